"""CPU: the host's own fp32 results that GPU tests compare with."""
import pytest
import torch

from conftest import HOST_THREADS


def _step(n, dim, relu, double):
    """the BatchNorm test's inputs, y and the gradients of x, weight and bias"""
    torch.manual_seed(n)
    bn = torch.nn.BatchNorm1d(dim)
    with torch.no_grad():
        bn.weight.uniform_(0.5, 1.5)
        bn.bias.uniform_(-0.5, 0.5)
    x, dtype = torch.randn(n, dim) * 2 + 3, torch.float64 if double else torch.float32
    gout = torch.randn(n, dim)
    bn, x = bn.to(dtype), x.to(dtype).requires_grad_(True)
    y = torch.relu(bn(x)) if relu else bn(x)
    y.backward(gout.to(dtype))
    return [y.detach(), x.grad, bn.weight.grad, bn.bias.grad]


@pytest.mark.parametrize("n,dim", [(777, 300), (5000, 600), (100, 32)])
@pytest.mark.parametrize("relu", [False, True])
def test_batchnorm_reference_is_near_64_bits(n, dim, relu):
    """within the tolerances that the GPU's result has around it, so that a right GPU result passes; with ReLU, a pre-activation on the wrong
    side of zero is another gradient"""
    before = torch.get_num_threads()
    torch.set_num_threads(HOST_THREADS)
    try:
        got, want = _step(n, dim, relu, False), _step(n, dim, relu, True)
    finally:
        torch.set_num_threads(before)
    for a, b, (rtol, atol) in zip(got, want, [(2e-5, 2e-5), (1e-4, 2e-5), (1e-4, 1e-4), (1e-4, 1e-4)]):
        torch.testing.assert_close(a.double(), b, rtol=0.7 * rtol, atol=0.7 * atol)
