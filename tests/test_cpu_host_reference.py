"""CPU: the host's own fp32 results that GPU tests compare with."""
import pytest
import torch

from conftest import HOST_THREADS


@pytest.mark.parametrize("n,dim", [(777, 300), (5000, 600), (100, 32)])
def test_batchnorm_reference_has_the_signs_of_64_bits(n, dim):
    """the inputs of the GPU's BatchNorm test: with ReLU behind it, a pre-activation on the wrong side of zero is another gradient"""
    torch.manual_seed(n)
    bn = torch.nn.BatchNorm1d(dim)
    with torch.no_grad():
        bn.weight.uniform_(0.5, 1.5)
        bn.bias.uniform_(-0.5, 0.5)
    x = torch.randn(n, dim) * 2 + 3
    exact = torch.nn.BatchNorm1d(dim).double()
    exact.load_state_dict(bn.state_dict())
    before = torch.get_num_threads()
    torch.set_num_threads(HOST_THREADS)
    try:
        got = bn(x)
    finally:
        torch.set_num_threads(before)
    assert torch.equal(got > 0, exact(x.double()) > 0)
