"""GPU: calls of the operators that go through torch's other machinery (traces, threads, other streams)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    from pretrain_gnns_amd import ops
    return ops


@pytest.mark.parametrize("shape", [(5, 300), (2, 3, 300)])
def test_a_trace_of_layer_norm_gives_the_values(shape):
    ops = _ops()
    ln = torch.nn.LayerNorm(300, device=DEV).requires_grad_(False)
    ln.weight.uniform_(0.5, 1.5)
    ln.bias.uniform_(-0.5, 0.5)
    traced = torch.jit.trace(lambda t: ops.layer_norm(t, ln, True) * 2, (torch.randn(shape, device=DEV),), check_trace=False)
    for _ in range(3):
        x = torch.randn(shape, device=DEV)
        junk = torch.full_like(x, float("nan"))  # what a result that nobody writes would be made of
        del junk
        assert torch.equal(traced(x), ops.layer_norm(x, ln, True) * 2)
