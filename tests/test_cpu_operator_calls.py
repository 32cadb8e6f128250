"""CPU: the host side of the operators' calls, the launches replaced by counters (no GPU here: nothing is launched)."""
import contextlib
import threading

import pytest
import torch
from torch.autograd import forward_ad

from pretrain_gnns_amd import _lib, ops


class _Counting:
    """the library as far as these tests go: workspaces of 1 KB, calls that convert their arguments and do nothing, counted by name"""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            kinds = _lib.PROTOTYPES[name][1]
            assert len(args) == len(kinds)
            for kind, value in zip(kinds, args):
                kind.from_param(value)
            if name.endswith("workspace_bytes"):
                return 1024
            self.calls.append(name)
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    """the calls' argument handling on CPU tensors"""
    lib = _Counting()
    monkeypatch.setattr(ops, "load", lambda: lib)
    monkeypatch.setattr(ops, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(ops, "stream_ptr", lambda *index: 0)
    monkeypatch.setattr(ops, "_ws_cache", {})
    monkeypatch.setattr(ops, "_ws_pool", {})
    monkeypatch.setattr(ops, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return lib


def _frozen_layer_norm(dim, **kw):
    return torch.nn.LayerNorm(dim, **kw).requires_grad_(False)


@pytest.mark.parametrize("kw", [{}, {"elementwise_affine": False}])
def test_layer_norm_drops_no_forward_tangent(lib, kw):
    """a tangent is refused as long as there is no rule for it, never dropped; a level without one changes nothing"""
    ln, x = _frozen_layer_norm(8, **kw), torch.randn(3, 8)
    with forward_ad.dual_level():
        assert forward_ad.unpack_dual(ops.layer_norm(x, ln)).tangent is None
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), pytest.raises(NotImplementedError, match="jvp"):
                ops.layer_norm(dual, ln)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ops.layer_norm(t, ln), (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("kw", [{}, {"bias": False}, {"elementwise_affine": False}])
def test_a_trace_of_layer_norm_holds_the_call(lib, kw):
    ln, x = _frozen_layer_norm(8, **kw), torch.randn(3, 8)
    traced = torch.jit.trace(lambda t: ops.layer_norm(t, ln, True), (x,), check_trace=False)
    assert "LayerNormReLU" in str(traced.graph)
    before = len(lib.calls)
    traced(torch.randn(5, 8))
    assert lib.calls[before:] == ["pgnn_layer_norm_fwd"]


def test_recorders_of_torch_calls_are_refused(lib):
    """they would keep the result's memory and not the launch that fills it"""
    from torch.fx.experimental.proxy_tensor import make_fx
    ln, x = _frozen_layer_norm(8), torch.randn(3, 8)
    for op in (lambda t: ops.layer_norm(t, ln), lambda t: ops.newton_schulz(t), lambda t: ops.newton_schulz([t, t])[1]):
        with pytest.raises(_lib.PgnnError, match="make_fx"):
            make_fx(op)(x)
    for op in (lambda t: ops.newton_schulz(t), lambda t: ops.newton_schulz([t, t])[1]):
        with pytest.raises(_lib.PgnnError, match="jit.trace"):
            torch.jit.trace(op, (x,), check_trace=False)
    assert not lib.calls
    ops.newton_schulz([x, x])
    assert lib.calls == ["pgnn_newton_schulz"]


def test_newton_schulz_drops_no_forward_tangent(lib):
    x = torch.randn(3, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for bad in (dual, [x, dual], dual * 2):
            with pytest.raises(NotImplementedError, match="tangent"):
                ops.newton_schulz(bad)
        assert not lib.calls
        ops.newton_schulz([x, x])
    ops.newton_schulz(x)
    assert lib.calls == ["pgnn_newton_schulz"] * 2


def test_every_host_thread_has_a_workspace_of_its_own(lib):
    """the launches of two threads' calls may alternate on one stream"""
    cpu = torch.device("cpu", 0)
    mine, others, both = ops._workspace(1000, cpu), [], threading.Barrier(2)

    def other():
        a = ops._workspace(1000, cpu)
        both.wait()  # (two threads that live at the same time)
        others.append((a, ops._workspace(1000, cpu)))

    threads = [threading.Thread(target=other) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({mine.data_ptr(), others[0][0].data_ptr(), others[1][0].data_ptr()}) == 3
    assert all(a.data_ptr() == b.data_ptr() for a, b in others) and ops._workspace(1000, cpu).data_ptr() == mine.data_ptr()


def test_muon_keeps_what_its_coefficients_were_made_for():
    """ns_steps beside coefficients for another number of steps would be read past their end"""
    from pretrain_gnns_amd import optim
    opt = object.__new__(optim.Muon)
    opt._steps, opt._eps, opt._adjust = 5, 1e-7, None
    assert (opt.ns_steps, opt.eps, opt.adjust_lr_fn) == (5, 1e-7, None)
    for name, value in (("ns_steps", 8), ("eps", 1.0), ("adjust_lr_fn", "match_rms_adamw")):
        with pytest.raises(AttributeError):
            setattr(opt, name, value)


def test_a_large_workspace_goes_back(lib):
    """what a call needs beyond the pool's size is not kept for the process"""
    cpu = torch.device("cpu", 0)
    small = ops._call_workspace(1 << 20, cpu)
    assert ops._call_workspace(1 << 20, cpu).data_ptr() == small.data_ptr()
    large = ops._call_workspace(100 << 20, cpu)
    assert large.numel() == 100 << 20
    assert sum(b.numel() for b in ops._ws_pool.values()) < 100 << 20
    assert ops._call_workspace(1 << 20, cpu).data_ptr() == small.data_ptr()


def test_use_layer_norm_leaves_frozen_gains_frozen():
    net = torch.nn.Sequential(torch.nn.BatchNorm1d(4), torch.nn.BatchNorm1d(4))
    net[0].weight.requires_grad_(False)
    net[1].bias.requires_grad_(False)
    ops.use_layer_norm(net)
    assert [p.requires_grad for p in net.parameters()] == [False, True, True, False]


def test_use_layer_norm_finds_every_batch_norm():
    """one that is in two places (and stays one), and the data-parallel form"""
    from pretrain_gnns_amd import parallel
    shared = torch.nn.BatchNorm1d(4)
    net = torch.nn.ModuleDict({"a": shared, "b": torch.nn.Sequential(torch.nn.Linear(4, 4), shared), "c": torch.nn.BatchNorm1d(4, affine=False)})
    ops.use_layer_norm(net)
    assert type(net["a"]) is torch.nn.LayerNorm and net["a"] is net["b"][1]
    assert type(net["c"]) is torch.nn.LayerNorm and net["c"].weight is None
    exact = parallel.use_exact_batchnorm(torch.nn.Sequential(torch.nn.BatchNorm1d(4)))
    assert type(ops.use_layer_norm(exact)[0]) is torch.nn.LayerNorm
