"""CPU: what the operators refuse, and their host-side rules (no GPU here: nothing is launched)."""
import pytest
import torch

from pretrain_gnns_amd import _lib, ops


def test_layer_norm_refusals():
    ln = torch.nn.LayerNorm(8)
    with pytest.raises(_lib.PgnnError, match="no CPU fallback"):
        ops.layer_norm(torch.zeros(2, 8), ln)
    lib = _lib.load()

    def fwd(rows, dim, xt=0, wt=0, x=4096, y=4096, ldx=None, ldy=None, mean=None, rstd=None):
        return lib.pgnn_layer_norm_fwd(x, dim if ldx is None else ldx, None, None, 1e-5, 0, y, dim if ldy is None else ldy, mean, rstd, rows, dim,
                                       xt, wt, None)

    assert fwd(0, 8) == 0                       # no rows: nothing to do
    assert fwd(2, 0) == 1 and fwd(-1, 8) == 1 and fwd(2, 1 << 30) == 1
    assert fwd(2, 8, xt=3) == 1 and fwd(2, 8, xt=0, wt=1) == 1 and fwd(2, 8, xt=1, wt=2) == 1
    assert fwd(2, 8, x=None) == 1 and fwd(2, 8, y=None) == 1
    assert fwd(2, 8, ldy=7) == 1 and fwd(2, 8, ldx=-1) == 1
    assert fwd(2, 8, mean=4096) == 1            # one statistic without the other
    assert b"layer_norm_fwd" in lib.pgnn_last_error()

    def bwd(rows, dim, dgamma=None, ws=None, ws_bytes=0, dy=4096, dx=4096, lddx=None, xt=0):
        return lib.pgnn_layer_norm_bwd(dy, dim, 4096, dim, None, None, 4096, 4096, 0, dx, dim if lddx is None else lddx, dgamma, None, rows, dim, xt, 0,
                                       ws, ws_bytes, None)

    assert bwd(0, 8) == 0 and bwd(5, 8, dx=None) == 0  # nothing asked for
    need = lib.pgnn_layer_norm_bwd_workspace_bytes(5, 8)
    assert need >= 2 * 8 * 4
    assert bwd(5, 8, dgamma=4096) == 3 and bwd(5, 8, dgamma=4096, ws=4096, ws_bytes=need - 1) == 3
    assert bwd(5, 8, dy=None) == 1 and bwd(5, 8, lddx=7) == 1 and bwd(5, 0) == 1 and bwd(5, 8, xt=-1) == 1
    assert lib.pgnn_layer_norm_bwd_workspace_bytes(-1, 8) == 0 and lib.pgnn_layer_norm_bwd_workspace_bytes(5, 0) == 0


def test_use_layer_norm_replaces_every_batch_norm():
    from pretrain_gnns_amd.bio import model as hbio
    from pretrain_gnns_amd.chem import model as hchem
    for net, count in ((hchem.GNN(3, 16), 3), (hbio.GNN(3, 16), 3), (hchem.GNN_graphpred(2, 16, 1), 2)):
        bns = {n: m for n, m in net.named_modules() if isinstance(m, torch.nn.BatchNorm1d)}
        assert len(bns) == count
        for m in bns.values():
            m.weight.data.uniform_(0.5, 1.5)
        net.eval()
        assert ops.use_layer_norm(net) is net
        lns = {n: m for n, m in net.named_modules() if isinstance(m, torch.nn.LayerNorm)}
        assert set(lns) == set(bns)
        for n, m in lns.items():
            assert m.eps == bns[n].eps and torch.equal(m.weight, bns[n].weight) and torch.equal(m.bias, bns[n].bias) and not m.training
        assert not any(isinstance(m, torch.nn.BatchNorm1d) for m in net.modules())
    with pytest.raises(_lib.PgnnError, match="no CPU fallback"):
        net(torch.zeros(1, 2, dtype=torch.long), torch.zeros(2, 0, dtype=torch.long), torch.zeros(0, 2, dtype=torch.long),
            torch.zeros(1, dtype=torch.long))


def _arrays(shapes):
    import ctypes
    n = len(shapes)
    return (ctypes.c_int64 * n)(*[r for r, _ in shapes]), (ctypes.c_int64 * n)(*[c for _, c in shapes]), n


def test_newton_schulz_refusals():
    import ctypes
    with pytest.raises(_lib.PgnnError, match="no CPU fallback"):
        ops.newton_schulz(torch.zeros(3, 4))
    lib = _lib.load()
    R, C, n = _arrays([(300, 600), (0, 7), (5, 4)])
    need = lib.pgnn_newton_schulz_workspace_bytes(R, C, n)
    assert need >= 4 * (2 * 600 * 320 + 2 * 300 * 320)  # X^T twice, A, B
    many = _arrays([(64, 64)] * 1000)
    assert lib.pgnn_newton_schulz_workspace_bytes(*many) < 60 * 100 * 1024  # taken in chunks
    for bad in ([(32769, 1)], [(1, 32769)], [(-1, 4)]):
        assert lib.pgnn_newton_schulz_workspace_bytes(*_arrays(bad)) == 0
    P = (ctypes.c_void_p * 3)(4096, 4096, 4096)
    L = (ctypes.c_int64 * 3)(600, 7, 4)

    def call(rows=R, cols=C, count=n, src=P, dst=P, ld=L, kind=0, coef=(3.4445, -4.775, 2.0315), steps=5, eps=1e-7, ws=None, ws_bytes=0):
        c = (ctypes.c_float * (3 * max(steps, 1)))(*(list(coef) * max(steps, 1)))
        return lib.pgnn_newton_schulz(src, ld, dst, rows, cols, count, kind, c, steps, eps, ws, ws_bytes, None)

    assert call() == 3 and call(ws=4096, ws_bytes=need - 1) == 3
    assert call(count=0) == 0 and call(*_arrays([(0, 7)])) == 0  # nothing to do
    assert call(kind=3) == 1 and call(steps=0) == 1 and call(steps=33) == 1
    assert call(eps=-1.0) == 1 and call(eps=float("nan")) == 1
    assert call(coef=(2.0, 2.0, 2.0)) == 1 and b"leaves every bound" in lib.pgnn_last_error()
    assert call(coef=(float("inf"), 0.0, 0.0)) == 1
    assert call(count=-1) == 1 and call(src=None) == 1 and call(dst=None) == 1 and call(rows=None) == 1
    assert call(src=(ctypes.c_void_p * 3)(None, 4096, 4096), ws=4096, ws_bytes=need) == 1
    assert call(ld=(ctypes.c_int64 * 3)(-1, 7, 4), ws=4096, ws_bytes=need) == 1
    rates = (ctypes.c_float * 3)(1.0, 1.0, 1.0)
    coef = (ctypes.c_float * 3)(1.5, -0.5, 0.0)

    def muon(params=P, momentum=P, ws=None, ws_bytes=0):
        return lib.pgnn_muon_step(params, P, momentum, rates, R, C, n, 0.95, 1, 1.0, coef, 1, 1e-7, ws, ws_bytes, None)

    assert muon() == 3 and muon(momentum=None) == 1
    assert muon(params=(ctypes.c_void_p * 3)(None, None, None), ws=4096, ws_bytes=need) == 1


def test_newton_schulz_coefficient_lists():
    make = ops._newton_schulz_coefficients
    assert list(make((1.5, -0.5, 0.0), 2)) == [1.5, -0.5, 0.0] * 2
    assert list(make([(1.5, -0.5, 0.0), (2, 0, 0)], 2)) == [1.5, -0.5, 0.0, 2, 0, 0]
    assert list(make([(1, 2, 3), (4, 5, 6), (7, 8, 9)], 3)) == [1, 2, 3, 4, 5, 6, 7, 8, 9]
    for bad in ([1, 2], [(1, 2, 3)] * 4, [(1, 2)] * 5):
        with pytest.raises(ValueError, match="coefficients"):
            make(bad, 5)


def test_muon_takes_gpu_matrices_only():
    from pretrain_gnns_amd import optim
    with pytest.raises(_lib.PgnnError, match="one GPU"):
        optim.Muon([torch.nn.Parameter(torch.zeros(3, 4))])
    with pytest.raises(ValueError, match="2-D"):
        optim.Muon([torch.nn.Parameter(torch.zeros(3))])
