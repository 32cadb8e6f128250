"""GPU: sums of products whose rounding is part of the result, bit by bit.  In each pair one product is rounded to fp32 and the other is fused
onto it; which one has been the same in every build.  Rows of four columns, so that a sum is two pairs and nothing else (the other lanes
add zeros), against exact rational arithmetic rounded to nearest even where the hardware rounds."""
from fractions import Fraction

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _round(x):
    """a rational number to the nearest fp32, ties to even"""
    near = np.float32(float(x))
    best = [near, np.nextafter(near, np.float32(-np.inf)), np.nextafter(near, np.float32(np.inf))]
    return min(best, key=lambda v: (abs(Fraction(float(v)) - x), int(v.view(np.uint32)) & 1))


def _q(v):
    return Fraction(float(v))


def _pair(a, b, c, d):
    """a b on top of c d, which is rounded first"""
    return _q(_round(_q(a) * _q(b) + _q(_round(_q(c) * _q(d)))))


def _first_fused(v, w):
    return _round(_pair(v[0], w[0], v[1], w[1]) + _pair(v[2], w[2], v[3], w[3]))


def _second_fused(v, w):
    return _round(_pair(v[1], w[1], v[0], w[0]) + _pair(v[3], w[3], v[2], w[2]))


def _ends_rounded(v, w):
    return _round(_pair(v[1], w[1], v[0], w[0]) + _pair(v[2], w[2], v[3], w[3]))


def _normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def test_the_oracle_tells_the_orders_apart():
    v, w = _normal(50, 4, seed=1).numpy(), _normal(4, seed=2).numpy()
    forms = [[f(row, w) for row in v] for f in (_first_fused, _second_fused, _ends_rounded)]
    assert all(a != b for k, a in enumerate(forms) for b in forms[:k])


def test_gat_logits_and_their_gradients():
    from pretrain_gnns_amd import _lib, ops
    n, d, heads = 30, 4, 2
    gen = torch.Generator().manual_seed(0)
    edge_index = torch.randint(0, n, (2, 50), generator=gen).to(DEV)
    edge_attr = torch.stack([torch.randint(0, 4, (50,), generator=gen), torch.randint(0, 3, (50,), generator=gen)], 1).to(DEV)
    g = ops.build_chem_graph(edge_index, edge_attr, n)
    xh, att, gout = _normal(n, heads * d, seed=1), _normal(heads, 2 * d, seed=2), _normal(n, d, seed=3)
    zero = torch.zeros(6, heads * d, device=DEV), torch.zeros(3, heads * d, device=DEV)  # (the bond tables: m = xh + 0)
    dx, da, dg = xh.to(DEV), att.to(DEV), gout.to(DEV)
    ctab, bias = torch.zeros(18, heads, device=DEV), torch.zeros(d, device=DEV)
    new = lambda *s: torch.zeros(*s, device=DEV)
    scores, z, alpha, cfa, out = new(n, 2 * heads), new(g.e + n, heads), new(g.e + n, heads), new(heads, n, 9), new(n, d)
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()
    graph = (p(g.in_ptr), p(g.in_src), p(g.in_code))
    assert lib.pgnn_gat_fwd(p(dx), heads * d, *graph, p(zero[0]), p(zero[1]), p(ctab), None, None, None, 0, p(da), p(bias), 0.2, p(scores), p(z),
                            p(alpha), p(cfa), p(out), d, n, d, st) == 0
    x, a = xh.view(n, heads, d).numpy(), att.numpy()
    want = [[_first_fused(x[i, h], a[h, :d]) for h in range(heads)] + [_second_fused(x[i, h], a[h, d:]) for h in range(heads)] for i in range(n)]
    assert np.array_equal(scores.cpu().numpy(), np.array(want, dtype=np.float32))

    # an edge's weight gradient dalpha = g . m / 2.  The call hands out dz = alpha (dalpha - sum alpha dalpha): with every alpha 2^-60 the
    # second term is far below half a step of the first, and with z > 0 nothing else touches it
    z.fill_(1.0)
    alpha.fill_(2.0 ** -60)
    dz, dsd, czf, wout, dxh = new(g.e + n, heads), new(heads, n, 2), new(heads, n, 9), new(max(g.e, 1), heads), new(n, heads * d)
    assert lib.pgnn_gat_bwd(p(dg), d, p(dx), heads * d, *graph, p(g.out_ptr), p(g.out_dst), p(zero[0]), p(zero[1]), None, None, None, 0, p(da), 0.2,
                            p(z), p(alpha), p(dz), p(dsd), p(czf), p(wout), p(dxh), heads * d, n, d, st) == 0
    ptr, src, gn = g.in_ptr.tolist(), g.in_src.tolist(), gout.numpy()
    want = [[_ends_rounded(gn[i], x[src[q] if q < ptr[i + 1] else i, h]) / np.float32(2) for h in range(heads)]
            for i in range(n) for q in range(ptr[i], ptr[i + 1] + 1)]
    assert np.array_equal(dz.cpu().numpy() * np.float32(2.0 ** 60), np.array(want, dtype=np.float32))


def test_context_prediction_scores():
    from pretrain_gnns_amd import ops
    for seed in range(6):
        hs, hc = _normal(1, 4, seed=10 + seed), _normal(1, 4, seed=20 + seed)
        one = torch.zeros(1, dtype=torch.int64, device=DEV)
        _, vals = ops.contextpred_loss(hs.to(DEV), one, hc.to(DEV), one, one, 1)  # one graph: the pair and its negative are the same
        x = float(_second_fused(hs[0].numpy(), hc[0].numpy()))
        others = [float(f(hs[0].numpy(), hc[0].numpy())) for f in (_first_fused, _ends_rounded)]
        loss = lambda v: max(-v, 0.0) + np.log(np.exp(-max(-v, 0.0)) + np.exp(-v - max(-v, 0.0)))
        off = abs(vals[0].item() - loss(x))
        assert off <= 1e-14 * (1 + abs(x))  # float64, a few roundings
        for other in others:
            assert other == x or off < abs(vals[0].item() - loss(other))
