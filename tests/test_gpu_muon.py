"""GPU: Newton-Schulz orthogonalisation (ops.newton_schulz) and the Muon step (optim.Muon) against their definitions in 64 bits.

Tolerance of the iteration: its operands are two fp16 planes (half a step of 2^-22 of the value where fp32 has 2^-24) and its sums are
fp32 like those of a plain fp32 product, whose accumulation over hundreds of terms outweighs the operands' rounding; a later step
magnifies what an earlier one lost (by up to |p'| = 3.9 with the usual coefficients), the same in both.  So in the Frobenius norm the
result may be 3 times as far from the 64-bit one as the same iteration in fp32 on the host, plus 2^-18 where the host's error happens to be
small (16 half steps of 2^-22), plus half a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
COEF = (3.4445, -4.7750, 2.0315)


def _ops():
    from pretrain_gnns_amd import ops
    return ops


def _iterate(g, coef=COEF, steps=5, eps=1e-7):
    """in g's own precision, on its device; the norm in 64 bits"""
    x = g / (g.double().norm() + eps).to(g.dtype) if g.dtype == torch.float64 else g * (1 / (g.double().norm() + eps)).to(g.dtype)
    tall = g.size(0) > g.size(1)
    x = x.t() if tall else x
    for t in range(steps):
        a, b, c = coef if not isinstance(coef[0], (tuple, list)) else coef[t]
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def _compare(got, g, **kw):
    want = _iterate(g.cpu().double(), **kw)
    host = _iterate(g.cpu().float(), **kw).double()
    scale = want.norm().item()
    tol = 3 * (host - want).norm().item() + 2.0 ** -18 * scale
    if got.dtype != torch.float32:
        tol += torch.finfo(got.dtype).eps / 2 * scale + 1e-7 * math.sqrt(want.numel())  # (fp16's subnormals: 2^-25)
    off = (got.cpu().double() - want).norm().item()
    assert off <= tol, "off by %.3g of %.3g, allowed %.3g" % (off, scale, tol)
    # no single value stands out: an error of all values together would be rms = off / sqrt(numel)
    worst = ((got.cpu().double() - want).abs() - (0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps) * want.abs()).max().item()
    assert worst <= max(64 * tol / math.sqrt(want.numel()), 1e-6), worst


def _matrix(rows, cols, seed=0, kind="gradient"):
    gen = torch.Generator().manual_seed(seed + 1000 * rows + cols)
    if kind == "gauss":
        return torch.randn(rows, cols, generator=gen)
    k = min(rows, cols)
    strength = torch.logspace(0, -2, k)
    return (torch.randn(rows, k, generator=gen) * strength) @ torch.randn(k, cols, generator=gen) + 0.1 * torch.randn(rows, cols, generator=gen)


SIZES = [(1, 1), (1, 7), (7, 1), (2, 3), (63, 65), (64, 64), (65, 63), (128, 1), (119, 300), (300, 119), (300, 600), (600, 300), (33, 1000),
         (257, 129), (900, 900)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_newton_schulz(rows, cols, dtype):
    g = _matrix(rows, cols).to(dtype)
    out = _ops().newton_schulz(g.to(DEV))
    assert out.shape == g.shape and out.dtype == dtype and out.is_contiguous()
    _compare(out, g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_newton_schulz_many_tiles(dtype):
    """enough tiles for the large-tile products: a batch, and one matrix"""
    ops = _ops()
    for g in (torch.stack([_matrix(700, 650, s) for s in range(16)]), torch.stack([_matrix(300, 1200, s) for s in range(60)])):
        g = g.to(dtype).to(DEV)
        out = ops.newton_schulz(g)
        assert out.shape == g.shape
        for b in (0, g.size(0) - 1):
            _compare(out[b], g[b])
        assert torch.equal(ops.newton_schulz(g), out)  # the same bits again
    one = _matrix(2900, 3001, 5).to(dtype).to(DEV)
    want = _iterate(one.double())
    rel = (_ops().newton_schulz(one).double() - want).norm() / want.norm()
    assert rel < (1e-5 if dtype == torch.float32 else 2.0 ** -8), rel  # half a step of bf16; fp32: 3 x what a product over 3000 terms loses


def test_newton_schulz_values_follow_the_polynomial():
    """the singular values are the scalar iteration's, the singular vectors stay"""
    gen = torch.Generator().manual_seed(0)
    u = torch.linalg.qr(torch.randn(40, 40, generator=gen, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(90, 40, generator=gen, dtype=torch.float64))[0]
    s = torch.logspace(0, -3, 40, dtype=torch.float64)
    g = ((u * s) @ v.t()).float()
    out = _ops().newton_schulz(g.to(DEV)).cpu().double()
    x = s / (s.norm() + 1e-7)
    for _ in range(5):
        x = x * (COEF[0] + x * x * (COEF[1] + x * x * COEF[2]))
    # fp32 rounds g by 2^-24 of its norm; the smallest singular value, 1e-3 of it, is magnified by up to 3.44^5 = 485: 485 * 2^-24 * sqrt(40)
    assert (out - (u * x) @ v.t()).abs().max().item() < 485 * 2.0 ** -24 * 40 ** 0.5


@pytest.mark.parametrize("coef,steps", [((2.0, -1.5, 0.5), 5), ((1.5, -0.5, 0.0), 12), (COEF, 1), (COEF, 32),
                                        ([(3.9, -6.0, 2.9), (3.4445, -4.775, 2.0315), (2.0, -1.5, 0.5)], 3), ((-1.875, 1.25, -0.375), 4)])
def test_newton_schulz_coefficients(coef, steps):
    for shape in ((70, 130), (130, 70)):
        g = _matrix(*shape)
        out = _ops().newton_schulz(g.to(DEV), steps=steps, coefficients=coef)
        if steps <= 12:
            _compare(out, g, coef=coef, steps=steps)
        else:  # the usual coefficients do not converge, they keep every value near 1: errors stay where they are after a few steps
            s = torch.linalg.svdvals(out.cpu().double())
            assert s.max() < 1.21 and s.min() > 0.6


def test_newton_schulz_lists_views_and_batches():
    ops = _ops()
    mats = [_matrix(r, c, i).to(DEV) for i, (r, c) in enumerate([(5, 9), (64, 64), (300, 17), (1, 1), (130, 260)] * 21)]  # three chunks of the job table
    mats.insert(2, torch.empty(0, 5, device=DEV))
    mats.insert(9, torch.empty(4, 0, device=DEV))
    outs = ops.newton_schulz(mats)
    assert [o.shape for o in outs] == [m.shape for m in mats]
    for i in (0, 1, 3, 4, 5, 6, 60, 106):
        assert torch.equal(outs[i], ops.newton_schulz(mats[i])), i  # alone or among others: the same bits
        if mats[i].numel():
            _compare(outs[i], mats[i])
    assert ops.newton_schulz([]) == []
    assert ops.newton_schulz(torch.empty(0, 3, 4, device=DEV)).shape == (0, 3, 4)
    g = _matrix(60, 100).to(DEV)
    want = ops.newton_schulz(g)
    wide = torch.full((60, 128), float("nan"), device=DEV)
    wide[:, 5:105] = g
    assert torch.equal(ops.newton_schulz(wide[:, 5:105]), want)        # a row stride of its own, rows that are not 16-byte aligned
    assert torch.equal(ops.newton_schulz(g.t().contiguous().t()), want)  # column major
    batch = torch.stack([g, 2 * g, -g]).view(3, 1, 60, 100)
    out = ops.newton_schulz(batch)
    assert out.shape == batch.shape and torch.equal(out[0, 0], want)
    # (-g gives -want up to rounding only: the f16 matrix instruction does not round its inner sums alike on both sides of zero)
    _compare(out[2, 0], -g)
    assert torch.equal(ops.newton_schulz(batch.transpose(0, 1)), out.transpose(0, 1))
    leaf = g.clone().requires_grad_(True)
    assert not ops.newton_schulz(leaf).requires_grad


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-9, 1e-7, 1.0, 1e18, 1e30])
def test_newton_schulz_of_any_size_of_gradient(scale):
    """norms far below eps, and ones whose square leaves fp32"""
    for shape in ((20, 30), (90, 65)):
        g = _matrix(*shape) * scale
        out = _ops().newton_schulz(g.to(DEV))
        want = _iterate(g.double())
        if scale < 1e-25:
            # X_0 = G / (|G| + 1e-7) is below 2^-60: under the range in which the planes keep their bits; it comes out as what is left, or 0
            assert out.isfinite().all() and (out.cpu().double() - want).abs().max().item() <= 2.0 ** -60
        else:
            rel = ((out.cpu().double() - want).norm() / want.norm()).item()
            assert rel < 2.0 ** -16, rel  # 5 steps that each lose 2^-22 and magnify what was lost by up to 3.9, to first order: in quadrature < 64 * 2^-22


@pytest.mark.parametrize("shape", [(20, 30), (90, 65)])
def test_newton_schulz_at_the_ends_of_the_types_range(shape):
    """a norm beyond fp32's largest number, whose inverse is below its smallest; subnormal values with eps = 0"""
    ops = _ops()
    for g, kw in ((_matrix(*shape).div(_matrix(*shape).abs().max()) * 3.3e38, {}), (_matrix(*shape) * 2.0 ** -140, {"eps": 0.0})):
        out = ops.newton_schulz(g.to(DEV), **kw)
        want = _iterate(g.double(), **kw)
        rel = ((out.cpu().double() - want).norm() / want.norm()).item()
        assert rel < 2.0 ** -16, rel  # (as in the test above)


# one tile more or one row more than a rule's limit: the one-launch form (64 x 384), the strips (320), and tiles that are formed in parts
# because they are few (700 x 650)
@pytest.mark.parametrize("rows,cols", [(64, 384), (385, 64), (65, 384), (320, 321), (321, 320), (384, 20), (700, 650), (520, 1030)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_newton_schulz_at_the_limits_of_its_rules(rows, cols, dtype):
    ops = _ops()
    g = _matrix(rows, cols).to(dtype)
    d = g.to(DEV)
    out = ops.newton_schulz(d)
    _compare(out, g)
    assert torch.equal(out, ops.newton_schulz(d))


@pytest.mark.parametrize("count,rows,cols,look", [(13, 330, 1100, (0, 5, 12)), (8, 1024, 1030, (0, 7)), (5, 1030, 900, (0, 4))])
def test_newton_schulz_left_over_tiles(count, rows, cols, look):
    """a few tiles more than compute units, in a graph as well: the parts' tickets are clear again behind every call"""
    ops = _ops()
    base = _matrix(rows, cols)
    gen = torch.Generator().manual_seed(5)
    g = torch.stack([base[torch.randperm(rows, generator=gen)] for _ in range(count)])  # (each matrix another one)
    d = g.to(DEV)
    out = ops.newton_schulz(d)
    for i in look:
        _compare(out[i], g[i])
    assert torch.equal(out, ops.newton_schulz(d))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ops.newton_schulz(d)
    for _ in range(3):
        again.zero_()
        graph.replay()
        eager = ops.newton_schulz(d)
        torch.cuda.synchronize()
        assert torch.equal(again, out) and torch.equal(eager, out)


def test_newton_schulz_beyond_32_bits():
    """planes of more than 2^31 bytes, one step, against fp32 products on the device"""
    rows, cols = 20011, 32768
    g = torch.randn(rows, cols, device=DEV).bfloat16()
    out = _ops().newton_schulz(g, steps=1)
    x = g.float()
    x *= (1 / (x.double().norm() + 1e-7)).float()
    gram = x @ x.t()
    b = torch.addmm(COEF[1] * gram, gram, gram, alpha=COEF[2])
    want = torch.addmm(x, b, x, beta=COEF[0])
    off = (out.float() - want).double().norm() / want.double().norm()
    assert off.item() <= 2.0 ** -8 + 2.0 ** -13  # half a step of bf16 per value; the fp32 products' own error is far below the second term


def test_newton_schulz_two_streams_at_once():
    """calls that overlap on two streams: each has its own workspace"""
    ops = _ops()
    a, b = _matrix(700, 650).to(DEV), _matrix(600, 800, 1).to(DEV)
    want = ops.newton_schulz(a), ops.newton_schulz(b)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for s, m in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                outs.append(ops.newton_schulz(m))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i & 1]) for i, o in enumerate(outs))


@pytest.mark.parametrize("shape", [(30, 40), (300, 100), (400, 500)])
def test_newton_schulz_in_place_at_the_c_entry(shape):
    import ctypes
    from pretrain_gnns_amd import _lib
    ops = _ops()
    for dtype in (torch.float32, torch.bfloat16):
        g = _matrix(*shape).to(dtype).to(DEV)
        want = ops.newton_schulz(g)
        lib = _lib.load()
        one = lambda v: (ctypes.c_int64 * 1)(v)
        R, C = one(shape[0]), one(shape[1])
        ws = torch.empty(lib.pgnn_newton_schulz_workspace_bytes(R, C, 1), dtype=torch.uint8, device=DEV)
        ptr = (ctypes.c_void_p * 1)(g.data_ptr())
        coef = (ctypes.c_float * 15)(*(COEF * 5))
        code = {torch.float32: 0, torch.bfloat16: 1}[dtype]
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.pgnn_newton_schulz(ptr, C, ptr, R, C, 1, code, coef, 5, 1e-7, ws.data_ptr(), ws.numel() - 1, stream) != 0  # too small
        assert lib.pgnn_newton_schulz(ptr, C, ptr, R, C, 1, code, coef, 5, 1e-7, ws.data_ptr(), ws.numel(), stream) == 0
        assert torch.equal(g, want)


def test_newton_schulz_zeros_and_bad_values():
    ops = _ops()
    z = torch.zeros(70, 90, device=DEV)
    assert not ops.newton_schulz(z).any() and not ops.newton_schulz(z, eps=1e-30).any()
    part = _matrix(70, 90).to(DEV)
    part[11] = 0.0
    out = ops.newton_schulz([part, part.t()])
    assert not out[0][11].any() and torch.equal(out[0].isfinite(), torch.ones_like(out[0], dtype=torch.bool))
    assert not out[1][:, 11].any()
    for bad in (float("nan"), float("inf"), float("-inf")):
        m = _matrix(70, 90).to(DEV)
        m[3, 4] = bad
        good = _matrix(30, 40).to(DEV)
        a, b = ops.newton_schulz([m, good])
        assert bool(a.isnan().all()) and torch.equal(b, ops.newton_schulz(good))


def test_newton_schulz_refusals():
    from pretrain_gnns_amd import _lib
    ops = _ops()
    g = torch.randn(4, 5, device=DEV)
    for bad in (0, 33):
        with pytest.raises(ValueError, match="steps"):
            ops.newton_schulz(g, steps=bad)
    with pytest.raises(ValueError, match="coefficients"):
        ops.newton_schulz(g, coefficients=[COEF] * 4)
    with pytest.raises(_lib.PgnnError, match="leaves every bound"):
        ops.newton_schulz(g, coefficients=(2.0, 2.0, 2.0))
    with pytest.raises(_lib.PgnnError, match="leaves every bound"):
        ops.newton_schulz(g, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(_lib.PgnnError, match="eps"):
        ops.newton_schulz(g, eps=-1.0)
    with pytest.raises(_lib.PgnnError, match="fp32, bf16 or fp16"):
        ops.newton_schulz(g.double())
    with pytest.raises(_lib.PgnnError, match="share type"):
        ops.newton_schulz([g, g.half()])
    with pytest.raises(ValueError, match="rows, cols"):
        ops.newton_schulz(g[0])
    with pytest.raises(_lib.PgnnError, match="32768"):
        ops.newton_schulz(torch.zeros(2, 32769, device=DEV))


def test_newton_schulz_streams_and_graphs():
    ops = _ops()
    g = [_matrix(119, 300).to(DEV), _matrix(600, 300).to(DEV)]
    want = ops.newton_schulz(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    static, graphs, outs = [t.clone() for t in g], [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.newton_schulz(static))
        graphs.append(gr)
    for k in range(3):
        for a, b in zip(static, g):
            a.copy_(b + 0.1 * k * b.abs())
        torch.cuda.synchronize()
        for gr in graphs:  # side by side on two streams: neither shares a workspace with the other or with the eager call
            with torch.cuda.stream(torch.cuda.Stream()):
                gr.replay()
        want = ops.newton_schulz(static)
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(want, o)), k


# ---------------------------------------------------------------------------------------------------------------- Muon
class _Oracle:
    """the step in 64 bits, and the bounds on the fp32 one's errors"""

    def __init__(self, params, **kw):
        self.kw = dict(lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, adjust_lr_fn=None)
        self.kw.update(kw)
        self.p = [p.detach().cpu().double().clone() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.slack = [torch.zeros_like(p) for p in self.p]

    def step(self, grads, **now):
        kw = dict(self.kw, **now)
        for i, g in enumerate(grads):
            if g is None:
                continue
            g = g.cpu().double()
            self.m[i] = kw["momentum"] * self.m[i] + g
            u = g + kw["momentum"] * self.m[i] if kw["nesterov"] else self.m[i]
            r, c = g.shape
            s = 0.2 * math.sqrt(max(r, c)) if kw["adjust_lr_fn"] else math.sqrt(max(1.0, r / c))
            o = _iterate(u)
            host = (_iterate(u.float()).double() - o).norm().item()
            self.p[i] = self.p[i] * (1 - kw["lr"] * kw["weight_decay"]) - kw["lr"] * s * o
            # a step: the direction's error (64 of its rms, see _compare), and three roundings of values up to |p| + lr s |o|
            step = kw["lr"] * s * (64 * (3 * host + 2.0 ** -18 * o.norm().item()) / math.sqrt(o.numel()) + 1e-6)
            self.slack[i] = self.slack[i] + step + 3 * 2.0 ** -24 * (self.p[i].abs() + kw["lr"] * s * o.abs())


SHAPES = [(600, 300), (300, 600), (119, 300), (4, 300), (1, 8), (9, 1), (64, 64)]


def _params(shapes=SHAPES, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=gen) / math.sqrt(s[1])).to(DEV)) for s in shapes]


@pytest.mark.parametrize("kw", [{}, {"nesterov": False, "lr": 0.02}, {"adjust_lr_fn": "match_rms_adamw", "weight_decay": 0.0},
                                {"momentum": 0.0, "lr": 0.1, "weight_decay": 1.0}])
def test_muon_steps(kw):
    from pretrain_gnns_amd import optim
    params = _params()
    opt = optim.Muon(params, **kw)
    ref = _Oracle(params, **kw)
    for t in range(4):
        opt.zero_grad()
        grads = [None if (t == 1 and i in (1, 4)) else _matrix(*p.shape, seed=t).to(DEV) * 1e-3 for i, p in enumerate(params)]
        for p, g in zip(params, grads):
            p.grad = g
        before = [g.clone() if g is not None else None for g in grads]
        if t == 2:  # a scheduler's hand
            opt.param_groups[0]["lr"] = 0.5 * float(opt.param_groups[0]["lr"])
        opt.step()
        ref.step(grads, lr=float(opt.param_groups[0]["lr"]))
        assert all(g is None or torch.equal(p.grad, g) for p, g in zip(params, before))
    for i, p in enumerate(params):
        m = opt.state[p]["momentum_buffer"]
        assert m.shape == p.shape
        # four fused multiply-adds: half a step each of values up to the largest so far
        assert ((m.cpu().double() - ref.m[i]).abs() <= 4 * 2.0 ** -24 * 4 * ref.m[i].abs().max()).all()
        off = (p.detach().cpu().double() - ref.p[i]).abs()
        assert (off <= ref.slack[i]).all(), (i, (off / ref.slack[i]).max().item())


@pytest.mark.parametrize("shapes", [[(3, 300), (64, 384), (1, 1)], [(6, 300), (300, 600), (400, 350), (119, 300), (1, 5)]])
def test_muon_lists_of_one_and_of_all_sizes(shapes):
    """a list that one launch takes, and one in which every kernel has a share"""
    from pretrain_gnns_amd import optim
    params = _params(shapes)
    opt = optim.Muon(params, lr=0.02)
    ref = _Oracle(params, lr=0.02)
    for t in range(3):
        grads = [_matrix(*p.shape, seed=t).to(DEV) for p in params]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        ref.step(grads)
    for i, p in enumerate(params):
        off = (p.detach().cpu().double() - ref.p[i]).abs()
        # the fp32 momentum differs from the oracle's in its last bit, and a direction magnifies that like any rounding of its input
        assert (off <= 2 * ref.slack[i]).all(), (i, (off / ref.slack[i]).max().item())


def test_muon_in_a_captured_step():
    from pretrain_gnns_amd import optim
    eager, captured = _params(), _params()
    a, b = optim.Muon(eager, lr=0.02), optim.Muon(captured, lr=0.02)
    grads = [_matrix(*p.shape).to(DEV) for p in captured]
    for p, g in zip(captured, grads):
        p.grad = g
    for p, g in zip(eager, grads):
        p.grad = g.clone()
    b.step()
    a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for t in range(3):
        for i, (p, g) in enumerate(zip(eager, grads)):
            new = _matrix(*p.shape, seed=10 + t).to(DEV)
            g.copy_(new)
            p.grad = new
        torch.cuda.synchronize()
        graph.replay()
        a.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, captured)), t
        assert all(torch.equal(a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"]) for p, q in zip(eager, captured))


def test_muon_refusals():
    from pretrain_gnns_amd import _lib, optim
    w = _params([(4, 5)])[0]
    with pytest.raises(ValueError, match="empty"):
        optim.Muon([])
    with pytest.raises(ValueError, match="2-D"):
        optim.Muon([w, torch.nn.Parameter(torch.zeros(4, device=DEV))])
    with pytest.raises(ValueError, match="twice"):
        optim.Muon([w, w])
    with pytest.raises(ValueError, match="adjust_lr_fn"):
        optim.Muon([w], adjust_lr_fn="other")
    with pytest.raises(ValueError, match="not negative"):
        optim.Muon([w], lr=-1.0)
    with pytest.raises(ValueError, match="steps"):
        optim.Muon([w], ns_steps=0)
    with pytest.raises(_lib.PgnnError, match="fp32"):
        optim.Muon([torch.nn.Parameter(torch.zeros(4, 5, device=DEV, dtype=torch.bfloat16))])
    with pytest.raises(_lib.PgnnError, match="contiguous"):
        optim.Muon([torch.nn.Parameter(torch.zeros(5, 4, device=DEV).t())])
    opt = optim.Muon([w])
    opt.step()  # nothing has a gradient: nothing happens
    assert not opt.state[w]["momentum_buffer"].any()
    w.grad = torch.ones(5, 4, device=DEV).t()
    with pytest.raises(_lib.PgnnError, match="contiguous fp32"):
        opt.step()
    opt.zero_grad()
    assert w.grad is None


def test_muon_looks_at_every_steps_tensors():
    """another gradient at the address of the last one, another momentum buffer"""
    from pretrain_gnns_amd import _lib, optim
    w = _params([(6, 6)])[0]
    opt = optim.Muon([w])
    w.grad = _matrix(6, 6).to(DEV)
    opt.step()
    before = w.detach().clone()
    w.grad = w.grad.t()  # same address
    with pytest.raises(_lib.PgnnError, match="contiguous fp32"):
        opt.step()
    w.grad = w.grad.t()
    for bad in (torch.zeros(6, 5, device=DEV), torch.zeros(6, 6, device=DEV, dtype=torch.float16), torch.zeros(6, 6)):
        opt.state[w]["momentum_buffer"] = bad
        with pytest.raises(_lib.PgnnError, match="momentum buffers"):
            opt.step()
    assert torch.equal(w, before)
    opt.state[w]["momentum_buffer"] = torch.zeros(6, 6, device=DEV)
    opt.step()
    assert not torch.equal(w, before)


def test_training_step_with_layer_norm_and_muon():
    """the masking step of a network with LayerNorms, its weights under Muon and the rest under Adam: the update is the definition's, from
    the gradients that the step left"""
    ops = _ops()
    from pretrain_gnns_amd import optim, train
    from pretrain_gnns_amd.chem import model as hmodel
    from pretrain_gnns_amd.data import synthetic
    torch.manual_seed(0)
    model = ops.use_layer_norm(hmodel.GNN(3, 100)).to(DEV)
    head, bonds = torch.nn.Linear(100, 119).to(DEV), torch.nn.Linear(100, 4).to(DEV)
    mods = [model, head, bonds]
    named = [(n, p) for m in mods for n, p in m.named_parameters()]
    weights = [p for n, p in named if p.dim() == 2 and "embedding" not in n]
    others = [p for _, p in named if all(p is not w for w in weights)]
    assert len(weights) == 3 * 2 + 2 and len(weights) + len(others) == len(named)
    opts = [optim.Muon(weights, lr=0.02), optim.Adam(others, lr=1e-3)]
    batch = synthetic.chem_masking_batch(16, seed=1)
    ref = _Oracle(weights, lr=0.02)
    for _ in range(3):
        before = [p.detach().clone() for p in others]
        loss = train.chem_masking_step(mods, opts, batch)[0]
        assert math.isfinite(loss)
        ref.step([p.grad for p in weights])
        assert any(not torch.equal(p, q) for p, q in zip(others, before))
    live = [i for i, p in enumerate(weights) if p.grad is not None]
    assert len(live) == 7  # the bond head has no part in this step
    for i in live:
        off = (weights[i].detach().cpu().double() - ref.p[i]).abs()
        # the fp32 momentum differs from the oracle's in its last bit, and a direction magnifies that like any rounding of its input
        assert (off <= 2 * ref.slack[i]).all(), i
