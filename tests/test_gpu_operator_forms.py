"""GPU: sizes at which the operators' kernels take a form that small cases do not reach -- the products' tile sizes and groups of waves, small
matrices beside large ones, and more rows than a layer norm has lane groups, on both sides of the widths where it takes more lanes to a row.
Everything is compared with 64 bits on the device."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
COEF = (3.4445, -4.7750, 2.0315)
U = 2.0 ** -24


def _ops():
    from pretrain_gnns_amd import ops
    return ops


# ------------------------------------------------------------------------------------------------------------ Newton-Schulz
def _iterate(g, steps=5, eps=1e-7):
    """in g's own precision; the norm in 64 bits"""
    tall = g.size(0) > g.size(1)
    x = g.t().contiguous() if tall else g
    x = x * (1 / (x.double().norm() + eps)).to(x.dtype)
    a, b, c = COEF
    for _ in range(steps):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def _bound(g):
    """the 64-bit result, and how far off the kernels' may be in the Frobenius norm: their operands are two fp16 planes (22 bits where fp32 has
    24) under fp32 sums, so 3 times what the same iteration in fp32 loses, and 16 half steps of 2^-22 where that happens to be little"""
    want = _iterate(g.double())
    lost = (_iterate(g.float()).double() - want).norm().item()
    return want, 3 * lost + 2.0 ** -18 * want.norm().item()


def _check(got, g):
    want, tol = _bound(g)
    own = 0.0
    if got.dtype != torch.float32:  # half a step of the result's type, half its smallest subnormal
        own = torch.finfo(got.dtype).eps / 2
        tol += own * want.norm().item() + torch.finfo(got.dtype).smallest_normal * own * math.sqrt(want.numel())
    off = (got.double() - want).abs()
    assert off.norm().item() <= tol, (off.norm().item(), tol)
    # no single value stands out: if all were off alike, each would be by tol / sqrt(numel)
    assert (off - 2 * own * want.abs()).max().item() <= max(64 * tol / math.sqrt(want.numel()), 1e-6)


def _gradient(rows, cols, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + 1000 * rows + cols)
    k = min(rows, cols)
    left = torch.randn(rows, k, device=DEV, generator=gen) * torch.logspace(0, -2, k, device=DEV)
    return left @ torch.randn(k, cols, device=DEV, generator=gen) + 0.1 * torch.randn(rows, cols, device=DEV, generator=gen)


# On 256 compute units: X X^T and A A have the tiles on and above the diagonal of k x k, B X all tiles of k x n (k <= n)
FORMS = [
    (1200, 1203),  # B X 361 tiles of 64 (two groups of waves, two stages)
    (1500, 1490),  # B X 576 of 64 (three stages)
    (2301, 1111),  # B X 666 of 64, tall
    (1111, 2301),  # the same, wide
    (1800, 1777),  # B X 812 of 64 as 210 of 128 (two groups), X X^T 406 of 64
    (2048, 2048),  # B X 256 of 128: as many as compute units
    (2500, 2300),  # B X 360 of 128 (one group): 104 left over; X X^T 666 of 64
    (2620, 3001),  # X X^T 861 of 64 as 231 of 128 in two groups, B X 504 of 128
    (3100, 4001),  # X X^T 325 of 128: 69 left over, in parts
]


@pytest.mark.parametrize("rows,cols", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_newton_schulz_in_every_form(rows, cols, dtype):
    ops = _ops()
    g = _gradient(rows, cols).to(dtype)
    out = ops.newton_schulz(g)
    _check(out, g)
    assert torch.equal(out, ops.newton_schulz(g))


def test_newton_schulz_batches_in_every_form():
    """several matrices to a launch, left-over tiles of the first ones in parts"""
    ops = _ops()
    for count, rows, cols in ((3, 900, 1000), (5, 640, 1100), (6, 1030, 1100), (20, 400, 420)):
        g = torch.stack([_gradient(rows, cols, seed) for seed in range(count)])
        out = ops.newton_schulz(g)
        for i in (0, count // 2, count - 1):
            _check(out[i], g[i])
        assert torch.equal(out, ops.newton_schulz(g))


LARGE, SMALL = [(1024, 1030)] * 5, [(4, 300), (119, 300), (320, 500), (500, 320), (64, 64), (1, 9)]


@pytest.mark.parametrize("shapes", [SMALL + LARGE, LARGE + SMALL, SMALL[:3] + LARGE[:3] + SMALL[3:] + LARGE[3:]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_newton_schulz_small_matrices_apart_from_large_ones(shapes, dtype):
    """360 tiles of 128 at k > 320 leave no compute unit idle, so the small matrices' second halves go into launches of their own"""
    ops = _ops()
    mats = [_gradient(r, c, i).to(dtype) for i, (r, c) in enumerate(shapes)]
    outs = ops.newton_schulz(mats)
    for m, o in zip(mats, outs):
        _check(o, m)
    again = ops.newton_schulz(mats)
    assert all(torch.equal(a, b) for a, b in zip(outs, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.newton_schulz(mats)
    for _ in range(3):
        for c in captured:
            c.zero_()
        graph.replay()
        ops.newton_schulz(mats[:3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, captured))


def _muon_check(shapes, steps=2, lr=0.02, decay=0.1, mu=0.95):
    from pretrain_gnns_amd import optim
    gen = torch.Generator(device=DEV).manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=gen) / math.sqrt(s[1])) for s in shapes]
    opt = optim.Muon(params, lr=lr, weight_decay=decay, momentum=mu)
    want = [p.detach().double() for p in params]
    momenta, slack = [torch.zeros_like(p) for p in want], [torch.zeros_like(p) for p in want]
    for t in range(steps):
        for i, p in enumerate(params):
            p.grad = _gradient(*p.shape, seed=100 * t + i)
        opt.step()
        for i, p in enumerate(params):
            g = p.grad.double()
            momenta[i] = mu * momenta[i] + g
            o, tol = _bound((g + mu * momenta[i]).float())
            rate = lr * math.sqrt(max(1.0, p.size(0) / p.size(1)))
            want[i] = want[i] * (1 - lr * decay) - rate * o
            # the direction's error, 64 of its rms for a single value, and three roundings of values up to |p| + rate |o|
            slack[i] += rate * (64 * tol / math.sqrt(o.numel()) + 1e-6) + 3 * U * (want[i].abs() + rate * o.abs())
    for i, p in enumerate(params):
        off = (p.detach().double() - want[i]).abs()
        # twice: the fp32 momentum differs from the 64-bit one in its last bit, and a direction magnifies that like any rounding of its input
        assert (off <= 2 * slack[i]).all(), (shapes[i], (off / slack[i]).max().item())
        m = opt.state[p]["momentum_buffer"].double()
        # one fused multiply-add per step, half a step of values up to the largest
        assert (m - momenta[i]).abs().max().item() <= 2 * steps * U * momenta[i].abs().max().item()


@pytest.mark.parametrize("shape", [(1203, 1200), (1490, 1500), (1111, 2301), (1800, 1777), (2500, 2300)])
def test_muon_in_every_form(shape):
    _muon_check([shape])


@pytest.mark.parametrize("shapes", [SMALL + LARGE, LARGE[:4] + SMALL + LARGE[4:]])
def test_muon_small_matrices_apart_from_large_ones(shapes):
    _muon_check(shapes)


@pytest.mark.parametrize("rows,cols", [(40, 300), (200, 400), (400, 500), (400, 200)])
@pytest.mark.parametrize("low", [1e-3, 1e-6])
def test_newton_schulz_of_graded_rows(rows, cols, low):
    """row by row (column by column of a tall matrix) what the planes promise: beside what fp32 products lose, every entry of X, A and B is
    off by up to 2^-37 of its bound, u <= 1.21, u^2 and 2.81.  Of a weak row, which grows by 3.4445 a step, a step adds 2^-37 (sqrt(n) u +
    sqrt(k) (4.775 u^3 + 2 * 2.0315 u^5 + 2.81 u)) at most, and a step's share grows as the row does: 1 / (1 - 1 / 3.4445) = 1.41 of the first's"""
    g = torch.randn(rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    k, n = min(rows, cols), max(rows, cols)
    grade = torch.logspace(0, math.log10(low), k, device=DEV)
    g = g * (grade[:, None] if rows <= cols else grade)
    out, want, host = _ops().newton_schulz(g).double(), _iterate(g.double()), _iterate(g).double()
    axis = 1 if rows <= cols else 0
    u = 1.21
    planes = 1.41 * 3.4445 ** 5 * 2.0 ** -37 * (math.sqrt(n) * u + math.sqrt(k) * (4.775 * u ** 3 + 2 * 2.0315 * u ** 5 + 2.81 * u))
    off, size = (out - want).norm(dim=axis), want.norm(dim=axis)
    assert (off <= 3 * (host - want).norm(dim=axis) + 2.0 ** -18 * size + planes).all()
    assert (out - want).norm().item() <= 3 * (host - want).norm().item() + 2.0 ** -18 * want.norm().item()  # and in the norm without that
    if low == 1e-3:
        assert (off / size).max().item() <= 2.0 ** -14  # (2^-10 of the largest: still within the planes' 22 bits)


# ------------------------------------------------------------------------------------------------------------ layer norm
def _layer_norm_check(rows, dim, dtype, gains, relu, seed=0):
    """per element, as the roundings of the arithmetic bound it.  A row's mean: at most 32 values in a lane and 12 partial sums, off by
    45 u max|x|, which moves the centred values and through the variance r = 1 / sqrt(var + eps); so xh is off by e = (1 + |xh|) 45 u max|x| r +
    30 u |xh|.  A gain's gradient: the rows of a lane group one after the other, with at least 256 groups from 8 192 rows on (and one or two
    rows each below), then the groups of a workgroup, then float64"""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(seed + rows + dim)
    normal = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    ln = torch.nn.LayerNorm(dim, device=DEV, dtype=gains)
    with torch.no_grad():
        ln.weight.copy_(1 + 0.3 * normal(dim))
        ln.bias.copy_(0.3 * normal(dim))
    x = (normal(rows, dim) * (0.3 + normal(rows, 1).abs()) + normal(dim)).to(dtype)
    dy = normal(rows, dim).to(dtype)
    xd, w, b = x.double(), ln.weight.detach().double(), ln.bias.detach().double()
    mean = xd.mean(1, keepdim=True)
    r = 1 / torch.sqrt((xd - mean).square().mean(1, keepdim=True) + ln.eps)
    xh = (xd - mean) * r
    pre = xh * w + b
    if relu:  # the mask of a pre-activation next to zero is a rounding question: no gradient flows through those
        dy = torch.where(pre.abs() < 1e-2, torch.zeros_like(dy), dy)
    y = pre.clamp(min=0) if relu else pre
    e = (1 + xh.abs()) * 45 * U * xd.abs().amax(1, keepdim=True) * r + 30 * U * xh.abs()
    h = dy.double() * (pre > 0) if relu else dy.double()
    g = h * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - m1 - xh * m2)
    dm1 = 50 * U * g.abs().mean(1, keepdim=True)
    dm2 = (g.abs() * e).mean(1, keepdim=True) + 50 * U * (g * xh).abs().mean(1, keepdim=True)
    dr = 45 * U * xd.abs().amax(1, keepdim=True) * r + 30 * U
    chain = rows / 256 + 16
    tols = [w.abs() * e + 4 * U * (pre.abs() + b.abs()),
            r * (dm1 + xh.abs() * dm2 + m2.abs() * e + 6 * U * (g.abs() + m1.abs() + (xh * m2).abs())) + dr * dx.abs(),
            (h.abs() * e).sum(0) + chain * U * (h * xh).abs().sum(0), chain * U * h.abs().sum(0)]
    wants = [y, dx, (h * xh).sum(0), h.sum(0)]
    x.requires_grad_(True)
    out = ops.layer_norm(x, ln, relu)
    got = [out] + list(torch.autograd.grad(out, (x, ln.weight, ln.bias), dy))
    for name, a, want, tol in zip(("y", "dx", "dgamma", "dbeta"), got, wants, tols):
        if a.dtype != torch.float32:
            half = torch.finfo(a.dtype).eps / 2
            tol = tol + half * (want.abs() + tol) + torch.finfo(a.dtype).smallest_normal * half
        over = ((a.detach().double() - want).abs() - tol).max().item()
        assert over <= 0, "%s: %.3g over its bound" % (name, over)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, ln, relu), out)


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# more rows than the launches have lane groups: 32 768 and 8 192 on 16 lanes (forward, backward), 8 192 and 2 048 on 64, 2 048 and 512 (256
# beyond 4 096 columns) on 256, 512 beyond 8 192 columns
@pytest.mark.parametrize("rows,dim,dtype,gains", [(70001, 300, F32, F32), (70001, 100, F16, F16), (20003, 400, BF16, F32), (20003, 1001, F32, F32),
                                                 (5001, 2049, F32, F32), (5001, 4096, BF16, F32), (5003, 6001, F16, F16), (1501, 8200, F32, F32),
                                                 (1501, 8200, BF16, BF16)])
@pytest.mark.parametrize("relu", [False, True])
def test_layer_norm_of_more_rows_than_lane_groups(rows, dim, dtype, gains, relu):
    _layer_norm_check(rows, dim, dtype, gains, relu)


@pytest.mark.parametrize("dim", [448, 449, 1792, 1793, 4096, 4097, 8192, 8193])
def test_layer_norm_at_the_limits_of_its_lanes_fp32(dim):
    _layer_norm_check(4500, dim, F32, F32, False)


@pytest.mark.parametrize("dim", [384, 385, 416, 448, 449, 1536, 1537, 1793, 4096, 4097, 8192, 8193])
@pytest.mark.parametrize("dtype,gains", [(BF16, F32), (F16, F16)])
def test_layer_norm_at_the_limits_of_its_lanes_16_bit(dim, dtype, gains):
    _layer_norm_check(4500, dim, dtype, gains, False)
