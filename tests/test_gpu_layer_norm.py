"""GPU: layer normalisation (csrc/layernorm.hip through ops.layer_norm) against its definition in 64 bits.

Tolerances are bounds on the rounding error of the arithmetic, evaluated per element (u = 2^-24, half a step of fp32):
a row's mean is a sum of at most 32 values per lane and 8 + 4 partial sums, so it is off by <= 45 u max|x|; that moves the centred
values, and through the variance 1 / sqrt(var + eps), so xh is off by e = (1 + |xh|) 45 u max|x| r + 30 u |xh|.  Rounding to the output's
type adds half a step of that type (torch.finfo(t).eps / 2 of the value, and half the smallest subnormal)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _ops():
    from pretrain_gnns_amd import ops
    return ops


def _half_step(value, dtype):
    if dtype == torch.float32:
        return 0 * value
    return value.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _oracle(x, w, b, eps, relu, dy=None):
    """y, dx, dgamma, dbeta in 64 bits and the bounds on their errors, from inputs on the CPU"""
    x, w, b = x.double(), w.double(), b.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    xh = (x - mean) * r
    pre = xh * w + b
    y = pre.clamp(min=0) if relu else pre
    e = (1 + xh.abs()) * 45 * U * x.abs().amax(1, keepdim=True) * r + 30 * U * xh.abs()
    out, tol = [y], [w.abs() * e + 4 * U * (pre.abs() + b.abs())]
    if dy is not None:
        h = dy.double() * (pre > 0) if relu else dy.double()
        g = h * w
        m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        dx = r * (g - m1 - xh * m2)
        dm1 = 50 * U * g.abs().mean(1, keepdim=True)
        dm2 = (g.abs() * e).mean(1, keepdim=True) + 50 * U * (g * xh).abs().mean(1, keepdim=True)
        dr = 45 * U * x.abs().amax(1, keepdim=True) * r + 30 * U  # relative error of r
        out += [dx, (h * xh).sum(0), h.sum(0)]
        # at most 300 additions in a lane's chain (the sizes here), then float64
        tol += [r * (dm1 + xh.abs() * dm2 + m2.abs() * e + 6 * U * (g.abs() + m1.abs() + (xh * m2).abs())) + dr * dx.abs(),
                (h.abs() * e).sum(0) + 300 * U * (h * xh).abs().sum(0), 300 * U * h.abs().sum(0)]
    return out, tol


def _near(got, want, tol, what):
    got = got.detach().double().cpu().reshape(want.shape)
    bound = tol + _half_step(want.abs() + tol, what[1])
    worst = ((got - want).abs() - bound).max().item() if want.numel() else -1.0
    assert worst <= 0, "%s: %.3g over its bound" % (what[0], worst)


def _module(shape, dtype, gain=True, bias=True, eps=1e-5, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ln = torch.nn.LayerNorm(shape, eps=eps, elementwise_affine=gain, bias=bias, device=DEV, dtype=dtype)
    with torch.no_grad():
        for p in (ln.weight, ln.bias):
            if p is not None:
                p.copy_((torch.randn(p.shape, generator=gen) * 0.3 + (p is ln.weight)).to(dtype))
    return ln


def _rows(rows, dim, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed + 17)
    x = torch.randn(rows, dim, generator=gen) * (0.3 + torch.rand(rows, 1, generator=gen)) + torch.randn(dim, generator=gen)
    return x.to(dtype), torch.randn(rows, dim, generator=gen).to(dtype)


def _check(x, dy, ln, relu, names="x"):
    """x, dy: [rows, dim] on the CPU"""
    ops = _ops()
    w = ln.weight.detach().cpu().reshape(-1) if ln.weight is not None else torch.ones(x.size(1))
    b = ln.bias.detach().cpu().reshape(-1) if ln.bias is not None else torch.zeros(x.size(1))
    if relu:  # the mask of a pre-activation next to zero is a rounding question: no gradient flows through those
        (pre,), _ = _oracle(x, w, b, ln.eps, False)
        dy = torch.where(pre.abs() < 1e-2, torch.zeros_like(dy), dy)
    want, tol = _oracle(x, w, b, ln.eps, relu, dy)
    xd = x.to(DEV).requires_grad_(True)
    y = ops.layer_norm(xd, ln, relu)
    assert y.dtype == x.dtype and y.shape == x.shape
    leaves = [xd] + [p for p in (ln.weight, ln.bias) if p is not None]
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    _near(y, want[0], tol[0], ("y", x.dtype))
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(xd, ln, relu), y)  # inference: the same arithmetic, nothing saved
    _near(grads[0], want[1], tol[1], ("dx", x.dtype))
    for p, g in zip(leaves[1:], grads[1:]):
        assert g.dtype == p.dtype
        k = 2 if p is ln.weight else 3
        _near(g, want[k], tol[k], ("dgamma" if k == 2 else "dbeta", p.dtype))


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
         (torch.float16, torch.float16)]
SHAPES = [(1, 1), (3, 2), (5, 7), (24, 300), (777, 300), (64, 301), (1030, 64), (130, 512), (130, 513), (33, 1023), (9, 2048), (9, 2049),
          (2, 4096), (3, 8192), (3, 8193), (2, 20001), (4500, 300)]


@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "%s-%s" % tuple(str(k)[6:] for k in t))
def test_layer_norm_forward_backward(rows, dim, types):
    ln = _module(dim, types[1], seed=rows + dim)
    x, dy = _rows(rows, dim, types[0], seed=rows)
    _check(x, dy, ln, relu=False)


@pytest.mark.parametrize("rows,dim", [(24, 300), (65, 301), (130, 1100), (7, 5000), (5, 9000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_norm_with_relu(rows, dim, dtype):
    ln = _module(dim, torch.float32, seed=3)
    x, dy = _rows(rows, dim, dtype, seed=4)
    _check(x, dy, ln, relu=True)


@pytest.mark.parametrize("gain,bias", [(True, False), (False, False)])
@pytest.mark.parametrize("dim", [30, 600, 3001, 8200])
def test_layer_norm_without_gains(dim, gain, bias):
    ln = _module(dim, torch.float32, gain, bias)
    x, dy = _rows(11, dim, torch.bfloat16)
    _check(x, dy, ln, relu=False)


def test_layer_norm_views_and_trailing_axes():
    ops = _ops()
    ln = _module((5, 60), torch.float32)
    flat = _module(300, torch.float32)
    with torch.no_grad():
        flat.weight.copy_(ln.weight.reshape(-1))
        flat.bias.copy_(ln.bias.reshape(-1))
    x, dy = _rows(24, 300, torch.float32)
    x, dy = x.to(DEV), dy.to(DEV)
    want = ops.layer_norm(x, flat)
    assert torch.equal(ops.layer_norm(x.view(4, 6, 5, 60), ln), want.view(4, 6, 5, 60))
    wide = torch.full((24, 311), float("nan"), device=DEV)  # columns of a wider buffer: what lies beside them is not read
    wide[:, 3:303] = x
    view = wide[:, 3:303].requires_grad_(True)
    got = ops.layer_norm(view, flat)
    assert torch.equal(got, want)
    (dx,) = torch.autograd.grad(got, view, dy)
    xl = x.clone().requires_grad_(True)
    (dx_want,) = torch.autograd.grad(ops.layer_norm(xl, flat), xl, dy)
    assert torch.equal(dx, dx_want) and dx.is_contiguous()
    t = x.t().contiguous().t().requires_grad_(True)  # column major
    assert torch.equal(ops.layer_norm(t, flat), want)
    # a gradient that is one value for all (sum) and one that is a row for all (expand)
    (a,) = torch.autograd.grad(ops.layer_norm(xl, flat).sum(), xl)
    (b,) = torch.autograd.grad(ops.layer_norm(xl, flat), xl, torch.ones_like(x))
    assert torch.equal(a, b)
    (a,) = torch.autograd.grad(ops.layer_norm(xl, flat), xl, dy[0].expand(24, 300))
    (b,) = torch.autograd.grad(ops.layer_norm(xl, flat), xl, dy[0].repeat(24, 1))
    assert torch.equal(a, b)
    one = x[3].clone()  # no leading axis at all
    assert torch.equal(ops.layer_norm(one, flat), want[3])
    same = x[:1].expand(24, 300)  # a row stride of zero
    assert torch.equal(ops.layer_norm(same, flat), want[:1].expand(24, 300))


def test_layer_norm_of_no_rows():
    ops = _ops()
    for dim in (300, 9000):
        ln = _module(dim, torch.float32)
        x = torch.empty(0, dim, device=DEV, requires_grad=True)
        y = ops.layer_norm(x, ln)
        assert y.shape == (0, dim)
        dx, dw, db = torch.autograd.grad(y, (x, ln.weight, ln.bias), torch.empty(0, dim, device=DEV))
        assert dx.shape == (0, dim) and not dw.any() and not db.any()


@pytest.mark.parametrize("dim", [300, 1500, 4000, 9000])
def test_layer_norm_keeps_bad_rows_apart(dim):
    ops = _ops()
    ln = _module(dim, torch.float32)
    x, dy = _rows(6, dim, torch.float32)
    clean = ops.layer_norm(x.to(DEV), ln)
    bad = x.clone()
    bad[1, 5], bad[3, dim - 1], bad[4, 0] = float("nan"), float("inf"), float("-inf")
    bad = bad.to(DEV).requires_grad_(True)
    y = ops.layer_norm(bad, ln, relu=True)
    rows = torch.tensor([0, 2, 5], device=DEV)
    assert torch.equal(y[rows], clean[rows].clamp(min=0)) and bool(y[[1, 3, 4]].isnan().all())
    (dx,) = torch.autograd.grad(y, bad, dy.to(DEV))
    assert bool(dx[rows].isfinite().all()) and bool(dx[[1, 3, 4]].isnan().any(1).all())


def test_layer_norm_constant_and_large_offset_rows():
    ln = _module(300, torch.float32)
    x, dy = _rows(4, 300, torch.float32)
    x[0] = 7.25          # no variance: eps alone under the root
    x[1] = 0.0
    x[2] += 3.0e4        # the mean is 3e4 standard deviations away
    _check(x, dy, ln, relu=False)


def test_layer_norm_gradient_against_differences():
    ops = _ops()
    dim, rows = 37, 5
    ln = _module(dim, torch.float32)
    x, dy = _rows(rows, dim, torch.float32)
    xd = x.to(DEV).requires_grad_(True)
    grads = torch.autograd.grad(ops.layer_norm(xd, ln), (xd, ln.weight, ln.bias), dy.to(DEV))
    at = [x.double(), ln.weight.detach().cpu().double(), ln.bias.detach().cpu().double()]
    f = lambda p: (_oracle(p[0], p[1], p[2], ln.eps, False)[0][0] * dy.double()).sum()
    gen = torch.Generator().manual_seed(1)
    for k, g in enumerate(grads):
        for _ in range(3):
            d = torch.randn(at[k].shape, generator=gen, dtype=torch.float64)
            step = 1e-5
            up, down = [t.clone() for t in at], [t.clone() for t in at]
            up[k] += step * d
            down[k] -= step * d
            diff = ((f(up) - f(down)) / (2 * step)).item()
            got = (g.double().cpu() * d).sum().item()
            # differences: step^2 times a third derivative of order 10 per value; the gradient: fp32, dim * rows terms
            assert abs(got - diff) <= 1e-6 * (g.double().cpu() * d).abs().sum().item() + 1e-7, (k, got, diff)


def test_layer_norm_only_what_is_asked_for():
    ops = _ops()
    ln = _module(300, torch.float32)
    x, dy = _rows(50, 300, torch.float32)
    xd = x.to(DEV).requires_grad_(True)
    full = torch.autograd.grad(ops.layer_norm(xd, ln), (xd, ln.weight, ln.bias), dy.to(DEV))
    ln.weight.requires_grad_(False)
    part = torch.autograd.grad(ops.layer_norm(xd, ln), (xd, ln.bias), dy.to(DEV))
    assert torch.equal(part[0], full[0]) and torch.equal(part[1], full[2])
    ln.weight.requires_grad_(True)
    only = torch.autograd.grad(ops.layer_norm(x.to(DEV), ln), (ln.weight, ln.bias), dy.to(DEV))
    assert torch.equal(only[0], full[1]) and torch.equal(only[1], full[2])
    ln.weight.requires_grad_(False)
    ln.bias.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(ops.layer_norm(xd, ln), xd, dy.to(DEV))[0], full[0])


def test_layer_norm_has_no_second_derivative():
    """a graph of the backward may be asked for; its use is refused, whatever the first gradient came from"""
    ops = _ops()
    ln = _module(30, torch.float32)
    x, dy = _rows(5, 30, torch.float32)
    x, dy = x.to(DEV).requires_grad_(True), dy.to(DEV)
    want = torch.autograd.grad(ops.layer_norm(x, ln), (x, ln.weight, ln.bias), dy)
    got = torch.autograd.grad(ops.layer_norm(x, ln), (x, ln.weight, ln.bias), dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    only, = torch.autograd.grad(ops.layer_norm(x, ln), ln.bias, dy, create_graph=True)
    for loss in (got[0].square().sum(), got[1].sum() + x.sum(), only.sum()):
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            loss.backward()
    y = ops.layer_norm(x, ln)
    g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        (y.sum() + g.sum()).backward()


def test_layer_norm_beyond_32_bits():
    """more than 2^31 values, dense and as rows far apart: the last rows as they come out of a small call"""
    ops = _ops()
    rows, dim = 2 ** 21 + 3, 1025
    ln = _module(dim, torch.float16)
    x = torch.zeros(rows, dim, dtype=torch.float16, device=DEV)
    dy = torch.zeros_like(x)
    few, dfew = _rows(8, dim, torch.float16)
    few, dfew = few.to(DEV), dfew.to(DEV)
    x[-8:], dy[-8:] = few, dfew
    x.requires_grad_(True)
    y = ops.layer_norm(x, ln)
    got = torch.autograd.grad(y, (x, ln.weight, ln.bias), dy)
    fl = few.clone().requires_grad_(True)
    want_y = ops.layer_norm(fl, ln)
    want = torch.autograd.grad(want_y, (fl, ln.weight, ln.bias), dfew)
    assert torch.equal(y[-8:], want_y) and torch.equal(got[0][-8:], want[0])
    assert torch.equal(y[0], ln.bias) and not got[0][:-8].any()
    # the same eight terms however they are grouped: twice 8 half steps of fp32 of their sum, at most 8 max|dy| sqrt(dim) (|xh| <= 32.02), which
    # is 2^-11.9 max|dy|, and two roundings to fp16
    for a, b in zip(got[1:], want[1:]):
        assert ((a.float() - b.float()).abs() <= torch.finfo(torch.float16).eps * b.float().abs() + 2.0 ** -11 * dfew.float().abs().max()).all()
    del x, y, dy, got
    wide = torch.zeros(1100, 2000003, dtype=torch.float16, device=DEV)
    part = wide[:, 7:7 + dim]
    part[-8:] = few
    assert torch.equal(ops.layer_norm(part, ln)[-8:].detach(), want_y.detach())


def test_layer_norm_streams_and_graphs():
    ops = _ops()
    ln = _module(300, torch.float32)
    x, dy = _rows(3000, 300, torch.float32)
    x, dy = x.to(DEV), dy.to(DEV)

    def step(x):
        xl = x.detach().requires_grad_(True)
        y = ops.layer_norm(xl, ln, relu=False)
        return (y.detach(),) + torch.autograd.grad(y, (xl, ln.weight, ln.bias), dy)

    want = step(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step(x)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    static, graphs, outs = x.clone(), [], []
    for _ in range(2):  # two graphs that may be replayed side by side: neither shares a workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(static))
        graphs.append(g)
    for k in range(3):
        new = x * (1 + k) + k
        static.copy_(new)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        want = step(new)
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(want, o)), k


@pytest.mark.parametrize("gnn_type", ["gin", "gcn", "graphsage", "gat"])
def test_networks_with_layer_norm(gnn_type):
    """the chem and bio networks with their BatchNorms replaced, against the oracle's with the same replacement"""
    ops = _ops()
    from oracle import bio as obio
    from oracle import chem as ochem
    from pretrain_gnns_amd.bio import model as hbio
    from pretrain_gnns_amd.chem import model as hchem
    from pretrain_gnns_amd.data import synthetic
    for omod, hmod, batch in ((ochem, hchem, synthetic.chem_plain_batch(8, seed=1)), (obio, hbio, synthetic.bio_masking_batch(4, seed=1))):
        torch.manual_seed(0)
        ref = ops.use_layer_norm(omod.GNN(3, 64, gnn_type=gnn_type)).double()
        assert not any(isinstance(m, torch.nn.BatchNorm1d) for m in ref.modules())
        hip = ops.use_layer_norm(hmod.GNN(3, 64, gnn_type=gnn_type))
        hip.load_state_dict(ref.state_dict())
        hip = hip.to(DEV)
        cpu = batch.clone().to("cpu")
        attr = cpu.edge_attr.double() if cpu.edge_attr.is_floating_point() else cpu.edge_attr
        x = cpu.x.double() if omod is ochem and cpu.x.is_floating_point() else cpu.x
        want = ref(x, cpu.edge_index, attr)
        got = hip(batch.x, batch.edge_index, batch.edge_attr)
        # three layers of fp32 products of 64 to 128 terms and norms: relative error per layer below 2^-24 * 200
        scale = want.abs().max().item()
        assert (got.detach().cpu().double() - want.detach()).abs().max().item() <= 3 * 200 * U * max(scale, 1.0)
        g = torch.randn(want.shape, generator=torch.Generator().manual_seed(5))
        want.backward(g.double())
        got.backward(g.to(DEV))
        grads = {n: p.grad for n, p in hip.named_parameters()}
        norms = [n for n, m in ref.named_modules() if isinstance(m, torch.nn.LayerNorm)]
        for n, p in ref.named_parameters():
            if p.grad is None:
                continue
            assert grads[n] is not None, n
            if n.rsplit(".", 1)[0] in norms or "weight" in n:
                rel = (grads[n].cpu().double() - p.grad).norm() / p.grad.norm().clamp(min=1e-12)
                assert rel < 2e-3, (n, rel.item())  # a pre-activation within 2^-20 of zero may switch a ReLU: one of thousands of terms
