"""GPU: calls of the operators that go through torch's other machinery (traces, threads, other streams)."""
import threading

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


def test_two_host_threads_on_one_stream():
    """calls of several launches each, from threads that share a stream: neither meets the other's planes or partial sums"""
    from pretrain_gnns_amd import optim
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(0)
    work = []
    for k in range(2):
        mats = [torch.randn(s, generator=gen, device=DEV) for s in ((300 + 60 * k, 600), (119, 300), (700, 650))]
        ln = torch.nn.LayerNorm(300 + 8 * k, device=DEV)
        x = torch.randn(5000, 300 + 8 * k, generator=gen, device=DEV)
        work.append((mats, ln, x))

    def job(k):
        mats, ln, x = work[k]
        out = list(ops.newton_schulz(mats))
        params = [torch.nn.Parameter(m.clone()) for m in mats]
        for p, m in zip(params, mats):
            p.grad = m
        optim.Muon(params, lr=0.02).step()
        xl = x.detach().requires_grad_(True)
        y = ops.layer_norm(xl, ln, True)
        return out + [p.detach() for p in params] + [y.detach()] + list(torch.autograd.grad(y, (xl, ln.weight, ln.bias), x))

    want = [job(0), job(1)]
    torch.cuda.synchronize()
    results, start = {}, threading.Barrier(2)

    def worker(k):
        start.wait()
        results[k] = [job(k) for _ in range(10)]

    threads = [threading.Thread(target=worker, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        assert len(results[k]) == 10
        for got in results[k]:
            assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def test_a_second_threads_smaller_launch_takes_no_lds_away():
    """the same kernel with 144 KB of LDS, from another thread with 104 KB, and with 144 KB again"""
    ops = _ops()
    large, small = torch.randn(64, 384, device=DEV), torch.randn(64, 200, device=DEV)
    want = ops.newton_schulz(large), ops.newton_schulz(small)
    got = []

    def other():
        got.append(ops.newton_schulz(small))
        torch.cuda.synchronize()

    thread = threading.Thread(target=other)
    thread.start()
    thread.join()
    assert torch.equal(got[0], want[1]) and torch.equal(ops.newton_schulz(large), want[0])


def test_muon_beside_torchs():
    """the same step from gradients far above eps (that class multiplies in bf16), and half of it where |U| is eps: eps is added"""
    from pretrain_gnns_amd import optim
    gen = torch.Generator().manual_seed(0)
    w, g = torch.randn(48, 96, generator=gen), torch.randn(48, 96, generator=gen)
    ours, theirs = torch.nn.Parameter(w.clone().to(DEV)), torch.nn.Parameter(w.clone())
    a = optim.Muon([ours], lr=1.0, weight_decay=0.1, momentum=0.9)
    b = torch.optim.Muon([theirs], lr=1.0, weight_decay=0.1, momentum=0.9)
    for k in range(3):
        ours.grad, theirs.grad = (g * (1 + k)).to(DEV), g * (1 + k)
        a.step()
        b.step()
        # M is their average times 1 / (1 - momentum): three roundings of either
        m, n = a.state[ours]["momentum_buffer"].cpu() * 0.1, b.state[theirs]["momentum_buffer"]
        assert ((m - n).abs() <= 8 * 2.0 ** -24 * (k + 1) * n.abs().max()).all()
        # five steps of three products in bf16, each term off by 2^-8 at most (as a random walk far less than 15 * 2^-8 of the direction)
        step = (theirs.detach() - w).norm()
        assert (ours.detach().cpu() - theirs.detach()).norm() <= 15 * 2.0 ** -8 * step
    # one linear step of which X_0 = U / (|U| + eps) is the result
    u = g * 1.9  # G + 0.9 M, M = G
    for eps, share in ((1e-7, 1.0), (u.norm().item(), 0.5), (3 * u.norm().item(), 0.25)):
        p = torch.nn.Parameter(torch.zeros(48, 96, device=DEV))
        p.grad = g.to(DEV)
        optim.Muon([p], lr=1.0, weight_decay=0.0, momentum=0.9, ns_coefficients=(1.0, 0.0, 0.0), ns_steps=1, eps=eps).step()
        want = -(u.double() / u.double().norm()) * share
        assert (p.detach().cpu().double() - want).norm() <= 2.0 ** -19 * share  # planes of 22 bits, eps and the norm rounded to fp32


def test_a_graph_from_before_a_muon_step_is_refused():
    """the step writes to the parameters: a backward pass that still wants their old values has to notice, as after any in-place update"""
    from pretrain_gnns_amd import optim
    p = torch.nn.Parameter(torch.randn(8, 12, device=DEV))
    opt = optim.Muon([p], lr=0.02)
    p.grad = torch.randn(8, 12, device=DEV)
    x = torch.randn(5, 8, device=DEV, requires_grad=True)
    loss = (x @ p).sum()
    before = p._version
    opt.step()
    assert p._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_muon_refuses_two_parameters_in_one_memory():
    from pretrain_gnns_amd import _lib, optim
    w = torch.randn(8, 12, device=DEV)
    a, b = torch.nn.Parameter(w), torch.nn.Parameter(w)
    c, d = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    for pair, tie in (((a, b), False), ((c, d), True)):
        opt = optim.Muon(pair, lr=0.02)
        for p in pair:
            p.grad = torch.ones(8, 12, device=DEV)
        if tie:
            opt.state[c]["momentum_buffer"] = opt.state[d]["momentum_buffer"]
        with pytest.raises(_lib.PgnnError, match="one place"):
            opt.step()
    assert torch.equal(a, w) and torch.equal(c, w) and torch.equal(d, w)
    b.grad = None  # one of them alone
    before = w.clone()
    optim.Muon((a, b), lr=0.02).step()
    assert torch.equal(a, b) and not torch.equal(a, before)


def test_muon_made_and_stepped_in_inference_mode():
    """tensors without version counters"""
    from pretrain_gnns_amd import optim
    w, g = torch.randn(8, 12, device=DEV), torch.randn(8, 12, device=DEV)
    outside, kept = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    with torch.inference_mode():
        inside = torch.nn.Parameter(w.clone())
        opts = [optim.Muon([inside], lr=0.02), optim.Muon([outside], lr=0.02)]
        inside.grad = g.clone()
    outside.grad = kept.grad = g
    plain = optim.Muon([kept], lr=0.02)
    for _ in range(2):
        plain.step()
        opts[1].step()
        with torch.inference_mode():
            opts[0].step()
    assert torch.equal(outside, kept) and torch.equal(inside, kept)


@pytest.mark.parametrize("shapes", [[(3, 300), (64, 384), (33, 1)], [(119, 301), (300, 600), (321, 35)], [(700, 651), (333, 1030)]])
def test_muon_with_weights_anywhere_in_memory(shapes):
    """parameters, gradients and momenta as parts of a buffer at any multiple of four bytes: the same bits as with tensors of their own, and
    what lies between them stays as it was"""
    from pretrain_gnns_amd import optim
    gen = torch.Generator(device=DEV).manual_seed(0)

    def parts():
        total = sum(r * c for r, c in shapes) + 8 * (len(shapes) + 1)
        buffer, at, views = torch.full((total,), float("nan"), device=DEV), 1, []
        for k, (r, c) in enumerate(shapes):
            views.append(buffer[at:at + r * c].view(r, c))
            at += r * c + 2 * k + 1  # (odd gaps)
        return buffer, views

    values = [[torch.randn(s, device=DEV, generator=gen) for s in shapes] for _ in range(3)]
    own = [torch.nn.Parameter(v.clone()) for v in values[0]]
    buffers, placed = zip(*(parts() for _ in range(3)))
    for views, vals in zip(placed, values):
        for view, val in zip(views, vals):
            view.copy_(val)
    between = [b.isnan() for b in buffers]
    apart = [torch.nn.Parameter(v) for v in placed[0]]
    opts = optim.Muon(own, lr=0.02), optim.Muon(apart, lr=0.02)
    for i, (p, q) in enumerate(zip(own, apart)):
        assert q.data_ptr() == placed[0][i].data_ptr()
        p.grad, q.grad = values[1][i], placed[1][i]
        opts[0].state[p]["momentum_buffer"].copy_(values[2][i])
        opts[1].state[q]["momentum_buffer"] = placed[2][i]
    for _ in range(2):
        for opt in opts:
            opt.step()
    for i, (p, q) in enumerate(zip(own, apart)):
        assert torch.equal(p, q) and torch.equal(opts[0].state[p]["momentum_buffer"], placed[2][i])
    assert all(torch.equal(b.isnan(), n) for b, n in zip(buffers, between))
