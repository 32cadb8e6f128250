"""The cases on which layer normalisation, Newton-Schulz orthogonalisation and the Muon step are measured.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) where ``own`` is
false, and calls the framework's kernels where it is true.  ``exact`` is the same from the definition in 64 bits.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, NS_EPS, LN_EPS = 5, 1e-7, 1e-5
LR, DECAY, MOMENTUM = 0.02, 0.1, 0.95
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # inference on one molecule: 24 atoms at the networks' width; nothing but latency
        {"name": "ln_one_molecule", "op": "layer_norm", "rows": 24, "dim": 300, "dtype": "fp32", "gamma": "fp32", "train": False, "pad": 0},
        # the atoms of 256 molecules, the batch of the masking step, forward and backward
        {"name": "ln_256_molecules", "op": "layer_norm", "rows": 6740, "dim": 300, "dtype": "fp32", "gamma": "fp32", "train": True, "pad": 0},
        # about 10 000 molecules on one card
        {"name": "ln_large_batch", "op": "layer_norm", "rows": 262144, "dim": 300, "dtype": "fp32", "gamma": "fp32", "train": True, "pad": 0},
        # wide rows in half precision with gains kept in 32 bits, as mixed-precision training has them
        {"name": "ln_wide_bf16", "op": "layer_norm", "rows": 16384, "dim": 4096, "dtype": "bf16", "gamma": "fp32", "train": True, "pad": 0},
        # an odd width, the rows a part of a wider buffer (columns of concatenated layer outputs)
        {"name": "ln_odd_fp16", "op": "layer_norm", "rows": 30011, "dim": 1023, "dtype": "fp16", "gamma": "fp16", "train": True, "pad": 5},
        # the atom-type head of the masking task
        {"name": "ns_head", "op": "newton_schulz", "batch": 1, "rows": 119, "cols": 300, "dtype": "fp32"},
        # both weights of a 5-layer network's mlps, as one batch
        {"name": "ns_gin_layers", "op": "newton_schulz", "batch": 10, "rows": 300, "cols": 600, "dtype": "fp32"},
        # odd sizes in half precision
        {"name": "ns_odd_bf16", "op": "newton_schulz", "batch": 1, "rows": 2301, "cols": 1111, "dtype": "bf16"},
        # one large square weight
        {"name": "ns_4096", "op": "newton_schulz", "batch": 1, "rows": 4096, "cols": 4096, "dtype": "fp32"},
        # the optimizer step of the 5-layer network at width 300, with its heads
        {"name": "muon_gin", "op": "muon", "layers": 5, "dim": 300, "hidden": 600, "classes": 119},
        # the same at width 1024, the largest that the networks take
        {"name": "muon_gin_1024", "op": "muon", "layers": 5, "dim": 1024, "hidden": 2048, "classes": 119},
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "newton_schulz", "muon"])
    if op == "layer_norm":
        dim = _log_uniform(rng, 16, 8192)
        rows = _log_uniform(rng, 1, min(262144, 262144 * 300 // dim))
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "gamma": rng.choice([dtype, "fp32"]), "train": rng.random() < 0.7,
                "pad": rng.choice([0, 0, rng.randrange(1, 9)])}
    if op == "newton_schulz":
        short = _log_uniform(rng, 16, 2048)
        long = _log_uniform(rng, short, min(4096, 8 * short))
        batch = _log_uniform(rng, 1, max(1, min(16, 2048 * 2048 // (short * long))))
        rows, cols = (short, long) if rng.random() < 0.5 else (long, short)
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    dim = _log_uniform(rng, 16, 1024)
    return {"op": op, "layers": rng.randrange(1, 9 if dim <= 512 else 6), "dim": dim, "hidden": rng.choice([dim, 2 * dim, dim + rng.randrange(1, dim)]),
            "classes": rng.randrange(2, 201)}


def _muon_shapes(case):
    shapes = []
    for _ in range(case["layers"]):
        shapes += [(case["hidden"], case["dim"]), (case["dim"], case["hidden"])]
    return shapes + [(case["classes"], case["dim"]), (4, case["dim"])]


def _ns_flops(k, n):
    k, n = min(k, n), max(k, n)
    return STEPS * (k * (k + 1) * n + k * k * (k + 1) + 2 * k * k * n)  # A and A A are symmetric: one half of each


def work(case):
    if case["op"] == "layer_norm":
        size = 4 if case["dtype"] == "fp32" else 2
        gamma = 4 if case["gamma"] == "fp32" else 2
        n = case["rows"] * case["dim"]
        if not case["train"]:
            return {"bytes": 2 * n * size + 2 * case["dim"] * gamma, "flops": 8 * n}
        # x and dy read, y and dx written; the output has to be whole before dy exists, so x is read for each direction
        return {"bytes": 5 * n * size + 6 * case["dim"] * gamma, "flops": 20 * n}
    if case["op"] == "newton_schulz":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * case["batch"] * case["rows"] * case["cols"] * size, "flops": case["batch"] * _ns_flops(case["rows"], case["cols"])}
    shapes = _muon_shapes(case)
    return {"bytes": 20 * sum(r * c for r, c in shapes), "flops": sum(_ns_flops(r, c) + 6 * r * c for r, c in shapes)}


def _gradient(gen, batch, rows, cols):
    """what a weight's gradient looks like: a product over examples whose features fall off in strength, a few strong directions
    that all examples share, and noise"""
    width = min(rows, cols)
    strength = torch.logspace(0, -2, width, device="cuda")
    left = torch.randn(batch, rows, width, device="cuda", generator=gen) * strength
    right = torch.randn(batch, width, cols, device="cuda", generator=gen)
    shared = torch.randn(batch, rows, 2, device="cuda", generator=gen) @ torch.randn(batch, 2, cols, device="cuda", generator=gen)
    return (left @ right + shared + 0.1 * torch.randn(batch, rows, cols, device="cuda", generator=gen)) * (1e-3 / math.sqrt(rows * cols))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "layer_norm":
        rows, dim, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
        ln = torch.nn.LayerNorm(dim, eps=LN_EPS, device="cuda", dtype=DTYPES[case["gamma"]])
        with torch.no_grad():
            ln.weight.copy_(1 + 0.2 * normal(dim))
            ln.bias.copy_(0.2 * normal(dim))
        # activations: columns of different strength and offset, rows of different strength
        x = (normal(rows, dim) * (0.5 + normal(dim).abs()) + 0.5 * normal(dim)) * (0.25 + normal(rows, 1).abs())
        buffer = torch.zeros(rows, dim + case["pad"], device="cuda", dtype=dtype)
        buffer[:, :dim] = x
        state = {"case": case, "ln": ln, "x": buffer[:, :dim]}
        if case["train"]:
            state["dy"] = normal(rows, dim).to(dtype)
            state["x"].requires_grad_(True)
        return state
    if case["op"] == "newton_schulz":
        return {"case": case, "g": _gradient(gen, case["batch"], case["rows"], case["cols"]).mul_(64).to(DTYPES[case["dtype"]])}
    params, buffers = [], []
    for rows, cols in _muon_shapes(case):
        p = torch.nn.Parameter(normal(rows, cols) / math.sqrt(cols))
        p.grad = _gradient(gen, 1, rows, cols)[0]
        params.append(p)
        buffers.append(_gradient(gen, 1, rows, cols)[0] * 10)
    state = {"case": case, "params": params, "buffers": buffers}
    if own:  # the optimizer that a program keeps, some steps into its training
        from pretrain_gnns_amd import optim
        state["optimizer"] = optim.Muon(params, lr=LR, weight_decay=DECAY, momentum=MOMENTUM, nesterov=True, ns_coefficients=COEFFICIENTS,
                                        eps=NS_EPS, ns_steps=STEPS)
        for p, b in zip(params, buffers):
            state["optimizer"].state[p]["momentum_buffer"].copy_(b)
    return state


def _plain_layer_norm(x, gamma, beta, dy):
    xf, w = x.float(), gamma.float()
    centred = xf - xf.mean(1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + LN_EPS)
    hat = centred * rstd
    y = (hat * w + beta.float()).to(x.dtype)
    if dy is None:
        return y
    dyf = dy.float()
    g = dyf * w
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return y, dx.to(x.dtype), (dyf * hat).sum(0).to(gamma.dtype), dyf.sum(0).to(gamma.dtype)


def _plain_newton_schulz(g):
    """[batch, rows, cols] in 32 bits; the norm, a sum of up to millions of squares, in 64"""
    norm = g.double().square().sum((1, 2), keepdim=True).sqrt()
    x = g / (norm + NS_EPS).float()
    if g.size(1) > g.size(2):
        x = x.transpose(1, 2).contiguous()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(1, 2).contiguous() if g.size(1) > g.size(2) else x


def _plain_muon(params, buffers):
    with torch.no_grad():
        direction, alike = [], {}
        for i, (p, m) in enumerate(zip(params, buffers)):
            m.mul_(MOMENTUM).add_(p.grad)
            u = p.grad + MOMENTUM * m
            direction.append(u.T if u.size(0) > u.size(1) else u)
            alike.setdefault(direction[i].shape, []).append(i)
        for members in alike.values():  # weights of one shape, and their transposes, as one batch
            ortho = _plain_newton_schulz(torch.stack([direction[i] for i in members]))
            for i, o in zip(members, ortho):
                p = params[i]
                rate = LR * math.sqrt(max(1.0, p.size(0) / p.size(1)))
                p.mul_(1 - LR * DECAY).sub_(o.T if p.size(0) > p.size(1) else o, alpha=rate)
    return [p.detach() for p in params] + list(buffers)


def run(state):
    op = state["case"]["op"]
    if op == "layer_norm":
        ln, x, dy = state["ln"], state["x"], state.get("dy")
        if not own:
            with torch.no_grad():
                return _plain_layer_norm(x, ln.weight, ln.bias, dy)
        from pretrain_gnns_amd import ops
        if dy is None:
            with torch.no_grad():
                return ops.layer_norm(x, ln)
        y = ops.layer_norm(x, ln)
        return (y.detach(),) + torch.autograd.grad(y, (x, ln.weight, ln.bias), dy)
    if op == "newton_schulz":
        if not own:
            return _plain_newton_schulz(state["g"].float()).to(state["g"].dtype)
        from pretrain_gnns_amd import ops
        return ops.newton_schulz(state["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    if not own:
        return _plain_muon(state["params"], state["buffers"])
    optimizer = state["optimizer"]
    optimizer.step()
    return [p.detach() for p in state["params"]] + [optimizer.state[p]["momentum_buffer"] for p in state["params"]]


def _exact_orthogonal(g):
    """the iteration as ONE polynomial in the Gram matrix S = G G^T of the short side, applied to G at the end: with X_t = Q_t X_0
    and A_t = Q_t S Q_t the factor R_t = a + b A_t + c A_t^2 gives Q_{t+1} = R_t Q_t"""
    if g.size(0) > g.size(1):
        return _exact_orthogonal(g.T).T
    x0 = g / (torch.linalg.matrix_norm(g) + NS_EPS)
    s = x0 @ x0.T
    eye = torch.eye(s.size(0), dtype=torch.float64, device=s.device)
    q = eye
    for _ in range(STEPS):
        a_t = q @ s @ q
        q = (COEFFICIENTS[0] * eye + COEFFICIENTS[1] * a_t + COEFFICIENTS[2] * (a_t @ a_t)) @ q
    return q @ x0


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "layer_norm":
            x, w, b = (t.detach().double() for t in (state["x"], state["ln"].weight, state["ln"].bias))
            var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            sigma = torch.sqrt(var + LN_EPS)
            y = (x - mean) / sigma * w + b
            if not case["train"]:
                return y
            dy = state["dy"].double()
            # the Jacobian of (x - mean) / sigma is symmetric: centre, remove the part along x - mean, divide by sigma
            t = dy * w
            t = t - t.mean(1, keepdim=True)
            along = (t * (x - mean)).sum(1, keepdim=True) / (case["dim"] * sigma.square())
            dx = (t - (x - mean) * along) / sigma
            return y, dx, (dy * (x - mean) / sigma).sum(0), dy.sum(0)
        if case["op"] == "newton_schulz":
            return torch.stack([_exact_orthogonal(g.double()) for g in state["g"]])
        params, buffers = [], []
        for p, m in zip(state["params"], state["buffers"]):
            g, m = p.grad.double(), m.double()
            m = g + MOMENTUM * m
            rate = LR * math.sqrt(max(1.0, p.size(0) / p.size(1)))
            params.append(p.detach().double() * (1 - LR * DECAY) - rate * _exact_orthogonal(g + MOMENTUM * m))
            buffers.append(m)
        return params + buffers
