"""``Adam``: torch.optim.Adam's update for the optimizers of the reference's train loops, as ONE kernel launch; ``Muon`` beside it.

The reference builds one ``optim.Adam`` per module (chem/pretrain_masking.py:134-136: model, linear_pred_atoms,
linear_pred_bonds) with the same hyper-parameters and calls ``zero_grad()`` / ``step()`` on each.  ``Adam`` here has the
same constructor and the same two methods; ``Adam.shared([...modules...], lr=..., weight_decay=...)`` returns one handle
per module that share a single kernel launch, so the reference's loop body runs unchanged::

    optimizer_model, optimizer_linear_pred_atoms, optimizer_linear_pred_bonds = Adam.shared(
        [model.parameters(), linear_pred_atoms.parameters(), linear_pred_bonds.parameters()], lr=args.lr, weight_decay=args.decay)

The update is torch's formula in fp32 (csrc/optim.hip); the step counter lives on the device, so a step can be captured
in a HIP graph.  Parameters without a gradient are skipped, like torch does; their moments stay untouched.

Limits, enforced rather than silent:
  * ONE step counter serves every parameter, where torch keeps ``state['step']`` per parameter and starts it at that
    parameter's first gradient.  A parameter that never gets a gradient (the bond head without --mask_edge) is simply skipped,
    which is torch's behaviour; a parameter whose FIRST gradient shows up after other parameters have already been stepped
    would get torch's bias correction for the wrong t, so ``launch()`` raises for it.
  * lr / betas / eps / weight_decay are read from ``param_groups[0]`` of the handles at every launch (an LR scheduler or a manual
    ``param_groups[0]['lr'] = x`` takes effect); the handles of one ``Adam.shared`` share a launch and must agree on them.
  * every handle of ``Adam.shared`` must call ``step()`` in every round: stepping a handle twice, or calling ``zero_grad()``
    while a round is incomplete, raises (the update of ALL handles would silently never be issued otherwise).
"""
import ctypes
import math

import torch

from . import _lib
from .ops import NEWTON_SCHULZ_COEFFICIENTS, _call_workspace, _newton_schulz_coefficients, _on_device, check, load, stream_ptr


def _zero_grads(params, set_to_none):
    for p in params:
        if p.grad is None:
            continue
        if set_to_none:
            p.grad = None
        else:
            if p.grad.grad_fn is not None:
                p.grad.detach_()
            else:
                p.grad.requires_grad_(False)  # (a gradient that is a view -- parallel.GradBucket's -- cannot be detached in place)
            p.grad.zero_()


class _Core:
    """the tensors of all handles, the flat moment buffers and the device step counter"""

    def __init__(self, params, lr, betas, eps, weight_decay):
        self.params = [p for p in params]
        if not self.params:
            raise ValueError("optimizer got an empty parameter list")
        for p in self.params:
            if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                raise _lib.PgnnError("pretrain_gnns_amd.optim.Adam: contiguous fp32 GPU parameters only")
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), (float(betas[0]), float(betas[1])), float(eps), float(weight_decay)
        dev = self.params[0].device
        offs, total = [], 0
        for p in self.params:
            offs.append(total)
            total += (p.numel() + 63) // 64 * 64
        self.offsets = offs
        self.exp_avg = torch.zeros(total, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(total, dtype=torch.float32, device=dev)
        self.step_words = torch.zeros(32, dtype=torch.int64, device=dev)  # updates applied, the kernel's cache of beta^step, its arrival tickets
        self.step_count = self.step_words[0]
        self.max_tensors = int(load().pgnn_adam_max_tensors())
        self.waiting = 0  # handles that still have to call step() before the shared launch goes out
        self._tables, self._table_key = [], None
        self.handles = 0
        self.owners = []       # the Adam handles (their param_groups carry the hyper-parameters)
        self.stepped = set()   # ids of the handles that have stepped in the current round
        self.launches = 0
        self._seen = set()     # ids of the parameters that took part in the first launch

    def hyper(self):
        """(lr, beta1, beta2, eps, weight_decay) as the handles' param_groups say NOW"""
        vals = None
        for h in self.owners:
            g = h.param_groups[0]
            v = (float(g["lr"]), float(g["betas"][0]), float(g["betas"][1]), float(g["eps"]), float(g["weight_decay"]))
            if vals is None:
                vals = v
            elif v != vals:
                raise _lib.PgnnError("pretrain_gnns_amd.optim.Adam.shared: the handles share ONE launch and must agree on lr / betas / eps / "
                                     "weight_decay (%r vs %r); use separate Adam instances for different hyper-parameters" % (vals, v))
        return vals if vals is not None else (self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay)

    @torch.no_grad()
    def launch(self):
        live = [(p, o) for p, o in zip(self.params, self.offsets) if p.grad is not None]
        ids = {id(p) for p, _ in live}
        if self.launches == 0:
            self._seen = ids
        elif not ids <= self._seen:
            raise _lib.PgnnError("pretrain_gnns_amd.optim.Adam: a parameter received its first gradient after %d updates of the others; the "
                                 "single device-side step count cannot give it torch's per-parameter bias correction" % self.launches)
        self.launches += 1
        lr, b1, b2, eps, wd = self.hyper()
        # the job tables (ctypes arrays of pointers / counts / offsets) are rebuilt only when a pointer moved: with the caching
        # allocator the gradients come back at the same addresses step after step, and building the tables was ~0.1 ms a step
        key = tuple([p.data_ptr() for p, _ in live] + [p.grad.data_ptr() for p, _ in live])
        if key != self._table_key:
            tables = []
            for i in range(0, len(live), self.max_tensors):
                part = live[i:i + self.max_tensors]
                n = len(part)
                for p, _ in part:
                    if p.grad.dtype != torch.float32 or not p.grad.is_contiguous() or p.grad.device != p.device:
                        raise _lib.PgnnError("pretrain_gnns_amd.optim.Adam: gradients must be contiguous fp32 on the parameter's device")
                tables.append(((ctypes.c_void_p * n)(*[p.data_ptr() for p, _ in part]),
                               (ctypes.c_void_p * n)(*[p.grad.data_ptr() for p, _ in part]),
                               (ctypes.c_int64 * n)(*[p.numel() for p, _ in part]), (ctypes.c_int64 * n)(*[o for _, o in part]), n))
            self._tables, self._table_key = tables, key
        lib, sp = load(), stream_ptr()
        for i, (P, G, C, O, n) in enumerate(self._tables):
            # every part reads the same step count: only the last part's launch advances it
            counter = self.step_words if i == len(self._tables) - 1 else self.step_words.clone()
            check(lib.pgnn_adam_step(P, G, C, O, n, self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), counter.data_ptr(), lr,
                                     b1, b2, eps, wd, sp), "pgnn_adam_step")


class Adam:
    """torch.optim.Adam(params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0): zero_grad() and step()."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, _core=None):
        self._own = list(params)
        self._core = _core if _core is not None else _Core(self._own, lr, betas, eps, weight_decay)
        self._core.handles += 1
        self._core.owners.append(self)
        self.param_groups = [{"params": self._own, "lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay}]

    @classmethod
    def shared(cls, param_lists, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0):
        """one handle per parameter list; the update of all of them is a single launch, issued by the LAST handle whose
        ``step()`` is called in a round (the reference calls them back to back)"""
        lists = [list(ps) for ps in param_lists]
        core = _Core([p for ps in lists for p in ps], lr, betas, eps, weight_decay)
        return [cls(ps, lr, betas, eps, weight_decay, _core=core) for ps in lists]

    def zero_grad(self, set_to_none=True):
        if self._core.waiting != 0:
            raise _lib.PgnnError("pretrain_gnns_amd.optim.Adam.shared: zero_grad() with %d of %d handles not stepped -- the shared update "
                                 "has NOT been issued; every handle must call step() each round" % (self._core.waiting, self._core.handles))
        _zero_grads(self._own, set_to_none)

    def step(self):
        core = self._core
        if core.waiting == 0:
            core.waiting = core.handles
            core.stepped.clear()
        if id(self) in core.stepped:
            raise _lib.PgnnError("pretrain_gnns_amd.optim.Adam.shared: this handle stepped twice before the others stepped once; every "
                                 "handle must call step() each round (the update is one launch for all of them)")
        core.stepped.add(id(self))
        core.waiting -= 1
        if core.waiting == 0:
            core.launch()

    @property
    def step_count(self):
        return self._core.step_count


class Muon:
    """Muon for the weight matrices of a network: zero_grad() and step(), one library call for all of them.

    Per matrix  M <- momentum M + G;  U = G + momentum M (nesterov) or M;  O = ops.newton_schulz(U, ns_steps, ns_coefficients, eps);
    p <- p (1 - lr weight_decay) - lr s O  with s = sqrt(max(1, rows / cols)) (``adjust_lr_fn`` None or "original") or
    0.2 sqrt(max(rows, cols)) ("match_rms_adamw": updates as large as Adam's).  The arguments are those of torch.optim.Muon, and so is the
    step but for three things.  The direction carries fp32's error (in the norm: ops.newton_schulz) where that class multiplies in bf16.
    ``eps`` is added to the norm where that class takes the larger of the two.  M is a sum where that class keeps an average (this M times
    1 - momentum), which is the same direction U / |U| but reaches eps at gradients 1 / (1 - momentum) times smaller: both matter for norms
    near eps only.

    It takes 2-D parameters only (contiguous fp32 on one GPU): biases, norms' gains and embedding tables belong to ``Adam``.  The
    reference's loop body takes both in its optimizer list::

        weights = [p for n, p in model.named_parameters() if p.dim() == 2 and "embedding" not in n]
        others = [p for p in model.parameters() if all(p is not w for w in weights)]
        optimizer_list = [Muon(weights, lr=0.02), Adam(others, lr=args.lr)]

    ``state[p]["momentum_buffer"]`` is p's M (zero before the first step).  A parameter without a gradient is skipped, momentum and
    all.  lr, momentum, nesterov and weight_decay are read from ``param_groups[0]`` at every step; a captured step keeps the captured ones.
    ns_steps, ns_coefficients, eps and adjust_lr_fn are fixed when it is made.
    """

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=NEWTON_SCHULZ_COEFFICIENTS, eps=1e-7,
                 ns_steps=5, adjust_lr_fn=None):
        self._own = list(params)
        if not self._own:
            raise ValueError("optimizer got an empty parameter list")
        if adjust_lr_fn not in (None, "original", "match_rms_adamw"):
            raise ValueError("Muon: adjust_lr_fn is None, \"original\" or \"match_rms_adamw\", got %r" % (adjust_lr_fn,))
        if lr < 0 or momentum < 0 or weight_decay < 0 or eps < 0:
            raise ValueError("Muon: lr, momentum, weight_decay and eps are not negative")
        self._coef = _newton_schulz_coefficients(ns_coefficients, ns_steps)
        for p in self._own:
            if p.dim() != 2:
                raise ValueError("Muon orthogonalises 2-D parameters only, got size %s: give the others to Adam" % (tuple(p.shape),))
            if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous() or p.device != self._own[0].device:
                raise _lib.PgnnError("pretrain_gnns_amd.optim.Muon: contiguous fp32 parameters on one GPU only")
        if len({id(p) for p in self._own}) != len(self._own):
            raise ValueError("Muon: a parameter appears twice")
        self._steps, self._eps, self._adjust = int(ns_steps), float(eps), adjust_lr_fn
        offs, total = [], 0
        for p in self._own:
            offs.append(total)
            total += (p.numel() + 63) // 64 * 64
        self._flat = torch.zeros(total, dtype=torch.float32, device=self._own[0].device)
        self.state = {p: {"momentum_buffer": self._flat[o:o + p.numel()].view(p.shape)} for p, o in zip(self._own, offs)}
        self.param_groups = [{"params": self._own, "lr": lr, "weight_decay": weight_decay, "momentum": momentum, "nesterov": nesterov}]
        self._sizes, self._tables = None, None  # of the live parameters: their sizes, and what follows from sizes alone

    # what the coefficients and the kept scales were made for: fixed
    ns_steps = property(lambda self: self._steps)
    eps = property(lambda self: self._eps)
    adjust_lr_fn = property(lambda self: self._adjust)

    def zero_grad(self, set_to_none=True):
        _zero_grads(self._own, set_to_none)

    def _scale(self, p):
        rows, cols = p.shape
        if self._adjust == "match_rms_adamw":
            return 0.2 * math.sqrt(max(rows, cols))
        return math.sqrt(max(1.0, rows / cols))

    @torch.no_grad()
    def step(self):
        live = [p for p in self._own if p.grad is not None and p.numel()]
        if not live:
            return
        lib, n, dev = load(), len(live), live[0].device
        grads, momenta = [p.grad for p in live], [self.state[p]["momentum_buffer"] for p in live]
        for kind, tensors in (("parameters", live), ("gradients", grads), ("momentum buffers", momenta)):
            for t, p in zip(tensors, live):
                if t.dtype is not torch.float32 or t.device != dev or t.shape != p.shape or not t.is_contiguous():
                    raise _lib.PgnnError("pretrain_gnns_amd.optim.Muon: %s must be contiguous fp32 of the parameter's size and on its device" % kind)
        sizes = [p.shape for p in live]
        if sizes != self._sizes:
            rows, cols = (ctypes.c_int64 * n)(*[r for r, _ in sizes]), (ctypes.c_int64 * n)(*[c for _, c in sizes])
            self._tables = rows, cols, lib.pgnn_newton_schulz_workspace_bytes(rows, cols, n), [self._scale(p) for p in live]
            self._sizes = sizes
        rows, cols, need, scales = self._tables
        written = [t.data_ptr() for t in live + momenta]
        if len(set(written)) != 2 * n:  # (all matrices of a call are updated at the same time)
            raise _lib.PgnnError("pretrain_gnns_amd.optim.Muon: two parameters, or momentum buffers, at one place in memory")
        P, M, G = (ctypes.c_void_p * n)(*written[:n]), (ctypes.c_void_p * n)(*written[n:]), (ctypes.c_void_p * n)(*[t.data_ptr() for t in grads])
        group = self.param_groups[0]
        lr = float(group["lr"])
        with _on_device(dev):
            ws = _call_workspace(need, dev)
            check(lib.pgnn_muon_step(P, G, M, (ctypes.c_float * n)(*[lr * s for s in scales]), rows, cols, n, float(group["momentum"]),
                                     int(bool(group["nesterov"])), 1.0 - lr * float(group["weight_decay"]), self._coef, self._steps, self._eps,
                                     ws.data_ptr(), ws.numel(), stream_ptr()), "pgnn_muon_step")
        # (a graph that still holds them must notice; tensors made in inference mode are in no graph and have no counter)
        torch.autograd.graph.increment_version([t for t in live + momenta if not t.is_inference()])
