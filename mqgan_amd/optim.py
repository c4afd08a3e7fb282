"""AdamW over many tensors on the HIP kernels (csrc/adamw.hip): decoupled weight decay, gradient-norm clipping, moments in f32 or
in 8 bits.  Beside train.FlatAdam, which is torch.optim.Adam (no decay) over one arena; the reference has Adam only (train.py:312).

A step is two or three launches whatever the number of tensors: the squares of the norm (with ``max_norm``), one small block that forms
the factors, the update.  Everything that changes from step to step is on the device, so a step may be captured into a graph: the replay
counts on, with the lr and the gradients' addresses of its capture.  One step at a time: a captured step and an eager one of the same
optimiser run one after the other (they share its workspace).
"""
import ctypes as C

import numpy as np
import torch

from . import _lib
from ._lib import AdamwDesc, AdamwTensor, MqganHipError, check, ptr, stream
from .ddp import FlatArena

GROUP = 256                                # elements that share an exponent base; every tensor's moments start on such a boundary
_GRAD_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CONTROL = 64                              # bytes of the control buffer in front of the per-tensor states


class AdamW:
    """``params``: a ddp.FlatArena, f32 tensors, or dicts {"params": tensors, "weight_decay": w, "lr_scale": s} (both optional).
    ``state_bits``: 32, or 8 (two bytes a parameter plus two for every 256; see csrc/adamw.hip for the format).
    ``decays``: which tensors of an arena decay (a function of the parameter; default all).
    ``seed``: of the 8-bit moments' random rounding.  A tensor without a gradient is left out of a step, as in torch.optim.AdamW:
    its moments and its step count stay.  Over an arena in gather mode whose gradients a ddp.GradReducer sums, that is a tensor without a
    gradient on any rank, so that all ranks step the same ones (make the optimiser before the first step's ``finish()``)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, seed=0, decays=None):
        self.arena = params if isinstance(params, FlatArena) else None
        if self.arena is not None:
            self.arena.track_presence = True
        groups = [{"params": params.params}] if self.arena is not None else list(params)
        if groups and not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        self.params, self.weight_decays, self.lr_scales, self.groups = [], [], [], []        # groups: positions of what shares a decay and a scale
        for g in groups:
            unknown = set(g) - {"params", "weight_decay", "lr_scale"}
            if unknown:
                raise ValueError(f"AdamW: a group has params, weight_decay and lr_scale, not {sorted(unknown)}")
            mine = {}
            for p in g["params"]:
                decayed = decays is None or bool(decays(p))
                mine.setdefault(decayed, []).append(len(self.params))
                self.params.append(p)
                self.weight_decays.append(float(g.get("weight_decay", weight_decay)) if decayed else 0.0)
                self.lr_scales.append(float(g.get("lr_scale", 1.0)))
            self.groups += [mine[k] for k in (True, False) if k in mine]
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW: a parameter is given twice")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: moments are held in 8 or 32 bits, not {state_bits}")
        if not (lr >= 0 and eps >= 0 and all(0 <= b < 1 for b in betas) and len(betas) == 2 and all(w >= 0 for w in self.weight_decays)):
            raise ValueError("AdamW: lr, eps and weight_decay >= 0 and two betas in [0, 1) are needed")
        self.device = self.params[0].device
        for i, p in enumerate(self.params):
            if not p.is_cuda or p.device != self.device:
                raise MqganHipError(f"AdamW: parameter {i} lives on {p.device}; every parameter belongs on one HIP device")
            if p.dtype != torch.float32 or not p.is_contiguous():
                raise MqganHipError(f"AdamW: parameter {i} is {p.dtype}{'' if p.is_contiguous() else ', not contiguous'}: parameters are "
                                    "contiguous f32 (they are their own master copy)")
        self.base_lr = self.lr = float(lr)
        self.betas, self.eps, self.state_bits, self.seed = (float(betas[0]), float(betas[1])), float(eps), state_bits, int(seed)
        n = len(self.params)
        sizes = [p.numel() for p in self.params]
        self.positions = np.concatenate([[0], np.cumsum([(s + GROUP - 1) // GROUP * GROUP for s in sizes])]).tolist()
        total = max(self.positions[-1], GROUP)
        new = lambda k, dt: torch.zeros(k, dtype=dt, device=self.device)  # noqa: E731
        if state_bits == 32:
            self.exp_avg, self.exp_avg_sq = new(total, torch.float32), new(total, torch.float32)
            self._bases = None
        else:
            self.exp_avg, self.exp_avg_sq = new(total, torch.uint8), new(total, torch.uint8)
            self._bases = new(total // GROUP, torch.uint8), new(total // GROUP, torch.uint8)
        lib = _lib.load()
        self._sizes, self._shapes = (C.c_int64 * n)(*sizes), [p.shape for p in self.params]
        self._table_bytes = lib.mq_adamw_table_bytes(self._sizes, n)
        if not self._table_bytes:
            raise MqganHipError("AdamW: too many elements")
        self._control = new(lib.mq_adamw_control_bytes(n) // 8, torch.int64)
        self._workspace = new(lib.mq_adamw_workspace(self._sizes, n) // 8, torch.float64)
        self._desc = AdamwDesc(n_tensors=n, state_bits=state_bits, beta1=self.betas[0], beta2=self.betas[1], eps=self.eps, seed=self.seed & (2 ** 64 - 1))
        self._addresses, self._captured = None, []
        self._bind([p.data_ptr() for p in self.params])

    # -- tables ---------------------------------------------------------------------------------
    def _bind(self, addresses):
        """(Re)build the device table of the tensors' addresses."""
        if torch.cuda.is_current_stream_capturing():
            raise MqganHipError("AdamW: a parameter moved since the last step; take one step outside the capture first")
        n, item = len(self.params), self.exp_avg.element_size()
        spans = sorted((a, a + 4 * s, i) for i, (a, s) in enumerate(zip(addresses, self._sizes)) if s)
        for (_, end, i), (start, _, j) in zip(spans, spans[1:]):
            if start < end:
                raise MqganHipError(f"AdamW: parameters {i} and {j} share memory")
        m, v = self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr()
        mb, vb = (b.data_ptr() for b in self._bases) if self._bases else (0, 0)
        rows = (AdamwTensor * n)()
        for i, (a, at) in enumerate(zip(addresses, self.positions)):
            rows[i] = AdamwTensor(a, m + at * item, v + at * item, mb and mb + at // GROUP, vb and vb + at // GROUP, self._sizes[i], at,
                                  self.weight_decays[i], self.lr_scales[i])
        host = torch.empty(self._table_bytes, dtype=torch.uint8)
        check(_lib.load().mq_adamw_table_fill(rows, n, self.state_bits, C.c_void_p(host.data_ptr()), self._table_bytes), "mq_adamw_table_fill")
        self._table = host.to(self.device)          # from pageable memory: complete when the call returns
        self._addresses = addresses

    # -- the step -------------------------------------------------------------------------------
    def zero_grad(self):
        if self.arena is not None:
            self.arena.zero_grad()
        else:
            for p in self.params:
                p.grad = None

    def _gradients(self, grads):
        if grads is not None:
            return grads
        arena = self.arena
        if arena is not None and arena.gather_mode:
            arena.gather()                          # whatever the reducer has not moved yet
            # A parameter without gradient is left out.  Once a reducer has summed the arena over ranks, that is one without gradient on EVERY
            # rank, which arena.present tells on the device: this rank's own .grad would have ranks step different tensors.
            everywhere = arena.present is not None
            return [arena.flat_grad[o:o + p.numel()] if everywhere or p.grad is not None else None for p, o in zip(self.params, arena.offsets)]
        return [p.grad for p in self.params]

    def step(self, max_norm=0.0, grad_scale=1.0, grads=None):
        """``max_norm`` > 0: clip the norm of all gradients to it (``grad_norm()`` then has the norm).  ``grad_scale``: factor on every
        gradient (1 / world size for summed ones).  ``grads``: the gradients (f32, bf16 or f16; None = none) in the order of the
        parameters, each of its parameter's shape or flat, instead of their ``.grad``."""
        if torch.cuda.current_device() != self.device.index:
            raise MqganHipError(f"AdamW: the parameters live on {self.device} but the current HIP device is cuda:{torch.cuda.current_device()}")
        if not max_norm >= 0.0:
            raise ValueError(f"AdamW: max_norm {max_norm}")
        params = self.params
        present = self.arena.present if self.arena is not None and grads is None else None
        grads = self._gradients(grads)
        if len(grads) != len(params):
            raise MqganHipError(f"AdamW: {len(grads)} gradients for {len(params)} parameters")
        held, addresses, types, device = [], [], bytearray(len(params)), self.device.index
        for i, (g, shape, size) in enumerate(zip(grads, self._shapes, self._sizes)):
            if g is None:
                addresses.append(0)
                continue
            t = _GRAD_TYPES.get(g.dtype)
            # of its parameter's shape as it was given, or as it is by now, or flat (an arena's): the same elements in the same order
            if t is None or g.get_device() != device or (g.shape != shape and (g.numel() != size or (g.dim() != 1 and g.shape != params[i].shape))):
                raise MqganHipError(f"AdamW: gradient {i} is {g.dtype} {tuple(g.shape)} on {g.device}; its parameter is {tuple(params[i].shape)} "
                                    f"on {self.device}")
            if not g.is_contiguous():
                g = g.contiguous()
                held.append(g)                      # until the launches are enqueued: the stream's order keeps its memory after that
            types[i] = t
            addresses.append(g.data_ptr())
        at = [p.data_ptr() for p in params]
        if at != self._addresses:
            for i, p in enumerate(params):
                if p.dtype != torch.float32 or not p.is_contiguous() or p.numel() != self._sizes[i] or p.device != self.device:
                    raise MqganHipError(f"AdamW: parameter {i} became {p.dtype} {tuple(p.shape)} on {p.device}")
            self._bind(at)
        if torch.cuda.is_current_stream_capturing():        # a graph reads them as long as it is replayed
            self._captured += [x for x in (self._table, present) if x is not None and not any(x is y for y in self._captured)]
        d = self._desc
        d.lr, d.max_norm, d.grad_scale = float(self.lr), float(max_norm), float(grad_scale)
        what = (C.byref(d), self._sizes, ptr(self._table), (C.c_void_p * len(params))(*addresses), (C.c_uint8 * len(params)).from_buffer(types))
        where = (ptr(self._control), ptr(self._workspace), self._workspace.numel() * 8, stream())
        if present is None:
            check(_lib.load().mq_adamw_step(*what, *where), "mq_adamw_step")
        else:
            check(_lib.load().mq_adamw_step_present(*what, ptr(present), *where), "mq_adamw_step_present")

    def grad_norm(self):
        """Norm of the scaled gradients before clipping, of the last step with ``max_norm`` > 0 (device scalar; reading it synchronises)."""
        f = self._control.view(torch.float64)
        return (f[0].sqrt() * f[4]).float()             # on the device both, so it is right after a replay too

    # -- moments and state ------------------------------------------------------------------------
    def moments(self, dtype=torch.float32):
        """(first, second) moments as flat tensors, tensor i's from ``positions[i]`` on, zeros between.  With f32 moments asked for in f32 they
        are the optimiser's own buffers; 8-bit moments are decoded (exactly, into f32 or bf16)."""
        if self.state_bits == 32:
            return self.exp_avg.to(dtype), self.exp_avg_sq.to(dtype)
        if dtype not in (torch.float32, torch.bfloat16):
            raise MqganHipError(f"AdamW: 8-bit moments decode into float32 or bfloat16, not {dtype}")
        m, v = (torch.empty(self.exp_avg.numel(), dtype=dtype, device=self.device) for _ in range(2))
        check(_lib.load().mq_moments8_decode(ptr(self.exp_avg), ptr(self._bases[0]), ptr(self.exp_avg_sq), ptr(self._bases[1]), m.numel(),
                                             int(dtype == torch.bfloat16), ptr(m), ptr(v), stream()), "mq_moments8_decode")
        return m, v

    def load_moments(self, exp_avg, exp_avg_sq, step=None):
        """Set the moments from flat f32 tensors laid out as ``moments()`` gives them (8 bits: rounded to nearest), and, with ``step``, every
        tensor's step count and the count of calls."""
        for x in (exp_avg, exp_avg_sq):
            if x.numel() != self.exp_avg.numel():
                raise MqganHipError(f"AdamW: moments of {x.numel()} elements, the layout has {self.exp_avg.numel()}")
        if self.state_bits == 32:
            self.exp_avg.copy_(exp_avg.reshape(-1))
            self.exp_avg_sq.copy_(exp_avg_sq.reshape(-1))
        else:
            m, v = (x.to(self.device, torch.float32).reshape(-1).contiguous() for x in (exp_avg, exp_avg_sq))
            check(_lib.load().mq_moments8_encode(ptr(m), ptr(v), m.numel(), ptr(self.exp_avg), ptr(self._bases[0]), ptr(self.exp_avg_sq),
                                                 ptr(self._bases[1]), stream()), "mq_moments8_encode")
        if step is not None:
            self._set_steps([int(step)] * len(self.params), int(step))

    def _steps(self):
        """Every tensor's step count, and the calls so far (synchronises)."""
        host = self._control.cpu()
        return host[_CONTROL // 8:].view(torch.int32)[::4].tolist(), int(host[1])

    def _set_steps(self, steps, calls):
        host = self._control.cpu()
        host[_CONTROL // 8:].view(torch.int32)[::4] = torch.tensor(steps, dtype=torch.int32)
        host[1] = calls
        self._control.copy_(host)

    @property
    def step_count(self):
        """Steps of the tensor that took most (synchronises)."""
        return max(self._steps()[0])

    def state_dict(self):
        """torch.optim.AdamW's format (moments in f32): one parameter group for every group given, and for the tensors of one that ``decays``
        leaves out, each with its own lr and weight decay.  A torch.optim.AdamW over the same groups takes it, and 8 and 32 bits take each
        other's; for 8 bits it has the codes and the seed besides, from which a run goes on bit for bit."""
        steps, calls = self._steps()
        m, v = self.moments()
        state = {}
        for i, (p, at, t) in enumerate(zip(self.params, self.positions, steps)):
            if t:
                state[i] = {"step": torch.tensor(float(t)), "exp_avg": m[at:at + p.numel()].view_as(p).clone(),
                            "exp_avg_sq": v[at:at + p.numel()].view_as(p).clone()}
        groups = [{"lr": self.lr * self.lr_scales[g[0]], "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decays[g[0]],
                   "amsgrad": False, "maximize": False, "foreach": None, "capturable": False, "differentiable": False, "fused": None,
                   "decoupled_weight_decay": True, "initial_lr": self.base_lr * self.lr_scales[g[0]], "lr_scale": self.lr_scales[g[0]],
                   "params": list(g)} for g in self.groups]
        sd = {"state": state, "param_groups": groups, "mqgan_amd_calls": calls, "mqgan_amd_lr": self.lr}
        if self.state_bits == 8:
            sd["mqgan_amd_moments8"] = {"codes": (self.exp_avg.clone(), self.exp_avg_sq.clone()), "bases": tuple(b.clone() for b in self._bases),
                                        "sizes": list(self._sizes), "seed": self.seed}
        return sd

    def load_state_dict(self, sd):
        """A state of this class or of torch.optim.AdamW (or Adam, train.FlatAdam).  Where its groups are this optimiser's - the same
        tensors for a state of this class, the same numbers of them otherwise - lr, scales, betas and eps come with it, as in torch, and weight
        decays where they are decoupled ones (Adam's is another thing); where they are not, lr alone (the first group's) does and the
        tensors go by their position."""
        own = "mqgan_amd_calls" in sd
        saved = sd.get("param_groups") or []
        ids = [[int(i) for i in g["params"]] for g in saved]
        if own:
            fits = ids == self.groups and "mqgan_amd_lr" in sd           # without: one group for all, as this class wrote them at first
        else:
            fits = [len(g) for g in ids] == [len(g) for g in self.groups]
        place = dict(zip((i for g in ids for i in g), (i for g in self.groups for i in g))) if fits else {}
        steps = [0] * len(self.params)
        total = self.exp_avg.numel()
        m, v = (torch.zeros(total, dtype=torch.float32, device=self.device) for _ in range(2))
        for i, st in sd.get("state", {}).items():
            i = place.get(int(i), int(i))
            if i >= len(self.params) or st["exp_avg"].numel() != self._sizes[i]:
                raise MqganHipError(f"AdamW: the state's entry {i} does not fit the parameters")
            at = self.positions[i]
            m[at:at + self._sizes[i]].copy_(st["exp_avg"].reshape(-1))
            v[at:at + self._sizes[i]].copy_(st["exp_avg_sq"].reshape(-1))
            steps[i] = int(float(st["step"]))
        held = sd.get("mqgan_amd_moments8")
        held = held if self.state_bits == 8 and held is not None and list(held["sizes"]) == list(self._sizes) else None
        mine = (self.exp_avg, self.exp_avg_sq) + (self._bases or ())
        theirs = tuple(held["codes"]) + tuple(held["bases"]) if held else ()
        if any(a.shape != b.shape or a.dtype != b.dtype for a, b in zip(mine, theirs)):
            raise MqganHipError("AdamW: the state's 8-bit moments do not fit the parameters")
        self._load_groups(saved, fits, sd.get("mqgan_amd_lr"))
        if held:
            for a, b in zip(mine, theirs):
                a.copy_(b)
            self.seed = int(held.get("seed", self.seed))
            self._desc.seed = self.seed & (2 ** 64 - 1)
        else:
            self.load_moments(m, v)
        self._set_steps(steps, int(sd.get("mqgan_amd_calls", max(steps))))

    def _load_groups(self, saved, fits, lr):
        """lr and, where the groups are this optimiser's, the rest of their settings."""
        if not saved:
            return
        if any(g.get("amsgrad") or g.get("maximize") for g in saved):
            raise MqganHipError("AdamW: the state is of an optimiser with amsgrad or maximize, which this one has not")
        lrs = [float(g.get("lr", self.lr)) for g in saved]
        if not fits:
            self.lr = lrs[0] if lr is None else float(lr)
            return
        betas, eps = ([tuple(float(b) for b in g.get("betas", self.betas)) for g in saved], [float(g.get("eps", self.eps)) for g in saved])
        if len(set(betas)) > 1 or len(set(eps)) > 1:
            raise MqganHipError("AdamW: the state's groups differ in betas or eps, which are one for all of this optimiser's")
        scales = [g.get("lr_scale") for g in saved]
        if lr is None or None in scales:                # not of this class: the first group's scale as it is here, the others' by their lr
            mine = [self.lr_scales[g[0]] for g in self.groups]
            lr = lrs[0] / mine[0] if mine[0] > 0 and lrs[0] > 0 else max(lrs)
            scales = [x / lr for x in lrs] if lr > 0 else mine
        self.lr = float(lr)
        self.betas, self.eps = betas[0], eps[0]
        d = self._desc
        d.beta1, d.beta2, d.eps = self.betas[0], self.betas[1], self.eps
        before = self.weight_decays, self.lr_scales
        self.weight_decays, self.lr_scales = list(before[0]), list(before[1])
        for group, g, scale in zip(self.groups, saved, scales):
            for i in group:
                self.lr_scales[i] = float(scale)
                if g.get("decoupled_weight_decay"):
                    self.weight_decays[i] = float(g.get("weight_decay", before[0][i]))
        if (self.weight_decays, self.lr_scales) != before:
            self._bind(self._addresses)                 # both stand in the table
