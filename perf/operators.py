"""What the operators on code scores and the AdamW step are measured on: cases, inputs, plain forms, 64-bit results.

Three operators:
  adamw    one optimisation step over many tensors: gradient norm clipping, decoupled weight decay, moments in f32 or in 8 bits
  balance  balance loss of a codebook with per-code counts, forward and backward
  sample   drawing a code per row of scores: temperature, top-k, top-p, min-p, given uniform numbers
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP = 256                    # elements of a tensor that share an exponent base in the 8-bit moments; tensors start on such a boundary
LR, BETAS, EPS, DECAY, STEP = 1e-4, (0.9, 0.999), 1e-8, 0.01, 100
SEED = 42


def listed():
    return [
        # the encoder's first layers alone, no clipping: what a small fine-tune steps; launches count
        {"name": "adamw32 small", "op": "adamw", "tensors": 12, "elements": 150_001, "bits": 32, "grad": "f32", "clip": False},
        # every tensor of the speech configuration's generator, clipped as its trainer does
        {"name": "adamw32 generator", "op": "adamw", "tensors": 260, "elements": 34_000_000, "bits": 32, "grad": "f32", "clip": True},
        # the same step with the moments in 8 bits
        {"name": "adamw8 generator", "op": "adamw", "tensors": 260, "elements": 34_000_000, "bits": 8, "grad": "f32", "clip": True},
        # generator and discriminators of a wide model in one step, gradients in bf16
        {"name": "adamw8 large", "op": "adamw", "tensors": 420, "elements": 150_000_000, "bits": 8, "grad": "bf16", "clip": True},
        # one short utterance against the [8, 5, 5, 5] code space
        {"name": "balance utterance", "op": "balance", "rows": 129, "codes": 1000, "per_row": 1, "dtype": "f32", "padded": 0.0},
        # a batch of 32 x 512 ragged frames at the benchmark's first codebook size
        {"name": "balance batch", "op": "balance", "rows": 16384, "codes": 1024, "per_row": 1, "dtype": "f32", "padded": 0.2},
        # few classes with two assignments a row: residual stages or experts
        {"name": "balance narrow", "op": "balance", "rows": 30011, "codes": 16, "per_row": 2, "dtype": "bf16", "padded": 0.1},
        # the benchmark's largest codebook
        {"name": "balance large", "op": "balance", "rows": 16384, "codes": 8192, "per_row": 1, "dtype": "bf16", "padded": 0.2},
        # one frame of one stream, every filter on: the latency of a token
        {"name": "sample one frame", "op": "sample", "rows": 1, "codes": 1000, "dtype": "f32", "top_k": 50, "top_p": 0.9, "min_p": 0.02, "by_row": False},
        # 48 streams, each with settings of its own, scores in bf16 over the code space with its special tokens
        {"name": "sample streams", "op": "sample", "rows": 48, "codes": 8003, "dtype": "bf16", "top_k": 0, "top_p": 0.95, "min_p": 0.0, "by_row": True},
        # a batch of utterances assigned at random instead of to the nearest code
        {"name": "sample batch", "op": "sample", "rows": 16384, "codes": 1024, "dtype": "f32", "top_k": 0, "top_p": 0.9, "min_p": 0.0, "by_row": False},
        # the same at the largest codebook, every filter on
        {"name": "sample large", "op": "sample", "rows": 16384, "codes": 8192, "dtype": "f32", "top_k": 100, "top_p": 0.95, "min_p": 0.01, "by_row": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw", "balance", "sample"])
    if op == "adamw":
        tensors = _log(rng, 1, 420)
        return {"op": op, "tensors": tensors, "elements": _log(rng, 1000 * tensors, 80_000_000), "bits": rng.choice([8, 32]),
                "grad": rng.choice(["f32", "bf16"]), "clip": rng.random() < 0.7}
    codes = _log(rng, 8, 8192)
    if op == "balance":
        return {"op": op, "rows": _log(rng, 1, 16384), "codes": codes, "per_row": rng.choice([1, 1, 2, 4]), "dtype": rng.choice(["f32", "bf16"]),
                "padded": rng.choice([0.0, 0.1, 0.5])}
    return {"op": op, "rows": _log(rng, 1, 16384), "codes": codes, "dtype": rng.choice(["f32", "bf16"]), "top_k": rng.choice([0, 1, 40, 200]),
            "top_p": rng.choice([1.0, 0.95, 0.8, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.05]), "by_row": rng.random() < 0.5}


# ----------------------------------------------------------------------------- adamw
def _sizes(case):
    """The weights first, which share out the elements, then two gains or biases for each, as weight-normed convolutions have them."""
    r = np.random.RandomState(case["tensors"])
    small = r.choice([1, 25, 80, 128, 256, 384, 512, 768], case["tensors"])
    share = np.where(np.arange(case["tensors"]) < _weights(case), 16.0 ** r.rand(case["tensors"]), 0.0)
    return np.where(share > 0, np.maximum(1, share / share.sum() * case["elements"]).astype(np.int64), small)


def _weights(case):
    return (case["tensors"] + 2) // 3


def _inputs_adamw(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    size = torch.from_numpy(_sizes(case))
    room = (size + GROUP - 1) // GROUP * GROUP
    start = room.cumsum(0) - room
    total = int(room.sum())
    owner = torch.repeat_interleave(torch.arange(len(size), device="cuda"), room.cuda())
    real = torch.arange(total, device="cuda") - start.cuda()[owner] < size.cuda()[owner]
    level = 10.0 ** (torch.rand(len(size), device="cuda", generator=gen) * 3 - 5)            # gradients of layers differ by orders
    param = torch.randn(total, device="cuda", generator=gen) * 0.05 * real
    usual = level[owner] * torch.exp(torch.randn(total, device="cuda", generator=gen)) * real
    exp_avg = 0.3 * usual * torch.randn(total, device="cuda", generator=gen)
    exp_avg_sq = usual.square() * (0.5 + torch.rand(total, device="cuda", generator=gen))
    flat = (usual * torch.randn(total, device="cuda", generator=gen)).to(DTYPES[case["grad"]])
    spans = list(zip(start.tolist(), size.tolist()))
    return {"op": "adamw", "case": case, "param": param, "params": [param[a:a + n] for a, n in spans], "grads": [flat[a:a + n].clone() for a, n in spans],
            "where": torch.nonzero(real).reshape(-1), "decay": (owner < _weights(case)).float() * DECAY, "exp_avg": exp_avg,
            "exp_avg_sq": exp_avg_sq, "max_norm": 1.0 if case["clip"] else 0.0, "step": STEP}


def _prepare_adamw(case, seed):
    s = _inputs_adamw(case, seed)
    m, v = s.pop("exp_avg"), s.pop("exp_avg_sq")
    if own:
        from mqgan_amd.optim import AdamW
        n, params = _weights(case), s.pop("params")                                          # weights decay; gains and biases do not
        groups = [{"params": params[:n]}, {"params": params[n:], "weight_decay": 0.0}]
        s["opt"] = AdamW([g for g in groups if g["params"]], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
        s["opt"].load_moments(m, v, step=STEP)
    elif case["bits"] == 8:
        s["m"], s["v"] = _encode(m, 4, None), _encode(v, 5, None)
    else:
        s["m"], s["v"] = m, v
    return s


def _mix(x):
    """The 32-bit finaliser that the random bits of the 8-bit moments come from, on int64 tensors that hold 32-bit words (or on a number)."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_words(n, step):
    """One 32-bit word for each position of the moments' layout, for one step."""
    seed = (SEED + step * 0xD1B54A32D192ED03) & 0xFFFFFFFFFFFFFFFF
    lo, hi = seed & 0xFFFFFFFF, seed >> 32
    k0 = lo ^ _mix(hi ^ 0x85EBCA6B)
    k1 = _mix((hi + _mix(lo ^ 0xC2B2AE35)) & 0xFFFFFFFF)
    i = torch.arange(n, device="cuda")
    return (_mix(((i & 0xFFFFFFFF) ^ k0) + (i >> 32) * 0x9E3779B1 & 0xFFFFFFFF) + k1) & 0xFFFFFFFF


def _encode(x, exponent_bits, words):
    """(codes uint8, base uint8 per group): sign (4 exponent bits) or none (5), `exponent_bits`, 3 mantissa bits over the group's base.
    words: 16 random bits each, or None for rounding to nearest."""
    bits = x.abs().view(torch.int32).reshape(-1, GROUP)
    top = torch.where(bits < 0x7F800000, bits, 0).amax(1, keepdim=True) >> 23
    base = (top + 1 - (2 ** exponent_bits - 1)).clamp(min=0)
    add = 0x7FFFF + ((bits >> 20) & 1) if words is None else (words.to(torch.int32) << 4).reshape(-1, GROUP)
    most = 2 ** (exponent_bits + 3)
    code = ((bits + add) >> 20) - 8 * base
    code = torch.where(code < 1, ((bits > 0) & (exponent_bits == 5)).int(), code)
    code = torch.where(bits >= 0x7F800000, torch.where(bits == 0x7F800000, most - 2, most - 1), code)
    if exponent_bits == 4:
        code = code | torch.where((x.reshape(-1, GROUP) < 0) & (code > 0), 128, 0)
    return code.to(torch.uint8).reshape(-1), base.to(torch.uint8).reshape(-1)


def _decode(held, exponent_bits):
    codes, base = held
    most = 2 ** (exponent_bits + 3)
    c = codes.reshape(-1, GROUP).int()
    k = c & (most - 1)
    bits = torch.where(k > 0, (k + 8 * base.int()[:, None]) << 20, 0)
    bits = torch.where(k >= most - 2, torch.where(k == most - 2, 0x7F800000, 0x7FC00000), bits)
    x = bits.to(torch.int32).view(torch.float32)
    return (torch.where(c >= 128, -x, x) if exponent_bits == 4 else x).reshape(-1)


def _adamw(s):
    case = s["case"]
    s["step"] += 1
    if own:
        s["opt"].step(max_norm=s["max_norm"], grads=s["grads"])
        m, v = s["opt"].moments(torch.bfloat16 if case["bits"] == 8 else torch.float32)
        return [s["param"], m, v]
    t = s["step"]
    g = torch.zeros_like(s["param"])
    g[s["where"]] = torch.cat(s["grads"]).float()
    if s["max_norm"]:
        norm = g.double().square().sum().sqrt()
        g = g * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    m, v = (_decode(s["m"], 4), _decode(s["v"], 5)) if case["bits"] == 8 else (s["m"], s["v"])
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g * g
    update = m / (v.sqrt() / math.sqrt(1 - BETAS[1] ** t) + EPS)
    s["param"].copy_(s["param"] * (1 - LR * s["decay"]) - LR / (1 - BETAS[0] ** t) * update)
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
        return [s["param"], m, v]
    words = _random_words(len(m), t)
    s["m"], s["v"] = _encode(m, 4, words >> 16), _encode(v, 5, words & 0xFFFF)
    return [s["param"], _decode(s["m"], 4).bfloat16(), _decode(s["v"], 5).bfloat16()]


def _exact_adamw(case, seed):
    s = _inputs_adamw(case, seed)
    t, n = STEP + 1, s["param"].numel()

    def held(codes, base, signed):
        c = codes.long()
        k = (c % 128 if signed else c) + 8 * base.long().repeat_interleave(GROUP)
        value = torch.ldexp(1.0 + (k % 8).double() / 8, (k // 8 - 127).double())
        return torch.where((c % 128 if signed else c) == 0, 0.0, torch.where((c >= 128) & signed, -value, value))

    def keep(x, exponent_bits, r):
        a = x.abs()
        top = torch.floor(torch.log2(a.reshape(-1, GROUP).amax(1).clamp(min=1e-300))).repeat_interleave(GROUP)
        low = top + 1 - (2 ** exponent_bits - 1)                                             # the lowest binade that has codes
        e = torch.floor(torch.log2(a.clamp(min=1e-300)))
        step = torch.exp2(e - 3)
        q = torch.floor(a / step + r.double() / 65536) * step
        first = torch.exp2(low) * 1.125                                                      # code 1
        q = torch.where((q < first) & (a > 0), first if exponent_bits == 5 else 0.0, q)
        return torch.where(a > 0, q, 0.0) * torch.sign(x)

    g = torch.zeros(n, dtype=torch.float64, device="cuda")
    g[s["where"]] = torch.cat([x.double() for x in s["grads"]])
    if s["max_norm"]:
        g *= min(1.0, s["max_norm"] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    m, v = s["exp_avg"], s["exp_avg_sq"]
    m, v = (held(*_encode(m, 4, None), True), held(*_encode(v, 5, None), False)) if case["bits"] == 8 else (m.double(), v.double())
    m = m + (1 - BETAS[0]) * (g - m)
    v = v + (1 - BETAS[1]) * (g * g - v)
    hat_m, hat_v = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    p = s["param"].double()
    p = p - LR * s["decay"].double() * p - LR * hat_m / (hat_v.sqrt() + EPS)
    if case["bits"] == 8:
        words = _random_words(n, t)
        m, v = keep(m, 4, words >> 16), keep(v, 5, words & 0xFFFF)
    return [p, m, v]


# ----------------------------------------------------------------------------- balance
def _prepare_balance(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    n, e, k = case["rows"], case["codes"], case["per_row"]
    favour = torch.randn(e, device="cuda", generator=gen)                                    # some codes are used more: what the loss is for
    logits = (2.0 * torch.randn(n, e, device="cuda", generator=gen) + favour).to(DTYPES[case["dtype"]])
    padded = torch.rand(n, device="cuda", generator=gen) < case["padded"]
    idx = torch.topk(logits.float(), k, dim=1).indices.int()
    return {"op": "balance", "logits": logits.requires_grad_(own), "idx": idx, "padded": padded.to(torch.uint8)}


def _balance(s):
    z, idx, padded = s["logits"], s["idx"], s["padded"]
    if own:
        from mqgan_amd.losses import code_balance_loss
        loss, counts = code_balance_loss(z, idx, padded)
        return [loss, counts, torch.autograd.grad(loss, z)[0]]
    e, k = z.shape[1], idx.shape[1]
    valid = padded == 0
    x = z.float()
    p = torch.exp(x - x.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True) * valid[:, None]
    nv = valid.sum().clamp(min=1)
    counts = torch.zeros(e, dtype=torch.int32, device=z.device)
    counts.index_add_(0, idx.reshape(-1), valid.int().repeat_interleave(k))
    f = counts.double() / (nv * k)
    mean = p.sum(0, dtype=torch.float64) / nv
    loss = (e * (f * mean).sum()).float()
    f = f.float()
    grad = (e / nv.double()).float() * p * (f - (p * f).sum(1, keepdim=True))
    return [loss, counts, grad.to(z.dtype)]


def _exact_balance(case, seed):
    s = _prepare_balance(case, seed)
    z = s["logits"].detach().double()
    keep = torch.nonzero(s["padded"] == 0).reshape(-1)
    e = z.shape[1]
    rows = z[keep]
    p = torch.softmax(rows, 1)
    chosen = s["idx"][keep].long()
    f = torch.bincount(chosen.reshape(-1), minlength=e).double()
    counts = f.to(torch.int32)
    f = f / max(1, chosen.numel())
    share = p @ f                                                                            # what of a row's mass lies on how used codes
    many = max(1, len(keep))
    grad = torch.zeros_like(z)
    grad[keep] = p * (f - share[:, None]) * (e / many)
    return [share.sum() * e / many, counts, grad]


# ----------------------------------------------------------------------------- sample
def _prepare_sample(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    n = case["rows"]
    logits = (3.0 * torch.randn(n, case["codes"], device="cuda", generator=gen)).to(DTYPES[case["dtype"]])
    s = {"op": "sample", "logits": logits, "u": torch.rand(n, device="cuda", generator=gen), "temperature": 0.8, "top_k": case["top_k"],
         "top_p": case["top_p"], "min_p": case["min_p"]}
    if case["by_row"]:
        s["temperature"] = 0.5 + torch.rand(n, device="cuda", generator=gen)
        s["top_p"] = 1 - (1 - case["top_p"]) * torch.rand(n, device="cuda", generator=gen)
        s["min_p"] = case["min_p"] * torch.rand(n, device="cuda", generator=gen)
        s["top_k"] = torch.randint(0, case["top_k"] + 1, (n,), device="cuda", generator=gen, dtype=torch.int32)
    return s


def _column(v, like):
    return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((1, 1), float(v), dtype=torch.float64, device=like.device)


def _sample(s):
    z, u = s["logits"], s["u"]
    if own:
        from mqgan_amd import ops
        idx, logp = ops.sample_codes(z, u, temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], return_logp=True)
        return [idx, logp]
    x, order = torch.sort(z.float(), dim=1, descending=True, stable=True)
    x = x.double()
    d = (x - x[:, :1]) / _column(s["temperature"], z)
    w = torch.exp(d)                                            # 64 bits: a draw next to a border has to fall on the right side of it
    rank = torch.arange(z.shape[1], device=z.device)[None]
    k = _column(s["top_k"], z)
    w = torch.where((k > 0) & (rank >= k), 0.0, w)
    before = w.cumsum(1) - w
    p = _column(s["top_p"], z)
    w = torch.where((p < 1) & (rank > 0) & (before >= p * w.sum(1, keepdim=True)), 0.0, w)
    w = torch.where(w >= _column(s["min_p"], z), w, 0.0)
    total = w.sum(1, keepdim=True)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    reach = by_index.cumsum(1)
    idx = ((reach > u.double()[:, None] * reach[:, -1:]) & (by_index > 0)).int().argmax(1, keepdim=True)
    logp = torch.log(by_index.gather(1, idx) / total)
    return [idx[:, 0], logp[:, 0].float()]


def _exact_sample(case, seed):
    """Without an order: a code's place is the number of codes before it, found for the codes above a bisected border of the score."""
    s = _prepare_sample(case, seed)
    z, n = s["logits"].double(), case["rows"]
    rows = lambda v: v.double() if isinstance(v, torch.Tensor) else torch.full((n,), float(v), dtype=torch.float64, device="cuda")  # noqa: E731
    t, k, top_p, min_p = rows(s["temperature"]), rows(s["top_k"]), rows(s["top_p"]), rows(s["min_p"])
    top = z.amax(1, keepdim=True)
    w = torch.exp((z - top) / t[:, None])

    def cut(w, ask):
        """Lowest score that `ask(mass or count strictly above it)` still takes, ties of it counted off in index order."""
        lo, hi = z.amin(1), top[:, 0].clone()
        for _ in range(70):
            mid = (lo + hi) / 2
            taken = ask(z > mid[:, None], w)
            lo, hi = torch.where(taken, lo, mid), torch.where(taken, mid, hi)
        at = torch.where(z <= hi[:, None], z, -math.inf).amax(1, keepdim=True)
        return at

    if bool((k > 0).any()):
        at = cut(w, lambda m, w: m.sum(1) < k)
        above, tie = z > at, z == at
        kept = above | (tie & (tie.long().cumsum(1) + above.sum(1, keepdim=True) <= k[:, None])) | (k <= 0)[:, None]
        w = w * kept
    if bool((top_p < 1).any()):
        goal = top_p * w.sum(1)
        at = cut(w, lambda m, w: (w * m).sum(1) < goal)
        above, tie = z > at, z == at
        ties = torch.where(tie, w, 0.0)
        before = (w * above).sum(1, keepdim=True) + ties.cumsum(1) - ties
        kept = above | (tie & (before < goal[:, None])) | (top_p >= 1)[:, None]
        first = torch.zeros_like(kept).scatter_(1, z.argmax(1, keepdim=True), True)
        w = w * (kept | first)
    w = w * (w >= min_p[:, None])
    reach = w.cumsum(1)
    goal = s["u"].double() * reach[:, -1]
    idx = torch.searchsorted(reach, goal[:, None], right=True).clamp(max=z.shape[1] - 1)
    return [idx[:, 0], torch.log(w.gather(1, idx) / reach[:, -1:])[:, 0]]


# ----------------------------------------------------------------------------- the interface
def prepare(case, seed):
    return {"adamw": _prepare_adamw, "balance": _prepare_balance, "sample": _prepare_sample}[case["op"]](case, seed)


def run(state):
    return {"adamw": _adamw, "balance": _balance, "sample": _sample}[state["op"]](state)


def exact(case, seed):
    return {"adamw": _exact_adamw, "balance": _exact_balance, "sample": _exact_sample}[case["op"]](case, seed)


def work(case):
    if case["op"] == "adamw":
        n = int(_sizes(case).sum())
        g = 4 if case["grad"] == "f32" else 2
        moments = 2 * (4 + 4) if case["bits"] == 32 else 2 * (1 + 1 + 2 / GROUP) + 2 * 2       # 8 bits: the values come back as bf16 too
        return {"bytes": n * (4 + 4 + g + moments), "flops": 16 * n}
    item = 4 if case["dtype"] == "f32" else 2
    n, e = case["rows"], case["codes"]
    if case["op"] == "balance":
        return {"bytes": n * e * item * 2 + n * case["per_row"] * 4 + n + e * 4 + 4, "flops": 12 * n * e}
    return {"bytes": n * e * item + n * (4 + 8 + 4), "flops": 8 * n * e}
