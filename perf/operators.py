"""Cases of the training-side row operators: token log-probabilities, the clipped policy loss and the
preference loss on logits, the residual path of a block (norm after it, gate, dropout, residual scale,
norm before the next one) and dropout from a counter-based generator.

`own` selects what run() calls: the framework's kernels, or the same operators written in elementary
torch operations.  Tensors are made on the GPU from the seed alone.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORED = -100            # label of a token that takes no part
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
BETA, SMOOTHING = 0.1, 0.05
EPS = 1e-6
SCALE = 0.7


def listed():
    return [
        # one sampled token: what a call costs before there is any work
        {"name": "policy 1x32000 bf16", "op": "policy", "batch": 1, "tokens": 1, "vocab": 32000, "dtype": "bf16", "masked": 0.0, "shift": False},
        # four sequences, logits shifted against their labels (views), a vocabulary of odd size
        {"name": "policy 4x1023x50021 bf16", "op": "policy", "batch": 4, "tokens": 1023, "vocab": 50021, "dtype": "bf16", "masked": 0.25, "shift": True},
        # a packed micro-batch over a large vocabulary; the largest case
        {"name": "policy 4096x151936 bf16", "op": "policy", "batch": 1, "tokens": 4096, "vocab": 151936, "dtype": "bf16", "masked": 0.1, "shift": False},
        # scores of sampled tokens under a reference model: forward only
        {"name": "logprobs 256x151936 f32", "op": "logprobs", "batch": 1, "tokens": 256, "vocab": 151936, "dtype": "f32", "masked": 0.0, "shift": False, "grad": False},
        # forward and backward for a loss of the user's own
        {"name": "logprobs 512x32768 f16", "op": "logprobs", "batch": 1, "tokens": 512, "vocab": 32768, "dtype": "f16", "masked": 0.0, "shift": False, "grad": True},
        # two short pairs
        {"name": "preference 2 pairs 317x32000 f16", "op": "preference", "pairs": 2, "rows": 317, "vocab": 32000, "dtype": "f16"},
        # sixteen ragged pairs in one packed batch, padded rows at its end
        {"name": "preference 16 pairs 3001x151936", "op": "preference", "pairs": 16, "rows": 3001, "vocab": 151936, "dtype": "bf16"},
        # one token on its way through a block when serving
        {"name": "block 1x4096 bf16", "op": "block", "batch": 1, "tokens": 1, "width": 4096, "dtype": "bf16", "gate": "none", "p": 0.0, "grad": False},
        # a training step of odd sizes, one gate row per sequence
        {"name": "block 8x125x1023 f32 train", "op": "block", "batch": 8, "tokens": 125, "width": 1023, "dtype": "f32", "gate": "sequence", "p": 0.1, "grad": True},
        # an ordinary training micro-batch, a gate for every element
        {"name": "block 4x4096x4096 bf16 train", "op": "block", "batch": 4, "tokens": 4096, "width": 4096, "dtype": "bf16", "gate": "element", "p": 0.1, "grad": True},
        # a small activation of odd width
        {"name": "dropout 257x333 f32", "op": "dropout", "rows": 257, "width": 333, "dtype": "f32", "p": 0.1},
        # activations of a training micro-batch, forward and backward
        {"name": "dropout 16384x8192 bf16", "op": "dropout", "rows": 16384, "width": 8192, "dtype": "bf16", "p": 0.1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["policy", "policy", "logprobs", "preference", "block", "block", "dropout"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    size = 4 if dtype == "f32" else 2
    if op in ("policy", "logprobs"):
        vocab = _log_int(rng, 200, 200000)
        batch = rng.choice([1, 1, 2, 3, 4])
        most = max(1, min(4096, 1_200_000_000 // (vocab * size)) // batch)
        case = {"op": op, "batch": batch, "tokens": _log_int(rng, 1, most), "vocab": vocab, "dtype": dtype,
                "masked": rng.choice([0.0, 0.1, 0.5]), "shift": rng.random() < 0.3}
        if op == "logprobs":
            case["grad"] = rng.random() < 0.5
        return case
    if op == "preference":
        vocab = _log_int(rng, 200, 200000)
        pairs = _log_int(rng, 1, 32)
        most = max(16, min(4096, 800_000_000 // (vocab * size)))
        return {"op": op, "pairs": pairs, "rows": _log_int(rng, 16, most), "vocab": vocab, "dtype": dtype}
    if op == "block":
        width = _log_int(rng, 64, 16384)
        if rng.random() < 0.7:
            width = -(-width // 64) * 64
        batch = rng.choice([1, 2, 4, 8])
        most = max(1, 130_000_000 // (width * size) // batch)
        return {"op": op, "batch": batch, "tokens": _log_int(rng, 1, min(16384, most)), "width": width, "dtype": dtype,
                "gate": rng.choice(["none", "vector", "sequence", "element"]), "p": rng.choice([0.0, 0.1, 0.5]), "grad": rng.random() < 0.6}
    rows = _log_int(rng, 1, 16384)
    width = _log_int(rng, 1, 8192)
    return {"op": op, "rows": rows, "width": width, "dtype": dtype, "p": round(rng.uniform(0.01, 0.9), 3)}


# ---------------------------------------------------------------------------------- inputs ----

def _logits(shape, dtype, labels, g, dev):
    """Logits of a model that mostly agrees with the sampled tokens."""
    x = torch.empty(shape, dtype=dtype, device=dev)
    flat, lab = x.view(-1, shape[-1]), labels.reshape(-1)
    for r in range(0, flat.shape[0], 512):
        v = torch.randn(flat[r:r + 512].shape, device=dev, generator=g) * 2.0
        at = lab[r:r + 512].clamp_min(0).unsqueeze(1)
        v.scatter_add_(1, at, 4.0 + 6.0 * torch.rand(at.shape, device=dev, generator=g))
        flat[r:r + 512] = v.to(dtype)
    return x


def _scores(x, labels):
    """Log-probabilities of the labels, to make the older policy's from."""
    flat, lab = x.reshape(-1, x.shape[-1]), labels.reshape(-1).clamp_min(0)
    got = torch.empty(flat.shape[0], dtype=torch.float64, device=x.device)
    for r in range(0, flat.shape[0], 512):
        v = flat[r:r + 512].double()
        got[r:r + 512] = v.gather(1, lab[r:r + 512].unsqueeze(1)).squeeze(1) - v.logsumexp(1)
    return got.view(labels.shape)


def _off_border(noise):
    """Keeps exp(-noise) a little away from both ends of the clip range, where rounding decides the branch."""
    for end in (-math.log(1.0 + CLIP_HIGH), -math.log(1.0 - CLIP_LOW)):
        noise = torch.where((noise - end).abs() < 1e-3, noise + 4e-3, noise)
    return noise


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    if op in ("policy", "logprobs"):
        b, t, v = case["batch"], case["tokens"], case["vocab"]
        full = t + 1 if case["shift"] else t
        labels = torch.randint(0, v, (b, full), device=dev, generator=g)
        lost = torch.rand(b, full, device=dev, generator=g) < case["masked"]
        lost[:, -1] = False
        if case["shift"]:
            # the logits at a position score the token behind it
            x = _logits((b, full, v), dtype, labels.roll(-1, 1), g, dev)[:, :-1]
            labels, lost = labels[:, 1:], lost[:, 1:]
        else:
            x = _logits((b, full, v), dtype, labels, g, dev)
        if b == 1:
            x, labels, lost = x[0], labels[0], lost[0]
        state = {"case": case, "logits": x, "labels": labels}
        if op == "logprobs":
            if case["masked"]:
                labels.masked_fill_(lost, IGNORED)
            state["grad_logp"] = torch.randn(labels.shape, device=dev, generator=g)
            return state
        logp = _scores(x, labels)
        state["old_logp"] = (logp + _off_border(0.2 * torch.randn(labels.shape, device=dev, generator=g))).float()
        state["ref_logp"] = (logp + 0.3 * torch.randn(labels.shape, device=dev, generator=g)).float()
        advantage = torch.randn((b, 1) if b > 1 else (1,), device=dev, generator=g) + 0.3 * torch.randn(labels.shape, device=dev, generator=g)
        state["advantages"] = advantage
        kept = (~lost).float()
        state["weights"] = kept / kept.sum().clamp_min(1.0)
        return state
    if op == "preference":
        n, v, p = case["rows"], case["vocab"], case["pairs"]
        share = 0.4 + torch.rand(2 * p, device=dev, generator=g)
        used = n - n // 16
        ends = (share.cumsum(0) / share.sum() * used).round().long()
        offsets = torch.cat([ends.new_zeros(1), ends])
        labels = torch.randint(0, v, (n,), device=dev, generator=g)
        x = _logits((n, v), dtype, labels, g, dev)
        row = torch.arange(n, device=dev)
        seq = (torch.searchsorted(offsets, row, right=True) - 1).clamp(0, 2 * p - 1)
        begin, end = offsets[seq], offsets[seq + 1]
        prompt = row < begin + (end - begin) // 4           # the prompt's tokens are not scored
        ref = (_scores(x, labels) + 0.3 * torch.randn(n, device=dev, generator=g)).float()
        labels = labels.masked_fill(prompt, IGNORED)
        return {"case": case, "logits": x, "labels": labels, "ref_logp": ref, "offsets": offsets}
    if op == "block":
        b, t, d = case["batch"], case["tokens"], case["width"]
        make = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
        gate = {"none": None, "vector": (d,), "sequence": (b, 1, d), "element": (b, t, d)}[case["gate"]]
        return {"case": case, "x": (3.0 * make(b, t, d)).to(dtype), "h": make(b, t, d).to(dtype),
                "post": (1.0 + 0.1 * make(d)).to(dtype), "next": (1.0 + 0.1 * make(d)).to(dtype),
                "gate": None if gate is None else torch.sigmoid(make(*gate)).to(dtype),
                "dx": make(b, t, d).to(dtype), "dy": make(b, t, d).to(dtype),
                "seed": 0x9E3779B97F4A7C15 ^ (seed * 0x2545F491), "offset": seed % 1000}
    x = torch.randn(case["rows"], case["width"], device=dev, generator=g).to(dtype)
    dy = torch.randn(case["rows"], case["width"], device=dev, generator=g).to(dtype)
    return {"case": case, "x": x, "dy": dy, "seed": 0x9E3779B97F4A7C15 ^ (seed * 0x2545F491), "offset": seed % 1000}


# ---------------------------------------------------------------------------------- one pass --

def run(state):
    op = state["case"]["op"]
    if own:
        return {"policy": _own_policy, "logprobs": _own_logprobs, "preference": _own_preference, "block": _own_block, "dropout": _own_dropout}[op](state)
    return {"policy": _policy, "logprobs": _logprobs, "preference": _preference, "block": _block, "dropout": _dropout}[op](state)


def _own_policy(s):
    import tensorplay_b200 as tpb
    loss, grad, logp, ratio, kl = tpb.policy_loss(s["logits"], s["labels"], s["old_logp"], s["advantages"], s["weights"], s["ref_logp"],
                                                  clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF)
    return {"loss": loss, "grad": grad, "logp": logp, "ratio": ratio, "kl": kl}


def _own_logprobs(s):
    import tensorplay_b200 as tpb
    logp, lse = tpb.token_logprobs(s["logits"], s["labels"])
    out = {"logp": logp, "lse": lse}
    if s["case"]["grad"]:
        out["grad"] = tpb.token_logprobs_backward(s["grad_logp"], s["logits"], s["labels"], lse)
    return out


def _own_preference(s):
    import tensorplay_b200 as tpb
    loss, grad, rewards, logp = tpb.preference_loss(s["logits"], s["labels"], s["ref_logp"], s["offsets"], beta=BETA, label_smoothing=SMOOTHING)
    return {"loss": loss, "grad": grad, "rewards": rewards, "logp": logp}


def _own_block(s):
    import tensorplay_b200 as tpb
    how = {"scale": SCALE, "p": s["case"]["p"], "seed": s["seed"], "offset": s["offset"]}
    x, y, rstd_post, rstd_next = tpb.block_residual(s["x"], s["h"], s["post"], s["next"], s["gate"], eps=EPS, **how)
    out = {"x": x, "y": y}
    if s["case"]["grad"]:
        # y went by x before its rounding: so do the gradients
        dx, dh, dpost, dnext, dgate = tpb.block_residual_backward(s["dx"], s["dy"], s["h"], x, rstd_post, rstd_next, s["post"], s["next"], s["gate"],
                                                                  x=s["x"], **how)
        out.update(dx=dx, dh=dh, dpost=dpost, dnext=dnext)
        if dgate is not None:
            out["dgate"] = dgate
    return out


def _own_dropout(s):
    import tensorplay_b200 as tpb
    p, seed, offset = s["case"]["p"], s["seed"], s["offset"]
    return {"y": tpb.dropout(s["x"], p, seed, offset), "dx": tpb.dropout_backward(s["dy"], p, seed, offset)}


def _log_normaliser(x):
    """(row maximum, log of the sum of exp(x - maximum)): their sum in 64 bits is the normaliser."""
    top = x.amax(-1, keepdim=True)
    return top, (x - top).exp().sum(-1, keepdim=True, dtype=torch.float64).log()


def _scored(x, labels):
    """Log-probabilities in 64 bits (differences of them are small), normalisers, and which tokens count."""
    kept = labels >= 0
    top, log_sum = _log_normaliser(x)
    at = x.gather(-1, labels.clamp_min(0).unsqueeze(-1))
    lse = top.double() + log_sum
    logp = torch.where(kept, (at.double() - lse).squeeze(-1), 0.0)
    return logp, lse, kept


def _grad_of(x, labels, lse, coef):
    """coef * (one at the label - softmax)."""
    out = (x - lse.float()).exp() * -coef.float().unsqueeze(-1)
    # the label's own entry, where one minus a probability near one loses digits
    at = labels.clamp_min(0).unsqueeze(-1)
    p = (x.gather(-1, at).double() - lse).exp()
    return out.scatter(-1, at, ((1.0 - p) * coef.double().unsqueeze(-1)).float())


def _policy(s):
    x, labels, w = s["logits"].float(), s["labels"], s["weights"].double()
    logp, lse, kept = _scored(x, labels)
    kept = kept & (w != 0)
    adv = s["advantages"].double()
    ratio = (logp - s["old_logp"].double()).exp()
    plain, held = ratio * adv, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
    d = s["ref_logp"].double() - logp
    kl = d.exp() - d - 1.0
    each = -torch.minimum(plain, held) + KL_COEF * kl
    slope = torch.where(plain <= held, -plain, 0.0) + KL_COEF * (1.0 - d.exp())
    loss = torch.where(kept, w * each, 0.0).sum()
    grad = _grad_of(x, labels, lse, torch.where(kept, w * slope, 0.0))
    zero = torch.zeros_like(logp)
    return {"loss": loss.float(), "grad": grad.to(s["logits"].dtype), "logp": torch.where(kept, logp, zero).float(),
            "ratio": torch.where(kept, ratio, zero).float(), "kl": torch.where(kept, kl, zero).float()}


def _logprobs(s):
    x, labels = s["logits"].float(), s["labels"]
    logp, lse, kept = _scored(x, labels)
    out = {"logp": logp.float(), "lse": torch.where(kept, lse.squeeze(-1), 0.0).float()}
    if s["case"]["grad"]:
        out["grad"] = _grad_of(x, labels, lse, torch.where(kept, s["grad_logp"], 0.0)).to(s["logits"].dtype)
    return out


def _preference(s):
    x, labels, offsets = s["logits"].float(), s["labels"], s["offsets"]
    n, pairs = x.shape[0], s["case"]["pairs"]
    logp, lse, kept = _scored(x, labels)
    row = torch.arange(n, device=x.device)
    seq = (offsets[1:].unsqueeze(1) <= row).sum(0)               # the sequence of every row, 2 * pairs behind the last one
    kept = kept & (seq < 2 * pairs)
    logp = torch.where(kept, logp, 0.0)
    each = torch.where(kept, logp - s["ref_logp"].double(), 0.0)
    sums = (each * (seq == torch.arange(2 * pairs, device=x.device).unsqueeze(1))).sum(1)
    margin = BETA * (sums[0::2] - sums[1::2])
    won, lost = 1.0 / (1.0 + (-margin).exp()), 1.0 / (1.0 + margin.exp())
    loss = (-(1.0 - SMOOTHING) * won.log() - SMOOTHING * lost.log()).mean()
    slope = BETA * (SMOOTHING * won - (1.0 - SMOOTHING) * lost) / pairs
    per_seq = torch.stack([slope, -slope], 1).reshape(-1)
    coef = torch.where(kept, per_seq[seq.clamp_max(2 * pairs - 1)], 0.0)
    grad = _grad_of(x, labels, lse, coef)
    return {"loss": loss.float(), "grad": grad.to(s["logits"].dtype), "rewards": (BETA * sums).float(), "logp": logp.float()}


M32 = 0xFFFFFFFF


def _kept(n, p, seed, offset, dev):
    """Truth values of n elements: ten rounds of Philox 4x32 on the counter (i // 8, offset) under the key
    `seed`; element i takes 16 bits of the block, and is kept if they reach p in units of 2^-16."""
    block = torch.arange(-(-n // 8), device=dev, dtype=torch.int64)
    c0, c1 = block & M32, block >> 32
    c2, c3 = torch.full_like(c0, offset & M32), torch.full_like(c0, (offset >> 32) & M32)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((m1 >> 32) & M32) ^ c1 ^ k0, m1 & M32, ((m0 >> 32) & M32) ^ c3 ^ k1, m0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    words = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1)
    return words.reshape(-1)[:n] >= _units(p)


def _units(p):
    """The drop probability in units of 2^-16, which is what 16 bits can express."""
    return int(math.floor(p * 65536.0 + 0.5))


def _factor(like, p, seed, offset):
    """0 for a dropped element and 1 / (1 - p) for a kept one."""
    if _units(p) == 0:
        return torch.ones((), device=like.device)
    keep = _kept(like.numel(), p, seed, offset, like.device).view(like.shape)
    return keep.float() * (65536.0 / (65536 - _units(p)))


def _dropout(s):
    f = _factor(s["x"], s["case"]["p"], s["seed"], s["offset"])
    return {"y": (s["x"].float() * f).to(s["x"].dtype), "dx": (s["dy"].float() * f).to(s["x"].dtype)}


def _norm_grad(dy, hat, rstd):
    """Gradient of hat = v * rstd with respect to v, for the gradient dy of hat."""
    return rstd * (dy - hat * (dy * hat).mean(-1, keepdim=True))


def _block(s):
    dtype = s["x"].dtype
    x, h, post, nxt = s["x"].float(), s["h"].float(), s["post"].float(), s["next"].float()
    f = _factor(h, s["case"]["p"], s["seed"], s["offset"])
    gate = torch.ones((), device=x.device) if s["gate"] is None else s["gate"].float()
    rstd_post = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hat = h * rstd_post
    branch = hat * post * f
    x_out = x + SCALE * gate * branch
    rstd_next = (x_out.square().mean(-1, keepdim=True) + EPS).rsqrt()
    x_hat = x_out * rstd_next
    out = {"x": x_out.to(dtype), "y": (x_hat * nxt).to(dtype)}
    if not s["case"]["grad"]:
        return out
    dy = s["dy"].float()
    total = s["dx"].float() + _norm_grad(dy * nxt, x_hat, rstd_next)
    dn = SCALE * gate * f * total
    out["dx"] = total.to(dtype)
    out["dh"] = _norm_grad(dn * post, hat, rstd_post).to(dtype)
    out["dpost"] = (dn * hat).sum((0, 1)).to(dtype)
    out["dnext"] = (dy * x_hat).sum((0, 1)).to(dtype)
    if s["gate"] is not None:
        dgate = SCALE * branch * total
        kind = s["case"]["gate"]
        dgate = dgate if kind == "element" else dgate.sum(1, keepdim=True) if kind == "sequence" else dgate.sum((0, 1))
        out["dgate"] = dgate.to(dtype)
    return out


# ---------------------------------------------------------------------------------- floors ----

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    op = case["op"]
    if op in ("policy", "logprobs"):
        n, v = case["batch"] * case["tokens"], case["vocab"]
        read = n * (1.0 - case["masked"]) * v * size
        write = n * v * size if op == "policy" or case["grad"] else 0.0
        return {"bytes": read + write + n * 40.0, "flops": n * (1.0 - case["masked"]) * v * (8.0 if write else 4.0)}
    if op == "preference":
        n, v = case["rows"], case["vocab"]
        scored = 0.75 * (n - n // 16)
        return {"bytes": (scored + n) * v * size + n * 20.0, "flops": scored * v * 8.0}
    if op == "block":
        n, d = case["batch"] * case["tokens"], case["width"]
        gate = {"none": 0, "vector": d, "sequence": case["batch"] * d, "element": n * d}[case["gate"]]
        forward = 4 * n * d + gate + 2 * d
        if not case["grad"]:
            return {"bytes": forward * float(size), "flops": 10.0 * n * d}
        # inputs once: x, h, gate, both weights, both gradients; outputs: x, y, dx, dh and the other gradients
        return {"bytes": (8 * n * d + 2 * gate + 4 * d) * float(size), "flops": 40.0 * n * d}
    n = case["rows"] * case["width"]
    return {"bytes": 4.0 * n * size, "flops": 4.0 * n}


# ---------------------------------------------------------------------------------- 64 bits ---

def exact(case, seed):
    s = prepare(case, seed)
    return {"policy": _exact_policy, "logprobs": _exact_logprobs, "preference": _exact_preference, "block": _exact_block, "dropout": _exact_dropout}[case["op"]](s)


def _rows64(x, labels, counts):
    """log softmax of the counted rows at their labels, by rows of a few hundred."""
    flat, lab, use = x.reshape(-1, x.shape[-1]), labels.reshape(-1), counts.reshape(-1)
    logp = torch.zeros(lab.shape, dtype=torch.float64, device=x.device)
    norm = torch.zeros_like(logp)
    for r in range(0, lab.shape[0], 256):
        v = flat[r:r + 256].double()
        norm[r:r + 256] = torch.logsumexp(v, 1)
        logp[r:r + 256] = v[torch.arange(v.shape[0], device=v.device), lab[r:r + 256].clamp(min=0)] - norm[r:r + 256]
    return torch.where(use, logp, 0.0).view(labels.shape), torch.where(use, norm, 0.0).view(labels.shape)


def _grad64(x, labels, norm, slope):
    """Derivative of slope . logp for all rows, in 32 bits at the end to save space."""
    flat, lab = x.reshape(-1, x.shape[-1]), labels.reshape(-1)
    norm, slope = norm.reshape(-1), slope.reshape(-1)
    out = torch.zeros(flat.shape, dtype=torch.float32, device=x.device)
    for r in range(0, lab.shape[0], 256):
        v = torch.exp(flat[r:r + 256].double() - norm[r:r + 256, None])
        v = -v
        v[torch.arange(v.shape[0], device=v.device), lab[r:r + 256].clamp(min=0)] += 1.0
        out[r:r + 256] = (torch.where(slope[r:r + 256, None] == 0, 0.0, v) * slope[r:r + 256, None]).float()
    return out.view(x.shape)


def _exact_policy(s):
    labels, w = s["labels"], s["weights"].double()
    use = (labels >= 0) & (w != 0)
    logp, norm = _rows64(s["logits"], labels, use)
    adv, gap = s["advantages"].double(), s["ref_logp"].double() - logp
    ratio = torch.exp(logp - s["old_logp"].double())
    out_of_range = torch.where(adv > 0, ratio > 1 + CLIP_HIGH, ratio < 1 - CLIP_LOW)
    end = torch.where(adv > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)
    gain = torch.where(out_of_range, end, ratio) * adv
    kl = torch.expm1(gap) - gap
    slope = KL_COEF * -torch.expm1(gap) - torch.where(out_of_range, 0.0, ratio * adv)
    mask = use.double()
    return {"loss": (mask * w * (KL_COEF * kl - gain)).sum(), "grad": _grad64(s["logits"], labels, norm, mask * w * slope),
            "logp": logp, "ratio": mask * ratio, "kl": mask * kl}


def _exact_logprobs(s):
    use = s["labels"] >= 0
    logp, norm = _rows64(s["logits"], s["labels"], use)
    out = {"logp": logp, "lse": norm}
    if s["case"]["grad"]:
        out["grad"] = _grad64(s["logits"], s["labels"], norm, use * s["grad_logp"].double())
    return out


def _exact_preference(s):
    bounds, count = s["offsets"].tolist(), s["labels"].shape[0]
    use = s["labels"] >= 0
    use[bounds[-1]:] = False
    logp, norm = _rows64(s["logits"], s["labels"], use)
    gain = torch.where(use, logp - s["ref_logp"].double(), 0.0)
    sums = torch.stack([gain[a:b].sum() for a, b in zip(bounds, bounds[1:])])
    margin = BETA * (sums[0::2] - sums[1::2])
    soft = torch.nn.functional.softplus
    loss = ((1 - SMOOTHING) * soft(-margin) + SMOOTHING * soft(margin)).sum() / margin.numel()
    down = BETA * (torch.sigmoid(margin) - (1 - SMOOTHING)) / margin.numel()
    slope = torch.zeros(count, dtype=torch.float64, device=gain.device)
    for j, (a, b) in enumerate(zip(bounds, bounds[1:])):
        slope[a:b] = down[j // 2] if j % 2 == 0 else -down[j // 2]
    return {"loss": loss, "grad": _grad64(s["logits"], s["labels"], norm, torch.where(use, slope, 0.0)), "rewards": BETA * sums, "logp": logp}


def _philox64(blocks, key, high):
    """The same generator on numpy's unsigned 64-bit integers."""
    import numpy as np
    low = np.uint64(M32)
    with np.errstate(over="ignore"):
        a = np.arange(blocks, dtype=np.uint64)
        ctr = [a & low, a >> np.uint64(32), np.full_like(a, high & M32), np.full_like(a, (high >> 32) & M32)]
        for r in range(10):
            left = ctr[0] * np.uint64(0xD2511F53)
            right = ctr[2] * np.uint64(0xCD9E8D57)
            ka = np.uint64(((key & M32) + r * 0x9E3779B9) & M32)
            kb = np.uint64((((key >> 32) & M32) + r * 0xBB67AE85) & M32)
            ctr = [(right >> np.uint64(32)) ^ ctr[1] ^ ka, right & low, (left >> np.uint64(32)) ^ ctr[3] ^ kb, left & low]
    return np.stack(ctr, 1).astype(np.uint32)


def _keep64(shape, p, seed, offset, dev):
    """Keep factors in 64 bits (the 16-bit halves of the words, low half first)."""
    count, units = math.prod(shape), round(p * 65536)
    if units == 0:
        return torch.ones(shape, dtype=torch.float64, device=dev)
    bits = _philox64((count + 7) // 8, seed, offset).view("<u2").reshape(-1)[:count]
    return torch.from_numpy((bits >= units).astype("float32")).to(dev).double().view(shape) / (1.0 - units / 65536.0)


def _exact_dropout(s):
    f = _keep64(tuple(s["x"].shape), s["case"]["p"], s["seed"], s["offset"], s["x"].device)
    return {"y": s["x"].double() * f, "dx": s["dy"].double() * f}


def _exact_block(s):
    c = s["case"]
    x, h, post, nxt = (s[k].double().requires_grad_(c["grad"]) for k in ("x", "h", "post", "next"))
    gate = None if s["gate"] is None else s["gate"].double().requires_grad_(c["grad"])
    keep = _keep64(tuple(h.shape), c["p"], s["seed"], s["offset"], h.device)
    n = post * h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * keep
    x_out = x + SCALE * (n if gate is None else n * gate)
    y = nxt * x_out / torch.sqrt((x_out * x_out).mean(-1, keepdim=True) + EPS)
    out = {"x": x_out.detach(), "y": y.detach()}
    if c["grad"]:
        wanted = [x, h, post, nxt] + ([] if gate is None else [gate])
        got = torch.autograd.grad([x_out, y], wanted, [s["dx"].double(), s["dy"].double()])
        out.update(zip(("dx", "dh", "dpost", "dnext", "dgate"), got))
    return out
