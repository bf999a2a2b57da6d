"""Plain 64-bit implementations of the training operators (torch float64, from the formulas), and the
bounds that the float32 kernels are held to.

Bounds.  u = eps(type) / 2 is one rounding of the output.  Objectives on logits: the exponent c (x - m) is a
difference and a product, two roundings of 2^-24 of its size (|c (x - m)| <= 48 in these tests for every entry
that counts: 5.8e-6 as an exponent of 2, 4.0e-6 of the value), ex2 is off by 2^-22, a sum of at most 64 float32
terms per thread by 64 * 2^-24 = 3.8e-6.  So a probability is off by at most P = 9e-6 of itself, and a
log-probability by at most P absolutely.  Where the normaliser comes back as a float32 (the separate backward
call) 2^-24 |lse| is added.
"""
import torch

P = 9e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half the smallest positive value of the type: what a result that underflows is off by
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, what=""):
    # a value beyond the largest of the type rounds to infinity
    top = torch.finfo(got.dtype).max
    got, want = got.double(), want.double()
    want = torch.where(want.abs() > top * (1 + 2.0 ** -9), want.sign() * float("inf"), want)
    tol = torch.as_tensor(tol, dtype=torch.float64, device=want.device).expand(want.shape)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN pattern differs"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    fine = want.isfinite()
    over = ((got - want).abs() - tol)[fine]
    if over.numel() and not bool((over <= 0).all()):
        i = int(over.argmax())
        raise AssertionError(f"{what}: {got[fine][i].item()!r} against {want[fine][i].item()!r}, over the bound {tol[fine][i].item():.3e} by {over[i].item():.3e}")


def scores(x, labels):
    """(logp, lse, takes part) in 64 bits; a label beyond the vocabulary gives NaN."""
    use = labels >= 0
    v = x.shape[-1]
    lse = torch.logsumexp(x.double(), -1)
    lse = torch.where(torch.isneginf(lse), torch.full_like(lse, float("nan")), lse)      # x - max is NaN there
    lse = torch.where(x.double().isposinf().any(-1), torch.full_like(lse, float("nan")), lse)
    at = x.double().gather(-1, labels.clamp(0, v - 1).unsqueeze(-1)).squeeze(-1)
    logp = torch.where(labels < v, at - lse, torch.full_like(lse, float("nan")))
    return torch.where(use, logp, 0.0), torch.where(use, lse, 0.0), use


def grad_of(x, labels, coef):
    """coef * (one at the label - softmax), and the bound of the kernels' error before rounding."""
    v = x.shape[-1]
    logp, lse, _ = scores(x, labels)
    p = (x.double() - lse.unsqueeze(-1)).exp()
    hit = torch.nn.functional.one_hot(labels.clamp(0, v - 1), v).bool() & ((labels >= 0) & (labels < v)).unsqueeze(-1)
    g = torch.where(hit, -torch.expm1(logp).unsqueeze(-1), -p)
    g = torch.where(labels.unsqueeze(-1) >= v, torch.full_like(g, float("nan")), g)
    c = coef.double().unsqueeze(-1)
    g = torch.where(c == 0, torch.zeros_like(g), g * c)
    return g, (c * p).abs() * P + g.abs() * 2.0 ** -21      # at the label d(1 - p) = dp as well; expm1, products


def policy(x, labels, old, adv, w, ref, low, high, kl_coef):
    logp, lse, use = scores(x, labels)
    old, adv, w = (t.double().expand(labels.shape) for t in (old, adv, w))
    use = use & (w != 0)
    logp = torch.where(use, logp, 0.0)
    r = (logp - old).exp()
    plain, held = r * adv, r.clamp(1 - low, 1 + high) * adv
    clipped = held < plain
    each = -torch.where(clipped, held, plain)
    slope = -torch.where(clipped, 0.0, plain)
    kl, dkl = torch.zeros_like(logp), torch.zeros_like(logp)
    if ref is not None:
        d = ref.double().expand(labels.shape) - logp
        kl, dkl = torch.expm1(d) - d, -torch.expm1(d)
        each, slope = each + kl_coef * kl, slope + kl_coef * dkl
    z = torch.zeros_like(logp)
    keep = lambda t: torch.where(use, t, z)  # noqa: E731
    out = {"logp": logp, "ratio": keep(r), "kl": keep(kl), "each": keep(w * each), "coef": keep(w * slope)}
    out["loss"] = out["each"].sum()
    out["kl_step"] = keep(dkl.abs())
    # what an error of P in logp does to each term
    out["loss_bound"] = keep(w.abs() * ((r * adv).abs() * 2 + kl_coef * dkl.abs()) * (P + 2.0 ** -21) + w.abs() * each.abs() * 2.0 ** -22).sum()
    out["coef_bound"] = keep(w.abs() * ((r * adv).abs() + kl_coef * (1 + dkl.abs())) * (P + 2.0 ** -21))
    return out


def preference(x, labels, ref, bounds, beta, e):
    """`bounds`: row ranges of the sequences over flattened rows."""
    xf, lf, rf = x.reshape(-1, x.shape[-1]), labels.reshape(-1), ref.reshape(-1).double()
    use = lf >= 0
    inside = torch.zeros_like(use)
    for a, b in bounds:
        inside[a:b] = True
    use = use & inside
    logp, _, _ = scores(xf, lf)
    logp = torch.where(use, logp, 0.0)
    gain = torch.where(use, logp - rf, 0.0)
    s = torch.stack([gain[a:b].sum() for a, b in bounds])
    m = beta * (s[0::2] - s[1::2])
    soft = torch.nn.functional.softplus
    loss = ((1 - e) * soft(-m) + e * soft(m)).mean()
    slope = beta * (e * torch.sigmoid(m) - (1 - e) * torch.sigmoid(-m)) / m.numel()
    coef = torch.zeros_like(logp)
    for q, (a, b) in enumerate(bounds):
        coef[a:b] = slope[q // 2] if q % 2 == 0 else -slope[q // 2]
    return {"loss": loss, "rewards": beta * s, "logp": logp.view(labels.shape), "coef": torch.where(use, coef, 0.0).view(labels.shape)}


def philox_factors(n, p, seed, offset, device):
    """Factors of n elements, one block at a time in Python integers."""
    units = int(p * 65536 + 0.5)
    if units == 0:
        return torch.ones(n, dtype=torch.float64, device=device)
    m = 0xFFFFFFFF
    out = []
    for i in range((n + 7) // 8):
        c = [i & m, i >> 32, offset & m, offset >> 32]
        k = [seed & m, seed >> 32]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
            k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
        for word in c:
            out += [word & 0xFFFF, word >> 16]
    f = 0.0 if units == 65536 else 65536.0 / (65536 - units)
    return torch.tensor([f if b >= units else 0.0 for b in out[:n]], dtype=torch.float64, device=device)


def block_forward(x, h, post, nxt, gate, scale, eps, f):
    x, h = x.double(), h.double()
    out = {}
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = h * rstd * post.double() if post is not None else h
    g = gate.double() if gate is not None else 1.0
    branch = scale * g * n * f
    out["x"] = x + branch
    out["x_bound"] = (x.abs() + branch.abs()) * 2.0 ** -20       # under 16 roundings of float32 on the way
    out["rstd_post"] = rstd.squeeze(-1)
    if nxt is not None:
        r = (out["x"].square().mean(-1, keepdim=True) + eps).rsqrt()
        out["rstd_next"] = r.squeeze(-1)
        out["y"] = out["x"] * r * nxt.double()
        out["y_bound"] = (r * nxt.double()).abs() * out["x_bound"] + out["y"].abs() * 2.0 ** -19
    return out


def block_backward(gx, gy, h, x_out, rstd_post, rstd_next, post, nxt, gate, gate_kind, scale, f):
    """Gradients and their bounds (1.2e-5 of the magnitudes that are summed: row sums of at most 64 float32
    terms per thread and a tree, 3.8e-6, twice over, and the products)."""
    e = 1.2e-5
    h = h.double()
    t = gx.double() if gx is not None else torch.zeros_like(h)
    tb = t.abs()
    out = {}
    if nxt is not None:
        r = rstd_next.double().unsqueeze(-1)
        xh = x_out.double() * r
        a = gy.double() * nxt.double()
        t = t + r * (a - xh * (a * xh).mean(-1, keepdim=True))
        tb = tb + r * (a.abs() + xh.abs() * (a * xh).abs().mean(-1, keepdim=True))
        terms = gy.double() * xh
        out["next"] = (terms, terms.abs())
    out["x"] = (t, tb * e)
    r = rstd_post.double().unsqueeze(-1) if post is not None else 1.0
    hat = h * r
    n = hat * post.double() if post is not None else h
    g = gate.double() if gate is not None else 1.0
    d, db = scale * g * f * t, (scale * g * f * tb).abs()
    if gate is not None:
        terms, mags = scale * f * n * t, (scale * f * n * tb).abs()
        out["gate"] = (terms, mags)
    if post is not None:
        out["post"] = (d * hat, db * hat.abs())
        b, bb = d * post.double(), db * post.double().abs()
        out["h"] = (r * (b - hat * (b * hat).mean(-1, keepdim=True)), r * (bb + hat.abs() * (bb * hat.abs()).mean(-1, keepdim=True)) * 2 * e)
    else:
        out["h"] = (d, db * 2 * e)
    # sums over rows: every term off by 2 e of its size, and a float32 running sum of at most `rows` terms
    rows = h.numel() // h.shape[-1]
    k = 2 * e + rows * 2.0 ** -24
    flat = lambda v: v.reshape(rows, -1)  # noqa: E731
    for name in ("next", "post"):
        if name in out:
            out[name] = tuple(flat(v).sum(0) for v in out[name])
            out[name] = (out[name][0], out[name][1] * k)
    if gate is not None:
        v, m = out["gate"]
        if gate_kind == "vector":
            out["gate"] = (flat(v).sum(0), flat(m).sum(0) * k)
        elif gate_kind == "sequence":
            out["gate"] = (v.sum(-2, keepdim=True), m.sum(-2, keepdim=True) * k)
        else:
            out["gate"] = (v, m * 2 * e)
    return out
