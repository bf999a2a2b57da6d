"""GPU tests of what the training operators keep of their 64-bit formulas where digits are easily lost, and of
calls that are rarely made.  Oracles in 64 bits; every bound is derived where it stands (u = eps / 2 is one
rounding of the output)."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import training_oracle as R
from test_gpu_training import EACH, KINDS, block_inputs, check_policy, check_preference, check_scores, labels_of, logits_of, policy_inputs
from training_oracle import close, u

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tpb():
    import tensorplay_b200
    return tensorplay_b200


# ------------------------------------------------------------------------------------ the residual path

SHAPES = pytest.mark.parametrize("shape", [(2, 3, 7), (3, 5, 64), (2, 3, 257), (3, 4, 512), (2, 30, 1000), (5, 2, 1023), (2, 9, 4096), (1, 3, 8200), (2, 2, 16384)],
                                 ids=lambda s: "x".join(map(str, s)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@KINDS
@SHAPES
def test_gradients_by_the_stream_before_it_is_rounded(cuda, tpb, dtype, kind, shape):
    """y comes from x_out before its rounding; with x the gradients do too.  The oracle differentiates at the 64-bit
    stream, which the kernels' float32 one is off by at most x_bound: that enters hat(x_out) as x_bound * rstd."""
    v = block_inputs(cuda, shape, dtype, kind, 3)
    scale, eps, how = 0.6, 1e-5, {"scale": 0.6, "p": 0.1, "seed": 11, "offset": 5}
    x_out, y, rp, rn = tpb.block_residual(v["x"], v["h"], v["post"], v["next"], v["gate"], eps=eps, **how)
    got = tpb.block_residual_backward(v["gx"], v["gy"], v["h"], None, rp, rn, v["post"], v["next"], v["gate"], x=v["x"], **how)
    f = R.philox_factors(v["h"].numel(), 0.1, 11, 5, cuda).view(shape)
    fine = R.block_forward(v["x"], v["h"], v["post"], v["next"], v["gate"], scale, eps, f)
    back = R.block_backward(v["gx"], v["gy"], v["h"], fine["x"], rp, rn, v["post"], v["next"], v["gate"], kind, scale, f)
    r, gy = rn.double().unsqueeze(-1), v["gy"].double()
    hat, off = (fine["x"] * r).abs(), fine["x_bound"] * r
    a = (gy * v["next"].double()).abs()
    # what the stream's own error does to dL/dx, and through it to the rest
    dt = r * (off * (a * hat).mean(-1, keepdim=True) + hat * (a * off).mean(-1, keepdim=True))
    extra = {"next": (gy.abs() * off).flatten(0, 1).sum(0), "x": dt}
    for name, g in zip(("x", "h", "post", "next", "gate"), got):
        if name not in back:
            assert g is None
            continue
        value, tol = (t.reshape(g.shape) for t in back[name])
        if name in ("h", "post", "gate"):
            # linear in dL/dx, whose magnitudes the bound multiplies by 2.4e-5 at least; dt is under 2^-19 of them
            tol = tol * 1.1
        else:
            tol = tol + extra[name].reshape(g.shape)
        close(g, value, tol + u(dtype) * value.abs() + R.TINY[dtype], f"gradient of {name}")


@KINDS
@SHAPES
def test_the_stream_is_formed_again_bit_for_bit(cuda, tpb, kind, shape):
    """In float32 x_out is not rounded further: by x or by x_out the gradients have to be the same bits."""
    v = block_inputs(cuda, shape, torch.float32, kind, 4)
    for post in (v["post"], None):
        for p in (0.0, 0.3):
            how = {"scale": -0.7, "p": p, "seed": 9, "offset": 1 << 35}
            x_out, y, rp, rn = tpb.block_residual(v["x"], v["h"], post, v["next"], v["gate"], **how)
            want = tpb.block_residual_backward(v["gx"], v["gy"], v["h"], x_out, rp, rn, post, v["next"], v["gate"], **how)
            for given in (None, x_out):
                got = tpb.block_residual_backward(v["gx"], v["gy"], v["h"], given, rp, rn, post, v["next"], v["gate"], x=v["x"], **how)
                for a, b in zip(got, want):
                    assert (a is None and b is None) or torch.equal(a, b)


@EACH
def test_x_in_place_of_x_out_as_a_view_and_without_a_next_norm(cuda, tpb, dtype):
    v = block_inputs(cuda, (3, 9, 211), dtype, "element", 21)
    for cut in (lambda t: t[:, 1:, 3:], lambda t: t[:, ::2, :208], lambda t: t[:, 2]):
        w = {k: cut(t) if t.dim() == 3 else t[:cut(v["x"]).shape[-1]] for k, t in v.items()}
        x_out, y, rp, rn = tpb.block_residual(w["x"], w["h"], w["post"], w["next"], w["gate"])
        got = tpb.block_residual_backward(w["gx"], w["gy"], w["h"], None, rp, rn, w["post"], w["next"], w["gate"], x=w["x"])
        c = {k: t.contiguous() for k, t in w.items()}
        want = tpb.block_residual_backward(c["gx"], c["gy"], c["h"], None, rp, rn, c["post"], c["next"], c["gate"], x=c["x"])
        for name, a, b in zip("xhpng", got, want):
            # other widths of thread and worker: the same sums in another order (the oracle's bounds cover either)
            close(a, b, 2 * u(dtype) * b.double().abs() + 1e-4 * b.double().abs().mean(), name)
    x_out, _, rp, _ = tpb.block_residual(v["x"], v["h"], v["post"], None, v["gate"])
    with_x = tpb.block_residual_backward(v["gx"], None, v["h"], None, rp, None, v["post"], None, v["gate"], x=v["x"])
    plain = tpb.block_residual_backward(v["gx"], None, v["h"], x_out, rp, None, v["post"], None, v["gate"])
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(with_x, plain))
    with pytest.raises(ValueError, match="x has shape"):
        tpb.block_residual_backward(v["gx"], v["gy"], v["h"], x_out, rp, rp, v["post"], v["next"], v["gate"], x=v["x"][:, :4])
    with pytest.raises(TypeError, match="x_out must be a tensor"):
        tpb.block_residual_backward(v["gx"], v["gy"], v["h"], None, rp, rp, v["post"], v["next"], v["gate"])


@EACH
def test_rows_of_no_elements(cuda, tpb, dtype):
    """The mean square of nothing is NaN, and so is rstd: it is written, not left as it was."""
    x, w = torch.empty(3, 5, 0, dtype=dtype, device=cuda), torch.empty(0, dtype=dtype, device=cuda)
    y, rstd = tpb.rms_norm(x, w, out=(torch.empty_like(x), torch.full((3, 5), 7.0, device=cuda)))
    assert y.shape == x.shape and bool(rstd.isnan().all())
    out = (torch.empty_like(x), torch.empty_like(x), *(torch.full((3, 5), 7.0, device=cuda) for _ in range(2)))
    _, _, rp, rn = tpb.block_residual(x, x, w, w, out=out)
    assert bool(rp.isnan().all()) and bool(rn.isnan().all())
    assert all(g is None or g.numel() == 0 for g in tpb.block_residual_backward(x, x, x, x, rp, rn, w, w))
    none = torch.empty(0, 8, dtype=dtype, device=cuda)
    assert tpb.rms_norm(none, torch.ones(8, dtype=dtype, device=cuda))[1].shape == (0,)


# ------------------------------------------------------------------------------------ objectives on logits

def exact_rows(x, labels):
    """(logp, p of every entry, 1 - p of the label) in 64 bits, from differences to the row's maximum and with the label
    left out of the sum: neither a large common value nor a p near 1 costs digits."""
    d = x.double() - x.double().amax(-1, keepdim=True)
    hit = torch.nn.functional.one_hot(labels, x.shape[-1]).bool()
    e = d.exp()
    others = torch.where(hit, 0.0, e).sum(-1)
    own = d.gather(-1, labels.unsqueeze(-1)).squeeze(-1)
    total = others + own.exp()
    logp = torch.where(own > others.log(), -torch.log1p(others / own.exp()), own - total.log())
    return logp, e / total.unsqueeze(-1), others / total, hit


def grad_rows(x, labels, coef):
    _, p, rest, hit = exact_rows(x, labels)
    return torch.where(hit, rest.unsqueeze(-1), -p) * coef.double().unsqueeze(-1)


def far_rows(cuda, dtype, vocab):
    """Rows around values that a float64 sum with log V does not hold beside it, or only in part."""
    top = torch.finfo(dtype).max
    fill = [-top, top / 2, -top / 3, 4e4, -3e3] + ([1e16, -2.0 ** 60, 3e7, 2.0 ** 28] if dtype != torch.float16 else [])
    x = torch.stack([torch.full((vocab,), f, device=cuda, dtype=torch.float64) for f in fill])
    x[:, 1::3] -= x[:, 1::3].abs() * (4 * u(dtype))          # a third of the entries a few steps lower
    x = x.to(dtype)
    # all entries alike, and a label that is one of the lower ones
    x = torch.cat([x, torch.full((2, vocab), -top, device=cuda, dtype=dtype)])
    labels = torch.arange(x.shape[0], device=cuda) % 4
    return x, labels


@EACH
@pytest.mark.parametrize("vocab", [5, 777, 20011])
def test_rows_around_large_values(cuda, tpb, dtype, vocab):
    """A row that a mask has filled with the type's lowest value is a uniform row: logp = -log V and a gradient.
    Bounds: P of the sums, as in the oracle's file; no term in |lse|."""
    x, lab = far_rows(cuda, dtype, vocab)
    n = x.shape[0]
    logp, p, rest, hit = exact_rows(x, lab)
    assert bool((logp[-2:] + torch.tensor(float(vocab)).log().to(cuda) < 1e-6).all()) and bool(logp[-2:].ne(0).all())
    tol = R.P + u(torch.float32) * logp.abs()
    close(tpb.token_logprobs(x, lab)[0], logp, tol, "logp of token_logprobs")
    one = torch.ones(n, device=cuda)
    old = logp.clamp_min(-50).float()                        # a ratio near 1, or 0 where the label is far below
    loss, grad, got, ratio, kl = tpb.policy_loss(x, lab, old, one, one / n)
    close(got, logp, tol, "logp of policy_loss")
    r = (logp - old.double()).exp()
    close(ratio, r, r * (R.P + 2.0 ** -21), "ratio")
    g = grad_rows(x, lab, -r / n)
    close(grad, g, g.abs() * (2 * R.P + 2.0 ** -20 + u(dtype)) + R.TINY[dtype], "gradient of policy_loss")
    n -= n % 2
    _, grad, rewards, got = tpb.preference_loss(x[:n], lab[:n], old[:n], torch.arange(n + 1, device=cuda), beta=0.3)
    close(got, logp[:n], tol[:n], "logp of preference_loss")
    s = torch.where(logp[:n] < -1e30, 0.0, 0.3 * (logp[:n] - old[:n].double()))
    m = (s[0::2] - s[1::2])
    near = (logp[:n].view(-1, 2) > -1e30).all(1)             # pairs whose margin is a number that float32 holds
    slope = -0.3 * torch.sigmoid(-m) / (n // 2)
    g = grad_rows(x[:n], lab[:n], torch.stack([slope, -slope], 1).flatten())
    keep = near.repeat_interleave(2)
    close(grad[keep], g[keep], (g.abs() * (2 * R.P + 0.3 * 2 * R.P + 2.0 ** -20 + u(dtype)) + R.TINY[dtype])[keep], "gradient of preference_loss")


@EACH
@pytest.mark.parametrize("ctas", [1, 2, 3, 5, 8])
def test_several_ctas_per_row(cuda, tpb, dtype, ctas, monkeypatch):
    """Rows shared by a cluster of CTAs, with the logits and the gradient on the same 16-byte boundaries and on
    different ones (every row of an odd vocabulary starts elsewhere), and as views that shift them further."""
    monkeypatch.setenv("TPB200_ROW_CTAS", str(ctas))
    for vocab, cut in ((20480, slice(None)), (20011, slice(None)), (20014, slice(1, None)), (20013, slice(3, -2))):
        x, lab, old, adv, w, ref = policy_inputs(cuda, (3, 7), vocab, dtype, vocab + ctas)
        x = x[..., cut]
        lab = torch.where(lab < x.shape[-1], lab, 0)
        lp, _, _ = R.scores(x, lab)              # the cut has changed it: the older policy's by the same rule again
        old = (lp + 0.05).float()
        check_policy(tpb, x, lab, old, adv, w, (lp - 0.3).float())
        check_policy(tpb, x[:, 1:], lab[:, 1:], old[:, 1:], adv[:, 1:], w[:, 1:], None, kl_coef=0.0)
        check_scores(tpb, x[:, ::2], lab[:, ::2])
        bounds = [(0, 4), (4, 9), (9, 20), (20, 21)]
        check_preference(tpb, x.reshape(21, -1), lab.flatten(), (lp + 0.2).float().flatten(), bounds, torch.tensor([0, 4, 9, 20, 21], device=cuda))


def confident(cuda, dtype, vocab, seed):
    """Rows whose token has nearly all of the probability, at the places where a row begins, ends and is split."""
    places = sorted({0, 1, vocab // 3, vocab // 2 + 1, vocab - 2, vocab - 1} & set(range(vocab)))
    heights = [10.0, 14.0, 17.0, 20.0, 28.0, 30.0, 45.0, 80.0]
    lab = torch.tensor([i for i in places for _ in heights], device=cuda)
    x = logits_of(cuda, (lab.numel(), vocab), dtype, seed, spread=2.0)
    up = torch.tensor(heights, device=cuda).repeat(len(places))
    return x.scatter(1, lab.unsqueeze(1), up.to(dtype).unsqueeze(1)), lab


@EACH
@pytest.mark.parametrize("vocab,shift", [(2, 0), (9, 0), (77, 1), (1000, 0), (32000, 0), (50021, 0), (50048, 3), (151936, 0)])
def test_tokens_with_a_probability_near_one(cuda, tpb, dtype, vocab, shift):
    """logp = -(1 - p) and the token's gradient are held to P of themselves, from 1 - p = 0.9 down to e^-80; the sum of the
    others is off by at most P of itself, e^-|g|, its logarithm and the products by 2^-20 of themselves.  No logp is
    positive, and a row of the gradient adds up to zero."""
    x, lab = confident(cuda, dtype, vocab + shift, 7 + vocab)
    x, lab = x[:, shift:], (lab - shift).clamp_min(0)
    logp, p, rest, hit = exact_rows(x, lab)
    rel = R.P + 2.0 ** -20
    got, lse = tpb.token_logprobs(x, lab)
    assert bool((got <= 0).all())
    close(got, logp, logp.abs() * rel + R.TINY[torch.float32], "logp of token_logprobs")
    close(lse, x.double().logsumexp(1), R.P + u(torch.float32) * lse.double().abs(), "lse")
    n = lab.numel()
    one = torch.ones(n, device=cuda)
    old = (logp + 0.1).float()
    loss, grad, got, ratio, _ = tpb.policy_loss(x, lab, old, one, one, grad_scale=64.0)
    close(got, logp, logp.abs() * rel + R.TINY[torch.float32], "logp of policy_loss")
    r = (logp - old.double()).exp()
    g = grad_rows(x, lab, -64.0 * r)
    # every entry: its own exponential (P) and the sum's
    tol = g.abs() * (2 * R.P + 2.0 ** -19 + u(dtype)) + R.TINY[dtype]
    close(grad, g, tol, "gradient of policy_loss")
    if dtype == torch.float32:
        # V terms of up to 2^-23 of themselves, each with its own exponential's error of 2^-22 and P / 8 of the sweep
        total, size = grad.double().sum(1).abs(), g.abs().sum(1)
        assert bool((total <= size * (R.P + 2.0 ** -22) + R.TINY[dtype] * vocab).all())
    n -= n % 2
    ref = (logp + 0.2).float()
    offsets = torch.arange(n + 1, device=cuda)
    _, grad, rewards, got = tpb.preference_loss(x[:n], lab[:n], ref[:n], offsets, beta=0.5, grad_scale=1024.0)
    close(got, logp[:n], logp[:n].abs() * rel + R.TINY[torch.float32], "logp of preference_loss")
    m = 0.5 * (logp - ref.double())[:n]
    slope = -1024.0 * 0.5 * torch.sigmoid(-(m[0::2] - m[1::2])) / (n // 2)
    g = grad_rows(x[:n], lab[:n], torch.stack([slope, -slope], 1).flatten())
    close(grad, g, g.abs() * (3 * R.P + 2.0 ** -19 + u(dtype)) + R.TINY[dtype], "gradient of preference_loss")


@EACH
@pytest.mark.parametrize("rows,vocab,spread,offset", [(2048, 32000, 2.0, 0.0), (512, 151936, 2.0, 0.0), (2048, 1000, 2.0, 0.0), (2048, 32000, 1.0, 40.0), (2048, 50021, 3.0, -12.0)])
def test_sums_are_not_off_to_one_side(cuda, tpb, dtype, rows, vocab, spread, offset):
    """The mean error of the float64 log-probabilities that a reward adds up (ref = the right value, rounded, so that the reward
    is small and its float32 holds it).  One row: roundings of 2^-22 and ex2's 1.5e-7, of either sign, averaged over its
    terms: at most 1.5e-7, over the rows 1.5e-7 / sqrt(rows) a standard deviation.  Equal logits have equal errors in every
    row, and 16-bit logits are equal often (near 40 a bfloat16 has four values to 1, and a row some twenty in all): with w_k
    the mean share of the value k, the errors of the values are independent, so that their mean has a standard deviation of
    1.5e-7 sqrt(sum of w_k^2), however many rows there are.  Four of both.  To one side: 1e-10 of the base; the
    arguments of ex2 are below 1, and 8.4e-8 (the difference of ex2's mean errors on either side of zero) count for
    the share of the sum above E, under 0.15: 1.3e-8."""
    g = torch.Generator(device=cuda).manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, device=cuda, generator=g) * spread + offset).to(dtype)
    lab = labels_of(cuda, (rows,), vocab, 5)
    want = torch.cat([exact_rows(x[i:i + 256], lab[i:i + 256])[0] for i in range(0, rows, 256)])
    ref = want.float()
    loss, _, rewards, _ = tpb.preference_loss(x, lab, ref, torch.tensor([0, rows // 2, rows], device=cuda), beta=1.0, need_grad=False)
    off = (rewards.double().sum() - (want - ref.double()).sum()).item() / rows
    share = 0.0
    if dtype != torch.float32:
        values, at = x.unique(return_inverse=True)
        w = torch.zeros(values.numel(), dtype=torch.float64, device=cuda)
        for i in range(0, rows, 256):
            w.scatter_add_(0, at[i:i + 256].flatten(), exact_rows(x[i:i + 256], lab[i:i + 256])[1].flatten() / rows)
        share = w.square().sum().sqrt().item()
    bound = 1.3e-8 + 4 * 1.5e-7 * (rows ** -0.5 + share)
    print(f"mean error {off:.3e}, bound {bound:.3e}")
    assert abs(off) <= bound


@EACH
@pytest.mark.parametrize("vocab", [2, 77, 8191, 32000, 50021])
def test_gradient_of_log_probabilities_where_lse_does_not_hold_them(cuda, tpb, dtype, vocab):
    """The separate backward call has lse as a float32 alone.  Rows whose token has nearly all of the probability, rows around
    large values, and logits with a large common part lose digits there: they are held to the bounds of the losses
    that have the sums (P twice, 2^-19).  Where lse serves, |lse| < 32, it costs p 2^-20 of itself."""
    x, lab = confident(cuda, dtype, vocab, 3 + vocab)
    far, at = far_rows(cuda, dtype, vocab)
    off = logits_of(cuda, (6, vocab), torch.float32, 5) + torch.tensor([31.0, -40.0, 500.0, -3000.0, 5000.0, 2e4], device=cuda).unsqueeze(1)
    x = torch.cat([x, far, off.to(dtype), logits_of(cuda, (40, vocab), dtype, 9, spread=6.0)])
    lab = torch.cat([lab, at.clamp_max(vocab - 1), labels_of(cuda, (46,), vocab, 6)])
    coef = torch.randn(lab.numel(), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)) * 8
    coef[::11] = 0.0
    logp, lse = tpb.token_logprobs(x, lab)
    for rows in (slice(None), slice(0, 1), slice(-46, None)):
        g = tpb.token_logprobs_backward(coef[rows], x[rows], lab[rows], lse[rows])
        want = grad_rows(x[rows], lab[rows], coef[rows])
        close(g, want, want.abs() * (2 * R.P + 2.0 ** -19 + u(dtype)) + R.TINY[dtype], "grad_logits")


@EACH
def test_an_infinite_kl_that_is_only_watched(cuda, tpb, dtype):
    """With kl_coef = 0 the KL term is reported, and is no part of the loss or of the gradient, whatever it is."""
    x, lab, old, adv, w, ref = policy_inputs(cuda, (7,), 301, dtype, 12, masked=0.0)
    plain = tpb.policy_loss(x, lab, old, adv, w, kl_coef=0.0)
    ref = ref.clone()
    ref[1], ref[2] = float("-inf"), 200.0                   # kl = inf - ... at d = -inf, e^d beyond float32 at d > 200
    loss, grad, logp, ratio, kl = tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.0)
    assert bool(kl[1:3].isinf().all()) and bool(kl[[0, 3, 4, 5, 6]].isfinite().all())
    for a, b in zip((loss, grad, logp, ratio), plain):
        assert torch.equal(a, b)
    x = x.clone()
    x[3, lab[3]] = float("-inf")                            # a token that a mask has taken out: logp = -inf, ratio 0, kl infinite
    loss, grad, logp, ratio, kl = tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.0)
    assert logp[3] == float("-inf") and ratio[3] == 0 and kl[3] == float("inf")
    assert bool(loss.isfinite()) and bool((grad[3] == 0).all()) and bool(grad.isfinite().all())
    # counted, it is an infinite loss
    assert bool(tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1)[0].isinf())


@EACH
def test_results_are_tensors_of_their_own(cuda, tpb, dtype):
    """No result is a view of another one or of scratch memory: keeping one keeps its own bytes, and each can be changed
    in place in a recorded graph."""
    x, lab, old, adv, w, ref = policy_inputs(cuda, (3, 5), 301, dtype, 12)
    v = block_inputs(cuda, (2, 3, 64), dtype, "vector", 13)
    x_out, y, rp, rn = block = tpb.block_residual(v["x"], v["h"], v["post"], v["next"], v["gate"])
    results = [*tpb.token_logprobs(x, lab), *tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1), *tpb.preference_loss(x[:2], lab[:2], ref[:2]), *block,
               *tpb.block_residual_backward(v["gx"], v["gy"], v["h"], x_out, rp, rn, v["post"], v["next"], v["gate"]), *tpb.rms_norm(v["x"], v["next"])]
    scale = torch.ones((), device=cuda, requires_grad=True)
    for i, t in enumerate(results):
        assert not t._is_view() and t.untyped_storage().nbytes() == t.numel() * t.element_size(), i
        t.mul_(scale.to(t.dtype)).sum().backward()
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in results)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))


# ------------------------------------------------------------------------------------ two host threads

def both_at_once(cuda, calls, times):
    """Every call `times` times in a host thread and on a stream of its own; what they raised, and their last results."""
    errors, got, go = [], [None] * len(calls), threading.Barrier(len(calls))

    def work(i):
        try:
            s = torch.cuda.Stream(cuda)
            s.wait_stream(torch.cuda.default_stream(cuda))
            with torch.cuda.stream(s):
                go.wait()
                for _ in range(times):
                    got[i] = calls[i]()
            s.synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return errors, got


@EACH
def test_two_host_threads_with_different_widths(cuda, tpb, dtype):
    """The limit of a kernel's shared memory belongs to the device: a thread's narrow rows must not lower it between
    another one's request and launch.  The calls go to the C ABI, one after the other as fast as threads make them."""
    from tensorplay_b200 import _lib
    L, calls, want = _lib.lib(), [], []
    for width in (8192, 320, 4096, 288):
        v = block_inputs(cuda, (1, 2, width), dtype, None, width)
        want.append(tpb.block_residual(v["x"], v["h"], v["post"], v["next"]))
        out = [torch.empty_like(t) for t in want[-1]]
        rows = _lib.pair(0, width)
        args = (v["x"].data_ptr(), rows, v["h"].data_ptr(), rows, None, None, v["post"].data_ptr(), v["next"].data_ptr(),
                tpb.training._TYPES[dtype], 1, 2, width, 1.0, 1e-6, 0.0, 0, 0, *(t.data_ptr() for t in out))

        def run(args=args, out=out, keep=v):
            stream = torch.cuda.current_stream(cuda).cuda_stream
            for _ in range(4000):
                _lib.check(L.tpb200_block_residual(*args, stream))
            return out
        calls.append(run)
    torch.cuda.synchronize()
    errors, got = both_at_once(cuda, calls, 2)
    assert not errors, errors[0]
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------ how they are called

def test_captured_where_the_data_decides(cuda, tpb):
    """One graph over rows that the backward call takes by lse in one replay and sums again in the next, over rows that
    change between near and far, and over the residual path by x; equal to eager calls every time."""
    vocab, n = 20011, 24
    x = torch.zeros(n, vocab, dtype=torch.bfloat16, device=cuda)
    lab, coef = torch.zeros(n, dtype=torch.int64, device=cuda), torch.ones(n, device=cuda)
    v = block_inputs(cuda, (2, 9, 640), torch.bfloat16, "sequence", 82)

    def run():
        logp, lse = tpb.token_logprobs(x, lab)
        g = tpb.token_logprobs_backward(coef, x, lab, lse)
        x_out, y, rp, rn = tpb.block_residual(v["x"], v["h"], v["post"], v["next"], v["gate"], p=0.1, seed=1)
        return [logp, lse, g, *tpb.policy_loss(x, lab, logp - 0.1, coef, coef, logp + 0.1, kl_coef=0.1), x_out, y,
                *tpb.block_residual_backward(v["gx"], v["gy"], v["h"], None, rp, rn, v["post"], v["next"], v["gate"], x=v["x"], p=0.1, seed=1)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept = run()
    sure, at = confident(cuda, torch.bfloat16, vocab, 5)
    far, far_at = far_rows(cuda, torch.bfloat16, vocab)
    for rows, labels in ((logits_of(cuda, (n, vocab), torch.bfloat16, 1), labels_of(cuda, (n,), vocab, 2, 0.2)), (sure[:n], at[:n]),
                         (torch.cat([far, sure])[:n], torch.cat([far_at, at])[:n]), (logits_of(cuda, (n, vocab), torch.bfloat16, 3), labels_of(cuda, (n,), vocab, 4))):
        x.copy_(rows)
        lab.copy_(labels)
        v["h"].copy_(logits_of(cuda, v["h"].shape, torch.bfloat16, int(labels[0]) + 7))
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        for a, b in zip(kept, eager):
            assert a is None or torch.equal(a, b)


def test_a_captured_dropout_drops_the_same_elements(cuda, tpb):
    """As documented: seed and offset are numbers of the call, so that a graph repeats the choice it was captured with."""
    x = torch.ones(1000, device=cuda)
    tpb.dropout(x, 0.5, 3, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tpb.dropout(x, 0.5, 3, 4)
    for scale in (1.0, 2.0):
        x.fill_(scale)
        graph.replay()
        assert torch.equal(y, tpb.dropout(x, 0.5, 3, 4)) and not torch.equal(y, tpb.dropout(x, 0.5, 3, 5))


def test_no_function_records_a_graph(cuda, tpb):
    """As documented: inputs that require gradients are read, and nothing is recorded."""
    x = torch.randn(4, 8, device=cuda, requires_grad=True)
    lab, one, w = labels_of(cuda, (4,), 8, 2), torch.ones(4, device=cuda), torch.ones(8, device=cuda, requires_grad=True)
    for t in (*tpb.token_logprobs(x, lab), *tpb.policy_loss(x, lab, one, one, one), *tpb.rms_norm(x, w), *tpb.block_residual(x, x.detach(), w, w), tpb.dropout(x, 0.5, 1)):
        assert not t.requires_grad


def test_under_the_range_checker(cuda):
    """The tests of this file with every global access compared with the ranges of its call."""
    from tensorplay_b200 import _lib
    if _lib.CHECKED:
        pytest.skip("already running under the checked build")
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.join("tests", "test_gpu_training_exact.py"), "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider",
                        "-k", "not host_threads and not captured and not one_side and not of_their_own"],
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), env=dict(os.environ, TPB200_CHECKED="1"), capture_output=True, text=True, timeout=1500)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
