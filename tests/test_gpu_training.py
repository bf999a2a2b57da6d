"""GPU parity of the training operators with their 64-bit formulas (training_oracle.py, where the bounds
are derived), at the sizes, strides and masks where they can go wrong."""
import os
import subprocess
import sys

import pytest
import torch

import training_oracle as R
from training_oracle import TYPES, close, u

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EACH = pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))


@pytest.fixture(scope="module")
def tpb():
    import tensorplay_b200
    return tensorplay_b200


def gen(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def logits_of(cuda, shape, dtype, seed, spread=3.0):
    return (torch.randn(shape, device=cuda, generator=gen(cuda, seed)) * spread).to(dtype)


def labels_of(cuda, shape, vocab, seed, masked=0.0):
    g = gen(cuda, seed)
    lab = torch.randint(0, vocab, shape, device=cuda, generator=g)
    return torch.where(torch.rand(shape, device=cuda, generator=g) < masked, torch.full_like(lab, -100), lab)


def check_scores(tpb, x, lab, seed=5):
    logp, lse = tpb.token_logprobs(x, lab)
    want, norm, use = R.scores(x, lab)
    close(logp, want, R.P + u(torch.float32) * want.abs().nan_to_num(0, 0, 0), "logp")
    close(lse, norm, R.P + u(torch.float32) * norm.abs().nan_to_num(0, 0, 0), "lse")
    assert logp.dtype == lse.dtype == torch.float32 and logp.shape == x.shape[:-1]
    gl = torch.randn(lab.shape, device=x.device, generator=gen(x.device, seed))
    g = tpb.token_logprobs_backward(gl, x, lab, lse)
    assert g.shape == x.shape and g.dtype == x.dtype and g.is_contiguous()
    coef = torch.where(use, gl, 0.0)
    want, tol = R.grad_of(x, lab, coef)
    # the normaliser came back as a float32: p is off by 2^-24 |lse| more
    p = want.abs() + coef.double().abs().unsqueeze(-1) * (want.abs() > 0)
    extra = (norm.abs().unsqueeze(-1).nan_to_num(0) + 1) * 2.0 ** -23 * p.nan_to_num(0)
    close(g, want, tol.nan_to_num(0) + extra + u(x.dtype) * want.abs().nan_to_num(0) + R.TINY[x.dtype], "grad_logits")
    return logp, lse, g


@EACH
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 33, 255, 1000, 4096, 5003, 32768, 70001])
def test_scores_of_every_row_length(cuda, tpb, dtype, vocab):
    rows = 5
    check_scores(tpb, logits_of(cuda, (rows, vocab), dtype, vocab), labels_of(cuda, (rows,), vocab, vocab + 1, 0.2))


@EACH
def test_scores_at_the_vocabulary_of_the_benchmark(cuda, tpb, dtype):
    check_scores(tpb, logits_of(cuda, (6, 151936), dtype, 3), labels_of(cuda, (6,), 151936, 4))
    check_scores(tpb, logits_of(cuda, (1, 151936), dtype, 5), labels_of(cuda, (1,), 151936, 6))
    check_scores(tpb, logits_of(cuda, (300, 151936), dtype, 7), labels_of(cuda, (300,), 151936, 8, 0.3))


@EACH
def test_scores_of_views(cuda, tpb, dtype):
    """Slices that shift rows against 16-byte boundaries, padded vocabularies, one row for all, no rows."""
    v = 1001
    base = logits_of(cuda, (3, 7, v + 6), dtype, 11)
    lab = labels_of(cuda, (3, 7), v - 3, 12, 0.2)
    for x, lb in ((base[:, :-1, :v], lab[:, 1:]), (base[..., 1:v + 1], lab), (base[:, ::2, 3:v], lab[:, ::2]), (base[1, :, 5:v], lab[1]),
                  (base[:, :1, :v], lab[:, :1]), (base[0, 0, :v], lab[0, 0]), (base[:, 3, 2:v], lab[:, 3])):
        logp, lse, g = check_scores(tpb, x, lb)
        again = check_scores(tpb, x.contiguous(), lb.contiguous())
        for a, b in zip((logp, lse, g), again):
            close(a, b, 2 * R.P + 2 * u(dtype) * b.double().abs(), "the same view, contiguous")
    one = base[0, :1, :v].expand(9, v)
    check_scores(tpb, one, labels_of(cuda, (9,), v, 13))
    four = logits_of(cuda, (2, 3, 2, 50), dtype, 14)
    check_scores(tpb, four, labels_of(cuda, (2, 3, 2), 50, 15))
    none = torch.empty(0, 50, dtype=dtype, device=cuda)
    logp, lse = tpb.token_logprobs(none, torch.empty(0, dtype=torch.int64, device=cuda))
    assert logp.shape == lse.shape == (0,)


@EACH
def test_scores_of_special_values(cuda, tpb, dtype):
    v = 777
    x = logits_of(cuda, (12, v), dtype, 21)
    lab = labels_of(cuda, (12,), v, 22)
    inf = float("inf")
    x[0, ::2] = -inf                       # half of the vocabulary masked
    lab[0] = 1
    x[1] = -inf
    x[1, 5] = 0.5                          # one entry left: probability 1
    lab[1] = 5
    x[2] = -inf                            # nothing left: NaN
    x[3, 100] = inf                        # NaN
    x[4, 200] = float("nan")
    lab[5] = -1                            # takes no part, whatever is there
    x[5] = float("nan")
    lab[6] = v                             # beyond the vocabulary: NaN for the row alone
    lab[7] = 1 << 40
    lab[8] = -(1 << 40)
    x[9] = torch.finfo(dtype).min          # equal entries of the lowest value
    x[10, 0] = -inf
    lab[10] = 0                            # a label of probability 0
    x[11] = torch.finfo(dtype).max / 2
    logp, lse = tpb.token_logprobs(x, lab)
    want, norm, use = R.scores(x, lab)
    close(logp, want, R.P + u(torch.float32) * (want.abs() + norm.abs()).nan_to_num(0, 0, 0), "logp")
    assert logp[1] == 0 and logp[5] == 0 and logp[10] == -inf and logp[8] == 0
    assert bool(logp[[2, 3, 4, 6, 7]].isnan().all())
    g = tpb.token_logprobs_backward(torch.ones(12, device=cuda), x, lab, lse)
    assert bool(g[[2, 3, 4, 6, 7]].isnan().any(1).all())
    assert bool((g[5] == 0).all()) and bool((g[8] == 0).all()) and bool((g[1] == 0).all())
    assert bool((g[0, ::2] == 0).all()) and g[10, 0] == 1
    for r in (0, 9, 10):
        w, _ = R.grad_of(x[r:r + 1], lab[r:r + 1], torch.ones(1, device=cuda))
        # |lse| reaches 1e38 in row 9: its logp is log(1/v) to within 64 bits of the sum only relative to the entries
        if r != 9:
            close(g[r:r + 1], w, (R.P + 2.0 ** -20) + u(dtype) * w.abs(), f"row {r}")


def policy_inputs(cuda, shape, vocab, dtype, seed, masked=0.2):
    g = gen(cuda, seed)
    x = logits_of(cuda, (*shape, vocab), dtype, seed + 1)
    lab = labels_of(cuda, shape, vocab, seed + 2)
    logp, _, _ = R.scores(x, lab)
    # ratios on both sides of the clip range, none within 1e-4 of its ends (0.8 and 1.3)
    noise = 0.4 * torch.randn(shape, device=cuda, generator=g, dtype=torch.float64)
    for end in (0.8, 1.3):
        near = ((-noise).exp() - end).abs() < 1e-3
        noise = torch.where(near, noise + 0.01, noise)
    old = (logp + noise).float()
    ref = (logp + 0.5 * torch.randn(shape, device=cuda, generator=g, dtype=torch.float64)).float()
    adv = torch.randn(shape, device=cuda, generator=g)
    w = (torch.rand(shape, device=cuda, generator=g) >= masked).float() / 7
    return x, lab, old, adv, w, ref


def check_policy(tpb, x, lab, old, adv, w, ref, kl_coef=0.1, grad_scale=1.0, **how):
    got = tpb.policy_loss(x, lab, old, adv, w, ref, clip_low=0.2, clip_high=0.3, kl_coef=kl_coef, grad_scale=grad_scale, **how)
    loss, grad, logp, ratio, kl = got
    want = R.policy(x, lab, old, adv, w, ref, 0.2, 0.3, kl_coef)
    f = u(torch.float32)
    close(logp, want["logp"], R.P + f * want["logp"].abs(), "logp")
    close(ratio, want["ratio"], want["ratio"] * (R.P + 2.0 ** -21), "ratio")
    close(kl, want["kl"], want["kl_step"] * R.P + want["kl"] * 2.0 ** -20 + 1e-10, "kl")
    close(loss, want["loss"], want["loss_bound"] + f * want["loss"].abs() + 1e-30, "loss")
    if how.get("need_grad", True):
        coef = want["coef"] * grad_scale
        g, tol = R.grad_of(x, lab, coef)
        unit = g.abs() / coef.abs().unsqueeze(-1).clamp_min(1e-300)
        tol = tol + unit * (want["coef_bound"] * abs(grad_scale)).unsqueeze(-1)
        # where the coefficient itself nearly cancels, its bound still counts for every entry of the row
        tol = torch.where(coef.unsqueeze(-1) == 0, torch.zeros_like(tol), tol)
        close(grad, g, tol + u(x.dtype) * g.abs() + R.TINY[x.dtype], "grad_logits")
        assert grad.dtype == x.dtype and grad.shape == x.shape and grad.is_contiguous()
    else:
        assert grad is None
    return got


@EACH
@pytest.mark.parametrize("shape,vocab", [((1,), 1), ((1,), 50), ((9,), 33), ((3, 5), 1003), ((40,), 4096), ((2, 3), 32001), ((17,), 151936)])
def test_policy_loss(cuda, tpb, dtype, shape, vocab):
    x, lab, old, adv, w, ref = policy_inputs(cuda, shape, vocab, dtype, vocab)
    check_policy(tpb, x, lab, old, adv, w, ref)
    check_policy(tpb, x, lab, old, adv, w, None, kl_coef=0.0, grad_scale=-128.0)
    check_policy(tpb, x, lab, old, adv, w, ref, need_grad=False)


@EACH
def test_policy_loss_views_and_broadcasts(cuda, tpb, dtype):
    x, lab, old, adv, w, ref = policy_inputs(cuda, (3, 8), 1003, dtype, 77)
    check_policy(tpb, x[:, :-1], lab[:, :-1], old[:, :-1], adv[:, :1], w[:, :-1], ref[:, :-1])
    check_policy(tpb, x[:, 1:, 1:], lab[:, 1:].clamp_max(900), old[:, 1:], adv[0, 0], w[:, 1:], ref[:, 1:])
    check_policy(tpb, x[1], lab[1], old[1], adv[1], torch.tensor(0.25, device=cuda), ref[1])


@EACH
def test_policy_loss_of_tokens_that_take_no_part(cuda, tpb, dtype):
    x, lab, old, adv, w, ref = policy_inputs(cuda, (6,), 700, dtype, 5, masked=0.0)
    x[1] = float("nan")
    w[1] = 0.0
    x[2] = float("inf")
    lab[2] = -100
    adv[1], old[2] = float("nan"), float("inf")
    check_policy(tpb, x, lab, old, adv, w, ref)
    zero = torch.zeros_like(w)
    loss, grad, logp, ratio, kl = tpb.policy_loss(x, lab, old, adv, zero, ref, kl_coef=0.1)
    for t in (loss, grad, logp, ratio, kl):
        assert bool((t == 0).all())
    lab[3] = 700
    loss, grad, logp, _, _ = tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1)
    assert bool(loss.isnan()) and bool(logp[3].isnan()) and bool(grad[3].isnan().all()) and not bool(grad[[0, 4, 5]].isnan().any())
    none = tpb.policy_loss(x[:0], lab[:0], old[:0], adv[:0], w[:0], ref[:0], kl_coef=0.1)
    assert none[0] == 0 and none[1].shape == (0, 700)


@EACH
def test_policy_gradient_against_differences(cuda, tpb, dtype):
    """d loss / d logit from loss values in 64 bits, for a few entries of a small case."""
    x, lab, old, adv, w, ref = policy_inputs(cuda, (4,), 19, dtype, 9, masked=0.0)
    _, grad, *_ = tpb.policy_loss(x, lab, old, adv, w, ref, clip_low=0.2, clip_high=0.3, kl_coef=0.1)
    step = 1e-5
    for r in range(4):
        for j in (0, 7, int(lab[r])):
            at = lambda d: R.policy(x.double().index_put((torch.tensor(r), torch.tensor(j)), torch.tensor(d, dtype=torch.float64), accumulate=True),  # noqa: E731, B023
                                    lab, old, adv, w, ref, 0.2, 0.3, 0.1)["loss"]
            slope = (at(step) - at(-step)) / (2 * step)
            # the difference is off by step^2 / 6 of the third derivative (under 100 here) and 1e-16 / step
            close(grad[r, j], slope, 1e-8 + 2e-5 * (w * adv.abs()).max().item() + u(dtype) * slope.abs().item() + R.TINY[dtype], f"entry {r}, {j}")


def check_preference(tpb, x, lab, ref, bounds, offsets=None, e=0.1, grad_scale=1.0, beta=0.3):
    loss, grad, rewards, logp = tpb.preference_loss(x, lab, ref, offsets, beta=beta, label_smoothing=e, grad_scale=grad_scale)
    want = R.preference(x, lab, ref, bounds, beta, e)
    f = u(torch.float32)
    close(logp, want["logp"], R.P + f * want["logp"].abs(), "logp")
    # every logp was rounded to float32 before it was summed
    count = max([b - a for a, b in bounds] + [1])
    s_tol = beta * count * (R.P + f * float(want["logp"].abs().max()) if want["logp"].numel() else 0.0)
    close(rewards, want["rewards"], s_tol + f * want["rewards"].abs(), "rewards")
    close(loss, want["loss"], 2 * s_tol + f * want["loss"].abs(), "loss")        # |d loss / d margin| <= 1
    coef = want["coef"] * grad_scale
    g, tol = R.grad_of(x, lab, coef)
    unit = g.abs() / coef.abs().unsqueeze(-1).clamp_min(1e-300)
    slope_tol = abs(grad_scale) * beta / (len(bounds) // 2) * 0.25 * 2 * s_tol    # sigmoid' <= 1/4
    close(grad, g, tol + unit * (slope_tol + 2.0 ** -23 * coef.abs().unsqueeze(-1)) + u(x.dtype) * g.abs() + R.TINY[x.dtype], "grad_logits")
    return loss, grad, rewards, logp


@EACH
@pytest.mark.parametrize("vocab", [1, 37, 1000, 32003])
def test_preference_loss_packed(cuda, tpb, dtype, vocab):
    """Ragged sequences, an empty one, one of one row, rows before the first and behind the last."""
    ends = [3, 9, 10, 10, 31, 40, 41]
    offsets = torch.tensor(ends, device=cuda)
    n = 47
    x, lab = logits_of(cuda, (n, vocab), dtype, vocab), labels_of(cuda, (n,), vocab, vocab + 1, 0.2)
    ref = torch.randn(n, device=cuda, generator=gen(cuda, 3)) - 6.0
    bounds = list(zip(ends, ends[1:]))
    x[:3], ref[:3], x[41:] = float("nan"), float("nan"), float("inf")      # rows of no sequence are not looked at
    lab[5] = -100
    x[5], ref[5] = float("nan"), float("nan")
    clean = x.clone()
    for r in (0, 1, 2, 5, *range(41, n)):
        clean[r] = 0
    keep = ref.nan_to_num(0.0)
    loss, grad, rewards, logp = check_preference(tpb, clean, lab, keep, bounds, offsets)
    got = tpb.preference_loss(x, lab, ref, offsets, beta=0.3, label_smoothing=0.1)
    for a, b in zip(got, (loss, grad, rewards, logp)):
        assert torch.equal(a, b)
    assert bool((grad[:3] == 0).all()) and bool((grad[41:] == 0).all()) and bool((logp[41:] == 0).all())
    same = tpb.preference_loss(x, lab, ref, offsets, beta=0.3, label_smoothing=0.1, need_grad=False)
    assert same[1] is None and torch.equal(same[0], loss)


@EACH
def test_preference_loss_padded(cuda, tpb, dtype):
    x, lab = logits_of(cuda, (6, 11, 517), dtype, 31), labels_of(cuda, (6, 11), 517, 32, 0.3)
    ref = torch.randn(6, 11, device=cuda, generator=gen(cuda, 33)) - 7.0
    bounds = [(q * 11, q * 11 + 11) for q in range(6)]
    check_preference(tpb, x, lab, ref, bounds, e=0.0, grad_scale=64.0)
    cut = [(q * 10, q * 10 + 10) for q in range(6)]
    check_preference(tpb, x[:, :-1], lab[:, 1:], ref[:, :-1], cut)


def test_preference_loss_far_margins(cuda, tpb):
    """Margins where sigmoid saturates: the loss is linear or zero, nothing overflows."""
    x, lab = logits_of(cuda, (4, 300), torch.float32, 41), labels_of(cuda, (4,), 300, 42)
    offsets = torch.arange(5, device=cuda)
    for far in (1e3, 1e5):
        ref = torch.tensor([far, 0.0, 0.0, far], device=cuda)
        loss, grad, rewards, _ = tpb.preference_loss(x, lab, ref, offsets, beta=0.5)
        want = R.preference(x, lab, ref, [(0, 1), (1, 2), (2, 3), (3, 4)], 0.5, 0.0)
        close(loss, want["loss"], 1e-4 + 2.0 ** -22 * far, "loss")
        close(rewards, want["rewards"], 1e-4 + 2.0 ** -22 * far, "rewards")
        assert bool(grad.isfinite().all()) and bool((grad[2:] == 0).all()) and bool((grad[:2] != 0).any())


def test_preference_loss_of_bad_offsets(cuda, tpb):
    """Offsets that decrease or leave the rows are not followed; the loss says so."""
    x, lab = logits_of(cuda, (10, 64), torch.float32, 51), labels_of(cuda, (10,), 64, 52)
    ref = torch.zeros(10, device=cuda)
    for bad in ([0, 6, 4], [0, 5, 11], [-2, 5, 10], [0, 5, 1 << 40]):
        loss, grad, _, _ = tpb.preference_loss(x, lab, ref, torch.tensor(bad, device=cuda))
        assert bool(loss.isnan()) and grad.shape == x.shape
    assert not bool(tpb.preference_loss(x, lab, ref, torch.tensor([0, 5, 10], device=cuda))[0].isnan())


# ------------------------------------------------------------------------------------ the residual path

def block_inputs(cuda, shape, dtype, kind, seed):
    g = gen(cuda, seed)
    make = lambda s, k=1.0: (k * torch.randn(s, device=cuda, generator=g)).to(dtype)  # noqa: E731
    d = shape[-1]
    gate = {None: None, "vector": (d,), "sequence": (*shape[:-2], 1, d), "element": shape}[kind]
    return {"x": make(shape, 2.0), "h": make(shape), "post": make((d,)) * 0.2 + 1, "next": make((d,)) * 0.2 + 1,
            "gate": None if gate is None else make(gate), "gx": make(shape), "gy": make(shape)}


def check_block(tpb, v, kind, scale=0.6, eps=1e-5, p=0.0, seed=0, offset=0, post=True, nxt=True, with_gx=True):
    x, h, gate = v["x"], v["h"], v["gate"]
    post, nxt = v["post"] if post else None, v["next"] if nxt else None
    how = {"scale": scale, "p": p, "seed": seed, "offset": offset}
    x_out, y, rp, rn = tpb.block_residual(x, h, post, nxt, gate, eps=eps, **how)
    f = R.philox_factors(h.numel(), p, seed, offset, x.device).view(h.shape)
    want = R.block_forward(x, h, post, nxt, gate, scale, eps, f)
    t = u(x.dtype)
    close(x_out, want["x"], want["x_bound"] + t * want["x"].abs() + R.TINY[x.dtype], "x_out")
    if post is not None:
        close(rp, want["rstd_post"], want["rstd_post"] * 2.0 ** -19, "rstd_post")
    if nxt is not None:
        close(rn, want["rstd_next"], want["rstd_next"] * 2.0 ** -18, "rstd_next")
        close(y, want["y"], want["y_bound"] + t * want["y"].abs() + R.TINY[x.dtype], "y")
    else:
        assert y is None and rn is None
    gx, gy = v["gx"] if with_gx else None, v["gy"] if nxt is not None else None
    got = tpb.block_residual_backward(gx, gy, h, x_out, rp, rn, post, nxt, gate, **how)
    back = R.block_backward(gx, gy, h, x_out, rp, rn, post, nxt, gate, kind, scale, f)
    for name, g in zip(("x", "h", "post", "next", "gate"), got):
        if name not in back:
            assert g is None, name
            continue
        value, tol = back[name]
        assert g.dtype == x.dtype and g.is_contiguous()
        close(g, value.reshape(g.shape), tol.reshape(g.shape) + t * value.abs().reshape(g.shape) + R.TINY[x.dtype], f"gradient of {name}")
    return (x_out, y, rp, rn), got


KINDS = pytest.mark.parametrize("kind", [None, "vector", "sequence", "element"], ids=["none", "vector", "sequence", "element"])


@EACH
@KINDS
@pytest.mark.parametrize("shape", [(2, 3, 1), (3, 4, 7), (2, 5, 64), (1, 1, 256), (3, 5, 257), (2, 7, 512), (2, 3, 1000), (5, 2, 1023), (2, 3, 4096)],
                         ids=lambda s: "x".join(map(str, s)))
def test_block(cuda, tpb, dtype, kind, shape):
    check_block(tpb, block_inputs(cuda, shape, dtype, kind, 3), kind)


@EACH
@pytest.mark.parametrize("width", [8192, 8200, 12296, 16384, 16383])
def test_block_of_wide_rows(cuda, tpb, dtype, width):
    check_block(tpb, block_inputs(cuda, (2, 2, width), dtype, "vector", 4), "vector")


@EACH
@pytest.mark.parametrize("p,width", [(0.1, 64), (0.5, 77), (0.9, 1032), (1.0, 40), (1e-6, 40)])
def test_block_with_dropout(cuda, tpb, dtype, p, width):
    v = block_inputs(cuda, (2, 4, width), dtype, "element", 6)
    check_block(tpb, v, "element", p=p, seed=(1 << 63) + 12345, offset=(1 << 40) + 7)
    v["gate"] = None
    check_block(tpb, v, None, p=p, seed=99, post=False)


@EACH
def test_block_without_one_of_the_norms(cuda, tpb, dtype):
    v = block_inputs(cuda, (3, 5, 320), dtype, "vector", 8)
    check_block(tpb, v, "vector", post=False)
    check_block(tpb, v, "vector", nxt=False)
    check_block(tpb, v, "vector", post=False, nxt=False)
    check_block(tpb, v, "vector", with_gx=False)
    check_block(tpb, v, "vector", nxt=False, with_gx=False)


@EACH
@KINDS
def test_block_of_many_rows(cuda, tpb, dtype, kind):
    """More rows than workers, groups that split unevenly, more groups than workers, two-dim inputs."""
    check_block(tpb, block_inputs(cuda, (3, 1201, 136), dtype, kind, 11), kind)
    check_block(tpb, block_inputs(cuda, (1501, 3, 1032), dtype, kind, 12), kind)
    check_block(tpb, block_inputs(cuda, (5003, 2, 72), dtype, kind, 13), kind)
    if kind != "sequence":
        check_block(tpb, block_inputs(cuda, (3001, 600), dtype, kind, 14), kind)
        check_block(tpb, block_inputs(cuda, (640,), dtype, kind, 15), kind)


@EACH
def test_block_of_views(cuda, tpb, dtype):
    wide = block_inputs(cuda, (3, 9, 211), dtype, "element", 21)
    for cut in (lambda t: t[:, 1:, 3:], lambda t: t[:, ::2, :208], lambda t: t[..., 1:129], lambda t: t[:, 2]):
        v = {k: cut(t) if t.dim() == 3 else t[:cut(wide["x"]).shape[-1]] for k, t in wide.items()}
        check_block(tpb, v, "element")
    v = dict(wide, x=wide["x"][:1, :1].expand(3, 9, 211), gx=wide["gx"][:, :1].expand(3, 9, 211))
    check_block(tpb, v, "element")
    many = block_inputs(cuda, (2, 3, 4, 40), dtype, "sequence", 22)
    check_block(tpb, many, "sequence")
    none = block_inputs(cuda, (2, 0, 64), dtype, "vector", 23)
    x_out, y, rp, rn = tpb.block_residual(none["x"], none["h"], none["post"], none["next"], none["gate"])
    got = tpb.block_residual_backward(none["gx"], none["gy"], none["h"], x_out, rp, rn, none["post"], none["next"], none["gate"])
    assert x_out.shape == got[0].shape == (2, 0, 64) and all(bool((g == 0).all()) for g in got[2:])


@EACH
def test_block_of_zeros_and_huge_values(cuda, tpb, dtype):
    v = block_inputs(cuda, (1, 4, 128), dtype, None, 24)
    v["h"][0, 0] = 0
    v["x"][0, 0] = 0
    v["h"][0, 1] = 1e-4
    big = 6e4 if dtype == torch.float16 else 1e18
    v["h"][0, 2] = big
    check_block(tpb, v, None)
    v["h"][0, 3, 5] = float("nan")
    x_out, y, _, _ = tpb.block_residual(v["x"], v["h"], v["post"], v["next"])
    assert bool(x_out[0, 3].isnan().all()) and not bool(x_out[0, :3].isnan().any()) and not bool(y[0, :3].isnan().any())


@EACH
@pytest.mark.parametrize("shape", [(1, 1), (5, 64), (3, 5, 1023), (2000, 256), (7, 16384)], ids=lambda s: "x".join(map(str, s)))
def test_rms_norm(cuda, tpb, dtype, shape):
    v = block_inputs(cuda, shape, dtype, None, 31)
    y, rstd = tpb.rms_norm(v["x"], v["next"], 1e-5)
    want = R.block_forward(v["x"], torch.zeros_like(v["x"]), None, v["next"], None, 1.0, 1e-5, 1.0)
    close(y, want["y"], want["y_bound"] + u(dtype) * want["y"].abs() + R.TINY[dtype], "y")
    close(rstd, want["rstd_next"], want["rstd_next"] * 2.0 ** -18, "rstd")
    gx, gw = tpb.rms_norm_backward(v["gy"], v["x"], v["next"], rstd)
    back = R.block_backward(None, v["gy"], v["x"], v["x"], None, rstd, None, v["next"], None, None, 0.0, 1.0)
    for name, g in (("x", gx), ("next", gw)):
        value, tol = back[name]
        close(g, value, tol + u(dtype) * value.abs() + R.TINY[dtype], f"gradient of {name}")


def test_block_gradients_against_differences(cuda, tpb):
    """Gradients of sum(c1 x_out + c2 y) from differences of the 64-bit formula."""
    v = block_inputs(cuda, (2, 3, 24), torch.float32, "sequence", 41)
    how = {"scale": 0.6, "p": 0.3, "seed": 5, "offset": 6}
    x_out, y, rp, rn = tpb.block_residual(v["x"], v["h"], v["post"], v["next"], v["gate"], eps=1e-5, **how)
    got = tpb.block_residual_backward(v["gx"], v["gy"], v["h"], x_out, rp, rn, v["post"], v["next"], v["gate"], **how)
    f = R.philox_factors(144, 0.3, 5, 6, cuda).view(2, 3, 24)

    def value(**change):
        w = {**v, **change}
        out = R.block_forward(w["x"], w["h"], w["post"], w["next"], w["gate"], 0.6, 1e-5, f)
        return (out["x"] * v["gx"].double()).sum() + (out["y"] * v["gy"].double()).sum()

    for name, g in zip(("x", "h", "post", "next", "gate"), got):
        for i in (0, 11, v[name].numel() - 1):
            at = lambda d: value(**{name: v[name].double().flatten().index_put((torch.tensor(i),), torch.tensor(d, dtype=torch.float64), accumulate=True).view(v[name].shape)})  # noqa: E731, B023
            slope = (at(1e-5) - at(-1e-5)) / 2e-5
            # third derivatives are under 1e3 here: 1e-10 * 1e3 / 6, float64 noise 1e-13 / 1e-5; the float32 kernels 1e-5
            close(g.flatten()[i], slope, 1e-4 * (1 + slope.abs().item()), f"{name}[{i}]")


# ------------------------------------------------------------------------------------ dropout

@EACH
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((8,), 0.1), ((13,), 0.5), ((5, 37), 0.25), ((3, 4, 64), 0.9), ((2, 1000), 1.0), ((7, 9), 0.0), ((0, 8), 0.5), ((), 0.5)])
def test_dropout(cuda, tpb, dtype, shape, p):
    x = logits_of(cuda, shape, dtype, 51)
    seed, offset = (1 << 64) - 3, (1 << 33) + 1
    f = R.philox_factors(x.numel(), p, seed, offset, cuda).view(x.shape)
    want = x.double() * f
    for fn in (tpb.dropout, tpb.dropout_backward):
        got = fn(x, p, seed, offset)
        assert got.dtype == dtype and got.shape == x.shape
        close(got, want, (u(dtype) + 2.0 ** -23) * want.abs() + R.TINY[dtype], "dropout")
        assert torch.equal(got == 0, want == 0)


@EACH
def test_dropout_of_views_draws_by_position(cuda, tpb, dtype):
    base = logits_of(cuda, (5, 7, 41), dtype, 52)
    for v in (base[:, 1:], base[:, ::2, 3:], base[1:, :, :40], base[..., :1], base[:1].expand(5, 7, 41), base[:, 2]):
        assert torch.equal(tpb.dropout(v, 0.4, 9, 2), tpb.dropout(v.contiguous(), 0.4, 9, 2))
    flat = base.flatten()
    assert torch.equal(tpb.dropout(flat[3:], 0.4, 9), tpb.dropout(flat[3:].clone(), 0.4, 9))


def test_dropout_share_and_independence(cuda, tpb):
    n = 1 << 20
    one = torch.ones(n, device=cuda)
    for p in (0.1, 0.5, 0.9):
        kept = tpb.dropout(one, p, 77) != 0
        # a binomial share: six standard deviations
        assert abs(kept.double().mean().item() - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5 + 2.0 ** -17
        other = tpb.dropout(one, p, 77, 1) != 0
        both = (kept & other).double().mean().item()
        assert abs(both - (1 - p) ** 2) < 6 * ((1 - p) ** 2 / n) ** 0.5 + 2.0 ** -15
    special = torch.tensor([float("nan"), float("inf")] * 500, device=cuda)
    got = tpb.dropout(special, 0.5, 3)
    dropped = tpb.dropout(torch.ones(1000, device=cuda), 0.5, 3) == 0
    assert bool((got[dropped] == 0).all()) and not bool(got[~dropped].isfinite().any())


# ------------------------------------------------------------------------------------ how they are called

def test_refusals(cuda, tpb):
    x, lab = logits_of(cuda, (4, 8), torch.float32, 1), labels_of(cuda, (4,), 8, 2)
    one = torch.ones(4, device=cuda)
    w = torch.ones(8, device=cuda)
    bad = [
        (TypeError, lambda: tpb.token_logprobs(x, lab.int())), (ValueError, lambda: tpb.token_logprobs(x, lab[:3])),
        (RuntimeError, lambda: tpb.token_logprobs(x, lab.cpu())), (NotImplementedError, lambda: tpb.token_logprobs(x.double(), lab)),
        (NotImplementedError, lambda: tpb.token_logprobs(x.t(), lab[:1].expand(8))),
        (ValueError, lambda: tpb.token_logprobs(x, lab, out=(one, one))), (ValueError, lambda: tpb.token_logprobs(x, lab, out=(one,))),
        (ValueError, lambda: tpb.token_logprobs_backward(one, x, lab, one, out=(x,))),
        (TypeError, lambda: tpb.token_logprobs_backward(one.double(), x, lab, one)),
        (ValueError, lambda: tpb.policy_loss(x, lab, one, one, one, kl_coef=0.1)), (TypeError, lambda: tpb.policy_loss(x, lab, one, one.half(), one)),
        (ValueError, lambda: tpb.policy_loss(x, lab, one, torch.ones(3, device=cuda), one)),
        (RuntimeError, lambda: tpb.policy_loss(x, lab, one, one, one, clip_low=2.0)),
        (ValueError, lambda: tpb.preference_loss(x, lab, one)), (ValueError, lambda: tpb.preference_loss(x, lab, one, torch.tensor([0, 4], device=cuda))),
        (TypeError, lambda: tpb.preference_loss(x, lab, one, torch.tensor([0, 2, 4], device=cuda, dtype=torch.int32))),
        (RuntimeError, lambda: tpb.preference_loss(x, lab, one, torch.tensor([0, 2, 4]))),
        (RuntimeError, lambda: tpb.preference_loss(x, lab, one, torch.tensor([0, 2, 4], device=cuda), label_smoothing=0.7)),
        (TypeError, lambda: tpb.rms_norm(x, w.half())), (ValueError, lambda: tpb.rms_norm(x, w[:7])), (TypeError, lambda: tpb.rms_norm(x, None)),
        (NotImplementedError, lambda: tpb.rms_norm(torch.zeros(2, 16385, device=cuda), torch.zeros(16385, device=cuda))),
        (ValueError, lambda: tpb.block_residual(x, x[:3])), (ValueError, lambda: tpb.block_residual(x, x, gate=w[:4])),
        (ValueError, lambda: tpb.block_residual(x, x, gate=one[:, None])), (RuntimeError, lambda: tpb.block_residual(x, x, p=1.5)),
        (ValueError, lambda: tpb.block_residual(x, x, seed=-1)), (ValueError, lambda: tpb.block_residual(x, x, offset=1 << 64)),
        (TypeError, lambda: tpb.block_residual_backward(x, None, x, x, None, None, None, w)),
        (ValueError, lambda: tpb.block_residual_backward(x, x, x, x, None, None)),
        (ValueError, lambda: tpb.block_residual_backward(x, x, x, x, None, None, None, w)),
        (RuntimeError, lambda: tpb.dropout(x, float("nan"), 1)), (ValueError, lambda: tpb.dropout(x, 0.5, 1 << 64)),
        (ValueError, lambda: tpb.dropout(x, 0.5, 1, out=(x,))),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"refusal {i} did not happen")
    torch.cuda.synchronize()


def test_outputs_passed_in(cuda, tpb):
    x, lab, old, adv, w, ref = policy_inputs(cuda, (6,), 300, torch.bfloat16, 61)
    fresh = tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1)
    out = tuple(torch.full_like(t, 7.0) for t in fresh)
    got = tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1, out=out)
    for a, b, c in zip(fresh, got, out):
        assert torch.equal(a, b) and b is c
    v = block_inputs(cuda, (2, 3, 64), torch.bfloat16, "vector", 62)
    fresh = tpb.block_residual(v["x"], v["h"], None, v["next"], v["gate"])
    out = tuple(None if t is None else torch.full_like(t, 7.0) for t in fresh)
    got = tpb.block_residual(v["x"], v["h"], None, v["next"], v["gate"], out=out)
    assert all(a is None or (torch.equal(a, b) and b is c) for a, b, c in zip(fresh, got, out))


@EACH
def test_same_bits_every_time_and_on_another_stream(cuda, tpb, dtype):
    x, lab, old, adv, w, ref = policy_inputs(cuda, (4, 60), 5001, dtype, 71)
    v = block_inputs(cuda, (3, 700, 1024), dtype, "vector", 72)

    def both():
        x_out, y, rp, rn = tpb.block_residual(v["x"], v["h"], v["post"], v["next"], v["gate"], p=0.1, seed=1)
        return [*tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1), *tpb.preference_loss(x, lab, ref),
                x_out, y, *tpb.block_residual_backward(v["gx"], v["gy"], v["h"], x_out, rp, rn, v["post"], v["next"], v["gate"], p=0.1, seed=1)]

    first = both()
    side = [torch.cuda.Stream() for _ in range(2)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for s in side:                     # the two streams' calls overlap
            with torch.cuda.stream(s):
                got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(first, g))


def test_captured_and_replayed(cuda, tpb):
    """Two graphs that live side by side, replayed on new inputs in any order, next to eager calls."""
    x, lab, old, adv, w, ref = policy_inputs(cuda, (30,), 3001, torch.bfloat16, 81)
    v = block_inputs(cuda, (2, 50, 640), torch.bfloat16, "sequence", 82)
    offsets = torch.tensor([0, 7, 19, 20, 30], device=cuda)

    def losses():
        return [*tpb.policy_loss(x, lab, old, adv, w, ref, kl_coef=0.1), *tpb.preference_loss(x, lab, ref, offsets)]

    def block():
        x_out, y, rp, rn = tpb.block_residual(v["x"], v["h"], v["post"], v["next"], v["gate"], p=0.1, seed=1)
        return [x_out, y, *tpb.block_residual_backward(v["gx"], v["gy"], v["h"], x_out, rp, rn, v["post"], v["next"], v["gate"], p=0.1, seed=1)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses(), block()
    torch.cuda.synchronize()
    graphs = []
    for fn in (losses, block):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kept = fn()
        graphs.append((g, kept, fn))
    for seed in (91, 92):
        x.copy_(logits_of(cuda, x.shape, x.dtype, seed))
        lab.copy_(labels_of(cuda, lab.shape, 3001, seed, 0.1))
        v["h"].copy_(logits_of(cuda, v["h"].shape, x.dtype, seed + 10))
        for order in ((0, 1), (1, 0)):
            for i in order:
                graphs[i][0].replay()
                eager = graphs[i][2]()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], eager))


def test_positions_beyond_31_bits(cuda, tpb):
    """A gradient of more than 2^31 elements, from one row of logits that stands for all (stride 0)."""
    v, n = 131075, 16400
    one = logits_of(cuda, (1, v), torch.bfloat16, 101)
    lab = labels_of(cuda, (n,), v, 102, 0.95)
    lab[-1] = v - 1
    x = one.expand(n, v)
    logp, lse = tpb.token_logprobs(x, lab)
    g = tpb.token_logprobs_backward(torch.ones(n, device=cuda), x, lab, lse)
    assert g.numel() > 1 << 31
    for r in (0, n // 2, n - 2, n - 1):
        want, tol = R.grad_of(one, lab[r:r + 1], (lab[r:r + 1] >= 0).double())
        close(g[r:r + 1], want, tol + want.abs() * (u(torch.bfloat16) + 2.0 ** -19) + 1e-30, f"row {r}")
    del g
    big = torch.zeros((1 << 31) + 24, dtype=torch.bfloat16, device=cuda)
    big[-24:] = 1.0
    got = tpb.dropout(big, 0.5, 7, 8)[-24:]
    f = []
    for b in range((1 << 28), (1 << 28) + 3):      # the last three blocks of the generator
        c, k, m = [b & 0xFFFFFFFF, b >> 32, 8, 0], [7, 0], 0xFFFFFFFF
        for _ in range(10):
            p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & m, (p0 >> 32) ^ c[3] ^ k[1], p0 & m]
            k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
        for word in c:
            f += [2.0 if word & 0xFFFF >= 32768 else 0.0, 2.0 if word >> 16 >= 32768 else 0.0]
    assert got.tolist() == f


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_current(cuda, tpb):
    other = torch.device("cuda", 1)
    x, lab = logits_of(cuda, (5, 300), torch.bfloat16, 1), labels_of(cuda, (5,), 300, 2)
    here, there = tpb.token_logprobs(x, lab), tpb.token_logprobs(x.to(other), lab.to(other))
    assert all(torch.equal(a, b.to(cuda)) for a, b in zip(here, there))


def test_a_training_step_of_a_small_model(cuda, tpb):
    """The operators together, as a model uses them: embedding, two gated blocks on a residual path with norms
    and dropout, logits, policy loss; every gradient against autograd in 64 bits."""
    B, Tn, D, V, layers = 2, 6, 48, 301, 2
    g = gen(cuda, 7)
    make = lambda *s, k=1.0: k * torch.randn(*s, device=cuda, generator=g)  # noqa: E731
    emb, head = make(V, D), make(D, V, k=0.15)
    w_in = [make(D, D, k=0.15) for _ in range(layers)]
    norms = [1 + 0.1 * make(D) for _ in range(2 * layers + 1)]              # first, then (post, next) of every block
    gates = [torch.sigmoid(make(B, 1, D)), torch.sigmoid(make(D))]
    tokens = torch.randint(0, V, (B, Tn + 1), device=cuda, generator=g)
    inp, lab = tokens[:, :-1], tokens[:, 1:]
    adv, w = make(B, 1), torch.full((B, Tn), 1.0 / (B * Tn), device=cuda)
    how = lambda i: {"scale": 0.7, "p": 0.2, "seed": 42, "offset": i}  # noqa: E731

    # 64 bits, autograd
    leaves = [t.double().requires_grad_(True) for t in (emb, head, *w_in, *norms, *gates)]
    e64, hd, win, nm, gt = leaves[0], leaves[1], leaves[2:4], leaves[4:9], leaves[9:]
    rms = lambda t, wt: t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * wt  # noqa: E731
    s = e64[inp]
    y = rms(s, nm[0])
    for i in range(layers):
        f = R.philox_factors(B * Tn * D, 0.2, 42, i, cuda).view(B, Tn, D)
        s = s + 0.7 * gt[i] * rms(y @ win[i], nm[1 + 2 * i]) * f
        y = rms(s, nm[2 + 2 * i])
    logits64 = y @ hd
    lp = torch.log_softmax(logits64, -1).gather(-1, lab.unsqueeze(-1)).squeeze(-1)
    old = (lp.detach() + torch.where(make(B, Tn) > 0, 0.1, -0.35)).float()      # ratios near 0.9 and 1.42: clipped ones among them
    ref = (lp.detach() + 0.2).float()
    r = (lp - old.double()).exp()
    d = ref.double() - lp
    loss64 = (w.double() * (-torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (d.exp() - d - 1))).sum()
    want = torch.autograd.grad(loss64, leaves)

    # the operators
    x = emb[inp]
    y, rstd0 = tpb.rms_norm(x, norms[0])
    saved = []
    stream, x0 = x, x
    for i in range(layers):
        h = y @ w_in[i]
        out, y2, rp, rn = tpb.block_residual(stream, h, norms[1 + 2 * i], norms[2 + 2 * i], gates[i], **how(i))
        saved.append((y, h, out, rp, rn))
        stream, y = out, y2
    loss, gl, *_ = tpb.policy_loss(y @ head, lab, old, adv, w, ref, kl_coef=0.1)
    close(loss, loss64, 1e-5 * (1 + loss64.abs().item()), "loss")
    got_norms, got_gates, got_w = [None] * (2 * layers + 1), [None] * layers, [None] * layers
    g_head = y.flatten(0, 1).t() @ gl.flatten(0, 1)
    gy, gx = gl @ head.t(), None
    for i in reversed(range(layers)):
        y_in, h, out, rp, rn = saved[i]
        gx, gh, got_norms[1 + 2 * i], got_norms[2 + 2 * i], got_gates[i] = tpb.block_residual_backward(
            gx, gy, h, out, rp, rn, norms[1 + 2 * i], norms[2 + 2 * i], gates[i], **how(i))
        got_w[i] = y_in.flatten(0, 1).t() @ gh.flatten(0, 1)
        gy = gh @ w_in[i].t()
    g0, got_norms[0] = tpb.rms_norm_backward(gy, x0, norms[0], rstd0)
    g_emb = torch.zeros_like(emb).index_put_((inp.flatten(),), (gx + g0).flatten(0, 1), accumulate=True)
    for i, (a, b) in enumerate(zip([g_emb, g_head, *got_w, *got_norms, *got_gates], want)):
        # float32 matrix products of 48 and 301 terms on the way, forward and back: a few 1e-6 of the largest entry
        close(a, b, 5e-5 * b.abs().max().item() + 1e-5 * b.abs(), f"gradient {i}")


def test_under_the_range_checker(cuda):
    """The same tests with every global access compared with the ranges of its call."""
    from tensorplay_b200 import _lib
    if _lib.CHECKED:
        pytest.skip("already running under the checked build")
    assert os.path.exists(os.path.join(ROOT, "tensorplay_b200", "libtpb200_checked.so")), "libtpb200_checked.so was not built"
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.join("tests", "test_gpu_training.py"), "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider",
                        "-k", "not another_stream and not beyond_31 and not captured and not share_and and not not_current"],
                       cwd=ROOT, env=dict(os.environ, TPB200_CHECKED="1"), capture_output=True, text=True, timeout=1500)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
    assert " passed" in r.stdout
