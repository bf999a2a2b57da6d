"""Training operators on rows, on top of the tpb200 C ABI: what a training step of a language model does
next to the reductions and softmax of `ops`.  No reference counterpart.

    token_logprobs(logits, labels) -> (logp, lse)
    token_logprobs_backward(grad_logp, logits, labels, lse) -> grad_logits
    policy_loss(logits, labels, old_logp, advantages, weights, ref_logp=None, ...) -> (loss, grad_logits, logp, ratio, kl)
    preference_loss(logits, labels, ref_logp, offsets=None, ...) -> (loss, grad_logits, rewards, logp)
    rms_norm(x, weight, eps=1e-6) -> (y, rstd)
    rms_norm_backward(grad_y, x, weight, rstd) -> (grad_x, grad_weight)
    block_residual(x, h, post_weight=None, next_weight=None, gate=None, ...) -> (x_out, y, rstd_post, rstd_next)
    block_residual_backward(...) -> (grad_x, grad_h, grad_post_weight, grad_next_weight, grad_gate)
    dropout(x, p, seed, offset=0) -> y                dropout_backward(grad_y, p, seed, offset=0) -> grad_x

float32, bfloat16 and float16 CUDA tensors (one type per call); everything is computed in float32 or
more and rounded once.  Rows are the last dim, which must have unit stride; the other dims may have any
strides as long as all but the last of them collapse to one.  Results are contiguous, and a gradient has
the type of what it is the gradient of.  The functions only enqueue on the current stream; scratch memory
comes from torch's allocator on every call, so that calls on other streams and captured graphs share none.

No function records an autograd graph, whatever its inputs require: the gradients come from the *_backward functions
and from the losses themselves (wrap them in a torch.autograd.Function to use them in one).  `seed` and `offset` of
a dropout are numbers of the call: a captured graph holds them, and every replay drops the same elements.
To drop others, capture once per offset, or call dropout outside of the graph.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from .ops import _check_out

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
MAX_WIDTH = 16384


def _check_tensor(x, what):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{what}: tpb200 kernels run on CUDA tensors only (got {x.device}); there is no CPU path")
    if x.dtype not in _TYPES:
        raise NotImplementedError(f"{what} not implemented for this dtype ({x.dtype}); float32, bfloat16 and float16 only")
    if x.dim() > _lib.MAX_DIMS:
        raise NotImplementedError(f"{what}: tensors of rank {x.dim()} are not supported")


@functools.lru_cache(maxsize=4096)
def _collapse(lead, st):
    """(outer, inner) strides as the ABI takes them for the leading sizes `lead` with strides `st`: the last
    is `inner`, the ones before it have to collapse to one; None if they do not."""
    if len(lead) == 0:
        return _lib.pair(0, 0)
    size, step = 1, 0
    for n, s in zip(reversed(lead[:-1]), reversed(st[:-1])):
        if n == 1:
            continue
        if size > 1 and s != size * step and 0 not in lead:
            return None
        if size == 1:
            step = s
        size *= n
    return _lib.pair(step, st[-1])


def _strides(x, lead, what, name):
    got = _collapse(lead, x.stride()[:len(lead)])
    if got is None:
        raise NotImplementedError(f"{what}: the leading dims of {name} do not collapse to one stride (use contiguous())")
    return got


def _split(lead):
    """(outer, inner) of the leading sizes."""
    if len(lead) == 1:
        return 1, lead[0]
    return (math.prod(lead[:-1]), lead[-1]) if lead else (1, 1)


def _row_strides(x, what, name):
    if x.dim() == 0:
        raise ValueError(f"{what}: {name} needs at least one dim")
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise NotImplementedError(f"{what}: the last dim of {name} must have unit stride (use contiguous())")
    return _strides(x, x.shape[:-1], what, name)


def _same(t, like, what, name, shape=None):
    """Another tensor of the same call: same type, device and (unless given) shape."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a tensor")
    if t.device != like.device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, expected {like.device}")
    if t.dtype != like.dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, expected {like.dtype}")
    want = like.shape if shape is None else shape
    if tuple(t.shape) != tuple(want):
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(want)}")
    return t


def _token(t, logits, dtype, what, name, broadcast=False):
    """A value per token: (pointer, strides).  `broadcast`: sizes of 1 and missing dims stand for all tokens."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a tensor")
    if t.device != logits.device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, expected {logits.device}")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} must be {dtype} (got {t.dtype})")
    lead = logits.shape[:-1]
    if t.shape != lead:
        if not broadcast:
            raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(lead)}")
        try:
            t = t.expand(lead)
        except RuntimeError:
            raise ValueError(f"{what}: {name} of shape {tuple(t.shape)} does not broadcast to {tuple(lead)}") from None
    return t.data_ptr(), _strides(t, lead, what, name)


def _logits(logits, labels, what):
    _check_tensor(logits, what)
    if logits.dim() < 1:
        raise ValueError(f"{what}: logits need at least one dim")
    strides = _row_strides(logits, what, "logits")
    outer, inner = _split(logits.shape[:-1])
    rows = (logits.data_ptr(), _TYPES[logits.dtype], outer, inner, logits.shape[-1], strides)
    return rows, _token(labels, logits, torch.int64, what, "labels")


def _new(shape, dtype, like):
    """A new contiguous tensor on the device of `like`; empty_like takes half the time of empty."""
    if dtype == like.dtype:
        if shape == like.shape and like.is_contiguous():
            return torch.empty_like(like)
        return like.new_empty(shape)
    return like.new_empty(shape, dtype=dtype)


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _outputs(what, like, out, specs):
    """New contiguous outputs, or the ones of `out` after a check; specs: (shape, dtype) or None each."""
    if out is None:
        outs, last = [], None
        for s in specs:
            # the same spec again: empty_like takes half the time of new_empty
            outs.append(None if s is None else torch.empty_like(outs[-1]) if s is last else _new(s[0], s[1], like))
            last = s
        return outs
    device = like.device
    if not isinstance(out, (tuple, list)) or len(out) != len(specs):
        raise ValueError(f"{what}: out must hold {len(specs)} tensors")
    for t, s in zip(out, specs):
        if s is None:
            if t is not None:
                raise ValueError(f"{what}: this call has no such output; pass None in its place")
        else:
            _check_out(t, s[0], s[1], device, what)
    return list(out)


def _no_overlap(what, outs, ins):
    """Outputs that the caller passes may not share memory with an input or with one another."""
    def span(t):
        lo = hi = 0
        for n, s in zip(t.shape, t.stride()):
            if n == 0:
                return None
            lo, hi = (lo + (n - 1) * s, hi) if s < 0 else (lo, hi + (n - 1) * s)
        size = t.element_size()
        return t.data_ptr() + lo * size, t.data_ptr() + (hi + 1) * size
    done = [s for s in map(span, (t for t in ins if t is not None)) if s]
    for t in outs:
        s = span(t) if t is not None else None
        if s is None:
            continue
        for u in done:
            if s[0] < u[1] and u[0] < s[1]:
                raise ValueError(f"{what}: out must not overlap an input or another output")
        done.append(s)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)     # torch.cuda.current_stream builds an object: 4 us


class _Stay:
    """The current device is the right one already (torch.cuda.device costs 3 us either way)."""

    def __enter__(self):
        pass

    def __exit__(self, *_):
        pass


_STAY = _Stay()


def _on(device):
    return _STAY if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


# ---------------------------------------------------------------------------- objectives on logits

def token_logprobs(logits, labels, *, out=None):
    """Log-probabilities of the labels under softmax(logits) along the last dim, and the normaliser:
    logp = logits[label] - lse, lse = log sum exp(logits), both float32 of shape logits.shape[:-1].

    `labels`: int64 of that shape; a negative label (e.g. -100) takes no part: its row is not read and its
    logp and lse are 0; a label beyond the vocabulary gives NaN.  `out=(logp, lse)`."""
    what = "token_logprobs"
    rows, lab = _logits(logits, labels, what)
    f32 = (logits.shape[:-1], torch.float32)
    with _on(logits.device):
        logp, lse = _outputs(what, logits, out, [f32, f32])
        if out is not None:
            _no_overlap(what, (logp, lse), (logits, labels))
        _lib.check(_lib.lib().tpb200_token_logprobs(*rows, *lab, logp.data_ptr(), lse.data_ptr(), _stream(logits.device)))
    return logp, lse


def token_logprobs_backward(grad_logp, logits, labels, lse, *, out=None):
    """Gradient of token_logprobs' logp: grad_logp * (one at the label - softmax(logits)), in the logits'
    type.  `grad_logp` (float32) broadcasts to the tokens; `lse` is the forward call's.  Rows whose float32 lse
    does not hold the digits (|lse| of 32 and more, a token with half of the probability) are summed again.
    `out=(grad_logits,)`."""
    what = "token_logprobs_backward"
    rows, lab = _logits(logits, labels, what)
    grad = _token(grad_logp, logits, torch.float32, what, "grad_logp", broadcast=True)
    _token(lse, logits, torch.float32, what, "lse")
    if not lse.is_contiguous():
        raise ValueError(f"{what}: lse must be contiguous, as token_logprobs returns it")
    with _on(logits.device):
        g, = _outputs(what, logits, out, [(logits.shape, logits.dtype)])
        if out is not None:
            _no_overlap(what, (g,), (logits, labels, grad_logp, lse))
        _lib.check(_lib.lib().tpb200_token_logprobs_backward(*grad, *rows, *lab, lse.data_ptr(), g.data_ptr(), _stream(logits.device)))
    return g


def policy_loss(logits, labels, old_logp, advantages, weights, ref_logp=None, *, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                grad_scale=1.0, need_grad=True, out=None):
    """Clipped policy loss with a KL term, and its gradient with respect to the logits, in one call.

        ratio = exp(logp - old_logp)              kl = exp(d) - d - 1,  d = ref_logp - logp
        loss = sum over tokens of weights * (-min(ratio * A, clip(ratio, 1 - clip_low, 1 + clip_high) * A) + kl_coef * kl)

    old_logp, advantages (A), weights and ref_logp are float32 and broadcast to labels.shape; the weights
    carry the mask and the mean.  A token of weight 0 or with a negative label takes no part: its row is not
    read, its logp, ratio, kl and gradient are 0.  Returns (loss, grad_logits, logp, ratio, kl): loss 0-dim,
    grad_logits = grad_scale * d loss / d logits in the logits' type (None without need_grad), the rest per
    token.  `out`: these five."""
    what = "policy_loss"
    rows, lab = _logits(logits, labels, what)
    args = [_token(t, logits, torch.float32, what, name, broadcast=True)
            for t, name in ((old_logp, "old_logp"), (advantages, "advantages"), (weights, "weights"))]
    args.append((None, None) if ref_logp is None else _token(ref_logp, logits, torch.float32, what, "ref_logp", broadcast=True))
    if ref_logp is None and kl_coef:
        raise ValueError(f"{what}: kl_coef needs ref_logp")
    device, lead = logits.device, logits.shape[:-1]
    L = _lib.lib()
    f32 = (lead, torch.float32)
    with _on(device):
        nbytes = L.tpb200_policy_loss_workspace_bytes(rows[2], rows[3])
        loss, grad, logp, ratio, kl = _outputs(what, logits, out, [((), torch.float32), (logits.shape, logits.dtype) if need_grad else None, f32, f32, f32])
        if out is not None:
            _no_overlap(what, (loss, grad, logp, ratio, kl), (logits, labels, old_logp, advantages, weights, ref_logp))
        ws = _scratch(nbytes, device)
        _lib.check(L.tpb200_policy_loss(*rows, *lab, *args[0], *args[1], *args[2], *args[3], clip_low, clip_high, kl_coef, grad_scale,
                                        loss.data_ptr(), _ptr(grad), logp.data_ptr(), ratio.data_ptr(), kl.data_ptr(), _ptr(ws), nbytes,
                                        _stream(device)))
    return loss, grad, logp, ratio, kl


def preference_loss(logits, labels, ref_logp, offsets=None, *, beta=0.1, label_smoothing=0.0, grad_scale=1.0, need_grad=True, out=None):
    """Preference loss on pairs of sequences (2p: chosen, 2p + 1: rejected), and its gradient.

        s_q = sum over sequence q of (logp - ref_logp),  rewards[q] = beta * s_q,  m_p = rewards[2p] - rewards[2p + 1]
        loss = mean over pairs of -(1 - e) * log sigmoid(m_p) - e * log sigmoid(-m_p),   e = label_smoothing

    Packed logits [tokens, vocab] come with `offsets`, int64 [2 * pairs + 1] on the device: sequence q is the
    rows offsets[q] .. offsets[q + 1] - 1 (non-decreasing, else the loss is NaN); rows in no sequence have a zero
    gradient.  Logits of more dims, without offsets, hold one sequence per leading index.  Tokens with a
    negative label take no part.  Returns (loss, grad_logits, rewards [2 * pairs], logp).  `out`: these four."""
    what = "preference_loss"
    rows, lab = _logits(logits, labels, what)
    ref = _token(ref_logp, logits, torch.float32, what, "ref_logp")
    device = logits.device
    if offsets is None:
        if logits.dim() < 3:
            raise ValueError(f"{what}: packed logits need offsets")
        sequences = rows[2]
    else:
        if logits.dim() != 2:
            raise ValueError(f"{what}: offsets go with packed logits [tokens, vocab]")
        if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int64 or offsets.dim() != 1 or not offsets.is_contiguous():
            raise TypeError(f"{what}: offsets must be a contiguous 1-D int64 tensor")
        if offsets.device != device:
            raise RuntimeError(f"{what}: offsets is on {offsets.device}, expected {device}")
        sequences = offsets.shape[0] - 1
    if sequences < 2 or sequences % 2:
        raise ValueError(f"{what}: an even number of sequences is needed (got {sequences})")
    L = _lib.lib()
    with _on(device):
        loss, grad, rewards, logp = _outputs(what, logits, out, [((), torch.float32), (logits.shape, logits.dtype) if need_grad else None,
                                                                 ((sequences,), torch.float32), (logits.shape[:-1], torch.float32)])
        if out is not None:
            _no_overlap(what, (loss, grad, rewards, logp), (logits, labels, ref_logp, offsets))
        nbytes = L.tpb200_preference_loss_workspace_bytes(rows[2], rows[3], sequences // 2)
        ws = _scratch(nbytes, device)
        _lib.check(L.tpb200_preference_loss(*rows, *lab, *ref, _ptr(offsets), sequences // 2, beta, label_smoothing, grad_scale,
                                            loss.data_ptr(), _ptr(grad), rewards.data_ptr(), logp.data_ptr(), _ptr(ws), nbytes, _stream(device)))
    return loss, grad, rewards, logp


# ---------------------------------------------------------------------------- the residual path

def _width(x, what):
    if x.dim() == 0:
        raise ValueError(f"{what}: at least one dim is needed")
    if x.shape[-1] > MAX_WIDTH:
        raise NotImplementedError(f"{what}: rows of at most {MAX_WIDTH} elements (got {x.shape[-1]})")
    outer, inner = _split(x.shape[:-1])
    return outer, inner, x.shape[-1]


def _weight(w, x, what, name):
    if w is None:
        return None
    _same(w, x, what, name, (x.shape[-1],))
    if not w.is_contiguous():
        raise ValueError(f"{what}: {name} must be contiguous")
    return w


def _gate(gate, x, what):
    """(kind, strides, gradient shape) of a gate of shape [width], x.shape with 1 in place of the rows of a
    sequence ([..., 1, width]), or x.shape."""
    if gate is None:
        return _lib.GATE["none"], None
    if not isinstance(gate, torch.Tensor):
        raise TypeError(f"{what}: gate must be a tensor")
    width, lead = x.shape[-1], x.shape[:-1]
    if tuple(gate.shape) == tuple(x.shape):
        _same(gate, x, what, "gate")
        return _lib.GATE["element"], _row_strides(gate, what, "gate")
    if tuple(gate.shape) == (width,):
        _same(gate, x, what, "gate", (width,))
        if gate.stride(0) != 1 and width > 1:
            raise NotImplementedError(f"{what}: the last dim of gate must have unit stride (use contiguous())")
        return _lib.GATE["vector"], _lib.pair(0, 0)
    if len(lead) >= 2 and tuple(gate.shape) == (*lead[:-1], 1, width):
        _same(gate, x, what, "gate", gate.shape)
        strides = _row_strides(gate, what, "gate")
        return _lib.GATE["sequence"], _lib.pair(strides[0], 0)
    raise ValueError(f"{what}: gate has shape {tuple(gate.shape)}, expected {(width,)}, {(*lead[:-1], 1, width)} or {tuple(x.shape)}")


def _counter(seed, offset, what):
    seed, offset = int(seed), int(offset)
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError(f"{what}: seed and offset must lie in [0, 2^64)")
    return seed, offset


def rms_norm(x, weight, eps=1e-6, *, out=None):
    """y = x / sqrt(mean(x^2) + eps) * weight over the last dim; returns (y, rstd), rstd float32 per row
    for the backward pass.  `out=(y, rstd)`."""
    what = "rms_norm"
    _check_tensor(x, what)
    size = _width(x, what)
    if weight is None:
        raise TypeError(f"{what}: weight must be a tensor")
    _weight(weight, x, what, "weight")
    strides = _row_strides(x, what, "x")
    with _on(x.device):
        y, rstd = _outputs(what, x, out, [(x.shape, x.dtype), (x.shape[:-1], torch.float32)])
        if out is not None:
            _no_overlap(what, (y, rstd), (x, weight))
        _lib.check(_lib.lib().tpb200_rms_norm(x.data_ptr(), _TYPES[x.dtype], *size, strides, weight.data_ptr(), eps, y.data_ptr(), rstd.data_ptr(),
                                              _stream(x.device)))
    return y, rstd


def _rstd(t, x, what, name):
    _same_f32 = isinstance(t, torch.Tensor) and t.dtype == torch.float32 and tuple(t.shape) == tuple(x.shape[:-1]) and t.is_contiguous()
    if not _same_f32:
        raise ValueError(f"{what}: {name} must be the forward call's (contiguous float32 of shape {tuple(x.shape[:-1])})")
    if t.device != x.device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, expected {x.device}")
    return t


def rms_norm_backward(grad_y, x, weight, rstd, *, out=None):
    """Gradients of rms_norm: (grad_x, grad_weight), both in the tensors' type.  `out`: these two."""
    what = "rms_norm_backward"
    _check_tensor(x, what)
    size = _width(x, what)
    if weight is None:
        raise TypeError(f"{what}: weight must be a tensor")
    _weight(weight, x, what, "weight")
    _same(grad_y, x, what, "grad_y")
    _rstd(rstd, x, what, "rstd")
    gs, xs = _row_strides(grad_y, what, "grad_y"), _row_strides(x, what, "x")
    L = _lib.lib()
    with _on(x.device):
        gx, gw = _outputs(what, x, out, [(x.shape, x.dtype), (weight.shape, x.dtype)])
        if out is not None:
            _no_overlap(what, (gx, gw), (grad_y, x, weight, rstd))
        nbytes = L.tpb200_rms_norm_backward_workspace_bytes(*size)
        ws = _scratch(nbytes, x.device)
        _lib.check(L.tpb200_rms_norm_backward(grad_y.data_ptr(), gs, x.data_ptr(), xs, _TYPES[x.dtype], *size, weight.data_ptr(), rstd.data_ptr(),
                                              gx.data_ptr(), gw.data_ptr(), _ptr(ws), nbytes, _stream(x.device)))
    return gx, gw


def block_residual(x, h, post_weight=None, next_weight=None, gate=None, *, scale=1.0, eps=1e-6, p=0.0, seed=0, offset=0, out=None):
    """The residual path behind a block, in one pass over x (the residual stream) and h (the block's output):

        n = rms_norm(h) * post_weight                     (n = h without post_weight)
        x_out = x + scale * gate * dropout(n, p, seed, offset)
        y = rms_norm(x_out) * next_weight                 (None without next_weight)

    `gate`: [width], one row per sequence ([..., 1, width]), or x.shape.  y goes by x_out before it is rounded.
    seed and offset as in dropout (a captured graph drops the same elements on every replay).
    Returns (x_out, y, rstd_post, rstd_next); the last two (float32 per row, None where there is no norm)
    are for the backward pass.  `out`: these four."""
    what = "block_residual"
    _check_tensor(x, what)
    size = _width(x, what)
    _same(h, x, what, "h")
    _weight(post_weight, x, what, "post_weight")
    _weight(next_weight, x, what, "next_weight")
    _, gs = _gate(gate, x, what)
    seed, offset = _counter(seed, offset, what)
    xs, hs = _row_strides(x, what, "x"), _row_strides(h, what, "h")
    f32 = (x.shape[:-1], torch.float32)
    same = (x.shape, x.dtype)
    with _on(x.device):
        outs = _outputs(what, x, out, [same, same if next_weight is not None else None, f32 if post_weight is not None else None,
                                              f32 if next_weight is not None else None])
        if out is not None:
            _no_overlap(what, outs, (x, h, post_weight, next_weight, gate))
        _lib.check(_lib.lib().tpb200_block_residual(x.data_ptr(), xs, h.data_ptr(), hs, _ptr(gate), gs, _ptr(post_weight), _ptr(next_weight),
                                                    _TYPES[x.dtype], *size, scale, eps, p, seed, offset, _ptr(outs[0]), _ptr(outs[1]),
                                                    _ptr(outs[2]), _ptr(outs[3]), _stream(x.device)))
    return tuple(outs)


def block_residual_backward(grad_x_out, grad_y, h, x_out, rstd_post, rstd_next, post_weight=None, next_weight=None, gate=None, *, x=None,
                            scale=1.0, p=0.0, seed=0, offset=0, out=None):
    """Gradients of block_residual for the gradients of x_out (None: zero) and y (with next_weight), from the
    block's output h and the forward call's x_out, rstd_post and rstd_next; weights, gate, scale, p, seed and
    offset as in that call.  Returns (grad_x, grad_h, grad_post_weight, grad_next_weight, grad_gate), None
    where there is no such input.  `out`: these five.

    y was computed from x_out before it was rounded.  With `x`, the forward call's, that x_out is formed again
    (x_out is not read then and may be None); without it the gradients go by x_out as it was rounded, and
    grad_next_weight of a 16-bit type is off by two roundings rather than one."""
    what = "block_residual_backward"
    _check_tensor(h, what)
    size = _width(h, what)
    _weight(post_weight, h, what, "post_weight")
    _weight(next_weight, h, what, "next_weight")
    kind, gs = _gate(gate, h, what)
    seed, offset = _counter(seed, offset, what)
    hs = _row_strides(h, what, "h")
    gxs = gys = xs = at = None
    if grad_x_out is not None:
        gxs = _row_strides(_same(grad_x_out, h, what, "grad_x_out"), what, "grad_x_out")
    if next_weight is not None:
        gys = _row_strides(_same(grad_y, h, what, "grad_y"), what, "grad_y")
        if x is not None:
            at, xs = x, _row_strides(_same(x, h, what, "x"), what, "x")
        if x is None or (x_out is not None and h.dtype == torch.float32):     # not rounded: the same bits without forming them again
            at, xs, x = x_out, _row_strides(_same(x_out, h, what, "x_out"), what, "x_out"), None
        _rstd(rstd_next, h, what, "rstd_next")
    elif grad_y is not None:
        raise ValueError(f"{what}: grad_y without next_weight")
    if post_weight is not None:
        _rstd(rstd_post, h, what, "rstd_post")
    same, row = (h.shape, h.dtype), ((h.shape[-1],), h.dtype)
    L = _lib.lib()
    with _on(h.device):
        outs = _outputs(what, h, out, [same, same, row if post_weight is not None else None, row if next_weight is not None else None,
                                              (gate.shape, h.dtype) if gate is not None else None])
        if out is not None:
            _no_overlap(what, outs, (grad_x_out, grad_y, h, x_out, at, rstd_post, rstd_next, post_weight, next_weight, gate))
        nbytes = L.tpb200_block_residual_backward_workspace_bytes(*size, post_weight is not None, next_weight is not None, kind)
        ws = _scratch(nbytes, h.device)
        call = L.tpb200_block_residual_backward if x is None else L.tpb200_block_residual_backward_from_x
        _lib.check(call(
            _ptr(grad_x_out), gxs, _ptr(grad_y), gys, h.data_ptr(), hs, _ptr(at), xs, _ptr(gate), gs, kind,
            _ptr(post_weight), _ptr(next_weight), _ptr(rstd_post), _ptr(rstd_next), _TYPES[h.dtype], *size, scale, p, seed, offset,
            _ptr(outs[0]), _ptr(outs[1]), _ptr(outs[2]), _ptr(outs[3]), _ptr(outs[4]), _ptr(ws), nbytes, _stream(h.device)))
    return tuple(outs)


# ---------------------------------------------------------------------------- dropout

def _dropout(x, p, seed, offset, out, what):
    _check_tensor(x, what)
    seed, offset = _counter(seed, offset, what)
    if x.dim() == 0:
        outer, inner, width, strides = 1, 1, 1, _lib.pair(0, 0)
    else:
        outer, inner = _split(x.shape[:-1])
        width, strides = x.shape[-1], _row_strides(x, what, "x")
    with _on(x.device):
        y, = _outputs(what, x, out, [(x.shape, x.dtype)])
        if out is not None:
            _no_overlap(what, (y,), (x,))
        _lib.check(_lib.lib().tpb200_dropout(x.data_ptr(), _TYPES[x.dtype], outer, inner, width, strides, p, seed, offset, y.data_ptr(), _stream(x.device)))
    return y


def dropout(x, p, seed, offset=0, *, out=None):
    """x with every element dropped with probability p (in units of 2^-16, rounded) and the kept ones
    multiplied by 1 / (1 - p).  The choice is a function of the element's position in row-major order, of
    `seed` and of `offset` (both 0 .. 2^64 - 1) alone: no mask is stored, and the same call on the gradient
    is the backward pass.  Use another offset for every call of a step; a captured graph keeps the one it was
    captured with, and drops the same elements on every replay.  `out=(y,)`."""
    return _dropout(x, p, seed, offset, out, "dropout")


def dropout_backward(grad_y, p, seed, offset=0, *, out=None):
    """Gradient of dropout(x, p, seed, offset): the same elements dropped, the same factor."""
    return _dropout(grad_y, p, seed, offset, out, "dropout_backward")
