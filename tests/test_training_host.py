"""CPU tests of the training operators: refusals that need no GPU (through the C ABI and the Python
functions), workspace sizes, and the generator's definition against its published known answers."""
import ctypes

import pytest
import torch

import training_oracle as R


@pytest.fixture(scope="module")
def lib():
    from tensorplay_b200 import _lib, build
    build.build_library()
    return _lib.lib()


PTR = ctypes.c_void_p(4096)      # never followed: every call here is refused or has nothing to do


def test_no_cpu_fallback():
    import tensorplay_b200 as tpb
    x, lab, one = torch.ones(4, 8), torch.zeros(4, dtype=torch.int64), torch.ones(4)
    for call in (lambda: tpb.token_logprobs(x, lab), lambda: tpb.token_logprobs_backward(one, x, lab, one),
                 lambda: tpb.policy_loss(x, lab, one, one, one), lambda: tpb.preference_loss(x, lab, one, torch.tensor([0, 2, 4])),
                 lambda: tpb.rms_norm(x, torch.ones(8)), lambda: tpb.rms_norm_backward(x, x, torch.ones(8), one),
                 lambda: tpb.block_residual(x, x), lambda: tpb.block_residual_backward(x, None, x, x, None, None),
                 lambda: tpb.dropout(x, 0.5, 1), lambda: tpb.dropout_backward(x, 0.5, 1)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(TypeError):
        tpb.dropout([1.0], 0.5, 1)


def test_logits_refusals(lib):
    from tensorplay_b200 import _lib
    S = _lib.pair(0, 8)

    def score(dtype=0, outer=1, inner=4, vocab=8, x=PTR, strides=S, lab=PTR, ls=S, o=PTR):
        return lib.tpb200_token_logprobs(x, dtype, outer, inner, vocab, strides, lab, ls, o, o, None)

    assert score(dtype=7) == _lib.ERR_UNSUPPORTED and b"bfloat16" in lib.tpb200_last_error()
    assert score(inner=-1) == _lib.ERR_INVALID
    assert score(inner=1 << 31) == _lib.ERR_UNSUPPORTED
    assert score(outer=1 << 20, inner=1 << 20) == _lib.ERR_UNSUPPORTED
    assert score(vocab=0) == _lib.ERR_INVALID and b"vocabulary is empty" in lib.tpb200_last_error()
    assert score(x=None) == _lib.ERR_INVALID
    assert score(strides=None) == _lib.ERR_INVALID
    assert score(o=None) == _lib.ERR_INVALID
    assert score(inner=0, x=None, lab=None, o=None) == _lib.OK            # no rows: nothing to do
    assert lib.tpb200_token_logprobs_backward(None, S, PTR, 0, 1, 4, 8, S, PTR, S, PTR, PTR, None) == _lib.ERR_INVALID

    def policy(low=0.2, high=0.2, kl=0.0, ref=None, ws=PTR, nws=32, loss=PTR, w=PTR):
        return lib.tpb200_policy_loss(PTR, 1, 1, 4, 8, S, PTR, S, PTR, S, PTR, S, w, S, ref, S, low, high, kl, 1.0, loss, None, PTR, PTR, PTR,
                                      ws, nws, None)

    nan = float("nan")
    for bad in ({"low": -0.1}, {"low": 1.5}, {"low": nan}, {"high": -0.1}, {"high": nan}, {"kl": -1.0}, {"kl": nan}, {"kl": 0.1}, {"loss": None}, {"w": None}):
        assert policy(**bad) == _lib.ERR_INVALID, bad
    assert policy(ws=None) == _lib.ERR_WORKSPACE and policy(nws=31) == _lib.ERR_WORKSPACE
    assert lib.tpb200_policy_loss_workspace_bytes(1, 4) == 32 and lib.tpb200_policy_loss_workspace_bytes(0, 4) == 0

    def prefer(outer=1, inner=4, offsets=PTR, pairs=1, e=0.0, ws=PTR, nws=4096, rewards=PTR):
        return lib.tpb200_preference_loss(PTR, 2, outer, inner, 8, S, PTR, S, PTR, S, offsets, pairs, 0.1, e, 1.0, PTR, None, rewards, PTR, ws, nws, None)

    assert prefer(pairs=0) == _lib.ERR_INVALID
    assert prefer(e=0.5) == _lib.ERR_INVALID and prefer(e=-0.1) == _lib.ERR_INVALID
    assert prefer(outer=2) == _lib.ERR_INVALID                       # offsets go with packed rows
    assert prefer(outer=3, offsets=None) == _lib.ERR_INVALID          # two sequences per pair
    assert prefer(rewards=None) == _lib.ERR_INVALID
    need = lib.tpb200_preference_loss_workspace_bytes(1, 4, 1)
    assert need > 0 and prefer(ws=None) == _lib.ERR_WORKSPACE and prefer(nws=need - 1) == _lib.ERR_WORKSPACE


def test_block_and_dropout_refusals(lib):
    from tensorplay_b200 import _lib
    S = _lib.pair(0, 8)

    def block(dtype=0, width=8, x=PTR, h=PTR, post=PTR, nxt=PTR, eps=1e-6, p=0.0, y=PTR, r=PTR):
        return lib.tpb200_block_residual(x, S, h, S, None, None, post, nxt, dtype, 1, 4, width, 1.0, eps, p, 0, 0, PTR, y, r, r, None)

    assert block(dtype=3) == _lib.ERR_UNSUPPORTED
    assert block(width=16385) == _lib.ERR_UNSUPPORTED and b"16384" in lib.tpb200_last_error()
    for bad in ({"x": None}, {"h": None}, {"y": None}, {"r": None}, {"eps": -1.0}, {"eps": float("nan")}, {"p": 1.1}, {"p": -0.1}, {"p": float("nan")}):
        assert block(**bad) == _lib.ERR_INVALID, bad

    def back(kind=0, gate=None, gy=PTR, ws=PTR, nws=1 << 30, inner=4, gpost=PTR):
        return lib.tpb200_block_residual_backward(PTR, S, gy, S, PTR, S, PTR, S, gate, S, kind, PTR, PTR, PTR, PTR, 0, 1, inner, 8, 1.0, 0.0, 0, 0,
                                                  PTR, PTR, gpost, PTR, PTR if kind else None, ws, nws, None)

    assert back(kind=4) == _lib.ERR_INVALID and back(kind=-1) == _lib.ERR_INVALID
    assert back(kind=1) == _lib.ERR_INVALID                         # a kind without a gate
    assert back(gy=None) == _lib.ERR_INVALID and back(gpost=None) == _lib.ERR_INVALID
    need = lib.tpb200_block_residual_backward_workspace_bytes(1, 4, 8, 1, 1, 0)
    assert need > 0 and back(ws=None) == _lib.ERR_WORKSPACE and back(nws=need - 1) == _lib.ERR_WORKSPACE
    assert lib.tpb200_block_residual_backward_workspace_bytes(1, 4, 20000, 1, 1, 0) == 0
    # a gate per sequence or for all rows takes more, one for every row does not
    assert lib.tpb200_block_residual_backward_workspace_bytes(1, 4, 8, 1, 1, 3) == need
    assert lib.tpb200_block_residual_backward_workspace_bytes(1, 4, 8, 1, 1, 1) > need
    assert lib.tpb200_rms_norm_backward_workspace_bytes(1, 4, 8) == lib.tpb200_block_residual_backward_workspace_bytes(1, 4, 8, 0, 1, 0)
    assert lib.tpb200_rms_norm(PTR, 0, 1, 4, 8, S, None, 1e-6, PTR, PTR, None) == _lib.ERR_INVALID
    assert lib.tpb200_rms_norm(None, 0, 1, 0, 8, S, None, 1e-6, None, None, None) == _lib.OK
    for p in (-0.5, 1.5, float("nan")):
        assert lib.tpb200_dropout(PTR, 0, 1, 4, 8, S, p, 0, 0, PTR, None) == _lib.ERR_INVALID
    assert lib.tpb200_dropout(PTR, 5, 1, 4, 8, S, 0.5, 0, 0, PTR, None) == _lib.ERR_UNSUPPORTED
    assert lib.tpb200_dropout(None, 0, 1, 4, 8, S, 0.5, 0, 0, PTR, None) == _lib.ERR_INVALID
    assert lib.tpb200_dropout(None, 0, 1, 4, 0, S, 0.5, 0, 0, None, None) == _lib.OK


def test_strides_of_views():
    from tensorplay_b200 import training as T
    strides = lambda *a: tuple(T._strides(*a))  # noqa: E731
    x = torch.empty(4, 6, 10)
    assert strides(x, x.shape[:-1], "t", "x") == (60, 10)
    assert strides(x[:, 1:], x[:, 1:].shape[:-1], "t", "x") == (60, 10)
    assert strides(x[0], (6,), "t", "x") == (0, 10)
    assert strides(x[0, 0], (), "t", "x") == (0, 0)
    y = torch.empty(2, 4, 6, 10)
    assert strides(y, y.shape[:-1], "t", "x") == (60, 10)
    z = torch.empty(1).expand(2, 4, 6)
    assert strides(z, (2, 4, 6), "t", "x") == (0, 0)
    with pytest.raises(NotImplementedError, match="collapse"):
        strides(y.transpose(0, 1), (4, 2, 6), "t", "x")
    with pytest.raises(NotImplementedError, match="unit stride"):
        T._row_strides(x.transpose(1, 2), "t", "x")
    assert T._split((2, 3, 5)) == (6, 5) and T._split(()) == (1, 1) and T._split((7,)) == (1, 7)


def test_generator_known_answers():
    """Known answers of Philox 4x32-10 published with the generator: all-zero and all-one counter and key."""
    m = 0xFFFFFFFF
    for word, want in ((0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)), (m, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD))):
        c, k = [word] * 4, [word] * 2
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
            k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
        assert tuple(c) == want
    # the first block of key 0, offset 0 as halves: 0xE8D5 0x6627 0xC58D 0xE169 ...
    f = R.philox_factors(8, 0.5, 0, 0, "cpu")
    halves = [0xE8D5, 0x6627, 0xC58D, 0xE169, 0xAC4C, 0xBC57, 0xDBD8, 0x9B00]
    assert f.tolist() == [2.0 if h >= 32768 else 0.0 for h in halves]


def test_backward_from_x_refusals(lib):
    """The call that takes x in place of x_out checks what the other one does, and needs h to form x_out."""
    from tensorplay_b200 import _lib
    S = _lib.pair(0, 8)

    def back(h=PTR, x=PTR, ws=PTR, nws=1 << 30):
        return lib.tpb200_block_residual_backward_from_x(PTR, S, PTR, S, h, S, x, S, None, S, 0, PTR, PTR, PTR, PTR, 0, 1, 4, 8, 1.0, 0.0, 0, 0,
                                                         PTR, PTR, PTR, PTR, None, ws, nws, None)

    assert back(h=None) == _lib.ERR_INVALID and back(x=None) == _lib.ERR_INVALID
    assert back(ws=None) == _lib.ERR_WORKSPACE
