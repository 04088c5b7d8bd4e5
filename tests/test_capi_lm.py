"""The language-model entry points' host side: argument checks that refuse a
call before any launch, empty extents, and the size queries.  No kernel runs
here (CPU only)."""

import ctypes

import pytest

INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 3
P = ctypes.c_void_p(256)  # a well-aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    import os

    from prlstm_b200 import _lib

    if not os.path.exists(_lib.LIB_PATH):
        from prlstm_b200 import build

        build.build()
    return _lib.load()


def rec_forward(lib, dtype=0, form=0, z=P, x=P, h=P, T=4, B=2, H=8, status=P):
    return lib.hs_recurrence_forward(dtype, form, z, 16, 8, x, 16, 8, None, None, 0, 0, h, 16, 8, None, None, T, B, H, status, None)


def rec_backward(lib, dtype=0, z=P, ckpt=P, dz=P, T=4, B=2, H=8, status=P):
    return lib.hs_recurrence_backward(dtype, 0, z, 16, 8, P, 16, 8, ckpt, 0, None, 0, 0, None, dz, 16, 8, P, 16, 8,
                                      None, T, B, H, status, None)


def emb_forward(lib, dtype=0, w=P, ld=8, bits=64, tok=P, out=P, N=4, V=10, D=8, status=P):
    return lib.hs_embedding_forward(dtype, w, ld, bits, tok, 1.0, out, N, V, D, status, None)


def emb_backward(lib, dtype=0, dout=P, bits=64, tok=P, dw=P, N=4, V=10, D=8, ws=P, nbytes=1 << 20, status=P):
    return lib.hs_embedding_backward(dtype, dout, bits, tok, -1, 1.0, dw, N, V, D, ws, nbytes, status, None)


def lp_forward(lib, dtype=0, x=P, ld=8, bits=64, tok=P, T=1.0, top=0, lp=P, top_lp=P, top_id=P, N=4, V=8, status=P):
    return lib.hs_token_logprobs_forward(dtype, x, ld, bits, tok, -100, T, top, lp, None, top_lp, top_id, None, N, V, status, None)


def lp_backward(lib, x=P, stats=P, ent=P, ids=P, ge=None, gt=None, dx=P, dld=8, top=0, N=4, V=8):
    return lib.hs_token_logprobs_backward(0, x, 8, 64, P, -100, 1.0, top, stats, ent, ids, None, ge, gt, dx, dld, N, V, None)


@pytest.mark.parametrize("call,bad", [
    (rec_forward, dict(dtype=3)), (rec_forward, dict(form=2)), (rec_forward, dict(T=-1)), (rec_forward, dict(z=None)),
    (rec_forward, dict(h=None)), (rec_forward, dict(status=None)), (rec_forward, dict(z=ctypes.c_void_p(258))),
    (rec_backward, dict(dtype=-1)), (rec_backward, dict(ckpt=None)), (rec_backward, dict(dz=None)),
    (rec_backward, dict(H=-2)), (rec_backward, dict(status=None)),
    (emb_forward, dict(bits=16)), (emb_forward, dict(w=None)), (emb_forward, dict(tok=None)), (emb_forward, dict(N=-1)),
    (emb_forward, dict(ld=7)), (emb_forward, dict(status=None)), (emb_forward, dict(tok=ctypes.c_void_p(260))),
    (emb_backward, dict(dtype=9)), (emb_backward, dict(dout=None)), (emb_backward, dict(dw=None)),
    (lp_forward, dict(top=33, V=64, ld=64)), (lp_forward, dict(top=9)), (lp_forward, dict(top=-1)), (lp_forward, dict(T=0.0)),
    (lp_forward, dict(T=float("nan"))), (lp_forward, dict(T=1e31)), (lp_forward, dict(V=0)), (lp_forward, dict(ld=7)),
    (lp_forward, dict(x=None)), (lp_forward, dict(lp=None)), (lp_forward, dict(top=2, top_id=None)), (lp_forward, dict(status=None)),
    (lp_forward, dict(x=ctypes.c_void_p(257))), (lp_forward, dict(bits=8)),
    (lp_backward, dict(stats=None)), (lp_backward, dict(dx=None)), (lp_backward, dict(dld=7)), (lp_backward, dict(ge=P, ent=None)),
    (lp_backward, dict(gt=P, top=2, ids=None)),
], ids=lambda v: v.__name__ if callable(v) else ",".join(v))
def test_refused_before_any_launch(lib, call, bad):
    assert call(lib, **bad) == INVALID
    assert lib.hs_last_error_message()


@pytest.mark.parametrize("call,bad", [
    (rec_forward, dict(T=(1 << 30) + 1)), (rec_forward, dict(B=1 << 20, H=1 << 20)), (emb_forward, dict(N=1 << 31)),
    (emb_backward, dict(V=1 << 31)), (lp_forward, dict(V=(1 << 30) + 1, ld=1 << 31)), (lp_forward, dict(N=(1 << 27) + 1))],
    ids=lambda v: v.__name__ if callable(v) else ",".join(v))
def test_too_large_is_unsupported(lib, call, bad):
    assert call(lib, **bad) == UNSUPPORTED


def test_workspace_is_checked(lib):
    need = lib.hs_embedding_workspace_bytes(4, 10, 8)
    assert need > 0
    assert emb_backward(lib, nbytes=need - 1) == WORKSPACE
    assert emb_backward(lib, ws=None) == WORKSPACE
    assert emb_backward(lib, ws=ctypes.c_void_p(128)) == WORKSPACE


def test_empty_extents_do_nothing(lib):
    assert rec_forward(lib, B=0) == rec_forward(lib, H=0) == rec_forward(lib, T=0, z=None) == 0
    assert rec_backward(lib, B=0) == rec_backward(lib, H=0) == rec_backward(lib, T=0, z=None) == 0
    assert emb_forward(lib, N=0, tok=None) == emb_forward(lib, D=0) == 0
    assert emb_backward(lib, V=0) == emb_backward(lib, D=0) == 0
    assert lp_forward(lib, N=0) == lp_backward(lib, N=0) == 0


def test_size_queries(lib):
    # a float32 state and a word of starts for each sequence and run of 16 steps
    assert lib.hs_recurrence_checkpoint_bytes(1, 2, 3) == 4 * 2 * (3 + 1)
    assert lib.hs_recurrence_checkpoint_bytes(16, 2, 3) == 4 * 2 * (3 + 1)
    assert lib.hs_recurrence_checkpoint_bytes(17, 2, 3) == 2 * 4 * 2 * (3 + 1)
    assert lib.hs_recurrence_checkpoint_bytes(0, 2, 3) == 0
    sizes = [lib.hs_embedding_workspace_bytes(n, 1000, 64) for n in (1, 1000, 16384, 16385, 100000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.hs_embedding_workspace_bytes(0, 10, 8) == 0
    assert lib.hs_status_string(6) == b"token id out of range"


def test_cpu_tensors_are_refused():
    import torch

    import prlstm_b200 as pk

    z = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        pk.gated_recurrence(z, z)
    with pytest.raises(RuntimeError, match="CUDA"):
        pk.embedding(torch.zeros(2, dtype=torch.int64), z[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        pk.token_logprobs(z[0], torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        pk.linear_recurrence(z.double(), z.double())
