"""Language-model operators over the C ABI: the gated linear recurrence, the
embedding, and the log probabilities of given tokens.  Host code only checks
arguments, allocates tensors and calls the library.

All of them take float32, bfloat16 and float16 CUDA tensors, compute in
float32 and run on the current stream of the tensors' device.  float64 is
refused, as in ``HeadStartLSTM``.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_GATED, _LINEAR = 0, 1
_MAX_TOP = 32


def _code(who, t):
    c = _CODE.get(t.dtype)
    if c is None:
        raise TypeError(f"{who}: prlstm_b200 computes in float32; got dtype {t.dtype} "
                        "(use float32, bfloat16 or float16)")
    return c


def _same_device(who, first, *rest):
    if not first.is_cuda:
        raise RuntimeError("prlstm_b200 runs on CUDA devices (B200, sm_100a) only; "
                           f"{who} got a tensor on {first.device}")
    for t in rest:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{who}: tensors on {first.device} and {t.device}")


def _call(name, dev, *args):
    """The library call on the current stream of `dev`, made with that device
    current."""
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)
    return _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)


def _p(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ------------------------------------------------------------------ recurrence
def _rows(t):
    """`t` with its last axis contiguous (a copy only where it is not)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _strides(t, batch_first):
    """Element strides of a step and of a sequence."""
    s = t.stride()
    return (s[1], s[0]) if batch_first else (s[0], s[1])


def _recurrence_forward(form, z, x, h0, starts, batch_first, keep, h_n=None):
    """(h, h_n, checkpoints) of checked arguments; z and x have contiguous rows."""
    B, T = (z.shape[0], z.shape[1]) if batch_first else (z.shape[1], z.shape[0])
    H, dev = z.shape[2], z.device
    h = torch.empty(z.shape, dtype=z.dtype, device=dev)
    if h_n is None:
        h_n = torch.empty(B, H, device=dev)
    ckpt = None
    if keep:
        nbytes = _lib.load().hs_recurrence_checkpoint_bytes(T, B, H)
        ckpt = torch.empty(nbytes // 4, device=dev)
    zs, xs, hs = _strides(z, batch_first), _strides(x, batch_first), _strides(h, batch_first)
    ss = (0, 0) if starts is None else _strides(starts, batch_first)
    _call("hs_recurrence_forward", dev, _CODE[z.dtype], form, _p(z), *zs, _p(x), *xs, _p(h0), _p(starts), *ss,
          _p(h), *hs, _p(h_n), _p(ckpt), T, B, H, _p(_lib.status_word(dev)))
    return h, h_n, ckpt


class RecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, x, h0, starts, form, batch_first):
        h, h_n, ckpt = _recurrence_forward(form, z, x, None if h0 is None else h0.float().contiguous(), starts,
                                           batch_first, True)
        ctx.save_for_backward(z, x, starts, ckpt)
        ctx.h0_dtype = None if h0 is None else h0.dtype
        ctx.form, ctx.batch_first = form, batch_first
        ctx.set_materialize_grads(False)
        return h, h_n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dh_n):
        z, x, starts, ckpt = ctx.saved_tensors
        bf, dev = ctx.batch_first, z.device
        B, T = (z.shape[0], z.shape[1]) if bf else (z.shape[1], z.shape[0])
        H = z.shape[2]
        dh = None if dh is None else _rows(dh)
        dh_n = None if dh_n is None else dh_n.float().contiguous()
        dz, dx = torch.empty(z.shape, dtype=z.dtype, device=dev), torch.empty(x.shape, dtype=x.dtype, device=dev)
        dh0 = torch.empty(B, H, device=dev) if ctx.h0_dtype is not None and ctx.needs_input_grad[2] else None
        gs = (0, 0) if dh is None else _strides(dh, bf)
        ss = (0, 0) if starts is None else _strides(starts, bf)
        _call("hs_recurrence_backward", dev, _CODE[z.dtype], ctx.form, _p(z), *_strides(z, bf), _p(x),
              *_strides(x, bf), _p(ckpt), _p(starts), *ss, _p(dh), *gs, _p(dh_n), _p(dz), *_strides(dz, bf),
              _p(dx), *_strides(dx, bf), _p(dh0), T, B, H, _p(_lib.status_word(dev)))
        return dz, dx, None if dh0 is None else dh0.to(ctx.h0_dtype), None, None, None


def _recurrence(who, form, z, x, h0, starts, batch_first):
    _code(who, z)
    _same_device(who, z, x, h0, starts)
    if z.dim() != 3 or x.shape != z.shape:
        raise RuntimeError(f"{who}: both tensors must be [T, B, H] ([B, T, H] with batch_first); got "
                           f"{tuple(z.shape)} and {tuple(x.shape)}")
    if x.dtype != z.dtype:
        raise TypeError(f"{who}: tensors of {z.dtype} and {x.dtype}")
    B, T = (z.shape[0], z.shape[1]) if batch_first else (z.shape[1], z.shape[0])
    if h0 is not None:
        if h0.dim() == 3 and h0.shape[0] == 1:
            h0 = h0.squeeze(0)
        if h0.shape != (B, z.shape[2]):
            raise RuntimeError(f"{who}: h0 must be [{B}, {z.shape[2]}]; got {tuple(h0.shape)}")
        _code(who, h0)
    if starts is not None:
        if starts.shape != z.shape[:2] or starts.dtype not in (torch.bool, torch.uint8):
            raise RuntimeError(f"{who}: starts must be a bool tensor of shape {tuple(z.shape[:2])}; got "
                               f"{starts.dtype} {tuple(starts.shape)}")
    z, x = _rows(z), _rows(x)
    if _wants_grad(z, x, h0):
        return RecurrenceFn.apply(z, x, h0, starts, form, batch_first)
    h0 = None if h0 is None else h0.float().contiguous()
    h, h_n, _ = _recurrence_forward(form, z, x, h0, starts, batch_first, False)
    return h, h_n


def gated_recurrence(z, x, h0=None, starts=None, batch_first: bool = False):
    """``h_t = f_t h_{t-1} + (1 - f_t) x_t`` with ``f = sigmoid(z)``, along time.

    ``z``, ``x``: [T, B, H] ([B, T, H] with ``batch_first``), float32, bfloat16
    or float16; slices of wider tensors are taken as they are.  ``h0``: [B, H]
    or None for zeros.  ``starts``: bool [T, B] ([B, T]); a marked step begins a
    new sequence (the state before it is dropped), for documents packed into
    rows.  Returns ``(h, h_n)``: h in the input's dtype, the state ``h_n``
    [B, H] after the last step in float32.  Differentiable in z, x and h0."""
    return _recurrence("gated_recurrence", _GATED, z, x, h0, starts, batch_first)


def linear_recurrence(a, b, h0=None, starts=None, batch_first: bool = False):
    """``h_t = a_t h_{t-1} + b_t``: ``gated_recurrence`` with both coefficients
    given, of either sign.  Differentiable in a, b and h0."""
    return _recurrence("linear_recurrence", _LINEAR, a, b, h0, starts, batch_first)


def _step(who, form, z, x, h, out_state):
    _code(who, z)
    _same_device(who, z, x, h, out_state)
    if z.dim() != 2 or x.shape != z.shape or h.shape != z.shape:
        raise RuntimeError(f"{who}: z, x and h must be [B, H]; got {tuple(z.shape)}, {tuple(x.shape)} and "
                           f"{tuple(h.shape)}")
    if x.dtype != z.dtype:
        raise TypeError(f"{who}: tensors of {z.dtype} and {x.dtype}")
    if h.dtype != torch.float32:
        raise TypeError(f"{who}: the state is float32; got {h.dtype}")
    if out_state is not None and (out_state.dtype != torch.float32 or out_state.shape != h.shape
                                  or not out_state.is_contiguous()):
        raise RuntimeError(f"{who}: out_state must be a contiguous float32 [B, H] tensor")
    if _wants_grad(z, x, h):
        raise RuntimeError(f"{who} is not differentiable; use the recurrence over [1, B, H], or torch.no_grad()")
    out, state, _ = _recurrence_forward(form, _rows(z).unsqueeze(0), _rows(x).unsqueeze(0), h.contiguous(), None,
                                        False, False, out_state)
    return out[0], state


def gated_recurrence_step(z, x, h, out_state=None):
    """One token of ``gated_recurrence``: z, x [B, H] and the float32 state h
    [B, H] to ``(out, state)``.  ``out_state`` names where the new state goes;
    it may be ``h`` itself (the state advances in place)."""
    return _step("gated_recurrence_step", _GATED, z, x, h, out_state)


def linear_recurrence_step(a, b, h, out_state=None):
    """One token of ``linear_recurrence`` (see ``gated_recurrence_step``)."""
    return _step("linear_recurrence_step", _LINEAR, a, b, h, out_state)


# ------------------------------------------------------------------ tokens
def _tokens(who, tokens):
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{who}: tokens must be int64 or int32; got {tokens.dtype}")
    return tokens if tokens.is_contiguous() else tokens.contiguous()


def _embedding_forward(tokens, weight, scale):
    (V, D), dev = weight.shape, weight.device
    out = torch.empty(*tokens.shape, D, dtype=weight.dtype, device=dev)
    _call("hs_embedding_forward", dev, _CODE[weight.dtype], _p(weight), weight.stride(0),
          8 * tokens.element_size(), _p(tokens), scale, _p(out), tokens.numel(), V, D, _p(_lib.token_status_word(dev)))
    return out


class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, padding_idx):
        _lib.poll(weight.device)
        ctx.save_for_backward(tokens)
        ctx.table = (weight.shape, weight.dtype)
        ctx.scale, ctx.padding_idx = scale, padding_idx
        return _embedding_forward(tokens, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (tokens,) = ctx.saved_tensors
        (V, D), dtype = ctx.table
        dev, N = dout.device, tokens.numel()
        dout = dout.contiguous()
        dweight = torch.empty(V, D, dtype=dtype, device=dev)
        ws = _lib.workspace(_lib.load().hs_embedding_workspace_bytes(N, V, D), dev)
        _call("hs_embedding_backward", dev, _CODE[dtype], _p(dout), 8 * tokens.element_size(), _p(tokens),
              ctx.padding_idx, ctx.scale, _p(dweight), N, V, D, _p(ws), ws.numel(), _p(_lib.token_status_word(dev)))
        _lib.note_launch(dev)
        return dweight, None, None, None


def embedding(tokens, weight, scale: float = 1.0, padding_idx: Optional[int] = None):
    """``scale * weight[tokens]``: tokens of any shape (int64 or int32), weight
    [V, D]; the result is ``tokens.shape + (D,)`` in the weight's dtype.

    The gradient of ``weight`` sums each token's rows in float32, in the order
    of the tokens, and is the same bit for bit from run to run; the row
    ``padding_idx`` gets none.  An id outside [0, V) gives a row of zeros and is
    reported by ``check_device_status()`` (and by a later training call)."""
    who = "embedding"
    _code(who, weight)
    _same_device(who, weight, tokens)
    if weight.dim() != 2:
        raise RuntimeError(f"{who}: weight must be [V, D]; got {tuple(weight.shape)}")
    tokens = _tokens(who, tokens)
    weight = _rows(weight)
    if weight.stride(0) < weight.shape[1]:
        weight = weight.contiguous()
    pad = -1
    if padding_idx is not None:
        pad = int(padding_idx) + (weight.shape[0] if padding_idx < 0 else 0)
        if not 0 <= pad < weight.shape[0]:
            raise RuntimeError(f"{who}: padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
    if _wants_grad(weight):
        return EmbeddingFn.apply(weight, tokens, float(scale), pad)
    return _embedding_forward(tokens, weight, float(scale))


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``, float32 (``top_index`` int64)."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def _logprobs_forward(logits, tokens, top, temperature, ignore_index, keep):
    N, V = logits.shape
    dev = logits.device
    both = torch.empty(2, N, device=dev)
    logprob, entropy = both[0], both[1]
    top_lp = torch.empty(N, top, device=dev) if top else None
    top_id = torch.empty(N, top, dtype=torch.int64, device=dev) if top else None
    stats = torch.empty(N, 2, device=dev) if keep else None
    _call("hs_token_logprobs_forward", dev, _CODE[logits.dtype], _p(logits), logits.stride(0),
          8 * tokens.element_size(), _p(tokens), ignore_index, temperature, top, _p(logprob), _p(entropy), _p(top_lp),
          _p(top_id), _p(stats), N, V, _p(_lib.token_status_word(dev)))
    return logprob, entropy, top_lp, top_id, stats


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature, ignore_index):
        _lib.poll(logits.device)
        logprob, entropy, top_lp, top_id, stats = _logprobs_forward(logits, tokens, top, temperature, ignore_index, True)
        ctx.save_for_backward(logits, tokens, entropy, top_id, stats)
        ctx.args = (top, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_id)
        return logprob, entropy, top_lp, top_id

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogprob, dentropy, dtop, _dindex):
        logits, tokens, entropy, top_id, stats = ctx.saved_tensors
        top, temperature, ignore_index = ctx.args
        N, V = logits.shape
        dev = logits.device
        dlogprob, dentropy, dtop = (None if t is None else t.float().contiguous() for t in (dlogprob, dentropy, dtop))
        dlogits = torch.empty(N, V, dtype=logits.dtype, device=dev)
        _call("hs_token_logprobs_backward", dev, _CODE[logits.dtype], _p(logits), logits.stride(0),
              8 * tokens.element_size(), _p(tokens), ignore_index, temperature, top, _p(stats), _p(entropy), _p(top_id),
              _p(dlogprob), _p(dentropy), _p(dtop), _p(dlogits), V, N, V)
        _lib.note_launch(dev)
        return dlogits, None, None, None, None


def token_logprobs(logits, tokens, top: int = 0, temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities (in nats) of ``tokens`` [...] under
    ``softmax(logits / temperature)``, logits [..., V], with the entropy of
    each distribution and its ``top`` (up to 32) most likely tokens.

    Differentiable in logits through ``logprob``, ``entropy`` and
    ``top_logprob``; ``-r.logprob.mean()`` is the cross-entropy loss.
    Alternatives are ordered by logit, equal logits by the lower index.  Rows
    whose token is ``ignore_index`` are not read and give 0 (``top_index`` -1)
    and no gradient.  Logits of -inf are masked out; a row with nothing left
    gives -inf, entropy 0 and no gradient; a row with a NaN or +inf gives NaN
    (``top_index`` -1).  A token outside [0, V) gives NaN and is reported by
    ``check_device_status()``."""
    who = "token_logprobs"
    _code(who, logits)
    _same_device(who, logits, tokens)
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise RuntimeError(f"{who}: logits [..., V] and tokens [...] do not match: {tuple(logits.shape)} and "
                           f"{tuple(tokens.shape)}")
    V = logits.shape[-1]
    if not 0 <= top <= min(_MAX_TOP, V):
        raise RuntimeError(f"{who}: top must be in 0..{min(_MAX_TOP, V)}; got {top}")
    if not 1e-30 <= temperature <= 1e30:
        raise RuntimeError(f"{who}: the temperature must be positive (1e-30 to 1e30); got {temperature}")
    shape = tokens.shape
    tokens = _tokens(who, tokens).view(-1)
    rows = logits if logits.dim() == 2 else logits.reshape(-1, V) if V else logits.reshape(tokens.numel(), 0)
    rows = _rows(rows)
    if rows.shape[0] > 1 and rows.stride(0) < V:
        rows = rows.contiguous()
    if _wants_grad(rows):
        lp, ent, top_lp, top_id = TokenLogprobsFn.apply(rows, tokens, int(top), float(temperature), int(ignore_index))
    else:
        lp, ent, top_lp, top_id, _ = _logprobs_forward(rows, tokens, int(top), float(temperature), int(ignore_index), False)
    if len(shape) != 1:
        lp, ent = lp.view(shape), ent.view(shape)
        if top:
            top_lp, top_id = top_lp.view(*shape, top), top_id.view(*shape, top)
    return TokenLogprobs(lp, ent, top_lp, top_id)
