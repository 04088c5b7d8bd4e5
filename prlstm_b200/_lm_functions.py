"""Language-model operators over the C ABI: the gated linear recurrence, the
embedding, and the log probabilities of given tokens.  Host code only checks
arguments, allocates tensors and calls the library.

All of them take float32, bfloat16 and float16 CUDA tensors, compute in
float32 and run on the current stream of the tensors' device.  float64 is
refused, as in ``HeadStartLSTM``.  Gradients are reverse-mode and of first
order; forward-mode tangents and functorch transforms are refused.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_GATED, _LINEAR = 0, 1
_MAX_TOP = 32
_RUN = 16  # steps between the recurrence's saved states

_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream() without the Python object (2 us a call)
_current_device = torch._C._cuda_getDevice


def _dtype_code(who, t):
    code = _CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{who}: prlstm_b200 computes in float32; got dtype {t.dtype} "
                        "(use float32, bfloat16 or float16)")
    return code


def _device_index(who, first, *rest):
    """The index of the CUDA device that all tensors are on.  Tensors that carry a
    forward-mode tangent are refused here: the results would have lost it."""
    if forward_ad._current_level >= 0:
        for t in (first, *rest):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{who} has no forward-mode derivative (its gradients are reverse-mode)")
    index = first.get_device()
    if index < 0:
        raise RuntimeError("prlstm_b200 runs on CUDA devices (B200, sm_100a) only; "
                           f"{who} got a tensor on {first.device}")
    for t in rest:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"{who}: tensors on {first.device} and {t.device}")
    return index


def _call(name, index, *args):
    """The library call on the current stream of device `index`, with that
    device current."""
    if index != _current_device():
        with torch.cuda.device(index):
            rc = _lib.function(name)(*args, _raw_stream(index))
    else:
        rc = _lib.function(name)(*args, _raw_stream(index))
    if rc:
        _lib.raise_error(name, rc)


def _p(t):
    return None if t is None else t.data_ptr()


def _float32(shape, like):
    """A float32 tensor on the device of `like`, whatever torch's default dtype is."""
    return torch.empty(shape, dtype=torch.float32, device=like.device)


def _once(backward):
    """A backward that may be differentiated no further: ``once_differentiable``
    where a graph of it is asked for, itself (4 us less a call) where not."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def _apply(fn):
    """``fn.apply``; the wrapper that torch puts around it is for functorch transforms
    (which refuse these functions) and left out where none is active, 5 us a call."""
    plain = super(torch.autograd.Function, fn).apply
    transforms = torch._C._are_functorch_transforms_active

    def apply(*args):
        return fn.apply(*args) if transforms() else plain(*args)

    return apply


# ------------------------------------------------------------------ recurrence
def _rows(t):
    """`t` with its last axis contiguous (a copy only where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _like(t):
    """An output laid out like `t`, its last axis contiguous.  (torch lays out the
    like of overlapping rows, windows say, by their strides, the last axis not
    always innermost.)"""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 or out.shape[-1] <= 1 else torch.empty_like(t, memory_format=torch.contiguous_format)


def _tensor(t, batch_first):
    """Address and element strides of a step and of a sequence, as the library
    takes a [T, B, ..] tensor (or none)."""
    if t is None:
        return None, 0, 0
    a, b = t.stride()[:2]
    return (t.data_ptr(), b, a) if batch_first else (t.data_ptr(), a, b)


def _extents(z, batch_first):
    """T, B, H."""
    a, b, H = z.shape
    return (b, a, H) if batch_first else (a, b, H)


def _recurrence_forward(code, index, form, z, x, h0, starts, batch_first, keep):
    """(h, h_n, checkpoints) of checked arguments; z and x have contiguous rows."""
    T, B, H = _extents(z, batch_first)
    h = _like(z)
    h_n = _float32((B, H), z) if h0 is None else torch.empty_like(h0)
    ckpt = _float32(-(-T // _RUN) * B * (H + 1), z) if keep else None  # states, masks of starts
    _call("hs_recurrence_forward", index, code, form, *_tensor(z, batch_first), *_tensor(x, batch_first), _p(h0),
          *_tensor(starts, batch_first), *_tensor(h, batch_first), h_n.data_ptr(), _p(ckpt), T, B, H,
          _lib.host_status(index).timeout_ptr)
    return h, h_n, ckpt


class RecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, x, h0, starts, code, index, form, batch_first):
        h, h_n, ckpt = _recurrence_forward(code, index, form, z, x, None if h0 is None else _state(h0), starts, batch_first,
                                           True)
        ctx.save_for_backward(z, x, ckpt)
        ctx.args = (code, index, form, batch_first, starts is not None, None if h0 is None else h0.dtype)
        ctx.set_materialize_grads(False)
        return h, h_n

    @staticmethod
    @_once
    def backward(ctx, dh, dh_n):
        z, x, ckpt = ctx.saved_tensors
        code, index, form, bf, with_starts, h0_dtype = ctx.args
        T, B, H = _extents(z, bf)
        dh = None if dh is None else _rows(dh)
        dh_n = None if dh_n is None else _state(dh_n)
        dz, dx = _like(z), _like(x)
        dh0 = _float32((B, H), z) if h0_dtype is not None and ctx.needs_input_grad[2] else None
        _call("hs_recurrence_backward", index, code, form, *_tensor(z, bf), *_tensor(x, bf), ckpt.data_ptr(),
              with_starts, *_tensor(dh, bf), _p(dh_n), *_tensor(dz, bf), *_tensor(dx, bf), _p(dh0), T, B, H,
              _lib.host_status(index).timeout_ptr)
        if dh0 is not None and h0_dtype is not torch.float32:
            dh0 = dh0.to(h0_dtype)
        return dz, dx, dh0, None, None, None, None, None


_recurrence_apply = _apply(RecurrenceFn)


def _state(t):
    """A [B, H] state as the library takes it."""
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.float().contiguous()


def _recurrence(who, form, z, x, h0, starts, batch_first):
    code, index = _dtype_code(who, z), _device_index(who, z, x, h0, starts)
    shape = z.shape
    if len(shape) != 3 or x.shape != shape:
        raise RuntimeError(f"{who}: both tensors must be [T, B, H] ([B, T, H] with batch_first); got "
                           f"{tuple(shape)} and {tuple(x.shape)}")
    if x.dtype is not z.dtype:
        raise TypeError(f"{who}: tensors of {z.dtype} and {x.dtype}")
    if h0 is not None:
        if h0.dim() == 3 and h0.shape[0] == 1:
            h0 = h0.squeeze(0)
        if h0.shape != (shape[0 if batch_first else 1], shape[2]):
            raise RuntimeError(f"{who}: h0 must be [{shape[0 if batch_first else 1]}, {shape[2]}]; got {tuple(h0.shape)}")
        _dtype_code(who, h0)
    if starts is not None and (starts.shape != shape[:2] or starts.dtype not in (torch.bool, torch.uint8)):
        raise RuntimeError(f"{who}: starts must be a bool tensor of shape {tuple(shape[:2])}; got "
                           f"{starts.dtype} {tuple(starts.shape)}")
    _lib.host_status(index).check()
    z, x = _rows(z), _rows(x)
    if torch.is_grad_enabled() and (z.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        return _recurrence_apply(z, x, h0, starts, code, index, form, batch_first)
    return _recurrence_forward(code, index, form, z, x, None if h0 is None else _state(h0), starts, batch_first, False)[:2]


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
    given, of either sign and any size (a state beyond float32's range is an infinity
    from that step on).  Differentiable in a, b and h0."""
    return _recurrence("linear_recurrence", _LINEAR, a, b, h0, starts, batch_first)


def _step(who, form, z, x, h, out_state):
    code, index = _dtype_code(who, z), _device_index(who, z, x, h, out_state)
    shape = z.shape
    if len(shape) != 2 or x.shape != shape or h.shape != shape:
        raise RuntimeError(f"{who}: z, x and h must be [B, H]; got {tuple(shape)}, {tuple(x.shape)} and {tuple(h.shape)}")
    if x.dtype is not z.dtype:
        raise TypeError(f"{who}: tensors of {z.dtype} and {x.dtype}")
    if h.dtype is not torch.float32:
        raise TypeError(f"{who}: the state is float32; got {h.dtype}")
    if (z.requires_grad or x.requires_grad or h.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError(f"{who} is not differentiable; use the recurrence over [1, B, H], or torch.no_grad()")
    z, x, h = _rows(z), _rows(x), h if h.is_contiguous() else h.contiguous()
    if out_state is None:
        out_state = torch.empty_like(h)
    elif out_state.dtype is not torch.float32 or out_state.shape != shape or not out_state.is_contiguous():
        raise RuntimeError(f"{who}: out_state must be a contiguous float32 [B, H] tensor")
    out = _like(z)
    B, H = shape
    status = _lib.host_status(index)
    status.check()
    _call("hs_recurrence_forward", index, code, form, z.data_ptr(), 0, z.stride(0), x.data_ptr(), 0, x.stride(0),
          h.data_ptr(), None, 0, 0, out.data_ptr(), 0, out.stride(0), out_state.data_ptr(), None, 1, B, H, status.timeout_ptr)
    return out, out_state


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
    """(contiguous tokens, their bits)."""
    bits = 64 if tokens.dtype is torch.int64 else 32 if tokens.dtype is torch.int32 else 0
    if not bits:
        raise TypeError(f"{who}: tokens must be int64 or int32; got {tokens.dtype}")
    return tokens if tokens.is_contiguous() else tokens.contiguous(), bits


def _embedding_forward(code, index, tokens, bits, weight, scale):
    V, D = weight.shape
    out = torch.empty((*tokens.shape, D), dtype=weight.dtype, device=weight.device)
    _call("hs_embedding_forward", index, code, weight.data_ptr(), weight.stride(0), bits, tokens.data_ptr(), scale,
          out.data_ptr(), tokens.numel(), V, D, _lib.host_status(index).token_ptr)
    return out


@lru_cache(maxsize=64)
def _embedding_workspace_bytes(N, V, D):
    return _lib.function("hs_embedding_workspace_bytes")(N, V, D)


class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, code, index, bits, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.args = (weight.shape, code, index, bits, scale, padding_idx)
        return _embedding_forward(code, index, tokens, bits, weight, scale)

    @staticmethod
    @_once
    def backward(ctx, dout):
        (tokens,) = ctx.saved_tensors
        shape, code, index, bits, scale, padding_idx = ctx.args
        V, D = shape
        N = tokens.numel()
        dout = dout if dout.is_contiguous() else dout.contiguous()
        dweight = dout.new_empty(shape)
        nbytes = _embedding_workspace_bytes(N, V, D)
        ws = dout.new_empty(nbytes // dout.element_size())  # (a multiple of 256 bytes)
        _call("hs_embedding_backward", index, code, dout.data_ptr(), bits, tokens.data_ptr(), padding_idx, scale,
              dweight.data_ptr(), N, V, D, ws.data_ptr(), nbytes, _lib.host_status(index).token_ptr)
        return dweight, None, None, None, None, None, None


_embedding_apply = _apply(EmbeddingFn)


def embedding(tokens, weight, scale: float = 1.0, padding_idx: Optional[int] = None):
    """``scale * weight[tokens]``: tokens of any shape (int64 or int32), weight
    [V, D]; the result is ``tokens.shape + (D,)`` in the weight's dtype.

    The gradient of ``weight`` sums each token's rows in float32, in the order
    of the tokens, and is the same bit for bit from run to run; the row
    ``padding_idx`` gets none.  An id outside [0, V) gives a row of zeros and is
    reported by ``check_device_status()`` and by later calls, until
    ``clear_device_status()``."""
    who = "embedding"
    code, index = _dtype_code(who, weight), _device_index(who, weight, tokens)
    if weight.dim() != 2:
        raise RuntimeError(f"{who}: weight must be [V, D]; got {tuple(weight.shape)}")
    tokens, bits = _tokens(who, tokens)
    V, D = weight.shape
    if weight.stride(0) < D or (D > 1 and weight.stride(1) != 1):
        weight = weight.contiguous()
    pad = -1
    if padding_idx is not None:
        pad = int(padding_idx) + (V if padding_idx < 0 else 0)
        if not 0 <= pad < V:
            raise RuntimeError(f"{who}: padding_idx {padding_idx} is outside the table of {V} rows")
    _lib.host_status(index).check()
    if weight.requires_grad and torch.is_grad_enabled():
        return _embedding_apply(weight, tokens, code, index, bits, float(scale), pad)
    return _embedding_forward(code, index, tokens, bits, weight, float(scale))


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``, float32 (``top_index`` int64)."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def _logprobs_forward(code, index, logits, tokens, bits, top, temperature, ignore_index, keep):
    N, V = logits.shape
    logprob = _float32(N, logits)
    entropy = torch.empty_like(logprob)
    top_lp = _float32((N, top), logits) if top else None
    top_id = torch.empty((N, top), dtype=torch.int64, device=logits.device) if top else None
    stats = _float32((N, 2), logits) if keep else None
    _call("hs_token_logprobs_forward", index, code, logits.data_ptr(), logits.stride(0), bits, tokens.data_ptr(),
          ignore_index, temperature, top, logprob.data_ptr(), entropy.data_ptr(), _p(top_lp), _p(top_id), _p(stats), N, V,
          _lib.host_status(index).token_ptr)
    return logprob, entropy, top_lp, top_id, stats


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, code, index, bits, top, temperature, ignore_index):
        logprob, entropy, top_lp, top_id, stats = _logprobs_forward(code, index, logits, tokens, bits, top, temperature,
                                                                    ignore_index, True)
        ctx.save_for_backward(logits, tokens, entropy, top_id, stats)
        ctx.args = (code, index, bits, top, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_id)
        return logprob, entropy, top_lp, top_id

    @staticmethod
    @_once
    def backward(ctx, dlogprob, dentropy, dtop, _dindex):
        logits, tokens, entropy, top_id, stats = ctx.saved_tensors
        code, index, bits, top, temperature, ignore_index = ctx.args
        N, V = logits.shape
        dlogprob, dentropy, dtop = (None if t is None else _state(t) for t in (dlogprob, dentropy, dtop))
        dlogits = torch.empty((N, V), dtype=logits.dtype, device=logits.device)
        _call("hs_token_logprobs_backward", index, code, logits.data_ptr(), logits.stride(0), bits, tokens.data_ptr(),
              ignore_index, temperature, top, stats.data_ptr(), entropy.data_ptr(), _p(top_id), _p(dlogprob), _p(dentropy),
              _p(dtop), dlogits.data_ptr(), V, N, V)
        return dlogits, None, None, None, None, None, None, None


_token_logprobs_apply = _apply(TokenLogprobsFn)


def token_logprobs(logits, tokens, top: int = 0, temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities (in nats) of ``tokens`` [...] under
    ``softmax(logits / temperature)``, logits [..., V], with the entropy of
    each distribution and its ``top`` (up to 32) most likely tokens.

    Differentiable in logits through ``logprob``, ``entropy`` and
    ``top_logprob``; ``-r.logprob.mean()`` is the cross-entropy loss.
    Alternatives are ordered by logit, equal logits by the lower index.  Rows
    whose token is ``ignore_index`` give 0 (``top_index`` -1) and no gradient,
    whatever their logits.  Logits of -inf are masked out; a row with nothing left
    gives -inf, entropy 0 and no gradient; a row with a NaN or +inf gives NaN
    (``top_index`` -1).  A token outside [0, V) gives NaN and is reported by
    ``check_device_status()`` and by later calls, until
    ``clear_device_status()``."""
    who = "token_logprobs"
    code, index = _dtype_code(who, logits), _device_index(who, logits, tokens)
    shape = tokens.shape
    if logits.dim() < 1 or logits.shape[:-1] != shape:
        raise RuntimeError(f"{who}: logits [..., V] and tokens [...] do not match: {tuple(logits.shape)} and {tuple(shape)}")
    V, top, temperature, ignore_index = logits.shape[-1], int(top), float(temperature), int(ignore_index)
    if not 0 <= top <= _MAX_TOP or top > V:
        raise RuntimeError(f"{who}: top must be in 0..{min(_MAX_TOP, V)}; got {top}")
    if not 1e-30 <= temperature <= 1e30:
        raise RuntimeError(f"{who}: the temperature must be positive (1e-30 to 1e30); got {temperature}")
    tokens, bits = _tokens(who, tokens)
    if len(shape) != 1:
        tokens, logits = tokens.view(-1), logits.reshape(tokens.numel(), V)
    rows = _rows(logits)
    if rows.shape[0] > 1 and rows.stride(0) < V:
        rows = rows.contiguous()
    _lib.host_status(index).check()
    if rows.requires_grad and torch.is_grad_enabled():
        lp, ent, top_lp, top_id = _token_logprobs_apply(rows, tokens, code, index, bits, top, temperature, ignore_index)
    else:
        lp, ent, top_lp, top_id, _ = _logprobs_forward(code, index, rows, tokens, bits, top, temperature, ignore_index, False)
    if len(shape) != 1:
        lp, ent = lp.view(shape), ent.view(shape)
        if top:
            top_lp, top_id = top_lp.view(*shape, top), top_id.view(*shape, top)
    return TokenLogprobs(lp, ent, top_lp, top_id)
