"""Cross attention: queries of one length, keys and values of another.

``cross_attention_b200`` is differentiable; ``cross_attention_forward_b200`` and
``cross_attention_backward_b200`` are its two directions as calls of their own, for callers that keep
the state between them themselves (a captured training step, a framework without autograd).
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib
from .functional import (_dtype_code, _mask_bytes, _on_device, _require_cuda, _require_no_tangent, _status, _status_words,
                         _stream_handle)

__all__ = ["cross_attention_b200", "cross_attention_forward_b200", "cross_attention_backward_b200", "AttentionState"]


class AttentionState(NamedTuple):
    """What the backward pass needs of the forward pass beside its result: ``rows`` ``[B, H, Lq, 2]`` (each
    row's maximum and the base-2 logarithm of its sum) and, for bf16, ``rounding`` ``[B, Lq, H, D]`` (what
    rounding took off the result, so that the scores' gradients do not lose it)."""
    rows: torch.Tensor
    rounding: torch.Tensor | None


def _laid_out(t: torch.Tensor, tensor_cores: bool) -> torch.Tensor:
    """``t`` outside autograd, with a contiguous last axis; for the tensor-core kernels also with every row on a
    16-byte boundary and no axis repeated in place (a copy where it is not)."""
    if t.requires_grad:
        t = t.detach()
    if t.is_contiguous():
        return t if not tensor_cores or t.data_ptr() % 16 == 0 else t.clone()
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return t.contiguous()
    if any(s < 0 for s in t.stride()):
        return t.contiguous()
    if tensor_cores and (t.data_ptr() % 16 or any(n > 1 and (s % 8 or s == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))):
        return t.clone(memory_format=torch.contiguous_format)
    return t


_NONE = (0, 0, 0, 0)
_MAX_SCALE = torch.finfo(torch.float32).max
_workspace_sizes: dict = {}      # of the library's answers, by what they depend on


def _tensor(t: torch.Tensor) -> tuple:
    b, l, h, _ = t.stride()
    return t.data_ptr(), b, l, h


class _Call:
    """Checked arguments of one call.  ``pack`` makes the library's descriptor of them (as bytes: setting the fields of a
    ctypes structure one by one costs more than the launch of a small problem)."""

    __slots__ = ("device", "code", "tensor_cores", "q", "k", "v", "sizes", "empty", "head", "bias", "bias_args", "bias_shape",
                 "mask", "mask_args")

    def __init__(self, q, k, v, bias, key_mask, scale, plain_kernels):
        if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
            raise ValueError("q, k and v must be [B, L, heads, D]")
        B, Lq, H, D = q.shape
        kshape = k.shape
        _, Lk, Hk, _ = kshape
        if kshape != v.shape or kshape[0] != B or kshape[3] != D:
            raise ValueError(f"k and v must both be [{B}, Lk, key heads, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
        if H and (Hk == 0 or H % Hk):
            raise ValueError(f"the {H} query heads must be a multiple of the {Hk} key heads")
        if D == 0:
            raise ValueError("the head dimension must not be empty")
        _require_cuda(q, "q")
        device, dtype = q.device, q.dtype
        code = _dtype_code(q)
        for name, t in (("k", k), ("v", v), ("bias", bias)):
            if t is not None and (t.dtype is not dtype or t.device != device):
                raise ValueError(f"{name} must be {dtype} on {device} like q, got {t.dtype} on {t.device}")
        tc = code == _lib.DTYPE_BF16 and D % 8 == 0 and D <= 128 and not plain_kernels
        self.device, self.code, self.tensor_cores = device, code, tc
        self.q, self.k, self.v = _laid_out(q, tc), _laid_out(k, tc), _laid_out(v, tc)
        self.sizes = (B, Lq, Lk, H, Hk, D)
        self.empty = B == 0 or Lq == 0 or H == 0
        scale = D ** -0.5 if scale is None else float(scale)
        if not abs(scale) <= _MAX_SCALE:
            raise ValueError(f"scale must be finite (in 32 bits), got {scale}")
        flags = _lib.ATTN_FLAG_PLAIN if plain_kernels else 0
        self.bias = self.bias_shape = self.mask = None
        self.bias_args, self.mask_args = (0, 0, 0, 0, 0, 0), (0, 0)
        if bias is not None:
            shape = tuple(bias.shape)
            if len(shape) not in (2, 3, 4):
                raise ValueError(f"bias must be [(B,) (H,) Lq, Lk], got {shape}")
            full = (1,) * (4 - len(shape)) + shape
            if full[0] not in (1, B) or full[1] not in (1, H) or full[2:] != (Lq, Lk):
                raise ValueError(f"bias must be [1 or {B}, 1 or {H}, {Lq}, {Lk}], got {shape}")
            self.bias_shape = shape
            bias = bias.detach() if bias.requires_grad else bias
            bias = bias[(None,) * (4 - len(shape))] if len(shape) < 4 else bias
            if not self.empty and Lk:
                if (bias.shape[3] > 1 and bias.stride(3) != 1) or min(bias.stride()) < 0:
                    bias = bias.contiguous()
                if tc and not _on_16_bytes(bias):
                    flags |= _lib.ATTN_FLAG_COPY_BIAS
            b, h, i, _ = bias.stride()
            self.bias, self.bias_args = bias, (bias.data_ptr(), b, h, i, full[0], full[1])
        if key_mask is not None:
            if tuple(key_mask.shape) != (B, Lk):
                raise ValueError(f"key_mask must be [B, Lk] = {(B, Lk)}, got {tuple(key_mask.shape)}")
            if key_mask.device != device:
                raise ValueError(f"key_mask is on {key_mask.device}, q on {device}")
            m = _mask_bytes(key_mask)
            self.mask, self.mask_args = m, (m.data_ptr(), m.stride(0))
        self.head = (_lib.ATTN_DESC.size, code, B, Lq, Lk, H, Hk, D, scale, flags)

    def pack(self, o, stats, o_lo, dout=_NONE, dq=_NONE, dk=_NONE, dv=_NONE, dbias=_NONE) -> bytes:
        """``trimul_attn_desc``; ``o`` ... ``dv`` as ``_tensor`` gives them."""
        return _lib.ATTN_DESC.pack(*self.head, *_tensor(self.q), *_tensor(self.k), *_tensor(self.v), *o, *dout, *dq, *dk, *dv,
                                   *self.bias_args, *self.mask_args, stats, o_lo, *dbias)

    def status(self):
        """The device's status words; none where a capture would have to create them."""
        if self.device.index not in _status and torch.cuda.is_current_stream_capturing():
            return None
        return _status_words(self.device).data_ptr()

    def workspace(self, desc: bytes, backward: bool, bias_grad: bool = False):
        """Scratch memory of its own for every call: calls on several streams, and graphs replayed side by side, share none."""
        key = (self.head, bias_grad, self.mask is not None, self.bias_args[4:], backward)
        n = _workspace_sizes.get(key)
        if n is None:
            size = C.c_size_t()
            _lib.check(_lib.load().trimul_b200_attn_workspace_bytes(desc, int(backward), C.byref(size)),
                       "trimul_b200_attn_workspace_bytes")
            n = size.value
            if len(_workspace_sizes) >= 1024:
                _workspace_sizes.clear()
            _workspace_sizes[key] = n
        return torch.empty(n, dtype=torch.uint8, device=self.device) if n else None


def _on_16_bytes(bias) -> bool:
    """Whether the tensor-core kernels can fetch this bf16 bias where it is."""
    if bias.data_ptr() % 16:
        return False
    (b, h, i, _), (sb, sh, si, _) = bias.shape, bias.stride()
    return (i == 1 or (si % 8 == 0 and si > 0)) and (h == 1 or (sh % 8 == 0 and sh > 0)) and (b == 1 or (sb % 8 == 0 and sb > 0))


def _like(t):
    """An uninitialised contiguous tensor of ``t``'s shape (``empty_like`` costs half of what ``empty`` does)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _rows_of(shape, like):
    """An uninitialised tensor whose rows start on 16-byte boundaries (a view into wider rows where they must)."""
    unit = 8 if like.dtype is torch.bfloat16 else 4
    pitch = -(-shape[-1] // unit) * unit
    t = like.new_empty((*shape[:-1], pitch))
    return t if pitch == shape[-1] else t.as_strided(shape, t.stride())


def _forward(call: _Call, state: bool):
    B, Lq, Lk, H, Hk, D = call.sizes
    with _on_device(call.device):
        out = _like(call.q)
        rows = out.new_empty((B, H, Lq, 2), dtype=torch.float32) if state else None
        rounding = torch.empty_like(out) if state and call.code == _lib.DTYPE_BF16 else None
        kept = AttentionState(rows, rounding) if state else None
        if call.empty or Lk == 0:
            if state:
                rows.zero_()
                if rounding is not None:
                    rounding.zero_()
            return out.zero_(), kept
        desc = call.pack(_tensor(out), rows.data_ptr() if state else 0, rounding.data_ptr() if rounding is not None else 0)
        ws = call.workspace(desc, False)
        rc = _lib.load().trimul_b200_attn_forward(desc, ws.data_ptr() if ws is not None else None,
                                                  ws.numel() if ws is not None else 0, _stream_handle(call.device),
                                                  call.status())
    _lib.check(rc, "trimul_b200_attn_forward")
    return out, kept


def cross_attention_forward_b200(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, bias: torch.Tensor | None = None,
                                 key_mask: torch.Tensor | None = None, scale: float | None = None,
                                 plain_kernels: bool = False) -> tuple:
    """``(result, AttentionState)`` of ``cross_attention_b200``, outside autograd; the state is what
    ``cross_attention_backward_b200`` takes."""
    return _forward(_Call(q, k, v, bias, key_mask, scale, plain_kernels), True)


def cross_attention_backward_b200(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                                  state: AttentionState, *, bias: torch.Tensor | None = None,
                                  key_mask: torch.Tensor | None = None, scale: float | None = None,
                                  bias_grad: bool = True, plain_kernels: bool = False) -> tuple:
    """``(dq, dk, dv, dbias)`` for the upstream gradient ``grad`` of ``cross_attention_forward_b200``'s result
    with the same arguments; ``dbias`` is None without a bias or with ``bias_grad=False``, and otherwise
    has the bias's shape (summed in fp32 over the axes along which it was shared, rounded once), its rows on
    16-byte boundaries.
    No atomics: the same call gives the same bits."""
    call = _Call(q, k, v, bias, key_mask, scale, plain_kernels)
    B, Lq, Lk, H, Hk, D = call.sizes
    for name, t in (("grad", grad), ("out", out)):
        if tuple(t.shape) != (B, Lq, H, D) or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must be {(B, Lq, H, D)} {q.dtype} on {q.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    rows, rounding = state
    if tuple(rows.shape) != (B, H, Lq, 2) or rows.dtype != torch.float32 or not rows.is_contiguous() or rows.device != q.device:
        raise ValueError("state does not belong to this call")
    if rounding is not None and (tuple(rounding.shape) != (B, Lq, H, D) or rounding.dtype != q.dtype
                                 or not rounding.is_contiguous() or rounding.device != q.device):
        raise ValueError("state does not belong to this call")
    grad, out = _laid_out(grad, call.tensor_cores), _laid_out(out, False)
    with _on_device(call.device):
        dq, dk = _like(call.q), _like(call.k)
        dv = torch.empty_like(dk)
        want = call.bias_shape is not None and bias_grad
        dbias = _rows_of(call.bias_shape, call.q) if want else None
        if call.empty or Lk == 0:
            for t in (dq, dk, dv, dbias):
                if t is not None:
                    t.zero_()
            return dq, dk, dv, dbias
        dbias_args = _NONE
        if want:
            full = dbias[(None,) * (4 - dbias.dim())]
            dbias_args = (full.data_ptr(), *full.stride()[:3])
        desc = call.pack(_tensor(out), rows.data_ptr(), rounding.data_ptr() if rounding is not None else 0, _tensor(grad),
                         _tensor(dq), _tensor(dk), _tensor(dv), dbias_args)
        ws = call.workspace(desc, True, want)
        rc = _lib.load().trimul_b200_attn_backward(desc, ws.data_ptr(), ws.numel(), _stream_handle(call.device), call.status())
    _lib.check(rc, "trimul_b200_attn_backward")
    return dq, dk, dv, dbias


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, key_mask, scale, plain_kernels):
        call = _Call(q, k, v, bias, key_mask, scale, plain_kernels)
        out, state = _forward(call, True)
        ctx.save_for_backward(q, k, v, bias, key_mask, out, *state)
        ctx.scale, ctx.plain_kernels = scale, plain_kernels
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, bias, key_mask, out, rows, rounding = ctx.saved_tensors
        dq, dk, dv, dbias = cross_attention_backward_b200(
            grad, q, k, v, out, AttentionState(rows, rounding), bias=bias, key_mask=key_mask, scale=ctx.scale,
            bias_grad=ctx.needs_input_grad[3], plain_kernels=ctx.plain_kernels)
        return dq, dk, dv, dbias, None, None, None


def cross_attention_b200(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, bias: torch.Tensor | None = None,
                         key_mask: torch.Tensor | None = None, scale: float | None = None,
                         plain_kernels: bool = False) -> torch.Tensor:
    """``softmax(scale * q k^T + bias) v`` over the kept keys, ``[B, Lq, H, D]``.

    ``q``: ``[B, Lq, H, D]``; ``k``, ``v``: ``[B, Lk, Hk, D]`` with ``Hk`` a divisor of ``H`` (query heads
    ``g * H / Hk ...`` share key head ``g``); any strides (a ``[B, heads, L, D]`` tensor is passed as its
    transposed view).  bf16 or fp32, the same for all; ``D`` at most 256.  ``bias``: ``[(B,) (H,) Lq, Lk]``,
    axes of size 1 shared; minus infinity masks a pair.  ``key_mask``: ``[B, Lk]``, False at keys that are
    left out, whose keys and values may hold anything, NaN included.  ``scale`` defaults to ``D ** -0.5``.
    A row without a kept key gives zeros (and zero gradients); a row whose scores hold a NaN gives NaN.

    bf16 with ``D`` a multiple of 8 up to 128 runs on the tensor cores, everything else (and
    ``plain_kernels=True``) on the CUDA cores in fp32 arithmetic.  The tensor-core kernels round the probabilities, and
    in the backward pass the scores' gradients, to bf16 on their way into a product (half a step each, beside the
    rounding of the result); ``plain_kernels=True`` keeps them in fp32.  Differentiable in ``q``, ``k``, ``v`` and
    ``bias``, in reverse mode; an input with a forward-mode tangent is refused."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, bias)):
        return _CrossAttention.apply(q, k, v, bias, key_mask, scale, plain_kernels)
    _require_no_tangent("cross_attention_b200", q, k, v, bias)
    return _forward(_Call(q, k, v, bias, key_mask, scale, plain_kernels), False)[0]
