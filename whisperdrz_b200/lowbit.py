"""Operands of the low-bit decode operators: a key/value cache in 8 bits with a scale for each block of 64 tokens and
head, and a linear layer's weights in 4 bits with group scales.  The reference holds both in 16 or 32 bits
(FlashKVCache, src/whisperdrz/model.py:98-147; nn.Linear, :258-261).  The calls that use them are methods of ``Engine``:
``qcache_store``, ``qcache_attention`` and ``linear_rows_packed``."""
from __future__ import annotations

import ctypes as C

import torch

from . import capi

BLOCK = capi.QCACHE_BLOCK
HEAD_DIM = 64
SEGMENT = 128   # weights of a row that are packed together


def rows_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a byte of one's rows is a byte of the other's.  Rows [n, width] with unit stride, none over another of its own."""
    n = a.shape[0]
    if n == 0:
        return False
    pa, pb = a.data_ptr(), b.data_ptr()
    wa, wb = a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
    sa = a.stride(0) * a.element_size() if n > 1 else wa
    sb = b.stride(0) * b.element_size() if n > 1 else wb
    if pa + (n - 1) * sa + wa <= pb or pb + (n - 1) * sb + wb <= pa:
        return False
    if sa == sb and wa <= (pb - pa) % sa <= sa - wb:     # columns of one product
        return False
    return any(max(0, (lo - wa - pa) // sa + 1) <= min(n - 1, (lo + wb - 1 - pa) // sa) for lo in range(pb, pb + n * sb, sb))


def _fixed(name: str) -> property:
    """A tensor that was checked, and whose address may have been handed on: it may be written into, not replaced."""
    return property(lambda self: self.__dict__["_" + name])


class QCache:
    """An 8-bit cache by its tensors: ``k`` / ``v`` int8 [n_slots, n_heads, 64 * n_blocks, 64], ``k_scale`` / ``v_scale``
    f32 [n_slots, n_heads, n_blocks].  A token's values are its int8 times the scale of its block of 64 tokens.  Slots may
    lie further apart than their size (a layer of a larger allocation); K and V alike."""

    k, v, k_scale, v_scale = map(_fixed, ("k", "v", "k_scale", "v_scale"))

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dim() != 4 or k.shape[3] != HEAD_DIM or k.shape[2] == 0 or k.shape[2] % BLOCK or k.shape != v.shape:
            raise ValueError(f"QCache: k and v are [slots, heads, 64 * blocks, 64], got {tuple(k.shape)} and {tuple(v.shape)}")
        want = (k.shape[0], k.shape[1], k.shape[2] // BLOCK)
        if tuple(k_scale.shape) != want or tuple(v_scale.shape) != want:
            raise ValueError(f"QCache: scales are {want}, got {tuple(k_scale.shape)} and {tuple(v_scale.shape)}")
        if k.dtype != torch.int8 or v.dtype != torch.int8 or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError("QCache: int8 values and float32 scales")
        if k.shape[0] < 1 or k.shape[1] < 1:
            raise ValueError("QCache: at least one slot and one head")
        if len({t.device for t in (k, v, k_scale, v_scale)}) != 1:
            raise ValueError("QCache: the tensors lie on different devices")
        for t in (k, v, k_scale, v_scale):
            if not t[0].is_contiguous():
                raise ValueError("QCache: a slot's part must be contiguous")
        n_slots, n_heads, n_tokens, _ = k.shape
        step = k.stride(0) if n_slots > 1 else k[0].numel()
        scale_step = k_scale.stride(0) if n_slots > 1 else k_scale[0].numel()
        if n_slots > 1 and (v.stride(0) != step or v_scale.stride(0) != scale_step):
            raise ValueError("QCache: k and v need the same distance from slot to slot, and their scales too")
        if step < k[0].numel() or scale_step < k_scale[0].numel():
            raise ValueError("QCache: the slots overlap")
        if step % 16 or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("QCache: values must start on 16 bytes")
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self.n_slots, self.n_heads, self.n_tokens, self.device, self.ordinal = n_slots, n_heads, n_tokens, k.device, k.get_device()
        self.desc = capi.QCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), step, scale_step,
                                    n_slots, n_heads, n_tokens // BLOCK)
        self.ref = C.byref(self.desc)
        self.apart = not (rows_overlap(k.flatten(1), v.flatten(1)) or rows_overlap(k_scale.flatten(1), v_scale.flatten(1)))
        self.scratch: dict = {}   # bytes of scratch by call shape, as the library told them

    @classmethod
    def empty(cls, n_slots: int, n_tokens: int, n_heads: int, device) -> "QCache":
        """A cache for ``n_tokens`` tokens a slot (rounded up to whole blocks), all zero."""
        blocks = max(1, (n_tokens + BLOCK - 1) // BLOCK)
        shape = (n_slots, n_heads, BLOCK * blocks, HEAD_DIM)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:2] + (blocks,), device=device), torch.zeros(shape[:2] + (blocks,), device=device))


class PackedLinear:
    """A linear layer's weights in 4 bits: ``weight`` uint8 [N, Kp / 2] in the order of include/wdz.h
    (wdz_linear_rows_packed), ``scale`` bf16 [N, Kp / group], optional ``bias`` [N], best in the type of the rows to
    come (one of the other type is converted in every call); Kp is ``in_features`` rounded up to a multiple of 128."""

    weight, scale, bias = map(_fixed, ("weight", "scale", "bias"))

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, in_features: int, group: int, bias: torch.Tensor | None = None):
        if group not in (32, 64, 128):
            raise ValueError(f"PackedLinear: groups of 32, 64 or 128 weights, got {group}")
        kp = (in_features + SEGMENT - 1) // SEGMENT * SEGMENT
        if in_features < 1 or weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] * 2 != kp or weight.dtype != torch.uint8:
            raise ValueError(f"PackedLinear: weight is uint8 [N, {kp // 2}], got {weight.dtype} {tuple(weight.shape)}")
        if tuple(scale.shape) != (weight.shape[0], kp // group) or scale.dtype != torch.bfloat16:
            raise ValueError(f"PackedLinear: scale is bfloat16 {(weight.shape[0], kp // group)}, got {scale.dtype} {tuple(scale.shape)}")
        if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype not in (torch.float32, torch.bfloat16)):
            raise ValueError("PackedLinear: bias is [N] in float32 or bfloat16")
        if any(t.device != weight.device for t in (scale, bias) if t is not None):
            raise ValueError("PackedLinear: the tensors lie on different devices")
        if not weight.is_contiguous() or not scale.is_contiguous() or weight.data_ptr() % 16 or scale.data_ptr() % 8:
            raise ValueError("PackedLinear: contiguous tensors, the weights on 16 bytes and the scales on 8")
        self._weight, self._scale, self.in_features, self.group = weight, scale, int(in_features), int(group)
        self.out_features, self.device, self.ordinal = weight.shape[0], weight.device, weight.get_device()
        self._bias = None if bias is None else bias.contiguous()
        self.at, self.scale_at = weight.data_ptr(), scale.data_ptr()


def pack_linear(weight: torch.Tensor, group: int = 64, bias: torch.Tensor | None = None) -> PackedLinear:
    """Rounds an nn.Linear weight [N, K] to 4 bits: per group of ``group`` inputs the scale is max|w| / 7 in bf16, and the
    values are round(w / scale) in [-8, 7]."""
    if group not in (32, 64, 128):
        raise ValueError(f"pack_linear: groups of 32, 64 or 128 weights, got {group}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"pack_linear: weight is [N, K], got {tuple(weight.shape)}")
    n, k = weight.shape
    kp = (k + SEGMENT - 1) // SEGMENT * SEGMENT
    w = torch.nn.functional.pad(weight.detach().float(), (0, kp - k)).view(n, kp // group, group)
    scale = (w.abs().amax(-1) / 7).bfloat16()
    div = scale.float()[..., None]
    q = torch.where(div > 0, w / torch.where(div > 0, div, torch.ones_like(div)), torch.zeros_like(w))
    return PackedLinear(pack_nibbles(q.round().clamp(-8, 7).to(torch.int32).view(n, kp)), scale.contiguous(), k, group, bias)


def pack_nibbles(q: torch.Tensor) -> torch.Tensor:
    """Whole numbers in [-8, 7], [N, K] with K a multiple of 128 -> uint8 [N, K / 2] in the kernel's order: a lane of the
    matrix instruction takes 16 bytes and finds in each of their four words eight neighbouring inputs of one group of 32."""
    n, k = q.shape
    u = (q.to(torch.int64) + 8).view(n, k // SEGMENT, 4, 4, 4, 2)     # segment, word i, lane t, pair j, odd
    j = torch.arange(4, device=q.device).view(4, 1)
    shift = 4 * j + 16 * torch.arange(2, device=q.device)
    words = (u << shift).sum((-1, -2)).transpose(2, 3).reshape(n, k // 8)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words)
    return words.to(torch.int32).contiguous().view(torch.uint8)
