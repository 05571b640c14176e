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


def rows_overlap(n: int, a: int, a_step: int, a_width: int, b: int, b_step: int, b_width: int) -> bool:
    """Whether a byte of one's ``n`` rows is a byte of the other's: first row's address, bytes from row to row and of a row (the
    step counts for nothing where n is 1, and no row lies over another of its own)."""
    if n < 2:
        return n == 1 and a < b + b_width and b < a + a_width
    if a + (n - 1) * a_step + a_width <= b or b + (n - 1) * b_step + b_width <= a:
        return False
    if a_step == b_step and a_width <= (b - a) % a_step <= a_step - b_width:     # columns of one product
        return False
    return any(max(0, (lo - a_width - a) // a_step + 1) <= min(n - 1, (lo + b_width - 1 - a) // a_step)
               for lo in range(b, b + n * b_step, b_step))


class _Operand:
    """Holds tensors that were checked and whose addresses have been handed on: they may be written into, not replaced.  A hook
    on writes, so that reading one costs no more than any attribute."""
    _fixed: tuple = ()
    _made = False

    def __setattr__(self, name, value):
        if self._made and name in self._fixed:
            raise AttributeError(f"{type(self).__name__}: {name} cannot be replaced")
        super().__setattr__(name, value)


class QCache(_Operand):
    """An 8-bit cache by its tensors: ``k`` / ``v`` int8 [n_slots, n_heads, 64 * n_blocks, 64], ``k_scale`` / ``v_scale``
    f32 [n_slots, n_heads, n_blocks].  A token's values are its int8 times the scale of its block of 64 tokens.  Slots may
    lie further apart than their size (a layer of a larger allocation); K and V alike."""

    _fixed = ("k", "v", "k_scale", "v_scale")

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
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_slots, self.n_heads, self.n_tokens, self.device, self.ordinal = n_slots, n_heads, n_tokens, k.device, k.get_device()
        self.desc = capi.QCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), step, scale_step,
                                    n_slots, n_heads, n_tokens // BLOCK)
        self.ref = C.byref(self.desc)
        size = n_heads * n_tokens * HEAD_DIM
        self.apart = not (rows_overlap(n_slots, self.desc.k, step, size, self.desc.v, step, size)
                          or rows_overlap(n_slots, self.desc.k_scale, 4 * scale_step, size // 1024, self.desc.v_scale, 4 * scale_step, size // 1024))
        self.scratch: dict = {}   # bytes of scratch by call shape, as the library told them
        self._made = True

    @classmethod
    def empty(cls, n_slots: int, n_tokens: int, n_heads: int, device) -> "QCache":
        """A cache for ``n_tokens`` tokens a slot (rounded up to whole blocks), all zero."""
        blocks = max(1, (n_tokens + BLOCK - 1) // BLOCK)
        shape = (n_slots, n_heads, BLOCK * blocks, HEAD_DIM)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:2] + (blocks,), device=device), torch.zeros(shape[:2] + (blocks,), device=device))


class PackedLinear(_Operand):
    """A linear layer's weights in 4 bits: ``weight`` uint8 [N, Kp / 2] in the order of include/wdz.h
    (wdz_linear_rows_packed), ``scale`` bf16 [N, Kp / group], optional ``bias`` [N], best in the type of the rows to
    come (one of the other type is converted in every call); Kp is ``in_features`` rounded up to a multiple of 128."""

    _fixed = ("weight", "scale", "bias")

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
        self.weight, self.scale, self.in_features, self.group = weight, scale, int(in_features), int(group)
        self.out_features, self.device, self.ordinal = weight.shape[0], weight.device, weight.get_device()
        self.bias = None if bias is None else bias.contiguous()
        self.at, self.scale_at = weight.data_ptr(), scale.data_ptr()
        self._made = True


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
