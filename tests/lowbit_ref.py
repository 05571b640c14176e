"""The low-bit operators in 64 bits, from their definitions (include/wdz.h), one row and one block at a time."""
import numpy as np

BLOCK, HEAD = 64, 64
TINY = 2.0 ** -117


def dequant(values, scale):
    """int8 [heads, tokens, 64], f32 [heads, blocks] -> f64."""
    return values.astype(np.float64) * np.repeat(scale.astype(np.float64), BLOCK, axis=1)[..., None]


def store(values, scale, rows, slots, positions, row_begin=None):
    """Rounds rows f32 [n, heads * 64] into values int8 [slots, heads, tokens, 64] / scale f32 [slots, heads, blocks], in
    place."""
    heads = values.shape[1]
    rows = rows.reshape(rows.shape[0], heads, HEAD).astype(np.float64)
    begin = range(len(slots) + 1) if row_begin is None else row_begin
    for i, (slot, p0) in enumerate(zip(slots, positions)):
        x = rows[begin[i]:begin[i + 1]]
        p1 = p0 + len(x)
        if not 0 <= slot < values.shape[0] or not len(x):
            continue
        for b in range(p0 // BLOCK, (p1 - 1) // BLOCK + 1):
            lo, hi = max(p0, b * BLOCK), min(p1, (b + 1) * BLOCK)
            for h in range(heads):
                new = x[lo - p0:hi - p0, h]
                top = np.abs(new[np.isfinite(new)]).max(initial=0.0)
                mine = np.float32(top / 127) if top >= TINY else np.float32(0)
                old = np.float32(0) if lo == b * BLOCK else scale[slot, h, b]
                now = max(old, mine)
                if now > old and lo > b * BLOCK:
                    kept = values[slot, h, b * BLOCK:lo].astype(np.float64)
                    values[slot, h, b * BLOCK:lo] = np.rint(kept * np.float64(old) / np.float64(now))
                with np.errstate(all="ignore"):
                    q = np.rint(new / np.float64(now)) if now > 0 else np.zeros_like(new)
                q = np.where(np.isnan(new), 0, np.clip(np.nan_to_num(q, nan=0, posinf=127, neginf=-127), -127, 127))
                values[slot, h, lo:hi] = q
                scale[slot, h, b] = now


def attend(q, k, v, k_scale, v_scale, slots, lens, scale):
    """f64 output [n, q_heads * 64] (NaN where the row is skipped) and, per query head, the pieces that an error bound
    needs: the largest sum |q_i k_i| over its tokens and the largest |v|."""
    n, heads = q.shape[0], k.shape[1]
    group = q.shape[1] // (heads * HEAD)
    q = q.astype(np.float64).reshape(n, heads, group, HEAD)
    out = np.full((n, heads, group, HEAD), np.nan)
    weight, top = np.zeros((n, heads, group)), np.zeros((n, heads, group))
    for r in range(n):
        if not 0 <= slots[r] < k.shape[0]:
            continue
        t = min(max(int(lens[r]), 0), k.shape[2])
        if t == 0:
            out[r] = 0
            continue
        blocks = (t + BLOCK - 1) // BLOCK
        kk = dequant(k[slots[r], :, :blocks * BLOCK], k_scale[slots[r], :, :blocks])[:, :t]
        vv = dequant(v[slots[r], :, :blocks * BLOCK], v_scale[slots[r], :, :blocks])[:, :t]
        s = scale * np.einsum("hgd,htd->hgt", q[r], kk)
        w = np.exp(s - s.max(-1, keepdims=True))
        out[r] = np.einsum("hgt,htd->hgd", w / w.sum(-1, keepdims=True), vv)
        # |q| in the kernel's fixed point is off by a part of the head's largest |q_i|: bound with that for every i
        most = np.abs(q[r]).max(-1)
        weight[r] = scale * most * np.abs(kk).sum(-1).max(-1)[:, None]
        top[r] = np.abs(vv).max((-2, -1))[:, None]
    return out.reshape(n, -1), weight, top


def unpack(packed, kp):
    """uint8 [N, kp / 2] -> whole numbers in [-8, 7], [N, kp]."""
    words = np.ascontiguousarray(packed).view(np.uint32).reshape(packed.shape[0], kp // 8)
    out = np.zeros((packed.shape[0], kp), dtype=np.int64)
    for w in range(kp // 8):
        seg, t, i = w // 16, w % 16 // 4, w % 4
        for e in range(8):
            bit = 4 * (e // 2) + 16 * (e % 2)
            out[:, seg * 128 + 32 * i + 8 * t + e] = ((words[:, w] >> bit) & 15).astype(np.int64) - 8
    return out
