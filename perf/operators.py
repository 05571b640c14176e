"""What the low-bit decode operators are measured on: the 8-bit key/value cache (storing rows into it, attending over it)
and the decoder's linear layer with 4-bit weights.

``own`` selects the side: False computes the operators in their plain form with elementary torch operations, True makes
the calls a user of the framework makes.  Both take the same inputs from ``prepare``.

The cache.  ``k`` and ``v`` are int8 [slots, heads, 64 * blocks, 64], ``k_scale`` and ``v_scale`` f32
[slots, heads, blocks]: a token's value is its int8 times the scale of its block of 64 tokens.

The packed weights.  Row n of the uint8 matrix holds K (padded to a multiple of 128) signed 4-bit values as value + 8.
Of every 128 of them, 32-bit word 4 t + i holds elements 32 i + 8 t ... + 7: bits 4 j of the word hold element 2 j, bits
4 (j + 4) element 2 j + 1.  The scales are bf16 [N, padded K / group].
"""
import math

import torch

own = False

HEAD = 64      # values of a head
BLOCK = 64     # tokens that share a scale
SEGMENT = 128  # weights of a row that are packed together


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one 30 s window decoded alone: every key of the encoder's 1500 positions for one new token (latency)
        _attend("attend_one_window", 1, 20, 1, 1500, False, "bf16"),
        # a serving engine with the default 32 slots, one decode step's cross-attention
        _attend("attend_32_windows", 32, 20, 1, 1500, False, "bf16"),
        # the benchmark's 384 chunks, one decode step's cross-attention: the dominant byte stream of the whole path
        _attend("attend_384_windows", 384, 20, 1, 1500, False, "bf16"),
        # the same step's self-attention: every row at its own depth of at most 448 tokens, some slots empty; fp32 engine
        _attend("attend_384_ragged", 384, 20, 1, 448, True, "f32"),
        # few rows over a long history with query heads that share their keys
        _attend("attend_long_shared", 2, 4, 4, 32749, False, "bf16"),
        # one finished prefill of 32 windows: K and V columns of the cross projection into their slots
        _store("store_32_windows", 32, 20, 1500, "bf16", 24, "windows"),
        # one decode step of the benchmark batch: one new row per slot, out of the fused QKV product
        _store("store_384_steps", 384, 20, 1, "f32", 7, "steps"),
        # prompts of uneven lengths that continue what their slots hold
        _store("store_24_prompts", 24, 20, 223, "bf16", 7, "prompts"),
        # a decoder layer's output projection for one row (latency)
        _linear("linear_one_row", 1, 1280, 1280, 64, "bf16", False),
        # the tied head over the vocabulary for one row: the largest weight of the decoder
        _linear("linear_head", 1, 51866, 1280, 128, "bf16", False),
        # the second half of the feed-forward block added into the residual stream, 16 rows
        _linear("linear_16_rows", 16, 1280, 5120, 32, "bf16", True),
        # the fp32 engine's first half, odd sizes
        _linear("linear_f32_odd", 5, 5003, 1237, 64, "f32", False),
    ]


def _attend(name, rows, heads, group, tokens, ragged, dtype):
    return {"name": name, "op": "attend", "rows": rows, "heads": heads, "group": group, "tokens": tokens, "ragged": ragged,
            "dtype": dtype}


def _store(name, runs, heads, length, dtype, blocks, kind):
    return {"name": name, "op": "store", "runs": runs, "heads": heads, "length": length, "dtype": dtype, "blocks": blocks,
            "kind": kind}


def _linear(name, rows, n, k, group, dtype, accumulate):
    return {"name": name, "op": "linear", "rows": rows, "n": n, "k": k, "group": group, "dtype": dtype, "accumulate": accumulate}


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "store", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "attend":
        heads, group = rng.choice([(20, 1), (20, 1), (4, 1), (2, 1), (8, 2), (4, 4), (1, 8)])
        rows = _log(rng, 1, 384)
        tokens = _log(rng, 1, 33000)
        tokens = max(1, min(tokens, 384 * 20 * 1500 // (rows * heads * group)))
        c = _attend("", rows, heads, group, tokens, rng.random() < 0.5, dtype)
    elif op == "store":
        kind = rng.choice(["windows", "steps", "prompts"])
        heads = rng.choice([2, 4, 20])
        runs = _log(rng, 1, 384)
        length = 1 if kind == "steps" else max(1, min(_log(rng, 2, 1500), 48000 // runs))
        blocks = (length + BLOCK - 1) // BLOCK + rng.randint(1 if kind == "prompts" else 0, 5)
        c = _store("", runs, heads, length, dtype, blocks, kind)
    else:
        rows, n, k = _log(rng, 1, 16), _log(rng, 64, 51866), _log(rng, 64, 5120)
        n = max(64, min(n, 51866 * 1280 // k))
        c = _linear("", rows, n, k, rng.choice([32, 64, 128]), dtype, rng.random() < 0.5)
    c.pop("name")
    return c


def _lengths(c):
    """Tokens that each row attends to, before the seed permutes them: all alike, or spread evenly with every sixteenth
    row empty."""
    if not c["ragged"]:
        return [c["tokens"]] * c["rows"]
    return [0 if i % 16 == 5 else 1 + int(c["tokens"] * ((i * 0.6180339887498949 + 0.5) % 1.0)) for i in range(c["rows"])]


def _run_lengths(c):
    if c["kind"] != "prompts":
        return [c["length"]] * c["runs"]
    return [1 + int(c["length"] * ((i * 0.6180339887498949 + 0.3) % 1.0)) for i in range(c["runs"])]


def work(c):
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "attend":
        lens, h, hq = _lengths(c), c["heads"], c["heads"] * c["group"]
        blocks = sum((n + BLOCK - 1) // BLOCK for n in lens)
        return {"bytes": 2 * h * (sum(lens) * HEAD + 4 * blocks) + 2 * c["rows"] * hq * HEAD * size,
                "flops": 4.0 * sum(lens) * hq * HEAD}
    if c["op"] == "store":
        rows = sum(_run_lengths(c))
        blocks = c["runs"] if c["kind"] == "steps" else sum((n + BLOCK - 1) // BLOCK for n in _run_lengths(c))
        return {"bytes": 2 * c["heads"] * (rows * HEAD * (size + 1) + 8 * blocks), "flops": 4.0 * rows * c["heads"] * HEAD}
    kp = (c["k"] + SEGMENT - 1) // SEGMENT * SEGMENT
    return {"bytes": c["n"] * (kp / 2 + 2 * kp / c["group"] + 4) + c["rows"] * (c["k"] * size + 4 * c["n"]),
            "flops": 2.0 * c["rows"] * c["n"] * c["k"]}


# --------------------------------------------------------------------- inputs
def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _cache(g, slots, heads, blocks):
    """A filled cache: int8 values as an absolute-maximum scale leaves them (a normal distribution that reaches +-127 near
    four standard deviations), scales around 0.03 that differ from block to block."""
    dev = g.device
    shape = (slots, heads, BLOCK * blocks, HEAD)

    def values():
        t = torch.empty(shape, dtype=torch.int8, device=dev)
        for i in range(0, slots, 32):   # in parts: the normal numbers of a large cache would not fit three times over
            part = torch.randn(t[i:i + 32].shape, generator=g, device=dev)
            t[i:i + 32] = (part * 32.0).round().clamp(-127, 127).to(torch.int8)
        return t

    def scales():
        return 0.03 * torch.exp(0.3 * torch.randn(slots, heads, blocks, generator=g, device=dev))

    return {"k": values(), "v": values(), "k_scale": scales(), "v_scale": scales()}


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = _dtype(c)
    if c["op"] == "attend":
        rows, h, hq = c["rows"], c["heads"], c["heads"] * c["group"]
        s = _cache(g, rows, h, (c["tokens"] + BLOCK - 1) // BLOCK)
        perm = torch.randperm(rows, generator=g, device=dev)
        s["lens"] = torch.tensor(_lengths(c), dtype=torch.int32).to(dev)[perm]
        s["slots"] = torch.randperm(rows, generator=g, device=dev).to(torch.int32)
        sharp = torch.exp(0.7 * torch.randn(1, hq, 1, generator=g, device=dev))   # flat heads and peaked ones
        s["q"] = (torch.randn(rows, hq, HEAD, generator=g, device=dev) * sharp).to(dt).view(rows, hq * HEAD)
        s["dtype"] = dt
        return _handle(s, c)
    if c["op"] == "store":
        runs, h, blocks = c["runs"], c["heads"], c["blocks"]
        slots = runs + 3
        s = _cache(g, slots, h, blocks)
        order = torch.randperm(runs, generator=g, device=dev)
        lens = torch.tensor(_run_lengths(c), dtype=torch.int32).to(dev)[order]
        s["row_begin"] = None if c["kind"] == "steps" else torch.cat([lens.new_zeros(1), lens.cumsum(0).to(torch.int32)])
        s["slots"] = torch.randperm(slots, generator=g, device=dev)[:runs].to(torch.int32)
        room = BLOCK * blocks - lens + 1
        first = (torch.rand(runs, generator=g, device=dev) * room).to(torch.int32)
        s["positions"] = torch.zeros_like(first) if c["kind"] == "windows" else first
        s["max_run"] = max(_run_lengths(c))
        rows, d = sum(_run_lengths(c)), h * HEAD
        loud = torch.exp(0.8 * torch.randn(3 * d, generator=g, device=dev))   # keys have a few loud channels
        rowsin = (torch.randn(rows, 3 * d, generator=g, device=dev) * loud).to(dt)   # a fused product: q | k | v
        s["new_k"], s["new_v"] = rowsin[:, d:2 * d], rowsin[:, 2 * d:]
        return _handle(s, c)
    n, k, grp = c["n"], c["k"], c["group"]
    kp = (k + SEGMENT - 1) // SEGMENT * SEGMENT
    q = (torch.randn(n, kp, generator=g, device=dev) * 2.5).round().clamp(-8, 7).to(torch.int32) + 8
    q[:, k:] = 8
    s = {"w": _pack(q), "w_scale": (0.01 * torch.exp(0.3 * torch.randn(n, kp // grp, generator=g, device=dev))).bfloat16()}
    s["x"] = torch.randn(c["rows"], k, generator=g, device=dev).to(dt)
    s["bias"] = (0.1 * torch.randn(n, generator=g, device=dev)).to(dt)
    s["residual"] = torch.randn(c["rows"], n, generator=g, device=dev) if c["accumulate"] else None
    s["group"], s["k_in"] = grp, k
    return _handle(s, c)


def _handle(s, c):
    """The objects that a program of this framework keeps: its engine, and its cache or weights by their tensors."""
    s["op"] = c["op"]
    if own:
        from whisperdrz_b200.lowbit import PackedLinear, QCache
        s["engine"] = _engine()
        if c["op"] == "linear":
            s["weights"] = PackedLinear(s["w"], s["w_scale"], s["k_in"], s["group"], s["bias"])
        else:
            s["cache"] = QCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


def _pack(u):
    """4-bit values + 8, int32 [N, K] with K a multiple of 128 -> uint8 [N, K / 2]."""
    n, k = u.shape
    w = u.view(n, k // SEGMENT, 4, 4, 4, 2)              # segment, i, t, j, odd
    shift = 4 * torch.arange(4, device=u.device, dtype=torch.int32).view(4, 1) + torch.tensor([0, 16], device=u.device, dtype=torch.int32)
    words = (w.to(torch.int64) << shift).sum((-1, -2))    # disjoint bits: the sum is the union
    words = words.transpose(2, 3).reshape(n, k // 8)      # word 4 t + i
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).contiguous().view(torch.uint8)


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "attend":
        return _attend_plain(s)
    if s["op"] == "store":
        return _store_plain(s)
    return _linear_plain(s)


def _attend_plain(s):
    slot, lens = s["slots"].long(), s["lens"]
    rows, h = slot.numel(), s["k"].shape[1]
    most = s["k"].shape[2]
    q = s["q"].float().view(rows, h, -1, HEAD)
    k = s["k"][slot].float() * s["k_scale"][slot].repeat_interleave(BLOCK, 2)[..., None]
    scores = (q @ k.transpose(2, 3)) * HEAD ** -0.5
    del k
    seen = torch.arange(most, device=q.device) < lens[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = s["v"][slot].float() * s["v_scale"][slot].repeat_interleave(BLOCK, 2)[..., None]
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(rows, -1).to(s["dtype"])


def _places(s):
    """Run, slot and position of every source row."""
    n = s["new_k"].shape[0]
    i = torch.arange(n, device=s["new_k"].device)
    if s["row_begin"] is None:
        run_of, first = i, i
    else:
        begin = s["row_begin"].long()
        run_of = torch.searchsorted(begin[1:], i, right=True)
        first = begin[run_of]
    return s["slots"].long()[run_of], s["positions"].long()[run_of] + i - first


def _store_one(s, new, values, scale, slot, pos):
    """The rows ``new`` into ``values`` / ``scale``, in place: a block that is entered at its first token starts with the
    new rows' own scale, one that is entered later keeps the larger of that and its old scale, and what it held is
    rounded to the new scale."""
    slots, h, blocks = scale.shape
    x = new.reshape(new.shape[0], h, HEAD).float()
    place = slot * blocks + pos // BLOCK
    top = torch.zeros(slots * blocks, h, device=x.device)
    top.scatter_reduce_(0, place[:, None].expand(-1, h), x.abs().amax(-1), "amax")
    fresh = torch.zeros(slots * blocks, dtype=torch.bool, device=x.device)
    fresh[place[pos % BLOCK == 0]] = True
    touched = torch.zeros_like(fresh)
    touched[place] = True
    old = scale.permute(0, 2, 1).reshape(slots * blocks, h)
    was = torch.where(fresh[:, None], torch.zeros_like(old), old)
    now = torch.where(touched[:, None], torch.maximum(was, (top.double() / 127.0).float()), old)
    # what the first, partly filled block of each run already holds
    rs, rp = s["slots"].long(), s["positions"].long()
    rb, kept = rp // BLOCK, rp % BLOCK
    tiles = values.view(slots, h, blocks, BLOCK, HEAD)
    held = tiles[rs, :, rb]
    before, after = old[rs * blocks + rb], now[rs * blocks + rb]
    again = (held.double() * before.double()[..., None, None] / after.double().clamp_min(1e-300)[..., None, None]).round()
    mine = (torch.arange(BLOCK, device=x.device) < kept[:, None])[:, None] & (after > before)[..., None]
    tiles[rs, :, rb] = torch.where(mine[..., None], again.to(torch.int8), held)
    mul = now[place].double()
    code = torch.where(mul[..., None] > 0, x.double() / mul.clamp_min(1e-300)[..., None], torch.zeros_like(x, dtype=torch.float64))
    values[slot, :, pos] = code.round().clamp(-127, 127).to(torch.int8)
    scale.copy_(now.view(slots, blocks, h).permute(0, 2, 1))


def _store_plain(s):
    slot, pos = _places(s)
    _store_one(s, s["new_k"], s["k"], s["k_scale"], slot, pos)
    _store_one(s, s["new_v"], s["v"], s["v_scale"], slot, pos)
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _linear_plain(s):
    n, kp = s["w"].shape[0], 2 * s["w"].shape[1]
    words = s["w"].view(torch.int32).view(n, kp // SEGMENT, 4, 4).transpose(2, 3)
    shift = 4 * torch.arange(4, device=words.device, dtype=torch.int32).view(4, 1) + torch.tensor([0, 16], device=words.device, dtype=torch.int32)
    q = ((words[..., None, None] >> shift) & 15).reshape(n, kp) - 8
    w = q.float().view(n, -1, s["group"]) * s["w_scale"].float()[..., None]
    y = s["x"].float() @ w.view(n, kp)[:, :s["k_in"]].T + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"]
    return y


# ------------------------------------------------------- the framework's calls
_held = {}


def _engine():
    """The program's engine: any engine offers the operators, so the smallest model serves."""
    if "engine" not in _held:
        from whisperdrz_b200.dims import ModelDimensions
        from whisperdrz_b200.engine import Engine
        from whisperdrz_b200.weights import init_state_dict
        dims = ModelDimensions.from_name("test-tiny")
        _held["engine"] = Engine(dims, init_state_dict(dims, 0), dtype=torch.float32, n_slots=1, max_clips=1, max_rows=1)
    return _held["engine"]


def _run_own(s):
    e = s["engine"]
    if s["op"] == "linear":
        return e.linear_rows_packed(s["x"], s["weights"], residual=s["residual"])
    cache = s["cache"]
    if s["op"] == "attend":
        return e.qcache_attention(s["q"], cache, s["slots"], s["lens"], out_dtype=s["dtype"])
    e.qcache_store(cache, s["new_k"], s["new_v"], s["slots"], s["positions"], row_begin=s["row_begin"], max_run=s["max_run"])
    return cache.k, cache.v, cache.k_scale, cache.v_scale


# ---------------------------------------------------------- in 64 bits, apart
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "attend":
        outs = []
        h, grp = c["heads"], c["group"]
        for slot, n, q in zip(s["slots"].tolist(), s["lens"].tolist(), s["q"].double().view(c["rows"], h, grp, HEAD)):
            o = torch.zeros(h, grp, HEAD, dtype=torch.float64, device=q.device)
            if n:
                block = torch.arange(n, device=q.device) // BLOCK
                k = torch.einsum("htd,ht->htd", s["k"][slot, :, :n].double(), s["k_scale"][slot].double()[:, block])
                v = torch.einsum("htd,ht->htd", s["v"][slot, :, :n].double(), s["v_scale"][slot].double()[:, block])
                weight = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / 8.0, -1)
                o = torch.einsum("hgt,htd->hgd", weight, v)
            outs.append(o.reshape(-1))
        return torch.stack(outs)
    if c["op"] == "store":
        # the int8 values are whole numbers; the scales have an exact value
        d = c["heads"] * HEAD
        begin = list(range(c["runs"] + 1)) if s["row_begin"] is None else s["row_begin"].tolist()
        scales = []
        for new, scale in ((s["new_k"], s["k_scale"].double()), (s["new_v"], s["v_scale"].double())):
            for r, (slot, p0) in enumerate(zip(s["slots"].tolist(), s["positions"].tolist())):
                rows = new[begin[r]:begin[r + 1]].double().abs().view(-1, c["heads"], HEAD).amax(-1)   # [n, heads]
                p1 = p0 + rows.shape[0]
                for b in range(p0 // BLOCK, (p1 - 1) // BLOCK + 1):
                    lo, hi = max(p0, BLOCK * b), min(p1, BLOCK * (b + 1))
                    mine = rows[lo - p0:hi - p0].amax(0) / 127
                    scale[slot, :, b] = mine if lo == BLOCK * b else torch.maximum(scale[slot, :, b], mine)
            scales.append(scale)
        return None, None, scales[0], scales[1]
    n, k, grp = c["n"], c["k"], c["group"]
    out = torch.zeros(c["rows"], n, dtype=torch.float64, device=s["x"].device)
    low, high = s["w"] & 15, s["w"] >> 4
    nibble = torch.stack([low, high], -1).view(n, -1, 8)       # in the order of a word's bits
    for j in range(8):                                         # bits 4 j of word 4 t + i: element 32 i + 8 t + 2 (j % 4) + j // 4
        at = torch.arange(nibble.shape[1], device=out.device)
        element = at // 16 * SEGMENT + 32 * (at % 4) + 8 * (at % 16 // 4) + 2 * (j % 4) + j // 4
        at, element = at[element < k], element[element < k]
        w = (nibble[:, at, j].double() - 8) * s["w_scale"][:, element // grp].double()
        out += s["x"][:, element].double() @ w.T
    out += s["bias"].double()
    return out if s["residual"] is None else out + s["residual"].double()
