"""The low-bit operators on the GPU against their definitions in 64 bits (lowbit_ref.py).

Tolerances, from the arithmetic that the interface promises (u = 2^-24, half a step of fp32):
  store      none: values and scales are equal.
  attention  a score is a 64-term fp32 sum: off by at most 70 u scale max|q| sum|k| (that also covers a query held in 23 or
             more bits of its head's largest value); the exponential and the weight's fixed point add 2^-21, the sums of n
             weights n 2^-23, all relative to the largest |v|; a bf16 result is rounded once, 2^-8 of its value.
  linear     an fp32 sum of K products in any order: (K + 8) u sum|x w|, and as much of the bias and the residual; bf16 rows
             are promised to 2^-46 of their largest value, sum|w| of that.
"""
import numpy as np
import pytest
import torch

import lowbit_ref as ref
from whisperdrz_b200.capi import WdzError
from whisperdrz_b200.dims import ModelDimensions
from whisperdrz_b200.lowbit import PackedLinear, QCache, pack_linear, pack_nibbles
from whisperdrz_b200.weights import init_state_dict

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def eng():
    from whisperdrz_b200.engine import Engine
    dims = ModelDimensions.from_name("test-tiny")
    e = Engine(dims, init_state_dict(dims, 0), dtype=F32, n_slots=1, max_clips=1, max_rows=1)
    yield e
    e.close()


def _filled(slots, heads, blocks, seed=0, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randint(-127, 128, (slots, heads, 64 * blocks, 64), generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2))
    ks, vs = (0.02 * torch.exp(spread * torch.randn(slots, heads, blocks, generator=g)) for _ in range(2))
    return k, v, ks, vs


def _cuda_cache(parts):
    return QCache(*(t.cuda() for t in parts))


# ---------------------------------------------------------------------- store
def _check_store(eng, parts, new_k, new_v, slots, positions, row_begin=None, max_run=None, device_index=True):
    want = [t.clone().numpy() for t in parts]
    ref.store(want[0], want[2], new_k.float().numpy(), slots, positions, row_begin)
    ref.store(want[1], want[3], new_v.float().numpy(), slots, positions, row_begin)
    c = _cuda_cache(parts)

    def index(x):
        return None if x is None else torch.tensor(x, dtype=torch.int32).cuda() if device_index else x

    eng.qcache_store(c, new_k.cuda(), new_v.cuda(), index(slots), index(positions), row_begin=index(row_begin), max_run=max_run)
    for got, w, name in zip((c.k, c.v, c.k_scale, c.v_scale), want, ("k", "v", "k_scale", "v_scale")):
        assert np.array_equal(got.cpu().numpy(), w, equal_nan=True), name
    return c


RUNS = {   # slots, positions, lengths
    "one token": ([1], [0], [1]),
    "last token": ([0], [255], [1]),
    "whole slot": ([2], [0], [256]),
    "across blocks": ([3, 1], [60, 100], [9, 130]),
    "into a block's end": ([0, 2, 3], [1, 63, 191], [63, 2, 65]),
    "empty and skipped": ([0, -1, 2, 7, 1], [5, 0, 0, 3, 250], [0, 4, 64, 5, 6]),
    "many": ([4, 3, 2, 1, 0], [0, 10, 64, 127, 200], [200, 37, 1, 128, 56]),
}


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [1, 3, 20])
@pytest.mark.parametrize("name", RUNS)
def test_store_runs(eng, name, heads, dtype):
    slots, positions, lens = RUNS[name]
    begin = [0] + np.cumsum(lens).tolist()
    g = torch.Generator().manual_seed(len(name) + heads)
    loud = torch.exp(torch.randn(heads * 64, generator=g))
    k, v = ((torch.randn(max(begin[-1], 1), heads * 64, generator=g) * loud).to(dtype) for _ in range(2))
    for hint in (None, 1, max(lens)):
        _check_store(eng, _filled(5, heads, 4, seed=heads), k, v, slots, positions, begin, max_run=hint)
    _check_store(eng, _filled(5, heads, 4, seed=heads), k, v, slots, positions, begin, device_index=False)
    eng.device_status()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 33, 384])
def test_store_steps(eng, rows, dtype):
    g = torch.Generator().manual_seed(rows)
    product = torch.randn(rows, 3 * 128, generator=g).to(dtype) * 3      # K and V as columns of a fused product
    slots = torch.randperm(rows + 2, generator=g)[:rows].tolist()
    positions = torch.randint(0, 128, (rows,), generator=g).tolist()
    k, v = product[:, 128:256], product[:, 256:]
    _check_store(eng, _filled(rows + 2, 2, 2, seed=rows), k, v, slots, positions)
    eng.device_status()


@pytest.mark.parametrize("heads", [1, 21, 45])
def test_store_steps_of_any_head_count(eng, heads):
    """More heads than a block takes at a time, K and V at different distances, scales that grow in some heads only."""
    g = torch.Generator().manual_seed(heads)
    d = heads * 64
    k = torch.randn(3, d + 64, generator=g)[:, :d]
    v = torch.randn(3, 2 * d, generator=g)[:, d:]
    k[0] *= 30
    v[1, ::2] *= 30
    _check_store(eng, _filled(4, heads, 2, seed=heads), k, v, [3, 0, 2], [63, 100, 64])
    _check_store(eng, _filled(4, heads, 2, seed=heads), k, v, [3, 0, 2], [63, 100, 64], [0, 1, 2, 3])   # as runs
    eng.device_status()


def test_store_token_by_token_fills_a_slot_like_the_definition(eng):
    parts = [t * 0 for t in _filled(2, 2, 3)]
    want = [t.clone().numpy() for t in parts]
    c = _cuda_cache(parts)
    g = torch.Generator().manual_seed(8)
    for t in range(130):
        k, v = (torch.randn(1, 128, generator=g) * (1 + t % 7) for _ in range(2))
        eng.qcache_store(c, k.cuda(), v.cuda(), [1], [t])
        ref.store(want[0], want[2], k.numpy(), [1], [t])
        ref.store(want[1], want[3], v.numpy(), [1], [t])
    for got, w in zip((c.k, c.v, c.k_scale, c.v_scale), want):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("start", [0, 3])
def test_store_extreme_values(eng, dtype, start):
    """Zeros, the smallest and largest numbers, ties, infinities and NaN; what is not finite is reported."""
    rows = torch.zeros(70, 128)
    g = torch.Generator().manual_seed(1)
    rows[:] = torch.randn(70, 128, generator=g)
    rows[5], rows[6, ::2], rows[7, ::3] = 0.0, 127.0, 63.5
    rows[64:, :64] = 0.0                 # a block of zeros in head 0
    rows[64:, 64:] *= 1e-38              # and of numbers below 2^-117 in head 1
    k, v = rows.to(dtype), (rows * 2.5e36).to(dtype)
    parts = _filled(1, 2, 2)
    _check_store(eng, parts, k, v, [0], [start], [0, 70])
    eng.device_status()
    k[1, 0], k[2, 70], v[3, 5], v[66, 100] = float("inf"), float("-inf"), float("nan"), float("nan")
    _check_store(eng, parts, k, v, [0], [start], [0, 70])
    with pytest.raises(WdzError) as err:
        eng.device_status()
    assert "WDZ_ENAN" in str(err.value)
    eng.device_status()                  # reported once


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_store_many_runs(eng, dtype):
    """Enough units that each belongs to one warp: uneven runs that continue their slots, scales that grow, odd values."""
    g = torch.Generator().manual_seed(11)
    runs, heads, blocks = 50, 20, 5
    lens = torch.randint(1, 201, (runs,), generator=g).tolist()
    positions = [int(torch.randint(0, 64 * blocks - n + 1, (1,), generator=g)) for n in lens]
    begin = [0] + np.cumsum(lens).tolist()
    k, v = ((torch.randn(begin[-1], heads * 64, generator=g) * 4).to(dtype) for _ in range(2))
    slots = torch.randperm(runs + 1, generator=g)[:runs].tolist()
    _check_store(eng, _filled(runs + 1, heads, blocks, seed=5), k, v, slots, positions, begin, max_run=200)
    eng.device_status()
    k[begin[3], 70], v[begin[20] + 1, 1279], v[begin[30], 0] = float("nan"), float("inf"), float("-inf")
    v[begin[40]:begin[41]] = 0
    _check_store(eng, _filled(runs + 1, heads, blocks, seed=5), k, v, slots, positions, begin, max_run=200)
    with pytest.raises(WdzError):
        eng.device_status()


def test_store_reports_runs_that_it_cannot_place(eng):
    """Positions and rows outside, a slot named twice: the run is left out, its neighbours are stored."""
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(12, 128, generator=g)
    parts = _filled(5, 2, 1)
    cases = [([0, 1], [0, 62], [0, 3, 6], [0]), ([0, 1], [0, -1], [0, 3, 6], [0]), ([0, 1], [0, 64], [0, 3, 6], [0]),
             ([0, 1], [0, 0], [0, 3, 13], [0]), ([0, 1], [0, 0], [-1, 3, 6], [1]), ([2, 1, 2], [0, 0, 9], [0, 3, 6, 9], [1, 2]),
             ([0, 1, 2], [2 ** 31 - 1, 0, 0], [0, 3, 6, 9], [1, 2])]
    for slots, positions, begin, good in cases:
        want = [t.clone().numpy() for t in parts]
        for w, s in ((want[0], want[2]), (want[1], want[3])):
            for i in good:
                ref.store(w, s, rows[begin[i]:begin[i + 1]].numpy(), [slots[i]], [positions[i]], [0, begin[i + 1] - begin[i]])
        c = _cuda_cache(parts)
        put = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
        eng.qcache_store(c, rows.cuda(), rows.cuda(), put(slots), put(positions), row_begin=put(begin))
        for got, w in zip((c.k, c.v, c.k_scale, c.v_scale), want):
            assert np.array_equal(got.cpu().numpy(), w), (slots, positions, begin)
        with pytest.raises(WdzError) as err:
            eng.device_status()
        assert "WDZ_EINVAL" in str(err.value)


def test_store_into_a_strided_layer_leaves_the_others(eng):
    full = torch.randint(-127, 128, (3, 4, 2, 128, 64), dtype=torch.int8).cuda()
    scale = torch.rand(3, 4, 2, 2).cuda()
    fk, fv, sk, sv = full.clone(), full.clone(), scale.clone(), scale.clone()
    c = QCache(fk[:, 2], fv[:, 2], sk[:, 2], sv[:, 2])
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(70, 128, generator=g), torch.randn(70, 128, generator=g)
    want = [t[:, 2].cpu().numpy().copy() for t in (full, full, scale, scale)]
    ref.store(want[0], want[2], k.numpy(), [2], [30], [0, 70])
    ref.store(want[1], want[3], v.numpy(), [2], [30], [0, 70])
    eng.qcache_store(c, k.cuda(), v.cuda(), [2], [30], row_begin=[0, 70])
    for got, w, was in zip((fk, fv, sk, sv), want, (full, full, scale, scale)):
        assert np.array_equal(got[:, 2].cpu().numpy(), w)
        rest = [0, 1, 3]
        assert torch.equal(got[:, rest], was[:, rest])


# ------------------------------------------------------------------ attention
def _check_attend(eng, parts, q, slots, lens, scale=0.125, out_dtype=F32, out=None, cache=None):
    arrays = [t.numpy() for t in parts]
    want, weight, top = ref.attend(q.float().numpy(), *arrays, slots, lens, scale)
    c = cache or _cuda_cache(parts)
    put = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = eng.qcache_attention(q.cuda(), c, put(slots), put(lens), scale=scale, out_dtype=out_dtype, out=out)
    assert got.dtype == out_dtype and tuple(got.shape) == tuple(want.shape)
    g = got.double().cpu().numpy()
    n = np.minimum(np.maximum(np.asarray(lens, dtype=np.float64), 0), parts[0].shape[2]).reshape(-1, 1, 1)
    tol = top * (2 * 70 * U * weight + 2.0 ** -21 + n * 2.0 ** -23)
    tol = np.repeat(tol.reshape(len(slots), -1), 64, axis=1) + (2.0 ** -8 if out_dtype == BF16 else U) * np.abs(want)
    seen = ~np.isnan(want)
    assert (np.abs(g - want)[seen] <= tol[seen]).all(), float((np.abs(g - want) / np.maximum(tol, 1e-30))[seen].max())
    norm = np.linalg.norm(want[seen])
    if norm:
        assert np.linalg.norm((g - want)[seen]) <= (2.0 ** -8 if out_dtype == BF16 else 1e-5) * norm
    if out is None:
        assert (g[~seen] == 0).all()
    return got


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("heads", [1, 4, 20])
def test_attention_lengths(eng, heads, group):
    lens = [0, 1, 2, 15, 16, 31, 33, 63, 64, 65, 127, 128, 129, 191, 192, 250, 256]
    rows = len(lens)
    parts = _filled(rows, heads, 4, seed=group)
    g = torch.Generator().manual_seed(heads)
    q = torch.randn(rows, heads * group * 64, generator=g) * 0.3
    slots = torch.randperm(rows, generator=g).tolist()
    _check_attend(eng, parts, q, slots, lens)


@pytest.mark.parametrize("q_dtype", [F32, BF16], ids=["qf32", "qbf16"])
@pytest.mark.parametrize("out_dtype", [F32, BF16], ids=["of32", "obf16"])
@pytest.mark.parametrize("rows,heads,group,tokens", [(1, 20, 1, 1500), (1, 2, 8, 2049), (3, 1, 1, 5000), (7, 3, 2, 700), (64, 4, 1, 448)])
def test_attention_types_and_shapes(eng, rows, heads, group, tokens, q_dtype, out_dtype):
    parts = _filled(rows, heads, (tokens + 63) // 64, seed=rows)
    g = torch.Generator().manual_seed(tokens)
    q = (torch.randn(rows, heads * group * 64, generator=g) * 0.3).to(q_dtype)
    lens = [1 + (tokens - 1) * (rows - i) // rows for i in range(rows)]
    _check_attend(eng, parts, q, list(range(rows))[::-1], lens, out_dtype=out_dtype)


def test_attention_of_peaked_and_flat_rows(eng):
    """Scores far apart (one weight is 1, the rest 0, wherever the maximum comes) and all alike."""
    parts = _filled(6, 2, 3, seed=9)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(6, 128, generator=g)
    q[0] *= 60
    q[1] *= 1e-6
    q[2] = 0
    q[3, ::7] *= 300
    q[4] *= 1e-34
    q[5, 3] = 3e30
    for scale in (0.125, 1.0, 0.0, 1e-30):
        n = 6 if scale < 0.1 else 5          # the query of 3e30 only where its scores stay in range
        _check_attend(eng, parts, q[:n], [0, 1, 2, 3, 4, 5][:n], [192, 192, 100, 192, 5, 64][:n], scale=scale)


def test_attention_rows_of_one_slot_and_clamped_lengths(eng):
    parts = _filled(3, 4, 2, seed=5)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(9, 256, generator=g)
    _check_attend(eng, parts, q, [1, 1, 1, 0, 0, 2, 2, 2, 2], [1, 2, 3, 128, 128, -5, 129, 2 ** 31 - 1, -2 ** 31])


@pytest.mark.parametrize("out_dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_leaves_skipped_rows_as_they_were(eng, out_dtype):
    parts = _filled(3, 2, 1, seed=5)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(5, 128, generator=g)
    slots, lens = [0, -1, 2, 3, 2 ** 31 - 1], [7, 7, 0, 9, 1]
    wide = torch.full((8, 256), 7.0, dtype=out_dtype, device="cuda")
    _check_attend(eng, parts, q, slots, lens, out_dtype=out_dtype, out=wide[:5, 64:192])
    assert (wide[[1, 3, 4]] == 7).all() and (wide[5:] == 7).all() and (wide[:, :64] == 7).all() and (wide[:, 192:] == 7).all()
    _check_attend(eng, parts, q, slots, lens, out_dtype=out_dtype)       # a fresh output has zeros there
    assert eng.qcache_attention(q[:0].cuda(), _cuda_cache(parts), [], []).shape == (0, 128)


def test_attention_of_strided_rows_and_layers(eng):
    parts = _filled(4, 2, 2, seed=1)
    many = [t.unsqueeze(1).repeat_interleave(3, 1).cuda() for t in parts]
    for t in many:
        t[:, 0], t[:, 2] = 0, 1
    cache = QCache(*(t[:, 1] for t in many))
    g = torch.Generator().manual_seed(6)
    product = torch.randn(4, 3 * 128, generator=g)
    _check_attend(eng, parts, product[:, 128:256], [3, 2, 1, 0], [128, 50, 64, 65], cache=cache)
    odd = torch.randn(4, 131, generator=g)[:, 1:129]          # rows that the kernel cannot take as they lie
    _check_attend(eng, parts, odd, [3, 2, 1, 0], [128, 50, 64, 65], cache=cache)


def test_attention_past_32_bits(eng):
    """Slots more than 2^31 values apart, and a slot of more than 2^31 values."""
    step = 2 ** 31 + 4096
    parts = _filled(2, 1, 1, seed=1)
    base = [torch.empty(step + 4096, dtype=torch.int8, device="cuda") for _ in range(2)]
    k, v = (b.as_strided((2, 1, 64, 64), (step, 4096, 64, 1)) for b in base)
    k.copy_(parts[0]); v.copy_(parts[1])
    cache = QCache(k, v, parts[2].cuda(), parts[3].cuda())
    q = torch.randn(2, 64, generator=torch.Generator().manual_seed(0))
    _check_attend(eng, parts, q, [1, 0], [64, 33], cache=cache)
    del base, k, v, cache
    heads = 2                                                   # head 1 of the slot starts past 2^31
    blocks = 2 ** 31 // 4096 + 2
    k = torch.zeros(1, heads, 64 * blocks, 64, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    scale = torch.zeros(1, heads, blocks, device="cuda")
    one = _filled(1, heads, 2, seed=2)
    k[:, :, :128], v[:, :, :128] = one[0].cuda(), one[1].cuda()
    ks, vs = scale.clone(), scale.clone()
    ks[:, :, :2], vs[:, :, :2] = one[2].cuda(), one[3].cuda()
    q = torch.randn(1, 128, generator=torch.Generator().manual_seed(0))
    _check_attend(eng, one, q, [0], [100], cache=QCache(k, v, ks, vs))
    # and its last tokens: everything before them has value 0 and, with a zero score, weight 1 each
    c = QCache(k, v, ks, vs)
    last = 64 * blocks
    rows = torch.randn(3, 128, generator=torch.Generator().manual_seed(1)).cuda()
    k.zero_(); v.zero_()
    eng.qcache_store(c, rows * 0, rows, [0], [last - 3], row_begin=[0, 3])
    got = eng.qcache_attention(torch.zeros(1, 128, device="cuda"), c, [0], [last], out_dtype=F32)
    want = ref.dequant(v[0, :, -64:].cpu().numpy(), vs[0, :, -1:].cpu().numpy()).sum(1).reshape(-1) / last
    # n weights of 1 in fp32 partial sums: n 2^-23 as above, though the sums are of whole numbers
    assert np.abs(got[0].double().cpu().numpy() - want).max() <= 2.0 ** -20 * np.abs(want).max()
    eng.device_status()


def test_attention_ignores_what_lies_behind_a_row(eng):
    """NaN scales of blocks behind the length, full-scale bytes behind it inside the last block."""
    parts = _filled(2, 2, 4, seed=4)
    parts[2][:, :, 2:] = float("nan")
    parts[3][:, :, 2:] = float("inf")
    clean = [t.clone() for t in parts]
    for t in clean[:2]:
        t[:, :, 70:] = 0
    for t in clean[2:]:
        t[:, :, 2:] = 0
    for t in parts[:2]:
        t[:, :, 70:] = -128
    q = torch.randn(2, 128, generator=torch.Generator().manual_seed(0))
    a = _check_attend(eng, clean, q, [0, 1], [70, 64])
    b = eng.qcache_attention(q.cuda(), _cuda_cache(parts), [0, 1], [70, 64], out_dtype=F32)
    assert torch.equal(a, b)


@pytest.mark.parametrize("what", ["q nan", "q inf", "k scale", "v scale"])
def test_attention_carries_nan_to_its_own_row_only(eng, what):
    parts = _filled(3, 2, 8, seed=4)
    q = torch.randn(3, 128, generator=torch.Generator().manual_seed(0))
    good = eng.qcache_attention(q.cuda(), _cuda_cache(parts), [0, 1, 2], [500, 500, 500], out_dtype=F32)
    if what == "q nan":
        q[1, 70] = float("nan")
    elif what == "q inf":
        q[1, 70] = float("inf")
    else:
        parts[2 if what == "k scale" else 3][1, 1, 5] = float("nan")
    got = eng.qcache_attention(q.cuda(), _cuda_cache(parts), [0, 1, 2], [500, 500, 500], out_dtype=F32)
    assert got[1, 64:].isnan().all()
    assert torch.equal(got[[0, 2]], good[[0, 2]]) and torch.equal(got[1, :64], good[1, :64])


def test_attention_gives_the_same_bits_every_time(eng):
    parts = _filled(3, 20, 24, seed=4)
    c = _cuda_cache(parts)
    q = torch.randn(3, 1280, generator=torch.Generator().manual_seed(0)).cuda()
    first = eng.qcache_attention(q, c, [0, 1, 2], [1500, 900, 64], out_dtype=F32)
    for _ in range(5):
        assert torch.equal(first, eng.qcache_attention(q, c, [0, 1, 2], [1500, 900, 64], out_dtype=F32))


# --------------------------------------------------------------------- linear
def _packed(n, k, group, seed, bias=None):
    g = torch.Generator().manual_seed(seed)
    kp = (k + 127) // 128 * 128
    q = torch.randint(-8, 8, (n, kp), generator=g)
    q[:, k:] = 0
    scale = (0.02 * torch.exp(0.5 * torch.randn(n, kp // group, generator=g))).bfloat16()
    b = None if bias is None else torch.randn(n, generator=g).to(bias)
    w = (q.numpy() * np.repeat(scale.float().numpy().astype(np.float64), group, axis=1))[:, :k]
    return PackedLinear(pack_nibbles(q).cuda(), scale.cuda(), k, group, None if b is None else b.cuda()), w, b


def _check_linear(eng, x, packed, w, b, residual=None, out=None):
    x64 = x.float().cpu().numpy().astype(np.float64)
    want, size = x64 @ w.T, np.abs(x64) @ np.abs(w).T
    for extra in (b, residual):
        if extra is not None:
            e = extra.float().cpu().numpy().astype(np.float64)
            want, size = want + e, size + np.abs(e)
    got = eng.linear_rows_packed(x.cuda(), packed, residual=residual, out=out)
    g = got.double().cpu().numpy()
    tol = (x.shape[1] + 8) * U * size
    if x.dtype == BF16:   # one or two rows are held in whole numbers of 2^(e - 45), e the exponent of the row's largest value:
        tol = tol + 2.0 ** -46 * np.abs(x64).max(1, keepdims=True, initial=0) * np.abs(w).sum(1)   # half a unit each, 2^-46 of it at most
    assert got.dtype == F32 and g.shape == want.shape
    assert (np.abs(g - want) <= tol).all(), float((np.abs(g - want) / np.maximum(tol, 1e-30)).max())
    assert np.linalg.norm(g - want) <= 1e-5 * max(np.linalg.norm(want), 1e-30)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1280, 1280), (1, 17, 130), (2, 64, 64), (3, 100, 1), (5, 33, 1237), (8, 256, 5120), (9, 31, 640),
                                   (16, 160, 256), (17, 48, 384), (33, 16, 136), (70, 15, 127), (2, 40, 9000), (1, 16, 20000),
                                   (4, 24, 8192), (5, 24, 14000), (12, 17, 9001), (3, 40, 5003)])
def test_linear_shapes(eng, m, n, k, group, dtype):
    packed, w, b = _packed(n, k, group, seed=m + n, bias=dtype if m % 2 else None)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k)).to(dtype)
    _check_linear(eng, x, packed, w, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 2, 4, 9, 16, 19])
def test_linear_of_many_features(eng, m, dtype):
    """Enough features that an SM has several blocks, and more inputs than one pass of theirs holds; the reference in 64 bits
    on the device."""
    n, k, group = 19001, 4250, 64
    g = torch.Generator(device="cuda").manual_seed(m)
    kp = (k + 127) // 128 * 128
    q = torch.randint(-8, 8, (n, kp), generator=g, device="cuda", dtype=torch.int32)
    q[:, k:] = 0
    scale = (0.02 * torch.exp(0.5 * torch.randn(n, kp // group, generator=g, device="cuda"))).bfloat16()
    w = (q.double().view(n, -1, group) * scale.double()[..., None]).view(n, kp)[:, :k]
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    r = torch.randn(m, n, generator=g, device="cuda")
    got = eng.linear_rows_packed(x, PackedLinear(pack_nibbles(q), scale, k, group), residual=r).double()
    want = x.double() @ w.T + r.double()
    tol = (k + 8) * U * (x.double().abs() @ w.abs().T + r.double().abs()) + 2.0 ** -46 * x.double().abs().amax(1, True) * w.abs().sum(1)
    assert bool(((got - want).abs() <= tol).all())
    assert float((got - want).norm() / want.norm()) <= 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 2, 4, 7, 16])
def test_linear_residual_and_bias(eng, m, dtype):
    packed, w, b = _packed(200, 512, 64, seed=m, bias=BF16 if dtype == F32 else F32)   # a bias of the other type
    x = torch.randn(m, 512, generator=torch.Generator().manual_seed(m)).to(dtype)
    b = b.to(dtype)     # a bias is rounded to the rows' type
    r = torch.randn(m, 200, generator=torch.Generator().manual_seed(m + 1)).cuda()
    was = r.clone()
    got = _check_linear(eng, x, packed, w, b, residual=r)
    assert torch.equal(r, was)
    y = r.clone()
    assert eng.linear_rows_packed(x.cuda(), packed, residual=y, out=y) is y      # into the residual stream, in place
    assert torch.equal(y, got)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("k", [256, 251])
def test_linear_rows_at_any_alignment(eng, k, dtype):
    packed, w, b = _packed(40, k, 32, seed=1)
    wide = torch.randn(6, k + 5, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    for first in range(4):
        _check_linear(eng, wide[:, first:first + k], packed, w, b)
    _check_linear(eng, wide[::2, :k], packed, w, b)
    flipped = torch.randn(k, 6, generator=torch.Generator().manual_seed(4)).to(dtype).cuda().T
    _check_linear(eng, flipped, packed, w, b)
    assert eng.linear_rows_packed(wide[:0, :k], packed).shape == (0, 40)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_linear_range_and_nan(eng, dtype):
    """Rows of very different sizes, rows of zeros, and NaN and infinity that stay in their row."""
    packed, w, b = _packed(64, 384, 64, seed=5)
    x = torch.randn(8, 384, generator=torch.Generator().manual_seed(3))
    x[6] *= 1e-33
    x[7] *= 1e-30
    x[7, 5] = 2e30
    x[0] *= 1e-20
    x[1] *= 1e20
    x[2] = 0
    x[3, 7] *= 1e6                       # one loud channel
    x = x.to(dtype)
    got = _check_linear(eng, x[:3], packed, w, b), _check_linear(eng, x[3:], packed, w, b)
    both = eng.linear_rows_packed(x.cuda(), packed)
    assert torch.equal(both[:3], got[0]) and torch.equal(both[3:], got[1])
    for i in range(8):                   # one and two rows go another way
        _check_linear(eng, x[i:i + 1], packed, w, b)
        if i < 7:
            _check_linear(eng, x[i:i + 2], packed, w, b)
    x[1, 100], x[4, 0] = float("nan"), float("inf")
    bad = eng.linear_rows_packed(x.cuda(), packed)
    assert bad[1].isnan().all()
    assert (~bad[4].isfinite()).all()
    keep = [0, 2, 3, 5, 6, 7]
    assert torch.equal(bad[keep], both[keep])
    for one, other in ((1, 0), (4, 5)):
        pair = eng.linear_rows_packed(x[[one, other]].cuda(), packed)
        assert (~pair[0].isfinite()).all() and torch.equal(pair[1], eng.linear_rows_packed(x[[other]].cuda(), packed)[0])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("k", [384, 381, 9001])
@pytest.mark.parametrize("m", [1, 2, 3, 9])
def test_linear_of_infinities_is_what_the_formula_gives(eng, m, k, dtype):
    """One infinity times a weight is an infinity of its sign, times a weight of zero NaN; two of them may cancel to NaN."""
    packed, w, b = _packed(70, k, 64, seed=m, bias=dtype)
    inf = float("inf")
    for places in ({5: inf}, {k - 1: -inf}, {0: inf, k - 1: inf}, {k // 2: -inf, 7: inf}, {k - 2: float("nan")}):
        x = torch.randn(m, k, generator=torch.Generator().manual_seed(k)).to(dtype)
        for at, v in places.items():
            x[m - 1, at] = v
        got = eng.linear_rows_packed(x.cuda(), packed).double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            want = (x[m - 1].double().numpy() * w).sum(1)
        assert not np.isfinite(want).any()
        np.testing.assert_array_equal(got[m - 1], want)   # NaN where NaN is wanted, and the same infinities
        assert np.isfinite(got[:m - 1]).all()


def test_pack_linear_on_the_device_is_the_same(eng):
    w = torch.randn(40, 333, generator=torch.Generator().manual_seed(0))
    a, b = pack_linear(w, 64), pack_linear(w.cuda(), 64)
    assert torch.equal(a.weight, b.weight.cpu()) and torch.equal(a.scale, b.scale.cpu())


def test_linear_from_packed_weights_is_near_the_weights(eng):
    w = torch.randn(96, 300, generator=torch.Generator().manual_seed(0)) / 17
    p = pack_linear(w, 32, bias=torch.ones(96))
    q = ref.unpack(p.weight.numpy(), 384)[:, :300]
    dense = q * np.repeat(p.scale.float().numpy().astype(np.float64), 32, axis=1)[:, :300]
    on = PackedLinear(p.weight.cuda(), p.scale.cuda(), 300, 32, p.bias.cuda())
    x = torch.randn(4, 300, generator=torch.Generator().manual_seed(1))
    _check_linear(eng, x, on, dense, p.bias)


# ------------------------------------------------- as a decode step uses them
def _step(eng, cache, qkv, out, x, slots, positions, lens):
    """x + out(attention(qkv(x))): the cached self-attention block of a decoder layer."""
    heads = cache.n_heads
    d = heads * 64
    p = eng.linear_rows_packed(x.to(BF16), qkv)
    eng.qcache_store(cache, p[:, d:2 * d], p[:, 2 * d:], slots, positions)
    a = eng.qcache_attention(p[:, :d], cache, slots, lens, out_dtype=BF16)
    return eng.linear_rows_packed(a, out, residual=x)


def test_decode_steps_run_together(eng):
    """Ten steps of a layer's self-attention for three slots of different depth against the same steps in 64 bits, each
    fed the kernels' own rows so that one step's rounding does not decide the next one's."""
    heads, d = 4, 256
    qkv, wq, bq = _packed(3 * d, d, 64, seed=1, bias=BF16)
    out, wo, bo = _packed(d, d, 32, seed=2, bias=BF16)
    parts = _filled(4, heads, 2, seed=3)
    cache = _cuda_cache(parts)
    host = [t.clone().numpy() for t in parts]
    slots, positions = [2, 0, 3], [0, 60, 101]
    g = torch.Generator().manual_seed(4)
    put = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    for step in range(10):
        x = torch.randn(3, d, generator=g)
        pos = [p + step for p in positions]
        y = _step(eng, cache, qkv, out, x.cuda(), put(slots), put(pos), put([p + 1 for p in pos]))
        p = eng.linear_rows_packed(x.cuda().to(BF16), qkv)
        _check_linear(eng, x.to(BF16), qkv, wq, bq)
        p = p.cpu().numpy()
        ref.store(host[0], host[2], p[:, d:2 * d], slots, pos)
        ref.store(host[1], host[3], p[:, 2 * d:], slots, pos)
        for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), host):
            assert np.array_equal(got.cpu().numpy(), w)
        a, _, _ = ref.attend(p[:, :d], *host, slots, [q + 1 for q in pos], 0.125)
        want = x.numpy().astype(np.float64) + a @ wo.T + bo.float().numpy()
        # the attention's bf16 rounding, 2^-8 of each value, through the product; all else is fp32
        tol = 1.01 * 2.0 ** -8 * (np.abs(a) @ np.abs(wo).T) + 1e-4 * np.abs(want).max()
        assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("rows,heads,group,tokens", [(1, 20, 1, 1500), (2, 4, 4, 20000), (40, 20, 1, 448)])
def test_attention_captured(eng, rows, heads, group, tokens):
    """Each way that a launch is cut (clusters, parts with scratch of the graph's own, a CTA a row), replayed with other
    lengths and other queries while an eager call runs beside it."""
    cache = _cuda_cache(_filled(rows, heads, (tokens + 63) // 64, seed=1))
    g = torch.Generator().manual_seed(2)
    q = torch.randn(rows, heads * group * 64, generator=g).cuda()
    slots = torch.arange(rows, dtype=torch.int32).cuda()
    lens = torch.full((rows,), tokens, dtype=torch.int32).cuda()
    eng.qcache_attention(q, cache, slots, lens, out_dtype=F32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = eng.qcache_attention(q, cache, slots, lens, out_dtype=F32)
    for n in (tokens, 1, tokens // 2, 0, tokens - 1):
        lens.fill_(n)
        q.copy_(torch.randn(q.shape, generator=g))
        want = eng.qcache_attention(q, cache, slots, lens, out_dtype=F32).clone()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graph.replay()
        beside = eng.qcache_attention(q, cache, slots, lens, out_dtype=F32)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(beside, want)
        if n == 0:
            assert (out == 0).all()
    eng.device_status()


def test_attention_in_place_of_its_queries(eng):
    parts = _filled(3, 4, 3, seed=1)
    q = torch.randn(3, 256, generator=torch.Generator().manual_seed(3))
    c = _cuda_cache(parts)
    want = eng.qcache_attention(q.cuda(), c, [2, 0, 1], [190, 64, 0], out_dtype=F32)
    both = q.cuda()
    assert eng.qcache_attention(both, c, [2, 0, 1], [190, 64, 0], out=both) is both
    assert torch.equal(both, want)


def test_operators_of_a_bf16_engine_without_overlapped_launches():
    """The other kind of engine, its default output type, and its launches without programmatic dependence."""
    from whisperdrz_b200 import capi
    from whisperdrz_b200.engine import Engine
    dims = ModelDimensions.from_name("test-small")
    e = Engine(dims, init_state_dict(dims, 0), dtype=BF16, n_slots=1, max_clips=1, max_rows=1, flags=capi.FLAG_NO_PDL)
    try:
        parts = _filled(3, 4, 2, seed=1)
        c = e.qcache(n_slots=3, n_tokens=100, n_heads=4)
        for t, p in zip((c.k, c.v, c.k_scale, c.v_scale), parts):
            t.copy_(p)
        q = torch.randn(3, 256, generator=torch.Generator().manual_seed(3))
        before = e.launch_count()
        got = e.qcache_attention(q.cuda(), c, [2, 0, 1], [100, 64, 1])
        assert got.dtype == BF16 and e.launch_count() == before + 1
        _check_attend(e, parts, q, [2, 0, 1], [100, 64, 1], out_dtype=BF16)
        _check_store(e, parts, q, q, [0, 2, 1], [3, 64, 127])
        packed, w, b = _packed(40, 300, 32, seed=1)
        _check_linear(e, q.new_ones(2, 300).to(BF16), packed, w, b)
        default = e.qcache()
        assert (default.n_slots, default.n_heads, default.n_tokens) == (1, dims.n_text_head, 1536)
        e.device_status()
    finally:
        e.close()


def test_calls_refuse_tensors_elsewhere(eng):
    c = _cuda_cache(_filled(2, 2, 1))
    q, i = torch.zeros(2, 128), torch.zeros(2, dtype=torch.int32)
    host = QCache(*_filled(2, 2, 1))
    for call in (lambda: eng.qcache_attention(q, c, i, i), lambda: eng.qcache_attention(q.cuda(), host, i, i),
                 lambda: eng.qcache_attention(q.cuda(), c, i, i, out=torch.zeros(2, 128)),
                 lambda: eng.qcache_store(c, q, q, [0, 1], [0, 0]), lambda: eng.qcache_store(host, q.cuda(), q.cuda(), [0, 1], [0, 0]),
                 lambda: eng.linear_rows_packed(torch.zeros(1, 128), _packed(4, 128, 32, 0)[0]),
                 lambda: eng.linear_rows_packed(torch.zeros(1, 128).cuda(), pack_linear(torch.zeros(4, 128)))):
        with pytest.raises(ValueError):
            call()


def test_steps_in_captured_graphs_and_on_side_streams(eng):
    """Two captured steps over two caches, replayed in turn and on different streams, and eager steps beside them."""
    heads, d = 2, 128
    qkv, _, _ = _packed(3 * d, d, 64, seed=1)
    out, _, _ = _packed(d, d, 32, seed=2)
    put = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    args = []
    for i in range(2):
        cache = _cuda_cache(_filled(3, heads, 2, seed=i))
        x = torch.randn(3, d, generator=torch.Generator().manual_seed(i)).cuda()
        args.append((cache, qkv, out, x, put([0, 2, 1]), put([0, 64, 99 + i]), put([1, 65, 100 + i])))
    want = [_step(eng, *a).clone() for a in args]     # storing the same row again changes nothing
    graphs, outs = [], []
    for a in args:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(eng, *a)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_step(eng, *a))
        graphs.append(gr)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for round_ in range(6):
        for i, gr in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                gr.replay()
        eager = _step(eng, *args[0][:3], args[0][3] * 1.0, *args[0][4:]) if round_ % 3 == 2 else None
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        if eager is not None:
            assert torch.equal(eager, want[0])
    eng.device_status()
