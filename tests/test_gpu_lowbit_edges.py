"""The low-bit operators at the ends of their ranges and on their rarer paths, on the GPU against the definitions in 64 bits
(lowbit_ref.py).  Tolerances are those of test_gpu_lowbit.py unless a test derives its own (u = 2^-24)."""
import numpy as np
import pytest
import torch

import lowbit_ref as ref
from test_gpu_lowbit import BF16, F32, U, _check_attend, _check_store, _cuda_cache, _filled, eng  # noqa: F401
from whisperdrz_b200 import capi
from whisperdrz_b200.capi import WdzError
from whisperdrz_b200.lowbit import PackedLinear, pack_nibbles

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ what is reported
def _misplaced_store(eng):
    c = _cuda_cache(_filled(2, 2, 1))
    rows = torch.zeros(1, 128, device="cuda")
    eng.qcache_store(c, rows, rows, torch.tensor([0], dtype=torch.int32).cuda(), torch.tensor([64], dtype=torch.int32).cuda())


def test_a_store_that_cannot_be_placed_leaves_a_transcription_alone(eng):
    """The decode loop's poll hears of its own kernels only, and what it leaves is told by device_status."""
    _misplaced_store(eng)
    eng.ts_poll()
    eng.decode_status()
    with pytest.raises(WdzError) as err:
        eng.device_status()
    assert "WDZ_EINVAL" in str(err.value)
    eng.device_status()


def test_each_kind_of_report_is_told_and_a_wait_that_ran_out_first(eng):
    """No kernel is made to hang: the words are set as one would leave them (the engine's own, the operators' waits, the
    operators' data)."""
    words = eng.workspace[:24].view(torch.int32).view(3, 2)
    assert (words == 0).all()
    _misplaced_store(eng)
    words[1, 0], words[1, 1] = -7, 2000005
    words[0, 0] = -6
    for name in ("WDZ_ETIMEOUT", "WDZ_ENAN", "WDZ_EINVAL"):
        with pytest.raises(WdzError) as err:
            eng.device_status()
        assert name in str(err.value)
    eng.device_status()
    words[0, 0] = -6
    with pytest.raises(WdzError) as err:
        eng.ts_poll()
    assert "WDZ_ENAN" in str(err.value)
    eng.ts_poll()
    eng.device_status()


# ---------------------------------------------------------------------- store
def test_store_of_a_padded_batch(eng):
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(9, 128, generator=g)
    for device_index in (True, False):
        _check_store(eng, _filled(3, 2, 1), rows[:4], rows[4:8], [2, -1, -1, 0], [5, 0, 0, 9], device_index=device_index)
        _check_store(eng, _filled(3, 2, 1), rows, rows.flip(0), [1, 3, 3, -1, -1], [5, 0, 0, 9, 70], [0, 4, 5, 6, 8, 9], device_index=device_index)
    eng.device_status()


# --------------------------------------------------------------------- linear
def _scaled(n, k, group, seed, scale):
    """Packed weights whose group scales are ``scale`` (a number, or one for each group) times 1 to 2."""
    g = torch.Generator().manual_seed(seed)
    kp = (k + 127) // 128 * 128
    q = torch.randint(-8, 8, (n, kp), generator=g)
    q[:, k:] = 0
    s = ((1 + torch.rand(n, kp // group, generator=g, dtype=torch.float64)) * torch.as_tensor(scale, dtype=torch.float64)).bfloat16()
    w = (q.numpy() * np.repeat(s.double().numpy(), group, axis=1))[:, :k]
    return PackedLinear(pack_nibbles(q).cuda(), s.cuda(), k, group), w


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("x_size,scale", [(1e-20, 1e33), (1e-35, 1e36), (1e-38, 1e37), (1.0, 1e33), (1e-3, 1e34), (30.0, 1e-33),
                                          (1e20, 1e-33), (1e35, 1e-38), (1e3, 1e30), (1e12, 1e-12)])
def test_linear_of_far_scales(eng, x_size, scale, m, group):
    """A result that fits fp32 comes out whatever the sizes of x and the scales; half a step of the smallest fp32 number, 2^-150,
    for each of the sums that a result below 2^-126 passes through: 16 at most here."""
    packed, w = _scaled(40, 300, group, seed=m, scale=scale)
    x = (torch.randn(m, 300, generator=torch.Generator().manual_seed(5)) * x_size).bfloat16()
    x64 = x.double().numpy()
    want, size = x64 @ w.T, np.abs(x64) @ np.abs(w).T
    got = eng.linear_rows_packed(x.cuda(), packed).double().cpu().numpy()
    tol = 308 * U * size + 2.0 ** -46 * np.abs(x64).max(1, keepdims=True) * np.abs(w).sum(1) + 16 * 2.0 ** -150
    assert size.max() < 1e38 and (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m", [1, 2])
def test_linear_of_groups_with_far_scales(eng, m, group):
    """Loud values under a small scale beside quiet ones, 2^-33 of them, under a large one that makes the result."""
    groups = 384 // group
    scale = torch.full((groups,), 1e-18, dtype=torch.float64)
    scale[groups // 3:] = 1e27
    packed, w = _scaled(40, 384, group, seed=m, scale=scale)
    x = torch.randn(m, 384, generator=torch.Generator().manual_seed(5)) * 1e8
    x[:, :128] *= 1e10
    x64 = x.bfloat16().double().numpy()
    got = eng.linear_rows_packed(x.bfloat16().cuda(), packed).double().cpu().numpy()
    # the elementwise bound of a row in whole numbers of 2^-45 of its largest value's power of two: half of one is up to 2^-46 of
    # 4e18, 6e4 on values of 1e8, so no bound relative to the result (1e-5 of its norm, say) follows from it here
    tol = 392 * U * (np.abs(x64) @ np.abs(w).T) + 2.0 ** -46 * np.abs(x64).max(1, keepdims=True) * np.abs(w).sum(1)
    assert (np.abs(got - x64 @ w.T) <= tol).all()


@pytest.mark.parametrize("m", [1, 3, 9])
@pytest.mark.parametrize("size", [1e-32, 1e-34, 1e-36, 1e-38, 1e-41])
def test_linear_of_tiny_f32_rows(eng, size, m):
    """Three bf16 pieces reach down to 2^-133: what a value holds below that is cut off."""
    packed, w = _scaled(40, 300, 64, seed=m, scale=0.02)
    x = torch.randn(m, 300, generator=torch.Generator().manual_seed(5)) * size
    x64 = x.double().numpy()
    want, total = x64 @ w.T, np.abs(x64) @ np.abs(w).T
    got = eng.linear_rows_packed(x.cuda(), packed).double().cpu().numpy()
    tol = 308 * U * total + 2.0 ** -133 * np.abs(w).sum(1) + 308 * 2.0 ** -150
    err = np.abs(got - want)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("m", [1, 2, 5])
def test_linear_of_a_bias_that_is_not_rounded(eng, m):
    """bf16 rows round a bias to their own type; as the residual it is added in f32."""
    packed, w = _scaled(200, 512, 64, seed=m, scale=0.02)
    b = torch.randn(200, generator=torch.Generator().manual_seed(1))
    x = torch.randn(m, 512, generator=torch.Generator().manual_seed(2)).bfloat16()
    x64 = x.double().numpy()
    got = eng.linear_rows_packed(x.cuda(), packed, residual=b.expand(m, 200).contiguous().cuda()).double().cpu().numpy()
    tol = 520 * U * (np.abs(x64) @ np.abs(w).T + np.abs(b.double().numpy())) + 2.0 ** -46 * np.abs(x64).max(1, keepdims=True) * np.abs(w).sum(1)
    assert (np.abs(got - (x64 @ w.T + b.double().numpy())) <= tol).all()
    own = PackedLinear(packed.weight, packed.scale, 512, 64, b.cuda())
    rounded = PackedLinear(packed.weight, packed.scale, 512, 64, b.bfloat16().cuda())
    assert torch.equal(eng.linear_rows_packed(x.cuda(), own), eng.linear_rows_packed(x.cuda(), rounded))


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("size", [1e-35, 1e-32, 1e-28, 1e-24, 1e30, 1e34])
def test_attention_over_values_of_any_size(eng, size, group):
    parts = _filled(3, 2, 4, seed=group)
    parts[3].mul_(size)
    q = torch.randn(3, 2 * group * 64, generator=torch.Generator().manual_seed(0)) * 0.3
    _check_attend(eng, parts, q, [2, 0, 1], [250, 64, 3])


@pytest.mark.parametrize("group", [1, 4])
def test_attention_over_blocks_of_far_scales(eng, group):
    parts = _filled(2, 2, 40, seed=group)
    size = torch.ones(2, 2, 40, dtype=torch.float64)
    size[0], size[0, :, 17:19], size[1, 1, 30] = 1e-28, 1e30, 1e36
    parts = (*parts[:3], (parts[3] * size).float())
    q = torch.randn(2, 2 * group * 64, generator=torch.Generator().manual_seed(0)) * 0.3
    for lens in ([1088, 1920], [2500, 2560], [1089, 1921]):
        _check_attend(eng, parts, q, [0, 1], lens)


def test_attention_with_the_largest_scale(eng):
    """Tiny queries times a scale near the largest number: scores of ordinary size."""
    parts = _filled(3, 2, 2, seed=3)
    q = torch.randn(3, 128, generator=torch.Generator().manual_seed(0)) * 1e-38
    _check_attend(eng, parts, q, [2, 0, 1], [128, 64, 3], scale=2.9e38)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("old", [1e-45, 1e-40, 1e-38, 3e-37, 4e-36])
def test_store_behind_a_scale_that_no_store_leaves(eng, old, dtype):
    """Blocks whose scale lies below 2^-124 (a caller's own cache), continued with rows below 2^-117, which leave it: quotients
    saturate at 127; and with ordinary rows, which replace it."""
    g = torch.Generator().manual_seed(2)
    small = torch.rand(5, 128, generator=g) * 1.1e-35 - 5.5e-36
    small[1, ::2], small[2], small[3, ::3] = 0.0, 1e-38, -1e-40
    for rows in (small, small * 3e35):
        parts = _filled(5, 2, 1)
        parts[2].fill_(old)
        parts[3].fill_(old * 2)
        _check_store(eng, parts, rows.to(dtype), rows.flip(0).to(dtype), [1], [3], [0, 5])
        _check_store(eng, parts, rows.to(dtype), rows.flip(0).to(dtype), [0, 1, 2, 3, 4], [3, 60, 9, 1, 63])
    eng.device_status()


def _raw_attend(eng, cache, q, slots, lens, out, clear, scratch_bytes):
    """The C call with a scratch of ``scratch_bytes``, none for 0."""
    put = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    heads = q.shape[1] // 64
    sl, ln = put(slots), put(lens)
    scratch = torch.full((max(scratch_bytes, 16),), 255, dtype=torch.uint8, device="cuda")   # its contents count for nothing
    rc = eng.lib.wdz_qcache_attention(eng.h, cache.ref, q.data_ptr(), q.stride(0), capi.WDZ_F32, heads, sl.data_ptr(), ln.data_ptr(),
                                      q.shape[0], 0.125, out.data_ptr(), out.stride(0), capi.WDZ_F32, clear,
                                      scratch.data_ptr() if scratch_bytes else None, scratch_bytes, eng._raw_stream())
    assert rc == 0
    return out


@pytest.mark.parametrize("heads,group,tokens", [(4, 4, 20000), (2, 1, 9000), (1, 2, 12001), (2, 8, 33000)])
def test_attention_of_long_rows_in_parts(eng, heads, group, tokens):
    """A few long rows over all SMs, with query heads that share their keys; and the same rows with no scratch, or too little."""
    parts = _filled(3, heads, (tokens + 63) // 64, seed=group, spread=0.2)
    q = torch.randn(3, heads * group * 64, generator=torch.Generator().manual_seed(1)) * 0.3
    lens = [tokens, 70, tokens // 2 + 1]
    cache = _cuda_cache(parts)
    got = _check_attend(eng, parts, q, [1, 2, 0], lens, cache=cache)
    need = eng.lib.wdz_qcache_attention_scratch(eng.h, cache.ref, heads * group, 3)
    assert need > 0
    on = q.cuda()
    for have in (need, 0, need - 4):
        out = _raw_attend(eng, cache, on, [1, 2, 0], lens, torch.full_like(on, 7.0), 0, have)
        if have == need:
            assert torch.equal(out, got)
        want, weight, top = ref.attend(q.numpy(), *(t.numpy() for t in parts), [1, 2, 0], lens, 0.125)
        tol = top * (2 * 70 * U * weight + 2.0 ** -21 + np.asarray(lens, dtype=np.float64).reshape(-1, 1, 1) * 2.0 ** -23)
        tol = np.repeat(tol.reshape(3, -1), 64, axis=1) + U * np.abs(want)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all(), have


def test_attention_in_parts_of_skipped_and_empty_rows(eng):
    cache = _cuda_cache(_filled(2, 2, 200, seed=1))
    q = torch.randn(4, 256, generator=torch.Generator().manual_seed(1)).cuda()
    slots, lens = [0, -1, 1, 2], [12000, 12000, 0, 5]
    need = eng.lib.wdz_qcache_attention_scratch(eng.h, cache.ref, 4, 4)
    assert need > 0
    for have in (need, 0):
        left = _raw_attend(eng, cache, q, slots, lens, torch.full((4, 256), 7.0, device="cuda"), 0, have)
        assert (left[[1, 3]] == 7).all() and (left[2] == 0).all() and left[0].isfinite().all() and (left[0] != 7).any()
        cleared = _raw_attend(eng, cache, q, slots, lens, torch.full((4, 256), 7.0, device="cuda"), 1, have)
        assert (cleared[1:] == 0).all() and torch.equal(cleared[0], left[0])
    kept = torch.full((4, 256), 7.0, device="cuda")
    put = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    assert torch.equal(eng.qcache_attention(q, cache, put(slots), put(lens), out=kept)[[1, 2, 3]], torch.tensor([7.0, 0.0, 7.0], device="cuda")[:, None].expand(3, 256))
    assert (eng.qcache_attention(q, cache, put(slots), put(lens))[1:] == 0).all()
    eng.device_status()
