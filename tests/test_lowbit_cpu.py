"""CPU checks of the low-bit operators: packing, the arguments that the calls refuse, and the rounding of the store as
its kernel computes it.  No GPU compute."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest
import torch

import lowbit_ref as ref
from whisperdrz_b200 import capi
from whisperdrz_b200.dims import ModelDimensions
from whisperdrz_b200.lowbit import PackedLinear, QCache, pack_linear, pack_nibbles


@pytest.fixture(scope="module")
def lib():
    from whisperdrz_b200 import build
    build.build()
    return capi.load()


@pytest.fixture(scope="module")
def handle(lib):
    """An engine that was created and never finalized: arguments are looked at before its state."""
    dims = ModelDimensions.from_name("test-tiny")
    shape = [getattr(dims, f) for f in ("n_mels", "n_audio_ctx", "n_audio_state", "n_audio_head", "n_audio_layer",
                                        "n_vocab", "n_text_ctx", "n_text_state", "n_text_head", "n_text_layer")]
    h = C.c_void_p()
    assert lib.wdz_engine_create(C.byref(capi.Config(*shape, capi.WDZ_F32, 1, 64, 1, 1, 0)), C.byref(h)) == capi.WDZ_OK
    yield h
    lib.wdz_engine_destroy(h)


@pytest.fixture()
def host():
    """The Python calls without a device behind them: what they refuse, they refuse before they reach the library."""
    from whisperdrz_b200.engine import Engine
    e = Engine.__new__(Engine)
    e.device, e._ordinal, e.dtype, e.h = torch.device("cpu"), -1, torch.float32, None
    return e


def _cache(slots=2, heads=2, blocks=2):
    return QCache.empty(slots, 64 * blocks, heads, "cpu")


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("n,k,group", [(3, 128, 32), (5, 200, 64), (1, 1, 128), (4, 1237, 32)])
def test_pack_linear_keeps_the_nearest_of_sixteen_values(n, k, group):
    g = torch.Generator().manual_seed(n * 1000 + k)
    w = torch.randn(n, k, generator=g)
    p = pack_linear(w, group, bias=torch.zeros(n))
    kp = 2 * p.weight.shape[1]
    assert kp % 128 == 0 and kp - k < 128 and p.in_features == k and p.out_features == n
    q = ref.unpack(p.weight.numpy(), kp)
    s = np.repeat(p.scale.float().numpy().astype(np.float64), group, axis=1)
    assert (q[:, k:] == 0).all()
    # half a step; the largest of a group lies at 7 steps of a scale that bf16 rounded by at most 2^-8
    assert (np.abs(q * s - np.pad(w.numpy().astype(np.float64), ((0, 0), (0, kp - k)))) <= s * (0.5 + 7 * 2.0 ** -8)).all()


def test_pack_nibbles_order():
    q = torch.randint(-8, 8, (3, 256), generator=torch.Generator().manual_seed(4))
    assert (ref.unpack(pack_nibbles(q).numpy(), 256) == q.numpy()).all()


def test_pack_linear_of_zeros_and_refusals():
    assert (ref.unpack(pack_linear(torch.zeros(2, 64)).weight.numpy(), 128) == 0).all()
    with pytest.raises(ValueError):
        pack_linear(torch.zeros(2, 64), group=48)
    with pytest.raises(ValueError):
        pack_linear(torch.zeros(64))
    p = pack_linear(torch.randn(4, 130), 64)
    for bad in (dict(group=32), dict(in_features=300), dict(scale=p.scale.float()), dict(weight=p.weight.to(torch.int32)),
                dict(bias=torch.zeros(3)), dict(scale=p.scale[:, :2]), dict(weight=p.weight[:, ::2])):
        with pytest.raises(ValueError):
            PackedLinear(**{**dict(weight=p.weight, scale=p.scale, in_features=130, group=64), **bad})


# ------------------------------------------------------------------- QCache
def test_qcache_takes_a_layer_of_a_larger_allocation_and_refuses_the_rest():
    k = torch.zeros(4, 3, 2, 128, 64, dtype=torch.int8)          # [slots, layers, heads, tokens, 64]
    s = torch.zeros(4, 3, 2, 2)
    c = QCache(k[:, 1], k.clone()[:, 1], s[:, 1], s.clone()[:, 1])
    assert (c.desc.slot_stride, c.desc.scale_slot_stride, c.desc.n_blocks) == (3 * 2 * 128 * 64, 12, 2)
    k, s = torch.zeros(4, 2, 128, 64, dtype=torch.int8), torch.zeros(4, 2, 2)
    for bad in ((k[..., :32], k[..., :32], s, s), (k[:, :, :100], k[:, :, :100], s, s), (k.float(), k, s, s), (k, k, s.double(), s),
                (k, k, s[..., :1], s), (k, k[:2], s, s), (k.transpose(1, 2), k.transpose(1, 2), s, s), (k[:0], k[:0], s[:0], s[:0]),
                (k, k, s.expand(4, 2, 2)[:, :, :1].expand(4, 2, 2), s), (k[:1].expand(4, 2, 128, 64), k, s, s)):
        with pytest.raises(ValueError):
            QCache(*bad)


# ----------------------------------------------------- refusals of the calls
def test_python_calls_refuse_bad_arguments(host):
    c = _cache()
    rows = torch.zeros(3, 128)
    good = (lambda: host.qcache_store(c, rows, rows, [0, 1, 2], [0, 0, 0]), lambda: host.qcache_attention(rows, c, [0, 1, 5], [1, 1, 1]),
            lambda: host.linear_rows_packed(torch.zeros(2, 130), pack_linear(torch.zeros(4, 130), 64)))
    for call in good:                        # good arguments get as far as the library, which this host does not have
        with pytest.raises(AttributeError):
            call()
    for bad in (dict(k=rows[:, :64]), dict(k=rows.double()), dict(v=rows[:2]), dict(v=rows.bfloat16()), dict(slots=[0, 0, 1]),
                dict(slots=[0, 1]), dict(positions=[0]), dict(row_begin=[0, 4]), dict(row_begin=[0, 2, 1], slots=[0, 1], positions=[0, 0]),
                dict(row_begin=[-1, 2], slots=[0], positions=[0]), dict(row_begin=[])):
        with pytest.raises(ValueError):
            host.qcache_store(**{**dict(cache=c, k=rows, v=rows, slots=[0, 1, 2], positions=[0, 0, 0]), **bad})
    q = torch.zeros(2, 128)
    for bad in (dict(q=torch.zeros(2, 192)), dict(q=torch.zeros(2, 9 * 128)), dict(q=q.half()), dict(q=torch.zeros(2, 0)), dict(slots=[0]),
                dict(lens=[1, 2, 3]), dict(out=torch.zeros(2, 64)), dict(out=torch.zeros(2, 128).half()), dict(out_dtype=torch.half),
                dict(out=torch.zeros(2, 256)[:, ::2]), dict(out=torch.zeros(2, 128), out_dtype=torch.bfloat16),
                dict(out=torch.zeros(2, 129)[:, 1:])):
        with pytest.raises(ValueError):
            host.qcache_attention(**{**dict(q=q, cache=c, slots=[0, 1], lens=[1, 1]), **bad})
    w = pack_linear(torch.zeros(4, 130), 64)
    x = torch.zeros(2, 130)
    for bad in (dict(x=x[:, :128]), dict(x=x.half()), dict(x=x[0]), dict(out=torch.zeros(2, 5)), dict(residual=torch.zeros(2, 4).bfloat16()),
                dict(out=torch.zeros(2, 8)[:, ::2])):
        with pytest.raises(ValueError):
            host.linear_rows_packed(**{**dict(x=x, w=w), **bad})


def _desc(**kw):
    d = dict(k=256, v=512, k_scale=1024, v_scale=2048, slot_stride=2 * 2 * 4096, scale_slot_stride=4, n_slots=2, n_heads=2, n_blocks=2)
    return capi.QCacheDesc(**{**d, **kw})


def test_abi_refuses_bad_arguments_before_it_looks_at_the_engine(lib, handle):
    """Addresses below are never followed: the calls end before a launch."""
    f32, bf16 = capi.WDZ_F32, capi.WDZ_BF16

    def store(cache=None, k=4096, ldk=128, v=8192, ldv=128, dtype=f32, n=3, rb=64, sl=64, ps=64, runs=2, most=3):
        return lib.wdz_qcache_store(handle, C.byref(cache or _desc()), k, ldk, v, ldv, dtype, n, rb, sl, ps, runs, most, None)

    def attend(cache=None, q=4096, ldq=128, qt=f32, hq=2, sl=64, ln=64, n=3, scale=0.125, out=8192, ldo=128, ot=bf16):
        return lib.wdz_qcache_attention(handle, C.byref(cache or _desc()), q, ldq, qt, hq, sl, ln, n, scale, out, ldo, ot, 0, None, 0, None)

    def linear(x=4096, ldx=130, xt=f32, M=2, K=130, w=4096, sc=4096, g=64, b=None, r=None, N=4, y=4096):
        return lib.wdz_linear_rows_packed(handle, x, ldx, xt, M, K, w, sc, g, b, r, N, y, None)

    not_ready = -4
    assert store() == not_ready and attend() == not_ready and linear() == not_ready
    caches = [_desc(k=None), _desc(v_scale=None), _desc(k=257), _desc(slot_stride=2 * 2 * 4096 - 16), _desc(slot_stride=2 * 2 * 4096 + 8),
              _desc(scale_slot_stride=3), _desc(n_slots=0), _desc(n_heads=0), _desc(n_blocks=0), _desc(n_blocks=2 ** 30), _desc(n_blocks=2 ** 24 + 1, slot_stride=2 ** 40, scale_slot_stride=2 ** 30), _desc(n_heads=4097),
              _desc(v_scale=2050)]
    for c in caches:
        assert store(cache=c) == -1 and attend(cache=c) == -1
    for bad in (dict(k=None), dict(v=None), dict(sl=None), dict(ps=None), dict(dtype=2), dict(n=-1), dict(runs=-1), dict(most=-1),
                dict(rb=None), dict(ldk=64), dict(ldv=126), dict(k=4100), dict(ldk=129), dict(ldk=132, dtype=bf16)):
        assert store(**bad) == -1, bad
    assert store(runs=70000) == -5
    assert store(n=0, runs=0, k=None) == 0 and attend(n=0, q=None) == 0 and linear(M=0, x=None) == 0
    for bad in (dict(q=None), dict(out=None), dict(sl=None), dict(ln=None), dict(qt=5), dict(ot=-1), dict(hq=3), dict(hq=0), dict(hq=18),
                dict(n=-1), dict(ldq=64), dict(ldo=120), dict(q=4098), dict(out=8196), dict(ldo=129, ot=f32),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-1.0)):
        assert attend(**bad) == -1, bad
    for bad in (dict(x=None), dict(w=None), dict(sc=None), dict(y=None), dict(xt=9), dict(M=-1), dict(N=0), dict(K=0), dict(g=16), dict(g=0),
                dict(ldx=129), dict(w=4104), dict(sc=4100), dict(K=2 ** 31 - 100), dict(x=4098), dict(b=4098), dict(r=4098), dict(y=4097)):
        assert linear(**bad) == -1, bad
    assert linear(M=8 * 65535 + 1) == -5
    assert lib.wdz_qcache_attention_scratch(handle, C.byref(_desc()), 2, -1) == -1
    assert lib.wdz_qcache_attention_scratch(handle, C.byref(_desc()), 2, 3) == 0
    assert lib.wdz_qcache_attention_scratch(handle, C.byref(_desc(n_blocks=512, slot_stride=2 ** 26, scale_slot_stride=2 ** 12)), 4, 1) > 0
    assert lib.wdz_qcache_store(None, C.byref(_desc()), 1, 1, 1, 1, 0, 1, None, 1, 1, 1, 1, None) == -1


# --------------------------------------------------- the store's arithmetic
def test_store_rounding_as_the_kernel_computes_it():
    """rint(x / s) from the products with the floats above and below 1 / s, and the sign of x - h s where they differ, in
    float32, against fractions: at every half step, one float to either side of it, and at random places, for scales of
    every mantissa size and rows in bf16."""
    rng = np.random.default_rng(0)
    f = np.float32
    magic = 12582912.0
    differed = 0
    for trial in range(80):
        top = f(rng.uniform(1, 2) * 2.0 ** int(rng.integers(-116, 100)))
        if trial % 2:
            top = torch.tensor(top).bfloat16().float().numpy()[()]
        s = f(top / f(127))
        inv = f(1) / s
        half_steps = (np.arange(-127, 127) + 0.5).astype(np.float64) * np.float64(s)
        x = half_steps.astype(f)
        x = np.concatenate([x, np.nextafter(x, f(np.inf)), np.nextafter(x, f(-np.inf)), (rng.uniform(-1, 1, 64) * top).astype(f), [top]])
        if trial % 4 == 1:
            x = torch.tensor(x).bfloat16().float().numpy()
        x = x[np.abs(x) <= top]

        def whole(m):   # a fused multiply-add with 1.5 2^23: the product has 48 bits, so 64 bits hold the sum before it is rounded
            return (x.astype(np.float64) * np.float64(m) + magic).astype(f).astype(np.float64) - magic

        a, b = whole(np.nextafter(inv, f(np.inf))), whole(np.nextafter(inv, f(0)))
        half = 0.5 * (a + b)
        sign = np.array([(Fraction(float(v)) > Fraction(float(h)) * Fraction(float(s))) - (Fraction(float(v)) < Fraction(float(h)) * Fraction(float(s)))
                         for v, h in zip(x, half)])
        even = np.where(a % 2 == 0, a, b)
        q = np.where(a == b, a, np.where(sign > 0, np.maximum(a, b), np.where(sign < 0, np.minimum(a, b), even)))
        differed += int((a != b).sum())
        want = np.array([round(Fraction(float(v)) / Fraction(float(s))) for v in x])   # half to even
        assert (q == want).all() and np.abs(q).max() <= 127
    assert differed > 200


def test_reference_store_continues_a_block():
    values, scale = np.zeros((1, 1, 64, 64), np.int8), np.zeros((1, 1, 1), np.float32)
    ref.store(values, scale, np.full((1, 64), 1.27, np.float32), [0], [0])
    ref.store(values, scale, np.full((1, 64), 12.7, np.float32), [0], [1])
    assert (values[0, 0, 0] == 13).all() and (values[0, 0, 1] == 127).all()   # 127 * 0.01 / 0.1 = 12.7
    ref.store(values, scale, np.full((1, 64), 1.27, np.float32), [0], [0])
    assert scale[0, 0, 0] == np.float32(np.float64(np.float32(1.27)) / 127)
