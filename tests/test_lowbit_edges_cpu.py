"""CPU checks of the low-bit operators' host side: what is refused, what is let through, and what the scheduler asks for."""
import numpy
import pytest
import torch

from test_lowbit_cpu import _cache, handle, host, lib  # noqa: F401
from test_scheduler_cpu import StubEngine, _patch_rules_dev
from whisperdrz_b200 import capi
from whisperdrz_b200.lowbit import QCache, pack_linear
from whisperdrz_b200.transcriber import Transcriber


def test_scheduler_asks_for_the_decode_loop_s_own_status():
    """A report of the operators on caller-held memory, which device_status would raise, is no failed decode step."""
    class Engine(StubEngine):
        asked = 0

        def device_status(self):
            raise AssertionError("the operators' reports are not the scheduler's")

        def decode_status(self):
            self.asked += 1

    eng = Engine()
    tr = Transcriber(eng, max_new_tokens=10, max_continuations=0)
    _patch_rules_dev(tr)
    assert len(tr.transcribe(torch.randn(16000 * 30)).raw_chunks) == 1
    assert eng.asked > 0


def test_a_padded_batch_names_no_slot_twice(host):  # noqa: F811
    """Runs of slots outside the cache are skipped, however many: only a slot of the cache may not come twice."""
    rows = torch.zeros(3, 128)
    for slots in ([0, -1, -1], [2, 2, 1], [-1, -1, -1], [5, 0, 5]):
        with pytest.raises(AttributeError):      # as far as the library, which this host does not have
            host.qcache_store(_cache(), rows, rows, slots, [0, 0, 0])
    for slots in ([1, -1, 1], [0, 0, 0]):
        with pytest.raises(ValueError):
            host.qcache_store(_cache(), rows, rows, slots, [0, 0, 0])


def test_linear_refuses_features_that_its_places_cannot_count(lib, handle):  # noqa: F811
    """A block covers up to 128 features at places of 32 bits: the last of nearly 2^31 would have wrapped below zero.  The
    addresses are never followed."""
    def linear(N):
        return lib.wdz_linear_rows_packed(handle, 4096, 128, capi.WDZ_BF16, 1, 128, 4096, 4096, 64, None, None, N, 4096, None)

    assert linear(2 ** 31 - 1) == -1 and linear(2 ** 31 - 128) == -1
    assert linear(2 ** 31 - 129) == -4       # as far as the engine, which is not ready


def test_rows_of_three_dimensions_are_heads_of_64(host):  # noqa: F811
    """[n, heads, 64] only: other splits of the same width lie in another order."""
    rows, q = torch.zeros(3, 2, 64), torch.zeros(3, 4, 64)
    for call in (lambda: host.qcache_store(_cache(), rows, rows, [0, 1, 2], [0, 0, 0]),
                 lambda: host.qcache_store(_cache(), rows.view(3, 128), rows, [0, 1, 2], [0, 0, 0]),
                 lambda: host.qcache_attention(q, _cache(), [0, 1, 1], [1, 1, 1])):
        with pytest.raises(AttributeError):      # as far as the library, which this host does not have
            call()
    for bad in (rows.transpose(1, 2), rows.view(3, 1, 128), rows.view(3, 4, 32)):
        with pytest.raises(ValueError):
            host.qcache_store(_cache(), bad, rows, [0, 1, 2], [0, 0, 0])
        with pytest.raises(ValueError):
            host.qcache_store(_cache(), rows, bad, [0, 1, 2], [0, 0, 0])
        with pytest.raises(ValueError):
            host.qcache_attention(bad, _cache(), [0, 1, 1], [1, 1, 1])


def test_index_tensors_keep_what_they_say(host):  # noqa: F811
    """64-bit entries that no int32 holds stay outside the cache instead of wrapping into it; lengths stay long."""
    far = torch.tensor([2 ** 32 + 1, -2 ** 32, 2 ** 31, 5, -1])
    assert host._index("slots", far, 5).tolist() == [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, -1]
    for t in (torch.uint8, torch.int16, torch.int32, torch.int64):
        x = host._index("lens", torch.tensor([3, 0], dtype=t), 2)
        assert x.dtype == torch.int32 and x.tolist() == [3, 0]
    for bad in (torch.tensor([1.5, 2.0]), torch.tensor([True, False]), torch.tensor([1, 2], dtype=torch.uint32), [1.5, 2.0], torch.tensor([1, 2, 3]), [1]):
        with pytest.raises(ValueError):
            host._index("slots", bad, 2)
    assert host._index("slots", [1, 2], 2).tolist() == [1, 2]
    assert host._index("slots", numpy.array([1, 2]), 2).tolist() == [1, 2]
    rows = torch.zeros(2, 128)
    with pytest.raises(ValueError):
        host.qcache_store(_cache(), rows, rows, [0.5, 1], [0, 0])
    with pytest.raises(ValueError):
        host.qcache_store(_cache(), rows, rows, [0], [0], row_begin=[0, 1.5])


def test_results_may_not_lie_over_what_is_still_read(host):  # noqa: F811
    """Blocks of a launch read x and q while others write: in place means the queries' own rows, or the residual."""
    w = pack_linear(torch.zeros(128, 128))
    x = torch.zeros(4, 128)
    buf = torch.zeros(9, 128)
    good = (dict(x=x), dict(x=x, out=torch.zeros(4, 128), residual=x), dict(x=x, out=buf[4:8], residual=buf[4:8]),
            dict(x=buf[:4], out=buf[4:8]), dict(x=buf[:4].bfloat16(), out=buf[:4]), dict(x=buf[:4], out=buf[4:8], residual=buf[:4]))
    bad = (dict(x=x, out=x), dict(x=buf[:4], out=buf[3:7]), dict(x=buf[4:8], out=buf[1:5]), dict(x=x, out=buf[:4], residual=buf[1:5]))
    for kw in good:
        with pytest.raises(AttributeError):      # as far as the library, which this host does not have
            host.linear_rows_packed(w=w, **kw)
    for kw in bad:
        with pytest.raises(ValueError):
            host.linear_rows_packed(w=w, **kw)
    p = torch.zeros(4, 384)                      # a fused product
    half = torch.zeros(8, 128, dtype=torch.bfloat16)
    good = (dict(q=p[:, :128], out=p[:, :128]), dict(q=p[:, :128], out=p[:, 128:256]), dict(q=p[:, 256:], out=p[:, :128]), dict(q=p[:2, :128], out=p[2:, :128]),
            dict(q=p[:1, :128], out=p[0:1, 128:256]), dict(q=half[:4], out=half[4:]), dict(q=p[:, 128:256], out=torch.zeros(4, 128)))
    bad = (dict(q=p[:, :128], out=p[:, 64:192]), dict(q=p[:3, :128], out=p[1:, :128]), dict(q=p[:, 64:192], out=p[:, :128]), dict(q=half[:4], out=half[1:5]),
           dict(q=x.view(-1).view(torch.bfloat16).view(8, 128)[:4], out=x), dict(q=p[1:, :128], out=p[:3, 64:192]))
    for kw in good:
        n = kw["q"].shape[0]
        with pytest.raises(AttributeError):
            host.qcache_attention(cache=_cache(4), slots=[0, 1, 2, 3][:n], lens=[1] * n, **kw)
    for kw in bad:
        n = kw["q"].shape[0]
        with pytest.raises(ValueError):
            host.qcache_attention(cache=_cache(4), slots=[0, 1, 2, 3][:n], lens=[1] * n, **kw)


def test_operands_keep_the_tensors_that_their_addresses_belong_to():
    """The kernels get addresses taken when the operand was made: another tensor in its place would leave them dangling."""
    c, w = _cache(), pack_linear(torch.zeros(4, 128), bias=torch.zeros(4))
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
        assert getattr(c.desc, name) == getattr(c, name).data_ptr()
    for name in ("weight", "scale"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name).clone())
    assert (w.at, w.scale_at) == (w.weight.data_ptr(), w.scale.data_ptr())


def test_a_bias_stays_the_one_that_was_checked():
    """Its length, type and device are looked at when the operand is made."""
    w = pack_linear(torch.zeros(4, 128), bias=torch.zeros(4))
    for bad in (torch.zeros(3), torch.zeros(4, device="meta"), None):
        with pytest.raises(AttributeError):
            w.bias = bad
    w.bias.fill_(2.0)
    assert (w.bias == 2).all()


def test_store_refuses_keys_and_values_in_one_place(host):  # noqa: F811
    """Rows of both would be rounded into the same bytes, in no order; attending over such a cache is all right."""
    rows = torch.zeros(2, 128)
    k, s = torch.zeros(2, 2, 128, 64, dtype=torch.int8), torch.zeros(2, 2, 2)
    both, scales = torch.zeros(2, 2, 2, 128, 64, dtype=torch.int8), torch.zeros(2, 2, 2, 2)     # K and V of a slot side by side
    for cache in (QCache(k, k, s, s), QCache(k, k.clone(), s, s), QCache(k, k, s, s.clone()), QCache(k[:1], k[:1], s[:1], s[1:])):
        with pytest.raises(ValueError):
            host.qcache_store(cache, rows, rows, [0, 1], [0, 0])
        with pytest.raises(AttributeError):      # as far as the library, which this host does not have
            host.qcache_attention(rows, cache, [0, 0], [1, 1])
    for cache in (QCache(both[:, 0], both[:, 1], scales[:, 0], scales[:, 1]), QCache(k[:1], k[1:], s[:1], s[1:])):
        with pytest.raises(AttributeError):
            host.qcache_store(cache, rows, rows, [0, 1], [0, 0])
