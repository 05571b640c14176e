"""Python host of the CUDA engine: owns the device tensors (torch is the
allocator), lends them to libwdz.so through the C ABI and exposes the engine
calls with torch tensors in and out.  Requires a CUDA device; there is no
fallback."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import capi, frontend
from .dims import ModelDimensions
from .lowbit import HEAD_DIM, PackedLinear, QCache, rows_overlap

_INDEX_DTYPES = (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64)
_TORCH_DTYPE = {torch.float32: capi.WDZ_F32, torch.bfloat16: capi.WDZ_BF16}


def pack_weights(sd: dict, dims: ModelDimensions, dtype: torch.dtype, device) -> dict[str, torch.Tensor]:
    """Reference state_dict (model.py names) -> the tensors the engine binds:
    q/k/v stacked per attention (key bias = 0, model.py:259), conv kernels
    tap-major ([out, tap * in + c]), cross-attention K/V projections of all
    decoder layers stacked into one [L * 2 * d, d] operand."""
    out: dict[str, torch.Tensor] = {}

    def put(name, t, dt=dtype):
        out[name] = t.detach().to(device=device, dtype=dt).contiguous()

    put("encoder.conv1.weight", sd["encoder.conv1.weight"].permute(0, 2, 1).reshape(dims.n_audio_state, -1))
    put("encoder.conv1.bias", sd["encoder.conv1.bias"])
    put("encoder.conv2.weight", sd["encoder.conv2.weight"].permute(0, 2, 1).reshape(dims.n_audio_state, -1))
    put("encoder.conv2.bias", sd["encoder.conv2.bias"])
    put("encoder.positional_embedding", sd["encoder.positional_embedding"], torch.float32)
    put("encoder.ln_post.weight", sd["encoder.ln_post.weight"])
    put("encoder.ln_post.bias", sd["encoder.ln_post.bias"])

    def block(p, cross):
        q, k, v = (sd[f"{p}.attn.{n}.weight"] for n in ("query", "key", "value"))
        put(f"{p}.attn.qkv.weight", torch.cat([q, k, v], 0))
        qb, vb = sd[f"{p}.attn.query.bias"], sd[f"{p}.attn.value.bias"]
        put(f"{p}.attn.qkv.bias", torch.cat([qb, torch.zeros_like(qb), vb], 0))
        names = ["attn_ln.weight", "attn_ln.bias", "attn.out.weight", "attn.out.bias", "mlp_ln.weight",
                 "mlp_ln.bias", "mlp.0.weight", "mlp.0.bias", "mlp.2.weight", "mlp.2.bias"]
        if cross:
            names += ["cross_attn_ln.weight", "cross_attn_ln.bias", "cross_attn.query.weight",
                      "cross_attn.query.bias", "cross_attn.out.weight", "cross_attn.out.bias"]
        for n in names:
            put(f"{p}.{n}", sd[f"{p}.{n}"])

    for i in range(dims.n_audio_layer):
        block(f"encoder.blocks.{i}", False)
    for i in range(dims.n_text_layer):
        block(f"decoder.blocks.{i}", True)
    put("decoder.token_embedding.weight", sd["decoder.token_embedding.weight"])
    put("decoder.positional_embedding", sd["decoder.positional_embedding"])
    put("decoder.ln.weight", sd["decoder.ln.weight"])
    put("decoder.ln.bias", sd["decoder.ln.bias"])
    kvw, kvb = [], []
    for i in range(dims.n_text_layer):
        p = f"decoder.blocks.{i}.cross_attn"
        kvw += [sd[f"{p}.key.weight"], sd[f"{p}.value.weight"]]
        kvb += [torch.zeros_like(sd[f"{p}.value.bias"]), sd[f"{p}.value.bias"]]
    put("decoder.cross_kv.weight", torch.cat(kvw, 0))
    put("decoder.cross_kv.bias", torch.cat(kvb, 0))
    return out


def pack_rules(rules: list[dict]) -> np.ndarray:
    """list of rule dicts -> array of ``wdz_rule_desc`` (uint8 [n, 128])."""
    arr = (capi.RuleDesc * max(len(rules), 1))()
    for i, r in enumerate(rules):
        d = arr[i]
        d.forced_id = r.get("forced_id", -1)
        d.mode = r.get("mode", capi.MODE_OR)
        d.arg0, d.arg1 = r.get("arg0", 0), r.get("arg1", 0)
        d.table_bits = r.get("table_bits", 0)
        d.prefix_begin, d.prefix_end = r.get("prefix_begin", 0), r.get("prefix_end", 0)
        d.or_table, d.allow_table = r.get("or_table", 0), r.get("allow_table", 0)
        for field, cap in (("set_ids", 6), ("clear_ids", 4), ("pen_ids", 10)):
            ids = list(dict.fromkeys(r.get(field, [])))
            if len(ids) > cap:
                raise ValueError(f"rule {i}: {len(ids)} {field} > {cap}")
            setattr(d, "n_" + field.split("_")[0], len(ids))
            for j, t in enumerate(ids):
                getattr(d, field)[j] = int(t)
    return np.frombuffer(bytes(arr), dtype=np.uint8).reshape(-1, 128)[: len(rules)].copy()


def pack_tables(tables: torch.Tensor, n_vocab: int) -> torch.Tensor:
    """bool [n_tables, V] -> uint32 bitsets as int32 tensor [max(n_tables, 32), ceil(V / 32)]."""
    words = (n_vocab + 31) // 32
    n = max(capi.MAX_TABLES, int(tables.shape[0]))
    t = np.zeros((n, words * 32), dtype=np.uint8)
    tb = tables.cpu().numpy().astype(np.uint8)
    t[: tb.shape[0], :n_vocab] = tb
    packed = np.packbits(t.reshape(n, words, 32), axis=-1, bitorder="little")
    return torch.from_numpy(packed.view(np.uint32).reshape(n, words).view(np.int32).copy())


class Engine:
    """One engine per GPU per process (the C library is not thread-safe)."""

    def __init__(self, dims: ModelDimensions, state_dict: dict, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda:0", n_slots: int = 32, max_tokens: int | None = None,
                 max_clips: int = 16, max_rows: int | None = None, flags: int = 0,
                 tables: torch.Tensor | None = None, lend_workspace: bool = True):
        if not torch.cuda.is_available():
            raise RuntimeError("whisperdrz_b200.Engine needs a CUDA device (no CPU path exists)")
        if dtype not in _TORCH_DTYPE:
            raise ValueError("dtype must be torch.float32 or torch.bfloat16")
        self.lib = capi.load()
        self.dims, self.dtype = dims, dtype
        self.device = torch.device(device)
        torch.cuda.set_device(self.device)
        self._ordinal = torch.cuda.current_device()   # of a device given without its number, too
        self.n_slots = n_slots
        self.max_tokens = max_tokens or dims.n_text_ctx
        self.max_clips = max_clips
        self.max_rows = max_rows or max(n_slots, 64)
        cfg = capi.Config(*[getattr(dims, f) for f in (
            "n_mels", "n_audio_ctx", "n_audio_state", "n_audio_head", "n_audio_layer",
            "n_vocab", "n_text_ctx", "n_text_state", "n_text_head", "n_text_layer")],
            _TORCH_DTYPE[dtype], n_slots, self.max_tokens, max_clips, self.max_rows, flags)
        self.cfg = cfg
        h = C.c_void_p()
        rc = self.lib.wdz_engine_create(C.byref(cfg), C.byref(h))
        if rc != capi.WDZ_OK:
            raise capi.WdzError(rc, "wdz_engine_create rejected the configuration")
        self.h = h
        dev = self.device
        self.weights = pack_weights(state_dict, dims, dtype, dev)
        L, d = dims.n_text_layer, dims.n_text_state
        self.self_k = torch.zeros(L, n_slots, self.max_tokens, d, dtype=dtype, device=dev)
        self.self_v = torch.zeros_like(self.self_k)
        self.cross_k = torch.zeros(L, n_slots, dims.n_audio_ctx, d, dtype=dtype, device=dev)
        self.cross_v = torch.zeros_like(self.cross_k)
        self.seq_lens_dev = torch.zeros(n_slots, dtype=torch.int32, device=dev)
        fb, lo, hi = frontend.mel_filterbank(dims.n_mels)
        self.consts = {
            "mel.twiddle": torch.from_numpy(frontend.twiddle()).to(dev),
            "mel.window": torch.from_numpy(frontend.hann_periodic()).to(dev),
            "mel.fb": torch.from_numpy(fb).to(dev),
            "mel.band_lo": torch.from_numpy(lo).to(dev),
            "mel.band_hi": torch.from_numpy(hi).to(dev),
        }
        self.tables_dev = None
        if tables is not None:
            self.tables_dev = pack_tables(tables, dims.n_vocab).to(dev)
        for name, t in self.weights.items():
            self._bind(name, t)
        for name, t in self.consts.items():
            self._bind(name, t)
        for name, t in (("cache.self_k", self.self_k), ("cache.self_v", self.self_v),
                        ("cache.cross_k", self.cross_k), ("cache.cross_v", self.cross_v),
                        ("cache.seq_lens", self.seq_lens_dev)):
            self._bind(name, t)
        if self.tables_dev is not None:
            self._bind("rules.tables", self.tables_dev)
        # lend_workspace=False: a host with no scratch memory to give; only the entry points that bring their own
        # scratch (logmel_static) work then, the others answer WDZ_ENOMEM
        self.workspace = None
        if lend_workspace:
            need = C.c_size_t()
            self._check(self.lib.wdz_workspace_bytes(self.h, C.byref(need)))
            self.workspace = torch.empty(need.value, dtype=torch.uint8, device=dev)
            self._check(self.lib.wdz_set_workspace(self.h, self.workspace.data_ptr(), need.value))
        self._check(self.lib.wdz_finalize(self.h))

    # ------------------------------------------------------------------ util
    def _bind(self, name: str, t: torch.Tensor) -> None:
        assert t.is_cuda and t.is_contiguous()
        self._check(self.lib.wdz_bind(self.h, name.encode(), t.data_ptr(), t.numel()))

    def _check(self, rc: int) -> None:
        if rc != capi.WDZ_OK:
            raise capi.WdzError(rc, self.lib.wdz_last_error(self.h).decode())

    def _stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def _i32(self, x) -> torch.Tensor:
        if isinstance(x, torch.Tensor):
            return x.to(device=self.device, dtype=torch.int32).contiguous()
        return torch.tensor(list(x), dtype=torch.int32, device=self.device)

    def close(self) -> None:
        if getattr(self, "h", None):
            torch.cuda.synchronize(self.device)
            self.lib.wdz_engine_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def device_status(self) -> None:
        """Raises if a kernel flagged an error: an exhausted wait, a NaN logits row, what the 8-bit cache was given.  Tells
        of one at a time, so ask until it returns."""
        self._check(self.lib.wdz_device_status(self.h, self._stream()))

    def decode_status(self) -> None:
        """``device_status`` for the engine's own kernels alone: a store into somebody's 8-bit cache is no failed step."""
        self._check(self.lib.wdz_decode_status(self.h, self._stream()))

    # ----------------------------------------------------------- measurement
    def launch_count(self) -> int:
        out = C.c_int64()
        self._check(self.lib.wdz_launch_count(self.h, C.byref(out)))
        return out.value

    def profile(self, enable: bool) -> None:
        self._check(self.lib.wdz_profile(self.h, int(enable)))

    def profile_read(self) -> dict:
        """{kind: {"ms", "launches", "work"}} for the launches recorded since profile(True)."""
        res = {}
        for name, kind in capi.PROF_KINDS.items():
            ms, n, work = C.c_double(), C.c_int64(), C.c_double()
            self._check(self.lib.wdz_profile_read(self.h, kind, C.byref(ms), C.byref(n), C.byref(work)))
            res[name] = {"ms": ms.value, "launches": n.value, "work": work.value}
        return res

    # ------------------------------------------------------------- front end
    def _checked_lengths(self, N: int, B: int, n_samples) -> torch.Tensor:
        """Per-clip sample counts as a device tensor; lengths that come from the host are validated there, so that
        the call does not have to wait for the GPU (a device tensor is read back once)."""
        if n_samples is None:
            shortest, ns = N, self._i32([N] * B)
        elif isinstance(n_samples, torch.Tensor):
            ns = self._i32(n_samples)
            shortest = int(ns.min())
        else:
            host = [int(v) for v in n_samples]
            shortest, ns = min(host), self._i32(host)
        if shortest < 400:
            raise ValueError("clips shorter than 400 samples cannot be reflect-padded")
        return ns

    def logmel(self, audio: torch.Tensor, n_samples=None, frame_offset=None) -> torch.Tensor:
        """audio f32 [B, N] (device) -> mel f32 [B, n_mels, 3000]."""
        audio = audio.to(device=self.device, dtype=torch.float32)
        if audio.dim() == 1:
            audio = audio[None]
        audio = audio.contiguous()
        B, N = audio.shape
        if N > 480000:
            raise ValueError("a window holds at most 30 s (480000 samples)")
        ns = self._checked_lengths(N, B, n_samples)
        fo = None if frame_offset is None else self._i32(frame_offset)
        mel = torch.empty(B, self.dims.n_mels, 3000, dtype=torch.float32, device=self.device)
        self._check(self.lib.wdz_logmel(self.h, audio.data_ptr(), N, ns.data_ptr(),
                                        None if fo is None else fo.data_ptr(), B, mel.data_ptr(), self._stream()))
        return mel

    def logmel_static(self, audio: torch.Tensor, n_samples=None, frame_offset=None) -> torch.Tensor:
        """``logmel`` through the entry point that brings its own scratch: for
        embedders that cannot lend the engine a workspace (all GPU memory
        already handed to another pool, or no tolerance for the stall of a
        device allocation).  At most 4 clips per call; calls share one built-in
        array, so do not overlap them on the GPU; make the first call on a
        device before any stream capture."""
        audio = audio.to(device=self.device, dtype=torch.float32)
        if audio.dim() == 1:
            audio = audio[None]
        audio = audio.contiguous()
        B, N = audio.shape
        if N > 480000:
            raise ValueError("a window holds at most 30 s (480000 samples)")
        ns = self._checked_lengths(N, B, n_samples)
        fo = None if frame_offset is None else self._i32(frame_offset)
        mel = torch.empty(B, self.dims.n_mels, 3000, dtype=torch.float32, device=self.device)
        self._check(self.lib.wdz_logmel_static(self.h, audio.data_ptr(), N, ns.data_ptr(),
                                               None if fo is None else fo.data_ptr(), B, mel.data_ptr(),
                                               self._stream()))
        return mel

    # --------------------------------------------------------------- encoder
    def encode(self, mel: torch.Tensor) -> torch.Tensor:
        mel = mel.to(device=self.device, dtype=torch.float32).contiguous()
        B = mel.shape[0]
        assert mel.shape[1:] == (self.dims.n_mels, 2 * self.dims.n_audio_ctx), mel.shape
        xa = torch.empty(B, self.dims.n_audio_ctx, self.dims.n_audio_state, dtype=self.dtype, device=self.device)
        self._check(self.lib.wdz_encode(self.h, mel.data_ptr(), B, xa.data_ptr(), self._stream()))
        return xa

    def linear(self, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, gelu: bool = False,
               cuda_cores_only: bool | int = False) -> torch.Tensor:
        """act(x @ w.T + bias) in the engine dtype through the engine's GEMM kernels (``cuda_cores_only``: True/1 =
        no tensor cores, 2 = the lone-CTA tcgen05 kernel, no CTA pairs)."""
        x = x.to(device=self.device, dtype=self.dtype).contiguous()
        w = w.to(device=self.device, dtype=self.dtype).contiguous()
        b = None if bias is None else bias.to(device=self.device, dtype=self.dtype).contiguous()
        M, K = x.shape
        N = w.shape[0]
        y = torch.empty(M, N, dtype=self.dtype, device=self.device)
        self._check(self.lib.wdz_linear(self.h, x.data_ptr(), M, K, w.data_ptr(), None if b is None else b.data_ptr(),
                                        N, int(gelu), y.data_ptr(), int(cuda_cores_only), self._stream()))
        return y

    def linear_rows(self, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
        """Decode-shaped product: x [M, K] (engine dtype) @ w[N, K].T (+ bias) -> f32 [M, N];
        with ``out`` given the result is added into it."""
        x = x.to(device=self.device, dtype=self.dtype).contiguous()
        w = w.to(device=self.device, dtype=self.dtype).contiguous()
        b = None if bias is None else bias.to(device=self.device, dtype=self.dtype).contiguous()
        M, K = x.shape
        N = w.shape[0]
        y = out if out is not None else torch.empty(M, N, dtype=torch.float32, device=self.device)
        self._check(self.lib.wdz_linear_rows(self.h, x.data_ptr(), M, K, w.data_ptr(),
                                             None if b is None else b.data_ptr(), N, int(out is not None),
                                             y.data_ptr(), self._stream()))
        return y

    def encoder_attention(self, qkv: torch.Tensor, cuda_cores_only: bool = False) -> torch.Tensor:
        """qkv [B, n_audio_ctx, 3d] -> [B, n_audio_ctx, d] (non-causal, scale 1/8) in the engine dtype."""
        qkv = qkv.to(device=self.device, dtype=self.dtype).contiguous()
        B, T, d3 = qkv.shape
        assert T == self.dims.n_audio_ctx and d3 == 3 * self.dims.n_audio_state and B <= self.max_clips
        out = torch.empty(B, T, d3 // 3, dtype=self.dtype, device=self.device)
        self._check(self.lib.wdz_encoder_attention(self.h, qkv.data_ptr(), B, out.data_ptr(), int(cuda_cores_only),
                                                   self._stream()))
        return out

    # --------------------------------------------------------------- decoder
    def cross_kv(self, xa: torch.Tensor, slots) -> None:
        xa = xa.to(self.dtype).contiguous()
        s = self._i32(slots)
        self._check(self.lib.wdz_cross_kv(self.h, xa.data_ptr(), s.data_ptr(), xa.shape[0], self._stream()))

    def slot_reset(self, slots) -> None:
        s = self._i32(slots)
        self._check(self.lib.wdz_slot_reset(self.h, s.data_ptr(), s.numel(), self._stream()))

    def seq_lens(self) -> list[int]:
        out = (C.c_int32 * self.n_slots)()
        self._check(self.lib.wdz_slot_seqlens(self.h, out, self._stream()))
        return list(out)

    def forward_rows(self, tokens, slots, positions, emit_rows=None, want_logits: bool = True):
        t, s, p = self._i32(tokens), self._i32(slots), self._i32(positions)
        n = t.numel()
        er = None if emit_rows is None else self._i32(emit_rows)
        n_emit = n if er is None else er.numel()
        logits = None
        if want_logits:
            logits = torch.empty(n_emit, self.dims.n_vocab, dtype=torch.float32, device=self.device)
        self._check(self.lib.wdz_forward_rows(
            self.h, t.data_ptr(), s.data_ptr(), p.data_ptr(), n, None if er is None else er.data_ptr(), n_emit,
            None if logits is None else logits.data_ptr(), self._stream()))
        return logits

    def prefill(self, xa: torch.Tensor, window_slots, prompts: list[list[int]], want_logits: bool = True):
        """Cross K/V + slot reset + prompt rows; returns the logits of each
        window's last prompt token, f32 [B, V]."""
        xa = xa.to(self.dtype).contiguous()
        ws = self._i32(window_slots)
        slots_l = [int(v) for v in ws.tolist()]
        tok, sl, pos, emit = [], [], [], []
        for b, pr in enumerate(prompts):
            for j, t in enumerate(pr):
                tok.append(int(t)); sl.append(slots_l[b]); pos.append(j)
            emit.append(len(tok) - 1)
        t, s, p, er = self._i32(tok), self._i32(sl), self._i32(pos), self._i32(emit)
        logits = None
        if want_logits:
            logits = torch.empty(len(emit), self.dims.n_vocab, dtype=torch.float32, device=self.device)
        self._check(self.lib.wdz_prefill(
            self.h, xa.data_ptr(), ws.data_ptr(), xa.shape[0], t.data_ptr(), s.data_ptr(), p.data_ptr(), t.numel(),
            er.data_ptr(), er.numel(), None if logits is None else logits.data_ptr(), self._stream()))
        return logits

    def rules_to_device(self, rules) -> torch.Tensor | None:
        if rules is None:
            return None
        if isinstance(rules, torch.Tensor):
            return rules
        return torch.from_numpy(pack_rules(rules)).to(self.device)

    def decode_step(self, tokens, slots, rules=None, want_logits: bool = False):
        """One step for the given (last token, slot) rows; returns next ids
        (int32, device) and optionally the f32 logits."""
        t, s = self._i32(tokens), self._i32(slots)
        n = t.numel()
        rd = self.rules_to_device(rules)
        out = torch.empty(n, dtype=torch.int32, device=self.device)
        logits = torch.empty(n, self.dims.n_vocab, dtype=torch.float32, device=self.device) if want_logits else None
        self._check(self.lib.wdz_decode_step(
            self.h, t.data_ptr(), s.data_ptr(), n, None if rd is None else rd.data_ptr(), out.data_ptr(),
            None if logits is None else logits.data_ptr(), self._stream()))
        return (out, logits) if want_logits else out

    # ------------------------------------------- rule state kept on the device
    def ts_reset(self, slots, max_new) -> None:
        s, m = self._i32(slots), self._i32(max_new)
        self._check(self.lib.wdz_ts_reset(self.h, s.data_ptr(), m.data_ptr(), s.numel(), self._stream()))

    def ts_first(self, logits: torch.Tensor, slots) -> None:
        logits = logits.to(device=self.device, dtype=torch.float32).contiguous()
        s = self._i32(slots)
        self._check(self.lib.wdz_ts_first(self.h, logits.data_ptr(), s.data_ptr(), s.numel(), self._stream()))

    def ts_steps(self, slots, k: int) -> None:
        s = self._i32(slots)
        self._check(self.lib.wdz_ts_steps(self.h, s.data_ptr(), s.numel(), int(k), self._stream()))

    def ts_poll(self) -> np.ndarray:
        """int32 [n_slots, 24]: max_new, n_new, timing_count, last_timing, last_was_timing, n_recent, done,
        last_token, recent[10], spare[6]."""
        out = np.empty((self.n_slots, 24), dtype=np.int32)
        self._check(self.lib.wdz_ts_poll(self.h, out.ctypes.data, self._stream()))
        return out

    def ts_tokens(self, slot: int, n: int) -> list[int]:
        out = np.empty(max(n, 1), dtype=np.int32)
        self._check(self.lib.wdz_ts_tokens(self.h, int(slot), out.ctypes.data, int(n), self._stream()))
        return out[:n].tolist()

    def reargmax(self, rows, rules) -> torch.Tensor:
        r = self._i32(rows)
        rd = self.rules_to_device(rules)
        out = torch.empty(r.numel(), dtype=torch.int32, device=self.device)
        self._check(self.lib.wdz_reargmax(self.h, r.data_ptr(), None if rd is None else rd.data_ptr(), r.numel(),
                                          out.data_ptr(), self._stream()))
        return out

    def rules_argmax(self, logits: torch.Tensor, rules, penalty: bool = True) -> torch.Tensor:
        logits = logits.to(device=self.device, dtype=torch.float32).contiguous()
        rd = self.rules_to_device(rules)
        out = torch.empty(logits.shape[0], dtype=torch.int32, device=self.device)
        self._check(self.lib.wdz_rules_argmax(self.h, logits.data_ptr(), None if rd is None else rd.data_ptr(),
                                              logits.shape[0], int(penalty), out.data_ptr(), self._stream()))
        return out

    # ------------------------------------------------- 8-bit cache, 4-bit weights
    def qcache(self, n_slots: int | None = None, n_tokens: int | None = None, n_heads: int | None = None) -> QCache:
        """An empty 8-bit cache on the engine's device; by default the engine's slots, its encoder positions and the
        decoder's heads (the shape of one layer's cross cache)."""
        return QCache.empty(self.n_slots if n_slots is None else n_slots, self.dims.n_audio_ctx if n_tokens is None else n_tokens,
                            self.dims.n_text_head if n_heads is None else n_heads, self.device)

    # The calls below take a few microseconds on the device, so their checks are written to cost little on the host.
    def _raw_stream(self) -> int:
        """The current stream's handle, without the object around it."""
        return torch._C._cuda_getCurrentRawStream(self._ordinal)

    def _here(self, name: str, ordinal: int) -> None:
        if ordinal != self._ordinal:
            raise ValueError(f"{name} does not lie on the engine's device")

    def _rows(self, name: str, t: torch.Tensor, width: int) -> torch.Tensor:
        """``t`` as rows [n, width] in a type and at places that the kernels take: no copy where it has them already."""
        if t.dim() == 3 and t.shape[2] == HEAD_DIM:
            t = t.flatten(1)
        if t.dtype not in _TORCH_DTYPE or t.dim() != 2 or t.shape[1] != width:
            raise ValueError(f"{name} must be [rows, {width}] in float32 or bfloat16, got {t.dtype} {tuple(t.shape)}")
        self._here(name, t.get_device())
        step, one = t.stride()
        if one != 1 or (step < width and t.shape[0] > 1) or step * t.element_size() % 16 or t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def _index(self, name: str, x, n: int) -> torch.Tensor:
        """An int32 index tensor of ``n`` entries on the device; host sequences are uploaded.  Entries that no int32 holds
        become its ends: outside every cache, longer than every row."""
        if isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.numel() == n and x.is_contiguous() and x.get_device() == self._ordinal:
            return x
        lo, hi = -2 ** 31, 2 ** 31 - 1
        if not isinstance(x, torch.Tensor):
            x = [min(max(v, lo), hi) for v in self._whole(name, x)]
        elif x.dtype not in _INDEX_DTYPES:
            raise ValueError(f"{name} must be whole numbers of a signed type or uint8, got {x.dtype}")
        elif x.dtype is torch.int64:
            x = x.clamp(lo, hi)
        x = self._i32(x)
        if x.numel() != n:
            raise ValueError(f"{name} must have {n} entries, got {tuple(x.shape)}")
        return x

    @staticmethod
    def _whole(name: str, values) -> list[int]:
        values = list(values)
        whole = [int(v) for v in values]
        if any(w != v for w, v in zip(whole, values)):
            raise ValueError(f"{name} must be whole numbers")
        return whole

    def qcache_store(self, cache: QCache, k: torch.Tensor, v: torch.Tensor, slots, positions, row_begin=None,
                     max_run: int | None = None) -> None:
        """Rounds rows of keys and values into an 8-bit cache, in place (what ``cross_kv`` and a decode step's append do
        in 16 bits, model.py:98-147).

        k, v: f32 or bf16 [n, heads * 64] (or [n, heads, 64]); columns of a fused product are taken as they lie.  Run i
        is rows row_begin[i] .. row_begin[i + 1] (``None``: one row a run) and goes to tokens positions[i], ... of slot
        slots[i].  A block of 64 tokens that a run enters at its first token gets the scale max|x| / 127 of the run's
        own values; one that is entered later keeps the larger of that and its scale, and what it holds is rounded to
        it.  A slot of the cache may be named once; ``max_run`` sizes the launch when row_begin is on the device (default: all
        rows).  Non-finite values, places outside the cache and slots named twice are told by ``device_status()``;
        slots outside the cache are skipped."""
        width = cache.n_heads * HEAD_DIM
        self._here("the cache", cache.ordinal)
        if not cache.apart:
            raise ValueError("qcache_store: the cache's keys and values lie in one place")
        k, v = self._rows("k", k, width), self._rows("v", v, width)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have the same shape and type")
        n = k.shape[0]
        rb = None
        if row_begin is None:
            n_runs, most = n, 1
        else:
            if not isinstance(row_begin, torch.Tensor):
                row_begin = self._whole("row_begin", row_begin)
                if not row_begin or row_begin[0] < 0 or row_begin[-1] > n or any(b > c for b, c in zip(row_begin, row_begin[1:])):
                    raise ValueError(f"row_begin must rise from 0 or more to at most {n}")
                if max_run is None:
                    max_run = max((c - b for b, c in zip(row_begin, row_begin[1:])), default=0)
            n_runs = len(row_begin) - 1
            if n_runs < 0:
                raise ValueError("row_begin has one entry more than there are runs")
            rb = self._index("row_begin", row_begin, n_runs + 1)
            most = n if max_run is None else int(max_run)
        if not isinstance(slots, torch.Tensor):
            slots = self._whole("slots", slots)
            kept = [x for x in slots if 0 <= x < cache.n_slots]   # the others are skipped, however often
            if len(set(kept)) != len(kept):
                raise ValueError("qcache_store: a slot is named twice")
        sl, ps = self._index("slots", slots, n_runs), self._index("positions", positions, n_runs)
        if n == 0 or n_runs == 0:
            return
        rc = self.lib.wdz_qcache_store(
            self.h, cache.ref, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), _TORCH_DTYPE[k.dtype], n,
            None if rb is None else rb.data_ptr(), sl.data_ptr(), ps.data_ptr(), n_runs, most, self._raw_stream())
        if rc:
            self._check(rc)

    def qcache_attention(self, q: torch.Tensor, cache: QCache, slots, lens, scale: float = HEAD_DIM ** -0.5,
                         out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Decode attention over an 8-bit cache (the cached branch of qkv_attention, model.py:336-359): row r's query
        heads attend to the first lens[r] tokens of slot slots[r].

        q: f32 or bf16 [n, q_heads * 64] (or [n, q_heads, 64]); q_heads is the cache's head count or a multiple of it up
        to 8, consecutive query heads sharing a key head.  Returns [n, q_heads * 64] in ``out_dtype`` (default: the
        engine's type), or fills ``out``, which may be q itself.  Length 0 gives zeros; a row whose slot lies outside the cache is left as it
        was (zeros when ``out`` is not given)."""
        if q.dim() == 3 and q.shape[2] == HEAD_DIM:
            q = q.flatten(1)
        elif q.dim() != 2:
            raise ValueError(f"q must be [rows, q_heads * {HEAD_DIM}] or [rows, q_heads, {HEAD_DIM}], got {tuple(q.shape)}")
        n, width = q.shape
        shared, rest = divmod(width, cache.n_heads * HEAD_DIM)
        if rest or not 1 <= shared <= 8:
            raise ValueError(f"q must have 1 to 8 times the cache's {cache.n_heads} heads of {HEAD_DIM}, got {tuple(q.shape)}")
        ordinal = self._ordinal
        if cache.ordinal != ordinal or q.get_device() != ordinal:
            raise ValueError("q and the cache must lie on the engine's device")
        code = _TORCH_DTYPE.get(q.dtype)
        if code is None:
            raise ValueError(f"q must be float32 or bfloat16, got {q.dtype}")
        step, one = q.stride()
        at = q.data_ptr()
        if one != 1 or (step < width and n > 1) or step % (8 if code else 4) or at % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            step, at = width, q.data_ptr()
        if out is None:
            to = _TORCH_DTYPE.get(out_dtype or self.dtype)
            if to is None:
                raise ValueError("out_dtype must be float32 or bfloat16")
            clear, out, out_step = 1, q.new_empty((n, width), dtype=out_dtype or self.dtype), width
        else:
            to, clear = _TORCH_DTYPE.get(out.dtype), 0
            if (to is None or out_dtype not in (None, out.dtype) or tuple(out.shape) != (n, width) or out.stride(1) != 1
                    or (n > 1 and out.stride(0) < width) or out.stride(0) % (8 if to else 4) or out.data_ptr() % 16):
                raise ValueError(f"out must be [{n}, {width}] rows in float32 or bfloat16 that start on 16 bytes")
            self._here("out", out.get_device())
            out_step = out.stride(0)
            to_at, q_size, out_size = out.data_ptr(), 2 if code else 4, 2 if to else 4
            same = to_at == at and to == code and (n == 1 or out_step == step)
            if not same and rows_overlap(n, at, step * q_size, width * q_size, to_at, out_step * out_size, width * out_size):
                raise ValueError("out may be q itself, but not lie over a part of it")
        slots, lens = self._index("slots", slots, n), self._index("lens", lens, n)
        if n == 0:
            return out
        need = cache.scratch.get((n, shared))
        if need is None:
            need = cache.scratch[(n, shared)] = max(0, self.lib.wdz_qcache_attention_scratch(self.h, cache.ref, width // HEAD_DIM, n))
        scratch = q.new_empty(need, dtype=torch.uint8) if need else None
        rc = self.lib.wdz_qcache_attention(
            self.h, cache.ref, at, step, code, width // HEAD_DIM, slots.data_ptr(), lens.data_ptr(), n, scale, out.data_ptr(),
            out_step, to, clear, scratch.data_ptr() if need else None, need, torch._C._cuda_getCurrentRawStream(ordinal))
        if rc:
            self._check(rc)
        return out

    def linear_rows_packed(self, x: torch.Tensor, w: PackedLinear, residual: torch.Tensor | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
        """``linear_rows`` with 4-bit weights (``lowbit.pack_linear``): x f32 or bf16 [M, K] @ W[N, K].T (+ bias)
        (+ residual f32 [M, N]) -> f32 [M, N].  ``residual`` and ``out`` may be the same tensor; ``out`` may not lie over x.

        Made for few rows: from about 48 bf16 rows on ``linear_rows`` on bf16 weights takes less time (include/wdz.h).
        As in ``linear_rows`` the bias has the rows' type: one of the other type is converted in every call, which rounds an
        f32 bias to bf16 under bf16 rows and costs a launch.  An f32 bias that must not be rounded goes in with ``residual``,
        which is added in f32."""
        code, ordinal = _TORCH_DTYPE.get(x.dtype), self._ordinal
        if code is None or x.dim() != 2:
            raise ValueError(f"x must be [rows, {w.in_features}] in float32 or bfloat16, got {x.dtype} {tuple(x.shape)}")
        M, K = x.shape
        if K != w.in_features:
            raise ValueError(f"x must be [rows, {w.in_features}], got {tuple(x.shape)}")
        if w.ordinal != ordinal or x.get_device() != ordinal:
            raise ValueError("x and the weights must lie on the engine's device")
        step, one = x.stride()
        if one != 1 or (step < K and M > 1):
            x = x.clone(memory_format=torch.contiguous_format)
            step = K
        N = w.out_features
        add = None
        if residual is not None:
            add = self._f32_rows("residual", residual, M, N).data_ptr()
        if out is None:
            out = x.new_empty((M, N), dtype=torch.float32)
        else:
            self._f32_rows("out", out, M, N)
            size, to_at = 2 if code else 4, out.data_ptr()
            if (rows_overlap(M, x.data_ptr(), step * size, K * size, to_at, 4 * N, 4 * N)
                    or (add is not None and add != to_at and abs(add - to_at) < 4 * M * N)):
                raise ValueError("out may be residual itself, but not lie over x or a part of residual")
        b = w.bias
        if b is not None and b.dtype is not x.dtype:
            b = b.to(x.dtype)   # not kept: the caller may write into the bias
        rc = self.lib.wdz_linear_rows_packed(
            self.h, x.data_ptr(), step, code, M, K, w.at, w.scale_at, w.group, None if b is None else b.data_ptr(), add, N,
            out.data_ptr(), torch._C._cuda_getCurrentRawStream(ordinal))
        if rc:
            self._check(rc)
        return out

    def _f32_rows(self, name: str, t: torch.Tensor, M: int, N: int) -> torch.Tensor:
        if t.dtype is not torch.float32 or tuple(t.shape) != (M, N) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 [{M}, {N}]")
        self._here(name, t.get_device())
        return t

    # ------------------------------------------------------- word-timing alignment
    def align_configure(self, heads) -> None:
        """(layer, head) pairs whose cross-attention tracks time (dtw_align.py:52-62)."""
        arr = np.ascontiguousarray(np.asarray(heads, dtype=np.int32).reshape(-1, 2))
        self._check(self.lib.wdz_align_configure(self.h, arr.ctypes.data, arr.shape[0]))
        self.align_heads = [tuple(int(v) for v in r) for r in arr]

    def align_capacity(self, t_pad: int) -> int:
        return int(self.lib.wdz_align_capacity(self.h, int(t_pad)))

    def align_matrix(self, tokens, lens, slots, audio_caps) -> torch.Tensor:
        """tokens int [B, T] (``alignment.build_full_tokens``), lens / slots / audio_caps [B] ->
        f32 [B, T, n_audio_ctx] on the device: the cost matrix before negation, rows past a chunk's length
        zero (dtw_align.py:1181-1195).  Slots must be distinct; more chunks than one call takes are run
        in several calls."""
        tok = torch.as_tensor(np.asarray(tokens), dtype=torch.int32)
        B, T = tok.shape
        if len(set(int(s) for s in slots)) != B:
            raise ValueError("align_matrix: the chunks of one call must sit in distinct slots")
        out = torch.empty(B, T, self.dims.n_audio_ctx, dtype=torch.float32, device=self.device)
        cap = self.align_capacity(T)
        if cap < 1:
            raise capi.WdzError(-5, f"no room to align chunks of {T} tokens (configure heads first)")
        tok_d = tok.to(self.device)
        lens_d, slots_d, caps_d = self._i32(lens), self._i32(slots), self._i32(audio_caps)
        for b0 in range(0, B, cap):
            n = min(cap, B - b0)
            self._check(self.lib.wdz_align_matrix(
                self.h, tok_d[b0:b0 + n].contiguous().data_ptr(), lens_d[b0:].data_ptr(), slots_d[b0:].data_ptr(),
                caps_d[b0:].data_ptr(), n, T, out[b0:].data_ptr(), self._stream()))
        return out

    def dtw(self, matrix: torch.Tensor, row0, n_rows, n_cols, limits=None):
        """Minimum-cost monotonic paths through ``-matrix[b, row0[b] : row0[b] + n_rows[b], : n_cols[b]]``
        (dtw_align.py:170-223).  ``limits`` = per chunk (lo, hi) int arrays [n_rows[b]]: columns outside
        [lo, hi) of a row cost +inf (anchor bands, dtw_align.py:589-641).  Returns [(text_idx, time_idx)]
        as int64 numpy arrays."""
        matrix = matrix.to(device=self.device, dtype=torch.float32)
        if matrix.dim() == 2:
            matrix = matrix[None]
        matrix = matrix.contiguous()
        B = matrix.shape[0]
        max_rows, max_cols = max(1, max(n_rows)), max(1, max(n_cols))
        lo_d = hi_d = None
        if limits is not None:
            lo = np.zeros((B, max_rows), dtype=np.int32)
            hi = np.zeros((B, max_rows), dtype=np.int32)
            for b, (l, h) in enumerate(limits):
                lo[b, : len(l)] = l
                hi[b, : len(h)] = h
            lo_d, hi_d = torch.from_numpy(lo).to(self.device), torch.from_numpy(hi).to(self.device)
        cap = max_rows + max_cols
        ti = torch.empty(B, cap, dtype=torch.int32, device=self.device)
        tj = torch.empty(B, cap, dtype=torch.int32, device=self.device)
        ln = torch.empty(B, dtype=torch.int32, device=self.device)
        row0_d, rows_d, cols_d = self._i32(row0), self._i32(n_rows), self._i32(n_cols)   # kept alive past the launch
        if min(int(r) for r in row0) < 0 or max(int(r) + int(n) for r, n in zip(row0, n_rows)) > matrix.shape[1] \
                or max_cols > matrix.shape[2]:
            raise ValueError("dtw: a chunk's rows or columns lie outside the matrix")
        self._check(self.lib.wdz_dtw(
            self.h, matrix.data_ptr(), matrix.stride(0), matrix.stride(1), row0_d.data_ptr(),
            rows_d.data_ptr(), cols_d.data_ptr(),
            None if lo_d is None else lo_d.data_ptr(), None if hi_d is None else hi_d.data_ptr(), max_rows, B,
            max_rows, max_cols, ti.data_ptr(), tj.data_ptr(), ln.data_ptr(), self._stream()))
        ti_h, tj_h, ln_h = ti.cpu().numpy(), tj.cpu().numpy(), ln.cpu().numpy()
        return [(ti_h[b, : ln_h[b]].astype(np.int64), tj_h[b, : ln_h[b]].astype(np.int64)) for b in range(B)]
