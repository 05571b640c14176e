// The 8-bit key/value cache: storing rows into it and attending over it.
//
//   value(slot, head, token, c) = int8[slot][head][token][c] * scale[slot][head][token / 64]     (K and V alike)
//
//   qcache_store_kernel, qcache_step_kernel - round rows into the cache: s = max|x| / 127 over the 64 tokens x 64 values
//       of a block, q = rint(x / s).  A block that is continued keeps the larger scale, and what it held is rounded to it.
//   qcache_attend_kernel, qcache_merge_kernel - one query row per (slot, length): softmax(scale * q K^T) V over the slot's first tokens.
#pragma once
#include "../../include/wdz.h"
#include "attention.cuh"
#include "common.cuh"
#include "gemv_packed.cuh"

namespace wdz {

constexpr int QC_BLOCK = WDZ_QCACHE_BLOCK;   // tokens that share a scale
constexpr int QC_HD = 64;
constexpr float QC_TINY = 6.0185310762e-36f;   // 2^-117: below it the store's remainders would underflow; such a block is zero
constexpr float QC_LEAST = 4.7019774033e-38f;  // 2^-124: no store leaves a smaller scale than that of QC_TINY, but a caller's cache may

struct QcView {
  int8_t *k, *v;
  float *ks, *vs;
  int64_t slot_stride, scale_stride;
  int n_slots, n_heads, n_blocks;
};

struct QcStoreParams {
  QcView c;
  const void *k, *v;
  int64_t ldk, ldv;
  int n_rows, n_runs;
  const int *row_begin, *slots, *positions;
};

// ---- store ---------------------------------------------------------------------------------------------------------
// Bound by the rows' bytes (2 or 4 a value) and the cache's (1).  rint(x / s) has to be exact, a value next to a half step
// included, at a few instructions a value: x is multiplied by the two floats next to 1 / s, above and below, and each product
// is rounded to a whole number by the same fused multiply-add with 1.5 2^23.  x / s lies strictly between the products and
// rounding is monotonic, so where the two agree that is the result.  Where they differ (near a half step: 1 value in 1000 of
// bf16 rows, whose quotients by a bf16 maximum often are nearly halves) the sign of x - h s, h the half between them, tells:
// h s has at most 32 bits and a fused multiply-add rounds only the difference, which keeps its sign.

// rint(x / s), half to even, for values that need not be finite, settled by the remainder x - q s: it has so few bits that a
// fused multiply-add gives it without rounding wherever it decides (q s is a multiple of s's last bit, x of s's last bit / 2
// or less, and |x - q s| <= s / 2 needs 24 of those).
__device__ __forceinline__ int qc_code(float x, float s, float inv) {
  const float lim = fminf(fmaxf(x * inv, -127.0f), 127.0f);   // infinities saturate; NaN becomes a bound and is set aside below
  float q = rintf(lim);
  const float d = fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (d > half || (d == half && odd)) q += 1.0f;
  if (d < -half || (d == -half && odd)) q -= 1.0f;
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  return x == x && s > 0.0f ? (int)q : 0;
}

// What a block's values are divided by: the scale, 1 / scale rounded, and the floats next to that.  Scale 0 makes zeros.
struct QcDivisor {
  float s, inv, above, below;
  __device__ explicit QcDivisor(float scale) : s(scale) {
    inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    above = scale > 0.0f ? __uint_as_float(__float_as_uint(inv) + 1) : 0.0f;
    below = scale > 0.0f ? __uint_as_float(__float_as_uint(inv) - 1) : 0.0f;
  }
};

__device__ __forceinline__ uint2 qc_bytes(const uint32_t (&n)[8]) {
  const uint32_t a = __byte_perm(n[0], n[1], 0x0040), b = __byte_perm(n[2], n[3], 0x0040);
  const uint32_t c = __byte_perm(n[4], n[5], 0x0040), d = __byte_perm(n[6], n[7], 0x0040);
  return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410));
}
// Eight finite values -> eight bytes.
__device__ __forceinline__ uint2 qc_code8(const float (&x)[8], const QcDivisor& by) {
  constexpr float MAGIC = 12582912.0f;   // 1.5 2^23: the sums' bits are its bits plus the whole number
  uint32_t n[8], other[8], differ = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    n[i] = __float_as_uint(fmaf(x[i], by.above, MAGIC));
    other[i] = __float_as_uint(fmaf(x[i], by.below, MAGIC));
    differ |= n[i] ^ other[i];
  }
  if (differ) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float half = 0.5f * ((__uint_as_float(n[i]) - MAGIC) + (__uint_as_float(other[i]) - MAGIC));
      const float d = fmaf(-half, by.s, x[i]);
      const uint32_t even = n[i] & 1 ? other[i] : n[i];
      n[i] = d > 0.0f ? max(n[i], other[i]) : d < 0.0f ? min(n[i], other[i]) : even;
    }
  }
  return qc_bytes(n);
}
// Eight values that need not be finite, and scales below QC_LEAST, which values below QC_TINY left as they were: 1 / scale may
// overflow there and values be more than 127 scales, so both are taken 2^64 times.
__device__ __forceinline__ uint2 qc_settle8(const float (&x)[8], float scale) {
  const float lift = scale < QC_LEAST ? 18446744073709551616.0f : 1.0f, s = scale * lift, inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  uint32_t n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = (uint32_t)qc_code(x[i] * lift, s, inv);
  return qc_bytes(n);
}

// What a block's bytes are multiplied by when its scale grows: s_old / s_new rounded, and the floats next to that.
struct QcRatio {
  float s_old, s_new, above, below;
  __device__ QcRatio(float o, float n) : s_old(o), s_new(n) {
    const uint32_t r = __float_as_uint(__fdiv_rn(o, n));
    above = __uint_as_float(r + 1);
    below = __uint_as_float(r ? r - 1 : 0);
  }
};

// rint(q s_old / s_new), half to even, of eight bytes: by the same bracket, and by the exact difference of the products, which
// 64 bits hold, where its ends differ.
__device__ __forceinline__ uint2 qc_recode8(uint2 w, const QcRatio& by) {
  constexpr float MAGIC = 12582912.0f;
  uint32_t n[8], differ = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    n[i] = __float_as_uint(fmaf(q, by.above, MAGIC));
    differ |= n[i] ^ __float_as_uint(fmaf(q, by.below, MAGIC));
  }
  if (differ) {
    const double so = by.s_old, sn = by.s_new, half = 0.5 * sn;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const int q = (int)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
      int m = __float2int_rn((float)q * by.above);
      const double d = (double)q * so - (double)m * sn;
      const bool odd = m & 1;
      if (d > half || (d == half && odd)) ++m;
      else if (d < -half || (d == -half && odd)) --m;
      if (i < 4) w.x = (w.x & ~(255u << (8 * i))) | (uint32_t)(m & 255) << (8 * i);
      else w.y = (w.y & ~(255u << (8 * i - 32))) | (uint32_t)(m & 255) << (8 * i - 32);
    }
    return w;
  }
  return qc_bytes(n);
}

// Pieces i0, i0 + step, .. below n, of eight bytes each, at(i) their places: rounded to a grown scale, four loads at a time.
template <typename At, typename By>
__device__ __forceinline__ void qc_recode(int i0, int n, int step, At at, By by) {
  for (int i = i0; i < n; i += 4 * step) {
    uint2 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) if (i + j * step < n) w[j] = *at(i + j * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) if (i + j * step < n) *at(i + j * step) = qc_recode8(w[j], by(i + j * step));
  }
}

// words: the engine's status words.  The first of a kind counts until it is read.
__device__ __forceinline__ void qc_report(DevStatus* words, int code, int detail) {
  DevStatus* st = words + (code == WDZ_ETIMEOUT ? STATUS_OP_WAIT : STATUS_OP_DATA);
  if (atomicCAS(&st->code, 0, code) == 0) st->detail = detail;
}

// The larger of two magnitudes, NaN if one is.
__device__ __forceinline__ float qc_max(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// Magnitudes in their bits' order: numbers, infinity, NaN.
__device__ __forceinline__ uint32_t qc_bits(float magnitude) { return __float_as_uint(magnitude) & 0x7fffffffu; }

// Eight neighbouring values of a row, as they lie.
template <typename T> struct QcRaw;
template <> struct QcRaw<bf16> {
  uint4 v = make_uint4(0, 0, 0, 0);
  __device__ QcRaw() {}
  __device__ explicit QcRaw(const uint8_t* staged) : v(*reinterpret_cast<const uint4*>(staged)) {}   // as the store kernel lays it
  __device__ void load(const void* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  // the largest magnitude so far and these; NaN stays
  __device__ float top(float m) const {
    __nv_bfloat162 x[4];
    memcpy(x, &v, 16);
    const __nv_bfloat162 y = __hmax2_nan(__hmax2_nan(__habs2(x[0]), __habs2(x[1])), __hmax2_nan(__habs2(x[2]), __habs2(x[3])));
    return qc_max(m, __bfloat162float(__hmax_nan(__low2bfloat16(y), __high2bfloat16(y))));
  }
};
template <> struct QcRaw<float> {
  float4 a = make_float4(0, 0, 0, 0), b = a;
  __device__ QcRaw() {}
  __device__ explicit QcRaw(const uint8_t* staged) : a(*reinterpret_cast<const float4*>(staged)), b(*reinterpret_cast<const float4*>(staged + 512)) {}
  __device__ void load(const void* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ float top(float m) const {
    float x[8];
    get(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = qc_max(m, fabsf(x[i]));
    return m;
  }
};
template <typename T>
__device__ __forceinline__ float qc_finite_top(const QcRaw<T>& r, float m) {   // the same without infinities and NaN
  float x[8];
  r.get(x);
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fabsf(x[i]) <= 3.402823466e38f ? fmaxf(m, fabsf(x[i])) : m;
  return m;
}

// A run's place; ok is false where it cannot be stored, `outside` where that has to be reported.
struct QcRun {
  int slot, p0, p1, r0;
  bool ok, outside;
  __device__ QcRun(const QcStoreParams& p, int run) {
    slot = p.slots[run];
    p0 = p.positions[run];
    r0 = p.row_begin ? p.row_begin[run] : run;
    const int r1 = p.row_begin ? p.row_begin[run + 1] : run + 1, room = p.c.n_blocks * QC_BLOCK;
    ok = slot >= 0 && slot < p.c.n_slots && r1 > r0;
    outside = ok && (r0 < 0 || r1 > p.n_rows || p0 < 0 || p0 > room - (r1 - r0));
    ok = ok && !outside;
    p1 = ok ? p0 + (r1 - r0) : 0;
  }
  // By all threads of the block, while the rows are on their way: does a later run name the slot?  The last one counts.
  __device__ bool named_again(const QcStoreParams& p, int run) const {
    int again = 0;
    for (int j = run + 1 + threadIdx.x; j < p.n_runs; j += blockDim.x) again |= p.slots[j] == slot;
    return __syncthreads_or(again);
  }
};

// Where a head's K or V lies.
struct QcPlace {
  int8_t* q;
  float* s;
  __device__ QcPlace(const QcView& c, int slot, int head, bool is_v) {
    q = (is_v ? c.v : c.k) + slot * c.slot_stride + (int64_t)head * c.n_blocks * (QC_BLOCK * QC_HD);
    s = (is_v ? c.vs : c.ks) + slot * c.scale_stride + (int64_t)head * c.n_blocks;
  }
};

__device__ __forceinline__ float qc_scale(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  return top >= QC_TINY ? __fdiv_rn(top, 127.0f) : 0.0f;
}

// Runs of any length.  A unit is a block of 64 tokens of one head, K or V, and belongs to one warp, which keeps it in shared
// memory between the maximum and the rounding, so the rows are read once.  A lane has 8 neighbouring values of a token, four
// tokens at a time, and reads back only what it brought itself (asynchronous copies): no barrier, and few registers, so that
// the many warps of an SM hide one another's copies.  With few units (SHARE = 4) four warps take a unit's tokens in turn and
// exchange the maximum: then the time is one unit's way through, not the SMs' rate.
// Measured (B200, bf16 rows of 20 heads): 32 windows of 1500 tokens 67 to 70 us, 5.3 to 5.5 TB/s of the 369 MB that have to
// move, issue slots 70 % and DRAM 56 % busy; the rows in registers instead 83 to 100 us (too few warps).  24 prompts of up to
// 223 tokens 10 us.
// Block = 2 units of a warp, or 1 of four; grid = (blocks of the longest run, groups of units, run).
template <typename T> constexpr int QC_UNIT = QC_BLOCK * QC_HD * (int)sizeof(T);   // bytes of a unit's rows

template <typename T, int SHARE>
__global__ void __launch_bounds__((SHARE == 1 ? 2 : SHARE) * 32) qcache_store_kernel(QcStoreParams p, DevStatus* status) {
  constexpr int PIECE = 8 * sizeof(T), STEP = 32 * PIECE;   // bytes of a lane's piece, of all lanes'
  extern __shared__ __align__(16) uint8_t qc_rows[];
  __shared__ uint32_t tops[2][4];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = SHARE > 1 ? warp : 0;
  const int unit = SHARE > 1 ? blockIdx.y : blockIdx.y * 2 + warp;
  uint8_t* mine = qc_rows + (SHARE > 1 ? 0 : warp) * QC_UNIT<T> + lane * 16;   // 16 bytes of each lane side by side
  pdl_wait();
  const QcRun run(p, blockIdx.z);
  const bool reports = blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0;
  if (!run.ok) {
    if (run.outside && reports) qc_report(status, WDZ_EINVAL, 2000000 + (int)blockIdx.z);
    return;
  }
  const bool is_v = unit >= p.c.n_heads;   // 2 n_heads units: the grid has no other
  const int head = is_v ? unit - p.c.n_heads : unit;
  const QcPlace place(p.c, run.slot, head, is_v);
  const int64_t ld = (is_v ? p.ldv : p.ldk) * (int64_t)sizeof(T);
  const char* src = reinterpret_cast<const char*>(is_v ? p.v : p.k) + (int64_t)head * (QC_HD * sizeof(T)) + PIECE * (lane & 7);
  auto over_unit = [&](float top, int round) {
    uint32_t bits = __reduce_max_sync(0xffffffffu, qc_bits(top));
    if (SHARE > 1) {   // the CTA is the unit; each round has words of its own, so one barrier is enough
      if (lane == 0) tops[round][warp] = bits;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < SHARE; ++i) bits = max(bits, tops[round][i]);
    }
    return bits;
  };
  bool asked = false;
  for (int b = run.p0 / QC_BLOCK + blockIdx.x; b * QC_BLOCK < run.p1; b += gridDim.x) {
    const int lo = max(run.p0, b * QC_BLOCK), hi = min(run.p1, (b + 1) * QC_BLOCK), t0 = b * QC_BLOCK + (lane >> 3);
    const int i0 = (lo - b * QC_BLOCK) >> 2, i1 = (hi - b * QC_BLOCK + 3) >> 2;   // steps of four tokens that the run reaches
    const int is = i0 + part;   // this warp's: is, is + SHARE, ..
    const char* from = src + (int64_t)(run.r0 + t0 + 4 * is - run.p0) * ld;   // followed only where the token is the run's
    const uint32_t to_smem = att_smem_u32(mine);
#pragma unroll 4
    for (int i = is; i < i1; i += SHARE, from += 4 * SHARE * ld) {
      const uint32_t bytes = t0 + 4 * i >= lo && t0 + 4 * i < hi ? 16 : 0;   // 0: zeros
      const char* at = bytes ? from : src;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to_smem + i * STEP), "l"(at), "r"(bytes) : "memory");
      if (PIECE == 32)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to_smem + i * STEP + 512), "l"(at + 16), "r"(bytes) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    const bool entered = lo > b * QC_BLOCK;   // behind the block's first token: what it holds stays
    const float old = entered ? place.s[b] : 0.0f;
    const bool again = !asked && run.named_again(p, blockIdx.z);
    asked = true;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (again) {   // nothing has been written yet
      if (reports) qc_report(status, WDZ_EINVAL, 2000000 + (int)blockIdx.z);
      return;
    }
    float top = 0.0f;
#pragma unroll 8
    for (int i = is; i < i1; i += SHARE) top = QcRaw<T>(mine + i * STEP).top(top);
    uint32_t bits = over_unit(top, 0);
    const bool odd = bits >= 0x7f800000u;
    if (odd) {   // an infinity or a NaN: the scale goes by the rest
      top = 0.0f;
#pragma unroll 1
      for (int i = is; i < i1; i += SHARE) top = qc_finite_top(QcRaw<T>(mine + i * STEP), top);
      bits = over_unit(top, 1);
      if (part == 0 && lane == 0) qc_report(status, WDZ_ENAN, 2000000 + (int)blockIdx.z);
    }
    const float now = fmaxf(old, qc_scale(bits));
    if (part == 0 && lane == 0) place.s[b] = now;   // every lane has read the old one
    int8_t* to = place.q + (int64_t)(b * QC_BLOCK + (lane >> 3)) * QC_HD + 8 * (lane & 7);
    if (now > old && entered) {
      const QcRatio ratio(old, now);
      uint2* kept = reinterpret_cast<uint2*>(place.q + (int64_t)b * (QC_BLOCK * QC_HD));
      qc_recode(part * 32 + lane, 8 * (lo - b * QC_BLOCK), 32 * SHARE, [&](int i) { return kept + i; }, [&](int) { return ratio; });
    }
    const QcDivisor by(now);
    if (odd || now < QC_LEAST) {
#pragma unroll 1
      for (int i = is; i < i1; i += SHARE) {
        float x[8];
        QcRaw<T>(mine + i * STEP).get(x);
        if (t0 + 4 * i >= lo && t0 + 4 * i < hi) *reinterpret_cast<uint2*>(to + 4 * i * QC_HD) = qc_settle8(x, now);
      }
    } else {
#pragma unroll 4
      for (int i = is; i < i1; i += SHARE) {
        float x[8];
        QcRaw<T>(mine + i * STEP).get(x);
        const uint2 w = qc_code8(x, by);
        if (t0 + 4 * i >= lo && t0 + 4 * i < hi) *reinterpret_cast<uint2*>(to + 4 * i * QC_HD) = w;
      }
    }
    if (SHARE > 1) __syncthreads();   // before the next block writes its words
  }
}

// One row a run (a decode step).  Block = a run; eight threads a head of K or V.  Where a scale grows, the whole block
// rounds the unit's earlier tokens to it together: alone, its eight threads would take up to 63 turns.
// Measured (384 f32 rows of 20 heads): 3.0 us, a launch's latency, where no scale grows; 6.8 us a step on average while 128
// random tokens are appended one by one; 70 us when nine in ten scales grow at once over half-filled blocks.
template <typename T>
__global__ void __launch_bounds__(320, 3) qcache_step_kernel(QcStoreParams p, DevStatus* status) {
  constexpr int UNITS = 320 / 8;
  __shared__ float olds[UNITS], news[UNITS];
  __shared__ int grown[UNITS], n_grown;
  pdl_trigger();
  const int c = threadIdx.x & 7, mine = threadIdx.x >> 3, units = 2 * p.c.n_heads;
  pdl_wait();
  const QcRun run(p, blockIdx.x);
  if (run.outside && threadIdx.x == 0) qc_report(status, WDZ_EINVAL, 2000000 + (int)blockIdx.x);
  if (!run.ok) return;
  if (run.named_again(p, blockIdx.x)) {
    if (threadIdx.x == 0) qc_report(status, WDZ_EINVAL, 2000000 + (int)blockIdx.x);
    return;
  }
  const int b = run.p0 / QC_BLOCK, kept = run.p0 % QC_BLOCK;
  for (int first = 0; first < units; first += UNITS) {
    const int unit = first + mine;
    const bool has = unit < units, is_v = unit >= p.c.n_heads;
    const int head = has ? (is_v ? unit - p.c.n_heads : unit) : 0;
    const QcPlace place(p.c, run.slot, head, is_v);
    __syncthreads();
    if (threadIdx.x == 0) n_grown = 0;
    QcRaw<T> raw;
    float old = 0.0f;
    if (has) {
      raw.load(reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)run.r0 * (is_v ? p.ldv : p.ldk) + head * QC_HD + 8 * c);
      if (kept) old = place.s[b];
    }
    uint32_t top = qc_bits(raw.top(0.0f));
    auto over8 = [&] {
#pragma unroll
      for (int i = 4; i > 0; i >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, i));
    };
    over8();
    const bool odd = top >= 0x7f800000u;
    if (__any_sync(0xffffffffu, odd)) {
      if (odd) top = qc_bits(qc_finite_top(raw, 0.0f));
      over8();
      if (odd && c == 0) qc_report(status, WDZ_ENAN, 2000000 + (int)blockIdx.x);
    }
    const float now = fmaxf(old, qc_scale(top));
    __syncthreads();
    if (has) {
      float x[8];
      raw.get(x);
      const QcDivisor by(now);
      *reinterpret_cast<uint2*>(place.q + (int64_t)run.p0 * QC_HD + 8 * c) = odd || now < QC_LEAST ? qc_settle8(x, now) : qc_code8(x, by);
      if (c == 0) {
        if (!kept || now > old) place.s[b] = now;
        if (kept && now > old) {
          const int i = atomicAdd(&n_grown, 1);   // the order of the list does not matter
          grown[i] = unit; olds[i] = old; news[i] = now;
        }
      }
    }
    __syncthreads();
    const int pieces = 8 * kept;   // of 8 bytes, a unit
    qc_recode(threadIdx.x, n_grown * pieces, blockDim.x,
              [&](int i) {
                const int g = grown[i / pieces];
                const QcPlace to(p.c, run.slot, g >= p.c.n_heads ? g - p.c.n_heads : g, g >= p.c.n_heads);
                return reinterpret_cast<uint2*>(to.q + (int64_t)b * (QC_BLOCK * QC_HD)) + i % pieces;
              },
              [&](int i) { return QcRatio(olds[i / pieces], news[i / pieces]); });
  }
}

// ---- attention ---------------------------------------------------------------------------------------------------------
struct QcAttendParams {
  QcView c;
  const void* q; int64_t ldq;
  void* out; int64_t ldo;
  const int *slots, *lens;
  int n_rows, group;        // query heads per key head
  float scale;
  bool clear_skipped;       // rows of slots outside the cache: zeros instead of what was there
  float* part;              // partial results [row, key head][parts], when the CTAs of a row are no cluster
};

// One query row per slot is a matrix-vector product, bound by the bytes of K and V.  Taking the bytes apart on the CUDA
// cores would cost more instructions than there are issue slots at the memory's rate (about 1400 a tile of 8 KB and
// scheduler), so both products run on the integer matrix instruction m16n8k32, which takes the cache's bytes as they lie:
//
//   scores   A = 16 tokens x 32 values of K (s8), B = the query, written as a whole number of 32 bits times a scale,
//            N = 2^24 d3 + 2^16 d2 + 2^8 d1 + d0 with signed bytes d: four of the instruction's eight columns.  Sums of
//            products of bytes are exact, so a score has the precision of an fp32 query.
//   output   A = 16 values x 32 tokens of V (s8), B = the softmax weights of the tokens, p in [0, 1] as four unsigned
//            bytes in units of 2^-32.
//
// A query head's columns are d1, d0, d3, d2: the two columns that a lane of the result holds are (d1, d0) or (d3, d2),
// and it folds them as 256 a + b in 32 bits.  Two heads of a group fill the eight columns.
//
// Tile = 64 tokens = one scale.  Lane (g, t) = (lane / 4, lane % 4).  Rows and contraction labels of the instruction
// are names only, so they are given out such that loads are whole 16- or 8-byte pieces of a token and no byte of K moves:
//   K    lane loads 16 values (16 t ..) of token 32 (j / 4) + 16 (g / 4) + 4 (j % 4) + g % 4, j = 0..7
//   V    lane loads 8 values (8 g ..) of token 32 ks + 16 r + 4 b + t; four tokens' bytes are transposed in registers
//   p    the four tokens (ks, r, b = 0..3, t) are the scores j = 4 ks + b of the lanes g = 4 r + t: one lane packs them
//        and one shuffle brings each word to its column.
//
// Measured (B200, 20 heads, one query head each; device time): 384 rows of 1500 tokens 206 us, 7.1 TB/s of K, V and scales
// (a plain version on the CUDA cores: 910 us); 32 rows 23 us; 384 rows of lengths spread over 448 tokens 40 us; one row
// 4.5 us; 2 rows of 32749 tokens, 4 key heads shared by 4 query heads each, 13.4 us with the merge.  Some 700 instructions a
// tile, prologue and merge among them, keep the issue slots 45 % busy at the largest size: the time is the memory's.
constexpr int QC_MAX_WARPS = 4;   // of a CTA
constexpr float QC_STEPS = 127.0f * 16777216.0f;   // a query's largest value in steps: rounding up leaves d3 a byte
constexpr float QC_ONE = 4294967040.0f;            // the weight 1 in steps: the largest fp32 below 2^32
constexpr float QC_LARGE = 18446744073709551616.0f;   // 2^64: block scales up to here are summed as they are

// A signed, B unsigned; the first of a sum starts from zeros.
__device__ __forceinline__ void qc_mma_su(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void qc_mma_su_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ float qc_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void qc_load16(const float* p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 x = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
  }
}
__device__ __forceinline__ void qc_load16(const bf16* p, float (&v)[16]) {
  float a[8], b[8];
  load_vec(p, a);
  load_vec(p + 8, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) { v[i] = a[i]; v[8 + i] = b[i]; }
}
__device__ __forceinline__ void qc_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void qc_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Merges n partial results (largest score m, sum l, weighted sum o) that lie `step` floats apart, for value c.
struct QcMerged { float m, l, o; };
__device__ __forceinline__ QcMerged qc_merge(const float* part, int step, int n, int c) {
  float M = -INFINITY;
  for (int i = 0; i < n; ++i) M = fmaxf(M, part[i * step + QC_HD]);
  QcMerged r{M, 0.0f, 0.0f};
  for (int i = 0; i < n; ++i) {
    const float l = part[i * step + QC_HD + 1];
    const float w = l == 0.0f ? 0.0f : qc_ex2(part[i * step + QC_HD] - M);   // l = 0: no tokens; NaN goes through
    r.l = fmaf(l, w, r.l);
    r.o = fmaf(part[i * step + c], w, r.o);
  }
  return r;
}

// A warp's tiles pass through a ring of its own in shared memory, K and V of a tile in turn, three places of 4 KB: one is
// worked on and two are under way (8 KB a warp).  One lane moves a piece (contiguous, 64 bytes a token, no more tokens than
// the row has) and its scale there with asynchronous copies, so the bytes in flight cost no registers and no warp waits for
// another.  Three places instead of four let a third more warps share an SM.  Waits are bounded.
constexpr int QC_TILE = QC_BLOCK * QC_HD;          // bytes of a tile of K, or V
constexpr int QC_PLACES = 3;
constexpr int QC_PLACE = QC_TILE + 16;             // and its scale
constexpr int QC_RING = QC_PLACES * (QC_PLACE + 8) + 8;   // places, their barriers; a multiple of 16

// Waits for a phase of a barrier, with a limit.  The clock is read only once the wait is seen to be a long one.
__device__ __forceinline__ bool qc_try(uint32_t bar, uint32_t phase) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(phase) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool qc_wait(uint32_t bar, uint32_t phase, DevStatus* status) {
  long long t0 = 0;
  for (int spin = 1; !qc_try(bar, phase); ++spin) {
    if ((spin & 63) == 0) {
      if (t0 == 0) t0 = clock64();
      else if (clock64() - t0 > ATT_WAIT_CYCLES) {
        qc_report(status, WDZ_ETIMEOUT, 2000000 + (int)blockIdx.x);
        return false;
      }
    }
  }
  return true;
}

struct QcRing {
  const uint8_t* base;
  uint32_t addr;              // of base in shared memory
  int place = 0, phase = 0;   // of the piece that is waited for next

  __device__ explicit QcRing(uint8_t* p) : base(p), addr(att_smem_u32(p)) {}
  __device__ const uint8_t* data() const { return base + place * QC_PLACE; }
  __device__ float scale() const { return *reinterpret_cast<const float*>(data() + QC_TILE); }
  __device__ uint32_t bar(int at) const { return addr + QC_PLACES * QC_PLACE + 8 * at; }
  __device__ void init() const {   // by one lane; two arrivals a piece: the bulk copy's and the scale's
#pragma unroll
    for (int i = 0; i < QC_PLACES; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 2;" ::"r"(bar(i)));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // by one lane: a piece of `tokens` tokens into place `at`
  __device__ void fetch(int at, const int8_t* from, const float* scale_from, int tokens) const {
    const uint32_t b = bar(at), dst = addr + at * QC_PLACE, bytes = (uint32_t)tokens * QC_HD;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(from), "r"(bytes), "r"(b) : "memory");
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + QC_TILE), "l"(scale_from) : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(b) : "memory");
  }
  __device__ void step() { if (++place == QC_PLACES) { place = 0; phase ^= 1; } }
  // by the warp: waits for the next piece.  False: the wait ran out and the status word voids the result; the `behind`
  // pieces that are still under way have been given a wait of their own, so that the ring may go.
  __device__ bool wait(int behind, DevStatus* status) {
    if (__all_sync(0xffffffffu, qc_wait(bar(place), phase, status))) return true;
    for (int j = 0; j < behind; ++j) {
      step();
      qc_wait(bar(place), phase, status);
    }
    return false;
  }
};

// A row's place in the cache.
struct QcRow {
  int r, hk, len;
  bool skipped;
  const int8_t *K, *V;
  const float *ks, *vs;
  __device__ QcRow(const QcAttendParams& p, uint32_t item) {
    r = (int)(item / (uint32_t)p.c.n_heads); hk = (int)(item - (uint32_t)r * p.c.n_heads);
    const int slot = p.slots[r];
    const int n = p.lens[r];
    skipped = slot < 0 || slot >= p.c.n_slots;
    len = skipped ? 0 : min(max(n, 0), p.c.n_blocks * QC_BLOCK);
    const int64_t at = skipped ? 0 : slot, head_at = (int64_t)hk * p.c.n_blocks;
    K = p.c.k + at * p.c.slot_stride + head_at * QC_TILE;
    V = p.c.v + at * p.c.slot_stride + head_at * QC_TILE;
    ks = p.c.ks + at * p.c.scale_stride + head_at;
    vs = p.c.vs + at * p.c.scale_stride + head_at;
  }
  __device__ int tiles() const { return (len + QC_BLOCK - 1) / QC_BLOCK; }
  __device__ int tokens(int tile) const { return min(QC_BLOCK, len - tile * QC_BLOCK); }
};

// The query's bytes: lane (g, t) makes column g, values 16 t .. 16 t + 15 of head g / 4 of the pair.
template <typename TQ, int NT>
__device__ __forceinline__ void qc_query(const QcAttendParams& p, int r, int hk, int g, int t, uint32_t (&qb)[NT][4], float (&q_mul)[NT]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = min(2 * nt + (g >> 2), p.group - 1);
    float x[16], top = 0.0f, odd = 0.0f;
    qc_load16(reinterpret_cast<const TQ*>(p.q) + (int64_t)r * p.ldq + (hk * p.group + h) * QC_HD + 16 * t, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) { top = fmaxf(top, fabsf(x[i])); odd = fmaf(x[i], 0.0f, odd); }
    if (odd != odd) top = INFINITY;   // an infinity or a NaN among them
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float lift = top < 1e-20f ? 18446744073709551616.0f : 1.0f;   // 2^64: keeps the quotient below finite
    const float steps = top > 0.0f ? QC_STEPS / (top * lift) : 0.0f;
    const uint32_t digit = ((g & 3) ^ 1) * 0x11 + 0x40;   // columns d1, d0, d3, d2: that byte of two numbers
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t n[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) n[b] = (uint32_t)__float2int_rn(x[4 * w + b] * lift * steps) + 0x80808080u;   // digits + 128
      qb[nt][w] = __byte_perm(__byte_perm(n[0], n[1], digit), __byte_perm(n[2], n[3], digit), 0x5410) ^ 0x80808080u;
    }
    // an infinite or NaN query: infinity times zero makes the row NaN
    const float mul = (top * lift) * (1.4426950408889634f / QC_STEPS) * p.scale / lift;   // the scale alone may be 3e38
    q_mul[nt] = __shfl_sync(0xffffffffu, mul, 16 * (t >> 1)) * (t & 1 ? 65536.0f : 1.0f);   // of the head whose scores this lane gets
  }
}

// One tile: scores, softmax weights, and their product with V added to acc.  release(place) is called when every lane has
// taken its bytes out of a place, behind() says how many pieces are under way.  False: a wait ran out.
template <int NT, bool ONE, typename Release, typename Behind>
__device__ __forceinline__ bool qc_tile(QcRing& ring, int tokens, int g, int t, const uint32_t (&qb)[NT][4],
                                        const float (&q_mul)[NT], float (&m)[NT], float (&l)[NT], float (&acc)[NT][8],
                                        float& shrink, DevStatus* status, Release release, Behind behind) {
  if (!ring.wait(behind(), status)) return false;
  uint32_t pb[NT][4];      // the weights' bytes: word 2 ks + r
  float alpha[NT];
  const float k_now = ring.scale();
  uint4 k[8];
  {
    const uint8_t* kt = ring.data() + (16 * (g >> 2) + (g & 3)) * QC_HD + 16 * t;
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = *reinterpret_cast<const uint4*>(kt + (32 * (j >> 2) + 4 * (j & 3)) * QC_HD);
  }
  __syncwarp();
  release(ring.place);
  ring.step();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float s[8];
    const float mul = q_mul[nt] * k_now;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int c[4];
      mma_s8_16832_first(c, k[2 * i].x, k[2 * i + 1].x, k[2 * i].y, k[2 * i + 1].y, qb[nt][0], qb[nt][1]);
      mma_s8_16832(c, k[2 * i].z, k[2 * i + 1].z, k[2 * i].w, k[2 * i + 1].w, qb[nt][2], qb[nt][3]);
      s[2 * i] = (float)(c[0] * 256 + c[1]) * mul;
      s[2 * i + 1] = (float)(c[2] * 256 + c[3]) * mul;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], 1);
    if (tokens < QC_BLOCK) {
      const int left = tokens - (16 * (g >> 2) + (g & 3));
#pragma unroll
      for (int j = 0; j < 8; ++j) if (32 * (j >> 2) + 4 * (j & 3) >= left) s[j] = -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float m_new = fmaxf(m[nt], top);
    alpha[nt] = qc_ex2(m[nt] - m_new);
    m[nt] = m_new;
    uint32_t n[8];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = qc_ex2(s[j] - m_new);
      sum += w;
      n[j] = __float2uint_rn(w * QC_ONE);
    }
    l[nt] = fmaf(l[nt], alpha[nt], sum);
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // tokens 32 h ..
      const uint32_t x01 = __byte_perm(n[4 * h], n[4 * h + 1], 0x5140), x23 = __byte_perm(n[4 * h + 2], n[4 * h + 3], 0x5140);
      const uint32_t y01 = __byte_perm(n[4 * h], n[4 * h + 1], 0x7362), y23 = __byte_perm(n[4 * h + 2], n[4 * h + 3], 0x7362);
      const uint32_t d0 = __byte_perm(x01, x23, 0x5410), d1 = __byte_perm(x01, x23, 0x7632);
      const uint32_t d2 = __byte_perm(y01, y23, 0x5410), d3 = __byte_perm(y01, y23, 0x7632);
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int from = (4 * rr + t) * 4;
        if (ONE) {
          const uint32_t got = __shfl_sync(0xffffffffu, t & 2 ? (t & 1 ? d2 : d3) : (t & 1 ? d0 : d1), from + (g & 3));
          pb[nt][2 * h + rr] = g < 4 ? got : 0u;
        } else {
          const uint32_t low = __shfl_sync(0xffffffffu, t & 1 ? d0 : d1, from + 2 * (g >> 2) + (g & 1));
          const uint32_t high = __shfl_sync(0xffffffffu, t & 1 ? d2 : d3, from + 2 * (g >> 2) + (g & 1));
          pb[nt][2 * h + rr] = g & 2 ? high : low;
        }
      }
    }
  }
  if (!ring.wait(behind(), status)) return false;
  // acc counts in the weights' steps times 1 / shrink: a step's share of a block's scale would underflow for values below
  // 1e-32, and the sums of scales above 2^64 might overflow, so from the first such block on they are 2^-64 of that.
  float v_now = ring.scale() * shrink;
  if (v_now > QC_LARGE) {
    shrink = 1.0f / QC_LARGE;
    v_now *= 1.0f / QC_LARGE;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[nt][i] *= 1.0f / QC_LARGE;
  }
  const uint8_t* vt = ring.data() + t * QC_HD + 8 * g;
  // V's bytes, four tokens of one value to a word: a[2 ks + r][value 8 g + i]
  uint32_t a[4][8];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint2 v[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) v[b] = *reinterpret_cast<const uint2*>(vt + 4 * (4 * w + b) * QC_HD);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t x0 = half ? v[0].y : v[0].x, x1 = half ? v[1].y : v[1].x;
      const uint32_t x2 = half ? v[2].y : v[2].x, x3 = half ? v[3].y : v[3].x;
      const uint32_t t0 = __byte_perm(x0, x1, 0x5140), t1 = __byte_perm(x2, x3, 0x5140);
      const uint32_t t2 = __byte_perm(x0, x1, 0x7362), t3 = __byte_perm(x2, x3, 0x7362);
      a[w][4 * half] = __byte_perm(t0, t1, 0x5410);
      a[w][4 * half + 1] = __byte_perm(t0, t1, 0x7632);
      a[w][4 * half + 2] = __byte_perm(t2, t3, 0x5410);
      a[w][4 * half + 3] = __byte_perm(t2, t3, 0x7632);
    }
  }
  __syncwarp();
  release(ring.place);
  ring.step();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int c[4];
      qc_mma_su_first(c, a[0][2 * i], a[0][2 * i + 1], a[1][2 * i], a[1][2 * i + 1], pb[nt][0], pb[nt][1]);
      qc_mma_su(c, a[2][2 * i], a[2][2 * i + 1], a[3][2 * i], a[3][2 * i + 1], pb[nt][2], pb[nt][3]);
      acc[nt][2 * i] = fmaf((float)(c[0] * 256 + c[1]), v_now, acc[nt][2 * i] * alpha[nt]);
      acc[nt][2 * i + 1] = fmaf((float)(c[2] * 256 + c[3]), v_now, acc[nt][2 * i + 1] * alpha[nt]);
    }
  }
  return true;
}

// NT: pairs of query heads of a key head.  ONE: a single query head (its scores then reach all four lanes of a group,
// and one shuffle a word is enough).  A cluster of CTAs takes an item (row, key head); its warps take tiles in turn, and
// the CTAs' partial results meet in the first CTA's shared memory.  Where a cluster is too small for a long row, `parts`
// lone CTAs take it and leave their partial results to qcache_merge_kernel.
template <typename TQ, typename TO, int NT, bool ONE>
__global__ void __launch_bounds__(QC_MAX_WARPS * 32) qcache_attend_kernel(QcAttendParams p, int cluster, int parts, DevStatus* status) {
  constexpr int HEADS = 2 * NT, STEP = HEADS * (QC_HD + 2);
  extern __shared__ __align__(128) uint8_t qc_smem[];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  QcRing ring(qc_smem + warp * QC_RING);
  float* warp_part = reinterpret_cast<float*>(qc_smem + warps * QC_RING);
  float* cta_part = warp_part + warps * STEP;
  const int g = lane >> 2, t = lane & 3;
  const int share = cluster * parts;   // CTAs of an item: a cluster, or `parts` lone ones, or one
  const int rank = blockIdx.x % (uint32_t)share;
  if (cluster > 1) qc_cluster_arrive();   // waited for below: every CTA of the cluster runs before another writes to it
  if (lane == 0) ring.init();
  __syncwarp();
  pdl_wait();
  const uint32_t item = blockIdx.x / (uint32_t)share;
  const QcRow row(p, item);
  if (lane == 0) asm volatile("fence.proxy.async.global;" ::: "memory");   // the bulk copies see what the kernels before wrote
  const int tiles = row.tiles(), stride = share * warps, tile0 = rank * warps + warp;
  const int mine = tile0 < tiles ? (tiles - tile0 + stride - 1) / stride : 0;   // tiles of this warp
  // pieces: K and V of the warp's tiles in turn
  int asked = 0;
  const int8_t *k_from = row.K + (int64_t)tile0 * QC_TILE, *v_from = row.V + (int64_t)tile0 * QC_TILE;
  const float *ks_from = row.ks + tile0, *vs_from = row.vs + tile0;
  int left = row.len - tile0 * QC_BLOCK;   // tokens from there on
  auto fetch = [&](int at) {
    if (asked == 2 * mine) return;
    const bool is_v = asked & 1;
    if (lane == 0) ring.fetch(at, is_v ? v_from : k_from, is_v ? vs_from : ks_from, min(left, QC_BLOCK));
    if (is_v) {
      k_from += (int64_t)stride * QC_TILE; v_from += (int64_t)stride * QC_TILE;
      ks_from += stride; vs_from += stride; left -= stride * QC_BLOCK;
    }
    ++asked;
  };
  for (int i = 0; i < QC_PLACES; ++i) fetch(i);
  uint32_t qb[NT][4];
  float q_mul[NT];
  qc_query<TQ, NT>(p, row.r, row.hk, g, t, qb, q_mul);
  float m[NT], l[NT], acc[NT][8], shrink = 1.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY; l[nt] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[nt][i] = 0.0f;
  }
  int taken = 0;
  for (int i = 0; i < mine; ++i) {
    if (!qc_tile<NT, ONE>(ring, row.tokens(tile0 + i * stride), g, t, qb, q_mul, m, l, acc, shrink, status, fetch,
                          [&] { return asked - ++taken; })) break;
  }

  // the warp's partial results
  const float step = (t & 1 ? 65536.0f : 1.0f) / QC_ONE * (shrink < 1.0f ? QC_LARGE : 1.0f);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 4);
    l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 8);
    l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 16);
    float* dst = warp_part + warp * STEP + (2 * nt + (t >> 1)) * (QC_HD + 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float mine = acc[nt][i] * step, o = mine + __shfl_xor_sync(0xffffffffu, mine, 1);
      if (!(t & 1)) dst[8 * g + i] = o;
    }
    if (g == 0 && !(t & 1)) { dst[QC_HD] = m[nt]; dst[QC_HD + 1] = l[nt]; }
  }
  __syncthreads();
  const bool write = !row.skipped || p.clear_skipped;
  auto store = [&](int h, int c, const QcMerged& x) {
    if (write) reinterpret_cast<TO*>(p.out)[(int64_t)row.r * p.ldo + (row.hk * p.group + h) * QC_HD + c] =
        from_f<TO>(row.len > 0 ? x.o / x.l : 0.0f);
  };
  if (parts > 1) {
    float* dst = p.part + ((int64_t)item * parts + rank) * STEP;
    for (int i = threadIdx.x; i < p.group * QC_HD; i += blockDim.x) {
      const int h = i >> 6, c = i & 63;
      const QcMerged x = qc_merge(warp_part + h * (QC_HD + 2), STEP, warps, c);
      dst[h * (QC_HD + 2) + c] = x.o;
      if (c < 2) dst[h * (QC_HD + 2) + QC_HD + c] = c ? x.l : x.m;
    }
    return;
  }
  if (cluster == 1) {
    for (int i = threadIdx.x; i < p.group * QC_HD; i += blockDim.x)
      store(i >> 6, i & 63, qc_merge(warp_part + (i >> 6) * (QC_HD + 2), STEP, warps, i & 63));
    return;
  }
  uint32_t home;   // cta_part of the cluster's first CTA
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(home) : "r"((uint32_t)__cvta_generic_to_shared(cta_part)));
  qc_cluster_wait();
  for (int i = threadIdx.x; i < p.group * QC_HD; i += blockDim.x) {
    const int h = i >> 6, c = i & 63;
    const QcMerged x = qc_merge(warp_part + h * (QC_HD + 2), STEP, warps, c);
    const uint32_t dst = home + 4 * (rank * STEP + h * (QC_HD + 2));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4 * c), "f"(x.o) : "memory");
    if (c < 2) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4 * (QC_HD + c)), "f"(c ? x.l : x.m) : "memory");
  }
  qc_cluster_arrive();
  qc_cluster_wait();
  if (rank == 0)
    for (int i = threadIdx.x; i < p.group * QC_HD; i += blockDim.x)
      store(i >> 6, i & 63, qc_merge(cta_part + (i >> 6) * (QC_HD + 2), STEP, cluster, i & 63));
}

// The partial results of a row's parts (qcache_attend_kernel with parts > 1), merged.  Block = 256 threads: a thread per
// part for the weights, then four groups of 64 that take every fourth part, eight loads at a time (a loop of single loads
// took 4 us longer); grid = (row, key head) x its query heads.
constexpr int QC_MAX_PARTS = 256;
template <typename TO>
__global__ void __launch_bounds__(256) qcache_merge_kernel(QcAttendParams p, int parts, int step) {
  __shared__ float weight[QC_MAX_PARTS], top[8], total[8], sums[4][QC_HD];
  pdl_trigger();
  const uint32_t item = blockIdx.x / (uint32_t)p.group;
  const int h = blockIdx.x % (uint32_t)p.group, tid = threadIdx.x, sub = tid >> 6, c = tid & 63;
  const int r = (int)(item / (uint32_t)p.c.n_heads), hk = (int)(item - (uint32_t)r * p.c.n_heads);
  pdl_wait();
  const int slot = p.slots[r];
  if ((slot < 0 || slot >= p.c.n_slots) && !p.clear_skipped) return;
  const float* part = p.part + (int64_t)item * parts * step + h * (QC_HD + 2);
  float m = -INFINITY, l = 0.0f;
  if (tid < parts) { m = part[tid * step + QC_HD]; l = part[tid * step + QC_HD + 1]; }
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  float t = warp_max(m);
  if ((tid & 31) == 0) top[tid >> 5] = t;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) t = fmaxf(t, top[i]);
  const float w = l == 0.0f ? 0.0f : qc_ex2(m - t);   // l = 0: no tokens; NaN goes through
  weight[tid] = w;
  const float s = warp_sum(l * w);
  if ((tid & 31) == 0) total[tid >> 5] = s;
  __syncthreads();
  int i = sub;
  for (; i + 28 < parts; i += 32) {   // eight parts' loads at a time
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = part[(i + 4 * j) * step + c];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j & 3] = fmaf(x[j], weight[i + 4 * j], o[j & 3]);
  }
  for (; i < parts; i += 4) o[0] = fmaf(part[i * step + c], weight[i], o[0]);
  sums[sub][c] = (o[0] + o[1]) + (o[2] + o[3]);
  __syncthreads();
  if (sub) return;
  float all = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) all += total[j];
  const float v = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
  // no tokens at all: the sum is 0
  reinterpret_cast<TO*>(p.out)[(int64_t)r * p.ldo + (hk * p.group + h) * QC_HD + c] = from_f<TO>(all == 0.0f ? 0.0f : v / all);
}

}  // namespace wdz
