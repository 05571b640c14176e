// The 8-bit key/value cache: storing rows into it and attending over it.
//
//   value(slot, head, token, c) = int8[slot][head][token][c] * scale[slot][head][token / 64]     (K and V alike)
//
//   qcache_store_kernel  - rounds rows into the cache: s = max|x| / 127 over the 64 tokens x 64 values of a block,
//       q = rint(x / s).  A block that is continued keeps the larger scale, and what it held is rounded to it.
//   qcache_attend_kernel - one query row per (slot, length): softmax(scale * q K^T) V over the slot's first tokens.
#pragma once
#include "../../include/wdz.h"
#include "common.cuh"

namespace wdz {

constexpr int QC_BLOCK = WDZ_QCACHE_BLOCK;   // tokens that share a scale
constexpr int QC_HD = 64;
constexpr float QC_TINY = 1.5046328e-36f;    // 2^-119: below it x / 127 would leave the normal range; such a block is zero

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

// rint(x / s), half to even, exactly: the rounded product with 1 / s is at most one off, and the remainder
// x - q s has so few bits that the fused multiply-add gives it without rounding wherever it decides.
__device__ __forceinline__ int qc_code(float x, float s, float inv) {
  const float lim = fminf(fmaxf(x * inv, -127.0f), 127.0f);   // infinities saturate; NaN becomes a bound and is set aside below
  float q = rintf(lim);
  const float d = fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (d > half || (d == half && odd)) q += 1.0f;
  if (d < -half || (d == -half && odd)) q -= 1.0f;
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  return x == x ? (int)q : 0;
}

// rint(q * s_old / s_new): both products fit a double, and the quotient is never nearer to a half than its rounding.
__device__ __forceinline__ int qc_recode(int q, double s_old, double s_new) {
  return __double2int_rn(__ddiv_rn((double)q * s_old, s_new));
}

__device__ __forceinline__ void qc_report(DevStatus* st, int code, int detail) {
  if (atomicCAS(&st->code, 0, code) == 0) st->detail = detail;
}

// Block = 64 threads (a thread per value of the head); grid = (blocks of the longest run, head and K / V, run).
template <typename T>
__global__ void __launch_bounds__(64) qcache_store_kernel(QcStoreParams p, DevStatus* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red[2];
  const int run = blockIdx.z, head = blockIdx.y >> 1, c = threadIdx.x;
  const bool is_v = blockIdx.y & 1;
  const int slot = p.slots[run], p0 = p.positions[run];
  const int r0 = p.row_begin ? p.row_begin[run] : run, r1 = p.row_begin ? p.row_begin[run + 1] : run + 1;
  const int room = p.c.n_blocks * QC_BLOCK;
  if (slot < 0 || slot >= p.c.n_slots || r1 <= r0) return;
  int dup = 0;
  for (int j = run + 1 + threadIdx.x; j < p.n_runs; j += 64) dup |= p.slots[j] == slot;
  if (r0 < 0 || r1 > p.n_rows || p0 < 0 || p0 > room - (r1 - r0) || __syncthreads_or(dup)) {
    if (threadIdx.x == 0) qc_report(status, WDZ_EINVAL, 2000000 + run);
    return;
  }
  const int p1 = p0 + (r1 - r0);
  int8_t* cv = (is_v ? p.c.v : p.c.k) + slot * p.c.slot_stride + (int64_t)head * room * QC_HD;
  float* cs = (is_v ? p.c.vs : p.c.ks) + slot * p.c.scale_stride + (int64_t)head * p.c.n_blocks;
  const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + head * QC_HD + c;
  const int64_t ld = is_v ? p.ldv : p.ldk;
  bool bad = false;
  for (int b = p0 / QC_BLOCK + blockIdx.x; b * QC_BLOCK < p1; b += gridDim.x) {
    const int lo = max(p0, b * QC_BLOCK), hi = min(p1, (b + 1) * QC_BLOCK);
    float top = 0.0f;
    for (int t = lo; t < hi; ++t) {
      const float x = to_f(src[(int64_t)(r0 + t - p0) * ld]);
      if (fabsf(x) <= 3.402823466e38f) top = fmaxf(top, fabsf(x)); else bad = true;
    }
    top = warp_max(top);
    __syncthreads();
    if ((c & 31) == 0) red[c >> 5] = top;
    __syncthreads();
    top = fmaxf(red[0], red[1]);
    const float old = lo > b * QC_BLOCK ? cs[b] : 0.0f;
    const float now = fmaxf(old, top >= QC_TINY ? __fdiv_rn(top, 127.0f) : 0.0f);
    if (now > old && lo > b * QC_BLOCK)
      for (int t = b * QC_BLOCK; t < lo; ++t) {
        int8_t* q = cv + (int64_t)t * QC_HD + c;
        *q = (int8_t)qc_recode(*q, old, now);
      }
    const float inv = now > 0.0f ? 1.0f / now : 0.0f;
    for (int t = lo; t < hi; ++t) {
      const float x = to_f(src[(int64_t)(r0 + t - p0) * ld]);
      cv[(int64_t)t * QC_HD + c] = now > 0.0f ? (int8_t)qc_code(x, now, inv) : (int8_t)0;
    }
    __syncthreads();
    if (c == 0) cs[b] = now;
  }
  if (bad) qc_report(status, WDZ_ENAN, 2000000 + run);
}

struct QcAttendParams {
  QcView c;
  const void* q; int64_t ldq;
  void* out; int64_t ldo;
  const int *slots, *lens;
  int n_rows, group;        // query heads per key head
  float scale;
  bool clear_skipped;       // rows of slots outside the cache: zeros instead of what was there
};

// A warp per (row, query head).
template <typename TQ, typename TO>
__global__ void __launch_bounds__(128) qcache_attend_kernel(QcAttendParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float qs[4][QC_HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hq = p.c.n_heads * p.group;
  const int64_t item = (int64_t)blockIdx.x * 4 + warp;
  if (item >= (int64_t)p.n_rows * hq) return;
  const int r = (int)(item / hq), h = (int)(item % hq), hk = h / p.group;
  const int slot = p.slots[r], room = p.c.n_blocks * QC_BLOCK;
  const bool skipped = slot < 0 || slot >= p.c.n_slots;
  if (skipped && !p.clear_skipped) return;
  const int len = skipped ? 0 : min(max(p.lens[r], 0), room);
  const TQ* q = reinterpret_cast<const TQ*>(p.q) + (int64_t)r * p.ldq + h * QC_HD;
  for (int c = lane; c < QC_HD; c += 32) qs[warp][c] = to_f(q[c]) * (p.scale * 1.4426950408889634f);
  __syncwarp();
  const int64_t at = skipped ? 0 : slot;
  const int8_t* K = p.c.k + at * p.c.slot_stride + (int64_t)hk * room * QC_HD;
  const int8_t* V = p.c.v + at * p.c.slot_stride + (int64_t)hk * room * QC_HD;
  const float* ks = p.c.ks + at * p.c.scale_stride + (int64_t)hk * p.c.n_blocks;
  const float* vs = p.c.vs + at * p.c.scale_stride + (int64_t)hk * p.c.n_blocks;
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int t0 = 0; t0 < len; t0 += 32) {
    const int t = t0 + lane;
    float s = -INFINITY;
    if (t < len) {
      s = 0.0f;
      const char4* row = reinterpret_cast<const char4*>(K + (int64_t)t * QC_HD);
      for (int c = 0; c < QC_HD / 4; ++c) {
        const char4 x = row[c];
        s += qs[warp][4 * c] * x.x + qs[warp][4 * c + 1] * x.y + qs[warp][4 * c + 2] * x.z + qs[warp][4 * c + 3] * x.w;
      }
      s *= ks[t / QC_BLOCK];
    }
    const float m_new = fmaxf(m, warp_max(s)), alpha = exp2f(m - m_new);
    const float w = t < len ? exp2f(s - m_new) : 0.0f;
    l = l * alpha + warp_sum(w);
    o0 *= alpha; o1 *= alpha;
    m = m_new;
    const float wv = t < len ? w * vs[t / QC_BLOCK] : 0.0f;
    for (int j = 0; j < min(32, len - t0); ++j) {
      const float pj = __shfl_sync(0xffffffffu, wv, j);
      o0 = fmaf(pj, (float)V[(int64_t)(t0 + j) * QC_HD + lane], o0);
      o1 = fmaf(pj, (float)V[(int64_t)(t0 + j) * QC_HD + 32 + lane], o1);
    }
  }
  const float inv = len > 0 ? 1.0f / l : 0.0f;
  TO* dst = reinterpret_cast<TO*>(p.out) + (int64_t)r * p.ldo + h * QC_HD;
  dst[lane] = from_f<TO>(o0 * inv);
  dst[32 + lane] = from_f<TO>(o1 * inv);
}

}  // namespace wdz
