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
#include "gemv_packed.cuh"

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

// ---- attention -----------------------------------------------------------------------------------------------------
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
constexpr int QC_MAX_WARPS = 8;
constexpr float QC_STEPS = 127.0f * 16777216.0f;   // a query's largest value in steps: rounding up leaves d3 a byte
constexpr float QC_ONE = 4294967040.0f;            // the weight 1 in steps: the largest fp32 below 2^32

__device__ __forceinline__ void qc_mma_su(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 qc_ld16(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 qc_ld8(const int8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
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

// NT: pairs of query heads of a key head.  ONE: a single query head (its scores then reach all four lanes of a group,
// and one shuffle a word is enough).  A cluster of CTAs takes an item (row, key head); its warps take tiles in turn, and
// the CTAs' partial results meet in the first CTA's shared memory.
template <typename TQ, typename TO, int NT, bool ONE>
__global__ void __launch_bounds__(QC_MAX_WARPS * 32) qcache_attend_kernel(QcAttendParams p, int cluster) {
  constexpr int HEADS = 2 * NT, STEP = HEADS * (QC_HD + 2), MAX_CLUSTER = NT == 4 ? 8 : 16;
  __shared__ float warp_part[QC_MAX_WARPS * STEP];
  __shared__ float cta_part[MAX_CLUSTER * STEP];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % cluster;
  const int64_t item = blockIdx.x / cluster;
  const int r = (int)(item / p.c.n_heads), hk = (int)(item % p.c.n_heads);
  if (cluster > 1) qc_cluster_arrive();   // waited for below: every CTA of the cluster runs before another writes to it
  pdl_wait();
  const int slot = p.slots[r];
  const bool skipped = slot < 0 || slot >= p.c.n_slots;
  const int len = skipped ? 0 : min(max(p.lens[r], 0), p.c.n_blocks * QC_BLOCK);
  const int64_t at = skipped ? 0 : slot;
  const int64_t head_at = (int64_t)hk * p.c.n_blocks;
  const int8_t* K = p.c.k + at * p.c.slot_stride + head_at * (QC_BLOCK * QC_HD);
  const int8_t* V = p.c.v + at * p.c.slot_stride + head_at * (QC_BLOCK * QC_HD);
  const float* ks = p.c.ks + at * p.c.scale_stride + head_at;
  const float* vs = p.c.vs + at * p.c.scale_stride + head_at;
  const int tiles = (len + QC_BLOCK - 1) / QC_BLOCK, stride = cluster * warps;
  int tile = rank * warps + warp;

  uint4 k[8];
  uint2 v[16];
  float k_mul = 0.0f, v_mul = 0.0f;
  const int k_at = (16 * (g >> 2) + (g & 3)) * QC_HD + 16 * t, v_at = t * QC_HD + 8 * g;
  auto load_k = [&](int tl) {
    const int8_t* b = K + (int64_t)tl * (QC_BLOCK * QC_HD) + k_at;
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = qc_ld16(b + (32 * (j >> 2) + 4 * (j & 3)) * QC_HD);
    k_mul = __ldg(ks + tl);
  };
  auto load_v = [&](int tl) {
    const int8_t* b = V + (int64_t)tl * (QC_BLOCK * QC_HD) + v_at;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = qc_ld8(b + 4 * j * QC_HD);
    v_mul = __ldg(vs + tl);
  };
  if (tile < tiles) { load_k(tile); load_v(tile); }

  // The query's bytes: lane (g, t) makes column g, values 16 t .. 16 t + 15 of head g / 4 of the pair.
  uint32_t qb[NT][4];
  float q_mul[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = min(2 * nt + (g >> 2), p.group - 1);
    float x[16], top = 0.0f;
    bool fine = true;
    qc_load16(reinterpret_cast<const TQ*>(p.q) + (int64_t)r * p.ldq + (hk * p.group + h) * QC_HD + 16 * t, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) { top = fmaxf(top, fabsf(x[i])); fine &= fabsf(x[i]) <= 3.402823466e38f; }
    if (!fine) top = INFINITY;
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float lift = top < 1e-20f ? 18446744073709551616.0f : 1.0f;   // 2^64: keeps the quotient below finite
    const float steps = top > 0.0f ? QC_STEPS / (top * lift) * lift : 0.0f;
    const int digit = (g & 3) ^ 1;   // columns d1, d0, d3, d2
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t n[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) n[b] = ((uint32_t)__float2int_rn(x[4 * w + b] * steps) + 0x80808080u) >> (8 * digit);
      const uint32_t lo = __byte_perm(n[0], n[1], 0x0040), hi = __byte_perm(n[2], n[3], 0x0040);
      qb[nt][w] = __byte_perm(lo, hi, 0x5410) ^ 0x80808080u;   // the digits are bytes less 128
    }
    // an infinite or NaN query: infinity times zero makes the row NaN
    const float mul = (top * lift) * (1.0f / QC_STEPS) * (p.scale * 1.4426950408889634f) / lift;
    q_mul[nt] = __shfl_sync(0xffffffffu, mul, 16 * (t >> 1)) * (t & 1 ? 65536.0f : 1.0f);   // of the head whose scores this lane gets
  }

  float m[NT], l[NT], acc[NT][8];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY; l[nt] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[nt][i] = 0.0f;
  }
  for (; tile < tiles; tile += stride) {
    const int next = tile + stride;
    const bool more = next < tiles;
    uint32_t pb[NT][4];      // the weights' bytes: word 2 ks + r
    float alpha[NT];
    const float k_now = k_mul;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float s[8];
      const float mul = q_mul[nt] * k_now;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int c[4] = {0, 0, 0, 0};
        mma_s8_16832(c, k[2 * i].x, k[2 * i + 1].x, k[2 * i].y, k[2 * i + 1].y, qb[nt][0], qb[nt][1]);
        mma_s8_16832(c, k[2 * i].z, k[2 * i + 1].z, k[2 * i].w, k[2 * i + 1].w, qb[nt][2], qb[nt][3]);
        s[2 * i] = (float)(c[0] * 256 + c[1]) * mul;
        s[2 * i + 1] = (float)(c[2] * 256 + c[3]) * mul;
      }
      if (nt == NT - 1 && more) load_k(next);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], 1);
      if ((tile + 1) * QC_BLOCK > len) {
        const int left = len - tile * QC_BLOCK - (16 * (g >> 2) + (g & 3));
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
    // V's bytes, four tokens of one value to a word: a[2 ks + r][value 8 g + i]
    uint32_t a[4][8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t x0 = half ? v[4 * w].y : v[4 * w].x, x1 = half ? v[4 * w + 1].y : v[4 * w + 1].x;
        const uint32_t x2 = half ? v[4 * w + 2].y : v[4 * w + 2].x, x3 = half ? v[4 * w + 3].y : v[4 * w + 3].x;
        const uint32_t t0 = __byte_perm(x0, x1, 0x5140), t1 = __byte_perm(x2, x3, 0x5140);
        const uint32_t t2 = __byte_perm(x0, x1, 0x7362), t3 = __byte_perm(x2, x3, 0x7362);
        a[w][4 * half] = __byte_perm(t0, t1, 0x5410);
        a[w][4 * half + 1] = __byte_perm(t0, t1, 0x7632);
        a[w][4 * half + 2] = __byte_perm(t2, t3, 0x5410);
        a[w][4 * half + 3] = __byte_perm(t2, t3, 0x7632);
      }
    }
    const float v_now = v_mul * ((t & 1 ? 65536.0f : 1.0f) / QC_ONE);
    if (more) load_v(next);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int c[4] = {0, 0, 0, 0};
        qc_mma_su(c, a[0][2 * i], a[0][2 * i + 1], a[1][2 * i], a[1][2 * i + 1], pb[nt][0], pb[nt][1]);
        qc_mma_su(c, a[2][2 * i], a[2][2 * i + 1], a[3][2 * i], a[3][2 * i + 1], pb[nt][2], pb[nt][3]);
        acc[nt][2 * i] = fmaf((float)(c[0] * 256 + c[1]), v_now, acc[nt][2 * i] * alpha[nt]);
        acc[nt][2 * i + 1] = fmaf((float)(c[2] * 256 + c[3]), v_now, acc[nt][2 * i + 1] * alpha[nt]);
      }
    }
  }

  // the warp's partial results
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 4);
    l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 8);
    l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 16);
    float* dst = warp_part + warp * STEP + (2 * nt + (t >> 1)) * (QC_HD + 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = acc[nt][i] + __shfl_xor_sync(0xffffffffu, acc[nt][i], 1);
      if (!(t & 1)) dst[8 * g + i] = o;
    }
    if (g == 0 && !(t & 1)) { dst[QC_HD] = m[nt]; dst[QC_HD + 1] = l[nt]; }
  }
  __syncthreads();
  const bool write = !skipped || p.clear_skipped;
  auto store = [&](int h, int c, const QcMerged& x) {
    if (write) reinterpret_cast<TO*>(p.out)[(int64_t)r * p.ldo + (hk * p.group + h) * QC_HD + c] =
        from_f<TO>(len > 0 ? x.o / x.l : 0.0f);
  };
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

}  // namespace wdz
