// tcb_page_decode.cu - attention over the paged cache row by row: decode steps
// and few rows over few positions (tcb_page_attn), and batches behind a shared
// prefix (tcb_prefix_attn: all of it, or the suffixes joined with partial results
// of the prefix).
//
// Mathematics: per (row, KV head) the G = H / KVH query heads that share
// the head are the 8 or 16 columns of two products on the tensor cores,
//   S^T = K Q^T   (16 positions x queries, per 16 positions)
//   O^T += V^T P^T (head elements x queries)
// with the running maximum m and sum l of the softmax per column, in powers of
// two (scores times scale * log2 e).  m follows a column only when a score
// passes it by more than kSlack (weights up to 2^kSlack, exact in f32 sums and
// far inside f16's range), so the usual 16 positions cost no maximum across
// lanes and no rescaling.
//
// Roundings: the weights, to the cache's type, are what the second product takes;
// the sum is of the rounded weights, whose errors then cancel in part.  Against 64
// bits a call errs by 2.1e-4 (f16) to 2.2e-3 (bf16), where one rounding of the
// result errs by 2.1e-4 and 1.7e-3.
//
// Bound: the K/V bytes, each read once: 3.63 GB for 64 sequences of up to 32768
// positions (window 16384, 8 KV heads of 128, bf16) in 555 to 570 us = 6370 to 6540
// GB/s, the copy rate.  Layout:
// every fragment comes straight from global memory into registers, without
// shared memory: the k slots of S^T are dealt so that a lane's A fragments of
// K are 16-byte pieces of one position (lane (g, t): positions g and g + 8,
// elements 32c + 8t ..; Q is read in the same order), and those of V^T are
// 16-byte pieces of four positions (2t, 2t+1, 2t+8, 2t+9), paired by byte
// permutes, with output row e of a lane group dealt to element 8g + e.  P^T
// becomes a B fragment by one matrix transpose (movmatrix) per 8 positions.
// A warp loads the next 16 positions' K as soon as it has formed S^T, and
// their V as soon as it has added P V, so both stay in flight.
//
// Split: a cluster of up to 8 CTAs shares the positions of one (request, KV
// head) in contiguous parts, 4 warps a CTA interleaved over 16-position
// groups; the partial (m, l, O) are joined within the CTA through shared
// memory and across the cluster through distributed shared memory, in a fixed
// order, with no scratch in HBM and no second launch.  Where a few long
// requests leave the GPU empty, several clusters share one: each rank leaves
// its slice of the joined partial in scratch, and the rank that comes last
// joins the slices.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "tcb_common.cuh"
#include "tcb_mv_ptx.cuh"
#include "tcb_page.h"

namespace tcb {
namespace pd {

constexpr float kSlack = 8.f;
constexpr uint32_t kAll = 0xFFFFFFFFu;

template <int DT>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (DT == TCB_F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// CTAs of 4 warps per SM that leave a thread the registers it needs without spills (168
// and 234 at head_dim 128).  At batch 64 with 3 CTAs: 554 us against 595 with
// 4 and 128 spilling registers.
template <int HD, int NT>
constexpr int kCtas = (NT == 1 ? 4 : 3) - (HD == 128);

// 16 bytes of the cache, read once: not kept in L1
__device__ __forceinline__ uint4 ld_cache(const uint16_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// two weights rounded to the cache's type, and what they were rounded to
template <int DT>
__device__ __forceinline__ uint32_t pack2(float &a, float &b) {
  uint32_t u;
  if constexpr (DT == TCB_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    u = *reinterpret_cast<const uint32_t *>(&h);
    const float2 f = __half22float2(h);
    a = f.x, b = f.y;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    u = *reinterpret_cast<const uint32_t *>(&h);
    a = __uint_as_float(u << 16), b = __uint_as_float(u & 0xFFFF0000u);
  }
  return u;
}

// 2^(m - top) for a partial whose maximum is m; an empty one weighs 0
__device__ __forceinline__ float join_weight(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

// where the partials of several clusters meet (parts > 1): element pairs
// [unit][part][query][HD] and (m, l) [unit][part][rank][query], one counter per
// (unit, rank); a unit is blockIdx.z * gridDim.y + blockIdx.y
struct Join {
  int parts, ranks;
  float *o;
  float2 *ml;
  unsigned *arrived;  // zero before and after a launch
};

template <int DT, int HD, int NT, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == 4 ? kCtas<HD, NT> : 1) k_page_decode(const __grid_constant__ PageAttnArgs a,
                                                                            const __grid_constant__ Join j,
                                                                            const __grid_constant__ PrefixPartials x) {
  constexpr int Q = 8 * NT, kThreads = 32 * kWarps;  // query columns
  constexpr int CK = HD / 32, CV = HD / 64;
  __shared__ float so[kWarps][Q][HD];
  __shared__ float sm[kWarps][Q], sl[kWarps][Q];
  __shared__ float cm[Q], cl[Q];  // the CTA's
  __shared__ float xm[Q], xl[Q], xg[kMaxPrefixParts][Q];  // the prefix's partials: maximum, sum, weights
  const int G = a.H / a.kv.n_kv_heads, tiles = (G + Q - 1) / Q;
  const int kh = blockIdx.y / tiles, h0 = (blockIdx.y % tiles) * Q;  // first query head within the group
  const int b = blockIdx.z / a.max_rows, at = blockIdx.z - b * a.max_rows, n_cta = gridDim.x;  // row `at` of request b
  const int n_rank = j.ranks, c = blockIdx.x % n_rank, part = blockIdx.x / n_rank;  // rank in the cluster; cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // behind the prefix's kernel too: what the kernels before that one wrote (lengths,
  // pages, K/V rows) is promised to a grid that has waited itself.  (Reading the
  // suffixes beside the prefix's tiles took 85.6 us where this takes 87.3, 64
  // requests behind 16384 positions.)
  mv::pdl_launch_dependents();  // before the wait: 7.3 us for one sequence, 7.6 after it
  mv::pdl_wait();
  // the row, and the positions up to its own
  int r = b, rows = 1;
  bool bad = false;
  if (a.row_start) {
    const int r0 = min(max(a.row_start[b], 0), a.T);
    rows = min(max(a.row_start[b + 1], r0), a.T) - r0;
    r = r0 + at;
    bad = rows > a.max_rows || a.row_start[b + 1] < a.row_start[b];
  }
  const bool live = at < rows;
  int len = a.kv_len[b];
  if (len < 0 || len > a.max_len || len > (long)a.width << a.page_shift) {
    bad = true;
    len = 0;
  }
  if (bad && threadIdx.x == 0) atomicExch(a.derr, TCB_ERR_BOUNDS);
  if (!live) return;  // every CTA of the cluster leaves
  len = max(len - rows + at + 1, 0);
  // visible: [0, first) (the first positions, or a prefix read here) and
  // [lo, len), first <= lo; in 16-position groups [0, ns) and [w0, w1)
  int lo, first;
  if (a.prefix) {
    lo = min(a.prefix_len, len);
    first = x.parts ? 0 : lo;
  } else {
    lo = a.window < 0 ? 0 : (int)max(0l, (long)len - a.window);
    first = min(a.sinks, lo);
    if (first == lo) lo = first = 0;
  }
  const int ns = (first + 15) >> 4, w0 = lo >> 4, w1 = lo < len ? (len + 15) >> 4 : w0;
  const int units = ns + w1 - w0;
  const int u0 = (int)((long)units * blockIdx.x / n_cta), u1 = (int)((long)units * (blockIdx.x + 1) / n_cta);

  // Q as the B operand: column g (and g + 8) is query head h0 + g
  uint32_t qf[NT][2 * CK][2];
  const long qrow = r * a.ldq + (long)(kh * G + h0) * HD;
#pragma unroll
  for (int x = 0; x < NT; x++) {
    const bool ok = h0 + 8 * x + g < G;
#pragma unroll
    for (int e = 0; e < CK; e++) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (ok)
        v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + qrow + (8 * x + g) * HD + 32 * e + 8 * t);
      qf[x][2 * e][0] = v.x, qf[x][2 * e][1] = v.y, qf[x][2 * e + 1][0] = v.z, qf[x][2 * e + 1][1] = v.w;
    }
  }
  float o[HD / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int x = 0; x < NT; x++) {
    m[x][0] = m[x][1] = -INFINITY;
    l[x][0] = l[x][1] = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 16; d++) o[d][x][0] = o[d][x][1] = o[d][x][2] = o[d][x][3] = 0.f;
  }

  const uint16_t *kp = static_cast<const uint16_t *>(a.kv.k) + kh * a.kv.head_stride + g * a.kv.pos_stride + 8 * t;
  const uint16_t *vp = static_cast<const uint16_t *>(a.kv.v) + kh * a.kv.head_stride + 2 * t * a.kv.pos_stride + 8 * g;
  const int *table = a.tables + b * a.ldt;
  // lane i holds the page of the warp's group `base + i * kWarps` (-1: none such)
  auto group_of = [&](int u) { return u < ns ? u : u - ns + w0; };
  auto page_of = [&](int u) {
    if (u >= u1) return 0;
    const int at = group_of(u) >> (a.page_shift - 4), pg = u < ns && a.prefix ? a.prefix[at] : table[at];
    return pg >= 0 && pg < a.kv.n_pages ? pg : -1;
  };
  const int base = u0 + warp, n_it = base < u1 ? (u1 - base + kWarps - 1) / kWarps : 0;
  int pages = page_of(base + lane * kWarps), next_pages = 0;
  if (n_it > 32) next_pages = page_of(base + (32 + lane) * kWarps);

  uint4 kf[2 * CK], vf[4][CV];
  // element offset of the group of iteration i, and whether its page is in the pools
  bool page_bad = false;
  auto locate = [&](int i, bool &ok) {
    const int pg = __shfl_sync(kAll, pages, i & 31);
    const int pos = group_of(base + i * kWarps) << 4;
    ok = pg >= 0;
    return (ok ? pg : 0) * a.kv.page_stride + (pos & (a.kv.page - 1)) * a.kv.pos_stride;
  };
  auto load_k = [&](long off) {
#pragma unroll
    for (int e = 0; e < CK; e++) {
      kf[e] = ld_cache(kp + off + 32 * e);
      kf[CK + e] = ld_cache(kp + off + 8 * a.kv.pos_stride + 32 * e);
    }
  };
  auto load_v = [&](long off) {
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
      for (int e = 0; e < CV; e++)
        vf[x][e] = ld_cache(vp + off + ((x & 1) + 8 * (x >> 1)) * a.kv.pos_stride + 64 * e);
  };
  bool ok = true;
  if (n_it > 0) {
    const long off = locate(0, ok);
    load_k(off);
    load_v(off);
  }
  for (int i = 0; i < n_it; i++) {
    const bool here = ok;
    const int key0 = group_of(base + i * kWarps) << 4;
    const bool early = base + i * kWarps < ns;
    const int from = early ? 0 : lo, to = early ? first : len;
    float s[NT][4];
#pragma unroll
    for (int x = 0; x < NT; x++) {
      s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
      for (int e = 0; e < CK; e++) {
        mma<DT>(s[x], kf[e].x, kf[CK + e].x, kf[e].y, kf[CK + e].y, qf[x][2 * e][0], qf[x][2 * e][1]);
        mma<DT>(s[x], kf[e].z, kf[CK + e].z, kf[e].w, kf[CK + e].w, qf[x][2 * e + 1][0], qf[x][2 * e + 1][1]);
      }
    }
    // the next group's K
    long off = 0;
    if (i + 1 < n_it) {
      if (((i + 1) & 31) == 0) {
        pages = next_pages;
        next_pages = page_of(base + (i + 33 + lane) * kWarps);
      }
      off = locate(i + 1, ok);
      load_k(off);
    }
    const bool edge = !here || key0 < from || key0 + 16 > to;
    auto sees = [&](int key) { return here && key >= from && key < to; };
    bool up = false;
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[x][e] *= a.scale_log2;
        if (edge && !sees(key0 + g + 8 * (e >> 1))) s[x][e] = -INFINITY;
        up |= s[x][e] > m[x][e & 1] + kSlack;
      }
    if (__any_sync(kAll, up)) {
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float top = fmaxf(s[x][e], s[x][2 + e]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, w));
          top = fmaxf(top, m[x][e]);
          const float keep = join_weight(m[x][e], top);
          m[x][e] = top;
          l[x][e] *= keep;
#pragma unroll
          for (int d = 0; d < HD / 16; d++) o[d][x][e] *= keep, o[d][x][2 + e] *= keep;
        }
    }
    uint32_t pf[NT][2];
#pragma unroll
    for (int x = 0; x < NT; x++) {
      const float m0 = m[x][0] == -INFINITY ? 0.f : m[x][0], m1 = m[x][1] == -INFINITY ? 0.f : m[x][1];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float p0 = exp2_fast(s[x][2 * e] - m0), p1 = exp2_fast(s[x][2 * e + 1] - m1);
        pf[x][e] = transpose8x8(pack2<DT>(p0, p1));
        l[x][0] += p0;
        l[x][1] += p1;
      }
    }
    if (edge) {  // what no query sees is not multiplied by 0 but left out
      page_bad |= !here;
#pragma unroll
      for (int x = 0; x < 4; x++)
        if (!sees(key0 + 2 * t + (x & 1) + 8 * (x >> 1)))
#pragma unroll
          for (int e = 0; e < CV; e++) vf[x][e] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < CV; e++) {
      const uint32_t *v0 = &vf[0][e].x, *v1 = &vf[1][e].x, *v2 = &vf[2][e].x, *v3 = &vf[3][e].x;
#pragma unroll
      for (int d = 0; d < 4; d++) {
        const uint32_t a0 = __byte_perm(v0[d], v1[d], 0x5410), a1 = __byte_perm(v0[d], v1[d], 0x7632);
        const uint32_t a2 = __byte_perm(v2[d], v3[d], 0x5410), a3 = __byte_perm(v2[d], v3[d], 0x7632);
#pragma unroll
        for (int x = 0; x < NT; x++) mma<DT>(o[4 * e + d][x], a0, a1, a2, a3, pf[x][0], pf[x][1]);
      }
    }
    if (i + 1 < n_it) load_v(off);
  }
  if (page_bad && lane == 0) atomicExch(a.derr, TCB_ERR_BOUNDS);

  // the CTA's partial: o[4e + d] of lane (g, t) holds, for queries 2t and 2t + 1,
  // elements 64e + 8g + 2d and the next
#pragma unroll
  for (int x = 0; x < NT; x++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[x][e] += __shfl_xor_sync(kAll, l[x][e], w);
      const int q = 8 * x + 2 * t + e;
      if (g == 0) sm[warp][q] = m[x][e], sl[warp][q] = l[x][e];
#pragma unroll
      for (int d = 0; d < HD / 16; d++)
        *reinterpret_cast<float2 *>(&so[warp][q][64 * (d >> 2) + 8 * g + 2 * (d & 3)]) =
            make_float2(o[d][x][e], o[d][x][2 + e]);
    }
  __syncthreads();
  constexpr int per_row = HD / 2;  // pairs of elements
  for (int i = threadIdx.x; i < Q * per_row; i += kThreads) {
    const int q = i / per_row, d = 2 * (i - q * per_row);
    float top = sm[0][q];
#pragma unroll
    for (int w = 1; w < kWarps; w++) top = fmaxf(top, sm[w][q]);
    float2 acc = make_float2(0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float f = join_weight(sm[w][q], top);
      const float2 v = *reinterpret_cast<const float2 *>(&so[w][q][d]);
      acc.x += f * v.x, acc.y += f * v.y;
      sum += f * sl[w][q];
    }
    *reinterpret_cast<float2 *>(&so[0][q][d]) = acc;  // read by this thread alone
    if (d == 0) cm[q] = top, cl[q] = sum;
  }
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  if (x.parts) {
    // per query the prefix's partials' joint maximum, sum and weights, kThreads / Q
    // lanes a query
    constexpr int lanes = kThreads / Q;
    const int q = threadIdx.x / lanes, at = threadIdx.x % lanes;
    const float2 *ml = x.ml + (long)r * a.H + kh * G + min(h0 + q, G - 1);
    const long all_rows = (long)a.T * a.H;
    float top = -INFINITY, sum = 0.f;
    for (int w = at; w < x.parts; w += lanes) top = fmaxf(top, __ldcg(ml + w * all_rows).x);
#pragma unroll
    for (int w = 1; w < lanes; w <<= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, w));
    for (int w = at; w < x.parts; w += lanes) {
      const float2 v = __ldcg(ml + w * all_rows);
      const float g = join_weight(v.x, top);
      xg[w][q] = g;
      sum += g * v.y;
    }
#pragma unroll
    for (int w = 1; w < lanes; w <<= 1) sum += __shfl_xor_sync(kAll, sum, w);
    if (at == 0) xm[q] = top, xl[q] = sum;
  }
  if (n_rank > 1) cluster.sync();
  else __syncthreads();
  // this rank's slice of the outputs, over the cluster's partials in rank order
  const int live_q = min(Q, G - h0);
  uint16_t *out = static_cast<uint16_t *>(a.out) + r * a.ldo + (long)(kh * G + h0) * HD;
  // a thread's element pairs: its i-th is number (i * n_rank + c) * kThreads + threadIdx.x
  constexpr int kItems = Q * per_row / kThreads;
  auto query_of = [&](int i) { return ((i * n_rank + c) * kThreads + (int)threadIdx.x) / per_row; };
  const int d = 2 * ((int)threadIdx.x % per_row);
  auto store = [&](float2 (&acc)[kItems], float (&top)[kItems], float (&sum)[kItems]) {
    if (x.parts) {  // the prefix's part, in the order of its partials
      const long all_rows = (long)a.T * a.H, row0 = (long)r * a.H + kh * G + h0;
      float2 pre[kItems];
#pragma unroll
      for (int i = 0; i < kItems; i++) pre[i] = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int w = 0; w < x.parts; w++)
#pragma unroll
        for (int i = 0; i < kItems; i++) {
          const int q = query_of(i);
          if (q >= live_q) continue;
          const float2 v = __ldcg(reinterpret_cast<const float2 *>(x.o + (w * all_rows + row0 + q) * HD + d));
          pre[i].x += xg[w][q] * v.x, pre[i].y += xg[w][q] * v.y;
        }
#pragma unroll
      for (int i = 0; i < kItems; i++) {
        const int q = query_of(i);
        if (q >= live_q) continue;
        const float joint = fmaxf(top[i], xm[q]), f = join_weight(top[i], joint), g = join_weight(xm[q], joint);
        acc[i].x = f * acc[i].x + g * pre[i].x, acc[i].y = f * acc[i].y + g * pre[i].y;
        sum[i] = f * sum[i] + g * xl[q];
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; i++) {
      const int q = query_of(i);
      if (q >= live_q) continue;
      float v0 = sum[i] == 0.f ? 0.f : __fdiv_rn(acc[i].x, sum[i]), v1 = sum[i] == 0.f ? 0.f : __fdiv_rn(acc[i].y, sum[i]);
      *reinterpret_cast<uint32_t *>(out + (long)q * HD + d) = pack2<DT>(v0, v1);
    }
  };
  const long unit = (long)blockIdx.z * gridDim.y + blockIdx.y;
  auto part_o = [&](int w, int q, int d) {
    return reinterpret_cast<float2 *>(j.o + ((unit * j.parts + w) * Q + q) * HD + d);
  };
  auto part_ml = [&](int w, int q) { return j.ml + ((unit * j.parts + w) * n_rank + c) * Q + q; };
  float2 acc[kItems];
  float top[kItems], sum[kItems];
#pragma unroll
  for (int i = 0; i < kItems; i++) {
    const int q = query_of(i);
    acc[i] = make_float2(0.f, 0.f);
    top[i] = -INFINITY, sum[i] = 0.f;
    if (q >= live_q) continue;
    for (int w = 0; w < n_rank; w++) top[i] = fmaxf(top[i], *cluster.map_shared_rank(&cm[q], w));
    for (int w = 0; w < n_rank; w++) {
      const float f = join_weight(*cluster.map_shared_rank(&cm[q], w), top[i]);
      const float2 v = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(&so[0][q][d], w));
      acc[i].x += f * v.x, acc[i].y += f * v.y;
      sum[i] += f * *cluster.map_shared_rank(&cl[q], w);
    }
    if (j.parts > 1) {
      __stcg(part_o(part, q, d), acc[i]);
      __stcg(part_ml(part, q), make_float2(top[i], sum[i]));  // the same value from every thread of the query
    }
  }
  if (j.parts == 1) store(acc, top, sum);
  if (n_rank > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
  if (j.parts == 1) return;
  // the last of the clusters' ranks c joins their slices, in cluster order
  __threadfence();
  __syncthreads();
  __shared__ bool last;
  if (threadIdx.x == 0) {
    unsigned *n = j.arrived + unit * n_rank + c;
    last = atomicAdd(n, 1u) == (unsigned)j.parts - 1;
    if (last) *n = 0;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
#pragma unroll
  for (int i = 0; i < kItems; i++) {
    const int q = query_of(i);
    acc[i] = make_float2(0.f, 0.f);
    top[i] = -INFINITY, sum[i] = 0.f;
    if (q >= live_q) continue;
    for (int w = 0; w < j.parts; w++) top[i] = fmaxf(top[i], __ldcg(part_ml(w, q)).x);
#pragma unroll 4
    for (int w = 0; w < j.parts; w++) {
      const float2 ml = __ldcg(part_ml(w, q)), v = __ldcg(part_o(w, q, d));
      const float f = join_weight(ml.x, top[i]);
      acc[i].x += f * v.x, acc[i].y += f * v.y;
      sum[i] += f * ml.y;
    }
  }
  store(acc, top, sum);
}

template <int DT, int HD, int NT, int W>
cudaError_t launch(const PageAttnArgs &a, const DecodePlan &pl, const Join &j, const PrefixPartials &x, cudaStream_t s) {
  return launch_serve(k_page_decode<DT, HD, NT, W>, dim3(pl.split, pl.units / (a.B * a.max_rows), a.B * a.max_rows), 32 * W, 0, j.ranks,
                      s, a, j, x);
}

}  // namespace pd

DecodePlan page_decode_plan(const PageAttnArgs &a, bool suffix) {
  DecodePlan pl{};
  const int G = a.H / a.kv.n_kv_heads;
  pl.nt = G <= 8 ? 1 : 2;
  const int q = 8 * pl.nt;
  long seen = a.window < 0 ? a.max_len : std::min<long>(a.max_len, (long)a.window + a.sinks + 32);
  if (suffix) seen = std::max(0, a.max_len - a.prefix_len) + 16;
  const long groups = (seen + 15) / 16;  // of 16 positions, in the longest request
  const long units = (long)a.B * a.max_rows * a.kv.n_kv_heads * ((G + q - 1) / q);
  pl.units = (int)units;
  // CTAs per unit, doubled
  //  - while one wave of CTAs holds them and a warp keeps 2 groups: one
  //    sequence with 1024 positions in sight takes 8.2 us with 8, 9.4 with 4;
  //    one of 32768 with one KV head 17.1 with 128, 64.9 with 8
  //  - up to a cluster, while there are fewer than about 4 waves and a warp keeps
  //    128 KB of K and V, to even out ragged lengths: 64 sequences of up to
  //    32768, 8 KV heads: 554 us with 4 (2048 CTAs), 574 with 8, 645 with 2
  const long room = 148l * ((pl.nt == 1 ? 4 : 3) - (a.kv.head_dim == 128));
  int split = 1;
  while (split < 128) {
    const long per_warp = groups / (2 * split * 4), ctas = units * split;
    if (2 * ctas <= room && per_warp >= 2) split *= 2;
    else if (split < 8 && ctas < 12 * 148 && per_warp * 16 * a.kv.head_dim * 4 >= 128 << 10) split *= 2;
    else break;
  }
  pl.split = split;
  // 8 warps a CTA where each CTA has an SM to itself and a warp its group: with 8 KV
  // heads, one sequence of 1000 positions takes 7.8 us a call with 8 warps and
  // 9.0 with 4, four of them 8.0 and 9.6.  Clusters of 8 such CTAs find room for
  // fewer than 16 at once (128 CTAs: 17.4 us with 8 warps, 12.1 with 4).
  pl.warps = pl.nt == 1 && groups > 4l * split && units * split <= (split >= 8 ? 64 : 148) ? 8 : 4;
  if (split > 8) {
    const size_t n = (size_t)units * (split / 8);
    pl.o_bytes = n * q * a.kv.head_dim * sizeof(float);
    pl.bytes = pl.o_bytes + n * 8 * q * sizeof(float2);
    pl.counters = (size_t)units * 8 * sizeof(unsigned);
  }
  return pl;
}

int launch_page_decode(tcb_ctx *ctx, const PageAttnArgs &a, const DecodePlan &pl, void *scratch, const PrefixPartials &x,
                       cudaStream_t s) {
  pd::Join j{};
  j.ranks = std::min(pl.split, 8);
  j.parts = pl.split / j.ranks;
  if (j.parts > 1) {
    const int rc = ctx_tick(ctx, pl.counters);
    if (rc != TCB_OK) return rc;
    j.o = static_cast<float *>(scratch);
    j.ml = reinterpret_cast<float2 *>(static_cast<char *>(scratch) + pl.o_bytes);
    j.arrived = static_cast<unsigned *>(ctx->tick.p);
  }
  const bool h = a.kv.dtype == TCB_F16, wide = a.kv.head_dim == 128;
  cudaError_t e;
  if (pl.warps == 8) {
    if (wide) e = h ? pd::launch<TCB_F16, 128, 1, 8>(a, pl, j, x, s) : pd::launch<TCB_BF16, 128, 1, 8>(a, pl, j, x, s);
    else e = h ? pd::launch<TCB_F16, 64, 1, 8>(a, pl, j, x, s) : pd::launch<TCB_BF16, 64, 1, 8>(a, pl, j, x, s);
  } else if (pl.nt == 1) {
    if (wide) e = h ? pd::launch<TCB_F16, 128, 1, 4>(a, pl, j, x, s) : pd::launch<TCB_BF16, 128, 1, 4>(a, pl, j, x, s);
    else e = h ? pd::launch<TCB_F16, 64, 1, 4>(a, pl, j, x, s) : pd::launch<TCB_BF16, 64, 1, 4>(a, pl, j, x, s);
  } else {
    if (wide) e = h ? pd::launch<TCB_F16, 128, 2, 4>(a, pl, j, x, s) : pd::launch<TCB_BF16, 128, 2, 4>(a, pl, j, x, s);
    else e = h ? pd::launch<TCB_F16, 64, 2, 4>(a, pl, j, x, s) : pd::launch<TCB_BF16, 64, 2, 4>(a, pl, j, x, s);
  }
  return e == cudaSuccess ? TCB_OK : ctx_fail(ctx, e);
}

}  // namespace tcb
