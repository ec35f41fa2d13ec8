// tcb_page_rows.cu - attention over the paged cache for requests of many rows
// (prompts, chunks of prompts; tcb_page_attn) and for the shared prefix of a
// batch (tcb_prefix_attn), on the fifth-generation tensor cores.
//
// Mathematics: flash attention.  A CTA holds two tiles of 128 query rows of
// one KV head; a row is a (row of q, query head of the group) pair, so the G
// query heads that share a KV head share its tiles.  Per tile of 128
// positions, S = Q K^T (tcgen05, f32 in tensor memory), the running maximum
// and sum of the softmax per row (one thread a row), P = 2^(S - m) rounded
// to the cache's type and written over S, and O += P V with O in tensor
// memory.  O is rescaled only when a row's maximum has grown by more than
// 2^kSlack (weights up to 2^kSlack are far inside f16's range, sums are f32).
// The tensor cores take P in the cache's type only; the sum is of the weights
// before that rounding (after it each would have to be unpacked).  Against 64 bits a
// call errs by 2.8e-4 (f16) and 2.2e-3 (bf16), where one rounding of the result
// errs by 2.1e-4 and 1.6e-3.
//
// Bound: at 128 elements a head a tile costs 1024 tensor cycles (S and P V)
// and 16384 exponentials, 1024 cycles of the SM's 16 a cycle: both pipes are
// kept busy by the two tiles, whose softmax and products alternate.  One MMA
// warp for both keeps them in turn (with one each they fall into step: 560 us
// where this took 465).
// Measured: 8192 rows, 32 heads on 8 KV heads of 128, window 4096, bf16: 401 us =
// 1030 TFLOP/s, 0.63 of the cuBLAS burst rate, at full clocks;
// 436 to 448 us = 920 to 950 TFLOP/s in a loop of such calls, 0.65 to 0.67 of cuBLAS
// under the power limit.  1.85 us per pair of tiles and 128 positions, and 11 of a CTA's
// 72 us at its start and end.  168 registers a thread, with 56 to 60 bytes
// spilled.
//
//   warp 0      K and V tiles by TMA from the pages (128-byte swizzle; one box
//               per page and 64 elements, one lane each), 2 stages of each
//   warp 1      tensor-memory allocation, MMA issue
//   warps 2, 3  V tiles at the edge of some row's sight (see below)
//   warps 4-7, 8-11  softmax of tile 0 and 1: thread = row = lane of tensor
//               memory; they also load Q and write the result
//
// Masked positions: a row's weight there is 0, but 0 times a non-finite V is
// not.  Tiles that some row of the CTA sees only in part are gone through by
// warps 2 and 3 before the product: positions that no row sees are zeroed (they may
// be unwritten memory), and non-finite V elements of those that some rows see
// are set to 0 and noted; if any were found, the rows that do see them add them
// at the end.  Tiles in full sight of every row need nothing.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tcb_common.cuh"
#include "tcb_mv_ptx.cuh"
#include "tcb_page.h"

namespace tcb {
namespace pr {

using mv::mbar_arrive;
using mv::mbar_expect_tx;
using mv::mbar_init;
using mv::mbar_try_wait;
using mv::sa;

constexpr int kRows = 128;   // rows of a query tile
constexpr int kTiles = 2;    // query tiles of a CTA
constexpr int kKeys = 128;   // positions of a K/V tile
constexpr int kStages = 2;   // of K and of V
constexpr int kThreads = 384;
constexpr float kSlack = 8.f;
constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kHalf = kKeys * 128;  // bytes of 64 elements (one swizzle row) of 128 rows

struct Args {
  PageAttnArgs a;
  int G, tiles;        // query heads per KV head; CTAs along a request's rows
  int split;           // CTAs along the positions
  int box;             // rows of a TMA box
  int joined;          // rows of q in one run (prefix): row index / G is the row of q
  int prows;           // rows with partial results: those of q, or, where q has more than the
                       // requests can have (`each` then), max_rows for every request
  bool each;
  float *po;           // split or prefix: partial results [split][prows * H][HD]
  float2 *pml;         // and their (maximum, sum)
  CUtensorMap tk, tv;
};

// ----------------------------------------------------------------- PTX

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// operand in shared memory, rows of 128 bytes (128-byte swizzle, 8-row groups
// 1024 bytes apart): K-major; and, for V, whose rows are the positions (the
// product's K) and whose columns the outputs, MN-major with 64-column blocks
// kHalf apart
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(kHalf >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// f32 accumulator, 16-bit operands (0 f16, 1 bf16), M 128, N n
constexpr uint32_t idesc(int bf16, int b_mn, int n) {
  return 1u << 4 | (uint32_t)bf16 << 7 | (uint32_t)bf16 << 10 | (uint32_t)b_mn << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(kRows >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sa(bar)) : "memory");
}

#define TCB_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define TCB_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 lanes x 32 columns of tensor memory, without the wait
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%"
      "20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : TCB_R8(r, 0), TCB_R8(r, 8), TCB_R8(r, 16), TCB_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%"
      "18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::TCB_W8(r, 0),
      TCB_W8(r, 8), TCB_W8(r, 16), TCB_W8(r, 24), "r"(addr)
      : "memory");
}
// waits for the loads; r (32 words) is used after it
#define TCB_X8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void tmem_wait_ld(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TCB_X8(r, 0), TCB_X8(r, 8), TCB_X8(r, 16), TCB_X8(r, 24)::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *tm, int x, int pos, int head, int page,
                                         uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(pos), "r"(head), "r"(page), "r"(sa(bar))
      : "memory");
}

// Every wait ends: after 2^22 tries (seconds), or when another role has given
// up, the waiter reports a timeout and leaves its loop.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t phase, volatile int *stop, int *err) {
  for (uint32_t i = 0; i < 1u << 22; i++) {
    if (mbar_try_wait(bar, phase)) return true;
    if (*stop) return false;
  }
  *stop = 1;
  atomicExch(err, TCB_ERR_TIMEOUT);
  return false;
}
// one thread of a converged warp
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// the same after another role has given up (copies and products in flight)
__device__ __forceinline__ void drain(uint64_t *bar, uint32_t phase) {
  for (uint32_t i = 0; i < 1u << 20; i++)
    if (mbar_try_wait(bar, phase)) return;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == TCB_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}
// whether one of the two 16-bit elements of u is infinite or NaN
template <int DT>
__device__ __forceinline__ bool nonfinite2(uint32_t u) {
  constexpr uint32_t e = DT == TCB_F16 ? 0x7C00u : 0x7F80u;
  return (u & e) == e || (u >> 16 & e) == e;
}

// pairs of f32 in one register pair: one instruction for two lanes
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// the larger of three, NaN if one is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// bits 0 .. n-1
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? kAll : (1u << n) - 1u; }

struct Bars {
  uint64_t kfull[kStages], kempty[kStages], vfull[kStages], vready[kStages], vempty[kStages];
  uint64_t qready, sfull[kTiles], phalf[kTiles], pready[kTiles], odone[kTiles];
  uint64_t checked, drained;
};

template <int HD>
struct Layout {
  static constexpr int kTile = HD / 64 * kHalf;  // bytes of a 128-row tile of Q, K or V
  static constexpr int kQ = 0, kK = kTiles * kTile, kV = kK + kStages * kTile, kBars = kV + kStages * kTile;
  static constexpr int kSmem = kBars + (int)sizeof(Bars) + 64 + 1024;
};

// Pair of query tiles number `item` of all requests in order, by the whole warp:
// its request, and which of that request's it is (the last, the longest, first).
// False: there are only `upto` of them.
constexpr int kEach = 4;  // requests a lane looks at at once
__device__ __forceinline__ bool find(const Args &p, int item, int &b, int &tile, long &upto) {
  const PageAttnArgs &a = p.a;
  const int lane = threadIdx.x & 31;
  upto = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32 * kEach) {
    const int mine = b0 + kEach * lane;
    int rs[kEach + 1], n[kEach], sum = 0;
#pragma unroll
    for (int e = 0; e <= kEach; e++) rs[e] = a.row_start[min(mine + e, a.B)];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      const int r0 = min(max(rs[e], 0), a.T), rows = min(min(max(rs[e + 1], r0), a.T) - r0, a.max_rows) * p.G;
      n[e] = mine + e < a.B ? (rows + kTiles * kRows - 1) / (kTiles * kRows) : 0;
      sum += n[e];
    }
    int to = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(kAll, to, d);
      if (lane >= d) to += v;
    }
    const uint32_t at = __ballot_sync(kAll, item < upto + to);
    if (at) {
      int off = (int)(item - (upto + to - sum)), e = 0;
#pragma unroll
      for (int i = 0; i < kEach - 1; i++)
        if (e == i && off >= n[i]) off -= n[i], e++;
      const int left = e == 0 ? n[0] : e == 1 ? n[1] : e == 2 ? n[2] : n[3];
      b = __shfl_sync(kAll, mine + e, __ffs(at) - 1);
      tile = __shfl_sync(kAll, left - 1 - off, __ffs(at) - 1);
      return true;
    }
    upto += __shfl_sync(kAll, to, 31);
  }
  return false;
}

// kPacked: CTAs count the requests' pairs of tiles (find), not tiles for each request
template <int DT, int HD, bool kPacked>
__global__ void __launch_bounds__(kThreads, 1) k_page_rows(const __grid_constant__ Args p) {
  using L = Layout<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Bars &bar = *reinterpret_cast<Bars *>(sm + L::kBars);
  // what the CTA's rows see: least and largest [lo, hi) and first positions
  __shared__ int hi_min, hi_max, lo_min, lo_max, first_min, first_max;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int stop;
  __shared__ int dirty, request;
  const PageAttnArgs &a = p.a;
  const int warp = __shfl_sync(kAll, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // the warp's number in a uniform register
  const int part = blockIdx.x % p.split, kh = blockIdx.y;
  int tile = p.tiles - 1 - (int)(blockIdx.x / p.split), b = blockIdx.z;  // the longest first

  mv::pdl_wait();
  mv::pdl_launch_dependents();
  if constexpr (kPacked) {
    long upto;
    if (blockIdx.x + blockIdx.y == 0 && warp == 0) {
      // requests without rows have no CTA that looks at their lengths; row
      // starts that fall may hold more tiles than there are CTAs
      for (int i = lane; i < a.B; i += 32) {
        const int l = a.kv_len[i];
        if (l < 0 || l > a.max_len || l > (long)a.width << a.page_shift || a.row_start[i + 1] < a.row_start[i]) atomicExch(a.derr, TCB_ERR_BOUNDS);
      }
    }
    if (!find(p, (int)(blockIdx.x / p.split), b, tile, upto)) return;
  }
  // the request's rows
  int r0 = 0, n = a.T, len = 0;
  if (!p.joined) {
    r0 = min(max(a.row_start[b], 0), a.T);
    n = min(max(a.row_start[b + 1], r0), a.T) - r0;
    len = a.kv_len[b];
    const bool bad = len < 0 || len > a.max_len || len > (long)a.width << a.page_shift;
    if ((bad || n > a.max_rows || a.row_start[b + 1] < a.row_start[b]) && threadIdx.x == 0) atomicExch(a.derr, TCB_ERR_BOUNDS);
    if (bad) len = 0;
    n = min(n, a.max_rows);
  }
  const int x0 = tile * kTiles * kRows, rows = n * p.G;  // (row, head) pairs: fewer than the bytes of q
  if (x0 >= rows) return;
  const int n_real = p.joined ? n : min(max(a.row_start[b + 1], r0), a.T) - r0;  // positions count from the true number of rows
  const int active = rows - x0 > kRows ? 2 : 1;  // query tiles with rows

  // softmax threads: the row and its Q, asked for before the setup (rows that do
  // not exist are zero): a warp takes its 32 rows one after the other, HD / 8
  // lanes a row
  const int qt = (warp >> 2) - 1, tid = threadIdx.x & 127;  // warps 4-7: 0, 8-11: 1
  const int x = x0 + qt * kRows + tid;
  const bool live = qt >= 0 && x < rows;
  const int xi = live ? (int)((unsigned)x / (unsigned)p.G) : 0;
  const int head = kh * p.G + (live ? x - xi * p.G : 0);
  const long r = r0 + xi;
  constexpr int kLanes = HD / 8;
  uint4 qv[kLanes];
  if (qt >= 0) {
    const long at = live && a.scale_log2 != 0.f ? r * a.ldq + (long)head * HD : -1;
#pragma unroll
    for (int i = 0; i < kLanes; i++) {
      const long off = __shfl_sync(kAll, at, i * (32 / kLanes) + lane / kLanes);
      qv[i] = make_uint4(0, 0, 0, 0);
      if (off >= 0) qv[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + off + 8 * (lane % kLanes));
    }
  }

  if (threadIdx.x == 0) {
    hi_min = lo_min = first_min = 0x7FFFFFFF;
    hi_max = lo_max = first_max = 0;
    stop = 0;
    dirty = 0;
    request = b;
    for (int i = 0; i < kStages; i++) {
      mbar_init(bar.kfull + i, 1);
      mbar_init(bar.kempty + i, 1);
      mbar_init(bar.vfull + i, 1);
      mbar_init(bar.vready + i, 2);
      mbar_init(bar.vempty + i, 1);
    }
    mbar_init(&bar.qready, kRows * kTiles);
    mbar_init(&bar.checked, 2);
    mbar_init(&bar.drained, 1);
    for (int i = 0; i < kTiles; i++) {
      mbar_init(bar.sfull + i, 1);
      mbar_init(bar.phalf + i, kRows);
      mbar_init(bar.pready + i, kRows);
      mbar_init(bar.odone + i, 1);
    }
    mv::fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(sa(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncthreads();

  // what the row sees
  int hi = 0, lo = 0, first = 0;
  if (live) {
    if (p.joined) {
      int kl = a.kv_len[xi];
      if (kl < 0 || kl > a.max_len || kl > (long)a.width << a.page_shift) kl = 0;  // the suffix's kernel reports it
      hi = min(kl, a.prefix_len);
    } else {
      const int pos = len - n_real + xi;
      hi = max(pos + 1, 0);
      lo = a.window < 0 ? 0 : (int)min((long)hi, max(0l, (long)pos - a.window + 1));
      first = min(a.sinks, lo);
      if (lo == hi) hi = first, lo = 0;  // no window: the first positions alone
      if (first >= lo) lo = first = 0;
    }
  }
  if (qt >= 0) {
    // rows that see something bound the tiles; every row bounds the full sight
    const int far = 0x7FFFFFFF;
    const int v[6] = {__reduce_min_sync(kAll, live ? hi : far), __reduce_max_sync(kAll, hi),
                      __reduce_min_sync(kAll, hi > 0 ? lo : far), __reduce_max_sync(kAll, lo),
                      __reduce_min_sync(kAll, hi > 0 ? first : far), __reduce_max_sync(kAll, first)};
    if (lane == 0) {
      atomicMin(&hi_min, v[0]), atomicMax(&hi_max, v[1]), atomicMin(&lo_min, v[2]);
      atomicMax(&lo_max, v[3]), atomicMin(&first_min, v[4]), atomicMax(&first_max, v[5]);
    }
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  // 128-position tiles: those of the first positions, then [t0, t1)
  const int ts = (first_max + kKeys - 1) / kKeys, t0 = max(min(lo_min, hi_max) / kKeys, ts);
  const int t1 = max((hi_max + kKeys - 1) / kKeys, t0);
  const int all = ts + t1 - t0;
  const int u0 = (int)((long)all * part / p.split), u1 = (int)((long)all * (part + 1) / p.split);
  auto key_of = [&](int u) { return (u < ts ? u : u - ts + t0) * kKeys; };
  auto in_full_sight = [&](int k0) {
    return k0 + kKeys <= hi_min && (k0 >= lo_max || k0 + kKeys <= first_min);
  };
  // a scale that is not positive goes into Q: its signs, or zeros
  const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // K and V: lane = (box of the tile, 64 elements)
      const int boxes = kKeys / p.box, at = lane / (HD / 64), half = lane % (HD / 64);
      const bool mine = at < boxes;
      const int *table = p.joined ? a.prefix : a.tables + b * a.ldt;
      auto page_at = [&](int u) {
        const int pos = key_of(u) + at * p.box;
        // outside the pools: zeros, for what no row sees (its pages may have been given back)
        if (u >= u1 || !mine || pos >= hi_max || (pos >= first_max && pos + p.box <= lo_min)) return a.kv.n_pages;
        const int pg = table[pos >> a.page_shift];
        if (pg >= 0 && pg < a.kv.n_pages) return pg;
        atomicExch(a.derr, TCB_ERR_BOUNDS);
        return a.kv.n_pages;
      };
      const uint32_t dst = half * kHalf + at * p.box * 128;
      int page = page_at(u0), nk = 0, nv = 0;  // tiles asked for
      bool ok = true;
      for (int u = u0; u < u1 && ok; u++) {
        const int i = u - u0, st = i % kStages;
        const uint32_t ph = ((i / kStages) & 1) ^ 1;
        const int y = (key_of(u) + at * p.box) & (a.kv.page - 1);
        const int next = page_at(u + 1);
        ok = wait(bar.kempty + st, ph, &stop, a.derr);
        if (!__all_sync(kAll, ok)) break;
        if (lane == 0) mbar_expect_tx(bar.kfull + st, L::kTile);
        __syncwarp();
        if (mine) tma_load(sa(sm + L::kK + st * L::kTile) + dst, &p.tk, half * 64, y, kh, page, bar.kfull + st);
        nk++;
        ok = wait(bar.vempty + st, ph, &stop, a.derr);
        if (!__all_sync(kAll, ok)) break;
        if (lane == 0) mbar_expect_tx(bar.vfull + st, L::kTile);
        __syncwarp();
        if (mine) tma_load(sa(sm + L::kV + st * L::kTile) + dst, &p.tv, half * 64, y, kh, page, bar.vfull + st);
        nv++;
        page = next;
      }
      // a whole run uses every tile; one given up waits for its copies here
      if (stop) {
        for (int t = nk - 1; t >= max(0, nk - kStages); t--) drain(bar.kfull + t % kStages, (t / kStages) & 1);
        for (int t = nv - 1; t >= max(0, nv - kStages); t--) drain(bar.vfull + t % kStages, (t / kStages) & 1);
      }
    } else if (warp == 1) {
      // The whole warp follows the barriers and one elected thread issues, so
      // that the descriptors stay in uniform registers.
      constexpr uint32_t ids = idesc(DT == TCB_BF16, 0, kKeys), ido = idesc(DT == TCB_BF16, 1, HD);
      const uint32_t base = sa(sm);
      auto s_mma = [&](int q, int st) {
        const uint64_t qd = desc_k(base + L::kQ + q * L::kTile), kd = desc_k(base + L::kK + st * L::kTile);
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          const uint64_t o = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
          mma_ss(tmem + q * kKeys, qd + o, kd + o, ids, k > 0);
        }
        commit(bar.sfull + q);
      };
      bool ok = u0 < u1 && wait(&bar.qready, 0, &stop, a.derr) && wait(bar.kfull, 0, &stop, a.derr);
      fence_after();
      if (ok && elect()) {
        for (int q = 0; q < active; q++) s_mma(q, 0);
        commit(bar.kempty);
      }
      __syncwarp();
      for (int u = u0; u < u1 && ok; u++) {
        const int i = u - u0, st = i % kStages, sn = (i + 1) % kStages;
        const uint64_t vd = desc_mn(base + L::kV + st * L::kTile);
        ok = wait(bar.vready + st, (i / kStages) & 1, &stop, a.derr);
        if (ok && u + 1 < u1) ok = wait(bar.kfull + sn, ((i + 1) / kStages) & 1, &stop, a.derr);
#pragma unroll
        for (int q = 0; q < kTiles; q++) {
          if (q >= active) break;
          // P V by halves of the positions: the first runs while the softmax
          // forms the second
          auto pv = [&](int half) {
#pragma unroll
            for (int k = 4 * half; k < 4 * half + 4; k++)
              mma_ts(tmem + kTiles * kKeys + q * HD, tmem + q * kKeys + 8 * k, vd + (k * 2048 >> 4), ido, i > 0 || k > 0);
          };
          ok = ok && wait(bar.phalf + q, i & 1, &stop, a.derr);
          if (!ok) break;
          fence_after();
          if (elect()) pv(0);
          __syncwarp();
          ok = wait(bar.pready + q, i & 1, &stop, a.derr);
          if (!ok) break;
          fence_after();
          if (elect()) {
            pv(1);
            // the next S goes over this P: the MMAs of one thread run in order
            if (u + 1 < u1) s_mma(q, sn);
            commit(bar.odone + q);
            if (q == active - 1) {
              commit(bar.vempty + st);
              if (u + 1 < u1) commit(bar.kempty + sn);
            }
          }
          __syncwarp();
        }
      }
      if (stop) {  // products in flight end before the tensor memory goes
        if (elect()) commit(&bar.drained);
        __syncwarp();
        drain(&bar.drained, 0);
      }
    } else {
      // V at the edge of some row's sight: positions that no row sees are
      // zeroed, those that only some see are searched for non-finite elements
      bool ok = true, found = false;
      for (int u = u0; u < u1 && ok; u++) {
        const int i = u - u0, st = i % kStages;
        ok = wait(bar.vfull + st, (i / kStages) & 1, &stop, a.derr);
        ok = __all_sync(kAll, ok);
        if (!ok) break;
        const int k0 = key_of(u);
        if (!in_full_sight(k0)) {
          // 8 lanes a row of 128 bytes (the swizzle stays within it), 8 rows at a time
          uint4 *v = reinterpret_cast<uint4 *>(sm + L::kV + st * L::kTile) + (threadIdx.x - 64);
          constexpr uint32_t e = DT == TCB_F16 ? 0x7C007C00u : 0x7F807F80u, one = DT == TCB_F16 ? 0x04000400u : 0x00800080u;
#pragma unroll 4
          for (int j0 = 0; j0 < kKeys; j0 += 8) {
            const int key = k0 + j0 + ((threadIdx.x - 64) >> 3);
            if (key < hi_min && (key >= lo_max || key < first_min)) continue;
            const bool none = key >= hi_max || (key < lo_min && key >= first_max);
#pragma unroll
            for (int h = 0; h < HD / 64; h++) {
              uint4 *at = v + (h * kKeys + j0) * 8;
              uint4 w = *at;
              // an exponent of ones carries into the sign's place
              const uint32_t bad = ((w.x & e) + one) | ((w.y & e) + one) | ((w.z & e) + one) | ((w.w & e) + one);
              if (none) {
                *at = make_uint4(0, 0, 0, 0);
              } else if (bad & 0x80008000u) {
                uint32_t *wd = &w.x;
#pragma unroll
                for (int d = 0; d < 4; d++) {
                  const uint32_t b = ((wd[d] & e) + one) & 0x80008000u;
                  wd[d] &= ~((b >> 15) * 0xFFFFu);
                }
                *at = w;
                found = true;
              }
            }
          }
          mv::fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.vready + st);
      }
      if (found) dirty = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.checked);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // Q into the swizzled tile
    if (qt < active) {
      const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
      for (int i = 0; i < kLanes; i++) {
        const int row = (warp & 3) * 32 + i * (32 / kLanes) + lane / kLanes, c = lane % kLanes;
        qv[i].x ^= sign, qv[i].y ^= sign, qv[i].z ^= sign, qv[i].w ^= sign;
        *reinterpret_cast<uint4 *>(sm + L::kQ + qt * L::kTile + row * 128 + (c >> 3) * kHalf + (((c & 7) ^ (row & 7)) << 4)) = qv[i];
      }
      mv::fence_proxy_async();
    }
    mbar_arrive(&bar.qready);
    if (qt < active) {
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
      const uint32_t ts_addr = tmem + lanes + qt * kKeys, to_addr = tmem + lanes + kTiles * kKeys + qt * HD;
      float m = -INFINITY;           // in scaled units
      uint64_t l0 = 0ull, l1 = 0ull;  // the sum, in four parts
      bool ok = true;
      for (int u = u0; u < u1; u++) {
        const int i = u - u0, k0 = key_of(u);
        ok = wait(bar.sfull + qt, i & 1, &stop, a.derr);
        if (!__all_sync(kAll, ok)) break;
        fence_after();
        uint32_t s[kKeys];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld(ts_addr + 32 * c, s + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_wait_ld(s + 32 * c);
        if (!in_full_sight(k0)) {
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int at = k0 + 32 * c;
            const uint32_t seen = below(hi - at) & (~below(lo - at) | below(first - at));
#pragma unroll
            for (int j = 0; j < 32; j++)
              if (!(seen >> j & 1)) s[32 * c + j] = 0xFF800000u;
          }
        }
        auto sf = [&](int j) { return __uint_as_float(s[j]); };
        float tops[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          tops[c] = max3_nan(sf(c), sf(c + 4), sf(c + 8));
#pragma unroll
          for (int j = c + 12; j < kKeys; j += 8) tops[c] = max3_nan(tops[c], sf(j), j + 4 < kKeys ? sf(j + 4) : sf(j));
        }
        float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]) * scale;
        if (!(top < INFINITY)) top = NAN;  // infinite and NaN scores make the row NaN
        const bool up = top > m + kSlack || top != top;
        if (i == 0) {
          if (up) m = top;
        } else if (__any_sync(kAll, up)) {
          // O is at rest once the last product is done
          ok = wait(bar.odone + qt, (i - 1) & 1, &stop, a.derr);
          if (!__all_sync(kAll, ok)) break;
          fence_after();
          // every row of the warp takes its new maximum, so that the next
          // time is far off
          const float next = top > m || up ? top : m;
          const float keep = next == m ? 1.f : m == -INFINITY ? 0.f : exp2f(m - next);
          m = next;
          l0 = fma2(l0, pair(keep, keep), 0ull);
          l1 = fma2(l1, pair(keep, keep), 0ull);
#pragma unroll 1
          for (int c = 0; c < HD / 32; c++) {
            uint32_t o[32];
            tmem_ld(to_addr + 32 * c, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
            tmem_st(to_addr + 32 * c, o);
          }
          tmem_wait_st();
        }
        const float sub = m == -INFINITY ? 0.f : m;
        const uint64_t mul = pair(scale, scale), off = pair(-sub, -sub);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t pk[32];
#pragma unroll
          for (int j = 0; j < 32; j++) {
            const uint64_t x = fma2(pair(sf(64 * c + 2 * j), sf(64 * c + 2 * j + 1)), mul, off);
            float2 w = split2(x);
            w = make_float2(exp2_fast(w.x), exp2_fast(w.y));
            if (j & 1) l1 = add2(l1, pair(w.x, w.y));
            else l0 = add2(l0, pair(w.x, w.y));
            pk[j] = pack2<DT>(w.x, w.y);
          }
          tmem_st(ts_addr + 32 * c, pk);
          tmem_wait_st();
          fence_before();
          mbar_arrive((c ? bar.pready : bar.phalf) + qt);
        }
      }
      const int iters = u1 - u0;
      if (iters > 0 && ok) ok = wait(bar.odone + qt, (iters - 1) & 1, &stop, a.derr);
      if (ok) ok = wait(&bar.checked, 0, &stop, a.derr);
      ok = __all_sync(kAll, ok);
      fence_after();
      const float2 la = split2(l0), lb = split2(l1);
      const float l = (la.x + la.y) + (lb.x + lb.y);
      const bool empty = iters == 0 || m == -INFINITY;
      const float inv = p.po ? 1.f : __fdiv_rn(1.f, empty ? 1.f : l);
      const long prow = ((long)part * p.prows + (p.each ? (long)request * a.max_rows + xi : r)) * a.H + head;
      if (p.po && live) p.pml[prow] = make_float2(empty ? -INFINITY : m, empty ? 0.f : l);
      uint32_t ahead[32];  // the next 32 columns, on their way while these are written
      if (iters > 0 && ok) tmem_ld(to_addr, ahead);
#pragma unroll 1
      for (int c = 0; c < HD / 32 && ok; c++) {
        uint32_t o[32];
        if (iters > 0) {
          tmem_wait_ld(ahead);
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = ahead[j];
          if (c + 1 < HD / 32) tmem_ld(to_addr + 32 * (c + 1), ahead);
        }
#pragma unroll
        for (int j = 0; j < 32; j++) o[j] = empty ? 0u : __float_as_uint(__uint_as_float(o[j]) * inv);
        if (dirty && live) {
          // the non-finite V elements of edge tiles, for the rows that see them
          const int *table = p.joined ? a.prefix : a.tables + request * a.ldt;
          for (int u = u0; u < u1; u++) {
            const int k0 = key_of(u);
            if (in_full_sight(k0)) continue;
            for (int key = k0; key < min(k0 + kKeys, hi); key++) {
              if (key < lo && key >= first) continue;
              const int pg = table[key >> a.page_shift];
              if (pg < 0 || pg >= a.kv.n_pages) continue;
              const uint32_t *v = reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(a.kv.v) + pg * a.kv.page_stride +
                                                                     kh * a.kv.head_stride + (key & (a.kv.page - 1)) * a.kv.pos_stride + 32 * c);
#pragma unroll
              for (int j = 0; j < 16; j++) {
                const uint32_t w = v[j];
                if (!nonfinite2<DT>(w)) continue;
                const uint16_t e0 = (uint16_t)w, e1 = (uint16_t)(w >> 16);
                if (nonfinite2<DT>(e0)) o[2 * j] = __float_as_uint(__uint_as_float(o[2 * j]) + (DT == TCB_BF16 ? bf16_to_f32(e0) : half_exact(e0)));
                if (nonfinite2<DT>(e1)) o[2 * j + 1] = __float_as_uint(__uint_as_float(o[2 * j + 1]) + (DT == TCB_BF16 ? bf16_to_f32(e1) : half_exact(e1)));
              }
            }
          }
        }
        // through this warp's part of the Q tile (its products are done), so that
        // whole sectors are written
        uint8_t *stage = sm + L::kQ + qt * L::kTile + (warp & 3) * 4096;
        __syncwarp();
        if (p.po) {
#pragma unroll
          for (int j = 0; j < 8; j++)
            *reinterpret_cast<uint4 *>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int row = 4 * i + (lane >> 3), j = lane & 7;
            const long to = __shfl_sync(kAll, live ? prow : -1, row);
            if (to >= 0) *reinterpret_cast<uint4 *>(p.po + to * HD + 32 * c + 4 * j) = *reinterpret_cast<const uint4 *>(stage + row * 128 + ((j ^ (row & 7)) << 4));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = pack2<DT>(__uint_as_float(o[8 * j + 2 * e]), __uint_as_float(o[8 * j + 2 * e + 1]));
            *reinterpret_cast<uint4 *>(stage + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          const long out_row = live ? r * a.ldo + (long)head * HD : -1;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = 8 * i + (lane >> 2), j = lane & 3;
            const long to = __shfl_sync(kAll, out_row, row);
            if (to >= 0)
              *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + to + 32 * c + 8 * j) = *reinterpret_cast<const uint4 *>(stage + row * 64 + ((j ^ (row >> 1 & 3)) << 4));
          }
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// out = the partials of every split joined in order, for the rows of requests
// (4 elements a thread; H * HD / 4 threads a row; prows and each as in Args)
template <int DT, int HD>
__global__ void __launch_bounds__(256) k_rows_join(const PageAttnArgs a, int split, int prows, bool each, const float *po, const float2 *pml) {
  mv::pdl_wait();
  mv::pdl_launch_dependents();
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = i / (HD / 4), rows = (long)prows * a.H;
  if (row >= rows) return;
  const int d = (int)(i - row * (HD / 4)) * 4;
  long r = row / a.H;
  const int head = (int)(row - r * a.H);
  // rows outside every request keep what they hold
  bool mine = false;
  if (each) {
    const int b = (int)(r / a.max_rows), at = (int)(r - (long)b * a.max_rows), r0 = min(max(a.row_start[b], 0), a.T);
    mine = at < min(a.row_start[b + 1], a.T) - r0;
    r = r0 + at;
  } else {
    for (int b = 0; b < a.B && !mine; b++) mine = r >= a.row_start[b] && r < min(a.row_start[b + 1], max(a.row_start[b], 0) + a.max_rows);
  }
  if (!mine) return;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < split; s++) top = fmaxf(top, pml[s * rows + row].x);
  for (int s = 0; s < split; s++) {
    const float2 ml = pml[s * rows + row];
    const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
    const float4 v = *reinterpret_cast<const float4 *>(po + (s * rows + row) * HD + d);
    acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
    sum += f * ml.y;
  }
  const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
  uint2 w = make_uint2(pack2<DT>(acc.x * inv, acc.y * inv), pack2<DT>(acc.z * inv, acc.w * inv));
  if (sum == 0.f) w = make_uint2(0, 0);
  *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + r * a.ldo + (long)head * HD + d) = w;
}

bool tensor_map(CUtensorMap *tm, const tcb_kv_pages &kv, const void *base, int box) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page, (cuuint64_t)kv.n_kv_heads, (cuuint64_t)kv.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv.pos_stride * 2, (cuuint64_t)kv.head_stride * 2, (cuuint64_t)kv.page_stride * 2};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, one[4] = {1, 1, 1, 1};
  return enc(tm, kv.dtype == TCB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
             const_cast<void *>(base), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int HD>
cudaError_t launch(const Args &p, bool packed, dim3 grid, cudaStream_t s) {
  auto go = [&](auto by_count) {
    constexpr auto kernel = k_page_rows<DT, HD, decltype(by_count)::value>;
    // the attribute belongs to the kernel on the current device
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<HD>::kSmem);
    return e != cudaSuccess ? e : launch_serve(kernel, grid, kThreads, Layout<HD>::kSmem, 1, s, p);
  };
  cudaError_t e = packed ? go(std::integral_constant<bool, true>()) : go(std::integral_constant<bool, false>());
  if (e == cudaSuccess && p.po && !p.joined) {
    const long n = (long)p.prows * p.a.H * (HD / 4);
    e = launch_serve(k_rows_join<DT, HD>, dim3((unsigned)((n + 255) / 256)), 256, 0, 1, s, p.a, p.split, p.prows, p.each, p.po, p.pml);
  }
  return e;
}

}  // namespace pr

RowsPlan page_rows_plan(const PageAttnArgs &a) {
  RowsPlan pl{};
  const bool joined = a.prefix != nullptr;
  const long rows = (long)(joined ? a.T : a.max_rows) * (a.H / a.kv.n_kv_heads);
  pl.tiles = (int)((rows + pr::kTiles * pr::kRows - 1) / (pr::kTiles * pr::kRows));
  const long seen = joined ? a.prefix_len : a.window < 0 ? a.max_len : std::min<long>(a.max_len, (long)a.window + a.sinks + 32);
  // CTAs: the longest request's pairs of tiles for every request, many of which
  // may be empty, or as many as the rows of all requests can fill, each of which
  // then looks for its own (up to 1 us), where that spares 3 empty CTAs an SM.
  // 256 requests of one row and one of 2048 (65000 spared): 920 us / 545; 4 of 64
  // and one of 2048 (952): 85.7 / 80.0; 7 of 64 to 515 (336): 28.3 / 27.3, and in
  // another case 29.7 / 30.9.
  pl.items = pl.tiles * (joined ? 1l : a.B);
  const long filled = (long)a.T * (a.H / a.kv.n_kv_heads) / (pr::kTiles * pr::kRows) + std::min(a.T, a.B);
  pl.packed = !joined && (pl.items - filled) * a.kv.n_kv_heads >= 3 * 148;
  if (pl.packed) pl.items = filled;
  const long keys = (seen + pr::kKeys - 1) / pr::kKeys, units = std::max(1l, pl.items * a.kv.n_kv_heads);
  // CTAs along the positions where the others leave SMs idle, two tiles each at the least
  pl.split = (int)std::max<long>(1, std::min<long>(148 / units, keys / 2));
  if (joined) pl.split = std::min(pl.split, kMaxPrefixParts);
  pl.partial = joined || pl.split > 1;
  // a padded batch has rows of q outside every request: no room for theirs
  pl.each = !joined && (long)a.B * a.max_rows < a.T;
  pl.prows = pl.each ? a.B * a.max_rows : a.T;
  if (pl.partial) {
    const size_t n = (size_t)pl.split * pl.prows * a.H;
    pl.o_bytes = n * a.kv.head_dim * sizeof(float);
    pl.bytes = pl.o_bytes + n * sizeof(float2);
  }
  return pl;
}

int launch_page_rows(tcb_ctx *ctx, const PageAttnArgs &a, const RowsPlan &pl, void *scratch, cudaStream_t s) {
  pr::Args p{};
  p.a = a;
  p.G = a.H / a.kv.n_kv_heads;
  p.tiles = pl.tiles;
  p.split = pl.split;
  p.joined = a.prefix != nullptr;
  p.box = std::min(a.kv.page, pr::kKeys);
  p.prows = pl.prows;
  p.each = pl.each;
  if (pl.partial) {
    p.po = static_cast<float *>(scratch);
    p.pml = reinterpret_cast<float2 *>(static_cast<char *>(scratch) + pl.o_bytes);
  }
  if (!pr::tensor_map(&p.tk, a.kv, a.kv.k, p.box) || !pr::tensor_map(&p.tv, a.kv, a.kv.v, p.box))
    return ctx_fail(ctx, cudaErrorInvalidValue);
  const dim3 grid((pl.packed ? (unsigned)pl.items : (unsigned)p.tiles) * p.split, a.kv.n_kv_heads, p.joined || pl.packed ? 1 : a.B);
  const bool h = a.kv.dtype == TCB_F16;
  cudaError_t e;
  if (a.kv.head_dim == 128) e = h ? pr::launch<TCB_F16, 128>(p, pl.packed, grid, s) : pr::launch<TCB_BF16, 128>(p, pl.packed, grid, s);
  else e = h ? pr::launch<TCB_F16, 64>(p, pl.packed, grid, s) : pr::launch<TCB_BF16, 64>(p, pl.packed, grid, s);
  return e == cudaSuccess ? TCB_OK : ctx_fail(ctx, e);
}

}  // namespace tcb
