// tcb_serve.cu - the serving operators' C entry points (page plan, K/V
// append, attention over the pages) with their argument checks, and the
// kernels of the plan and the append.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/tcb.h"
#include "tcb_common.cuh"
#include "tcb_ctx.h"
#include "tcb_mv_ptx.cuh"
#include "tcb_page.h"

namespace {

bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128 || page == 256; }
int log2i(int v) { return v <= 1 ? 0 : 1 + log2i(v / 2); }
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// bytes of an array (none where n is 0)
struct Span {
  const void *p;
  long n;
  uintptr_t at() const { return reinterpret_cast<uintptr_t>(p); }
};
bool meet(const Span &a, const Span &b) { return a.n > 0 && b.n > 0 && a.at() < b.at() + b.n && b.at() < a.at() + a.n; }
// whether a lies in one of `count` rows of `n` bytes, `step` apart
bool meets_rows(const Span &a, const void *rows, int count, long n, long step) {
  if (count < 1 || !meet(a, {rows, (count - 1) * step + n})) return false;
  if (count == 1 || a.at() < reinterpret_cast<uintptr_t>(rows)) return true;
  const long off = (long)(a.at() - reinterpret_cast<uintptr_t>(rows)) % step;  // from the start of its row
  return off < n || off + a.n > step;
}

// ------------------------------------------------------------ page plan

struct PlanArgs {
  int B, page, page_shift, width, free_cap, rows;
  const int *cached, *fresh;
  int *tables;
  long ldt;
  const int *free_pages, *n_free;
  int *row_start, *kv_len;
  int64_t *slots;
  int *positions, *balance, *taken;
};

// exclusive sum over the CTA's threads, and the total
template <int NT>
__device__ __forceinline__ long block_scan(long v, long *warp_sums, long &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  // every warp scans the warps' sums
  const long own = lane < NT / 32 ? warp_sums[lane] : 0;
  long y = own;
#pragma unroll
  for (int o = 1; o < NT / 32; o <<= 1) {
    const long z = __shfl_up_sync(0xFFFFFFFFu, y, o);
    if (lane >= o) y += z;
  }
  total = __shfl_sync(0xFFFFFFFFu, y, NT / 32 - 1);
  return __shfl_sync(0xFFFFFFFFu, y - own, warp) + x - v;
}

// the pages that a request lacks, -1 where its lengths, rows or table do not
// hold it (row_end: one past its last row)
__device__ __forceinline__ long pages_lacking(const PlanArgs &a, long cached, long fresh, long row_end) {
  const long end = cached + fresh;
  if (cached < 0 || fresh < 0 || row_end > a.rows || end > (long)a.width << a.page_shift || end > 0x7FFFFFFF) return -1;
  return ((end + a.page - 1) >> a.page_shift) - ((cached + a.page - 1) >> a.page_shift);
}

// Every CTA scans all requests (two loads and two scans over at most
// TCB_PAGE_PLAN_MAX requests) and keeps the row and page offsets in shared
// memory, so the rows and table entries can be written by the whole grid in
// one launch without waiting on one another.  Thread t holds the requests
// t * items .. of its part; sums are 64-bit, so no length overflows them.
template <int NT>
__global__ void __launch_bounds__(NT) k_page_plan(const PlanArgs a) {
  extern __shared__ int sh[];
  int *rs = sh;              // [B + 1] first row of each request
  int *pg = sh + a.B + 1;    // [B] pages taken before it; -1: refused
  int *cs = pg + a.B;        // [B] positions cached
  __shared__ long sums[NT / 32];
  __shared__ int taken_s;
  __shared__ long long asked_s;
  tcb::mv::pdl_wait();
  tcb::mv::pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int items = (a.B + NT - 1) / NT;
  const int b0 = tid * items, b1 = min(a.B, b0 + items);
  const long n_free = min(max(*a.n_free, 0), a.free_cap);
  if (tid == 0) taken_s = 0, asked_s = 0;

  // the lengths, read once where a thread has one request
  const int c0 = b0 < b1 ? a.cached[b0] : 0, f0 = b0 < b1 ? a.fresh[b0] : 0;
  auto cached = [&](int b) { return b == b0 ? c0 : a.cached[b]; };
  auto fresh = [&](int b) { return b == b0 ? f0 : a.fresh[b]; };
  long sum = 0, total;
  for (int b = b0; b < b1; b++) sum += max(fresh(b), 0);
  long row = block_scan<NT>(sum, sums, total);
  // the pages each request lacks, 0 where it does not fit its rows or table
  const long r0 = row;
  long lacks = 0;
  for (int b = b0; b < b1; b++) {
    const long f = fresh(b);
    rs[b] = (int)min(row, (long)a.rows);
    row += max(f, 0l);
    lacks += max(pages_lacking(a, cached(b), f, row), 0l);
  }
  if (tid == 0) rs[a.B] = (int)min(total, (long)a.rows);
  long page = block_scan<NT>(lacks, sums, total);
  row = r0;
  int taken = 0;       // by the last request that gets pages
  long long asked = 0;  // up to the last one that is not refused
  for (int b = b0; b < b1; b++) {
    const long c = cached(b), f = fresh(b);
    cs[b] = (int)c;
    row += max(f, 0l);
    const long need = pages_lacking(a, c, f, row);
    const bool granted = need == 0 || (need > 0 && page + need <= n_free);
    pg[b] = granted ? (int)min(page, n_free) : -1;
    if (granted && need) taken = (int)(page + need);
    if (granted) asked = page + need;
    if (blockIdx.x == 0) {
      a.row_start[b] = rs[b];
      a.kv_len[b] = granted ? (int)(c + f) : 0;
    }
    page += max(need, 0l);
  }
  if (blockIdx.x == 0 && taken) atomicMax(&taken_s, taken);
  if (blockIdx.x == 0 && asked) atomicMax(&asked_s, asked);
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    a.row_start[a.B] = rs[a.B];
    *a.balance = (int)max(n_free - asked_s, -2147483647ll);
    if (a.taken) *a.taken = taken_s;
  }

  // table entries: a warp per request
  const int warps = gridDim.x * (NT / 32), lane = tid & 31;
  for (int b = blockIdx.x * (NT / 32) + (tid >> 5); b < a.B; b += warps) {
    if (pg[b] < 0) continue;
    const int c = cs[b];
    const int have = (int)(((long)c + a.page - 1) >> a.page_shift);
    const int need = (int)(((long)c + a.fresh[b] + a.page - 1) >> a.page_shift) - have;
    for (int j = lane; j < need; j += 32) a.tables[b * a.ldt + have + j] = a.free_pages[n_free - 1 - pg[b] - j];
  }
  // rows: the request by bisection of the row offsets; a page that this call
  // hands out is read from the free list, not from the table
  for (long r = (long)blockIdx.x * NT + tid; r < a.rows; r += (long)gridDim.x * NT) {
    int64_t slot = -1;
    int pos = -1;
    if (r < rs[a.B]) {
      int lo = 0, hi = a.B;  // the last request whose first row is at or before r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (rs[mid] <= r) lo = mid;
        else hi = mid;
      }
      if (pg[lo] >= 0) {
        const int c = cs[lo];
        pos = c + (int)(r - rs[lo]);
        const int have = (int)(((long)c + a.page - 1) >> a.page_shift), at = pos >> a.page_shift;
        const int g = at < have ? a.tables[lo * a.ldt + at] : a.free_pages[n_free - 1 - pg[lo] - (at - have)];
        if (g >= 0) slot = ((int64_t)g << a.page_shift) + (pos & (a.page - 1));
      }
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
  }
}

// ------------------------------------------------------------ append

// 8 consecutive elements of a row
template <int XT, bool VEC>
__device__ __forceinline__ void load8(const void *x, long i, float (&f)[8]) {
  if constexpr (VEC && XT == TCB_F32) {
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
    const float4 lo = __ldcs(p), hi = __ldcs(p + 1);
    f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
  } else if constexpr (VEC) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + i));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint16_t b = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      f[e] = XT == TCB_BF16 ? tcb::bf16_to_f32(b) : tcb::half_exact(b);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = tcb::load_act(x, i + e, XT);
  }
}
// the same in the cache's type, each rounded once (not at all where the types are one)
template <int XT, bool VEC>
__device__ __forceinline__ uint4 load_cache8(const void *x, long i, int dtype) {
  if constexpr (VEC && XT != TCB_F32)
    if (XT == dtype) return __ldcs(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + i));
  float f[8];
  load8<XT, VEC>(x, i, f);
  uint32_t o[4];
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 8; e++) nan |= f[e] != f[e];
  if (!nan) {  // the conversions differ from the library's rounding in a NaN's payload alone
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (dtype == TCB_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
        o[e] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
        o[e] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    o[e] = dtype == TCB_BF16 ? tcb::f32_to_bf16(f[2 * e]) | (uint32_t)tcb::f32_to_bf16(f[2 * e + 1]) << 16
                             : tcb::f32_to_f16(f[2 * e]) | (uint32_t)tcb::f32_to_f16(f[2 * e + 1]) << 16;
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A thread keeps one place in the rows (8 elements of a head) and walks rows,
// kRows at a time: their slots, then their K and V, are asked for together
// (16-byte loads where the rows are 16-byte aligned; the cache always is).
// HBM-bound: T * KVH * hd * (x bytes + 2) * 2 bytes; 130 MB (16391 rows of 8
// heads of 128, bf16) in 24.6 us = 5300 GB/s, against 37.5 us with one row at a
// time and the place found by divisions.
constexpr int kAppendThreads = 256, kAppendRows = 4;
template <int XT, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(const tcb_kv_pages kv, int page_shift, int T, const void *k,
                                                              long ldk, const void *v, long ldv, const int64_t *slots,
                                                              int *derr) {
  tcb::mv::pdl_wait();
  tcb::mv::pdl_launch_dependents();
  const int per_head = kv.head_dim / 8, places = kv.n_kv_heads * per_head;
  const int across = min(places, kAppendThreads);  // threads along a row; the CTA's other threads take other rows
  const int c = blockIdx.y * across + threadIdx.x % across, sub = threadIdx.x / across, rows = kAppendThreads / across;
  if (c >= places || sub >= rows) return;
  const int h = c / per_head, d = (c - h * per_head) * 8;
  const long x0 = (long)h * kv.head_dim + d, dst0 = h * kv.head_stride + d;
  const int64_t n_slots = (int64_t)kv.n_pages << page_shift;
  const long step = (long)gridDim.x * rows;
  for (long r0 = (long)blockIdx.x * rows + sub; r0 < T; r0 += step * kAppendRows) {
    int64_t slot[kAppendRows];
    uint4 kx[kAppendRows], vx[kAppendRows];
#pragma unroll
    for (int i = 0; i < kAppendRows; i++) slot[i] = r0 + i * step < T ? slots[r0 + i * step] : -1;
#pragma unroll
    for (int i = 0; i < kAppendRows; i++)
      if (r0 + i * step < T) {
        kx[i] = load_cache8<XT, VEC>(k, (r0 + i * step) * ldk + x0, kv.dtype);
        vx[i] = load_cache8<XT, VEC>(v, (r0 + i * step) * ldv + x0, kv.dtype);
      }
#pragma unroll
    for (int i = 0; i < kAppendRows; i++) {
      if (slot[i] < 0) continue;
      if (slot[i] >= n_slots) {
        if (c == 0) atomicExch(derr, TCB_ERR_BOUNDS);
        continue;
      }
      const long dst = (slot[i] >> page_shift) * kv.page_stride + (slot[i] & (kv.page - 1)) * kv.pos_stride + dst0;
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(kv.k) + dst) = kx[i];
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(kv.v) + dst) = vx[i];
    }
  }
}

int check_pages(const tcb_kv_pages *kv) {
  if (!kv || !kv->k || !kv->v) return TCB_ERR_NULL;
  if (kv->dtype != TCB_F16 && kv->dtype != TCB_BF16) return TCB_ERR_DTYPE;
  if (!page_ok(kv->page) || kv->n_pages < 1 || kv->n_kv_heads < 1 || (kv->head_dim != 64 && kv->head_dim != 128))
    return TCB_ERR_SHAPE;
  if (kv->pos_stride < kv->head_dim || kv->head_stride < kv->head_dim || kv->page_stride < kv->head_dim)
    return TCB_ERR_SHAPE;
  if ((kv->pos_stride | kv->head_stride | kv->page_stride) % 8 || !aligned(kv->k, 16) || !aligned(kv->v, 16))
    return TCB_ERR_ALIGN;
  return TCB_OK;
}

// what tcb_page_attn and tcb_prefix_attn share
int check_attn(const tcb_kv_pages *kv, int B, int T, int H, const void *q, long ldq, const void *out, long ldo,
               const int *kv_len, const int *tables, int width, long ldt, int max_len, float scale) {
  int rc = check_pages(kv);
  if (rc != TCB_OK) return rc;
  if (B < 0 || T < 0 || H < 1 || H % kv->n_kv_heads || B > 65535 || width < 0 || max_len < 0) return TCB_ERR_SHAPE;
  if (!isfinite(scale)) return TCB_ERR_SHAPE;
  if (B == 0 || T == 0) return TCB_OK;
  if (ldq < (long)H * kv->head_dim || ldo < (long)H * kv->head_dim || (B > 1 && ldt < width)) return TCB_ERR_SHAPE;
  if (!q || !out || !kv_len || (width > 0 && !tables)) return TCB_ERR_NULL;
  if (!aligned(q, 16) || !aligned(out, 16) || ldq % 8 || ldo % 8) return TCB_ERR_ALIGN;
  if (!aligned(kv_len, 4) || !aligned(tables, 4)) return TCB_ERR_ALIGN;
  return TCB_OK;
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace

extern "C" {

int tcb_page_plan(tcb_ctx *ctx, int B, int page, const int *cached, const int *fresh, int *tables, int width,
                  long ldt, const int *free_pages, int free_cap, const int *n_free, int rows, int *row_start,
                  int *kv_len, int64_t *slots, int *positions, int *balance, int *taken,
                  void *stream) {
  if (!ctx) return TCB_ERR_NULL;
  if (B < 0 || !page_ok(page) || width < 0 || (B > 1 && ldt < width) || free_cap < 0 || rows < 0) return TCB_ERR_SHAPE;
  if (B > TCB_PAGE_PLAN_MAX) return TCB_ERR_TOO_LARGE;
  if (!row_start || !balance || !n_free || (B && (!cached || !fresh || !kv_len || (width && !tables))) ||
      (free_cap && !free_pages) || (rows && (!slots || !positions)))
    return TCB_ERR_NULL;
  for (const void *p : {(const void *)cached, (const void *)fresh, (const void *)tables, (const void *)free_pages,
                        (const void *)n_free, (const void *)row_start, (const void *)kv_len, (const void *)positions,
                        (const void *)balance, (const void *)taken})
    if (!aligned(p, 4)) return TCB_ERR_ALIGN;
  if (!aligned(slots, 8)) return TCB_ERR_ALIGN;
  // CTAs still read what others have read and CTA 0 or their neighbours write: no
  // output lies in an input, in the tables' rows or in another output
  const Span in[] = {{cached, 4l * B}, {fresh, 4l * B}, {free_pages, 4l * free_cap}, {n_free, 4}};
  const Span out[] = {{row_start, 4 * (B + 1l)}, {kv_len, 4l * B}, {slots, 8l * rows}, {positions, 4l * rows}, {balance, 4}, {taken, taken ? 4 : 0}};
  for (const Span &o : out) {
    for (const Span &i : in)
      if (meet(o, i)) return TCB_ERR_UNSUPPORTED;
    for (const Span *p = out; p != &o; p++)
      if (meet(o, *p)) return TCB_ERR_UNSUPPORTED;
    if (meets_rows(o, tables, B, 4l * width, 4 * ldt)) return TCB_ERR_UNSUPPORTED;
  }
  for (const Span &i : in)
    if (meets_rows(i, tables, B, 4l * width, 4 * ldt)) return TCB_ERR_UNSUPPORTED;
  int rc = tcb::ctx_bind(ctx);
  if (rc != TCB_OK) return rc;
  PlanArgs a{B, page, log2i(page), width, free_cap, rows, cached, fresh, tables, ldt, free_pages, n_free,
             row_start, kv_len, slots, positions, balance, taken};
  const size_t smem = (3 * (size_t)B + 1) * sizeof(int);
  // 128 threads while each has at most one request (3.4 us for 16 requests), else
  // 1024 (1024 requests with 110 thousand rows: 6.8 us, 8.2 with 256)
  auto go = [&](auto kernel, int nt, int most) {
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (3 * TCB_PAGE_PLAN_MAX + 1) * (int)sizeof(int));
      if (e != cudaSuccess) return e;
    }
    const long want = std::max<long>((rows + nt - 1) / nt, (B + nt / 32 - 1) / (nt / 32));
    return tcb::launch_serve(kernel, dim3((unsigned)std::min<long>(std::max<long>(want, 1), most)), nt, smem, 1,
                             static_cast<cudaStream_t>(stream), a);
  };
  const cudaError_t e = B <= 128 ? go(k_page_plan<128>, 128, 8 * ctx->sms) : go(k_page_plan<1024>, 1024, ctx->sms);
  return e == cudaSuccess ? TCB_OK : tcb::ctx_fail(ctx, e);
}

int tcb_kv_append(tcb_ctx *ctx, const tcb_kv_pages *kv, int T, const void *k, long ldk, const void *v, long ldv,
                  int xdtype, const int64_t *slots, void *stream) {
  if (!ctx) return TCB_ERR_NULL;
  int rc = check_pages(kv);
  if (rc != TCB_OK) return rc;
  if (xdtype != TCB_F32 && xdtype != TCB_F16 && xdtype != TCB_BF16) return TCB_ERR_DTYPE;
  if (T < 0) return TCB_ERR_SHAPE;
  if (T == 0) return TCB_OK;
  if (std::min(ldk, ldv) < (long)kv->n_kv_heads * kv->head_dim) return TCB_ERR_SHAPE;
  if (!k || !v || !slots) return TCB_ERR_NULL;
  const size_t xe = xdtype == TCB_F32 ? 4 : 2;
  if (!aligned(k, xe) || !aligned(v, xe) || !aligned(slots, 8)) return TCB_ERR_ALIGN;
  if ((rc = tcb::ctx_bind(ctx)) != TCB_OK) return rc;
  const bool vec = aligned(k, 16) && aligned(v, 16) && (ldk | ldv) * (long)xe % 16 == 0;
  const int places = kv->n_kv_heads * (kv->head_dim / 8), across = std::min(places, kAppendThreads);
  const long rows = kAppendThreads / across, waves = (T + rows - 1) / rows;
  const int most = 8 * ctx->sms;
  const dim3 grid((unsigned)std::min<long>(waves, most), (unsigned)((places + across - 1) / across));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sh = log2i(kv->page);
  auto go = [&](auto kernel) {
    return tcb::launch_serve(kernel, grid, kAppendThreads, 0, 1, s, *kv, sh, T, k, ldk, v, ldv, slots, ctx->derr);
  };
  cudaError_t e;
  if (xdtype == TCB_F32) e = vec ? go(k_kv_append<TCB_F32, true>) : go(k_kv_append<TCB_F32, false>);
  else if (xdtype == TCB_F16) e = vec ? go(k_kv_append<TCB_F16, true>) : go(k_kv_append<TCB_F16, false>);
  else e = vec ? go(k_kv_append<TCB_BF16, true>) : go(k_kv_append<TCB_BF16, false>);
  return e == cudaSuccess ? TCB_OK : tcb::ctx_fail(ctx, e);
}

int tcb_page_attn(tcb_ctx *ctx, const tcb_kv_pages *kv, int B, int T, int H, const void *q, long ldq, void *out,
                  long ldo, const int *row_start, const int *kv_len, const int *tables, int width, long ldt,
                  int max_rows, int max_len, float scale, int window, int sinks, void *stream) {
  if (!ctx) return TCB_ERR_NULL;
  int rc = check_attn(kv, B, T, H, q, ldq, out, ldo, kv_len, tables, width, ldt, max_len, scale);
  if (rc != TCB_OK) return rc;
  if (max_rows < 0 || sinks < 0) return TCB_ERR_SHAPE;
  if (B == 0 || T == 0 || max_rows == 0) return TCB_OK;
  if (!row_start) return TCB_ERR_NULL;
  if (!aligned(row_start, 4)) return TCB_ERR_ALIGN;
  if ((rc = tcb::ctx_bind(ctx)) != TCB_OK) return rc;
  tcb::PageAttnArgs a{*kv, log2i(kv->page), B, T, H, q, ldq, out, ldo, row_start, kv_len, tables, width, ldt,
                      nullptr, 0, std::min(max_rows, T), max_len, scale * kLog2e, window, sinks, ctx->derr};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Few rows over few positions go row by row too, each reading its positions
  // again (mostly from L2), where that is at most 20 MB: with 8 KV heads of 128,
  // row by row / by tiles in us: one request of 4 rows over 1024 positions 9.3 /
  // 15.5, of 8 rows 18.2 / 15.4; 4 requests of 2 rows over 256 8.3 / 11.8, over 1024
  // 18.4 / 15.5
  const double seen = window < 0 ? max_len : std::min<double>(max_len, (double)window + sinks);
  const double read = (double)B * a.max_rows * seen * kv->n_kv_heads * kv->head_dim * 4;
  if (a.max_rows == 1 || (read <= 20e6 && (long)B * a.max_rows <= 65535)) {
    const tcb::DecodePlan pl = tcb::page_decode_plan(a, false);
    if ((rc = tcb::ctx_scratch(ctx, pl.bytes)) != TCB_OK) return rc;
    return tcb::launch_page_decode(ctx, a, pl, ctx->sv.p, {}, s);
  }
  const tcb::RowsPlan pl = tcb::page_rows_plan(a);
  if ((rc = tcb::ctx_scratch(ctx, pl.bytes)) != TCB_OK) return rc;
  return tcb::launch_page_rows(ctx, a, pl, ctx->sv.p, s);
}

int tcb_prefix_attn(tcb_ctx *ctx, const tcb_kv_pages *kv, int B, int H, const void *q, long ldq, void *out, long ldo,
                    const int *prefix, int prefix_len, const int *kv_len, const int *tables, int width, long ldt,
                    int max_len, float scale, void *stream) {
  if (!ctx) return TCB_ERR_NULL;
  int rc = check_attn(kv, B, B, H, q, ldq, out, ldo, kv_len, tables, width, ldt, max_len, scale);
  if (rc != TCB_OK) return rc;
  if (prefix_len < 0) return TCB_ERR_SHAPE;
  if (B == 0) return TCB_OK;
  if (prefix_len && !prefix) return TCB_ERR_NULL;
  if (!aligned(prefix, 4)) return TCB_ERR_ALIGN;
  if ((rc = tcb::ctx_bind(ctx)) != TCB_OK) return rc;
  tcb::PageAttnArgs a{*kv, log2i(kv->page), B, B, H, q, ldq, out, ldo, nullptr, kv_len, tables, width, ldt,
                      prefix_len ? prefix : nullptr, prefix_len, 1, max_len, scale * kLog2e, -1, 0, ctx->derr};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // The prefix in a product of all requests' rows, or read by each request like
  // its own positions (mostly from L2): the first costs about 10 us and 1.2 ns
  // a position more, the second a quarter of a microsecond per MB.  With 8 KV
  // heads of 128 and 4 query heads each, apart / read by each, in us: 4 requests
  // behind 1024 positions 18.6 / 9.9, behind 4096 20.6 / 26.0; 16 behind 256 17.6 /
  // 10.3, behind 1024 18.5 / 23.9; 64 behind 256 26.7 / 25.1, behind 4096 33.9 / 146
  const double read = (double)B * prefix_len * kv->n_kv_heads * kv->head_dim * 4;
  const bool apart = read > 40e6 + 4800. * prefix_len;
  const tcb::DecodePlan dp = tcb::page_decode_plan(a, apart);
  tcb::RowsPlan rp{};
  if (apart) rp = tcb::page_rows_plan(a);
  const size_t at = (rp.bytes + 255) / 256 * 256;
  if ((rc = tcb::ctx_scratch(ctx, at + dp.bytes)) != TCB_OK) return rc;
  char *ws = static_cast<char *>(ctx->sv.p);
  tcb::PrefixPartials x{};
  if (apart) {
    if ((rc = tcb::launch_page_rows(ctx, a, rp, ws, s)) != TCB_OK) return rc;
    x = {rp.split, reinterpret_cast<const float *>(ws), reinterpret_cast<const float2 *>(ws + rp.o_bytes)};
  }
  return tcb::launch_page_decode(ctx, a, dp, ws + at, x, s);
}

}  // extern "C"
