// tcb_logits.cu - penalties, biases and masks on logits and the pick of the
// first maximum (tcb_logits_penalize), in one pass over the logits.
//
// A CTA takes one tile of one row, kPer tokens a thread, and asks for its
// logits, mask words and first history tokens at once.  It counts the history in
// a table of the tile's tokens in shared memory (integer atomics: their order
// does not change a count), notes the last bias entry of each token, changes the
// logits in registers and writes them once.  The largest value of a row is found
// as a 64-bit maximum of (value in an order-preserving form, ~token), so the
// order in which CTAs arrive does not change it and equal values go to the lowest
// token.
//
// Bound: the logits read and written once (HBM): 68 MB in 36 us for 64 rows of
// 128256 (f32, histories of up to 8192 tokens, biases and masks), 18 us without
// history, biases, masks and pick.  The rest is the counting (10 us), the masks
// and biases (4 each) and the pick; a row's tiles scan its whole history.
// Measured slower: the CTAs of a cluster sharing the scan through distributed
// shared memory (48 us), changing the touched tokens from a list with full warps
// (43), 8 tokens a thread (42).
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/tcb.h"
#include "tcb_common.cuh"
#include "tcb_ctx.h"
#include "tcb_mv_ptx.cuh"
#include "tcb_page.h"

namespace {

using namespace tcb;

constexpr int kPer = 16;                  // tokens of a thread, in groups of 4
constexpr int kMaxThreads = 512;
constexpr int kAhead = 2;                 // pairs of history tokens a thread has asked for
constexpr uint32_t kSeen = 0x80000000u;  // the token is in the prompt
// the state of a row's pick between its CTAs; zero before and after a call
struct Pick {
  unsigned long long best;  // 0: nothing allowed so far
  unsigned long long arrived;
};

// four elements from index i on; VEC: aligned to the four
template <int DT, bool VEC>
__device__ __forceinline__ float4 load4(const void *p, int i, int n) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (VEC) {
    if (n >= 4) {
      if constexpr (DT == TCB_F32) return __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i));
      const uint2 u = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i));
      auto f = [](uint32_t h) { return DT == TCB_BF16 ? bf16_to_f32((uint16_t)h) : half_exact(h & 0xFFFFu); };
      return make_float4(f(u.x), f(u.x >> 16), f(u.y), f(u.y >> 16));
    }
  }
  if (n > 0) v.x = load_act(p, i, DT);
  if (n > 1) v.y = load_act(p, i + 1, DT);
  if (n > 2) v.z = load_act(p, i + 2, DT);
  if (n > 3) v.w = load_act(p, i + 3, DT);
  return v;
}
template <int DT, bool VEC>
__device__ __forceinline__ void store4(void *p, int i, int n, const float (&v)[4]) {
  if constexpr (VEC) {
    if (n >= 4) {
      if constexpr (DT == TCB_F32) {
        __stcs(reinterpret_cast<float4 *>(static_cast<float *>(p) + i), make_float4(v[0], v[1], v[2], v[3]));
      } else {
        auto h = [](float f) { return (uint32_t)(DT == TCB_BF16 ? f32_to_bf16(f) : f32_to_f16(f)); };
        __stcs(reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i),
               make_uint2(h(v[0]) | h(v[1]) << 16, h(v[2]) | h(v[3]) << 16));
      }
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (e < n) store_out(p, i + e, DT, v[e], false);
}

template <int XT, int OT, bool VEC>
__global__ void __launch_bounds__(kMaxThreads, 2) k_penalize(const __grid_constant__ tcb_logits_args a, Pick *picks,
                                                             int *derr) {
  extern __shared__ __align__(16) uint32_t sh[];
  const int tid = threadIdx.x, nt = blockDim.x, tile = kPer * nt;
  uint32_t *count = sh;         // [tile] generated occurrences, kSeen
  uint32_t *entry = sh + tile;  // [tile] 1 + last bias entry, 0: none (only with biases)
  __shared__ unsigned long long best_s;
  const int b = blockIdx.y, t0 = blockIdx.x * tile, n = min(tile, a.V - t0);
  mv::pdl_wait();
  const bool counted = a.history, biased = a.n_bias > 0;

  const char *in_row = static_cast<const char *>(a.logits) + b * a.ld * (XT == TCB_F32 ? 4 : 2);
  char *out_row = static_cast<char *>(a.out) + b * a.ldo * (OT == TCB_F32 ? 4 : 2);

  // everything that is read first is asked for before anything is waited for
  float4 x[kPer / 4];
#pragma unroll
  for (int u = 0; u < kPer / 4; u++) {
    const int i = 4 * (u * nt + tid);
    x[u] = load4<XT, VEC>(in_row, t0 + i, n - i);
  }
  const int total = a.history ? min(max(a.total_len[b], 0), a.hist_width) : 0;
  const int prompt = a.history && a.prompt_len ? a.prompt_len[b] : 0;
  const int64_t *hist = a.history + b * a.ldh;
  const bool pairs = reinterpret_cast<uintptr_t>(hist) % 16 == 0;
  auto two = [&](int i) {
    longlong2 v = make_longlong2(-1, -1);
    if (pairs && i + 1 < total) return *reinterpret_cast<const longlong2 *>(hist + i);
    if (i < total) v.x = hist[i];
    if (i + 1 < total) v.y = hist[i + 1];
    return v;
  };
  longlong2 ids[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; k++) ids[k] = two(2 * (tid + k * nt));
  int bias_id = tid < a.n_bias ? a.bias_ids[b * a.ldb + tid] : -1;
  const uint32_t *mask = nullptr;
  if (a.mask) {
    const int m = a.mask_row ? a.mask_row[b] : b;
    if (m >= a.n_masks) {
      if (tid == 0) atomicExch(derr, TCB_ERR_BOUNDS);
    } else if (m >= 0) {
      mask = a.mask + m * a.ldm;
    }
  }
  uint32_t word[kPer / 4];
#pragma unroll
  for (int u = 0; u < kPer / 4; u++) {
    const int i = 4 * (u * nt + tid);
    const uint32_t in = (1u << min(max(n - i, 0), 4)) - 1u;  // tokens of the four that are in the row
    word[u] = mask && i < n ? mask[(t0 + i) >> 5] >> ((t0 + i) & 31) & in : in;
  }
  if (tid == 0) best_s = 0;
  for (int i = tid; i < (biased ? 2 : counted ? 1 : 0) * tile / 4; i += nt) reinterpret_cast<uint4 *>(sh)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  auto one = [&](int64_t id, int i) {
    const uint32_t t = (uint32_t)id - (uint32_t)t0;
    if ((uint64_t)id >> 32 || t >= (uint32_t)n) return;
    if (i < prompt) atomicOr(count + t, kSeen);
    else atomicAdd(count + t, 1u);
  };
  for (int i = 2 * tid; i < total; i += 2 * kAhead * nt) {
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const longlong2 v = ids[k];
      ids[k] = two(i + 2 * (k + kAhead) * nt);
      one(v.x, i + 2 * k * nt);
      one(v.y, i + 2 * k * nt + 1);
    }
  }
  for (int i = tid; i < a.n_bias; i += nt) {
    const uint32_t t = (uint32_t)bias_id - (uint32_t)t0;
    if (bias_id >= 0 && t < (uint32_t)n) atomicMax(entry + t, (uint32_t)i + 1);
    if (i + nt < a.n_bias) bias_id = a.bias_ids[b * a.ldb + i + nt];
  }
  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f, pres = a.presence ? a.presence[b] : 0.f;
  __syncthreads();
  float best = -INFINITY;
  int best_t = -1;  // a thread's tokens come in rising order: the first of equal values stays
#pragma unroll
  for (int u = 0; u < kPer / 4; u++) {
    const int i = 4 * (u * nt + tid);
    if (counted && i < n) {
      const uint4 c4 = *reinterpret_cast<const uint4 *>(count + i);
      uint32_t left = (c4.x != 0) | (c4.y != 0) << 1 | (c4.z != 0) << 2 | (c4.w != 0) << 3;
      while (left) {  // few tokens of a warp's 128 are in the history: one at a time, whichever of the four it is
        const int e = __ffs(left) - 1;
        left &= left - 1;
        const uint32_t c = e < 2 ? (e ? c4.y : c4.x) : e == 2 ? c4.z : c4.w, made = c & ~kSeen;
        float w = e < 2 ? (e ? x[u].y : x[u].x) : e == 2 ? x[u].z : x[u].w;
        w = w > 0.f ? __fdiv_rn(w, rep) : __fmul_rn(w, rep);
        if (made) w = __fsub_rn(__fsub_rn(w, __fmul_rn(freq, (float)made)), pres);
        x[u].x = e == 0 ? w : x[u].x;
        x[u].y = e == 1 ? w : x[u].y;
        x[u].z = e == 2 ? w : x[u].z;
        x[u].w = e == 3 ? w : x[u].w;
      }
    }
    if (biased && i < n) {
      const uint4 e4 = *reinterpret_cast<const uint4 *>(entry + i);
      const float *bias = a.bias + b * a.ldb - 1;
      if (e4.x) x[u].x = __fadd_rn(x[u].x, bias[e4.x]);
      if (e4.y) x[u].y = __fadd_rn(x[u].y, bias[e4.y]);
      if (e4.z) x[u].z = __fadd_rn(x[u].z, bias[e4.z]);
      if (e4.w) x[u].w = __fadd_rn(x[u].w, bias[e4.w]);
    }
    auto last = [&](float &v, int e) {
      if (!(word[u] >> e & 1)) v = -INFINITY;
      if (v > best) best = v, best_t = t0 + i + e;
    };
    last(x[u].x, 0);
    last(x[u].y, 1);
    last(x[u].z, 2);
    last(x[u].w, 3);
    const float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    store4<OT, VEC>(out_row, t0 + i, n - i, v);
  }
  mv::pdl_launch_dependents();  // here, not at the start: CTAs of the next kernel would wait in the room of this one's
  if (a.token) {
    // the warp's largest value (in its order-preserving form; -0 and +0 are equal), then its lowest token
    const uint32_t f = f_bits(best + 0.f), key = best_t < 0 ? 0u : f & 0x80000000u ? ~f : f | 0x80000000u;
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, key);
    const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, key == top ? (uint32_t)best_t : 0xFFFFFFFFu);
    if ((tid & 31) == 0 && top) atomicMax(&best_s, (unsigned long long)top << 32 | (0xFFFFFFFFu - low));
    __syncthreads();
    if (tid == 0) {
      Pick *p = picks + b;
      if (best_s) atomicMax(&p->best, best_s);
      __threadfence();
      if (atomicAdd(&p->arrived, 1ull) == gridDim.x - 1) {
        const unsigned long long k = atomicExch(&p->best, 0ull);
        p->arrived = 0;
        a.token[b] = k ? (int64_t)(0xFFFFFFFFu - (uint32_t)k) : -1;
      }
    }
  }
}

template <int XT, int OT>
cudaError_t launch(const tcb_logits_args &a, int threads, Pick *picks, int *derr, cudaStream_t s) {
  const int tile = kPer * threads, xe = XT == TCB_F32 ? 16 : 8, oe = OT == TCB_F32 ? 16 : 8;  // bytes of four
  const bool vec = reinterpret_cast<uintptr_t>(a.logits) % xe == 0 && reinterpret_cast<uintptr_t>(a.out) % oe == 0 &&
                   a.ld % 4 == 0 && a.ldo % 4 == 0;
  const dim3 grid((a.V + tile - 1) / tile, a.B);
  const size_t smem = (a.n_bias ? 2 : a.history ? 1 : 0) * tile * sizeof(uint32_t);
  auto go = [&](auto kernel) {
    // the attributes belong to the kernel on the current device: asked for with
    // every launch that needs them
    cudaError_t e = cudaSuccess;
    if (smem > 48 << 10) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMaxThreads * kPer * 4);
    if (e == cudaSuccess && smem) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    return e != cudaSuccess ? e : launch_serve(kernel, grid, threads, smem, 1, s, a, picks, derr);
  };
  return vec ? go(k_penalize<XT, OT, true>) : go(k_penalize<XT, OT, false>);
}

template <int XT>
cudaError_t launch_to(const tcb_logits_args &a, int threads, Pick *picks, int *derr, cudaStream_t s) {
  if (a.odtype == TCB_F32) return launch<XT, TCB_F32>(a, threads, picks, derr, s);
  if (a.odtype == TCB_F16) return launch<XT, TCB_F16>(a, threads, picks, derr, s);
  return launch<XT, TCB_BF16>(a, threads, picks, derr, s);
}

bool type_ok(int dt) { return dt == TCB_F32 || dt == TCB_F16 || dt == TCB_BF16; }
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

extern "C" int tcb_logits_penalize(tcb_ctx *ctx, const tcb_logits_args *p, void *stream) {
  if (!ctx || !p) return TCB_ERR_NULL;
  tcb_logits_args a = *p;
  if (!type_ok(a.dtype) || !type_ok(a.odtype)) return TCB_ERR_DTYPE;
  if (a.B < 0 || a.B > 65535 || a.V < 0 || a.n_bias < 0 || a.n_masks < 0 || a.hist_width < 0) return TCB_ERR_SHAPE;
  if (a.B == 0 || a.V == 0) return TCB_OK;
  if (!a.logits || !a.out) return TCB_ERR_NULL;
  if (a.ld < a.V || a.ldo < a.V) return TCB_ERR_SHAPE;
  const size_t xe = a.dtype == TCB_F32 ? 4 : 2, oe = a.odtype == TCB_F32 ? 4 : 2;
  if (a.logits == a.out && (a.dtype != a.odtype || a.ld != a.ldo)) return TCB_ERR_UNSUPPORTED;
  if (!aligned(a.logits, xe) || !aligned(a.out, oe) || !aligned(a.token, 8) || !aligned(a.history, 8) ||
      !aligned(a.prompt_len, 4) || !aligned(a.total_len, 4) || !aligned(a.repetition, 4) || !aligned(a.frequency, 4) ||
      !aligned(a.presence, 4) || !aligned(a.bias_ids, 4) || !aligned(a.bias, 4) || !aligned(a.mask, 4) ||
      !aligned(a.mask_row, 4))
    return TCB_ERR_ALIGN;
  if (a.history && (!a.total_len || (a.B > 1 && a.ldh < a.hist_width))) return a.total_len ? TCB_ERR_SHAPE : TCB_ERR_NULL;
  if (!a.bias_ids) a.n_bias = 0;
  if (a.n_bias && (!a.bias || (a.B > 1 && a.ldb < a.n_bias))) return a.bias ? TCB_ERR_SHAPE : TCB_ERR_NULL;
  if (a.mask && (a.n_masks < 1 || (a.n_masks > 1 && a.ldm < (a.V + 31) / 32))) return TCB_ERR_SHAPE;
  int rc = ctx_bind(ctx);
  if (rc != TCB_OK || (rc = ctx_tick(ctx, (size_t)a.B * sizeof(Pick))) != TCB_OK) return rc;
  // tiles as large as leave the GPU a CTA per SM: one sequence of 128256 logits
  // takes 5.5 us with 128 threads (63 CTAs), 64 of them with histories of up to 8192
  // tokens 37 us with 512, 39 with 256, 45 with 128 (the history is read once
  // per tile)
  int threads = 128;
  while (threads < kMaxThreads && (long)a.B * ((a.V + 2 * threads * kPer - 1) / (2 * threads * kPer)) >= 148) threads *= 2;
  Pick *picks = static_cast<Pick *>(ctx->tick.p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.dtype == TCB_F32   ? launch_to<TCB_F32>(a, threads, picks, ctx->derr, s)
                        : a.dtype == TCB_F16 ? launch_to<TCB_F16>(a, threads, picks, ctx->derr, s)
                                             : launch_to<TCB_BF16>(a, threads, picks, ctx->derr, s);
  return e == cudaSuccess ? TCB_OK : ctx_fail(ctx, e);
}
