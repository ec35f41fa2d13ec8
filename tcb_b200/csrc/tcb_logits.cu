// tcb_logits.cu - penalties, biases and masks on logits and the pick of the
// first maximum (tcb_logits_penalize), in one pass over the logits.
//
// A CTA takes one tile of one row.  It counts the row's history in a table
// of the tile's tokens in shared memory (integer atomics: their order does
// not change a count), notes the last bias entry of each token, and then
// reads, changes and writes its logits once.  The largest value of a row is
// found as a 64-bit maximum of (value in an order-preserving form, ~token),
// so the order in which CTAs arrive does not change it and equal values go
// to the lowest token.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/tcb.h"
#include "tcb_common.cuh"
#include "tcb_ctx.h"

namespace {

using namespace tcb;

constexpr int kThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;  // the token is in the prompt

// the state of a row's pick between its CTAs; zero before and after a call
struct Pick {
  unsigned long long best;  // 0: nothing allowed so far
  unsigned long long arrived;
};

__device__ __forceinline__ unsigned long long pick_key(float x, int t) {
  const uint32_t u = f_bits(x + 0.f);  // -0 and +0 are equal
  return (unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xFFFFFFFFu - (uint32_t)t);
}

__global__ void __launch_bounds__(kThreads) k_penalize(const tcb_logits_args a, int tile, Pick *picks, int *derr) {
  extern __shared__ uint32_t sh[];
  uint32_t *count = sh;         // [tile] generated occurrences, kSeen
  uint32_t *entry = sh + tile;  // [tile] 1 + last bias entry, 0: none
  __shared__ unsigned long long best_s;
  const int b = blockIdx.y, t0 = blockIdx.x * tile, n = min(tile, a.V - t0), tid = threadIdx.x;
  for (int i = tid; i < n; i += kThreads) {
    count[i] = 0;
    entry[i] = 0;
  }
  if (tid == 0) best_s = 0;
  __syncthreads();
  if (a.history) {
    const int total = min(max(a.total_len[b], 0), a.hist_width);
    const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
    const int64_t *hist = a.history + b * a.ldh;
    for (int i = tid; i < total; i += kThreads) {
      const int64_t t = hist[i] - t0;
      if (t < 0 || t >= n) continue;
      if (i < prompt) atomicOr(count + t, kSeen);
      else atomicAdd(count + t, 1u);
    }
  }
  for (int i = tid; i < a.n_bias; i += kThreads) {
    const long t = (long)a.bias_ids[b * a.ldb + i] - t0;
    if (t >= 0 && t < n) atomicMax(entry + t, (uint32_t)i + 1);
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[b] : 1.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f, pres = a.presence ? a.presence[b] : 0.f;
  const uint32_t *mask = nullptr;
  if (a.mask) {
    const int m = a.mask_row ? a.mask_row[b] : b;
    if (m >= a.n_masks) {
      if (tid == 0) atomicExch(derr, TCB_ERR_BOUNDS);
    } else if (m >= 0) {
      mask = a.mask + m * a.ldm;
    }
  }
  unsigned long long best = 0;
  for (int i = tid; i < n; i += kThreads) {
    const int t = t0 + i;
    float x = load_out(a.logits, b * a.ld + t, a.dtype);
    const uint32_t c = count[i];
    if (c) {
      const float made = (float)(c & ~kSeen);
      x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (c & ~kSeen) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, made)), pres);
    }
    if (entry[i]) x = __fadd_rn(x, a.bias[b * a.ldb + entry[i] - 1]);
    if (mask && !(mask[t >> 5] >> (t & 31) & 1)) x = -INFINITY;
    store_out(a.out, b * a.ldo + t, a.odtype, x, false);
    if (x > -INFINITY) best = max(best, pick_key(x, t));
  }
  if (!a.token) return;
  if (best) atomicMax(&best_s, best);
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
  const int tile = 4096;
  const dim3 grid((a.V + tile - 1) / tile, a.B);
  k_penalize<<<grid, kThreads, 2 * tile * sizeof(uint32_t), static_cast<cudaStream_t>(stream)>>>(
      a, tile, static_cast<Pick *>(ctx->tick), ctx->derr);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TCB_OK : ctx_fail(ctx, e);
}
