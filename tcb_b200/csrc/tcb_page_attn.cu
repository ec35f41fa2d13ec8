// tcb_page_attn.cu - attention over the paged cache (tcb_page_attn,
// tcb_prefix_attn): one warp per (row, query head).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "tcb_common.cuh"
#include "tcb_page.h"

namespace tcb {
namespace pa {

__device__ __forceinline__ float elem(uint16_t b, int dt) { return dt == TCB_BF16 ? bf16_to_f32(b) : half_exact(b); }

// Lane l holds elements l, l + 32, .. of the head.  The warp walks the
// visible positions with the running maximum and sum of the softmax.
template <int HD>
__global__ void __launch_bounds__(128) k_page_attn_row(const PageAttnArgs a) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.y, b = blockIdx.z, i = blockIdx.x * 4 + (threadIdx.x >> 5);
  int r = b, n = 1;
  if (a.row_start) {
    const int r0 = min(max(a.row_start[b], 0), a.T), r1 = min(max(a.row_start[b + 1], r0), a.T);
    n = r1 - r0;
    r = r0 + i;
    if (n > a.max_rows && lane == 0) atomicExch(a.derr, TCB_ERR_BOUNDS);
  }
  if (i >= min(n, a.max_rows)) return;
  int len = a.kv_len[b];
  if (len < 0 || len > a.max_len || len > (long)a.width << a.page_shift) {
    if (lane == 0) atomicExch(a.derr, TCB_ERR_BOUNDS);
    len = 0;
  }
  const int p = len - n + i, dt = a.kv.dtype;
  const uint16_t *qp = static_cast<const uint16_t *>(a.q) + r * a.ldq + (long)h * HD;
  const uint16_t *kp = static_cast<const uint16_t *>(a.kv.k), *vp = static_cast<const uint16_t *>(a.kv.v);
  const long hoff = (long)(h / (a.H / a.kv.n_kv_heads)) * a.kv.head_stride;
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < N; e++) q[e] = elem(qp[lane + 32 * e], dt), o[e] = 0.f;
  const int lo = a.window < 0 ? 0 : max(0l, (long)p - a.window + 1);
  for (int j = min(a.sinks, lo) > 0 ? 0 : lo; j <= p; j++) {
    if (j < lo && j >= a.sinks) j = lo;
    if (j > p) break;
    const int at = j >> a.page_shift;
    const int g = j < a.prefix_len ? a.prefix[at] : a.tables[b * a.ldt + at];
    if (g < 0 || g >= a.kv.n_pages) {
      if (lane == 0) atomicExch(a.derr, TCB_ERR_BOUNDS);
      continue;
    }
    const long off = g * a.kv.page_stride + hoff + (j & (a.kv.page - 1)) * a.kv.pos_stride;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) s = fmaf(q[e], elem(kp[off + lane + 32 * e], dt), s);
    s = warp_sum(s) * a.scale_log2;
    // a NaN score makes the row NaN; an infinite one keeps the sums' rules
    const float top = s != s ? s : fmaxf(m, s);
    const float keep = m == top ? 1.f : exp2f(m - top);
    const float w = s == top ? 1.f : exp2f(s - top);
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < N; e++) o[e] = o[e] * keep + w * elem(vp[off + lane + 32 * e], dt);
    m = top;
  }
  uint16_t *op = static_cast<uint16_t *>(a.out) + r * a.ldo + (long)h * HD;
#pragma unroll
  for (int e = 0; e < N; e++) {
    const float x = l == 0.f ? 0.f : __fdiv_rn(o[e], l);
    op[lane + 32 * e] = dt == TCB_BF16 ? f32_to_bf16(x) : f32_to_f16(x);
  }
}

}  // namespace pa

int launch_page_attn(tcb_ctx *ctx, const PageAttnArgs &a, cudaStream_t s) {
  if (a.max_rows == 1 && a.row_start) return launch_page_decode(ctx, a, s);
  const dim3 grid((a.max_rows + 3) / 4, a.H, a.B);
  if (a.kv.head_dim == 64) pa::k_page_attn_row<64><<<grid, 128, 0, s>>>(a);
  else pa::k_page_attn_row<128><<<grid, 128, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TCB_OK : ctx_fail(ctx, e);
}

}  // namespace tcb
