// tcb_page.h - the paged cache as the serving kernels take it, and their
// host-side launchers (internal to libtcb).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/tcb.h"
#include "tcb_ctx.h"

namespace tcb {

// Launch of a serving kernel (clusters of `cluster` CTAs along x): its CTAs may
// be placed while the last kernel of the stream ends, so every one of them
// waits for that kernel (mv::pdl_wait) before it touches memory, and lets the
// next kernel do the same (mv::pdl_launch_dependents).  Between the small
// kernels of a step this hides most of a launch.
template <class... Params, class... Args>
inline cudaError_t launch_serve(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s,
                                const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// attention over the pages (tcb_page_attn, tcb_prefix_attn), arguments checked
struct PageAttnArgs {
  tcb_kv_pages kv;
  int page_shift;  // log2(kv.page)
  int B, T, H;
  const void *q;
  long ldq;
  void *out;
  long ldo;
  const int *row_start;  // nullptr: row b is request b (one row each)
  const int *kv_len;
  const int *tables;
  int width;
  long ldt;
  const int *prefix;  // pages of the shared prefix, nullptr without one
  int prefix_len;
  int max_rows, max_len;
  float scale_log2;  // scale * log2(e): softmax in powers of two
  int window, sinks;  // window < 0: none
  int *derr;
};

// Requests of many rows, and the shared prefix of a batch (a.prefix set: all
// T rows against its positions): tcb_page_rows.cu.  With more than one CTA
// along the positions, and for a prefix, the kernel leaves partial results
// in scratch: o[split][prows * H][head_dim] and, o_bytes on, (maximum, sum)
// pairs [split][prows * H], where prows is T, or B * max_rows (`each`) where that
// is less; a prefix's are joined by the kernel of its suffixes.
struct RowsPlan {
  int tiles, split;
  long items;   // pairs of query tiles that have CTAs (for each KV head and part)
  bool packed;  // counted over all requests
  bool partial;
  int prows;
  bool each;
  size_t o_bytes, bytes;
};
RowsPlan page_rows_plan(const PageAttnArgs &a);
int launch_page_rows(tcb_ctx *ctx, const PageAttnArgs &a, const RowsPlan &pl, void *scratch, cudaStream_t s);

// Row by row (tcb_page_decode.cu): every row reads the positions it sees.  With a.prefix set: its positions
// from those pages, the others from the tables; or, with `parts` > 0, the
// positions from a.prefix_len on (suffix), joined with partial results as above.
struct DecodePlan {
  int nt, units, split, warps;
  size_t o_bytes, bytes;  // scratch of the join across clusters
  size_t counters;        // bytes of zeroed counters
};
constexpr int kMaxPrefixParts = 64;
struct PrefixPartials {
  int parts;
  const float *o;
  const float2 *ml;
};
DecodePlan page_decode_plan(const PageAttnArgs &a, bool suffix);
int launch_page_decode(tcb_ctx *ctx, const PageAttnArgs &a, const DecodePlan &pl, void *scratch, const PrefixPartials &x,
                       cudaStream_t s);

}  // namespace tcb
