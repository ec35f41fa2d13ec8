// tcb_page.h - the paged cache as the serving kernels take it, and their
// host-side launchers (internal to libtcb).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/tcb.h"
#include "tcb_ctx.h"

namespace tcb {

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

// requests of one row (tcb_page_decode.cu)
int launch_page_decode(tcb_ctx *ctx, const PageAttnArgs &a, cudaStream_t s);
int launch_page_attn(tcb_ctx *ctx, const PageAttnArgs &a, cudaStream_t s);

}  // namespace tcb
