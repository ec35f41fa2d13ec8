// tcb_ctx.h - the context behind the opaque tcb_ctx handle (internal).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include <mutex>

struct tcb_ctx {
  int dev = 0;
  int sms = 148;
  void *ws = nullptr;  // scratch owned by the context, grown on demand
  size_t ws_cap = 0;
  int *derr = nullptr;  // device error word (bounded waits that gave up)
  void *sk = nullptr;   // split-K scratch of the matvec kernels (zeroed; kernels leave it zeroed)
  size_t sk_cap = 0;
  void *hx = nullptr;   // tcb_qgemm_host: x staged on the device
  size_t hx_cap = 0;
  void *hc = nullptr;   // tcb_qgemm_host: c of a caller whose c the GPU cannot reach
  size_t hc_cap = 0;
  // the serving operators' scratch, and their arrival counters and pick words
  // (zeroed; launches leave them zeroed).  An outgrown buffer is kept until the
  // context goes: a captured graph may still name it (each is at least twice the
  // one before).
  struct Kept {
    void *p = nullptr;
    size_t cap = 0;
    void *old[64] = {nullptr};
    int n_old = 0;
  } sv, tick;
  std::mutex mu;
  char err[256] = {0};
};

// the context's helpers behind the C entry points (tcb_capi.cu)
namespace tcb {
int ctx_fail(tcb_ctx *ctx, cudaError_t e);        // record the error, TCB_ERR_CUDA
int ctx_bind(tcb_ctx *ctx);                       // make the context's device current
int ctx_scratch(tcb_ctx *ctx, size_t bytes);      // at least `bytes` of scratch in ctx->sv.p
int ctx_tick(tcb_ctx *ctx, size_t bytes);         // at least `bytes` of zeroed counters in ctx->tick.p
}  // namespace tcb
