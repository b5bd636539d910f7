// What the RMS norm's launches take.
#pragma once
#include <hip/hip_runtime_api.h>

struct RmsNormArgs {
  const void* x;
  const void* res;    // or null
  const void* dy;     // backward only, as dh (or null: h has no gradient of its own)
  const void* dh;
  const float* w;
  void* y;            // output rows, contiguous: fp32 / bf16, or e4m3 where q_scale is given; backward: dx
  void* h;            // x + res (only with res)
  float* rstd;        // forward: written unless null
  float* q_scale;
  float* part;        // backward: [blocks][dim] partial sums of dw, or null
  float* dw;
  long rows, ld_x, ld_res, ld_dy, ld_dh;
  int dim, bf16;
  float eps;
  int blocks;         // backward: rows of `part` (dtf_rms_norm_bwd_blocks; 0: no `part`)
};

extern "C" int dtf_rms_norm_fwd(const RmsNormArgs* a, hipStream_t st);
extern "C" int dtf_rms_norm_bwd_blocks(long rows, int dim);
extern "C" int dtf_rms_norm_bwd(const RmsNormArgs* a, hipStream_t st);
