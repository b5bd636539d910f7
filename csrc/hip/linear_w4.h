// What a product with 4-bit weights takes.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

enum { X_F32 = 0, X_BF16 = 1, X_E4M3 = 2 };  // LinearW4Args::xtype

struct LinearW4Args {
  const void* x;         // [M][ldx]
  const void* wq;        // [Nt][Kt][64][16] bytes, Nt = ceil(N / 16), Kt = ceil(K / 128)
  const uint16_t* scales;// bf16 [Nt][Kt * 128 / G][16]
  const float* bias;     // [N] or null
  const float* x_scale;  // [M] or null
  void* y;               // [M][N] fp32 or bf16
  long M, ldx;
  int N, K, group, xtype, relu, out_bf16;
};

extern "C" int dtf_linear_w4(const LinearW4Args* a, hipStream_t st);
extern "C" int dtf_linear_w4_tiles(long rows, int outputs, int k, int xtype);
extern "C" int dtf_linear_w4_waves(long rows, int outputs, int k, int xtype);
