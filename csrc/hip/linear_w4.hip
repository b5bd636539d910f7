// Products of a few rows with 4-bit weights:  y[m][n] = relu?( x_scale[m] * sum_k x[m][k] e2m1(code[k][n]) s[k/G][n] + bias[n] )
//
// For single rows and small batches the weights' bytes are what the product costs (half a byte each, and 2 / G for the scales), so they
// are laid out once as the matrix instruction wants them: a wave loads 16 outputs x 128 k as one contiguous KB.  Four
// v_mfma_f32_16x16x32_bf16 take it: A = the weights, turned into bf16 two at a time by v_cvt_scalef32_pk_bf16_fp4 (0, 0.5 .. 6 are exact),
// B = up to 16 rows of x.  With a single row 15 columns of B are idle, which costs nothing: the instruction is not what bounds the kernel,
// and unpacking to fp32 for vector FMAs would need three times the VALU work.  The group's scales are applied in fp32 to the
// accumulator of the group (G = 32, 64, 128: 1, 2, 4 instructions).
//
// x: bf16; e4m3 (exact in bf16) with a scale a row; or fp32, each row as three columns of B, x = hi + mid + lo in bf16 by cutting the
// mantissa (8 + 8 + 8 bits: the sum is exact), added up at the end: fp32 rows lose nothing to the matrix instruction's type.
//
// The waves of a workgroup split k (tile t goes to wave t mod waves, so that the workgroup streams contiguously) and add their partial
// results in LDS, in the waves' order.
#include "common.h"
#include "linear_w4.h"

namespace {
constexpr int ERR = -22;
}

template <int XT> struct XType { using T = float; static constexpr int P = 3; };  // P: columns of B a row takes
template <> struct XType<X_BF16> { using T = uint16_t; static constexpr int P = 1; };
template <> struct XType<X_E4M3> { using T = uint8_t; static constexpr int P = 1; };

__device__ __forceinline__ uint32_t word_of(float e) { return __float_as_uint(e); }
__device__ __forceinline__ uint32_t word_of(uint16_t e) { return e; }
__device__ __forceinline__ uint32_t word_of(uint8_t e) { return e; }
// eight consecutive k of a row as loaded
template <int XT> struct XRaw { uint32_t w[2 * sizeof(typename XType<XT>::T)]; };
template <int XT> __device__ __forceinline__ XRaw<XT> x_load(const typename XType<XT>::T* p) {
  XRaw<XT> r;
  __builtin_memcpy(&r, p, sizeof(r));  // (wide loads also where a row starts at an odd element)
  return r;
}
// the same where the row ends among or before them: zeros from there on, nothing behind the row is read
template <int XT> __device__ __forceinline__ XRaw<XT> x_load_end(const typename XType<XT>::T* row, int k, int K) {
  using T = typename XType<XT>::T;
  constexpr int PER = 4 / sizeof(T);  // elements a word
  XRaw<XT> r;
#pragma unroll
  for (int i = 0; i < (int)(2 * sizeof(T)); ++i) {
    r.w[i] = 0;
#pragma unroll
    for (int h = 0; h < PER; ++h) {
      const int at = k + i * PER + h;
      const T e = row[min(at, K - 1)];
      r.w[i] |= at < K ? word_of(e) << (8 * (int)sizeof(T) * h) : 0u;
    }
  }
  return r;
}
// as bf16; fp32: the part of x that column `plane` of the three takes
template <int XT> __device__ __forceinline__ bf16x8 x_bf16(const XRaw<XT>& r, int plane) {
  uint32_t u[4];
  if constexpr (XT == X_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = r.w[i];
  } else if constexpr (XT == X_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.w[i], 1.f, false));
      u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.w[i], 1.f, true));
    }
  } else {
    // the upper 16 bits are taken off as often as the plane's number says (masks instead of branches: the planes are a wave's lanes).
    // Both differences are exact.  Column 0 takes a NaN or an infinity as it is (the difference with 0 makes a NaN quiet, so that one
    // whose bits all lie in the lower half survives); infinity less itself, a NaN, is none of the others' business.
    const uint32_t once = plane >= 1 ? 0xffff0000u : 0u, twice = plane >= 2 ? 0xffff0000u : 0u;
    float part[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __uint_as_float(r.w[i]), y = x - __uint_as_float(r.w[i] & once);
      part[i] = y - __uint_as_float(__float_as_uint(y) & twice);
      part[i] = plane >= 1 && part[i] != part[i] ? 0.f : part[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (__float_as_uint(part[2 * i]) >> 16) | (__float_as_uint(part[2 * i + 1]) & 0xffff0000u);
  }
  return __builtin_bit_cast(bf16x8, make_uint4(u[0], u[1], u[2], u[3]));
}
__device__ __forceinline__ bf16x8 e2m1_bf16(uint32_t w) {  // eight codes, the low nibble of the low byte first
  return __builtin_bit_cast(bf16x8, make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0)),
                                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1)),
                                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2)),
                                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3))));
}

// v as the lane g of each four lanes holds it (NG: how many of the four hold different values)
template <int NG> __device__ __forceinline__ uint32_t from_lane_of_four(uint32_t v, int g) {
  if constexpr (NG == 1) return v;
  switch (g) {
    case 0: return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x00, 0xf, 0xf, true);
    case 1: return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x55, 0xf, 0xf, true);
    case 2: return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xaa, 0xf, 0xf, true);
    default: return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xff, 0xf, 0xf, true);
  }
}

// GJ: matrix instructions (32 k each) that share a scale; R: tiles of 16 outputs a wave
template <int XT, int GJ, int R> __global__ __launch_bounds__(512) void linear_w4_kernel(const LinearW4Args a) {
  using T = typename XType<XT>::T;
  constexpr int P = XType<XT>::P, MC = 16 / P, NG = 4 / GJ;
  extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][R][16 n][16 columns]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, kb = lane >> 4, col = lane & 15;
  const int nt_all = (a.N + 15) / 16, kt_all = (a.K + 127) / 128, nt0 = blockIdx.x * R, plane = col % P;
  const long m0 = (long)blockIdx.y * MC, mine = min(m0 + col / P, a.M - 1);  // (columns behind the last row repeat it: not stored)
  const T* row = static_cast<const T*>(a.x) + mine * a.ldx;
  const uint4* wq[R];
  const uint16_t* sc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long nt = min(nt0 + r, nt_all - 1);
    wq[r] = static_cast<const uint4*>(a.wq) + nt * kt_all * 64 + lane;
    sc[r] = a.scales + (nt * kt_all * NG + col % NG) * 16 + 4 * kb;  // (the tile's groups are shared out over each four lanes)
  }
  f32x4 acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Weights {
    uint4 w[R];
    uint2 s[R];
  };
  auto load = [&](Weights& t, int kt) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      t.w[r] = wq[r][(long)kt * 64];
      t.s[r] = *reinterpret_cast<const uint2*>(sc[r] + (long)kt * NG * 16);
    }
  };
  auto multiply = [&](const Weights& t, const XRaw<XT> (&x)[4]) {
    bf16x8 b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = x_bf16<XT>(x[j], plane);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = g * GJ; j < (g + 1) * GJ; ++j)
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e2m1_bf16(reinterpret_cast<const uint32_t*>(&t.w[r])[j]), b[j], d, 0, 0, 0);
        const uint2 q = make_uint2(from_lane_of_four<NG>(t.s[r].x, g), from_lane_of_four<NG>(t.s[r].y, g));
        const float s4[4] = {__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u)};
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][i] = fmaf(d[i], s4[i], acc[r][i]);
      }
  };
  // Whole tiles of k.  All loads of a tile are on their way before the first is waited for (left to itself the compiler puts each load of x
  // next to its use, a round trip to the caches each: 17 us instead of 9.5 for one row of 16384 by 2048 outputs).  Two tiles at a time
  // gained nothing further: eight to sixteen waves a CU hide the rest.
  const int whole = a.K / 128;
  for (int kt = wave; kt < whole; kt += waves) {
    Weights t;
    XRaw<XT> x[4];
    load(t, kt);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = x_load<XT>(row + kt * 128 + 32 * j + 8 * kb);
    __builtin_amdgcn_sched_barrier(0);
    multiply(t, x);
  }
  if (whole < kt_all && wave == whole % waves) {  // the rest of k
    Weights t;
    XRaw<XT> x[4];
    load(t, whole);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = x_load_end<XT>(row, whole * 128 + 32 * j + 8 * kb, a.K);
    multiply(t, x);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[((wave * R + r) * 16 + 4 * kb + i) * 16 + col] = acc[r][i];
  __syncthreads();
  for (int o = threadIdx.x; o < R * 16 * MC; o += blockDim.x) {
    const int n = o % (R * 16), mm = o / (R * 16);
    const long m = m0 + mm;
    const int out = nt0 * 16 + n;
    if (m >= a.M || out >= a.N) continue;
    float s = 0.f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int p = 0; p < P; ++p) s += part[(w * R * 16 + n) * 16 + mm * P + p];
    if (a.x_scale) s *= a.x_scale[m];
    if (a.bias) s += a.bias[out];
    if (a.relu) s = s < 0.f ? 0.f : s;  // (a NaN stays one)
    if (a.out_bf16) static_cast<uint16_t*>(a.y)[m * a.N + out] = f2bf(s);
    else static_cast<float*>(a.y)[m * a.N + out] = s;
  }
}

namespace {
template <int XT, int GJ, int R> void go(const LinearW4Args& a, int passes, hipStream_t st) {
  // eight waves split k (16 were as fast at best; 4 took 9 instead of 7 us where 65 workgroups share 25 tiles of k, and are even elsewhere)
  const int nt = (a.N + 15) / 16, kt = (a.K + 127) / 128, waves = kt < 8 ? kt : 8;
  hipLaunchKernelGGL((linear_w4_kernel<XT, GJ, R>), dim3((nt + R - 1) / R, passes), dim3(64 * waves), sizeof(float) * waves * R * 256, st, a);
}
// More rows than the columns of B hold (16; fp32 5) take a pass over the weights for each such set, side by side in one launch: several
// column tiles a wave were slower, because x is what a wave reads most (16 rows of bf16 are four times a tile's weights): 64 rows of bf16,
// 4096 x 16384: 30.6 us, with four column tiles a wave 35.5.  For the same reason the tiles of outputs a wave takes are as many as leave
// the chip filled.  Measured, us with 1 / 2 / 4 tiles, by tiles of outputs x passes (k 4096): 256 (2048 outputs, 32 rows bf16) 6.8 / 8.2 / 10.5;
// 512 (8192, 16 rows bf16) 11.2 / 8.6 / 10.7; 1024 (16384, 16 rows bf16) 19.5 / 13.4 / 11.3, (16384, 5 rows fp32) 20.2 / 14.1 / 13.0.
template <int XT, int GJ> void with_tiles(const LinearW4Args& a, hipStream_t st) {
  constexpr int MC = 16 / XType<XT>::P;
  const int passes = (int)((a.M + MC - 1) / MC);
  const long sets = (long)((a.N + 15) / 16) * passes;
  if (sets >= 1024) go<XT, GJ, 4>(a, passes, st);
  else if (sets >= 512) go<XT, GJ, 2>(a, passes, st);
  else go<XT, GJ, 1>(a, passes, st);
}
template <int XT> void with_group(const LinearW4Args& a, hipStream_t st) {
  if (a.group == 32) with_tiles<XT, 1>(a, st);
  else if (a.group == 64) with_tiles<XT, 2>(a, st);
  else with_tiles<XT, 4>(a, st);
}
}  // namespace

DTF_API int dtf_linear_w4(const LinearW4Args* p, hipStream_t st) {
  if (!p || !p->x || !p->wq || !p->scales || !p->y || p->M <= 0 || p->N <= 0 || p->K <= 0 || p->ldx < 0) return ERR;
  if ((p->group != 32 && p->group != 64 && p->group != 128) || p->xtype < 0 || p->xtype > 2) return ERR;
  if ((uintptr_t)p->wq % 16 || (uintptr_t)p->scales % 8 || p->M > 65535L * 5) return ERR;  // (grid.y: five rows and more each)
  if (p->xtype == X_F32) with_group<X_F32>(*p, st);
  else if (p->xtype == X_BF16) with_group<X_BF16>(*p, st);
  else with_group<X_E4M3>(*p, st);
  DTF_CHECK_LAUNCH();
  return 0;
}
