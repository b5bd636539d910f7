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

// eight consecutive k of a row as loaded
template <int XT> struct XRaw { typename XType<XT>::T e[8]; };
template <int XT, bool VEC> __device__ __forceinline__ XRaw<XT> x_load(const typename XType<XT>::T* row, int k, int K) {
  XRaw<XT> r;
  if constexpr (VEC) {  // (K % 8 == 0: eight of a kind.  Behind the end: the row's first eight, cleared by x_clear)
    const auto* p = row + (k < K ? k : 0);
    if constexpr (sizeof(r) == 8) *reinterpret_cast<uint2*>(&r) = *reinterpret_cast<const uint2*>(p);
    else
#pragma unroll
      for (int i = 0; i < (int)(sizeof(r) / 16); ++i) reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = row[min(k + i, K - 1)];
  }
  return r;
}
// as bf16, with zeros behind the row's end; fp32: the part of x that column `plane` of the three takes
template <int XT, bool VEC> __device__ __forceinline__ bf16x8 x_bf16(const XRaw<XT>& r, int k, int K, int plane) {
  uint32_t u[4];
  if constexpr (XT == X_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = reinterpret_cast<const uint32_t*>(&r)[i];
  } else if constexpr (XT == X_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(&r)[i];
      u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
      u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t part[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = r.e[2 * i + h];
        const uint32_t b = __float_as_uint(x), top = b & 0xffff0000u;
        const float rest = x - __uint_as_float(top);                    // exact: the low 16 bits of the mantissa
        const uint32_t mid = __float_as_uint(rest) & 0xffff0000u;
        const float low = rest - __uint_as_float(mid);
        const bool finite = (b & 0x7f800000u) != 0x7f800000u;           // an infinity goes into the first column alone
        // (a NaN whose bits all lie in the part that is cut off stays one)
        part[h] = plane == 0 ? (finite || (b & 0x7fffffffu) == 0x7f800000u ? top : top | 0x00400000u)
                             : !finite ? 0u : plane == 1 ? mid : __float_as_uint(low);
      }
      u[i] = (part[0] >> 16) | (part[1] & 0xffff0000u);
    }
  }
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = k < K ? u[i] : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (k + 2 * i < K ? u[i] & 0xffffu : 0u) | (k + 2 * i + 1 < K ? u[i] & 0xffff0000u : 0u);
  }
  return __builtin_bit_cast(bf16x8, make_uint4(u[0], u[1], u[2], u[3]));
}
__device__ __forceinline__ bf16x8 e2m1_bf16(uint32_t w) {  // eight codes, the low nibble of the low byte first
  return __builtin_bit_cast(bf16x8, make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0)),
                                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1)),
                                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2)),
                                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3))));
}

// GJ: matrix instructions (32 k each) that share a scale; R: tiles of 16 outputs a wave; C: tiles of 16 columns of B a wave
template <int XT, bool VEC, int GJ, int R, int C> __global__ __launch_bounds__(1024) void linear_w4_kernel(const LinearW4Args a) {
  using T = typename XType<XT>::T;
  constexpr int P = XType<XT>::P, MC = C * 16 / P, NG = 4 / GJ;
  extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][R][16 n][C * 16 columns]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, kb = lane >> 4, col = lane & 15;
  const int nt_all = (a.N + 15) / 16, kt_all = (a.K + 127) / 128, nt0 = blockIdx.x * R;
  const long m0 = (long)blockIdx.y * MC;
  const T* rows[C];
  int plane[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {  // (columns behind the last row repeat it: nothing of theirs is stored)
    const long m = m0 + (16 * c + col) / P;
    rows[c] = static_cast<const T*>(a.x) + (m < a.M ? m : a.M - 1) * a.ldx;
    plane[c] = (16 * c + col) % P;
  }
  const uint4* wq[R];
  const uint16_t* sc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long nt = min(nt0 + r, nt_all - 1);
    wq[r] = static_cast<const uint4*>(a.wq) + nt * kt_all * 64 + lane;
    sc[r] = a.scales + nt * kt_all * NG * 16 + 4 * kb;
  }
  f32x4 acc[R][C];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kt = wave; kt < kt_all; kt += waves) {
    uint4 w[R];
    uint2 s[R][NG];
    XRaw<XT> x[C][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      w[r] = wq[r][(long)kt * 64];
#pragma unroll
      for (int g = 0; g < NG; ++g) s[r][g] = *reinterpret_cast<const uint2*>(sc[r] + ((long)kt * NG + g) * 16);
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[c][j] = x_load<XT, VEC>(rows[c], kt * 128 + 32 * j + 8 * kb, a.K);
    bf16x8 b[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) b[c][j] = x_bf16<XT, VEC>(x[c][j], kt * 128 + 32 * j + 8 * kb, a.K, plane[c]);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 t[C];
#pragma unroll
        for (int c = 0; c < C; ++c) t[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = g * GJ; j < (g + 1) * GJ; ++j) {
          const bf16x8 wa = e2m1_bf16(reinterpret_cast<const uint32_t*>(&w[r])[j]);
#pragma unroll
          for (int c = 0; c < C; ++c) t[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa, b[c][j], t[c], 0, 0, 0);
        }
        const float s4[4] = {bf2f(s[r][g].x & 0xffffu), bf2f(s[r][g].x >> 16), bf2f(s[r][g].y & 0xffffu), bf2f(s[r][g].y >> 16)};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][c][i] = fmaf(t[c][i], s4[i], acc[r][c][i]);
      }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[((wave * R + r) * 16 + 4 * kb + i) * (C * 16) + 16 * c + col] = acc[r][c][i];
  __syncthreads();
  for (int o = threadIdx.x; o < R * 16 * MC; o += blockDim.x) {
    const int n = o % (R * 16), mm = o / (R * 16);
    const long m = m0 + mm;
    const int out = nt0 * 16 + n;
    if (m >= a.M || out >= a.N) continue;
    float s = 0.f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int p = 0; p < P; ++p) s += part[(w * R * 16 + n) * (C * 16) + mm * P + p];
    if (a.x_scale) s *= a.x_scale[m];
    if (a.bias) s += a.bias[out];
    if (a.relu) s = s < 0.f ? 0.f : s;  // (a NaN stays one)
    if (a.out_bf16) static_cast<uint16_t*>(a.y)[m * a.N + out] = f2bf(s);
    else static_cast<float*>(a.y)[m * a.N + out] = s;
  }
}

namespace {
template <int XT, bool VEC, int GJ, int R, int C> void go(const LinearW4Args& a, int waves, hipStream_t st) {
  constexpr int MC = C * 16 / XType<XT>::P;
  const int nt = (a.N + 15) / 16;
  hipLaunchKernelGGL((linear_w4_kernel<XT, VEC, GJ, R, C>), dim3((nt + R - 1) / R, (unsigned)((a.M + MC - 1) / MC)), dim3(64 * waves),
                     sizeof(float) * waves * R * 256 * C, st, a);
}
template <int XT, bool VEC, int GJ> void with_tiles(const LinearW4Args& a, hipStream_t st) {
  const long cols = a.M * XType<XT>::P;
  const int nt = (a.N + 15) / 16, kt = (a.K + 127) / 128;
  // waves of a workgroup: as many as there are k tiles, up to 16; 8 where the outputs alone fill the chip (256 CUs of 32 waves)
  const int most = nt >= 512 ? 8 : 16, waves = kt < most ? kt : most;
  // (fp32 rows hold more registers: at most two tiles of columns, one where elements are loaded one by one)
  if constexpr (XT != X_F32)
    if (cols > 32) return go<XT, VEC, GJ, 1, 4>(a, waves < 8 ? waves : 8, st);
  if constexpr (XT != X_F32 || VEC)
    if (cols > 16) return go<XT, VEC, GJ, 1, 2>(a, waves < 8 ? waves : 8, st);
  go<XT, VEC, GJ, 1, 1>(a, waves, st);
}
template <int XT, bool VEC> void with_group(const LinearW4Args& a, hipStream_t st) {
  if (a.group == 32) with_tiles<XT, VEC, 1>(a, st);
  else if (a.group == 64) with_tiles<XT, VEC, 2>(a, st);
  else with_tiles<XT, VEC, 4>(a, st);
}
template <int XT> void with_rows(const LinearW4Args& a, hipStream_t st) {
  constexpr int size = (int)sizeof(typename XType<XT>::T), piece = 8 * size < 16 ? 8 * size : 16;  // bytes of one load
  if (a.K % 8 == 0 && (uintptr_t)a.x % piece == 0 && a.ldx * size % piece == 0) with_group<XT, true>(a, st);
  else with_group<XT, false>(a, st);
}
}  // namespace

DTF_API int dtf_linear_w4(const LinearW4Args* p, hipStream_t st) {
  if (!p || !p->x || !p->wq || !p->scales || !p->y || p->M <= 0 || p->N <= 0 || p->K <= 0 || p->ldx < 0) return ERR;
  if ((p->group != 32 && p->group != 64 && p->group != 128) || p->xtype < 0 || p->xtype > 2) return ERR;
  if ((uintptr_t)p->wq % 16 || (uintptr_t)p->scales % 8 || p->M > 65535L * 5) return ERR;  // (grid.y: five rows and more each)
  if (p->xtype == X_F32) with_rows<X_F32>(*p, st);
  else if (p->xtype == X_BF16) with_rows<X_BF16>(*p, st);
  else with_rows<X_E4M3>(*p, st);
  DTF_CHECK_LAUNCH();
  return 0;
}
