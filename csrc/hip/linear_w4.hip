// Products of a few rows with 4-bit weights:  y[m][n] = relu?( x_scale[m] * sum_k x[m][k] e2m1(code[k][n]) s[k/G][n] + bias[n] )
//
// For single rows and small batches the weights' bytes are what the product costs (half a byte each, and 2 / G for the scales), so they
// are laid out once as the matrix instruction wants them: a wave loads 16 outputs x 128 k as one contiguous KB.  Four
// v_mfma_f32_16x16x32_bf16 take it: A = the weights, turned into bf16 two at a time by v_cvt_scalef32_pk_bf16_fp4 (0, 0.5 .. 6 are exact),
// B = 16 rows of x.  With a single row 15 columns of B are idle, which costs nothing: the instruction is not what bounds the kernel,
// and unpacking to fp32 for vector FMAs would need three times the VALU work.  The group's scales are applied in fp32 to the
// accumulator of the group (G = 32, 64, 128: 1, 2, 4 instructions).  16384 x 16384 take 28-29 us for 1 row (bf16, G = 64) and 16 (e4m3,
// G = 128): 4.9 TB/s of weights, where a large copy reaches 5.1.
//
// x: bf16; e4m3 (exact in bf16) with a scale a row; or fp32, each row as three columns of B, x = hi + mid + lo in bf16 by cutting the
// mantissa (8 + 8 + 8 bits: the sum is exact), added up at the end: fp32 rows lose nothing to the matrix instruction's type.
//
// The waves of a workgroup split k (tile t goes to wave t mod waves, so that the workgroup streams contiguously) and add their partial
// results in LDS, in the waves' order.
#include "common.h"
#include "linear_w4.h"
#include <algorithm>

namespace {
constexpr int ERR = -22;
}

template <int XT> struct XType { using T = float; static constexpr int P = 3; };  // P: columns of B a row takes
template <> struct XType<X_BF16> { using T = uint16_t; static constexpr int P = 1; };
template <> struct XType<X_E4M3> { using T = uint8_t; static constexpr int P = 1; };

__device__ __forceinline__ uint32_t word_of(float e) { return __float_as_uint(e); }
__device__ __forceinline__ uint32_t word_of(uint16_t e) { return e; }
__device__ __forceinline__ uint32_t word_of(uint8_t e) { return e; }
// 16 bytes of a row: 4, 8 or 16 elements
struct XPiece {
  uint32_t w[4];
};
// The piece at k of a row of K elements, zeros behind its end.  One that reaches over the end is loaded as the row's last 16 bytes and
// shifted into place; a row shorter than that goes element by element.
template <typename T> __device__ __forceinline__ XPiece last_piece(const T* row, int k, int K) {
  constexpr int E = 16 / sizeof(T), PER = 4 / sizeof(T);
  XPiece x;
  if (K >= E) {
    uint64_t h[2];
    __builtin_memcpy(h, row + min(k, K - E), 16);
    const int over = max(k - (K - E), 0) * 8 * (int)sizeof(T);  // bits to drop at the low end
    const uint64_t lo = over >= 64 ? h[1] >> (over & 63) : over ? h[0] >> over | h[1] << (64 - over) : h[0];
    const uint64_t hi = over >= 64 ? 0 : h[1] >> over;
    const bool in = k < K;
    x.w[0] = in ? (uint32_t)lo : 0u;
    x.w[1] = in ? (uint32_t)(lo >> 32) : 0u;
    x.w[2] = in ? (uint32_t)hi : 0u;
    x.w[3] = in ? (uint32_t)(hi >> 32) : 0u;
  } else {
    T e[E];
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = row[min(k + i, K - 1)];
    __builtin_amdgcn_sched_barrier(0);  // (all loads first)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const uint32_t v = k + i < K ? word_of(e[i]) << (8 * (int)sizeof(T) * (i % PER)) : 0u;
      x.w[i / PER] = i % PER ? x.w[i / PER] | v : v;
    }
  }
  return x;
}
// A tile of x (the rows of this pass x 128 k) goes through LDS: the wave loads it in one piece, 16 bytes a lane, turns it into bf16 and
// writes it as the columns of B; then every lane reads its parts of its column.  Loaded from memory in B's order, a lane's column at a time,
// few rows are read by up to 16 lanes each (and converted as often), and the load unit, not memory, is what bounds the kernel.
// PITCH: 16 columns' parts of 16 bytes fall into all 64 banks.
constexpr int PITCH = 128 + 8;
template <int XT, bool CHECKED> __device__ __forceinline__ void store_columns(uint16_t* tile, int row, int k, const XPiece& x, float& sum) {
  if constexpr (XT == X_BF16) {
    *reinterpret_cast<uint4*>(tile + row * PITCH + k) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
  } else if constexpr (XT == X_E4M3) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w[i], 1.f, false));
      u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w[i], 1.f, true));
    }
    uint4* to = reinterpret_cast<uint4*>(tile + row * PITCH + k);
    to[0] = make_uint4(u[0], u[1], u[2], u[3]);
    to[1] = make_uint4(u[4], u[5], u[6], u[7]);
  } else {
    // the upper 16 bits, those of the rest, and what is left: both differences are exact
    uint32_t part[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = __uint_as_float(x.w[i]);
      float rest = v - __uint_as_float(x.w[i] & 0xffff0000u);
      part[0][i] = x.w[i];
      if constexpr (CHECKED) {
        // the first column takes a NaN or an infinity (a NaN made quiet, so that one whose bits all lie in the lower half survives); infinity
        // less itself, a NaN, is none of the others' business
        part[0][i] |= v != v ? 0x00400000u : 0u;
        rest = rest == rest ? rest : 0.f;
      } else {
        sum += rest;  // (of finite values: finite)
      }
      part[1][i] = __float_as_uint(rest);
      part[2][i] = __float_as_uint(rest - __uint_as_float(part[1][i] & 0xffff0000u));
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<uint2*>(tile + (3 * row + p) * PITCH + k) =
          make_uint2(__builtin_amdgcn_perm(part[p][1], part[p][0], 0x07060302u), __builtin_amdgcn_perm(part[p][3], part[p][2], 0x07060302u));
  }
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

// GJ: matrix instructions (32 k each) that share a scale; R: tiles of 16 outputs a wave; C: tiles of 16 columns of B; PIECES: of x a lane,
// one for few rows
template <int XT, int GJ, int R, int C, int PIECES> __global__ __launch_bounds__(C > 1 ? 256 : R > 1 ? 512 : 768) void linear_w4_kernel(const LinearW4Args a) {
  using T = typename XType<XT>::T;
  constexpr int P = XType<XT>::P, MC = C * 16 / P, NG = 4 / GJ;
  constexpr int E = 16 / sizeof(T), PER_ROW = 128 / E;  // elements of a piece, pieces of a row
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // a tile of x for each wave; at the end [waves][R][16 n][C * 16 columns] sums
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, kb = lane >> 4, col = lane & 15;
  const int nt_all = (a.N + 15) / 16, kt_all = (a.K + 127) / 128, nt0 = blockIdx.x * R;
  const long m0 = (long)blockIdx.y * MC;
  const int rows = (int)min((long)MC, a.M - m0);  // of this pass
  const T* const x0 = static_cast<const T*>(a.x) + m0 * a.ldx;
  uint16_t* const tile = reinterpret_cast<uint16_t*>(lds) + wave * C * 16 * PITCH;
  const uint16_t* column[C];
#pragma unroll
  for (int c = 0; c < C; ++c) column[c] = tile + min(16 * c + col, rows * P - 1) * PITCH + 8 * kb;  // (columns behind the last repeat it: not stored)
  const uint4* wq[R];
  const uint16_t* sc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long nt = min(nt0 + r, nt_all - 1);
    wq[r] = static_cast<const uint4*>(a.wq) + nt * kt_all * 64 + lane;
    sc[r] = a.scales + (nt * kt_all * NG + col % NG) * 16 + 4 * kb;  // (the tile's groups are shared out over each four lanes)
  }
  f32x4 acc[R][C];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
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
  auto put = [&](const XPiece (&x)[PIECES]) {  // a tile of x into LDS
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * 64 + lane;
      store_columns<XT, false>(tile, min(c / PER_ROW, MC - 1), c % PER_ROW * E, x[i], sum);  // (rows behind the last hold it again)
    }
    if (XT == X_F32 && __any(sum != sum)) {  // a NaN or an infinity: once more
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int c = i * 64 + lane;
        store_columns<XT, true>(tile, min(c / PER_ROW, MC - 1), c % PER_ROW * E, x[i], sum);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (a wave's own tile: its LDS accesses are done in order)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  auto multiply = [&](const Weights& t) {  // with the tile of x that is in LDS
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bf16x8 b[GJ][C];
#pragma unroll
      for (int j = 0; j < GJ; ++j)
#pragma unroll
        for (int c = 0; c < C; ++c) b[j][c] = *reinterpret_cast<const bf16x8*>(column[c] + 32 * (g * GJ + j));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        f32x4 d[C];
#pragma unroll
        for (int c = 0; c < C; ++c) d[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GJ; ++j) {
          const bf16x8 w = e2m1_bf16(reinterpret_cast<const uint32_t*>(&t.w[r])[g * GJ + j]);
#pragma unroll
          for (int c = 0; c < C; ++c) d[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, b[j][c], d[c], 0, 0, 0);
        }
        const uint2 q = make_uint2(from_lane_of_four<NG>(t.s[r].x, g), from_lane_of_four<NG>(t.s[r].y, g));
        const float s4[4] = {__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u)};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][c][i] = fmaf(d[c][i], s4[i], acc[r][c][i]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  };
  // Whole tiles of k; the next tile's loads are on their way while one is multiplied.
  const int whole = a.K / 128;
  auto fetch = [&](XPiece (&x)[PIECES], int kt) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * 64 + lane;
      __builtin_memcpy(&x[i], x0 + min(c / PER_ROW, rows - 1) * a.ldx + kt * 128 + c % PER_ROW * E, 16);
    }
  };
  if (wave < whole) {
    Weights t, t2;
    XPiece x[PIECES];
    fetch(x, wave);
    load(t, wave);
    for (int kt = wave; kt < whole; kt += 2 * waves) {
      // (behind the end: this one again, not multiplied.  Without a branch, so that the compiler counts the loads that are still out and
      // waits for the older half alone: behind a branch it waits for all, 8.9 instead of 7.6 us for one row of 16384 by 2048 outputs)
      const int second = kt + waves < whole ? kt + waves : kt, third = kt + 2 * waves < whole ? kt + 2 * waves : kt;
      put(x);
      fetch(x, second);
      load(t2, second);
      __builtin_amdgcn_sched_barrier(0);
      multiply(t);
      if (second == kt) break;
      put(x);
      fetch(x, third);
      load(t, third);
      __builtin_amdgcn_sched_barrier(0);
      multiply(t2);
    }
  }
  if (whole < kt_all && wave == whole % waves) {  // the rest of k: zeros behind it, nothing behind a row's end is read
    Weights t;
    XPiece x[PIECES];
    load(t, whole);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * 64 + lane;
      x[i] = last_piece(x0 + min(c / PER_ROW, rows - 1) * a.ldx, whole * 128 + c % PER_ROW * E, a.K);
    }
    put(x);
    multiply(t);
  }
  __syncthreads();
  float* const part = reinterpret_cast<float*>(lds);
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
// Eight waves split k (4: 11.1 instead of 7.5 us for one row of 16384 by 2048 outputs), twelve where k is long and the CUs have one workgroup each
// at most (6.5; 15: 6.6; with 4096 k 3.5 instead of 3.4).  Four where each has more to do, and its registers and LDS are more (7: 17.7 instead
// of 15.6 us for 32 rows bf16, 4096 x 16384).  Fewer where a launch would have 2^32 threads (they are cut off without an error).
int pick_waves(long groups, long passes, int r, int c, int kt) {
  const int most = c > 1 ? 4 : r == 1 && kt >= 64 && groups * passes <= 256 ? 12 : 8;
  return (int)std::min<long>(std::min(kt, most), 0xffffffffL / (64 * groups));
}
template <int XT, int GJ, int R, int C> void go(const LinearW4Args& a, int passes, hipStream_t st) {
  constexpr int ROW = 128 * sizeof(typename XType<XT>::T), MC = C * 16 / XType<XT>::P, MOST = (MC * ROW + 1023) / 1024;  // bytes of a tile's row; KB of a tile
  const int nt = (a.N + 15) / 16, kt = (a.K + 127) / 128;
  const dim3 grid((nt + R - 1) / R, passes);
  const int waves = pick_waves(grid.x, passes, R, C, kt);
  static_assert(32 * PITCH >= R * 1024, "a wave's sums take the place of its tiles of x");
  const int lds = 32 * PITCH * C * waves;
  if constexpr (C == 1) {
    if (a.M * ROW <= 1024) {
      hipLaunchKernelGGL((linear_w4_kernel<XT, GJ, R, C, 1>), grid, dim3(64 * waves), lds, st, a);
      return;
    }
  }
  hipLaunchKernelGGL((linear_w4_kernel<XT, GJ, R, C, MOST>), grid, dim3(64 * waves), lds, st, a);
}
// How many tiles of outputs (R) and of 16 columns of B (C) a wave takes.  More of the first: a tile of x is loaded and turned less often; of
// the second: a tile of weights is loaded and unpacked less often.  Rows that the columns do not hold take another pass over the weights, side by
// side in one launch.  What decides is how the workgroups come out on the 256 CUs, so the time is estimated as
//   first[C][R] * (1 + more * (rounds - 1)),   rounds = workgroups / 256, upwards
// where first is what one round takes (us measured for k = 4096) and another one adds less, because two workgroups share a CU by then; less still
// for short k, where much of a workgroup's time is waiting at its ends.  Measured, us (chosen: *):
//   C = 1, R = 1 / 2 / 3 / 4     3 rows fp32, 5000 x 4160 (260 tiles of outputs)  8.8 / 8.5* / 9.8 / 11.7    1 row bf16, 16384 x 9600 (600)  17.0 / 19.5 / 14.9* / 17.2
//                                16 rows e4m3, 5000 x 12288 (768)  10.6 / 11.8 / 10.0* / 11.4                the same, 16384 x 16384  39.1 / 31.6 / - / 29.6*
//   C = 1, C = 2, R = 2 / 3 / 4  32 rows bf16, 4096 x 16384  17.5, 15.3* / 18.4 / 16.6                       10 rows fp32, 16384 x 16384  60.4, 59.9 / - / 46.4*
//   C = 1, C = 3, R = 2 / 3 / 4  16 rows fp32, 4096 x 8192  17.3, 14.2* / 16.5 / 20.2                        the same, 16384 x 16384  98, 66 / 71 / 59*
// Three column tiles help fp32 rows alone (48 rows bf16, 4096 x 8192: 13.0 instead of 13.8), four are slower than two for all but the largest.
// A tile of columns that would hold no row is never worth it, whatever the estimate says (1 row bf16, 4096 x 262144: 150 us with one, 105 without).
struct Tiles { int r, c, passes; };
Tiles pick_tiles(long rows, int outputs, int k, int xtype) {
  static const float first[3][4] = {{4.7f, 6.1f, 8.1f, 9.1f}, {0.f, 10.6f, 13.2f, 16.f}, {0.f, 13.6f, 16.3f, 19.7f}};
  static const float more1[4] = {.5f, .62f, .62f, 1.f};
  const int most_c = xtype == X_F32 ? 3 : 2, parts = xtype == X_F32 ? 3 : 1, size = xtype == X_F32 ? 4 : xtype == X_BF16 ? 2 : 1;
  const long nt = ((long)outputs + 15) / 16;
  const bool few = rows * 128 * size <= 1024;  // (x takes a wave one load a tile: 2 rows bf16, 2866 x 5194: 4.5 instead of 4.9 us)
  float least = 0.f;
  Tiles best{0, 0, 0};
  for (int c = 1; c <= most_c && (c == 1 || (c - 1) * 16 / parts < rows); ++c)  // (a further tile of columns only for rows that the ones before do not hold)
    for (int r = c == 1 ? 1 : 2; r <= 4; ++r) {  // (one tile of outputs with several of columns comes out best for next to nothing)
      const long held = c * 16 / parts, p = (rows + held - 1) / held, rounds = ((nt + r - 1) / r * p + 255) / 256;
      const float more = c == 1 && r == 1 && rounds == 2 && few ? .25f : c == 1 ? more1[r - 1] : k < 8192 ? .4f : .6f;
      const float t = first[c - 1][r - 1] * (1.f + more * (float)(rounds - 1));
      if (best.c == 0 || t < least) least = t, best = {r, c, (int)p};
    }
  return best;
}
template <int XT, int GJ> void with_tiles(const LinearW4Args& a, hipStream_t st) {
  const Tiles t = pick_tiles(a.M, a.N, a.K, XT);
  switch (4 * t.c + t.r - 5) {
    case 0: return go<XT, GJ, 1, 1>(a, t.passes, st);
    case 1: return go<XT, GJ, 2, 1>(a, t.passes, st);
    case 2: return go<XT, GJ, 3, 1>(a, t.passes, st);
    case 3: return go<XT, GJ, 4, 1>(a, t.passes, st);
    case 5: return go<XT, GJ, 2, 2>(a, t.passes, st);
    case 6: return go<XT, GJ, 3, 2>(a, t.passes, st);
    case 7: return go<XT, GJ, 4, 2>(a, t.passes, st);
  }
  if constexpr (XT == X_F32) {
    switch (4 * t.c + t.r - 5) {
      case 9: return go<XT, GJ, 2, 3>(a, t.passes, st);
      case 10: return go<XT, GJ, 3, 3>(a, t.passes, st);
      case 11: return go<XT, GJ, 4, 3>(a, t.passes, st);
    }
  }
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
  if ((uintptr_t)p->wq % 16 || (uintptr_t)p->scales % 8 || p->M > 65535L * 5 || p->K > 0x7fffff00 || p->N > 0x7fffff00)
    return ERR;  // (grid.y: five rows and more each; sums with a tile stay inside an int)
  if (p->xtype == X_F32) with_group<X_F32>(*p, st);
  else if (p->xtype == X_BF16) with_group<X_BF16>(*p, st);
  else with_group<X_E4M3>(*p, st);
  DTF_CHECK_LAUNCH();
  return 0;
}

// The tiles that a wave takes for these sizes: 16 * (tiles of 16 columns) + tiles of outputs
DTF_API int dtf_linear_w4_tiles(long rows, int outputs, int k, int xtype) {
  if (rows <= 0 || outputs <= 0 || k <= 0 || xtype < 0 || xtype > 2) return ERR;
  const Tiles t = pick_tiles(rows, outputs, k, xtype);
  return 16 * t.c + t.r;
}
// The waves of each of its workgroups
DTF_API int dtf_linear_w4_waves(long rows, int outputs, int k, int xtype) {
  if (rows <= 0 || outputs <= 0 || k <= 0 || xtype < 0 || xtype > 2) return ERR;
  const Tiles t = pick_tiles(rows, outputs, k, xtype);
  return pick_waves((((long)outputs + 15) / 16 + t.r - 1) / t.r, t.passes, t.r, t.c, (int)(((long)k + 127) / 128));
}
