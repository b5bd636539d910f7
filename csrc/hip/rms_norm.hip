// RMS norm of rows with the residual's addition, its backward pass, and a forward pass whose output is e4m3 with a scale a row.
//
//   h = x + res      rstd = 1 / sqrt(mean(h^2) + eps)      y = h rstd w                       (all in fp32, rounded where it is stored)
//   g = dy w         dx = dres = dh + rstd (g - h rstd^2 mean(g h))        dw = sum over rows of dy h rstd
//
// y comes from the sum as it stands in registers, not from the rounded h that is stored for the residual stream: one rounding each.
// The backward pass therefore adds x and res again instead of reading h: with bf16 rows dw from the rounded h would be 2e-3 off.
// The pass is bound by memory: a row is read once, kept in registers (a wave or a workgroup a row) and written once.  Measured: 16384 x 4096
// bf16 with residual 94 us (5.7 TB/s); 8192 x 2048 bf16 with residual 24.7 us forward (5.4 TB/s), 29.2 + 3.9 us backward (5.7 TB/s, and dw's sums).
// dw: every workgroup of the backward pass adds up its rows in registers and writes one row of partial sums; a second kernel adds
// those in a fixed order (no atomics: the same result on every run).
#include "common.h"
#include "rms_norm.h"
#include <algorithm>
#include <type_traits>

namespace {
constexpr int ERR = -22;
constexpr float E4M3_MAX = 448.f;
constexpr float TINY = 0x1p-100f;  // a row whose largest magnitude is below this is scaled as if it were this: 448 / max stays finite
}  // namespace

template <typename T, int VEC> struct Piece {  // VEC consecutive elements as loaded (T: float, or uint16_t for bf16)
  T e[VEC];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return e[i];
    else return bf2f(e[i]);
  }
  __device__ __forceinline__ void set(int i, float v) {
    if constexpr (sizeof(T) == 4) e[i] = v;
    else e[i] = f2bf(v);
  }
};
// (wide accesses whatever the address: rows of odd lengths start anywhere)
template <typename T, int VEC> __device__ __forceinline__ Piece<T, VEC> load_piece(const T* p) {
  Piece<T, VEC> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int VEC> __device__ __forceinline__ void store_piece(T* p, const Piece<T, VEC>& r) { __builtin_memcpy(p, &r, sizeof(r)); }
template <int VEC> __device__ __forceinline__ void load_w(const float* p, float* w) { __builtin_memcpy(w, p, VEC * sizeof(float)); }
// Piece number c of a row: the last one ends where the row ends and covers some elements of the one before again (the same values are
// computed and stored twice); `skip` says how many, so that sums count them once.  Numbers behind the last: that one again, all skipped.
template <int VEC> struct Place {
  int start, skip;
  bool in;
  __device__ __forceinline__ Place(int c, int dim) : start(min(c * VEC, dim - VEC)), skip(min(c * VEC - start, VEC)), in(c * VEC < dim) {}
};
// VEC floats as e4m3 (to nearest even)
template <int VEC> __device__ __forceinline__ void store_e4m3(uint8_t* p, const float* y) {
  if constexpr (VEC == 1) *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], 0.f, 0, false);
  else {
    uint32_t u[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      u[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      u[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], (int)u[i], true);
    }
    __builtin_memcpy(p, u, VEC);
  }
}

// sum (or largest bits) over the NT threads of a row; `slot`: NT / 64 floats of LDS that no other reduction in flight uses
template <int NT> __device__ __forceinline__ float row_sum(float v, float* slot) {
  v = wave_sum(v);
  if constexpr (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += slot[i];
  return s;
}
template <int NT> __device__ __forceinline__ uint32_t row_max(uint32_t v, float* slot) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  if constexpr (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) reinterpret_cast<uint32_t*>(slot)[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s = max(s, reinterpret_cast<uint32_t*>(slot)[i]);
  return s;
}
// The scale of a row of e4m3 and what its values are multiplied by, from the bits of its largest magnitude (an order in which NaN is
// the largest: a row that holds one gets a scale of NaN; a row of zeros the scale 0)
__device__ __forceinline__ void e4m3_scale(uint32_t bits, float& scale, float& inv) {
  const float m = __uint_as_float(bits), c = m < TINY ? TINY : m;
  scale = m == 0.f ? 0.f : c / E4M3_MAX;
  inv = E4M3_MAX / c;
}

// NT threads a row (a wave: four rows a workgroup; or the whole workgroup), IT pieces of VEC elements a thread
template <typename T, int VEC, int NT, int IT, bool RES, bool OUT8>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void rms_norm_fwd_kernel(const RmsNormArgs a) {
  constexpr int RPB = NT < 256 ? 256 / NT : 1;
  __shared__ float slots[2][NT < 256 ? 1 : NT / 64];
  const int t = threadIdx.x % NT;
  const long row = (long)blockIdx.x * RPB + threadIdx.x / NT;
  if (row >= a.rows) return;  // (whole waves; a workgroup a row has none)
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* res = static_cast<const T*>(a.res) + row * a.ld_res;
  Piece<T, VEC> px[IT], pr[IT];
  float w[IT][VEC];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const Place<VEC> at(k * NT + t, a.dim);
    px[k] = load_piece<T, VEC>(x + at.start);
    if constexpr (RES) pr[k] = load_piece<T, VEC>(res + at.start);
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) load_w<VEC>(a.w + Place<VEC>(k * NT + t, a.dim).start, w[k]);
  float v[IT][VEC], ss = 0.f;
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const Place<VEC> at(k * NT + t, a.dim);
    Piece<T, VEC> ph;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[k][i] = px[k].get(i);
      if constexpr (RES) v[k][i] += pr[k].get(i);
      ss += i >= at.skip ? v[k][i] * v[k][i] : 0.f;
      ph.set(i, v[k][i]);
    }
    if constexpr (RES)
      if (at.in) store_piece<T, VEC>(static_cast<T*>(a.h) + row * a.dim + at.start, ph);
  }
  const float rstd = 1.f / sqrtf(row_sum<NT>(ss, slots[0]) / (float)a.dim + a.eps);
  if (a.rstd && t == 0) a.rstd[row] = rstd;
  uint32_t big = 0;
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[k][i] = v[k][i] * rstd * w[k][i];
      if constexpr (OUT8) big = max(big, __float_as_uint(v[k][i]) & 0x7fffffffu);  // (repeated pieces change no maximum)
    }
  float scale = 0.f, inv = 0.f;
  if constexpr (OUT8) {
    e4m3_scale(row_max<NT>(big, slots[1]), scale, inv);
    if (t == 0) a.q_scale[row] = scale;
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const Place<VEC> place(k * NT + t, a.dim);
    if (!place.in) continue;
    const long at = row * a.dim + place.start;
    if constexpr (OUT8) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[k][i] *= inv;
      store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + at, v[k]);
    } else {
      Piece<T, VEC> p;
#pragma unroll
      for (int i = 0; i < VEC; ++i) p.set(i, v[k][i]);
      store_piece<T, VEC>(static_cast<T*>(a.y) + at, p);
    }
  }
}

// Rows that do not fit the registers of a workgroup (fp32 above 8192 values, bf16 above 16384): the row is read again (from the caches) for each of the two
// or three passes, one element a load.  2048 x 32768 bf16 with residual: forward 169 us (3.2 TB/s of what has to move), dx 337, dw 157 + 12.
template <typename T, bool RES, bool OUT8>
__global__ __launch_bounds__(1024) void rms_norm_fwd_long_kernel(const RmsNormArgs a) {
  __shared__ float slots[2][16];
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* res = static_cast<const T*>(a.res) + row * a.ld_res;
  auto at = [&](int c) {
    float v = load_piece<T, 1>(x + c).get(0);
    if constexpr (RES) v += load_piece<T, 1>(res + c).get(0);
    return v;
  };
  float ss = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float v = at(c);
    ss += v * v;
    if constexpr (RES) {
      Piece<T, 1> p;
      p.set(0, v);
      store_piece<T, 1>(static_cast<T*>(a.h) + row * a.dim + c, p);
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<1024>(ss, slots[0]) / (float)a.dim + a.eps);
  if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  float scale = 0.f, inv = 0.f;
  if constexpr (OUT8) {
    uint32_t big = 0;
    for (int c = threadIdx.x; c < a.dim; c += 1024) big = max(big, __float_as_uint(at(c) * rstd * a.w[c]) & 0x7fffffffu);
    e4m3_scale(row_max<1024>(big, slots[1]), scale, inv);
    if (threadIdx.x == 0) a.q_scale[row] = scale;
  }
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float y = at(c) * rstd * a.w[c], q = y * inv;
    if constexpr (OUT8) store_e4m3<1>(static_cast<uint8_t*>(a.y) + row * a.dim + c, &q);
    else {
      Piece<T, 1> p;
      p.set(0, y);
      store_piece<T, 1>(static_cast<T*>(a.y) + row * a.dim + c, p);
    }
  }
}

// 16 columns of dw from all rows: 256 threads = 16 columns x 16 sets of rows, then the sets' sums in order
template <typename T, bool RES> __device__ __forceinline__ void dw_columns(const RmsNormArgs& a, int c0, float (*sums)[17]) {
  const int c = c0 + (threadIdx.x & 15), set = threadIdx.x >> 4, cc = min(c, a.dim - 1);
  float s = 0.f;
#pragma unroll 8
  for (long row = set; row < a.rows; row += 16) {
    float h = load_piece<T, 1>(static_cast<const T*>(a.x) + row * a.ld_x + cc).get(0);
    if constexpr (RES) h += load_piece<T, 1>(static_cast<const T*>(a.res) + row * a.ld_res + cc).get(0);
    s += load_piece<T, 1>(static_cast<const T*>(a.dy) + row * a.ld_dy + cc).get(0) * (h * a.rstd[row]);
  }
  sums[set][threadIdx.x & 15] = s;
  __syncthreads();
  if (set || c >= a.dim) return;
  for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x & 15];
  a.dw[c] = s;
}

// Every workgroup takes rows blockIdx, blockIdx + gridDim, ... (four at a time with a wave a row); w and the sums of dw stay in registers.
// SPLIT, for few rows: dw does not wait for the rows' sums, so that further workgroups of the same launch take it, 16 columns each, and
// no partial sums go through memory.
template <typename T, int VEC, int NT, int IT, bool RES, bool DH, bool SPLIT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void rms_norm_bwd_kernel(const RmsNormArgs a) {
  constexpr int RPB = NT < 256 ? 256 / NT : 1;
  __shared__ float slots[2][NT < 256 ? 1 : NT / 64];
  __shared__ __attribute__((aligned(16))) float sums[NT < 256 ? IT * NT * VEC : 1];
  if constexpr (SPLIT) {
    __shared__ float sets[16][17];
    const int rows_wg = (int)((a.rows + RPB - 1) / RPB);
    if ((int)blockIdx.x >= rows_wg) return dw_columns<T, RES>(a, ((int)blockIdx.x - rows_wg) * 16, sets);
  }
  const int t = threadIdx.x % NT, group = threadIdx.x / NT;
  const float over = 1.f / (float)a.dim;
  float w[IT][VEC], acc[IT][VEC];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    load_w<VEC>(a.w + Place<VEC>(k * NT + t, a.dim).start, w[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[k][i] = 0.f;
  }
  int parity = 0;
  for (long row = (long)blockIdx.x * RPB + group; row < a.rows; row += SPLIT ? a.rows : (long)gridDim.x * RPB) {
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* res = static_cast<const T*>(a.res) + row * a.ld_res;
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const T* dh = static_cast<const T*>(a.dh) + row * a.ld_dh;
    Piece<T, VEC> px[IT], pr[IT], pd[IT], pg[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int start = Place<VEC>(k * NT + t, a.dim).start;
      px[k] = load_piece<T, VEC>(x + start);
      if constexpr (RES) pr[k] = load_piece<T, VEC>(res + start);
      pd[k] = load_piece<T, VEC>(dy + start);
      if constexpr (DH) pg[k] = load_piece<T, VEC>(dh + start);
    }
    const float rstd = a.rstd[row];
    float dot = 0.f, n[IT][VEC];  // n = h rstd
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int skip = Place<VEC>(k * NT + t, a.dim).skip;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = pd[k].get(i);
        n[k][i] = px[k].get(i);
        if constexpr (RES) n[k][i] += pr[k].get(i);
        n[k][i] *= rstd;
        if constexpr (!SPLIT) acc[k][i] += d * n[k][i];
        dot += i >= skip ? d * w[k][i] * n[k][i] : 0.f;
      }
    }
    const float mean = row_sum<NT>(dot, slots[parity]) * over;  // (two sets of slots: one barrier a row)
    parity ^= 1;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const Place<VEC> at(k * NT + t, a.dim);
      if (!at.in) continue;
      Piece<T, VEC> p;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float v = rstd * (pd[k].get(i) * w[k][i] - n[k][i] * mean);
        if constexpr (DH) v += pg[k].get(i);
        p.set(i, v);
      }
      store_piece<T, VEC>(static_cast<T*>(a.y) + row * a.dim + at.start, p);
    }
  }
  if (SPLIT || !a.part) return;
  if constexpr (NT < 256) {  // the four waves' sums, in the waves' order
    for (int g = 0; g < RPB; ++g) {
      if (group == g)
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float* s = &sums[(k * VEC + i) * NT + t];
            acc[k][i] = g ? *s + acc[k][i] : acc[k][i];
            *s = acc[k][i];
          }
      __syncthreads();
    }
    if (group != RPB - 1) return;
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const Place<VEC> at(k * NT + t, a.dim);
    if (at.in) __builtin_memcpy(a.part + (long)blockIdx.x * a.dim + at.start, acc[k], VEC * sizeof(float));
  }
}

template <typename T> __device__ __forceinline__ float h_at(const RmsNormArgs& a, long row, int c) {
  float v = load_piece<T, 1>(static_cast<const T*>(a.x) + row * a.ld_x + c).get(0);
  if (a.res) v += load_piece<T, 1>(static_cast<const T*>(a.res) + row * a.ld_res + c).get(0);
  return v;
}
template <typename T> __global__ __launch_bounds__(1024) void rms_norm_bwd_long_kernel(const RmsNormArgs a, long first) {
  __shared__ float slots[16];
  const long row = first + blockIdx.x;
  const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
  const T* dh = static_cast<const T*>(a.dh) + row * a.ld_dh;
  const float rstd = a.rstd[row];
  float dot = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += 1024) dot += load_piece<T, 1>(dy + c).get(0) * a.w[c] * (h_at<T>(a, row, c) * rstd);
  const float mean = row_sum<1024>(dot, slots) / (float)a.dim;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    float v = rstd * (load_piece<T, 1>(dy + c).get(0) * a.w[c] - h_at<T>(a, row, c) * rstd * mean);
    if (a.dh) v += load_piece<T, 1>(dh + c).get(0);
    Piece<T, 1> p;
    p.set(0, v);
    store_piece<T, 1>(static_cast<T*>(a.y) + row * a.dim + c, p);
  }
}
// the long rows' partial sums of dw: workgroup (column block, slice of the rows)
template <typename T> __global__ __launch_bounds__(256) void rms_norm_dw_long_kernel(const RmsNormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float s = 0.f;
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y)
    s += load_piece<T, 1>(static_cast<const T*>(a.dy) + row * a.ld_dy + c).get(0) * (h_at<T>(a, row, c) * a.rstd[row]);
  a.part[(long)blockIdx.y * a.dim + c] = s;
}

// dw: 64 columns a workgroup, 16 waves that take every sixteenth row of partial sums; then the waves' sums in order
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* __restrict__ part, float* __restrict__ dw, int blocks, int dim, int first) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = first + blockIdx.x * 64 + lane, cc = min(c, dim - 1);
  float s = 0.f;
#pragma unroll 8
  for (int b = wave; b < blocks; b += 16) s += part[(long)b * dim + cc];
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || c >= dim) return;
  for (int i = 1; i < 16; ++i) s += sums[i][lane];
  dw[c] = s;
}

namespace {
template <int VEC_, int NT_, int IT_> struct Shape { static constexpr int VEC = VEC_, NT = NT_, IT = IT_; };

// The threads of a row and the pieces of a thread (16 bytes: 4 floats or 8 bf16 values), so that a thread holds at most 32 elements: a
// wave a row while that is enough (no barrier, four rows a workgroup), then 256 or 1024 threads.  `few`: rows that leave most of the chip
// idle take 256 threads at once.  Rows shorter than a piece go element by element.  False: the row does not fit.
template <int VEC, typename F> bool with_shape(int dim, bool few, F f) {
  const int pieces = (dim + VEC - 1) / VEC;
  if (dim < VEC) f(Shape<1, 64, 1>{});
  else if (pieces <= 64) f(Shape<VEC, 64, 1>{});
  else if (few && pieces <= 256) f(Shape<VEC, 256, 1>{});
  else if (pieces <= 128) f(Shape<VEC, 64, 2>{});
  else if (pieces <= 256) f(Shape<VEC, 64, 4>{});
  else if (pieces <= 512) f(Shape<VEC, 256, 2>{});
  else if (pieces <= 1024) f(Shape<VEC, 256, 4>{});
  else if (pieces <= 2048) f(Shape<VEC, 1024, 2>{});
  else return false;
  return true;
}
template <typename F> bool with_type(const RmsNormArgs& a, F f) {
  const bool few = a.rows <= 1024;
  if (a.bf16) return with_shape<8>(a.dim, few, [&](auto s) { f(uint16_t{}, s); });
  return with_shape<4>(a.dim, few, [&](auto s) { f(float{}, s); });
}
constexpr long MOST = 1L << 21;  // workgroups of a launch: its threads have to be fewer than 2^32 (more are cut off without an error)
bool bad(const RmsNormArgs* a) {
  return !a || !a->x || !a->w || !a->y || a->rows <= 0 || a->dim <= 0 || a->rows > 0x7fffffffL || a->ld_x < 0 || a->ld_res < 0 || a->ld_dy < 0 || a->ld_dh < 0;
}
}  // namespace

static void fwd_rows(const RmsNormArgs& a, hipStream_t st) {
  const bool done = with_type(a, [&](auto type, auto s) {
    using T = decltype(type);
    using S = decltype(s);
    constexpr int RPB = S::NT < 256 ? 256 / S::NT : 1, BT = S::NT < 256 ? 256 : S::NT;
    const dim3 grid((unsigned)((a.rows + RPB - 1) / RPB));
    if (a.res) {
      if (a.q_scale) hipLaunchKernelGGL((rms_norm_fwd_kernel<T, S::VEC, S::NT, S::IT, true, true>), grid, dim3(BT), 0, st, a);
      else hipLaunchKernelGGL((rms_norm_fwd_kernel<T, S::VEC, S::NT, S::IT, true, false>), grid, dim3(BT), 0, st, a);
    } else {
      if (a.q_scale) hipLaunchKernelGGL((rms_norm_fwd_kernel<T, S::VEC, S::NT, S::IT, false, true>), grid, dim3(BT), 0, st, a);
      else hipLaunchKernelGGL((rms_norm_fwd_kernel<T, S::VEC, S::NT, S::IT, false, false>), grid, dim3(BT), 0, st, a);
    }
  });
  if (!done) {
    auto go = [&](auto type) {
      using T = decltype(type);
      const dim3 grid((unsigned)a.rows);
      if (a.res) {
        if (a.q_scale) hipLaunchKernelGGL((rms_norm_fwd_long_kernel<T, true, true>), grid, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((rms_norm_fwd_long_kernel<T, true, false>), grid, dim3(1024), 0, st, a);
      } else {
        if (a.q_scale) hipLaunchKernelGGL((rms_norm_fwd_long_kernel<T, false, true>), grid, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((rms_norm_fwd_long_kernel<T, false, false>), grid, dim3(1024), 0, st, a);
      }
    };
    if (a.bf16) go(uint16_t{}); else go(float{});
  }
}

DTF_API int dtf_rms_norm_fwd(const RmsNormArgs* p, hipStream_t st) {
  if (bad(p) || (p->res && !p->h)) return ERR;
  const long size = p->bf16 ? 2 : 4;
  const auto skip = [](auto* q, long bytes) { return q ? (decltype(q))((uintptr_t)q + bytes) : q; };
  for (long r = 0; r < p->rows; r += MOST) {
    RmsNormArgs a = *p;
    a.rows = p->rows - r < MOST ? p->rows - r : MOST;
    a.x = skip(a.x, r * a.ld_x * size);
    a.res = skip(a.res, r * a.ld_res * size);
    a.h = skip(a.h, r * a.dim * size);
    a.y = skip(a.y, r * a.dim * (a.q_scale ? 1 : size));
    a.rstd = skip(a.rstd, r * 4);
    a.q_scale = skip(a.q_scale, r * 4);
    fwd_rows(a, st);
    DTF_CHECK_LAUNCH();
  }
  return 0;
}

// How many rows of partial sums `part` the backward pass of these sizes writes; 0: none (dw in the same launch as dx).
// One kernel / two, us of both: 100 x 1024 fp32 2.9 / 7.2, 512 x 1024 fp32 5.1 / 7.8, 512 x 2048 bf16 6.0 / 9.8, 1000 x 2048 bf16 10.0 / 9.8 (x and dy
// are read twice, and a thread takes a sixteenth of the rows).
DTF_API int dtf_rms_norm_bwd_blocks(long rows, int dim) {
  if (rows <= 0 || dim <= 0) return ERR;
  if (rows <= 512 && dim <= 4096) return 0;
  return (int)(rows < 512 ? rows : 512);
}

DTF_API int dtf_rms_norm_bwd(const RmsNormArgs* p, hipStream_t st) {
  if (bad(p) || !p->dy || !p->rstd || p->blocks != dtf_rms_norm_bwd_blocks(p->rows, p->dim) || (p->dw && p->blocks && !p->part)) return ERR;
  const RmsNormArgs a = *p;
  const bool done = with_type(a, [&](auto type, auto s) {
    using T = decltype(type);
    using S = decltype(s);
    const dim3 block(S::NT < 256 ? 256 : S::NT);
    auto go = [&](auto res, auto dh) {
      constexpr bool RES = decltype(res)::value, DH = decltype(dh)::value;
      if constexpr (S::NT <= 256)
        if (a.blocks == 0) {
          const long rows_wg = S::NT < 256 ? (a.rows + 256 / S::NT - 1) / (256 / S::NT) : a.rows;
          hipLaunchKernelGGL((rms_norm_bwd_kernel<T, S::VEC, S::NT, S::IT, RES, DH, true>), dim3((unsigned)rows_wg + (a.dw ? (a.dim + 15) / 16 : 0)),
                             block, 0, st, a);
          return;
        }
      hipLaunchKernelGGL((rms_norm_bwd_kernel<T, S::VEC, S::NT, S::IT, RES, DH, false>), dim3(a.blocks), block, 0, st, a);
    };
    if (a.res) {
      if (a.dh) go(std::true_type{}, std::true_type{}); else go(std::true_type{}, std::false_type{});
    } else {
      if (a.dh) go(std::false_type{}, std::true_type{}); else go(std::false_type{}, std::false_type{});
    }
  });
  if (!done) {
    auto go = [&](auto type) {
      using T = decltype(type);
      for (long r = 0; r < a.rows; r += MOST) hipLaunchKernelGGL((rms_norm_bwd_long_kernel<T>), dim3((unsigned)(a.rows - r < MOST ? a.rows - r : MOST)), dim3(1024), 0, st, a, r);
      if (a.part) hipLaunchKernelGGL((rms_norm_dw_long_kernel<T>), dim3(dtf_cdiv(a.dim, 256), a.blocks), dim3(256), 0, st, a);
    };
    if (a.bf16) go(uint16_t{}); else go(float{});
  }
  DTF_CHECK_LAUNCH();
  if (a.dw && a.blocks)
    for (long c = 0; c < a.dim; c += 64 * MOST)
      hipLaunchKernelGGL(rms_norm_dw_kernel, dim3((unsigned)((std::min(a.dim - c, 64 * MOST) + 63) / 64)), dim3(1024), 0, st, a.part, a.dw, a.blocks, a.dim, (int)c);
  DTF_CHECK_LAUNCH();
  return 0;
}
