// AdamW over many separate tensors in one launch, moments held in 32 or in 8 bits (optim/adamw.py).
//
//   m = b1 m + (1-b1) g          p = p (1 - lr wd) - lr/(1-b1^t) * m / (sqrt(v)/sqrt(1-b2^t) + eps)
//   v = b2 v + (1-b2) g^2
//
// A step streams p, g and the moments once: 28 bytes an element (fp32, 32-bit moments) down to 10 (bf16, 8-bit moments).  The
// parameters and gradients are wherever the program put them; the moments lie in arenas in which every tensor starts at a multiple
// of 256 elements.  Two kernels a step (`begin` once for every 200 tensors, `apply` once for every pair of parameter and gradient types in use): `begin` takes the pointers by value (a captured graph keeps them, and nothing is kept by an
// address from one call to the next), advances every tensor's step counter and works out its bias corrections; `apply` runs over a
// fixed list of 2048-element chunks of all tensors.
//
// Measured: 190 tensors of 24 M fp32 elements, 8-bit moments, 72 us (5.3 TB/s); 64 of 268 M bf16 elements 494-545 us (5.0-5.5 TB/s), where about
// 65 issue slots an element keep the vector units two thirds busy (at 105, before the conversion and the root were shortened, they were
// the bound: 678 us); MNIST's eight tensors with 32-bit moments 18.5 us (5.0 TB/s).  Where a tensor or its gradient does not start at a multiple of 16
// bytes its elements are moved one by one: the 268 M as 64 allocations of their own, all values random, 490-600 us, one element further on 820-860.
// A second pair of types is a second launch over all chunks, whose workgroups leave at once where it is not theirs: 38-41 us for 131 000.
//
// 8-bit moments: 256 elements share a scale.  m and r = sqrt(v) (the root halves the range that the code has to span) are e4m3 times
// a power of two that brings the block's largest magnitude into [128, 256).  They are rounded stochastically, with 16 bits of a hash
// of seed, step, block and element: with b2 = 0.999 one step moves r by 0.05 % of itself and e4m3's grid is 6-12 %, so rounding to
// nearest would freeze it after some thirty steps, while the expectation of the stochastic rounding follows the average exactly.  A
// power of two keeps the grid in place while the largest magnitude stays in its binade, so a value that does not move is not
// rounded again.  r > 0 never becomes 0: the denominator must not vanish under an m that was kept.  Infinities and NaN are held as
// NaN and do not touch the scale: the other elements of their block keep their values.
#include "common.h"
#include "adamw.h"

#pragma clang fp contract(off)  // the moments are rounded operation by operation, as the eager form on the CPU rounds them

namespace {
constexpr int BLOCK = 256;    // elements that share a scale
constexpr int CHUNK = 2048;   // elements of a workgroup: 8 a lane, so that 16-bit operands move 16 bytes a lane
constexpr int NARGS = 200;    // tensors whose pointers one `begin` launch takes (its arguments, 4096 bytes, would hold 232)
}  // namespace

struct AdamWLive {  // what `begin` leaves for `apply`, one a tensor
  void* p;
  const void* g;
  long n, at;       // elements; the tensor's place in the arenas
  float lr1, ic2;   // lr / (1-b1^t), 1 / sqrt(1-b2^t)
  uint32_t key;     // of this step's random bits
  int kind;         // bit 0: bf16 parameters, bit 1: bf16 gradients, bit 2: both allow 16-byte accesses; -1: no gradient
};

struct AdamWPointers {
  int first, count;
  void* p[NARGS];
  const void* g[NARGS];
  int8_t kind[NARGS];
};
static_assert(sizeof(AdamWPointers) + sizeof(AdamWLaunch) <= 4096, "kernel arguments");

// xor-shift and odd multipliers (fractional digits of sqrt(2) and sqrt(3))
__device__ __forceinline__ uint32_t adamw_mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

__global__ __launch_bounds__(256) void adamw_begin_kernel(const AdamWLaunch a, const AdamWPointers ptr) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= ptr.count) return;
  const int k = ptr.first + i;
  AdamWLive l;
  l.p = ptr.p[i];
  l.g = ptr.g[i];
  l.n = a.shape[2 * k];
  l.at = a.shape[2 * k + 1];
  l.kind = ptr.kind[i];
  if (l.kind >= 0) {
    const int t = a.step[k] + 1;
    a.step[k] = t;
    double p1 = 1.0, p2 = 1.0, b1 = a.beta1, b2 = a.beta2;  // b^t by repeated squaring
    for (unsigned e = (unsigned)t; e; e >>= 1) {
      if (e & 1u) { p1 *= b1; p2 *= b2; }
      b1 *= b1;
      b2 *= b2;
    }
    l.lr1 = (float)(a.lr / (1.0 - p1));
    l.ic2 = (float)(1.0 / sqrt(1.0 - p2));
    l.key = adamw_mix(a.seed + (uint32_t)t * 0x9E3779B9u);
  }
  static_cast<AdamWLive*>(a.live)[k] = l;
}

template <typename T> struct Raw8 { uint4 q[sizeof(T) / 2]; };  // eight elements as loaded (T: float, or uint16_t for bf16)

template <typename T> __device__ __forceinline__ float raw_get(const Raw8<T>& r, int i) {
  if constexpr (sizeof(T) == 4) return reinterpret_cast<const float*>(&r)[i];
  else return bf2f(reinterpret_cast<const uint16_t*>(&r)[i]);
}
template <typename T> __device__ __forceinline__ void raw_set(Raw8<T>& r, int i, float v) {
  if constexpr (sizeof(T) == 4) reinterpret_cast<float*>(&r)[i] = v;
  else reinterpret_cast<uint16_t*>(&r)[i] = f2bf(v);  // to nearest even
}
template <typename T> __device__ __forceinline__ Raw8<T> raw_load(const T* src, long e0, long n, bool whole) {
  Raw8<T> r;
  if (whole) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(T) / 2); ++j) r.q[j] = reinterpret_cast<const uint4*>(src + e0)[j];
  } else {  // a tensor's last elements, or one that is not aligned: inside the tensor whatever the lane, zeros behind it
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T e = src[e0 + i < n ? e0 + i : n - 1];
      reinterpret_cast<T*>(&r)[i] = e0 + i < n ? e : T(0);
    }
  }
  return r;
}
template <typename T> __device__ __forceinline__ void raw_store(T* dst, long e0, long n, bool whole, const Raw8<T>& r) {
  if (whole) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(T) / 2); ++j) reinterpret_cast<uint4*>(dst + e0)[j] = r.q[j];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e0 + i < n) dst[e0 + i] = reinterpret_cast<const T*>(&r)[i];
  }
}

// The largest of the 32 lanes of a block: as bits, so that the order of the integers is that of the magnitudes.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o, 64));
  return x;
}
constexpr uint32_t INF_BITS = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_magnitude(float x) { return magnitude(x) < INF_BITS ? magnitude(x) : 0u; }

// The nearest float to sqrt(x) for x = 0, infinity, NaN and from 2^-96 on, by Tuckerman's rounding test: v_sqrt_f32 is at most one step off,
// and the signs of x - (s - step) s and x - (s + step) s say which neighbour is right.  (The tests compare moments with the CPU's nearest root, bit for bit.)  sqrtf also scales small arguments: 19 instead of
// 9 instructions, which count here (see adamw_apply_kernel).
__device__ __forceinline__ float sqrt_from_2_96(float x) {
  const float s = __builtin_amdgcn_sqrtf(x), lo = __uint_as_float(__float_as_uint(s) - 1u), hi = __uint_as_float(__float_as_uint(s) + 1u);
  const float r = fmaf(-lo, s, x) <= 0.f ? lo : s;
  return fmaf(-hi, s, x) > 0.f ? hi : r;
}
// x to e4m3, |x| <= 256: v_cvt_sr_fp8_f32 adds the random bits' upper 20 below the three mantissa bits that stay and cuts (on the grid of
// 2^-9 below 2^-6), which rounds up with the probability of the fraction.  What is not finite becomes NaN.
__device__ __forceinline__ uint32_t stochastic_e4m3(float x, uint32_t random, uint32_t word, int byte) {
  switch (byte) {
    case 0: return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x, random, (int)word, 0);
    case 1: return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x, random, (int)word, 1);
    case 2: return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x, random, (int)word, 2);
    default: return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x, random, (int)word, 3);
  }
}
__device__ __forceinline__ void e4m3_floats(uint2 c, float* out) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(h ? c.y : c.x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(h ? c.y : c.x, true);
    out[4 * h] = lo.x; out[4 * h + 1] = lo.y; out[4 * h + 2] = hi.x; out[4 * h + 3] = hi.y;
  }
}

template <typename P, typename G, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_apply_kernel(const AdamWLaunch a) {
  const int2 chunk = static_cast<const int2*>(a.chunks)[blockIdx.x];
  const AdamWLive l = static_cast<const AdamWLive*>(a.live)[chunk.x];
  if (l.kind < 0 || (l.kind & 3) != (sizeof(P) == 2) + 2 * (sizeof(G) == 2)) return;  // no gradient, or another launch's types
  const long e0 = (long)chunk.y * CHUNK + threadIdx.x * 8;
  if ((e0 & ~(long)(BLOCK - 1)) >= l.n) return;  // (the 32 lanes of a block leave together)
  const bool whole = (l.kind & 4) && e0 + 8 <= l.n;
  P* const p = static_cast<P*>(l.p);
  const Raw8<G> rg = raw_load(static_cast<const G*>(l.g), e0, l.n, whole);
  Raw8<P> rp = raw_load(p, e0, l.n, whole);
  const long s0 = l.at + e0;  // the place in the arenas (behind the tensor's end they hold zeros up to the block's end, and keep them)
  const float b1 = a.b1, ob1 = a.ob1, b2 = a.b2, ob2 = a.ob2;
  float m[8], v[8], r[8];
  if constexpr (EIGHT) {
    const uint2 cm = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + s0);
    const uint2 cr = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + s0);
    const float ms = a.m_scale[s0 / BLOCK], rs = a.r_scale[s0 / BLOCK];
    e4m3_floats(cm, m);
    e4m3_floats(cr, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] *= ms;
      v[i] *= rs;
      v[i] *= v[i];
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      reinterpret_cast<float4*>(m)[h] = reinterpret_cast<const float4*>(static_cast<const float*>(a.m) + s0)[h];
      reinterpret_cast<float4*>(v)[h] = reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + s0)[h];
    }
  }
  float vmin = 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float g = raw_get(rg, i) * a.grad_scale;
    m[i] = b1 * m[i] + ob1 * g;
    v[i] = b2 * v[i] + ob2 * (g * g);
    vmin = fminf(vmin, v[i]);
  }
  if (!EIGHT || vmin < 0x1p-96f) {  // (zeros too; 32-bit moments are bound by memory either way)
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = sqrtf(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = sqrt_from_2_96(v[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) raw_set(rp, i, raw_get(rp, i) * a.decay - l.lr1 * (m[i] / (r[i] * l.ic2 + a.eps)));
  raw_store(p, e0, l.n, whole, rp);
  if constexpr (EIGHT) {
    uint32_t mmax = 0, rmax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mmax = max(mmax, magnitude(m[i]));
      rmax = max(rmax, __float_as_uint(r[i]));  // (r is not negative; a NaN is larger than infinity whatever its sign)
    }
    if (max(mmax, rmax) >= INF_BITS) {  // the scale is that of the finite ones
      mmax = rmax = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mmax = max(mmax, finite_magnitude(m[i]));
        rmax = max(rmax, finite_magnitude(r[i]));
      }
    }
    // scale 2^(e-7) for a largest magnitude in [2^e, 2^(e+1)); 2^-126 where that would be no normal number
    const uint32_t mf = max(block_max(mmax) >> 23, 8u), rf = max(block_max(rmax) >> 23, 8u);
    const float minv = __uint_as_float((261u - mf) << 23), rinv = __uint_as_float((261u - rf) << 23);
    const uint32_t key = adamw_mix(l.key ^ (uint32_t)(s0 / BLOCK)) + ((uint32_t)s0 & (BLOCK - 1));
    uint32_t cm[2] = {0, 0}, cr[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t random = adamw_mix(key + i);  // 16 bits for each of the two
      cm[i / 4] = stochastic_e4m3(m[i] * minv, random << 16, cm[i / 4], i % 4);
      const float q = r[i] * rinv;
      cr[i / 4] = stochastic_e4m3(r[i] > 0.f ? fmaxf(q, 0x1p-9f) : q, random & 0xffff0000u, cr[i / 4], i % 4);  // (2^-9: the smallest value)
    }
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + s0) = make_uint2(cm[0], cm[1]);
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + s0) = make_uint2(cr[0], cr[1]);
    if ((threadIdx.x & 31) == 0) {
      a.m_scale[s0 / BLOCK] = __uint_as_float((mf - 7u) << 23);
      a.r_scale[s0 / BLOCK] = __uint_as_float((rf - 7u) << 23);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      reinterpret_cast<float4*>(static_cast<float*>(a.m) + s0)[h] = reinterpret_cast<const float4*>(m)[h];
      reinterpret_cast<float4*>(static_cast<float*>(a.v) + s0)[h] = reinterpret_cast<const float4*>(v)[h];
    }
  }
}

template <typename P, typename G> static void adamw_apply(const AdamWLaunch& all, hipStream_t st) {
  constexpr int MOST = 1 << 23;  // chunks of a launch: its threads have to be fewer than 2^32 (more are cut off without an error)
  for (long first = 0; first < all.nchunks; first += MOST) {
    AdamWLaunch a = all;
    a.chunks = static_cast<const int2*>(all.chunks) + first;
    a.nchunks = (int)(all.nchunks - first < MOST ? all.nchunks - first : MOST);
    if (a.bits == 8) hipLaunchKernelGGL((adamw_apply_kernel<P, G, true>), dim3(a.nchunks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((adamw_apply_kernel<P, G, false>), dim3(a.nchunks), dim3(256), 0, st, a);
  }
}

DTF_API int dtf_sizeof_adamw_live() { return (int)sizeof(AdamWLive); }

DTF_API int dtf_adamw(const AdamWLaunch* a, const uint64_t* p, const uint64_t* g, const uint8_t* kind, hipStream_t st) {
  if (!a || !p || !g || !kind || a->ntensors < 0 || a->nchunks < 0 || (a->bits != 8 && a->bits != 32)) return -22;
  if (a->ntensors == 0 || a->nchunks == 0) return 0;
  if (!a->shape || !a->chunks || !a->live || !a->step || !a->m || !a->v || (a->bits == 8 && (!a->m_scale || !a->r_scale))) return -22;
  unsigned types = 0;
  for (int first = 0; first < a->ntensors; first += NARGS) {
    AdamWPointers q;
    q.first = first;
    q.count = a->ntensors - first < NARGS ? a->ntensors - first : NARGS;
    for (int i = 0; i < q.count; ++i) {
      const uint64_t pp = p[first + i], gg = g[first + i];
      const int k = kind[first + i] & 3;
      if (gg && (!pp || pp % ((k & 1) ? 2 : 4) || gg % ((k & 2) ? 2 : 4))) return -22;
      q.p[i] = reinterpret_cast<void*>(pp);
      q.g[i] = reinterpret_cast<const void*>(gg);
      q.kind[i] = (int8_t)(gg ? k | (((pp | gg) & 15) == 0 ? 4 : 0) : -1);
      if (gg) types |= 1u << k;
    }
    hipLaunchKernelGGL(adamw_begin_kernel, dim3((q.count + 255) / 256), dim3(256), 0, st, *a, q);
    DTF_CHECK_LAUNCH();
  }
  // one launch for each pair of types that is there (usually one); the workgroups of other pairs leave at once
  if (types & 1u) adamw_apply<float, float>(*a, st);
  if (types & 2u) adamw_apply<uint16_t, float>(*a, st);
  if (types & 4u) adamw_apply<float, uint16_t>(*a, st);
  if (types & 8u) adamw_apply<uint16_t, uint16_t>(*a, st);
  DTF_CHECK_LAUNCH();
  return 0;
}
