// The optimiser's step over all tensors of a model (no reference kernel: the reference trains with PyTorch's
// optimiser), in a few launches whatever the number of tensors.
//
//   g' = g min(1, max_norm / (|g| + 1e-6))                       (with a global norm; skipped unless finite)
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tables of tensors travel as kernel parameters (no copy, no device memory; captured by value).  Every
// tensor is cut into blocks of 256 elements, its state starts at a multiple of 256 in the group's flat state.
//
// 8-bit moments.  The 256 values of a block share the power of two of the largest magnitude (one byte, fp32's
// exponent field; 255 = a value was not finite, the whole block then stands for NaN).  Over it, m is a sign, 4
// exponent and 3 fraction bits, sqrt(v) 4 exponent and 4 fraction bits, with gradual underflow: the high bits of the
// fp32 pattern of |x| 2^(-e - 112), whose subnormals fall where the small format's do.  The bits below are dropped
// after adding an offset from an additive sequence over (element, step), one a moment, so a value that stays is
// rounded up as often as it is near the upper neighbour: round-to-nearest would never move an average whose step is
// 1 - b2 = 1e-3 of itself.  What passes the largest code stays there, so a block's largest sqrt(v) moves on only
// when one step takes it to the next power of two; 4,000 steps of random gradients leave sqrt(v) 1.4% low in
// the mean and a block's largest one 40%, gradients that never change leave it at 1/8 to 1/4 of its value.
// sqrt(v) over 0 is never rounded to 0 (the update would divide by eps).
// The moments' operations are single rounded fp32 ones in a fixed order, so the codes are reproducible bit for bit.
//
// With 32-bit moments it is bound by memory: 24.5M fp32 parameters in 240 tensors (28 bytes each) take 99 us, 6.9 TB/s.
// With 8-bit ones (16 bytes) 82 us where the bytes take 60; 120M bf16 parameters (10 bytes) 318 us where they take 184:
// 66 instructions an element keep the integer pipe two thirds busy.  The clipping norm of the 24.5M takes 21 to 27 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>

#include "e2a_common.cuh"

namespace {

constexpr int kBlock = 256;          // elements that share a scale
constexpr int kThreads = 256;
constexpr int kUnit = 8 * kBlock;    // elements that a CTA takes at a time: one block a warp
constexpr int kTensors = 512;        // tensors in one launch's table (18.4 KB of kernel parameters)
constexpr int kNormCtas = 1184;      // partial sums of squares of one launch (8 per SM)
// CTAs of one step, each a contiguous range: a few waves so that they even out; with 8 bits one wave, whose start
// (its tensor, its scalars) then counts once (24.5M fp32 parameters: 16 a SM 126 us, 4 a SM 94 us)
constexpr int kStepCtas32 = 148 * 16, kStepCtas8 = 148 * 4;

struct Table {
  uint64_t p[kTensors];
  uint64_t g[kTensors];
  int64_t numel[kTensors];
  int64_t offset[kTensors];
  int32_t first[kTensors + 1];       // first unit of every tensor
  int32_t n;
};

struct Slots { int32_t slot[kTensors]; };

struct Scalars { float size, root; int32_t t, pad; };
struct Globals { float decay, coef; int32_t skip, pad; };

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// The tensor that owns unit b: the last j with first[j] <= b (empty tensors own none).
__device__ __forceinline__ int tensor_of(const Table& t, int32_t b) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

// ---- 8-bit values -------------------------------------------------------------------------------
// The roundings' offsets: sums i a + t b mod 2^32 of element and step by odd 32-bit fractions of the powers of the
// root of x^5 = x + 1; the upper 20 bits for the first moment, the upper 19 for the second.
constexpr uint32_t kIndexStepM = 0xDB4F0B91u, kTimeStepM = 0xBBE05633u;
constexpr uint32_t kIndexStepS = 0xA0F2EC75u, kTimeStepS = 0x89E18285u;

__device__ __forceinline__ float two_to_112() { return __uint_as_float((112u + 127u) << 23); }
__device__ __forceinline__ float two_to_m112() { return __uint_as_float((127u - 112u) << 23); }
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b == 255u ? 0x7FC00000u : b << 23); }

// The shared exponent of a block from the largest magnitude's bits (integer order is value order, NaN above).
__device__ __forceinline__ uint32_t shared_exponent(uint32_t largest) {
  if (largest >= 0x7F800000u) return 255u;
  return min(max(largest >> 23, 27u), 253u);
}

__device__ __forceinline__ float unpack_m(uint32_t code, float scale) {
  const float y = __fmul_rn(__fmul_rn(__uint_as_float((code & 127u) << 20), two_to_112()), scale);
  return code > 127u ? -y : y;
}
__device__ __forceinline__ float unpack_s(uint32_t code, float scale) {
  return __fmul_rn(__fmul_rn(__uint_as_float(code << 19), two_to_112()), scale);
}

__device__ __forceinline__ uint32_t pack_m(float m, uint32_t b, uint32_t dither) {
  if (b == 255u) return 0u;
  const float z = __fmul_rn(__fmul_rn(fabsf(m), __uint_as_float((254u - b) << 23)), two_to_m112());
  return min((__float_as_uint(z) + dither) >> 20, 127u) | ((__float_as_uint(m) >> 24) & 128u);
}
__device__ __forceinline__ uint32_t pack_s(float s, uint32_t b, uint32_t dither) {
  if (b == 255u) return 0u;
  const float z = __fmul_rn(__fmul_rn(s, __uint_as_float((254u - b) << 23)), two_to_m112());
  return max(min((__float_as_uint(z) + dither) >> 19, 255u), s > 0.f ? 1u : 0u);
}

// ---- the step ------------------------------------------------------------------------------------
struct Hyper {
  double lr, log_beta1, log_beta2, decay;    // the betas' logarithms to base 2
  const float* lr_dev;
  const float* norm;
  float max_norm;
};

// Per tensor t <- t + 1, lr / (1 - b1^t) and 1 / sqrt(1 - b2^t) in 64 bits, rounded once.
__global__ void k_adamw_scalars(const __grid_constant__ Slots slots, Hyper h, int32_t* __restrict__ step, int n,
                                Scalars* __restrict__ s, Globals* __restrict__ g) {
  float norm = 0.f;
  bool skip = false;
  if (h.norm) {
    norm = *h.norm;
    skip = !isfinite(norm);
  }
  const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int32_t k = slots.slot[j];
    const int32_t t = step[k] + 1;
    if (!skip) step[k] = t;
    Scalars v;
    v.size = (float)(lr / (1.0 - exp2(t * h.log_beta1)));
    v.root = (float)(1.0 / sqrt(1.0 - exp2(t * h.log_beta2)));
    v.t = t;
    v.pad = 0;
    s[j] = v;
  }
  if (threadIdx.x == 0) {
    Globals v;
    v.decay = (float)(1.0 - lr * h.decay);
    v.coef = h.norm ? fminf(__fdiv_rn(h.max_norm, __fadd_rn(norm, 1e-6f)), 1.f) : 1.f;
    v.skip = skip;
    v.pad = 0;
    *g = v;
  }
}

__device__ __forceinline__ float reciprocal(float x) {      // within 1 unit; 0 for inf, inf below 2^-126
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float root_approx(float x) {     // within 2^-23; 0 below 2^-126
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What all elements of a launch share.
struct Rates { float b1, a1, b2, a2, eps, one; };

// a b + c d, each product and the sum rounded on its own.  The sum is a fused product with a 1 that the compiler
// does not know: it may contract a packed product and sum into one rounding.
__device__ __forceinline__ float2 sum_of_products(float2 a, float b, float2 c, float d, float one) {
  return f2_fma(f2_mul(a, f2(b)), f2(one), f2_mul(c, f2(d)));
}

// One element's moments; every operation rounded on its own (see above).
__device__ __forceinline__ float next_m(float m, float g, const Rates& r) {
  return __fadd_rn(__fmul_rn(m, r.b1), __fmul_rn(g, r.a1));
}
__device__ __forceinline__ float next_v(float v, float g, const Rates& r) {
  return __fadd_rn(__fmul_rn(v, r.b2), __fmul_rn(__fmul_rn(g, g), r.a2));
}
// p decay - m / (s root + eps) size: nothing is kept of it but p, so the quotient may be a unit or two off.
__device__ __forceinline__ float next_p(float p, float m, float s, const Globals& gl, const Scalars& sc, float eps) {
  return fmaf(-m * reciprocal(fmaf(s, sc.root, eps)), sc.size, p * gl.decay);
}

// Four neighbouring values of a tensor of n from element i on, 0 beyond its end; one load where the tensor's
// address allows it (`vec`) and all four exist.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) {
    if (sizeof(T) == 4) return *reinterpret_cast<const float4*>(p + i);
    const uint2 w = *reinterpret_cast<const uint2*>(p + i);
    const T* h = reinterpret_cast<const T*>(&w);
    return make_float4(to_f(h[0]), to_f(h[1]), to_f(h[2]), to_f(h[3]));
  }
  float4 v = f4_zero();
  if (i < n) v.x = to_f(p[i]);
  if (i + 1 < n) v.y = to_f(p[i + 1]);
  if (i + 2 < n) v.z = to_f(p[i + 2]);
  if (i + 3 < n) v.w = to_f(p[i + 3]);
  return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool vec, float4 v) {
  const T h[4] = {from_f<T>(v.x), from_f<T>(v.y), from_f<T>(v.z), from_f<T>(v.w)};
  if (vec && i + 4 <= n) {
    if (sizeof(T) == 4)
      *reinterpret_cast<float4*>(p + i) = v;
    else
      *reinterpret_cast<uint2*>(p + i) = *reinterpret_cast<const uint2*>(h);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = h[k];
  }
}

// Eight values of a thread: elements 4 l and 128 + 4 l on of its warp's block.
struct Eight { float v[8]; };

template <typename T>
__device__ __forceinline__ Eight load8(const T* p, int64_t i, int64_t n, bool vec) {
  Eight o;
  *reinterpret_cast<float4*>(o.v) = load4(p, i, n, vec);
  *reinterpret_cast<float4*>(o.v + 4) = load4(p, i + 128, n, vec);
  return o;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t i, int64_t n, bool vec, const Eight& v) {
  store4(p, i, n, vec, *reinterpret_cast<const float4*>(v.v));
  store4(p, i + 128, n, vec, *reinterpret_cast<const float4*>(v.v + 4));
}

// Where a thread's values lie: its first element, the tensor's elements, and that element's sums for the offsets.
struct Where {
  int64_t i, n;
  uint32_t um, us;
};

// A thread's codes of a block and the block's shared exponents.
struct Codes {
  uint32_t m[2], s[2], em, es;
};

// The new codes for any values, and the new parameters if they are not there yet.  By value, and g read again: the
// rarely made call must not tie the caller's values to memory or registers.
template <typename T>
__device__ __noinline__ Codes block_exact(const Codes h, T* p, const T* g, bool vec, bool with_p, bool clip,
                                          const Where w, const Globals gl, const Scalars sc, const Rates r) {
  Eight m, s;
  Eight pv = load8(p, w.i, w.n, vec);
  const Eight gv = load8(g, w.i, w.n, vec);
  uint32_t top_m = 0, top_s = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float ge = clip ? __fmul_rn(gv.v[e], gl.coef) : gv.v[e];
    const float r0 = unpack_s((h.s[e / 4] >> (8 * (e % 4))) & 255u, scale_of(h.es));
    m.v[e] = next_m(unpack_m((h.m[e / 4] >> (8 * (e % 4))) & 255u, scale_of(h.em)), ge, r);
    s.v[e] = __fsqrt_rn(next_v(__fmul_rn(r0, r0), ge, r));
    pv.v[e] = next_p(pv.v[e], m.v[e], s.v[e], gl, sc, r.eps);
    if (w.i + e % 4 + 128 * (e / 4) >= w.n) m.v[e] = s.v[e] = 0.f;     // a block holds no more than its tensor
    top_m = max(top_m, __float_as_uint(m.v[e]) & 0x7FFFFFFFu);
    top_s = max(top_s, __float_as_uint(s.v[e]) & 0x7FFFFFFFu);
  }
  if (with_p) store8(p, w.i, w.n, vec, pv);
  Codes o{};
  o.em = shared_exponent(__reduce_max_sync(0xffffffffu, top_m));
  o.es = shared_exponent(__reduce_max_sync(0xffffffffu, top_s));
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t at = e % 4 + 128 * (e / 4);
    o.m[e / 4] |= pack_m(m.v[e], o.em, (w.um + at * kIndexStepM) >> 12) << (8 * (e % 4));
    o.s[e / 4] |= pack_s(s.v[e], o.es, (w.us + at * kIndexStepS) >> 13) << (8 * (e % 4));
  }
  return o;
}

__device__ __forceinline__ float max_or_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Byte `k` of a word as its top byte, and four words' top bytes as one word.
__device__ __forceinline__ uint32_t byte_on_top(uint32_t w, int k) { return __byte_perm(w, 0u, (k << 12) | 0x444u); }
__device__ __forceinline__ uint32_t top_bytes(const uint32_t* w) {
  return __byte_perm(__byte_perm(w[0], w[1], 0x0073u), __byte_perm(w[2], w[3], 0x0073u), 0x5410u);
}

// The step of a whole block of ordinary values, in about half of block_exact's instructions (its time is theirs: 82
// an element took 408 us on 120M bf16 values, 66 take 318): packed fp32 arithmetic, scales as one product,
// and square roots within 2^-23.  A root's code is the exact one's unless the rounding offset brings it
// within a few units of the next code; where that, or a value's range, is in doubt for any of the warp, `sure` is
// false and the codes are not to be used.  The parameters are stored either way.
template <typename T>
__device__ __forceinline__ Codes block_fast(const Codes& h, T* pt, const T* gt, bool vec, bool clip, const Where& w,
                                            const Globals& gl, const Scalars& sc, const Rates& r, bool* sure) {
  // scales 2^(e + 112) of the old codes, in range for e <= 15 (the caller has looked)
  const float2 fm = f2(__uint_as_float((h.em + 112u) << 23)), fs = f2(__uint_as_float((h.es + 112u) << 23));
  float2 m[4], s[4];
  float top_m = 0.f, top_s = 0.f;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float4 p4 = load4(pt, w.i + 128 * half, w.n, vec);
    const float4 g4 = load4(gt, w.i + 128 * half, w.n, vec);
    float2 v[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float2 g = q ? make_float2(g4.z, g4.w) : make_float2(g4.x, g4.y);
      if (clip) g = f2_mul(g, f2(gl.coef));
      const uint32_t a0 = byte_on_top(h.m[half], 2 * q), a1 = byte_on_top(h.m[half], 2 * q + 1);
      const uint32_t b0 = byte_on_top(h.s[half], 2 * q) >> 5, b1 = byte_on_top(h.s[half], 2 * q + 1) >> 5;
      // magnitude to bits 20..26 (19..26), sign to bit 31
      const float2 m0 = f2_mul(make_float2(__uint_as_float((uint32_t)((int32_t)a0 >> 4) & 0x87F00000u),
                                           __uint_as_float((uint32_t)((int32_t)a1 >> 4) & 0x87F00000u)), fm);
      const float2 s0 = f2_mul(make_float2(__uint_as_float(b0), __uint_as_float(b1)), fs);
      m[2 * half + q] = sum_of_products(m0, r.b1, g, r.a1, r.one);
      v[q] = sum_of_products(f2_mul(s0, s0), r.b2, f2_mul(g, g), r.a2, r.one);
      s[2 * half + q] = make_float2(root_approx(v[q].x), root_approx(v[q].y));
    }
    // a second moment over 0 but below 2^-126, whose root is not 0 (a 0's bits less 1 are the largest)
    if (min(min(__float_as_uint(v[0].x) - 1u, __float_as_uint(v[0].y) - 1u),
            min(__float_as_uint(v[1].x) - 1u, __float_as_uint(v[1].y) - 1u)) < 0x007FFFFFu) {
#pragma unroll
      for (int q = 0; q < 2; ++q) s[2 * half + q] = make_float2(__fsqrt_rn(v[q].x), __fsqrt_rn(v[q].y));
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int e = 2 * half + q;
      const float2 p = q ? make_float2(p4.z, p4.w) : make_float2(p4.x, p4.y);
      const float2 d = f2_fma(s[e], f2(sc.root), f2(r.eps));
      const float2 up = f2_mul(m[e], make_float2(reciprocal(d.x), reciprocal(d.y)));
      const float2 next = f2_fma(up, f2(-sc.size), f2_mul(p, f2(gl.decay)));
      if (q) {
        p4.z = next.x;
        p4.w = next.y;
      } else {
        p4.x = next.x;
        p4.y = next.y;
      }
      top_m = max_or_nan(top_m, fabsf(m[e].x), fabsf(m[e].y));
      top_s = max_or_nan(top_s, s[e].x, s[e].y);
    }
    store4(pt, w.i + 128 * half, w.n, vec, p4);
  }
  Codes o;
  const uint32_t bits_s = __reduce_max_sync(0xffffffffu, __float_as_uint(top_s) & 0x7FFFFFFFu);
  o.em = shared_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m) & 0x7FFFFFFFu));
  o.es = shared_exponent(bits_s);
  // in range for one product each (NaN and infinities are above), and the exponent not in doubt
  *sure = o.em <= 127 + 14 && o.es <= 127 + 14 && o.es >= 127 - 40 && ((bits_s + 4u) & 0x7FFFFFu) >= 8u;
  if (!*sure) return o;
  const float zm = __uint_as_float((254u - 112u - o.em) << 23);
  const float2 zs = f2(__uint_as_float((254u - 112u - o.es) << 23));
  uint32_t doubt = 8u;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t cm[4], cs[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float2 mv = m[2 * half + q], sv = s[2 * half + q], z = f2_mul(sv, zs);
      const float me[2] = {mv.x, mv.y}, se[2] = {sv.x, sv.y}, ze[2] = {z.x, z.y};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t at = 2 * q + k + 128 * half;
        const uint32_t tm = __float_as_uint(__fmul_rn(fabsf(me[k]), zm)) + ((w.um + at * kIndexStepM) >> 12);
        cm[2 * q + k] = (min(tm, 0x07FFFFFFu) << 4) | (__float_as_uint(me[k]) & 0x80000000u);
        // over zero at least the smallest code; 4 more than the sum, so that what is in doubt lies in 0..7 of the
        // dropped bits
        const float least = fminf(se[k], __uint_as_float(1u << 19));
        const uint32_t ts = __float_as_uint(fmaxf(ze[k], least)) + ((w.us + at * kIndexStepS) >> 13) + 4u;
        doubt = min(doubt, ts & 0x7FFFFu);
        cs[2 * q + k] = min(ts, 0x07FFFFFFu) << 5;
      }
    }
    o.m[half] = top_bytes(cm);
    o.s[half] = top_bytes(cs);
  }
  *sure = !__any_sync(0xffffffffu, doubt < 8u);
  return o;
}

// Asks for a later block's lines, a lane each: parameters, gradients and codes.
template <typename T>
__device__ __forceinline__ void prefetch_block(const T* p, const T* g, const uint8_t* m, const uint8_t* s) {
  constexpr int LINES = kBlock * (int)sizeof(T) / 128;
  const int lane = threadIdx.x & 31;
  const char* at = lane < LINES ? (const char*)p + lane * 128
                   : lane < 2 * LINES ? (const char*)g + (lane - LINES) * 128
                   : lane < 2 * LINES + 2 ? (const char*)m + (lane - 2 * LINES) * 128
                                          : (const char*)s + (lane - 2 * LINES - 2) * 128;
  if (lane < 2 * LINES + 4) asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
}

// A CTA walks a contiguous range of units; a warp owns one block of 256 of each, lane l the values 4 l and
// 128 + 4 l on (16-byte loads of fp32, 4-byte ones of codes, all neighbouring).
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads, 4)
k_adamw(const __grid_constant__ Table tab, int32_t n_units, int32_t per_cta, void* __restrict__ exp_avg,
        void* __restrict__ exp_avg_sq, uint8_t* __restrict__ scale_m, uint8_t* __restrict__ scale_v,
        const Scalars* __restrict__ scal, const Globals* __restrict__ glob, const Rates r, bool clip) {
  const Globals gl = *glob;
  if (gl.skip) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t from = blockIdx.x * per_cta, to = min(from + per_cta, n_units);
  int j = tensor_of(tab, from);
  for (int32_t b = from; b < to; ++b) {
    while (b >= tab.first[j + 1]) ++j;
    const int64_t i0 = (int64_t)(b - tab.first[j]) * kUnit + warp * kBlock, n = tab.numel[j];
    if (i0 >= n) continue;
    const int64_t i = i0 + 4 * lane, at = tab.offset[j] + i;
    const Scalars s = scal[j];
    T* pt = reinterpret_cast<T*>(tab.p[j]);
    const T* gt = reinterpret_cast<const T*>(tab.g[j]);
    const bool vec = ((tab.p[j] | tab.g[j]) & (4 * sizeof(T) - 1)) == 0;
    if (BITS == 32) {
      Eight p = load8(pt, i, n, vec), g = load8(gt, i, n, vec);
      float* mt = (float*)exp_avg + at;
      float* vt = (float*)exp_avg_sq + at;
      Eight m, v;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        *reinterpret_cast<float4*>(m.v + 4 * k) = *reinterpret_cast<const float4*>(mt + 128 * k);
        *reinterpret_cast<float4*>(v.v + 4 * k) = *reinterpret_cast<const float4*>(vt + 128 * k);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (clip) g.v[e] = __fmul_rn(g.v[e], gl.coef);
        m.v[e] = next_m(m.v[e], g.v[e], r);
        v.v[e] = next_v(v.v[e], g.v[e], r);
        p.v[e] = next_p(p.v[e], m.v[e], __fsqrt_rn(v.v[e]), gl, s, r.eps);
      }
      store8(pt, i, n, vec, p);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        *reinterpret_cast<float4*>(mt + 128 * k) = *reinterpret_cast<const float4*>(m.v + 4 * k);
        *reinterpret_cast<float4*>(vt + 128 * k) = *reinterpret_cast<const float4*>(v.v + 4 * k);
      }
    } else {
      uint32_t* mt = reinterpret_cast<uint32_t*>((uint8_t*)exp_avg + at);
      uint32_t* vt = reinterpret_cast<uint32_t*>((uint8_t*)exp_avg_sq + at);
      const Codes h{{mt[0], mt[32]}, {vt[0], vt[32]}, scale_m[at / kBlock], scale_v[at / kBlock]};
      if (i0 + kUnit + kBlock <= n)      // the warp's next block
        prefetch_block(pt + i0 + kUnit, gt + i0 + kUnit, (const uint8_t*)exp_avg + (at - 4 * lane) + kUnit,
                       (const uint8_t*)exp_avg_sq + (at - 4 * lane) + kUnit);
      const Where w{i, n, (uint32_t)i * kIndexStepM + (uint32_t)s.t * kTimeStepM,
                    (uint32_t)i * kIndexStepS + (uint32_t)s.t * kTimeStepS};
      // whole blocks of moments below 2^16; a block of NaN has exponent 255
      const bool ordinary = i0 + kBlock <= n && max(h.em, h.es) <= 127 + 15;
      bool sure = false;
      Codes o;
      if (ordinary) o = block_fast(h, pt, gt, vec, clip, w, gl, s, r, &sure);
      if (!sure) o = block_exact(h, pt, gt, vec, !ordinary, clip, w, gl, s, r);
      mt[0] = o.m[0];
      mt[32] = o.m[1];
      vt[0] = o.s[0];
      vt[32] = o.s[1];
      if (lane == 0) {
        scale_m[at / kBlock] = (uint8_t)o.em;
        scale_v[at / kBlock] = (uint8_t)o.es;
      }
    }
  }
}

// Whole blocks of 256, eight values a thread at a time.
__global__ void __launch_bounds__(kThreads)
k_moments_unpack(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v, const uint8_t* __restrict__ scale_m,
                 const uint8_t* __restrict__ scale_v, int64_t n, float* __restrict__ out_m,
                 float* __restrict__ out_v) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t b = blockIdx.x * (int64_t)(kThreads / 32) + (threadIdx.x >> 5); b < n / kBlock; b += step) {
    const float sm = scale_of(scale_m[b]), ss = scale_of(scale_v[b]);
    uint32_t cm[2], cv[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      cm[k] = __ldg(reinterpret_cast<const uint32_t*>(m + b * kBlock) + lane + 32 * k);
      cv[k] = __ldg(reinterpret_cast<const uint32_t*>(v + b * kBlock) + lane + 32 * k);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = unpack_m((cm[k] >> (8 * e)) & 255u, sm);
        const float r = unpack_s((cv[k] >> (8 * e)) & 255u, ss);
        y[e] = __fmul_rn(r, r);
      }
      __stcs(reinterpret_cast<float4*>(out_m + b * kBlock) + lane + 32 * k, make_float4(x[0], x[1], x[2], x[3]));
      __stcs(reinterpret_cast<float4*>(out_v + b * kBlock) + lane + 32 * k, make_float4(y[0], y[1], y[2], y[3]));
    }
  }
}

// ---- the global norm: partial sums in 64 bits, added up in order -----------------------------------
__device__ __forceinline__ double cta_sum(double s, double* sh) {
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.;
  for (int w = 0; w < kThreads / 32; ++w) s += sh[w];
  return s;
}

// The sum of eight squares in 64 bits, where every product is exact and the sum as good as.  An fp32 value's bits
// are those of the 64-bit one but for the exponent's bias (896 more) and its place, which two or three integer
// operations do faster than the conversion unit (240M bf16 values: 131 us with conversions).  That holds for
// ordinary values: zeros and subnormals come out as at most 2^-126, which a sum over 1e-20 does not see.  Other
// groups, with infinities and NaN among them, are converted.
__device__ __forceinline__ double squares(const float4 a, const float4 b) {
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  float rough = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) rough = fmaf(v[k], v[k], rough);
  double d[2] = {0., 0.};
  if (rough > 1e-20f && rough < 1e38f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t bits = __float_as_uint(v[k]) & 0x7FFFFFFFu;
      const double x = __hiloint2double((int)((bits >> 3) + (896u << 20)), (int)(bits << 29));
      d[k & 1] = fma(x, x, d[k & 1]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) d[k & 1] = fma((double)v[k], (double)v[k], d[k & 1]);
  }
  return d[0] + d[1];
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
k_sum_squares(const __grid_constant__ Table tab, int32_t n_units, int32_t per_cta, double* __restrict__ part) {
  __shared__ double sh[kThreads / 32];
  double s = 0.;
  const int32_t from = blockIdx.x * per_cta, to = min(from + per_cta, n_units);
  int j = tensor_of(tab, from);
  for (int32_t b = from; b < to; ++b) {
    while (b >= tab.first[j + 1]) ++j;
    const int64_t i0 = (int64_t)(b - tab.first[j]) * kUnit, n = tab.numel[j];
    const T* g = reinterpret_cast<const T*>(tab.g[j]);
    // four whole units at a time, their 16-byte loads all in flight (one unit at a time: 240M bf16 values 131 us)
    if ((tab.g[j] & 15) == 0 && b + 4 <= min(to, tab.first[j + 1]) && i0 + 4 * kUnit <= n) {
      const uint4* q = reinterpret_cast<const uint4*>(g + i0) + threadIdx.x;
      uint4 raw[sizeof(T) * 2];
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) * 2; ++k) raw[k] = __ldg(q + k * kThreads);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (sizeof(T) == 4) {
          s += squares(*reinterpret_cast<const float4*>(&raw[(2 * k) % (sizeof(T) * 2)]),
                       *reinterpret_cast<const float4*>(&raw[(2 * k + 1) % (sizeof(T) * 2)]));
        } else {
          const T* h = reinterpret_cast<const T*>(&raw[k]);
          s += squares(make_float4(to_f(h[0]), to_f(h[1]), to_f(h[2]), to_f(h[3])),
                       make_float4(to_f(h[4]), to_f(h[5]), to_f(h[6]), to_f(h[7])));
        }
      }
      b += 3;
      continue;
    }
    const bool vec = (tab.g[j] & (4 * sizeof(T) - 1)) == 0;
    s += squares(load4(g, i0 + 4 * threadIdx.x, n, vec), load4(g, i0 + 4 * (threadIdx.x + kThreads), n, vec));
  }
  const double all = cta_sum(s, sh);
  if (threadIdx.x == 0) part[blockIdx.x] = all;
}

__global__ void __launch_bounds__(kThreads)
k_norm(const double* __restrict__ part, int64_t n, float* __restrict__ norm) {
  __shared__ double sh[kThreads / 32];
  double s = 0.;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) s += part[i];
  s = cta_sum(s, sh);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

int64_t blocks_of(int64_t numel) { return (numel + kBlock - 1) / kBlock; }
int64_t units_of(int64_t numel) { return (numel + kUnit - 1) / kUnit; }

size_t width_of(int dtype) { return dtype == 0 ? 4 : 2; }

// Fills a launch's table with tensors [from, ...): as many as fit.  Returns the next tensor, units in *n_units.
int64_t fill(Table* t, int64_t from, int64_t n_tensors, const uint64_t* p, const uint64_t* g, const int64_t* numel,
             const int64_t* offset, int32_t* n_units) {
  int64_t units = 0, j = from;
  int k = 0;
  for (; j < n_tensors && k < kTensors; ++j, ++k) {
    const int64_t nu = units_of(numel[j]);
    if (k > 0 && units + nu > (1ll << 30)) break;
    t->p[k] = p ? p[j] : 0;
    t->g[k] = g[j];
    t->numel[k] = numel[j];
    t->offset[k] = offset ? offset[j] : 0;
    t->first[k] = (int32_t)units;
    units += nu;
  }
  t->first[k] = (int32_t)units;
  t->n = k;
  *n_units = (int32_t)units;
  return j;
}

bool bad_tensors(const uint64_t* t, const int64_t* numel, int64_t n, int dtype) {
  if (dtype < 0 || dtype > 2 || n < 0 || (n > 0 && (!t || !numel))) return true;
  for (int64_t j = 0; j < n; ++j)
    if (numel[j] < 0 || numel[j] > (1ll << 37) || (numel[j] > 0 && (!t[j] || t[j] % width_of(dtype)))) return true;
  return false;
}

struct Span { uint64_t begin, end; bool written; };

// True when a written tensor shares memory with another written or read one.
int overlap(const uint64_t* p, const uint64_t* g, const int64_t* numel, int64_t n, size_t width, bool* found) {
  Span* s = new (std::nothrow) Span[2 * n + 1];
  if (!s) return E2A_ERR_WORKSPACE;
  const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  int64_t k = 0, half = 0;
  for (int64_t j = 0; j < n; ++j)
    if (numel[j] > 0) s[k++] = {p[j], p[j] + (uint64_t)numel[j] * width, true};
  half = k;
  for (int64_t j = 0; j < n; ++j)
    if (numel[j] > 0) s[k++] = {g[j], g[j] + (uint64_t)numel[j] * width, false};
  // lists in the order of their addresses, as one allocation's views are, need no sort
  if (!std::is_sorted(s, s + half, before)) std::sort(s, s + half, before);
  if (!std::is_sorted(s + half, s + k, before)) std::sort(s + half, s + k, before);
  if (half < k && half > 0 && before(s[half], s[half - 1])) std::sort(s, s + k, before);
  uint64_t written = 0, any = 0;      // furthest ends so far
  *found = false;
  for (int64_t i = 0; i < k; ++i) {
    if (s[i].begin < written || (s[i].written && s[i].begin < any)) *found = true;
    any = std::max(any, s[i].end);
    if (s[i].written) written = std::max(written, s[i].end);
  }
  delete[] s;
  return E2A_OK;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == 0) return f((float*)nullptr);
  if (dtype == 1) return f((__nv_bfloat16*)nullptr);
  return f((__half*)nullptr);
}

}  // namespace

extern "C" {

size_t e2a_grad_norm_workspace_bytes(int64_t n_tensors) {
  return n_tensors <= 0 ? 0 : (size_t)((n_tensors + kTensors - 1) / kTensors + 1) * kNormCtas * sizeof(double);
}

int e2a_sum_squares(const uint64_t* tensors, const int64_t* numel, int64_t n_tensors, int dtype, void* workspace,
                    size_t workspace_bytes, int64_t* n_partials, void* stream) {
  if (bad_tensors(tensors, numel, n_tensors, dtype) || !n_partials || e2a_misaligned(8, workspace)) return E2A_ERR_ARG;
  *n_partials = 0;
  double* part = (double*)workspace;
  const int64_t room = (int64_t)(workspace_bytes / sizeof(double));
  for (int64_t j = 0; j < n_tensors;) {
    static thread_local Table t;
    int32_t units = 0;
    j = fill(&t, j, n_tensors, nullptr, tensors, numel, nullptr, &units);
    if (units == 0) continue;
    const int32_t per = (units + kNormCtas - 1) / kNormCtas, ctas = (units + per - 1) / per;
    if (!part || *n_partials + ctas > room) return E2A_ERR_WORKSPACE;
    const int rc = by_type(dtype, [&](auto* x) -> int {
      using T = std::remove_pointer_t<decltype(x)>;
      k_sum_squares<T><<<ctas, kThreads, 0, (cudaStream_t)stream>>>(t, units, per, part + *n_partials);
      E2A_CHECK_LAUNCH();
      return E2A_OK;
    });
    if (rc != E2A_OK) return rc;
    *n_partials += ctas;
  }
  return E2A_OK;
}

int e2a_norm_of_squares(const void* partials, int64_t n_partials, float* norm, void* stream) {
  if (n_partials < 0 || (n_partials > 0 && !partials) || !norm) return E2A_ERR_ARG;
  if (e2a_misaligned(8, partials) || e2a_misaligned(4, norm)) return E2A_ERR_ARG;
  k_norm<<<1, kThreads, 0, (cudaStream_t)stream>>>((const double*)partials, n_partials, norm);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
}

int e2a_grad_norm(const uint64_t* tensors, const int64_t* numel, int64_t n_tensors, int dtype, void* workspace,
                  size_t workspace_bytes, float* norm, void* stream) {
  int64_t n = 0;
  const int rc = e2a_sum_squares(tensors, numel, n_tensors, dtype, workspace, workspace_bytes, &n, stream);
  return rc == E2A_OK ? e2a_norm_of_squares(workspace, n, norm, stream) : rc;
}

size_t e2a_adamw_workspace_bytes(int64_t n_tensors) {
  return n_tensors <= 0 ? 0 : sizeof(Globals) + (size_t)n_tensors * sizeof(Scalars);
}

int e2a_adamw_step(const uint64_t* params, const uint64_t* grads, const int64_t* numel, const int64_t* state_offset,
                   const int32_t* slots, int64_t n_tensors, int dtype, int state_bits, void* exp_avg, void* exp_avg_sq,
                   uint8_t* exp_avg_scale, uint8_t* exp_avg_sq_scale, int64_t state_elements, int32_t* step, double lr,
                   const float* lr_device, double beta1, double beta2, double eps, double weight_decay,
                   const float* grad_norm, double max_norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_tensors(params, numel, n_tensors, dtype) || bad_tensors(grads, numel, n_tensors, dtype)) return E2A_ERR_ARG;
  if (state_bits != 32 && state_bits != 8) return E2A_ERR_ARG;
  if (!(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1. && eps >= 0.)) return E2A_ERR_ARG;
  if (eps > 0. && eps < 0x1p-126) return E2A_ERR_ARG;      // the kernels' reciprocal takes it for 0
  if (grad_norm && !(max_norm > 0.)) return E2A_ERR_ARG;
  if (n_tensors == 0) return E2A_OK;
  if (!state_offset || !slots || !exp_avg || !exp_avg_sq || !step || n_tensors > (1 << 24)) return E2A_ERR_ARG;
  if (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) return E2A_ERR_ARG;
  if (e2a_misaligned(state_bits == 32 ? 16 : 4, exp_avg, exp_avg_sq) ||
      e2a_misaligned(4, step, lr_device, grad_norm) || e2a_misaligned(16, workspace))
    return E2A_ERR_ARG;
  int64_t end = 0;
  for (int64_t j = 0; j < n_tensors; ++j) {
    if (state_offset[j] < end || state_offset[j] % kBlock || (j > 0 && slots[j] <= slots[j - 1]) || slots[j] < 0)
      return E2A_ERR_ARG;
    end = state_offset[j] + blocks_of(numel[j]) * kBlock;
  }
  if (end > state_elements) return E2A_ERR_ARG;
  bool shared = false;
  int rc = overlap(params, grads, numel, n_tensors, width_of(dtype), &shared);
  if (rc != E2A_OK) return rc;
  if (shared) return E2A_ERR_ARG;
  if (!workspace || workspace_bytes < e2a_adamw_workspace_bytes(n_tensors)) return E2A_ERR_WORKSPACE;
  Globals* glob = (Globals*)workspace;
  Scalars* scal = (Scalars*)(glob + 1);
  cudaStream_t st = (cudaStream_t)stream;
  const Hyper h{lr, std::log2(beta1), std::log2(beta2), weight_decay, lr_device, grad_norm, (float)max_norm};
  const Rates r{(float)beta1, (float)(1. - beta1), (float)beta2, (float)(1. - beta2), (float)eps, 1.f};
  for (int64_t j = 0; j < n_tensors;) {
    static thread_local Table t;
    static thread_local Slots slot;
    const int64_t from = j;
    int32_t units = 0;
    j = fill(&t, j, n_tensors, params, grads, numel, state_offset, &units);
    std::copy(slots + from, slots + j, slot.slot);
    k_adamw_scalars<<<1, kTensors, 0, st>>>(slot, h, step, t.n, scal + from, glob);
    E2A_CHECK_LAUNCH();
    if (units == 0) continue;
    rc = by_type(dtype, [&](auto* x) -> int {
      using T = std::remove_pointer_t<decltype(x)>;
      auto* kernel = state_bits == 32 ? k_adamw<T, 32> : k_adamw<T, 8>;
      const int32_t most = state_bits == 32 ? kStepCtas32 : kStepCtas8;
      const int32_t per = (units + most - 1) / most, ctas = (units + per - 1) / per;
      kernel<<<ctas, kThreads, 0, st>>>(t, units, per, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale,
                                        scal + from, glob, r, grad_norm != nullptr);
      E2A_CHECK_LAUNCH();
      return E2A_OK;
    });
    if (rc != E2A_OK) return rc;
  }
  return E2A_OK;
}

int e2a_moments_unpack(const uint8_t* exp_avg, const uint8_t* exp_avg_sq, const uint8_t* exp_avg_scale,
                       const uint8_t* exp_avg_sq_scale, int64_t n, float* out_avg, float* out_avg_sq, void* stream) {
  if (n < 0) return E2A_ERR_ARG;
  if (n == 0) return E2A_OK;
  if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !out_avg || !out_avg_sq) return E2A_ERR_ARG;
  if (n % kBlock || e2a_misaligned(4, exp_avg, exp_avg_sq) || e2a_misaligned(16, out_avg, out_avg_sq)) return E2A_ERR_ARG;
  const int64_t b = (n / kBlock + kThreads / 32 - 1) / (kThreads / 32);
  k_moments_unpack<<<(int)(b < 148 * 64 ? b : 148 * 64), kThreads, 0, (cudaStream_t)stream>>>(
      exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, n, out_avg, out_avg_sq);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
}

}  // extern "C"
