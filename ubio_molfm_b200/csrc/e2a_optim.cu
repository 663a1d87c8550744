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
// 8-bit moments.  The 256 values of a block share a power of two, that of the largest magnitude or the next (one
// byte, fp32's exponent field; 255 = a value was not finite, the whole block then stands for NaN).  Over it, m is a sign, 4
// exponent and 3 fraction bits, sqrt(v) 4 exponent and 4 fraction bits, with gradual underflow: the high bits
// of the fp32 pattern of |x| 2^(-e - 112), whose subnormals fall where the small format's do.  The bits below
// are dropped after adding an offset, mixed bits of (element, step), so a value is rounded up as often as it is
// near the upper neighbour: round-to-nearest would never move an average whose step is 1 - b2 = 1e-3 of itself
// (an additive sequence in place of mixed bits locks to the value that it rounds: an average that grows by 1e-3
// a step fell 6% behind in 2,000 steps).  sqrt(v) > 0 is never rounded to 0 (the update would divide by eps).
// Every operation is a single rounded fp32 one in a fixed order, so the codes are reproducible bit for bit.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <new>
#include <type_traits>

#include "e2a_common.cuh"

namespace {

constexpr int kBlock = 256;          // elements that share a scale
constexpr int kTensors = 512;        // tensors in one launch's table (18.4 KB of kernel parameters)
constexpr int kNormCtas = 592;       // partial sums of squares of one launch (4 per SM)

struct Table {
  uint64_t p[kTensors];
  uint64_t g[kTensors];
  int64_t numel[kTensors];
  int64_t offset[kTensors];
  int32_t first[kTensors + 1];       // first block of every tensor
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

// The tensor that owns block b: the last j with first[j] <= b (empty tensors own none).
__device__ __forceinline__ int tensor_of(const Table& t, int32_t b) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

// ---- 8-bit values -------------------------------------------------------------------------------
// Mixed bits of (element, step): sums and products by odd 32-bit fractions (of the powers of the root of
// x^5 = x + 1) with shifts between them.  The first moment's offset is the upper 20 bits, the second's the
// lower 19.
__device__ __forceinline__ uint32_t mixed(uint32_t i, uint32_t t) {
  uint32_t u = i * 0xDB4F0B91u + t * 0xBBE05633u;
  u = (u ^ (u >> 16)) * 0xA0F2EC75u;
  u = (u ^ (u >> 15)) * 0x89E18285u;
  return u ^ (u >> 16);
}

__device__ __forceinline__ float two_to_112() { return __uint_as_float((112u + 127u) << 23); }
__device__ __forceinline__ float two_to_m112() { return __uint_as_float((127u - 112u) << 23); }
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b == 255u ? 0x7FC00000u : b << 23); }

// The shared exponent of a block from the largest magnitude's bits (integer order is value order, NaN above):
// the next one where rounding up could pass the largest code, or a slowly growing average would stop there.
__device__ __forceinline__ uint32_t shared_exponent(uint32_t largest, int fraction) {
  if (largest >= 0x7F800000u) return 255u;
  return min(max((largest + (1u << (23 - fraction))) >> 23, 27u), 253u);
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
  return min((__float_as_uint(z) + dither) >> 20, 127u) | (m < 0.f ? 128u : 0u);
}
__device__ __forceinline__ uint32_t pack_s(float s, uint32_t b, uint32_t dither) {
  if (b == 255u) return 0u;
  const float z = __fmul_rn(__fmul_rn(s, __uint_as_float((254u - b) << 23)), two_to_m112());
  return max(min((__float_as_uint(z) + dither) >> 19, 255u), s > 0.f ? 1u : 0u);
}

// ---- the step ------------------------------------------------------------------------------------
struct Hyper {
  double lr, beta1, beta2, decay;
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
    v.size = (float)(lr / (1.0 - pow(h.beta1, (double)t)));
    v.root = (float)(1.0 / sqrt(1.0 - pow(h.beta2, (double)t)));
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

struct Moments { float p, m, v; };

// One element's update; every operation rounded on its own (see above).
__device__ __forceinline__ Moments update(float p, float g, float m, float v, const Globals& gl, const Scalars& s,
                                          float b1, float a1, float b2, float a2, float eps, bool clip) {
  if (clip) g = __fmul_rn(g, gl.coef);
  Moments o;
  o.m = __fadd_rn(__fmul_rn(m, b1), __fmul_rn(g, a1));
  o.v = __fadd_rn(__fmul_rn(v, b2), __fmul_rn(__fmul_rn(g, g), a2));
  const float d = __fadd_rn(__fmul_rn(__fsqrt_rn(o.v), s.root), eps);
  o.p = __fsub_rn(__fmul_rn(p, gl.decay), __fmul_rn(__fdiv_rn(o.m, d), s.size));
  return o;
}

template <typename T, int BITS>
__global__ void __launch_bounds__(kBlock)
k_adamw(const __grid_constant__ Table tab, int32_t n_blocks, void* __restrict__ exp_avg, void* __restrict__ exp_avg_sq,
        uint8_t* __restrict__ scale_m, uint8_t* __restrict__ scale_v, const Scalars* __restrict__ scal,
        const Globals* __restrict__ glob, float b1, float a1, float b2, float a2, float eps, bool clip) {
  __shared__ uint32_t top[2][kBlock / 32];
  const Globals gl = *glob;
  if (gl.skip) return;
  for (int32_t b = blockIdx.x; b < n_blocks; b += gridDim.x) {
    const int j = tensor_of(tab, b);
    const int64_t i = (int64_t)(b - tab.first[j]) * kBlock + threadIdx.x;
    const int64_t at = tab.offset[j] + i;
    const bool in = i < tab.numel[j];
    const Scalars s = scal[j];
    T* p = reinterpret_cast<T*>(tab.p[j]);
    const T* g = reinterpret_cast<const T*>(tab.g[j]);
    if (BITS == 32) {
      if (!in) continue;
      float* m = (float*)exp_avg;
      float* v = (float*)exp_avg_sq;
      const Moments o = update(to_f(p[i]), to_f(g[i]), m[at], v[at], gl, s, b1, a1, b2, a2, eps, clip);
      p[i] = from_f<T>(o.p);
      m[at] = o.m;
      v[at] = o.v;
    } else {
      uint8_t* m = (uint8_t*)exp_avg;
      uint8_t* v = (uint8_t*)exp_avg_sq;
      Moments o{0.f, 0.f, 0.f};
      float sv = 0.f;
      if (in) {
        const float r = unpack_s(v[at], scale_of(scale_v[at / kBlock]));
        o = update(to_f(p[i]), to_f(g[i]), unpack_m(m[at], scale_of(scale_m[at / kBlock])), __fmul_rn(r, r), gl, s, b1,
                   a1, b2, a2, eps, clip);
        p[i] = from_f<T>(o.p);
        sv = __fsqrt_rn(o.v);
      }
      const uint32_t lm = __reduce_max_sync(0xffffffffu, __float_as_uint(o.m) & 0x7FFFFFFFu);
      const uint32_t lv = __reduce_max_sync(0xffffffffu, __float_as_uint(sv) & 0x7FFFFFFFu);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) {
        top[0][threadIdx.x >> 5] = lm;
        top[1][threadIdx.x >> 5] = lv;
      }
      __syncthreads();
      uint32_t em = 0, ev = 0;
      for (int w = 0; w < kBlock / 32; ++w) {
        em = max(em, top[0][w]);
        ev = max(ev, top[1][w]);
      }
      em = shared_exponent(em, 3);
      ev = shared_exponent(ev, 4);
      if (in) {
        const uint32_t u = mixed((uint32_t)i, (uint32_t)s.t);
        m[at] = (uint8_t)pack_m(o.m, em, u >> 12);
        v[at] = (uint8_t)pack_s(sv, ev, u & 0x7FFFFu);
      }
      if (threadIdx.x == 0) {
        scale_m[at / kBlock] = (uint8_t)em;
        scale_v[at / kBlock] = (uint8_t)ev;
      }
    }
  }
}

__global__ void k_moments_unpack(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                 const uint8_t* __restrict__ scale_m, const uint8_t* __restrict__ scale_v, int64_t n,
                                 float* __restrict__ out_m, float* __restrict__ out_v) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    out_m[i] = unpack_m(m[i], scale_of(scale_m[i / kBlock]));
    const float s = unpack_s(v[i], scale_of(scale_v[i / kBlock]));
    out_v[i] = __fmul_rn(s, s);
  }
}

// ---- the global norm -------------------------------------------------------------------------------
// Squares are exact in 64 bits and summed there: the norm is the correctly rounded one but for ties.
template <typename T>
__global__ void __launch_bounds__(kBlock)
k_sum_squares(const __grid_constant__ Table tab, int32_t n_blocks, double* __restrict__ part) {
  __shared__ double sh[kBlock / 32];
  double s = 0.;
  for (int32_t b = blockIdx.x; b < n_blocks; b += gridDim.x) {
    const int j = tensor_of(tab, b);
    const int64_t i = (int64_t)(b - tab.first[j]) * kBlock + threadIdx.x;
    if (i < tab.numel[j]) {
      const double g = (double)to_f(reinterpret_cast<const T*>(tab.g[j])[i]);
      s += g * g;
    }
  }
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBlock / 32; ++w) s += sh[w];
    part[blockIdx.x] = s;
  }
}

__global__ void k_norm(const double* __restrict__ part, int64_t n, float* __restrict__ norm) {
  __shared__ double sh[kBlock / 32];
  double s = 0.;
  for (int64_t i = threadIdx.x; i < n; i += kBlock) s += part[i];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBlock / 32; ++w) s += sh[w];
    *norm = (float)sqrt(s);
  }
}

int64_t blocks_of(int64_t numel) { return (numel + kBlock - 1) / kBlock; }

size_t width_of(int dtype) { return dtype == 0 ? 4 : 2; }

// Fills a launch's table with tensors [from, ...): as many as fit.  Returns the next tensor, blocks in *n_blocks.
int64_t fill(Table* t, int64_t from, int64_t n_tensors, const uint64_t* p, const uint64_t* g, const int64_t* numel,
             const int64_t* offset, int32_t* n_blocks) {
  int64_t blocks = 0, j = from;
  int k = 0;
  for (; j < n_tensors && k < kTensors; ++j, ++k) {
    const int64_t nb = blocks_of(numel[j]);
    if (k > 0 && blocks + nb > (1ll << 30)) break;
    t->p[k] = p ? p[j] : 0;
    t->g[k] = g[j];
    t->numel[k] = numel[j];
    t->offset[k] = offset ? offset[j] : 0;
    t->first[k] = (int32_t)blocks;
    blocks += nb;
  }
  t->first[k] = (int32_t)blocks;
  t->n = k;
  *n_blocks = (int32_t)blocks;
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
  int64_t k = 0;
  for (int64_t j = 0; j < n; ++j) {
    if (numel[j] == 0) continue;
    s[k++] = {p[j], p[j] + (uint64_t)numel[j] * width, true};
    s[k++] = {g[j], g[j] + (uint64_t)numel[j] * width, false};
  }
  std::sort(s, s + k, [](const Span& a, const Span& b) { return a.begin < b.begin; });
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

int grid_of(int32_t n_blocks) { return n_blocks < 148 * 8 ? n_blocks : 148 * 8; }

}  // namespace

extern "C" {

size_t e2a_grad_norm_workspace_bytes(int64_t n_tensors) {
  return n_tensors <= 0 ? 0 : (size_t)((n_tensors + kTensors - 1) / kTensors + 1) * kNormCtas * sizeof(double);
}

int e2a_sum_squares(const uint64_t* tensors, const int64_t* numel, int64_t n_tensors, int dtype, void* workspace,
                    size_t workspace_bytes, int64_t* n_partials, void* stream) {
  if (bad_tensors(tensors, numel, n_tensors, dtype) || !n_partials) return E2A_ERR_ARG;
  *n_partials = 0;
  double* part = (double*)workspace;
  const int64_t room = (int64_t)(workspace_bytes / sizeof(double));
  for (int64_t j = 0; j < n_tensors;) {
    static thread_local Table t;
    int32_t blocks = 0;
    j = fill(&t, j, n_tensors, nullptr, tensors, numel, nullptr, &blocks);
    if (blocks == 0) continue;
    const int ctas = blocks < kNormCtas ? blocks : kNormCtas;
    if (!part || *n_partials + ctas > room) return E2A_ERR_WORKSPACE;
    const int rc = by_type(dtype, [&](auto* x) -> int {
      using T = std::remove_pointer_t<decltype(x)>;
      k_sum_squares<T><<<ctas, kBlock, 0, (cudaStream_t)stream>>>(t, blocks, part + *n_partials);
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
  k_norm<<<1, kBlock, 0, (cudaStream_t)stream>>>((const double*)partials, n_partials, norm);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
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
  if (grad_norm && !(max_norm > 0.)) return E2A_ERR_ARG;
  if (n_tensors == 0) return E2A_OK;
  if (!state_offset || !slots || !exp_avg || !exp_avg_sq || !step || n_tensors > (1 << 24)) return E2A_ERR_ARG;
  if (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) return E2A_ERR_ARG;
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
  const Hyper h{lr, beta1, beta2, weight_decay, lr_device, grad_norm, (float)max_norm};
  const float b1 = (float)beta1, a1 = (float)(1. - beta1), b2 = (float)beta2, a2 = (float)(1. - beta2);
  for (int64_t j = 0; j < n_tensors;) {
    static thread_local Table t;
    static thread_local Slots slot;
    const int64_t from = j;
    int32_t blocks = 0;
    j = fill(&t, j, n_tensors, params, grads, numel, state_offset, &blocks);
    std::copy(slots + from, slots + j, slot.slot);
    k_adamw_scalars<<<1, kTensors, 0, st>>>(slot, h, step, t.n, scal + from, glob);
    E2A_CHECK_LAUNCH();
    if (blocks == 0) continue;
    rc = by_type(dtype, [&](auto* x) -> int {
      using T = std::remove_pointer_t<decltype(x)>;
      auto* kernel = state_bits == 32 ? k_adamw<T, 32> : k_adamw<T, 8>;
      kernel<<<grid_of(blocks), kBlock, 0, st>>>(t, blocks, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale,
                                                 scal + from, glob, b1, a1, b2, a2, (float)eps, grad_norm != nullptr);
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
  const int64_t b = blocks_of(n);
  k_moments_unpack<<<(int)(b < 148 * 32 ? b : 148 * 32), kBlock, 0, (cudaStream_t)stream>>>(
      exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, n, out_avg, out_avg_sq);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
}

}  // extern "C"
