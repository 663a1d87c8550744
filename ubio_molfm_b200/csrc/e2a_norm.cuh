// Layer norm with an optional SiLU over rows of W values (nn.LayerNorm followed by nn.SiLU in the radial
// and scalar MLPs, module_utils.py:2151-2178, 2240-2274), as training needs it: the weight's and bias's
// gradients, and the backward of the backward that a loss on forces asks for.
//
//   xh = (x - mean) r,  r = (var + eps)^-1/2,  z = w xh + b,  y = act(z)            (biased variance)
//   backward        a = g act'(z),  h = a w,  dx = r (h - <h> - xh <h xh>)           (<.> = row mean)
//                   dw = sum_rows a xh,  db = sum_rows a
//   second order, for cotangents u of dx, p of dw and q of db:
//                   c = <u xh>,  t = r (u - <u> - xh c)        (the norm's Jacobian, symmetric, times u)
//                   v = w t + p xh + q,  e = g act''(z) v
//                   dg = act'(z) v,  k = e w + a p - r (u <h xh> + h c)
//                   dx = r (k - <k> - xh <k xh> - xh <h t>),  dw = sum a t + e xh,  db = sum e
//
// All of it is bound by memory once the arithmetic is packed and the exponential the special function unit's: the
// forward moves 2 values an element, the backward 3, the second order 5.  640,210 x 128 fp32 (328 MB an operand):
// 102, 164 and 244 us, that is 6.4, 6.0 and 6.7 TB/s where a copy runs at 6.5; 97,865 x 512 fp32: 66 and 94 us;
// 16,384 x 4,096 bf16 without activation: 49 and 83 us (5.4 and 4.9 TB/s: one row a CTA, its sums behind barriers).
//
// The statistics are two-pass in fp32, of the differences to the row's first value, and kept per row.  Column sums: a thread's own rows in fp32 chains of at most
// 128, which join the CTA's partial rows in memory; those are added up in CTA order in 64 bits.  No atomics.  Rows
// of more than 8,192 values take loops over memory (first part below), whose sums are in 64 bits throughout.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "e2a_common.cuh"

namespace {

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// SiLU and its first two derivatives: s = 1 / (1 + exp(-z)), y = z s, y' = s (1 + z (1 - s)),
// y'' = s (1 - s) (2 + z (1 - 2 s)).  Without activation 1 and 0.  The exponential and the reciprocal are the
// special function unit's (s within about 2e-7): with expf and a division the forward was bound by them, 212 us
// on 640,210 x 128 fp32 where its bytes take 100, and is at 102 like this.
struct Act { float y, d1, d2; };
__device__ __forceinline__ Act activation(float z, bool silu) {
  if (!silu) return {z, 1.f, 0.f};
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return {z * s, s * (1.f + z * (1.f - s)), s * (1.f - s) * (2.f + z * (1.f - 2.f * s))};
}

// The same of two neighbouring values in packed fp32 arithmetic.
__device__ __forceinline__ float2 sigmoid(float2 z) {
  const float2 t = f2_mul(z, f2(-1.44269504f));
  float2 e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  e = f2_add(e, f2(1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
  return s;
}
struct Act2 { float2 d1, d2; };
template <bool SILU, bool SECOND>
__device__ __forceinline__ Act2 derivatives(float2 z) {
  if (!SILU) return {f2(1.f), f2(0.f)};
  const float2 s = sigmoid(z), rest = f2_fma(s, f2(-1.f), f2(1.f));
  Act2 a;
  a.d1 = f2_mul(s, f2_fma(z, rest, f2(1.f)));
  a.d2 = SECOND ? f2_mul(f2_mul(s, rest), f2_fma(z, f2_fma(s, f2(-2.f), f2(1.f)), f2(2.f))) : f2(0.f);
  return a;
}

struct Norm {
  const float* gamma;  // NULL = 1
  const float* beta;   // NULL = 0
  const float* p;      // cotangents of dw and db (second order; NULL = 0)
  const float* q;
  int64_t W;
  bool silu;
};

__device__ __forceinline__ float at(const float* v, int64_t c, float without) { return v ? __ldg(v + c) : without; }

// Means over a row's columns, by a warp: f(c, p) adds column c's terms to p.  AT_ONCE of them (a few at the row's end) add
// up in fp32, the rest in 64 bits.
template <int AT_ONCE, int K, typename F>
__device__ __forceinline__ void row_means(int64_t W, double (&mean)[K], F f) {
#pragma unroll
  for (int k = 0; k < K; ++k) mean[k] = 0.;
  int64_t c = threadIdx.x & 31;
  for (; c + 32 * (AT_ONCE - 1) < W; c += 32 * AT_ONCE) {
    float p[K] = {};
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) f(c + 32 * j, p);
#pragma unroll
    for (int k = 0; k < K; ++k) mean[k] += p[k];
  }
  float p[K] = {};
  for (; c < W; c += 32) f(c, p);
#pragma unroll
  for (int k = 0; k < K; ++k) mean[k] += p[k];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mean[k] += __shfl_xor_sync(0xffffffffu, mean[k], o);
    mean[k] /= W;
  }
}

template <typename T>
__global__ void k_ln_fwd(const T* __restrict__ x, int64_t ldx, Norm n, int64_t rows, float eps, T* __restrict__ y,
                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  const int lane = threadIdx.x & 31;
  const int64_t nw = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t r = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; r < rows; r += nw) {
    const T* xr = x + r * ldx;
    const float x0 = to_f(xr[0]);      // see k_row_fwd
    double shift[1], var[1];
    row_means<8>(n.W, shift, [&](int64_t c, float* p) { p[0] += to_f(xr[c]) - x0; });
    const float by = (float)shift[0], mean = x0 + by;
    row_means<8>(n.W, var, [&](int64_t c, float* p) {
      const float d = (to_f(xr[c]) - x0) - by;
      p[0] = fmaf(d, d, p[0]);
    });
    const float rstd = (float)rsqrt(var[0] + eps);
    for (int64_t c = lane; c < n.W; c += 32) {
      const float z = ((to_f(xr[c]) - x0) - by) * rstd * at(n.gamma, c, 1.f) + at(n.beta, c, 0.f);
      y[r * n.W + c] = from_f<T>(activation(z, n.silu).y);
    }
    if (lane == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

template <typename T>
__global__ void k_ln_bwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ g, int64_t ldg, Norm n,
                         const float* __restrict__ mean_in, const float* __restrict__ rstd_in, int64_t rows,
                         T* __restrict__ dx) {
  const int lane = threadIdx.x & 31;
  const int64_t nw = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t r = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; r < rows; r += nw) {
    const T* xr = x + r * ldx;
    const T* gr = g + r * ldg;
    const float mean = mean_in[r], rstd = rstd_in[r];
    double m[2];
    row_means<4>(n.W, m, [&](int64_t c, float* p) {
      const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd;
      const float h = to_f(gr[c]) * activation(xh * w + at(n.beta, c, 0.f), n.silu).d1 * w;
      p[0] += h;
      p[1] = fmaf(h, xh, p[1]);
    });
    const float s1 = (float)m[0], s2 = (float)m[1];
    for (int64_t c = lane; c < n.W; c += 32) {
      const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd;
      const float h = to_f(gr[c]) * activation(xh * w + at(n.beta, c, 0.f), n.silu).d1 * w;
      dx[r * n.W + c] = from_f<T>(rstd * (h - s1 - xh * s2));
    }
  }
}

template <typename T>
__global__ void k_ln_bwd2(const T* __restrict__ x, int64_t ldx, const T* __restrict__ g, int64_t ldg,
                          const T* __restrict__ u, int64_t ldu, Norm n, const float* __restrict__ mean_in,
                          const float* __restrict__ rstd_in, int64_t rows, T* __restrict__ dg, T* __restrict__ dx,
                          float* __restrict__ row_u, float* __restrict__ row_c) {
  const int lane = threadIdx.x & 31;
  const int64_t nw = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t r = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; r < rows; r += nw) {
    const T* xr = x + r * ldx;
    const T* gr = g + r * ldg;
    const T* ur = u + r * ldu;
    const float mean = mean_in[r], rstd = rstd_in[r];
    double m[5], e[2];
    row_means<4>(n.W, m, [&](int64_t c, float* p) {
      const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd, uv = to_f(ur[c]);
      const float h = to_f(gr[c]) * activation(xh * w + at(n.beta, c, 0.f), n.silu).d1 * w;
      p[0] += uv;
      p[1] = fmaf(uv, xh, p[1]);
      p[2] += h;
      p[3] = fmaf(h, xh, p[3]);
      p[4] = fmaf(h, uv, p[4]);
    });
    const float su = (float)m[0], sc = (float)m[1], s2 = (float)m[3];
    const double ht = rstd * (m[4] - m[2] * m[0] - m[3] * m[1]);
    // one column's dg and k
    const auto column = [&](int64_t c, float* xh, float* dgv) {
      *xh = (to_f(xr[c]) - mean) * rstd;
      const float w = at(n.gamma, c, 1.f), uv = to_f(ur[c]), gv = to_f(gr[c]);
      const Act a = activation(*xh * w + at(n.beta, c, 0.f), n.silu);
      const float pc = at(n.p, c, 0.f), t = rstd * (uv - su - *xh * sc);
      const float v = w * t + pc * *xh + at(n.q, c, 0.f);
      const float ga = gv * a.d1;
      *dgv = a.d1 * v;
      return gv * a.d2 * v * w + ga * pc - rstd * (uv * s2 + ga * w * sc);
    };
    row_means<2>(n.W, e, [&](int64_t c, float* p) {
      float xh, dgv;
      const float k = column(c, &xh, &dgv);
      p[0] += k;
      p[1] = fmaf(k, xh, p[1]);
    });
    const float k1 = (float)e[0], k2 = (float)(e[1] + ht);
    for (int64_t c = lane; c < n.W; c += 32) {
      float xh, dgv;
      const float k = column(c, &xh, &dgv);
      dg[r * n.W + c] = from_f<T>(dgv);
      dx[r * n.W + c] = from_f<T>(rstd * (k - k1 - xh * k2));
    }
    if (lane == 0) {
      row_u[r] = su;
      row_c[r] = sc;
    }
  }
}

// Column sums of one chunk of rows: [chunk][2][W] in 64 bits.  Thread (col, y): rows y, y + 8, ... .
template <typename T, bool SECOND>
__global__ void k_ln_cols(const T* __restrict__ x, int64_t ldx, const T* __restrict__ g, int64_t ldg,
                          const T* __restrict__ u, int64_t ldu, Norm n, const float* __restrict__ mean_in,
                          const float* __restrict__ rstd_in, const float* __restrict__ row_u,
                          const float* __restrict__ row_c, int64_t rows, int64_t chunk_rows,
                          double* __restrict__ part) {
  __shared__ double sh[2][8][32];
  const int64_t c = blockIdx.x * (int64_t)32 + threadIdx.x;
  const int64_t r0 = blockIdx.y * chunk_rows, r1 = min(rows, r0 + chunk_rows);
  double sw = 0., sb = 0.;
  if (c < n.W) {
    const float w = at(n.gamma, c, 1.f), b = at(n.beta, c, 0.f), pc = at(n.p, c, 0.f), qc = at(n.q, c, 0.f);
    for (int64_t r = r0 + threadIdx.y; r < r1; r += 8) {
      const float xh = (to_f(x[r * ldx + c]) - mean_in[r]) * rstd_in[r], gv = to_f(g[r * ldg + c]);
      const Act a = activation(xh * w + b, n.silu);
      if (SECOND) {
        const float t = rstd_in[r] * (to_f(u[r * ldu + c]) - row_u[r] - xh * row_c[r]);
        const float e = gv * a.d2 * (w * t + pc * xh + qc);
        sw += gv * a.d1 * t + e * xh;
        sb += e;
      } else {
        sw += gv * a.d1 * xh;
        sb += gv * a.d1;
      }
    }
  }
  sh[0][threadIdx.y][threadIdx.x] = sw;
  sh[1][threadIdx.y][threadIdx.x] = sb;
  __syncthreads();
  if (threadIdx.y < 2 && c < n.W) {
    double s = 0.;
    for (int i = 0; i < 8; ++i) s += sh[threadIdx.y][i][threadIdx.x];
    part[(blockIdx.y * 2 + threadIdx.y) * n.W + c] = s;
  }
}

__global__ void k_ln_cols_sum(const double* __restrict__ part, int64_t chunks, int64_t W, float* __restrict__ dw,
                              float* __restrict__ db) {
  const int64_t c = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (c >= 2 * W) return;
  float* out = c < W ? dw : db;
  if (!out) return;
  double s = 0.;
  for (int64_t i = 0; i < chunks; ++i) s += part[i * 2 * W + c];
  out[c < W ? c : c - W] = (float)s;
}

// ------------------------------------------------------------------------------------------------
// Rows in registers.  A team of TEAM threads holds a row, VEC neighbouring values (16 bytes, or one where the
// strides or addresses allow no more) V times a thread; the next row's loads are issued before the current one is
// worked on, so they are in flight all the time.  Teams of at most a warp share a CTA of 256 threads and meet only
// in shuffles; wider rows take a CTA each.
// ------------------------------------------------------------------------------------------------
template <typename T, int VEC> struct Pack;
template <> struct Pack<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ void widen(const Raw& t, float* v) {
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  }
  static __device__ __forceinline__ Raw narrow(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }
};
template <typename T, typename T2> struct Pack16 {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const Raw& t, float* v) {
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T2 h = *reinterpret_cast<const T2*>(&w[i]);
      v[2 * i] = to_f(h.x);
      v[2 * i + 1] = to_f(h.y);
    }
  }
  static __device__ __forceinline__ Raw narrow(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T2 h;
      h.x = from_f<T>(v[2 * i]);
      h.y = from_f<T>(v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Pack<__nv_bfloat16, 8> : Pack16<__nv_bfloat16, __nv_bfloat162> {};
template <> struct Pack<__half, 8> : Pack16<__half, __half2> {};
template <typename T> struct Pack<T, 1> {
  using Raw = T;
  static __device__ __forceinline__ void widen(const Raw& t, float* v) { v[0] = to_f(t); }
  static __device__ __forceinline__ Raw narrow(const float* v) { return from_f<T>(v[0]); }
};

// fp32 vectors of the affine parameters: VEC at a time in 16-byte loads (they come from fresh or parameter
// allocations; the host checks), without them the constant.
template <int VEC>
__device__ __forceinline__ void load_affine(const float* p, int c, float without, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = without;
  } else if (VEC == 1) {
    v[0] = __ldg(p + c);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      const float4 t = ldg4(p + c + k);
      v[k] = t.x; v[k + 1] = t.y; v[k + 2] = t.z; v[k + 3] = t.w;
    }
  }
}

// Sums over a team of N values a thread; every thread of the team gets them.  CTA-wide teams alternate between
// two halves of `sh`, so one barrier a sum is enough.
template <int TEAM, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* sh, int& turn) {
#pragma unroll
  for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if (TEAM > 32) {
    constexpr int WARPS = TEAM / 32;
    float* half = sh + turn * WARPS * 5;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) half[i * WARPS + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += half[i * WARPS + w];
      v[i] = s;
    }
  }
}

template <typename T_, int VEC_, int V_, int TEAM_>
struct Shape {
  using T = T_;
  using P = Pack<T, VEC_>;
  static constexpr int VEC = VEC_, V = V_, TEAM = TEAM_;
  static constexpr int THREADS = TEAM > 32 ? TEAM : 256;
  static constexpr int TEAMS = THREADS / TEAM;   // rows that a CTA holds at a time
  static constexpr int N = VEC * V;
  // vectors of a thread that are never beyond the row's end: by_shape takes every shape but the narrowest (a single
  // vector, or four single values in a team of 8) for rows that fill more than half of it
  static constexpr int SURE = VEC == 1 && TEAM == 8 ? 0 : V / 2;
  // those of them that are loaded and stored without asking (150,000 x 262 fp32 second order 275 -> 243 us, 8,192 x 8,192
  // bf16 454 -> 388 us; in narrower shapes of 16-byte vectors the registers fall worse: 16,384 x 4,096 bf16 157 -> 230 us)
  static constexpr int UNASKED = VEC == 1 || TEAM == 512 ? SURE : 0;
  static constexpr int SCRATCH = TEAM > 32 ? 2 * 5 * (TEAM / 32) : 1;                    // team_sum
};

// The rows a thread works on, of K operands at once, one row ahead of their use in registers.  (Two to four rows
// ahead in shared memory by asynchronous copies took 3 to 15% longer at every shape tried.)
template <class S, int K>
struct Rows {
  using T = typename S::T;
  using Raw = typename S::P::Raw;
  const T* p[K];
  int64_t ld[K], rows, step;
  int W;
  Raw next[K][S::V];

  __device__ __forceinline__ void load(int64_t row) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < S::V; ++i) {
        const int c = (threadIdx.x % S::TEAM + S::TEAM * i) * S::VEC;
        next[k][i] = row < rows && (i < S::UNASKED || c < W) ? __ldg(reinterpret_cast<const Raw*>(p[k] + row * ld[k] + c)) : Raw{};
      }
    }
  }
  // The values of `row` (zero beyond the rows' and the row's end), the next row's on their way.
  __device__ __forceinline__ void take(int64_t row, float (&v)[K][S::N]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < S::V; ++i) S::P::widen(next[k][i], v[k] + i * S::VEC);
    }
    load(row + step);
  }
};

// A thread's values as pairs.  The vectors' own pairs with 16-byte loads, neighbours of its V single ones without.
#define E2A_PAIR(v, e) (reinterpret_cast<float2*>(v)[e])

// gamma, beta, p, q at a thread's columns, `without` beyond the row's end too.
template <class S>
__device__ __forceinline__ void columns(const float* p, int W, float without, float (&v)[S::N]) {
#pragma unroll
  for (int i = 0; i < S::V; ++i) {
    const int c = (threadIdx.x % S::TEAM + S::TEAM * i) * S::VEC;
    load_affine<S::VEC>(i < S::UNASKED || c < W ? p : nullptr, c, without, v + i * S::VEC);
  }
}

// Sets a thread's values beyond the row's end.
template <class S>
__device__ __forceinline__ void fill_beyond(float (&v)[S::N], int W, float value) {
#pragma unroll
  for (int i = S::SURE; i < S::V; ++i) {
    if (((int)(threadIdx.x % S::TEAM) + S::TEAM * i) * S::VEC >= W) {
#pragma unroll
      for (int k = 0; k < S::VEC; ++k) v[i * S::VEC + k] = value;
    }
  }
}

template <class S, bool SILU>
__global__ void __launch_bounds__(S::THREADS)
k_row_fwd(const typename S::T* __restrict__ x, int64_t ldx, Norm n, int64_t rows, float eps,
          typename S::T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  using Raw = typename S::P::Raw;
  __shared__ float sh[S::SCRATCH];
  int turn = 0;
  const int me = threadIdx.x % S::TEAM, W = (int)n.W;
  const int64_t step = gridDim.x * (int64_t)S::TEAMS;
  const float inv = 1.f / W;
  int64_t row = blockIdx.x * (int64_t)S::TEAMS + threadIdx.x / S::TEAM;
  Rows<S, 1> in{{x}, {ldx}, rows, step, W};
  in.load(row);
  // The statistics are those of the differences to the row's first value, which are exact for values near each other:
  // no error grows with the mean, and a row of one value, whatever it is, has variance 0.
  typename S::T first{};
  if (S::TEAM > 32 && row < rows) first = __ldg(x + row * ldx);
  for (int64_t base = blockIdx.x * (int64_t)S::TEAMS; base < rows; base += step, row += step) {
    alignas(8) float v[1][S::N];
    in.take(row, v);
    float x0;
    if (S::TEAM > 32) {
      x0 = to_f(first);
      if (row + step < rows) first = __ldg(x + (row + step) * ldx);
    } else {
      x0 = __shfl_sync(0xffffffffu, v[0][0], 0, S::TEAM < 32 ? S::TEAM : 32);
    }
    fill_beyond<S>(v[0], W, x0);
    float2 two = f2(0.f);
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      E2A_PAIR(v[0], e) = f2_add(E2A_PAIR(v[0], e), f2(-x0));
      two = f2_add(two, E2A_PAIR(v[0], e));
    }
    float sum[1] = {two.x + two.y};
    team_sum<S::TEAM>(sum, sh, turn);
    const float shift = sum[0] * inv, mean = x0 + shift;
    fill_beyond<S>(v[0], W, shift);
    two = f2(0.f);
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      E2A_PAIR(v[0], e) = f2_add(E2A_PAIR(v[0], e), f2(-shift));
      two = f2_fma(E2A_PAIR(v[0], e), E2A_PAIR(v[0], e), two);
    }
    sum[0] = two.x + two.y;
    constexpr bool EARLY = S::TEAM > 32 || S::N <= 8;     // beside the sum, where registers allow
    alignas(8) float ga[S::N], be[S::N];
    if (EARLY) {
      columns<S>(n.gamma, W, 1.f, ga);
      columns<S>(n.beta, W, 0.f, be);
    }
    team_sum<S::TEAM>(sum, sh, turn);
    const float rstd = rsqrtf(sum[0] * inv + eps);
    if (row >= rows) continue;      // a team of a warp or less: the others go on; a CTA's rows all exist
    if (me == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    if (!EARLY) {
      columns<S>(n.gamma, W, 1.f, ga);
      columns<S>(n.beta, W, 0.f, be);
    }
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      const float2 z = f2_fma(f2_mul(E2A_PAIR(v[0], e), f2(rstd)), E2A_PAIR(ga, e), E2A_PAIR(be, e));
      E2A_PAIR(v[0], e) = SILU ? f2_mul(z, sigmoid(z)) : z;
    }
#pragma unroll
    for (int i = 0; i < S::V; ++i) {
      const int c = (me + S::TEAM * i) * S::VEC;
      if (i < S::UNASKED || c < W) *reinterpret_cast<Raw*>(y + row * W + c) = S::P::narrow(v[0] + i * S::VEC);
    }
  }
}

// Adds the column sums that the CTA's threads hold to its partial rows part[2][W], and clears them.
template <class S>
__device__ __forceinline__ void flush_cols(float (&dw)[S::N], float (&db)[S::N], float* __restrict__ part, int W,
                                           bool first, float* sh) {
  const int me = threadIdx.x % S::TEAM;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&d)[S::N] = which ? db : dw;
    float* out = part + which * W;
    if (S::TEAM > 32) {
#pragma unroll
      for (int i = 0; i < S::V; ++i) {
#pragma unroll
        for (int k = 0; k < S::VEC; ++k) {
          const int c = (me + S::TEAM * i) * S::VEC + k;
          if (c < W) out[c] = first ? d[i * S::VEC + k] : out[c] + d[i * S::VEC + k];
        }
      }
    } else {
#pragma unroll
      for (int o = 16; o >= S::TEAM; o >>= 1) {
#pragma unroll
        for (int k = 0; k < S::N; ++k) d[k] += __shfl_xor_sync(0xffffffffu, d[k], o);
      }
      constexpr int WARPS = S::THREADS / 32, COLS = S::TEAM * S::N;
      __syncthreads();
      if ((threadIdx.x & 31) < S::TEAM) {
#pragma unroll
        for (int i = 0; i < S::V; ++i) {
#pragma unroll
          for (int k = 0; k < S::VEC; ++k)
            sh[(threadIdx.x >> 5) * COLS + (me + S::TEAM * i) * S::VEC + k] = d[i * S::VEC + k];
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < W; c += S::THREADS) {
        float s = first ? 0.f : out[c];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += sh[w * COLS + c];
        out[c] = s;
      }
    }
#pragma unroll
    for (int k = 0; k < S::N; ++k) d[k] = 0.f;
  }
}

constexpr int kChain = 128;   // rows that a thread adds up in fp32 before its sums join the partial rows

// The statistics of the row after next, loaded ahead.
struct Stats {
  float mean, rstd;
  __device__ __forceinline__ void load(const float* mean_in, const float* rstd_in, int64_t row, int64_t rows) {
    mean = row < rows ? __ldg(mean_in + row) : 0.f;
    rstd = row < rows ? __ldg(rstd_in + row) : 0.f;
  }
};

// Pair e of a row's normalised values, from x: 0 beyond the row's end, where x counts as 0 and mean rstd can pass fp32's
// range (a row of one huge value).  There the mean is taken for 0 (MEAN) or the result; which of them costs registers
// differs: 640,210 x 128 fp32 second order 256 against 265 us, 16,384 x 4,096 bf16 backward 105 against 92 us.
template <class S, bool MEAN>
__device__ __forceinline__ float2 normalised(float2 x, int e, int W, const Stats& st) {
  float2 less = f2(-st.mean);
  bool beyond[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = (2 * e + k) / S::VEC;
    beyond[k] = i >= S::SURE && ((int)(threadIdx.x % S::TEAM) + S::TEAM * i) * S::VEC >= W;
    if (MEAN && beyond[k]) (k ? less.y : less.x) = 0.f;
  }
  float2 xh = f2_mul(f2_add(x, less), f2(st.rstd));
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!MEAN && beyond[k]) (k ? xh.y : xh.x) = 0.f;
  }
  return xh;
}

// part NULL: dx alone; dx NULL: the column sums alone.  Beyond a row's end g is 0: so are a and h.
template <class S, bool SILU>
__global__ void __launch_bounds__(S::THREADS, 512 / S::THREADS)
k_row_bwd(const typename S::T* __restrict__ x, int64_t ldx, const typename S::T* __restrict__ g, int64_t ldg, Norm n,
          const float* __restrict__ mean_in, const float* __restrict__ rstd_in, int64_t rows,
          typename S::T* __restrict__ dx, float* __restrict__ part) {
  using Raw = typename S::P::Raw;
  __shared__ float sh[S::TEAM > 32 ? S::SCRATCH : S::THREADS / 32 * S::TEAM * S::N];
  int turn = 0;
  const int me = threadIdx.x % S::TEAM, W = (int)n.W;
  const int64_t step = gridDim.x * (int64_t)S::TEAMS;
  const float inv = 1.f / W;
  alignas(8) float dw[S::N], db[S::N];
#pragma unroll
  for (int k = 0; k < S::N; ++k) dw[k] = db[k] = 0.f;
  int held = 0;
  bool first = true;
  if (part) part += blockIdx.x * (int64_t)(2 * W);
  int64_t row = blockIdx.x * (int64_t)S::TEAMS + threadIdx.x / S::TEAM;
  Rows<S, 2> operands{{x, g}, {ldx, ldg}, rows, step, W};
  operands.load(row);
  Stats next;
  next.load(mean_in, rstd_in, row, rows);
  for (int64_t base = blockIdx.x * (int64_t)S::TEAMS; base < rows; base += step, row += step) {
    alignas(8) float v[2][S::N], ga[S::N], be[S::N];
    operands.take(row, v);
    const Stats st = next;
    next.load(mean_in, rstd_in, row + step, rows);
    columns<S>(n.gamma, W, 0.f, ga);
    if (SILU) columns<S>(n.beta, W, 0.f, be);
    if (!n.gamma) {
#pragma unroll
      for (int k = 0; k < S::N; ++k) ga[k] = 1.f;
    }
    float2 s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      float2 &xh = E2A_PAIR(v[0], e), &h = E2A_PAIR(v[1], e);
      xh = normalised<S, false>(xh, e, W, st);
      if (SILU) h = f2_mul(h, derivatives<SILU, false>(f2_fma(xh, E2A_PAIR(ga, e), E2A_PAIR(be, e))).d1);
      E2A_PAIR(dw, e) = f2_fma(h, xh, E2A_PAIR(dw, e));
      E2A_PAIR(db, e) = f2_add(h, E2A_PAIR(db, e));
      h = f2_mul(h, E2A_PAIR(ga, e));
      s1 = f2_add(s1, h);
      s2 = f2_fma(h, xh, s2);
    }
    if (dx) {
      float sums[2] = {s1.x + s1.y, s2.x + s2.y};
      team_sum<S::TEAM>(sums, sh, turn);
      const float2 m1 = f2(-sums[0] * inv * st.rstd), m2 = f2(-sums[1] * inv * st.rstd);
#pragma unroll
      for (int e = 0; e < S::N / 2; ++e)
        E2A_PAIR(v[1], e) = f2_fma(E2A_PAIR(v[1], e), f2(st.rstd), f2_fma(E2A_PAIR(v[0], e), m2, m1));
#pragma unroll
      for (int i = 0; i < S::V; ++i) {
        const int c = (me + S::TEAM * i) * S::VEC;
        if (row < rows && (i < S::UNASKED || c < W)) *reinterpret_cast<Raw*>(dx + row * W + c) = S::P::narrow(v[1] + i * S::VEC);
      }
    }
    if (part && ++held == kChain) {
      flush_cols<S>(dw, db, part, W, first, sh);
      first = false;
      held = 0;
    }
  }
  if (part && (held || first)) flush_cols<S>(dw, db, part, W, first, sh);
}

// Second order.  With B = r act', C = r g act'' w and d = u - <u> - xh c (t = r d):  dg = B w d (+ act' (p xh + q)),
// e = C d,  dw = sum g B d + e xh,  k = w (e - c g B) - r <h xh> u; p and q join v = w t + p xh + q where they are.
template <class S, bool SILU, bool PQ>
__global__ void __launch_bounds__(S::THREADS, (S::N > 8 && S::THREADS <= 256 ? 256 : 512) / S::THREADS)
k_row_bwd2(const typename S::T* __restrict__ x, int64_t ldx, const typename S::T* __restrict__ g, int64_t ldg,
           const typename S::T* __restrict__ u, int64_t ldu, Norm n, const float* __restrict__ mean_in,
           const float* __restrict__ rstd_in, int64_t rows, typename S::T* __restrict__ dg,
           typename S::T* __restrict__ dx, float* __restrict__ part) {
  using Raw = typename S::P::Raw;
  __shared__ float sh[S::TEAM > 32 ? S::SCRATCH : S::THREADS / 32 * S::TEAM * S::N];
  int turn = 0;
  const int me = threadIdx.x % S::TEAM, W = (int)n.W;
  const int64_t step = gridDim.x * (int64_t)S::TEAMS;
  const float inv = 1.f / W;
  alignas(8) float dw[S::N], db[S::N];
#pragma unroll
  for (int k = 0; k < S::N; ++k) dw[k] = db[k] = 0.f;
  int held = 0;
  bool first = true;
  if (part) part += blockIdx.x * (int64_t)(2 * W);
  int64_t row = blockIdx.x * (int64_t)S::TEAMS + threadIdx.x / S::TEAM;
  Rows<S, 3> operands{{x, g, u}, {ldx, ldg, ldu}, rows, step, W};
  operands.load(row);
  Stats next;
  next.load(mean_in, rstd_in, row, rows);
  for (int64_t base = blockIdx.x * (int64_t)S::TEAMS; base < rows; base += step, row += step) {
    alignas(8) float v[3][S::N], ga[S::N], be[S::N], B[S::N], C[S::N];
    operands.take(row, v);
    const Stats st = next;
    next.load(mean_in, rstd_in, row + step, rows);
    columns<S>(n.gamma, W, 1.f, ga);
    if (SILU) columns<S>(n.beta, W, 0.f, be);
    const float2 r = f2(st.rstd);
    float2 s[5];      // u, u xh, r h, r h xh, r h u; beyond the row's end g and u are 0
#pragma unroll
    for (int i = 0; i < 5; ++i) s[i] = f2(0.f);
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      float2& xh = E2A_PAIR(v[0], e);
      const float2 gv = E2A_PAIR(v[1], e), uv = E2A_PAIR(v[2], e), w = E2A_PAIR(ga, e);
      xh = normalised<S, true>(xh, e, W, st);
      const Act2 a = derivatives<SILU, true>(SILU ? f2_fma(xh, w, E2A_PAIR(be, e)) : xh);
      E2A_PAIR(B, e) = SILU ? f2_mul(a.d1, r) : r;
      E2A_PAIR(C, e) = SILU ? f2_mul(f2_mul(gv, a.d2), f2_mul(w, r)) : f2(0.f);
      const float2 rh = f2_mul(f2_mul(gv, E2A_PAIR(B, e)), w);
      s[0] = f2_add(s[0], uv);
      s[1] = f2_fma(uv, xh, s[1]);
      s[2] = f2_add(s[2], rh);
      s[3] = f2_fma(rh, xh, s[3]);
      s[4] = f2_fma(rh, uv, s[4]);
    }
    float s5[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) s5[i] = s[i].x + s[i].y;
    team_sum<S::TEAM>(s5, sh, turn);
    const float su = s5[0] * inv, sc = s5[1] * inv, m2 = s5[3] * inv;     // <u>, c, r <h xh>
    const float ht = s5[4] * inv - s5[2] * inv * su - m2 * sc;            // <h t>
    const bool in = row < rows;
    float2 k1 = f2(0.f), k2 = f2(0.f);
    alignas(8) float pc[S::N], qc[S::N];
    if (PQ) {
      columns<S>(n.p, W, 0.f, pc);
      columns<S>(n.q, W, 0.f, qc);
    }
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      const float2 xh = E2A_PAIR(v[0], e), w = E2A_PAIR(ga, e), gv = E2A_PAIR(v[1], e);
      float2& uv = E2A_PAIR(v[2], e);
      float2 d = f2_fma(xh, f2(-sc), f2_add(uv, f2(-su)));
      const float2 gB = f2_mul(gv, E2A_PAIR(B, e));
      float2 er = f2_mul(E2A_PAIR(C, e), d);
      float2 out = f2_mul(f2_mul(E2A_PAIR(B, e), w), d);
      float2 kk = f2_fma(gB, f2(-sc), er);
      if (PQ) {      // v's other share o = p xh + q: act' o, e + g act'' o, k + act' g p
        const float2 o = f2_fma(E2A_PAIR(pc, e), xh, E2A_PAIR(qc, e));
        const Act2 a = derivatives<SILU, true>(SILU ? f2_fma(xh, w, E2A_PAIR(be, e)) : xh);
        out = f2_fma(a.d1, o, out);
        const float2 more = f2_mul(f2_mul(gv, a.d2), o);
        kk = f2_add(kk, more);
        er = f2_add(er, more);
        kk = f2_mul(kk, w);
        kk = f2_fma(f2_mul(gv, a.d1), E2A_PAIR(pc, e), kk);
      } else {
        kk = f2_mul(kk, w);
      }
      kk = f2_fma(uv, f2(-m2), kk);
      E2A_PAIR(dw, e) = f2_fma(gB, d, E2A_PAIR(dw, e));
      if (SILU) {
        E2A_PAIR(dw, e) = f2_fma(er, xh, E2A_PAIR(dw, e));
        E2A_PAIR(db, e) = f2_add(er, E2A_PAIR(db, e));
      }
      E2A_PAIR(v[1], e) = out;
      uv = kk;
    }
#pragma unroll
    for (int i = 0; i < S::V; ++i) {
      const int c = (me + S::TEAM * i) * S::VEC;
      if (i < S::UNASKED || c < W) {
        if (in) *reinterpret_cast<Raw*>(dg + row * W + c) = S::P::narrow(v[1] + i * S::VEC);
      } else {
#pragma unroll
        for (int k = 0; k < S::VEC; ++k) v[2][i * S::VEC + k] = 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e) {
      k1 = f2_add(k1, E2A_PAIR(v[2], e));
      k2 = f2_fma(E2A_PAIR(v[2], e), E2A_PAIR(v[0], e), k2);
    }
    float s2[2] = {k1.x + k1.y, k2.x + k2.y};
    team_sum<S::TEAM>(s2, sh, turn);
    k1 = f2(-s2[0] * inv * st.rstd);
    k2 = f2(-(s2[1] * inv + ht) * st.rstd);
#pragma unroll
    for (int e = 0; e < S::N / 2; ++e)
      E2A_PAIR(v[2], e) = f2_fma(E2A_PAIR(v[2], e), r, f2_fma(E2A_PAIR(v[0], e), k2, k1));
#pragma unroll
    for (int i = 0; i < S::V; ++i) {
      const int c = (me + S::TEAM * i) * S::VEC;
      if (in && (i < S::UNASKED || c < W)) *reinterpret_cast<Raw*>(dx + row * W + c) = S::P::narrow(v[2] + i * S::VEC);
    }
    if (part && ++held == kChain) {
      flush_cols<S>(dw, db, part, W, first, sh);
      first = false;
      held = 0;
    }
  }
  if (part && (held || first)) flush_cols<S>(dw, db, part, W, first, sh);
}

// Column c of the partial rows, added up in row order by 32 threads in 64 bits.
__global__ void __launch_bounds__(1024)
k_part_sum(const float* __restrict__ part, int n_part, int W, float* __restrict__ dw, float* __restrict__ db) {
  __shared__ double sh[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  double s = 0.;
  if (c < 2 * W) {
#pragma unroll 4
    for (int i = threadIdx.y; i < n_part; i += 32) s += part[(int64_t)i * 2 * W + c];
  }
  sh[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sh[threadIdx.x][threadIdx.y];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < 2 * W) {
    float* out = col < W ? dw : db;
    if (out) out[col < W ? col : col - W] = (float)s;
  }
}

// The widest row that teams hold in registers; wider ones take the loops over memory above.
constexpr int64_t kMaxTeamWidth = 8192;

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 16-byte loads and stores need every row of every operand to start on 16 bytes.
template <typename T>
bool vectors_fit(const Norm& n, const void* const* rows_of, const int64_t* ld, int count) {
  constexpr int VEC = 16 / sizeof(T);
  if (n.W % VEC) return false;
  for (int i = 0; i < count; ++i)
    if (!aligned16(rows_of[i]) || ld[i] % VEC) return false;
  return aligned16(n.gamma) && aligned16(n.beta) && aligned16(n.p) && aligned16(n.q);
}

// Calls f with the Shape for rows of W values: two vectors a thread while a warp holds the row so, then 16 values,
// then WIDE in teams of a CTA, the smallest that holds a row.  640,210 x 128 fp32: 16 values a thread take the
// backward from 161 to 190 us; 16,384 x 4,096 bf16: 32 take the forward from 62 to 49 us, the backward from 81 to
// 99 us (registers).
template <typename T, int WIDE, typename F>
int by_shape(int64_t W, bool vec, F f) {
  constexpr int VEC = 16 / sizeof(T), V16 = 16 / VEC, VW = WIDE / VEC;
  if (vec) {
    if (W <= 4 * VEC) return f(Shape<T, VEC, 1, 4>{});
    if (W <= 8 * VEC) return f(Shape<T, VEC, 2, 4>{});
    if (W <= 16 * VEC) return f(Shape<T, VEC, 2, 8>{});
    if (W <= 32 * VEC) return f(Shape<T, VEC, 2, 16>{});
    if (W <= 64 * VEC) return f(Shape<T, VEC, 2, 32>{});
    if constexpr (VEC < 8) {      // 16 values a thread are two vectors otherwise
      if (W <= 512) return f(Shape<T, VEC, V16, 32>{});
    }
    if constexpr (WIDE > 16) {
      if (W <= 32 * WIDE) return f(Shape<T, VEC, VW, 32>{});
    }
    if (W <= 64 * WIDE) return f(Shape<T, VEC, VW, 64>{});
    if (W <= 128 * WIDE) return f(Shape<T, VEC, VW, 128>{});
    if constexpr (WIDE > 16) {
      return f(Shape<T, VEC, VW, 256>{});
    } else {
      if (W <= 256 * WIDE) return f(Shape<T, VEC, VW, 256>{});
      return f(Shape<T, VEC, V16, 512>{});
    }
  }
  if (W <= 32) return f(Shape<T, 1, 4, 8>{});
  if (W <= 64) return f(Shape<T, 1, 4, 16>{});
  if (W <= 128) return f(Shape<T, 1, 4, 32>{});
  if (W <= 256) return f(Shape<T, 1, 8, 32>{});
  // 8 values a thread at most beyond a warp, too, where their gradients' sums are held (150,000 x 262 fp32 backward: 519
  // us with 16, 117 us), 16 in the forward (71 us; 75 us where 8 took 96)
  if constexpr (WIDE > 16) {
    if (W <= 512) return f(Shape<T, 1, 16, 32>{});
    if (W <= 1024) return f(Shape<T, 1, 16, 64>{});
    if (W <= 2048) return f(Shape<T, 1, 16, 128>{});
    if (W <= 4096) return f(Shape<T, 1, 16, 256>{});
  } else {
    if (W <= 512) return f(Shape<T, 1, 8, 64>{});
    if (W <= 1024) return f(Shape<T, 1, 8, 128>{});
    if (W <= 2048) return f(Shape<T, 1, 8, 256>{});
    if (W <= 4096) return f(Shape<T, 1, 8, 512>{});
  }
  return f(Shape<T, 1, 16, 512>{});
}

// Partial rows of column sums, one per CTA of a row kernel.
int64_t most_parts(int64_t rows, int64_t W) {
  const int64_t most = W <= 1024 ? 148 * 16 : 148 * 8;
  return rows < most ? rows : most;
}

// CTAs of a row kernel: as many as the device holds at once, never more than there are batches of rows.
template <auto Kernel, class S>
int row_grid(int64_t rows, int64_t W, int* grid) {
  if (W < S::TEAM * S::VEC * S::SURE) return E2A_ERR_ARG;      // what Shape says of by_shape
  static std::atomic<int> resident_on[64];
  int dev = 0;
  E2A_CUDA(cudaGetDevice(&dev));
  std::atomic<int>& known = resident_on[dev & 63];
  int resident = dev < 64 ? known.load(std::memory_order_relaxed) : 0;
  if (resident == 0) {
    int sms = 0, per = 0;
    E2A_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    E2A_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, Kernel, S::THREADS, 0));
    resident = sms * (per > 0 ? per : 1);
    known.store(resident, std::memory_order_relaxed);
  }
  const int64_t batches = (rows + S::TEAMS - 1) / S::TEAMS, most = most_parts(rows, W);
  const int64_t g = batches < resident ? batches : resident;
  *grid = (int)(g < most ? g : most);
  return E2A_OK;
}

int sum_parts(const float* part, int n_part, int64_t W, float* dw, float* db, cudaStream_t st) {
  k_part_sum<<<(unsigned)((2 * W + 31) / 32), dim3(32, 32), 0, st>>>(part, n_part, (int)W, dw, db);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
}

int grid_rows(int64_t rows) {
  int64_t b = (rows + kThreads / 32 - 1) / (kThreads / 32);
  return (int)(b > 148 * 64 ? 148 * 64 : b);
}

int64_t chunk_count(int64_t rows) { return rows < 512 ? 1 : (rows / 512 > 1024 ? 1024 : rows / 512); }

template <typename T>
int launch_cols(bool second, const T* x, int64_t ldx, const T* g, int64_t ldg, const T* u, int64_t ldu, Norm n,
                const float* mean, const float* rstd, const float* row_u, const float* row_c, int64_t rows, double* part,
                float* dw, float* db, cudaStream_t st) {
  const int64_t chunks = chunk_count(rows), per = (rows + chunks - 1) / chunks;
  const dim3 grid((unsigned)((n.W + 31) / 32), (unsigned)chunks), block(32, 8);
  if (second)
    k_ln_cols<T, true><<<grid, block, 0, st>>>(x, ldx, g, ldg, u, ldu, n, mean, rstd, row_u, row_c, rows, per, part);
  else
    k_ln_cols<T, false><<<grid, block, 0, st>>>(x, ldx, g, ldg, u, ldu, n, mean, rstd, row_u, row_c, rows, per, part);
  E2A_CHECK_LAUNCH();
  k_ln_cols_sum<<<(unsigned)((2 * n.W + 255) / 256), 256, 0, st>>>(part, chunks, n.W, dw, db);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
}

bool bad_shape(int64_t rows, int64_t W, int64_t ld) { return rows < 0 || W <= 0 || W > (1ll << 30) || ld < 0; }

// Rows start at multiples of their type's size, the fp32 vectors and the workspace at multiples of theirs.
template <typename... P>
bool bad_rows(int dtype, const P*... p) { return e2a_misaligned(dtype == 0 ? 4 : 2, p...); }

bool bad_mode(int dtype, int act) { return dtype < 0 || dtype > 2 || (act != 0 && act != 1); }

size_t part_bytes(int64_t rows, int64_t W) {
  return e2a_align_up(W <= kMaxTeamWidth ? (size_t)most_parts(rows, W) * 2 * W * 4
                                         : (size_t)chunk_count(rows) * 2 * W * 8, 256);
}

template <typename F>
int by_type(int dtype, F f) {
  switch (dtype) {
    case 0: return f((float*)nullptr);
    case 1: return f((__nv_bfloat16*)nullptr);
    case 2: return f((__half*)nullptr);
    default: return E2A_ERR_ARG;
  }
}

template <typename F>
int by_flag(bool flag, F f) {
  return flag ? f(std::true_type{}) : f(std::false_type{});
}

int zero_cols(float* dw, float* db, int64_t W, cudaStream_t st) {
  if (dw) E2A_CUDA(cudaMemsetAsync(dw, 0, W * sizeof(float), st));
  if (db) E2A_CUDA(cudaMemsetAsync(db, 0, W * sizeof(float), st));
  return E2A_OK;
}

}  // namespace
