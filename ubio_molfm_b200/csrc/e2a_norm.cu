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
// One warp per row; the statistics are two-pass in fp32 and kept per row.  The column sums run over chunks
// of rows in 64 bits, one partial per chunk, added up in chunk order (no atomics).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
// y'' = s (1 - s) (2 + z (1 - 2 s)).  Without activation 1 and 0.
struct Act { float y, d1, d2; };
__device__ __forceinline__ Act activation(float z, bool silu) {
  if (!silu) return {z, 1.f, 0.f};
  const float s = 1.f / (1.f + expf(-z));
  return {z * s, s * (1.f + z * (1.f - s)), s * (1.f - s) * (2.f + z * (1.f - 2.f * s))};
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

template <typename T>
__global__ void k_ln_fwd(const T* __restrict__ x, int64_t ldx, Norm n, int64_t rows, float eps, T* __restrict__ y,
                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  const int lane = threadIdx.x & 31;
  const int64_t nw = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t r = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; r < rows; r += nw) {
    const T* xr = x + r * ldx;
    float s = 0.f;
    for (int64_t c = lane; c < n.W; c += 32) s += to_f(xr[c]);
    const float mean = e2a_warp_sum(s) / n.W;
    float v = 0.f;
    for (int64_t c = lane; c < n.W; c += 32) {
      const float d = to_f(xr[c]) - mean;
      v += d * d;
    }
    const float rstd = 1.f / sqrtf(e2a_warp_sum(v) / n.W + eps);
    for (int64_t c = lane; c < n.W; c += 32) {
      const float z = (to_f(xr[c]) - mean) * rstd * at(n.gamma, c, 1.f) + at(n.beta, c, 0.f);
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
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = lane; c < n.W; c += 32) {
      const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd;
      const float h = to_f(gr[c]) * activation(xh * w + at(n.beta, c, 0.f), n.silu).d1 * w;
      s1 += h;
      s2 += h * xh;
    }
    s1 = e2a_warp_sum(s1) / n.W;
    s2 = e2a_warp_sum(s2) / n.W;
    for (int64_t c = lane; c < n.W; c += 32) {
      const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd;
      const float h = to_f(gr[c]) * activation(xh * w + at(n.beta, c, 0.f), n.silu).d1 * w;
      dx[r * n.W + c] = from_f<T>(rstd * (h - s1 - xh * s2));
    }
  }
}

// The row means the second order needs: {<u>, <u xh>, <h>, <h xh>, <h u>} and, from them, t.
struct RowMeans { float u, c, h1, h2, ht; };

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
    float su = 0.f, sc = 0.f, s1 = 0.f, s2 = 0.f, su2 = 0.f;
    for (int64_t c = lane; c < n.W; c += 32) {
      const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd, uv = to_f(ur[c]);
      const float h = to_f(gr[c]) * activation(xh * w + at(n.beta, c, 0.f), n.silu).d1 * w;
      su += uv;
      sc += uv * xh;
      s1 += h;
      s2 += h * xh;
      su2 += h * uv;
    }
    su = e2a_warp_sum(su) / n.W;
    sc = e2a_warp_sum(sc) / n.W;
    s1 = e2a_warp_sum(s1) / n.W;
    s2 = e2a_warp_sum(s2) / n.W;
    const float ht = rstd * (e2a_warp_sum(su2) / n.W - s1 * su - s2 * sc);
    float k1 = 0.f, k2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass == 1) {
        k1 = e2a_warp_sum(k1) / n.W;
        k2 = e2a_warp_sum(k2) / n.W + ht;
      }
      for (int64_t c = lane; c < n.W; c += 32) {
        const float w = at(n.gamma, c, 1.f), xh = (to_f(xr[c]) - mean) * rstd, uv = to_f(ur[c]), gv = to_f(gr[c]);
        const Act a = activation(xh * w + at(n.beta, c, 0.f), n.silu);
        const float pc = at(n.p, c, 0.f), t = rstd * (uv - su - xh * sc);
        const float v = w * t + pc * xh + at(n.q, c, 0.f);
        const float ga = gv * a.d1;
        const float k = gv * a.d2 * v * w + ga * pc - rstd * (uv * s2 + ga * w * sc);
        if (pass == 0) {
          k1 += k;
          k2 += k * xh;
        } else {
          dg[r * n.W + c] = from_f<T>(a.d1 * v);
          dx[r * n.W + c] = from_f<T>(rstd * (k - k1 - xh * k2));
        }
      }
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

bool bad_mode(int dtype, int act) { return dtype < 0 || dtype > 2 || (act != 0 && act != 1); }

size_t part_bytes(int64_t rows, int64_t W) { return e2a_align_up((size_t)chunk_count(rows) * 2 * W * 8, 256); }

template <typename F>
int by_type(int dtype, F f) {
  switch (dtype) {
    case 0: return f((float*)nullptr);
    case 1: return f((__nv_bfloat16*)nullptr);
    case 2: return f((__half*)nullptr);
    default: return E2A_ERR_ARG;
  }
}

int zero_cols(float* dw, float* db, int64_t W, cudaStream_t st) {
  if (dw) E2A_CUDA(cudaMemsetAsync(dw, 0, W * sizeof(float), st));
  if (db) E2A_CUDA(cudaMemsetAsync(db, 0, W * sizeof(float), st));
  return E2A_OK;
}

}  // namespace

extern "C" {

int e2a_layer_norm_fwd(const void* x, int64_t ldx, int dtype, const float* gamma, const float* beta, int64_t rows,
                       int64_t W, float eps, int act, void* y, float* mean, float* rstd, void* stream) {
  if (bad_shape(rows, W, ldx) || bad_mode(dtype, act)) return E2A_ERR_ARG;
  if (rows == 0) return E2A_OK;
  if (!x || !y || !mean || !rstd) return E2A_ERR_ARG;
  const Norm n{gamma, beta, nullptr, nullptr, W, act == 1};
  return by_type(dtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    k_ln_fwd<T><<<grid_rows(rows), kThreads, 0, (cudaStream_t)stream>>>((const T*)x, ldx, n, rows, eps, (T*)y, mean,
                                                                        rstd);
    E2A_CHECK_LAUNCH();
    return E2A_OK;
  });
}

size_t e2a_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t W) {
  return rows <= 0 || W <= 0 ? 0 : part_bytes(rows, W);
}

int e2a_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t lddy, int dtype, const float* gamma,
                       const float* beta, const float* mean, const float* rstd, int64_t rows, int64_t W, int act,
                       void* dx, float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_shape(rows, W, ldx) || lddy < 0 || bad_mode(dtype, act)) return E2A_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) return zero_cols(dgamma, dbeta, W, st);
  if (!x || !dy || !mean || !rstd) return E2A_ERR_ARG;
  if ((dgamma || dbeta) && (!workspace || workspace_bytes < part_bytes(rows, W))) return E2A_ERR_WORKSPACE;
  const Norm n{gamma, beta, nullptr, nullptr, W, act == 1};
  return by_type(dtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (dx) {
      k_ln_bwd<T><<<grid_rows(rows), kThreads, 0, st>>>((const T*)x, ldx, (const T*)dy, lddy, n, mean, rstd, rows,
                                                        (T*)dx);
      E2A_CHECK_LAUNCH();
    }
    if (!dgamma && !dbeta) return E2A_OK;
    return launch_cols<T>(false, (const T*)x, ldx, (const T*)dy, lddy, nullptr, 0, n, mean, rstd, nullptr, nullptr,
                          rows, (double*)workspace, dgamma, dbeta, st);
  });
}

size_t e2a_layer_norm_bwd2_workspace_bytes(int64_t rows, int64_t W) {
  return rows <= 0 || W <= 0 ? 0 : part_bytes(rows, W) + 2 * e2a_align_up((size_t)rows * sizeof(float), 256);
}

int e2a_layer_norm_bwd2(const void* x, int64_t ldx, const void* dy, int64_t lddy, const void* u, int64_t ldu, int dtype,
                        const float* gamma, const float* beta, const float* mean, const float* rstd, const float* p,
                        const float* q, int64_t rows, int64_t W, int act, void* d_dy, void* dx, float* dgamma,
                        float* dbeta, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_shape(rows, W, ldx) || lddy < 0 || ldu < 0 || bad_mode(dtype, act)) return E2A_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) return zero_cols(dgamma, dbeta, W, st);
  if (!x || !dy || !u || !mean || !rstd || !d_dy || !dx) return E2A_ERR_ARG;
  E2aArena ar{(char*)workspace, workspace_bytes, 0};
  double* part = (double*)ar.take(part_bytes(rows, W));
  float* row_u = (float*)ar.take(rows * sizeof(float));
  float* row_c = (float*)ar.take(rows * sizeof(float));
  if (!part || !row_u || !row_c) return E2A_ERR_WORKSPACE;
  const Norm n{gamma, beta, p, q, W, act == 1};
  return by_type(dtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    k_ln_bwd2<T><<<grid_rows(rows), kThreads, 0, st>>>((const T*)x, ldx, (const T*)dy, lddy, (const T*)u, ldu, n, mean,
                                                       rstd, rows, (T*)d_dy, (T*)dx, row_u, row_c);
    E2A_CHECK_LAUNCH();
    if (!dgamma && !dbeta) return E2A_OK;
    return launch_cols<T>(true, (const T*)x, ldx, (const T*)dy, lddy, (const T*)u, ldu, n, mean, rstd, row_u, row_c,
                          rows, part, dgamma, dbeta, st);
  });
}

}  // extern "C"
