// Layer norm: forward and first-order backward entry points (the mathematics and the kernels: e2a_norm.cuh).  With
// E2A_ROW_TYPE the kernels for that type of rows, without it the entry points: the compiler works on four parts at once.
#include "e2a_norm.cuh"

struct E2aLnFwd {
  const void* x; int64_t ldx;
  const float *gamma, *beta;
  int64_t rows, W;
  float eps;
  int act;
  void* y;
  float *mean, *rstd;
  cudaStream_t st;
};
struct E2aLnBwd {
  const void* x; int64_t ldx;
  const void* dy; int64_t lddy;
  const float *gamma, *beta, *mean, *rstd;
  int64_t rows, W;
  int act;
  void* dx;
  float *dgamma, *dbeta;
  void* workspace;
  cudaStream_t st;
};

template <typename T>
int e2a_ln_fwd(const E2aLnFwd& a);
template <typename T>
int e2a_ln_bwd(const E2aLnBwd& a);

#ifdef E2A_ROW_TYPE

template <typename T>
int e2a_ln_fwd(const E2aLnFwd& a) {
  const Norm n{a.gamma, a.beta, nullptr, nullptr, a.W, a.act == 1};
  const T* x = (const T*)a.x;
  if (a.W <= kMaxTeamWidth) {
    const void* of[] = {x, a.y};
    const int64_t ld[] = {a.ldx, a.W};
    return by_shape<T, 32>(a.W, vectors_fit<T>(n, of, ld, 2), [&](auto shape) -> int {
      using S = decltype(shape);
      return by_flag(n.silu, [&](auto silu) -> int {
        constexpr auto kernel = &k_row_fwd<S, silu.value>;
        int grid = 0;
        if (const int rc = row_grid<kernel, S>(a.rows, a.W, &grid)) return rc;
        kernel<<<grid, S::THREADS, 0, a.st>>>(x, a.ldx, n, a.rows, a.eps, (T*)a.y, a.mean, a.rstd);
        E2A_CHECK_LAUNCH();
        return E2A_OK;
      });
    });
  }
  k_ln_fwd<T><<<grid_rows(a.rows), kThreads, 0, a.st>>>(x, a.ldx, n, a.rows, a.eps, (T*)a.y, a.mean, a.rstd);
  E2A_CHECK_LAUNCH();
  return E2A_OK;
}
template int e2a_ln_fwd<E2A_ROW_TYPE>(const E2aLnFwd&);

template <typename T>
int e2a_ln_bwd(const E2aLnBwd& a) {
  const Norm n{a.gamma, a.beta, nullptr, nullptr, a.W, a.act == 1};
  const T *x = (const T*)a.x, *dy = (const T*)a.dy;
  const bool cols = a.dgamma || a.dbeta;
  if (!a.dx && !cols) return E2A_OK;
  if (a.W <= kMaxTeamWidth) {
    const void* of[] = {x, dy, a.dx};
    const int64_t ld[] = {a.ldx, a.lddy, a.W};
    return by_shape<T, 16>(a.W, vectors_fit<T>(n, of, ld, 3), [&](auto shape) -> int {
      using S = decltype(shape);
      float* part = cols ? (float*)a.workspace : nullptr;
      return by_flag(n.silu, [&](auto silu) -> int {
        constexpr auto kernel = &k_row_bwd<S, silu.value>;
        int grid = 0;
        if (const int rc = row_grid<kernel, S>(a.rows, a.W, &grid)) return rc;
        kernel<<<grid, S::THREADS, 0, a.st>>>(x, a.ldx, dy, a.lddy, n, a.mean, a.rstd, a.rows, (T*)a.dx, part);
        E2A_CHECK_LAUNCH();
        return part ? sum_parts(part, grid, a.W, a.dgamma, a.dbeta, a.st) : E2A_OK;
      });
    });
  }
  if (a.dx) {
    k_ln_bwd<T><<<grid_rows(a.rows), kThreads, 0, a.st>>>(x, a.ldx, dy, a.lddy, n, a.mean, a.rstd, a.rows, (T*)a.dx);
    E2A_CHECK_LAUNCH();
  }
  if (!cols) return E2A_OK;
  return launch_cols<T>(false, x, a.ldx, dy, a.lddy, nullptr, 0, n, a.mean, a.rstd, nullptr, nullptr, a.rows,
                        (double*)a.workspace, a.dgamma, a.dbeta, a.st);
}
template int e2a_ln_bwd<E2A_ROW_TYPE>(const E2aLnBwd&);

#else

extern "C" {

int e2a_layer_norm_fwd(const void* x, int64_t ldx, int dtype, const float* gamma, const float* beta, int64_t rows,
                       int64_t W, float eps, int act, void* y, float* mean, float* rstd, void* stream) {
  if (bad_shape(rows, W, ldx) || bad_mode(dtype, act)) return E2A_ERR_ARG;
  if (rows == 0) return E2A_OK;
  if (!x || !y || !mean || !rstd) return E2A_ERR_ARG;
  if (bad_rows(dtype, x, y) || e2a_misaligned(4, gamma, beta, mean, rstd)) return E2A_ERR_ARG;
  const E2aLnFwd a{x, ldx, gamma, beta, rows, W, eps, act, y, mean, rstd, (cudaStream_t)stream};
  return by_type(dtype, [&](auto* t) { return e2a_ln_fwd<std::remove_pointer_t<decltype(t)>>(a); });
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
  if (bad_rows(dtype, x, dy, dx) || e2a_misaligned(4, gamma, beta, mean, rstd, dgamma, dbeta) ||
      e2a_misaligned(16, workspace))
    return E2A_ERR_ARG;
  if ((dgamma || dbeta) && (!workspace || workspace_bytes < part_bytes(rows, W))) return E2A_ERR_WORKSPACE;
  const E2aLnBwd a{x, ldx, dy, lddy, gamma, beta, mean, rstd, rows, W, act, dx, dgamma, dbeta, workspace, st};
  return by_type(dtype, [&](auto* t) { return e2a_ln_bwd<std::remove_pointer_t<decltype(t)>>(a); });
}

}  // extern "C"
#endif
