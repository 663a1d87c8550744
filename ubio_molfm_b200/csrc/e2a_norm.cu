// Layer norm: forward and first-order backward entry points (the mathematics and the kernels: e2a_norm.cuh).
#include "e2a_norm.cuh"

extern "C" {

int e2a_layer_norm_fwd(const void* x, int64_t ldx, int dtype, const float* gamma, const float* beta, int64_t rows,
                       int64_t W, float eps, int act, void* y, float* mean, float* rstd, void* stream) {
  if (bad_shape(rows, W, ldx) || bad_mode(dtype, act)) return E2A_ERR_ARG;
  if (rows == 0) return E2A_OK;
  if (!x || !y || !mean || !rstd) return E2A_ERR_ARG;
  if (bad_rows(dtype, x, y) || e2a_misaligned(4, gamma, beta, mean, rstd)) return E2A_ERR_ARG;
  const Norm n{gamma, beta, nullptr, nullptr, W, act == 1};
  return by_type(dtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (W <= kMaxTeamWidth) {
      const void* of[] = {x, y};
      const int64_t ld[] = {ldx, W};
      return by_shape<T, 32>(W, vectors_fit<T>(n, of, ld, 2), [&](auto shape) -> int {
        using S = decltype(shape);
        return by_flag(n.silu, [&](auto silu) -> int {
          constexpr auto kernel = &k_row_fwd<S, silu.value>;
          int grid = 0;
          if (const int rc = row_grid<kernel, S>(rows, W, &grid)) return rc;
          kernel<<<grid, S::THREADS, 0, (cudaStream_t)stream>>>((const T*)x, ldx, n, rows, eps, (T*)y, mean, rstd);
          E2A_CHECK_LAUNCH();
          return E2A_OK;
        });
      });
    }
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
  if (bad_rows(dtype, x, dy, dx) || e2a_misaligned(4, gamma, beta, mean, rstd, dgamma, dbeta) ||
      e2a_misaligned(16, workspace))
    return E2A_ERR_ARG;
  if ((dgamma || dbeta) && (!workspace || workspace_bytes < part_bytes(rows, W))) return E2A_ERR_WORKSPACE;
  const Norm n{gamma, beta, nullptr, nullptr, W, act == 1};
  return by_type(dtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!dx && !dgamma && !dbeta) return E2A_OK;
    if (W <= kMaxTeamWidth) {
      const void* of[] = {x, dy, dx};
      const int64_t ld[] = {ldx, lddy, W};
      return by_shape<T, 16>(W, vectors_fit<T>(n, of, ld, 3), [&](auto shape) -> int {
        using S = decltype(shape);
        float* part = dgamma || dbeta ? (float*)workspace : nullptr;
        return by_flag(n.silu, [&](auto silu) -> int {
          constexpr auto kernel = &k_row_bwd<S, silu.value>;
          int grid = 0;
          if (const int rc = row_grid<kernel, S>(rows, W, &grid)) return rc;
          kernel<<<grid, S::THREADS, 0, st>>>((const T*)x, ldx, (const T*)dy, lddy, n, mean, rstd, rows, (T*)dx, part);
          E2A_CHECK_LAUNCH();
          return part ? sum_parts(part, grid, W, dgamma, dbeta, st) : E2A_OK;
        });
      });
    }
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

}  // extern "C"
