// Layer norm: second-order backward entry points (the mathematics and the kernels: e2a_norm.cuh).
#include "e2a_norm.cuh"

extern "C" {

size_t e2a_layer_norm_bwd2_workspace_bytes(int64_t rows, int64_t W) {
  if (rows <= 0 || W <= 0) return 0;
  return part_bytes(rows, W) + (W <= kMaxTeamWidth ? 0 : 2 * e2a_align_up((size_t)rows * sizeof(float), 256));
}

int e2a_layer_norm_bwd2(const void* x, int64_t ldx, const void* dy, int64_t lddy, const void* u, int64_t ldu, int dtype,
                        const float* gamma, const float* beta, const float* mean, const float* rstd, const float* p,
                        const float* q, int64_t rows, int64_t W, int act, void* d_dy, void* dx, float* dgamma,
                        float* dbeta, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_shape(rows, W, ldx) || lddy < 0 || ldu < 0 || bad_mode(dtype, act)) return E2A_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) return zero_cols(dgamma, dbeta, W, st);
  if (!x || !dy || !u || !mean || !rstd || !d_dy || !dx) return E2A_ERR_ARG;
  if (bad_rows(dtype, x, dy, u, d_dy, dx) || e2a_misaligned(4, gamma, beta, mean, rstd, p, q, dgamma, dbeta) ||
      e2a_misaligned(16, workspace))
    return E2A_ERR_ARG;
  E2aArena ar{(char*)workspace, workspace_bytes, 0};
  double* part = (double*)ar.take(part_bytes(rows, W));
  const bool loops = W > kMaxTeamWidth;      // <u> and c of every row, for the column sums' own pass
  float* row_u = loops ? (float*)ar.take(rows * sizeof(float)) : nullptr;
  float* row_c = loops ? (float*)ar.take(rows * sizeof(float)) : nullptr;
  if (!part || (loops && (!row_u || !row_c))) return E2A_ERR_WORKSPACE;
  const Norm n{gamma, beta, p, q, W, act == 1};
  return by_type(dtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (W <= kMaxTeamWidth) {
      const void* of[] = {x, dy, u, d_dy, dx};
      const int64_t ld[] = {ldx, lddy, ldu, W, W};
      return by_shape<T, 16>(W, vectors_fit<T>(n, of, ld, 5), [&](auto shape) -> int {
        using S = decltype(shape);
        float* sums = dgamma || dbeta ? (float*)part : nullptr;
        return by_flag(n.silu, [&](auto silu) -> int {
          return by_flag(p || q, [&](auto pq) -> int {
            constexpr auto kernel = &k_row_bwd2<S, silu.value, pq.value>;
            int grid = 0;
            if (const int rc = row_grid<kernel, S>(rows, W, &grid)) return rc;
            kernel<<<grid, S::THREADS, 0, st>>>((const T*)x, ldx, (const T*)dy, lddy, (const T*)u, ldu, n, mean, rstd,
                                                    rows, (T*)d_dy, (T*)dx, sums);
            E2A_CHECK_LAUNCH();
            return sums ? sum_parts(sums, grid, W, dgamma, dbeta, st) : E2A_OK;
          });
        });
      });
    }
    k_ln_bwd2<T><<<grid_rows(rows), kThreads, 0, st>>>((const T*)x, ldx, (const T*)dy, lddy, (const T*)u, ldu, n, mean,
                                                       rstd, rows, (T*)d_dy, (T*)dx, row_u, row_c);
    E2A_CHECK_LAUNCH();
    if (!dgamma && !dbeta) return E2A_OK;
    return launch_cols<T>(true, (const T*)x, ldx, (const T*)dy, lddy, (const T*)u, ldu, n, mean, rstd, row_u, row_c,
                          rows, part, dgamma, dbeta, st);
  });
}

}  // extern "C"
