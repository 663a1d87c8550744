// Layer norm: second-order backward entry points (the mathematics and the kernels: e2a_norm.cuh).  With E2A_ROW_TYPE
// the kernels for that type of rows, without it the entry points: the compiler works on four parts at once.
#include "e2a_norm.cuh"

struct E2aLnBwd2 {
  const void* x; int64_t ldx;
  const void* dy; int64_t lddy;
  const void* u; int64_t ldu;
  const float *gamma, *beta, *mean, *rstd, *p, *q;
  int64_t rows, W;
  int act;
  void *d_dy, *dx;
  float *dgamma, *dbeta;
  double* part;
  float *row_u, *row_c;
  cudaStream_t st;
};

template <typename T>
int e2a_ln_bwd2(const E2aLnBwd2& a);

#ifdef E2A_ROW_TYPE

template <typename T>
int e2a_ln_bwd2(const E2aLnBwd2& a) {
  const Norm n{a.gamma, a.beta, a.p, a.q, a.W, a.act == 1};
  const T *x = (const T*)a.x, *dy = (const T*)a.dy, *u = (const T*)a.u;
  if (a.W <= kMaxTeamWidth) {
    const void* of[] = {x, dy, u, a.d_dy, a.dx};
    const int64_t ld[] = {a.ldx, a.lddy, a.ldu, a.W, a.W};
    return by_shape<T, 16>(a.W, vectors_fit<T>(n, of, ld, 5), [&](auto shape) -> int {
      using S = decltype(shape);
      float* sums = a.dgamma || a.dbeta ? (float*)a.part : nullptr;
      return by_flag(n.silu, [&](auto silu) -> int {
        return by_flag(a.p || a.q, [&](auto pq) -> int {
          constexpr auto kernel = &k_row_bwd2<S, silu.value, pq.value>;
          int grid = 0;
          if (const int rc = row_grid<kernel, S>(a.rows, a.W, &grid)) return rc;
          kernel<<<grid, S::THREADS, 0, a.st>>>(x, a.ldx, dy, a.lddy, u, a.ldu, n, a.mean, a.rstd, a.rows, (T*)a.d_dy,
                                                (T*)a.dx, sums);
          E2A_CHECK_LAUNCH();
          return sums ? sum_parts(sums, grid, a.W, a.dgamma, a.dbeta, a.st) : E2A_OK;
        });
      });
    });
  }
  k_ln_bwd2<T><<<grid_rows(a.rows), kThreads, 0, a.st>>>(x, a.ldx, dy, a.lddy, u, a.ldu, n, a.mean, a.rstd, a.rows,
                                                         (T*)a.d_dy, (T*)a.dx, a.row_u, a.row_c);
  E2A_CHECK_LAUNCH();
  if (!a.dgamma && !a.dbeta) return E2A_OK;
  return launch_cols<T>(true, x, a.ldx, dy, a.lddy, u, a.ldu, n, a.mean, a.rstd, a.row_u, a.row_c, a.rows, a.part,
                        a.dgamma, a.dbeta, a.st);
}
template int e2a_ln_bwd2<E2A_ROW_TYPE>(const E2aLnBwd2&);

#else

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
  const E2aLnBwd2 a{x, ldx, dy, lddy, u, ldu, gamma, beta, mean, rstd, p, q, rows, W, act, d_dy, dx, dgamma, dbeta,
                    part, row_u, row_c, st};
  return by_type(dtype, [&](auto* t) { return e2a_ln_bwd2<std::remove_pointer_t<decltype(t)>>(a); });
}

}  // extern "C"
#endif
