// Products with many vectors (q4_gemm.cu): arguments as in q4.h, n_vec >= 1 for the products.
#pragma once
#include "q4.h"

namespace mx {
namespace q4 {

template <typename V>
cudaError_t product_many(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s);
template <typename V>
cudaError_t product_t_many(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                           cudaStream_t s);
template <typename V>
cudaError_t grad_many(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy,
                      V *d_scales, V *d_res, cudaStream_t s);
// *flag = whether a bounded wait of an earlier call on the current device ended without its barrier (async copy)
cudaError_t waits_ran_out(int *flag, cudaStream_t s);
cudaError_t waits_ran_out_few(int *flag, cudaStream_t s);
cudaError_t waits_ran_out_grad(int *flag, cudaStream_t s);
cudaError_t waits_ran_out_quant(int *flag, cudaStream_t s);

}  // namespace q4
}  // namespace mx
