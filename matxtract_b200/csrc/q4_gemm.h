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
// where the kernels of each file write on the current device that a bounded wait ended without what it waited for
cudaError_t late_flag(int **flag);
cudaError_t late_flag_few(int **flag);
cudaError_t late_flag_quant(int **flag);
cudaError_t late_flag_grad(int **flag);

}  // namespace q4
}  // namespace mx
