// Products with a 4-bit matrix and the gradients of its numbers, straight from the definitions.
#include "q4.h"
#include "q4_gemm.h"

namespace mx {
namespace q4 {
namespace {

constexpr int WARPS = 8;
constexpr int FEW = 8;  // vectors up to which these kernels run; the tensor core kernels' tiles are wider

template <typename V>
__device__ __forceinline__ int step_at(const Matrix<V> &m, int i, int k) {
    const int c = m.codes[i * m.code_ld + k / 2] >> 4 * (k & 1) & 15;
    return c - zero_of(m, i, k / m.group);
}

__device__ __forceinline__ float warp_sum(float v) {
    for (int d = 16; d; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// one warp a result
template <typename V>
__global__ void product_kernel(Matrix<V> m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y) {
    const long long at = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int i = (int)(at % m.n_rows);
    const long long t = at / m.n_rows;
    if (t >= n_vec) return;
    float sum = 0.f;
    for (int k = lane; k < m.n_cols; k += 32)
        sum += to_float(m.scales[(long long)i * m.n_groups + k / m.group]) * (step_at(m, i, k) * to_float(x[t * ld_x + k]));
    if (m.res_ptr) {
        int b, e;
        res_range(m, i, b, e);
        for (int j = b + lane; j < e; j += 32) {
            const int k = m.res_col[j];
            if (k >= 0 && k < m.n_cols) sum += to_float(m.res_val[j]) * to_float(x[t * ld_x + k]);
        }
    }
    sum = warp_sum(sum);
    if (lane == 0) y[t * ld_y + i] = from_float<V>(sum);
}

// one thread a result
template <typename V>
__global__ void product_t_kernel(Matrix<V> m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx) {
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int k = (int)(at % m.n_cols);
    const long long t = at / m.n_cols;
    if (t >= n_vec) return;
    float sum = 0.f;
    for (int i = 0; i < m.n_rows; ++i) {
        const float d = to_float(dy[t * ld_dy + i]);
        sum += step_at(m, i, k) * to_float(m.scales[(long long)i * m.n_groups + k / m.group]) * d;
        if (m.res_ptr) {
            int b, e;
            res_range(m, i, b, e);
            for (int j = first_at_least(m.res_col, b, e, k); j < e && m.res_col[j] == k; ++j)
                sum += to_float(m.res_val[j]) * d;
        }
    }
    dx[t * ld_dx + k] = from_float<V>(sum);
}

template <typename V>
__device__ __forceinline__ float dot_over_vectors(int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy) {
    float sum = 0.f;
    for (long long t = 0; t < n_vec; ++t) sum += to_float(dy[t * ld_dy]) * to_float(x[t * ld_x]);
    return sum;
}

// one warp a scale
template <typename V>
__global__ void grad_scales_kernel(Matrix<V> m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy,
                                   V *d_scales) {
    const long long at = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (at >= (long long)m.n_rows * m.n_groups) return;
    const int i = (int)(at / m.n_groups), g = (int)(at % m.n_groups);
    const int k1 = (int)min((long long)m.n_cols, ((long long)g + 1) * m.group);
    float sum = 0.f;
    for (int k = g * m.group + lane; k < k1; k += 32)
        sum += step_at(m, i, k) * dot_over_vectors(n_vec, x + k, ld_x, dy + i, ld_dy);
    sum = warp_sum(sum);
    if (lane == 0) d_scales[at] = from_float<V>(sum);
}

// one warp a row, one thread an entry
template <typename V>
__global__ void grad_residual_kernel(Matrix<V> m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy,
                                     V *d_res) {
    const int i = blockIdx.x * WARPS + threadIdx.x / 32;
    if (i >= m.n_rows) return;
    int b, e;
    res_range(m, i, b, e);
    for (int j = b + threadIdx.x % 32; j < e; j += 32) {
        const int k = m.res_col[j];
        if (k >= 0 && k < m.n_cols) d_res[j] = from_float<V>(dot_over_vectors(n_vec, x + k, ld_x, dy + i, ld_dy));
    }
}

unsigned blocks_for(long long units, int per_block) { return (unsigned)((units + per_block - 1) / per_block); }

}  // namespace

template <typename V>
cudaError_t product(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s) {
    if (n_vec > FEW) return product_many(m, n_vec, x, ld_x, y, ld_y, s);
    product_kernel<<<blocks_for((long long)m.n_rows * n_vec, WARPS), 32 * WARPS, 0, s>>>(m, n_vec, x, ld_x, y, ld_y);
    return cudaGetLastError();
}

template <typename V>
cudaError_t product_t(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                      cudaStream_t s) {
    if (n_vec > FEW) return product_t_many(m, n_vec, dy, ld_dy, dx, ld_dx, s);
    product_t_kernel<<<blocks_for((long long)m.n_cols * n_vec, 256), 256, 0, s>>>(m, n_vec, dy, ld_dy, dx, ld_dx);
    return cudaGetLastError();
}

template <typename V>
cudaError_t grad(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy, V *d_scales,
                 V *d_res, cudaStream_t s) {
    if (n_vec > FEW) return grad_many(m, n_vec, x, ld_x, dy, ld_dy, d_scales, d_res, s);
    if (d_scales)
        grad_scales_kernel<<<blocks_for((long long)m.n_rows * m.n_groups, WARPS), 32 * WARPS, 0, s>>>(
            m, n_vec, x, ld_x, dy, ld_dy, d_scales);
    if (d_res)
        grad_residual_kernel<<<blocks_for(m.n_rows, WARPS), 32 * WARPS, 0, s>>>(m, n_vec, x, ld_x, dy, ld_dy, d_res);
    return cudaGetLastError();
}

#define INSTANTIATE(V)                                                                                                \
    template cudaError_t product<V>(const Matrix<V> &, int, const V *, long long, V *, long long, cudaStream_t);      \
    template cudaError_t product_t<V>(const Matrix<V> &, int, const V *, long long, V *, long long, cudaStream_t);    \
    template cudaError_t grad<V>(const Matrix<V> &, int, const V *, long long, const V *, long long, V *, V *,        \
                                 cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
