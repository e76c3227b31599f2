// Shared by the translation units of the 4-bit matrix operators (mx_q4_*): what a kernel sees of a matrix, and the
// launchers.  include/mx_capi.h has the definitions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mx_capi.h"

namespace mx {
namespace q4 {

// A checked mx_q4_matrix; V is the type of scales, residual values and vectors.
template <typename V>
struct Matrix {
    int n_rows, n_cols, group, n_groups;
    long long code_ld;
    const uint8_t *codes;
    const V *scales;
    const uint8_t *zeros;  // may be null: 8
    const int *res_ptr;    // may be null: no residual
    const int *res_col;
    const V *res_val;
    int res_cap;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename V>
__device__ __forceinline__ V from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Entries [begin, end) of row i, clamped into the buffers whatever the row pointers hold.  Entries' places are unsigned: a
// loop goes on behind the last one by its step, and a residual may have 2^31 - 1.
template <typename V>
__device__ __forceinline__ void res_range(const Matrix<V> &m, int i, unsigned &begin, unsigned &end) {
    const int b = max(0, min(m.res_ptr[i], m.res_cap));
    begin = b;
    end = max(b, min(m.res_ptr[i + 1], m.res_cap));
}

template <typename V>
__device__ __forceinline__ int zero_of(const Matrix<V> &m, int i, int g) {
    return m.zeros ? m.zeros[(long long)i * m.n_groups + g] & 15 : 8;
}

// First entry of [begin, end) whose column is at least k (columns ascend).
__device__ __forceinline__ unsigned first_at_least(const int *col, unsigned begin, unsigned end, int k) {
    while (begin < end) {
        const unsigned mid = begin + (end - begin) / 2;
        if (col[mid] < k)
            begin = mid + 1;
        else
            end = mid;
    }
    return begin;
}

template <typename V>
cudaError_t quantize(const mx_q4_matrix &m, int w_dtype, const void *w, long long ld_w, float threshold, cudaStream_t s);
template <typename V>
cudaError_t expand(const Matrix<V> &m, V *w, long long ld_w, cudaStream_t s);
template <typename V>
cudaError_t product(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s);
template <typename V>
cudaError_t product_t(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                      cudaStream_t s);
template <typename V>
cudaError_t grad(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy, V *d_scales,
                 V *d_res, cudaStream_t s);

}  // namespace q4
}  // namespace mx
