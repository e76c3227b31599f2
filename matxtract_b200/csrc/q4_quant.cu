// 4-bit matrices: dense -> codes + scales + zero points + CSR residual (mx_q4_quantize) and back (mx_q4_expand).
#include <math.h>

#include "q4.h"

namespace mx {
namespace q4 {
namespace {

constexpr int WARPS = 8;

// w / s to the nearest whole number, ties to even.  The quotient's own rounding can put it on the wrong side of a
// border (w may have 24 bits), the remainder cannot: q * s has 4 + 11 bits, so that w - q * s is exact near a border.
__device__ __forceinline__ float nearest_quotient(float w, float s) {
    float q = rintf(fminf(fmaxf(w / s, -32.f), 32.f));
    const float r = fmaf(-q, s, w);
    const float twice = 2.f * fabsf(r);
    if (twice > s || (twice == s && ((int)q & 1))) q += copysignf(1.f, r);
    return q;
}

template <typename W>
__device__ __forceinline__ bool is_far(W w, float threshold) { return fabsf(to_float(w)) > threshold; }

// counts[i] = entries of row i above the threshold; one warp a row
template <typename W>
__global__ void count_kernel(int n_rows, int n_cols, const W *w, long long ld, float threshold, int *counts) {
    const int row = blockIdx.x * WARPS + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (row >= n_rows) return;
    int n = 0;
    for (int k = lane; k < n_cols; k += 32) n += is_far(w[row * ld + k], threshold);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) counts[row] = n;
}

// ptr[0] = 0, ptr[i + 1] = sum of ptr[1 .. i + 1] (as far as int32 holds it), in one block
__global__ void __launch_bounds__(1024) scan_kernel(int n, int *ptr) {
    __shared__ long long sums[32];
    __shared__ long long carry;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        carry = 0;
        ptr[0] = 0;
    }
    __syncthreads();
    for (int base = 0; base < n; base += 1024) {
        const int i = base + threadIdx.x;
        long long v = i < n ? ptr[i + 1] : 0;
        for (int d = 1; d < 32; d *= 2) {
            const long long u = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += u;
        }
        if (lane == 31) sums[warp] = v;
        __syncthreads();
        long long before = carry;
        for (int k = 0; k < warp; ++k) before += sums[k];
        if (i < n) ptr[i + 1] = (int)min(before + v, (long long)INT_MAX);
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + v;
        __syncthreads();
    }
}

// one warp a row, 64 columns (2 a lane) at a time; a group is gone through twice, for its range and for its codes
template <typename V, typename W, bool ZEROS>
__global__ void quantize_kernel(int n_rows, int n_cols, int group, int n_groups, const W *w, long long ld,
                                float threshold, uint8_t *codes, long long code_ld, V *scales, uint8_t *zeros,
                                const int *res_ptr, int *res_col, V *res_val, int res_cap) {
    const int row = blockIdx.x * WARPS + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (row >= n_rows) return;
    const W *wr = w + row * ld;
    uint8_t *cr = codes + row * code_ld;
    const bool split = res_ptr != nullptr;
    long long at = split ? res_ptr[row] : 0;
    for (int g = 0; g < n_groups; ++g) {
        const int k0 = g * group, k1 = min((long long)n_cols, (long long)k0 + group);
        float lo = 0.f, hi = 0.f;
        bool nan = false;
        for (int k = k0 + lane; k < k1; k += 32) {
            const float v = to_float(wr[k]);
            if (split && fabsf(v) > threshold) continue;
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
            nan |= isnan(v);
        }
        for (int d = 16; d; d /= 2) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        nan = __any_sync(0xffffffffu, nan);
        const V s16 = from_float<V>(nan ? nanf("") : ZEROS ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f);
        const float s = to_float(s16);
        const bool usable = s > 0.f && s <= 3.4028235e38f;
        const float z = ZEROS ? (usable ? fminf(nearest_quotient(-lo, s), 15.f) : 0.f) : 8.f;
        if (lane == 0) {
            scales[(long long)row * n_groups + g] = s16;
            if (ZEROS) zeros[(long long)row * n_groups + g] = (uint8_t)z;
        }
        for (int k = k0 + 2 * lane; k - 2 * lane < k1; k += 64) {
            bool far[2] = {false, false};
            int c[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (k + j < k1) {
                    const float v = to_float(wr[k + j]);
                    far[j] = split && fabsf(v) > threshold;
                    const float q = usable && !far[j] ? nearest_quotient(v, s) : 0.f;
                    c[j] = (int)fminf(fmaxf(q + z, ZEROS ? 0.f : 1.f), 15.f);
                }
            if (k < k1) cr[k / 2] = (uint8_t)(c[0] | c[1] << 4);
            if (split) {
                const unsigned even = __ballot_sync(0xffffffffu, far[0]), odd = __ballot_sync(0xffffffffu, far[1]);
                const unsigned below = (1u << lane) - 1;
                const long long p = at + __popc(even & below) + __popc(odd & below);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const long long e = p + (j && far[0]);
                    if (far[j] && e < res_cap) {
                        res_col[e] = k + j;
                        res_val[e] = from_float<V>(to_float(wr[k + j]));
                    }
                }
                at += __popc(even) + __popc(odd);
            }
        }
    }
}

// one warp a row: the codes' values first, then the entries of the residual on top of them
template <typename V>
__global__ void expand_kernel(Matrix<V> m, V *w, long long ld) {
    const int row = blockIdx.x * WARPS + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (row >= m.n_rows) return;
    const uint8_t *cr = m.codes + row * m.code_ld;
    const V *sr = m.scales + (long long)row * m.n_groups;
    auto value = [&](int k) {
        const int g = k / m.group, c = cr[k / 2] >> 4 * (k & 1) & 15;
        return to_float(sr[g]) * (float)(c - zero_of(m, row, g));
    };
    for (int k = lane; k < m.n_cols; k += 32) w[row * ld + k] = from_float<V>(value(k));
    if (!m.res_ptr) return;
    __syncwarp();
    int b, e;
    res_range(m, row, b, e);
    for (int i = b + lane; i < e; i += 32) {
        const int k = m.res_col[i];
        if (k < 0 || k >= m.n_cols || (i > b && m.res_col[i - 1] == k)) continue;
        float v = value(k);
        for (int j = i; j < e && m.res_col[j] == k; ++j) v += to_float(m.res_val[j]);
        w[row * ld + k] = from_float<V>(v);
    }
}

template <typename V, typename W>
cudaError_t quantize_from(const mx_q4_matrix &m, const W *w, long long ld, float threshold, cudaStream_t s) {
    const int n_groups = (int)(((long long)m.n_cols + m.group - 1) / m.group);
    const int blocks = (m.n_rows + WARPS - 1) / WARPS;
    if (m.res_row_ptr) {
        if (blocks) count_kernel<<<blocks, 32 * WARPS, 0, s>>>(m.n_rows, m.n_cols, w, ld, threshold, m.res_row_ptr + 1);
        scan_kernel<<<1, 1024, 0, s>>>(m.n_rows, m.res_row_ptr);
    }
    if (blocks) {
        auto k = m.zeros ? quantize_kernel<V, W, true> : quantize_kernel<V, W, false>;
        k<<<blocks, 32 * WARPS, 0, s>>>(m.n_rows, m.n_cols, m.group, n_groups, w, ld, threshold,
                                        static_cast<uint8_t *>(m.codes), m.code_ld, static_cast<V *>(m.scales),
                                        static_cast<uint8_t *>(m.zeros), m.res_row_ptr, m.res_col_ind,
                                        static_cast<V *>(m.res_val), m.res_cap);
    }
    return cudaGetLastError();
}

}  // namespace

template <typename V>
cudaError_t quantize(const mx_q4_matrix &m, int w_dtype, const void *w, long long ld, float threshold, cudaStream_t s) {
    if (w_dtype == MX_FP32) return quantize_from<V>(m, static_cast<const float *>(w), ld, threshold, s);
    if (w_dtype == MX_FP16) return quantize_from<V>(m, static_cast<const __half *>(w), ld, threshold, s);
    return quantize_from<V>(m, static_cast<const __nv_bfloat16 *>(w), ld, threshold, s);
}

template <typename V>
cudaError_t expand(const Matrix<V> &m, V *w, long long ld, cudaStream_t s) {
    expand_kernel<<<(m.n_rows + WARPS - 1) / WARPS, 32 * WARPS, 0, s>>>(m, w, ld);
    return cudaGetLastError();
}

#define INSTANTIATE(V)                                                                                              \
    template cudaError_t quantize<V>(const mx_q4_matrix &, int, const void *, long long, float, cudaStream_t);      \
    template cudaError_t expand<V>(const Matrix<V> &, V *, long long, cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
