// 4-bit matrices: dense -> codes + scales + zero points + CSR residual (mx_q4_quantize) and back (mx_q4_expand).
#include <math.h>

#include "q4.h"
#include "q4_values.cuh"

namespace mx {
namespace q4 {
namespace {

constexpr int WARPS = 8;
// A warp's piece of a row: 8 chunks of 256 columns, 8 neighbouring columns a lane, all asked for at once.  Short pieces
// fill the GPU with few rows too; their entries follow one another in the residual's order.
constexpr int CHUNK = 256, CHUNKS = 8, PIECE = CHUNK * CHUNKS;
constexpr int BLOCK = 256;  // pieces whose counts are summed up in one number

// w / s to the nearest whole number, ties to even.  The quotient's own rounding can put it on the wrong side of a
// border (w may have 24 bits), the remainder cannot: q * s has 4 + 11 bits, so that w - q * s is exact near a border.
__device__ __forceinline__ float nearest_from(float q, float w, float s) {
    const float r = fmaf(-q, s, w);
    const float twice = 2.f * fabsf(r);
    if (twice > s || (twice == s && ((int)q & 1))) q += copysignf(1.f, r);
    return q;
}
__device__ __forceinline__ float nearest_quotient(float w, float s) {
    return nearest_from(rintf(fminf(fmaxf(w / s, -32.f), 32.f)), w, s);
}

// scale and zero point of a group whose values reach from lo <= 0 to hi >= 0
template <typename V, bool ZEROS>
struct Scale {
    V stored;
    float s, z;
    bool usable;
    __device__ __forceinline__ Scale(float lo, float hi, bool nan) {
        stored = from_float<V>(nan ? nanf("") : ZEROS ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f);
        s = to_float(stored);
        usable = s > 0.f && s <= 3.4028235e38f;
        z = ZEROS ? (usable ? fminf(nearest_quotient(-lo, s), 15.f) : 0.f) : 8.f;
    }
};

// 8 neighbouring values of a row from column k on, 0 from column `end` on, not yet taken apart
template <typename W>
struct Raw {
    uint4 u[sizeof(W) / 2];
    __device__ __forceinline__ void load(const W *row, int k, int end, bool wide) {
        if (wide && k + 8 <= end) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(W) / 2; ++j) u[j] = __ldg(reinterpret_cast<const uint4 *>(row + k) + j);
        } else {
            W v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < end ? row[k + j] : from_float<W>(0.f);
#pragma unroll
            for (int j = 0; j < (int)sizeof(W) / 2; ++j) u[j] = reinterpret_cast<const uint4 *>(v)[j];
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const W *w = reinterpret_cast<const W *>(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float(w[j]);
    }
};

// counts[piece] = entries above the threshold, sums[b] = those of the pieces b BLOCK .. (b + 1) BLOCK - 1
template <typename W>
__global__ void __launch_bounds__(32 * WARPS) count_kernel(int n_rows, int n_cols, int per_row, const W *w, long long ld,
                                                           bool wide, float threshold, int *counts, int *sums) {
    const long long piece = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (piece >= (long long)n_rows * per_row) return;
    const W *row = w + piece / per_row * ld;
    const int k0 = (int)(piece % per_row) * PIECE + 8 * lane;
    Raw<W> raw[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) raw[c].load(row, k0 + c * CHUNK, n_cols, wide);
    int n = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        float v[8];
        raw[c].values(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) n += fabsf(v[j]) > threshold;
    }
    // what lies behind the last column counts as 0, which is above a negative threshold
    if (threshold < 0.f)
        for (int c = 0; c < CHUNKS; ++c) n -= 8 - min(max(n_cols - (k0 + c * CHUNK), 0), 8);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) {
        counts[piece] = n;
        if (n) atomicAdd(sums + piece / BLOCK, n);  // whole numbers: the order does not matter
    }
}

// Entries in front of a warp's piece, for each warp of a block of neighbouring pieces.
__device__ __forceinline__ long long entries_before(long long piece, const int *counts, const int *sums) {
    const int lane = threadIdx.x % 32;
    const long long block = piece / BLOCK;
    long long n = 0;
    for (long long b = lane; b < block; b += 32) n += sums[b];
    for (long long p = block * BLOCK + lane; p < piece; p += 32) n += counts[p];
    for (int d = 16; d; d /= 2) n += __shfl_xor_sync(0xffffffffu, n, d);
    return n;
}

template <typename V>
struct Out {
    int n_rows, n_cols, group, n_groups, per_row;
    uint8_t *codes;
    long long code_ld;
    V *scales;
    uint8_t *zeros;
    const int *counts, *sums;  // residual only
    int *res_ptr, *res_col;
    V *res_val;
    int res_cap;
};

__device__ __forceinline__ int clamped(long long n) { return (int)min(n, (long long)INT_MAX); }

// Entries of eight neighbouring columns that go to the residual, lanes in order; `at`: the warp's place.
template <typename V, typename W>
__device__ __forceinline__ void hand_out(const Out<V> &o, const float (&v)[8], unsigned far, int k, long long &at) {
    const int n = __popc(far), lane = threadIdx.x % 32;
    if (!__any_sync(0xffffffffu, n)) return;
    int before = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += u;
    }
    long long e = at + before - n;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (far >> j & 1) {
            if (e < o.res_cap) {
                o.res_col[e] = k + j;
                o.res_val[e] = from_float<V>(v[j]);
            }
            ++e;
        }
    at += __shfl_sync(0xffffffffu, before, 31);
}

// One warp a piece, for groups of 32, 64, ... 2048 columns: SPAN chunks a group (1: up to 256 columns, lanes of one chunk).
// Reading W is what bounds it; the division by the scale is a multiplication unless a value comes near a border.
template <typename V, typename W, bool ZEROS, int SPAN>
__global__ void __launch_bounds__(32 * WARPS) quantize_kernel(const Out<V> o, const W *w, long long ld, bool wide,
                                                              float threshold) {
    const long long piece = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (piece >= (long long)o.n_rows * o.per_row) return;
    const int row = (int)(piece / o.per_row), start = (int)(piece % o.per_row) * PIECE;
    const W *from = w + row * ld;
    uint8_t *codes = o.codes + row * o.code_ld;
    const int lanes = SPAN > 1 ? 32 : o.group / 8;  // that share a group in a chunk
    Raw<W> raw[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) raw[c].load(from, start + c * CHUNK + 8 * lane, o.n_cols, wide);
    const bool split = o.res_ptr != nullptr;
    long long at = 0;
    if (split) {
        at = entries_before(piece, o.counts, o.sums);
        if (lane == 0 && start + PIECE >= o.n_cols) o.res_ptr[row + 1] = clamped(at + o.counts[piece]);
        if (lane == 0 && piece == 0) o.res_ptr[0] = 0;
    }
#pragma unroll
    for (int c0 = 0; c0 < CHUNKS; c0 += SPAN) {
        if (start + c0 * CHUNK >= o.n_cols) break;
        float lo = 0.f, hi = 0.f;
        bool nan = false;
#pragma unroll
        for (int c = c0; c < c0 + SPAN; ++c) {
            float v[8];
            raw[c].values(v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = split && fabsf(v[j]) > threshold ? 0.f : v[j];
                if (ZEROS) {
                    lo = fminf(lo, x);
                    hi = fmaxf(hi, x);
                } else {
                    hi = fmaxf(hi, fabsf(x));
                }
                nan |= x != x;
            }
        }
        for (int d = lanes / 2; d; d /= 2) {
            if (ZEROS) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        // a NaN concerns the lanes of its own group
        const unsigned nans = __ballot_sync(0xffffffffu, nan);
        nan = (nans >> (lane & ~(lanes - 1)) & (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1)) != 0;
        const Scale<V, ZEROS> g(lo, hi, nan);
        const int k0 = start + c0 * CHUNK + 8 * lane;
        if (lane % lanes == 0 && k0 < o.n_cols) {
            const long long to = (long long)row * o.n_groups + k0 / o.group;
            o.scales[to] = g.stored;
            if (ZEROS) o.zeros[to] = (uint8_t)g.z;
        }
        // a product with the reciprocal is off by 2^-22 of itself at most, where the scale was not rounded to few bits
        const bool quick = g.usable && g.s > 6.2e-5f;
        const float inverse = quick ? 1.f / g.s : 0.f;
#pragma unroll
        for (int c = c0; c < c0 + SPAN; ++c) {
            const int k = k0 + (c - c0) * CHUNK;
            float v[8];
            raw[c].values(v);
            unsigned far = 0;
            if (split) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (fabsf(v[j]) > threshold && k + j < o.n_cols) far |= 1u << j;
                hand_out<V, W>(o, v, far, k, at);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (far >> j & 1) v[j] = 0.f;
            }
            constexpr float MAGIC = 12582912.f;  // 1.5 * 2^23: adding it rounds to whole numbers, ties to even
            const float base = MAGIC + g.z;
            float q[8], worst = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float t = v[j] * inverse;
                q[j] = __fadd_rn(t, MAGIC) - MAGIC;
                worst = fmaxf(worst, fabsf(t - q[j]));
            }
            if (__any_sync(0xffffffffu, worst > 0.499f || !quick)) {
                if (quick) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[j] = nearest_from(q[j], v[j], g.s);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[j] = g.usable ? nearest_quotient(v[j], g.s) : 0.f;
                }
            }
            uint32_t word = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = fminf(fmaxf(q[j] + base, ZEROS ? MAGIC : MAGIC + 1.f), MAGIC + 15.f);
                word |= (__float_as_uint(f) & 15u) << 4 * j;
            }
            if (k + 8 <= o.n_cols) {
                *reinterpret_cast<uint32_t *>(codes + k / 2) = word;
            } else {
                // the last bytes; a half behind the last column is 0
                for (int j = 0; j < 8 && k + j < o.n_cols; j += 2)
                    codes[(k + j) / 2] = (uint8_t)(k + j + 1 < o.n_cols ? word >> 4 * j : word >> 4 * j & 15);
            }
        }
    }
}

// Any other group: one warp a row, 64 columns (2 a lane) at a time; a group is gone through twice, for its range and for
// its codes.
template <typename V, typename W, bool ZEROS>
__global__ void quantize_any_kernel(const Out<V> o, const W *w, long long ld, float threshold) {
    const int row = blockIdx.x * WARPS + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (row >= o.n_rows) return;
    const W *wr = w + row * ld;
    uint8_t *cr = o.codes + row * o.code_ld;
    const bool split = o.res_ptr != nullptr;
    long long at = 0;
    if (split) {
        at = entries_before((long long)row * o.per_row, o.counts, o.sums);
        const long long next = entries_before((row + 1ll) * o.per_row, o.counts, o.sums);
        if (lane == 0) {
            o.res_ptr[row + 1] = clamped(next);
            if (row == 0) o.res_ptr[0] = 0;
        }
    }
    for (int g = 0; g < o.n_groups; ++g) {
        const int k0 = g * o.group, k1 = (int)min((long long)o.n_cols, (long long)k0 + o.group);
        float lo = 0.f, hi = 0.f;
        bool nan = false;
        for (int k = k0 + lane; k < k1; k += 32) {
            const float v = to_float(wr[k]);
            if (split && fabsf(v) > threshold) continue;
            lo = fminf(lo, v);
            hi = fmaxf(hi, v);
            nan |= v != v;
        }
        for (int d = 16; d; d /= 2) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        const Scale<V, ZEROS> s(lo, hi, __any_sync(0xffffffffu, nan));
        if (lane == 0) {
            o.scales[(long long)row * o.n_groups + g] = s.stored;
            if (ZEROS) o.zeros[(long long)row * o.n_groups + g] = (uint8_t)s.z;
        }
        for (int k = k0 + 2 * lane; k - 2 * lane < k1; k += 64) {
            bool far[2] = {false, false};
            int c[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (k + j < k1) {
                    const float v = to_float(wr[k + j]);
                    far[j] = split && fabsf(v) > threshold;
                    const float q = s.usable && !far[j] ? nearest_quotient(v, s.s) : 0.f;
                    c[j] = (int)fminf(fmaxf(q + s.z, ZEROS ? 0.f : 1.f), 15.f);
                }
            if (k < k1) cr[k / 2] = (uint8_t)(c[0] | c[1] << 4);
            if (split) {
                const unsigned even = __ballot_sync(0xffffffffu, far[0]), odd = __ballot_sync(0xffffffffu, far[1]);
                const unsigned below = (1u << lane) - 1;
                const long long p = at + __popc(even & below) + __popc(odd & below);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const long long e = p + (j && far[0]);
                    if (far[j] && e < o.res_cap) {
                        o.res_col[e] = k + j;
                        o.res_val[e] = from_float<V>(to_float(wr[k + j]));
                    }
                }
                at += __popc(even) + __popc(odd);
            }
        }
    }
}

// One warp a piece: the codes' values first, then the entries of the residual on top of them.
template <typename V>
__global__ void __launch_bounds__(32 * WARPS) expand_kernel(Matrix<V> m, int per_row, V *w, long long ld, bool wide) {
    const long long piece = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (piece >= (long long)m.n_rows * per_row) return;
    const int row = (int)(piece / per_row), start = (int)(piece % per_row) * PIECE;
    const uint8_t *codes = m.codes + row * m.code_ld;
    const V *scales = m.scales + (long long)row * m.n_groups;
    V *to = w + row * ld;
    uint32_t c[CHUNKS];
    V s[CHUNKS];
    int z[CHUNKS];
    GroupOf at(start + 8 * lane, m.group, CHUNK);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int k = start + j * CHUNK + 8 * lane;
        c[j] = 0;
        s[j] = from_float<V>(0.f);
        z[j] = 8;
        if (k < m.n_cols) {
            c[j] = __ldg(reinterpret_cast<const uint32_t *>(codes + k / 2));  // a row of codes ends on 16 bytes
            s[j] = scales[at.g];
            z[j] = zero_of(m, row, at.g);
        }
        at.move();
    }
    int begin = 0, end = 0;
    if (m.res_ptr) res_range(m, row, begin, end);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int k = start + j * CHUNK + 8 * lane;
        const uint4 v = values<V>(c[j], Pair<V>::both(s[j]), z[j]);
        if (wide && k + 8 <= m.n_cols) {
            *reinterpret_cast<uint4 *>(to + k) = v;
        } else {
            const V *e = reinterpret_cast<const V *>(&v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < m.n_cols) to[k + i] = e[i];
        }
    }
    if (begin >= end) return;
    __syncwarp();
    const int stop = min(m.n_cols, start + PIECE);
    for (int i = begin + lane; i < end; i += 32) {
        const int k = m.res_col[i];
        if (k < start || k >= stop || (i > begin && m.res_col[i - 1] == k)) continue;
        const int g = k / m.group, code = codes[k / 2] >> 4 * (k & 1) & 15;
        float v = to_float(scales[g]) * (float)(code - zero_of(m, row, g));
        for (int j = i; j < end && m.res_col[j] == k; ++j) v += to_float(m.res_val[j]);
        to[k] = from_float<V>(v);
    }
}

template <typename V, typename W, bool ZEROS>
cudaError_t quantize_as(const Out<V> &o, const W *w, long long ld, bool wide, float threshold, cudaStream_t s) {
    const long long blocks = ceil_div((long long)o.n_rows * o.per_row, WARPS);
    const unsigned grid = (unsigned)blocks, threads = 32 * WARPS;
    switch (o.group) {
        case 32:
        case 64:
        case 128:
        case 256: quantize_kernel<V, W, ZEROS, 1><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
        case 512: quantize_kernel<V, W, ZEROS, 2><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
        case 1024: quantize_kernel<V, W, ZEROS, 4><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
        case 2048: quantize_kernel<V, W, ZEROS, 8><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
        default:
            quantize_any_kernel<V, W, ZEROS><<<(unsigned)ceil_div(o.n_rows, WARPS), threads, 0, s>>>(o, w, ld, threshold);
    }
    return cudaGetLastError();
}

template <typename V, typename W>
cudaError_t quantize_from(const mx_q4_matrix &m, const W *w, long long ld, float threshold, cudaStream_t s) {
    if (m.n_rows == 0 || m.n_cols == 0) {
        if (!m.res_row_ptr) return cudaSuccess;
        return cudaMemsetAsync(m.res_row_ptr, 0, sizeof(int) * (m.n_rows + 1ll), s);
    }
    Out<V> o = {};
    o.n_rows = m.n_rows;
    o.n_cols = m.n_cols;
    o.group = m.group;
    o.n_groups = (int)ceil_div(m.n_cols, m.group);
    o.per_row = (int)ceil_div(m.n_cols, PIECE);
    o.codes = static_cast<uint8_t *>(m.codes);
    o.code_ld = m.code_ld;
    o.scales = static_cast<V *>(m.scales);
    o.zeros = static_cast<uint8_t *>(m.zeros);
    const bool wide = (uintptr_t)w % 16 == 0 && (m.n_rows == 1 || ld * sizeof(W) % 16 == 0);
    const long long pieces = (long long)m.n_rows * o.per_row, blocks = ceil_div(pieces, BLOCK);
    if (ceil_div(pieces, WARPS) > INT_MAX) return cudaErrorInvalidConfiguration;
    Workspace work(s);
    if (m.res_row_ptr) {
        int *counts = nullptr;
        cudaError_t e = work.take((void **)&counts, sizeof(int) * (pieces + blocks));
        if (e != cudaSuccess) return e;
        int *sums = counts + pieces;
        if ((e = cudaMemsetAsync(sums, 0, sizeof(int) * blocks, s)) != cudaSuccess) return e;
        count_kernel<<<(unsigned)ceil_div(pieces, WARPS), 32 * WARPS, 0, s>>>(m.n_rows, m.n_cols, o.per_row, w, ld, wide,
                                                                              threshold, counts, sums);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        o.counts = counts;
        o.sums = sums;
        o.res_ptr = m.res_row_ptr;
        o.res_col = m.res_col_ind;
        o.res_val = static_cast<V *>(m.res_val);
        o.res_cap = m.res_cap;
    }
    return m.zeros ? quantize_as<V, W, true>(o, w, ld, wide, threshold, s)
                   : quantize_as<V, W, false>(o, w, ld, wide, threshold, s);
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
    const int per_row = (int)ceil_div(m.n_cols, PIECE);
    const long long blocks = ceil_div((long long)m.n_rows * per_row, WARPS);
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    const bool wide = (uintptr_t)w % 16 == 0 && (m.n_rows == 1 || ld % 8 == 0);
    expand_kernel<<<(unsigned)blocks, 32 * WARPS, 0, s>>>(m, per_row, w, ld, wide);
    return cudaGetLastError();
}

#define INSTANTIATE(V)                                                                                              \
    template cudaError_t quantize<V>(const mx_q4_matrix &, int, const void *, long long, float, cudaStream_t);      \
    template cudaError_t expand<V>(const Matrix<V> &, V *, long long, cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
