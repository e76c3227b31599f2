// Products of a 4-bit matrix with few vectors (decoding), and the gradients of its numbers from few vectors.
//
// What bounds these is reading the codes once; the arithmetic only has to keep up.  Codes go from global memory to
// registers, become c - z as exact 16-bit values (no scale yet) and feed mma.sync with 32-bit sums, whose 8 columns are
// the vectors; the tensor memory path (q4_gemm.cu) costs 5 us before its first result, more than all of these calls'
// work.  The order of a contraction's terms is free, so a lane takes the codes as they lie in memory (16 bytes of a row)
// and the vectors are fetched to match.  Sums over a group's columns are taken first and multiplied by the group's scale
// in 32 bits, so that no weight is rounded.
#include <algorithm>

#include "q4.h"
#include "q4_gemm.h"
#include "q4_ptx.cuh"
#include "q4_values.cuh"

namespace mx {
namespace q4 {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;

template <typename V>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// values k .. k + 7 of a vector, 0 from `end` on; `wide`: k is on a 16-byte border
template <typename V>
__device__ __forceinline__ uint4 eight(const V *x, int k, int end, bool wide) {
    if (wide && k + 8 <= end) return __ldg(reinterpret_cast<const uint4 *>(x + k));
    V v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < end ? x[k + j] : from_float<V>(0.f);
    return *reinterpret_cast<uint4 *>(v);
}

// The 32 codes that a lane has of one row of 128 columns.  S is the width that shares a scale: the four lanes of a row
// have neighbouring quarters of every S columns, so that one mma never mixes two groups.  Word w begins at column
// place<S>(w, quarter).
template <int S>
__device__ __forceinline__ int place(int w, int quarter) {
    return S == 128 ? 32 * quarter + 8 * w : S == 64 ? 64 * (w / 2) + 16 * quarter + 8 * (w % 2) : 32 * w + 8 * quarter;
}
template <int S>
__device__ __forceinline__ void row_codes(uint32_t (&c)[4], const uint8_t *row, int k, int quarter, int row_bytes) {
    if (S == 128) {
        const int at = k / 2 + 16 * quarter;
        const uint4 v = at < row_bytes ? __ldg(reinterpret_cast<const uint4 *>(row + at)) : make_uint4(0, 0, 0, 0);
        c[0] = v.x, c[1] = v.y, c[2] = v.z, c[3] = v.w;
    } else if (S == 64) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int at = k / 2 + 32 * j + 8 * quarter;
            const uint2 v = at < row_bytes ? __ldg(reinterpret_cast<const uint2 *>(row + at)) : make_uint2(0, 0);
            c[2 * j] = v.x, c[2 * j + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = k / 2 + 16 * j + 4 * quarter;
            c[j] = at < row_bytes ? __ldg(reinterpret_cast<const uint32_t *>(row + at)) : 0;
        }
    }
}

template <typename V>
struct Few {
    Matrix<V> m;
    int n_vec, splits;
    const V *x, *dy;
    long long ld_x, ld_dy;
    bool wide_x, wide_dy;
    V *out;
    long long ld_out;
    V *d_res;
};

// d[tile] += steps of 16 rows x 8 columns (one word of two rows) times the vectors' values at those columns
template <typename V, int NT>
__device__ __forceinline__ void word_product(float (&d)[NT][4], uint32_t up, uint32_t low, int z_up, int z_low,
                                             const uint4 (&x)[NT]) {
    typename Pair<V>::T p[4], q[4];
    Pair<V>::steps(up, z_up, p);
    Pair<V>::steps(low, z_low, q);
    // codes j and j + 4 share a register; the vectors' values are paired alike
    const uint32_t a0[4] = {raw(p[0]), raw(q[0]), raw(p[1]), raw(q[1])}, a1[4] = {raw(p[2]), raw(q[2]), raw(p[3]), raw(q[3])};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mma16<V>(d[n], a0, __byte_perm(x[n].x, x[n].z, 0x5410), __byte_perm(x[n].x, x[n].z, 0x7632));
        mma16<V>(d[n], a1, __byte_perm(x[n].y, x[n].w, 0x5410), __byte_perm(x[n].y, x[n].w, 0x7632));
    }
}

// y = W x for up to 8 NT vectors.  A block has 16 rows; its warps take the 128-column pieces in turn, and the blocks of
// a cluster (where there are too few rows to occupy the GPU) take contiguous parts of them; the parts are added in the
// order of warps and ranks.
template <typename V, int S, int NT>
__global__ void __launch_bounds__(THREADS) product_few_kernel(const Few<V> g) {
    __shared__ float part[WARPS][8 * NT][17];
    __shared__ float sum[8 * NT][16];
    const Matrix<V> &m = g.m;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, line = lane / 4, quarter = lane % 4;
    const int rank = g.splits > 1 ? (int)cluster_rank() : 0, row0 = blockIdx.x / g.splits * 16;
    const int pieces = (int)(((long long)m.n_cols + 127) / 128);
    const int from = (int)((long long)pieces * rank / g.splits), to = (int)((long long)pieces * (rank + 1) / g.splits);
    const int row_bytes = (int)(((long long)m.n_cols + 31) / 32 * 16);
    const int i0 = min(row0 + line, m.n_rows - 1), i1 = min(row0 + line + 8, m.n_rows - 1);  // the last row again: unused
    const uint8_t *up = m.codes + i0 * m.code_ld, *low = m.codes + i1 * m.code_ld;
    const long long s_up = (long long)i0 * m.n_groups, s_low = (long long)i1 * m.n_groups;
    constexpr int SEGMENTS = 128 / S;

    // the residual's first entries of this warp's two rows are on their way while the codes are worked on
    int begin[2] = {0, 0}, end[2] = {0, 0};
    const bool has_residual = m.res_ptr && rank == 0;
    if (has_residual)
        for (int j = 0; j < 2; ++j)
            if (row0 + 2 * warp + j < m.n_rows) res_range(m, row0 + 2 * warp + j, begin[j], end[j]);

    float total[NT][4] = {};
    GroupOf at((from + warp) * 128, m.group, WARPS * 128);
    struct Piece {
        uint32_t up[4], low[4];
        V s_up[SEGMENTS], s_low[SEGMENTS];
        int z_up[SEGMENTS], z_low[SEGMENTS];
    };
    auto fetch = [&](Piece &p, int piece) {
        row_codes<S>(p.up, up, piece * 128, quarter, row_bytes);
        row_codes<S>(p.low, low, piece * 128, quarter, row_bytes);
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) {
            const int gr = min(at.after(j * (S / 32)), m.n_groups - 1);
            p.s_up[j] = m.scales[s_up + gr];
            p.s_low[j] = m.scales[s_low + gr];
            p.z_up[j] = m.zeros ? m.zeros[s_up + gr] & 15 : 8;
            p.z_low[j] = m.zeros ? m.zeros[s_low + gr] & 15 : 8;
        }
        at.move();
    };
    auto work = [&](const Piece &p, int piece) {
        uint4 x[4][NT];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int t = 8 * n + line;
                x[w][n] = t < g.n_vec ? eight(g.x + t * g.ld_x, piece * 128 + place<S>(w, quarter), m.n_cols, g.wide_x)
                                      : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) {
            float d[NT][4] = {};
#pragma unroll
            for (int w = j * (S / 32); w < (j + 1) * (S / 32); ++w)
                word_product<V, NT>(d, p.up[w], p.low[w], p.z_up[j], p.z_low[j], x[w]);
            const float a = to_float(p.s_up[j]), b = to_float(p.s_low[j]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                total[n][0] = fmaf(a, d[n][0], total[n][0]);
                total[n][1] = fmaf(a, d[n][1], total[n][1]);
                total[n][2] = fmaf(b, d[n][2], total[n][2]);
                total[n][3] = fmaf(b, d[n][3], total[n][3]);
            }
        }
    };
    // two pieces ahead
    Piece p[3];
    int piece = from + warp;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (piece + WARPS * j < to) fetch(p[j], piece + WARPS * j);
    int first[2];
    V value[2];
    if (has_residual)
        for (int j = 0; j < 2; ++j)
            if (begin[j] + lane < end[j]) {
                first[j] = m.res_col[begin[j] + lane];
                value[j] = m.res_val[begin[j] + lane];
            }
    while (piece < to) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            if (piece < to) {
                if (piece + 2 * WARPS < to) fetch(p[(j + 2) % 3], piece + 2 * WARPS);
                work(p[j], piece);
            }
            piece += WARPS;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[warp][8 * n + 2 * quarter + j % 2][line + 8 * (j / 2)] = total[n][j];
    if (has_residual) {
        __syncwarp();
        for (int j = 0; j < 2; ++j) {
            float r[8 * NT] = {};
            for (int e = begin[j] + lane; e < end[j]; e += 32) {
                const int k = e < begin[j] + 32 ? first[j] : m.res_col[e];
                if (k < 0 || k >= m.n_cols) continue;
                const float v = to_float(e < begin[j] + 32 ? value[j] : m.res_val[e]);
#pragma unroll
                for (int t = 0; t < 8 * NT; ++t)
                    if (t < g.n_vec) r[t] = fmaf(v, to_float(g.x[t * g.ld_x + k]), r[t]);
            }
#pragma unroll
            for (int t = 0; t < 8 * NT; ++t) {
                if (t >= g.n_vec) break;
                for (int d = 16; d; d /= 2) r[t] += __shfl_xor_sync(0xffffffffu, r[t], d);
                if (lane == 0) part[warp][t][2 * warp + j] += r[t];
            }
        }
    }
    __syncthreads();
    const int row = threadIdx.x % 16, t = threadIdx.x / 16;
    if (t < 8 * NT) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += part[w][t][row];
        if (g.splits > 1) {
            sum[t][row] = s;
        } else if (t < g.n_vec && row0 + row < m.n_rows) {
            g.out[t * g.ld_out + row0 + row] = from_float<V>(s);
        }
    }
    if (g.splits > 1) {
        __syncthreads();
        cluster_barrier();
        if (rank == 0 && t < g.n_vec && row0 + row < m.n_rows) {
            float s = 0.f;
            for (int r = 0; r < g.splits; ++r) s += cluster_load(smem_addr(&sum[t][row]), r);
            g.out[t * g.ld_out + row0 + row] = from_float<V>(s);
        }
        __syncwarp();
        cluster_barrier();
    }
}

// Gradients from up to 8 NT vectors.  A block has 16 rows and a part of the groups, a warp whole groups of them: the
// sums over a group's columns for each vector are the product's, then they are weighed with dy instead of the scale.
// S = 0: one group at a time, in pieces of 128 columns; else 128 / S groups at a time.
template <typename V, int S, int NT>
__global__ void __launch_bounds__(THREADS) grad_few_kernel(const Few<V> g) {
    const Matrix<V> &m = g.m;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, line = lane / 4, quarter = lane % 4;
    const int row0 = blockIdx.x / g.splits * 16, rank = blockIdx.x % g.splits;
    const int row_bytes = (int)(((long long)m.n_cols + 31) / 32 * 16);
    const bool real0 = row0 + line < m.n_rows, real1 = row0 + line + 8 < m.n_rows;
    const int i0 = min(row0 + line, m.n_rows - 1), i1 = min(row0 + line + 8, m.n_rows - 1);
    if (g.out) {
        const uint8_t *up = m.codes + i0 * m.code_ld, *low = m.codes + i1 * m.code_ld;
        const long long s_up = (long long)i0 * m.n_groups, s_low = (long long)i1 * m.n_groups;
        float dy[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 8 * n + 2 * quarter + j % 2;
                dy[n][j] = t < g.n_vec ? to_float(g.dy[t * g.ld_dy + (j < 2 ? i0 : i1)]) : 0.f;
            }
        constexpr int WIDTH = S ? S : 128, SEGMENTS = 128 / WIDTH;
        const int units = (m.n_groups + SEGMENTS - 1) / SEGMENTS;
        for (int u = rank * WARPS + warp; u < units; u += g.splits * WARPS) {
            const int k0 = u * SEGMENTS * m.group;
            const int k1 = S ? m.n_cols : (int)min((long long)m.n_cols, (long long)k0 + m.group);
            float d[SEGMENTS][NT][4] = {};
            int z_up[SEGMENTS], z_low[SEGMENTS];
#pragma unroll
            for (int j = 0; j < SEGMENTS; ++j) {
                const int gr = min(u * SEGMENTS + j, m.n_groups - 1);
                z_up[j] = m.zeros ? m.zeros[s_up + gr] & 15 : 8;
                z_low[j] = m.zeros ? m.zeros[s_low + gr] & 15 : 8;
            }
            for (int k = k0; k < (S ? k0 + 1 : k1); k += 128) {
                uint32_t a[4], b[4];
                row_codes<WIDTH>(a, up, k, quarter, row_bytes);
                row_codes<WIDTH>(b, low, k, quarter, row_bytes);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint4 x[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const int t = 8 * n + line;
                        x[n] = t < g.n_vec ? eight(g.x + t * g.ld_x, k + place<WIDTH>(w, quarter), k1, g.wide_x)
                                           : make_uint4(0, 0, 0, 0);
                    }
                    const int j = w / (WIDTH / 32);
                    word_product<V, NT>(d[j], a[w], b[w], z_up[j], z_low[j], x);
                }
            }
#pragma unroll
            for (int j = 0; j < SEGMENTS; ++j) {
                float e0 = 0.f, e1 = 0.f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    e0 = fmaf(dy[n][0], d[j][n][0], fmaf(dy[n][1], d[j][n][1], e0));
                    e1 = fmaf(dy[n][2], d[j][n][2], fmaf(dy[n][3], d[j][n][3], e1));
                }
#pragma unroll
                for (int x = 1; x < 4; x *= 2) {
                    e0 += __shfl_xor_sync(0xffffffffu, e0, x);
                    e1 += __shfl_xor_sync(0xffffffffu, e1, x);
                }
                const int gr = u * SEGMENTS + j;
                if (quarter == 0 && gr < m.n_groups) {
                    if (real0) g.out[s_up + gr] = from_float<V>(e0);
                    if (real1) g.out[s_low + gr] = from_float<V>(e1);
                }
            }
        }
    }
    if (g.d_res && rank == 0) {
        for (int r = 2 * warp; r < 2 * warp + 2 && row0 + r < m.n_rows; ++r) {
            const int i = row0 + r;
            int begin, end;
            res_range(m, i, begin, end);
            float dy[8 * NT];
#pragma unroll
            for (int t = 0; t < 8 * NT; ++t) dy[t] = t < g.n_vec ? to_float(g.dy[t * g.ld_dy + i]) : 0.f;
            for (int e = begin + lane; e < end; e += 32) {
                const int k = m.res_col[e];
                if (k < 0 || k >= m.n_cols) continue;
                float s = 0.f;
#pragma unroll
                for (int t = 0; t < 8 * NT; ++t)
                    if (t < g.n_vec) s = fmaf(dy[t], to_float(g.x[t * g.ld_x + k]), s);
                g.d_res[e] = from_float<V>(s);
            }
        }
    }
}

// dx = dy W for up to 8 vectors.  A block has 256 columns, its warps take 16 rows at a time; the contraction runs over
// rows, whose scales differ, so the values are s (c - z), rounded once to the type.  The blocks of a cluster share the
// rows.  A lane holds 32 columns of four rows; two rows' codes of a column are brought into one register.
constexpr int COLS = 256, VEC = 8, VEC_STRIDE = 268, WARP_PART = VEC * VEC_STRIDE;
__device__ __forceinline__ int part_at(int t, int k) { return t * VEC_STRIDE + k + k / 32; }

template <typename V>
__global__ void __launch_bounds__(THREADS) product_t_few_kernel(const Few<V> g) {
    extern __shared__ float parts[];  // [warp][vector][column], columns a little apart
    const Matrix<V> &m = g.m;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, line = lane / 4, quarter = lane % 4;
    const int rank = g.splits > 1 ? (int)cluster_rank() : 0, k0 = blockIdx.x / g.splits * COLS;
    const int steps = (int)(((long long)m.n_rows + 15) / 16);
    const int from = (int)((long long)steps * rank / g.splits), to = (int)((long long)steps * (rank + 1) / g.splits);
    const int k = k0 + 32 * line, gr = min(k / m.group, m.n_groups - 1);
    const bool inside = k < m.n_cols;
    float d[16][4] = {};
    struct Rows {
        uint32_t c[4][4];
        V s[4];
        int z[4];
        uint2 dy;
    };
    auto fetch = [&](Rows &r, int step) {
        const int i0 = step * 16 + 4 * quarter;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j;
            const bool real = inside && i < m.n_rows;
            const uint4 v = real ? __ldg(reinterpret_cast<const uint4 *>(m.codes + i * m.code_ld + k / 2)) : make_uint4(0, 0, 0, 0);
            r.c[j][0] = v.x, r.c[j][1] = v.y, r.c[j][2] = v.z, r.c[j][3] = v.w;
            r.s[j] = real ? m.scales[(long long)i * m.n_groups + gr] : from_float<V>(0.f);
            r.z[j] = real && m.zeros ? m.zeros[(long long)i * m.n_groups + gr] & 15 : 8;
        }
        r.dy = make_uint2(0, 0);
        if (line < g.n_vec) {
            const V *p = g.dy + line * g.ld_dy + i0;
            if (g.wide_dy && i0 + 4 <= m.n_rows) {
                r.dy = __ldg(reinterpret_cast<const uint2 *>(p));
            } else {
                V v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = i0 + j < m.n_rows ? p[j] : from_float<V>(0.f);
                r.dy = *reinterpret_cast<uint2 *>(v);
            }
        }
    };
    auto work = [&](const Rows &r) {
        typename Pair<V>::T s[2] = {Pair<V>::two(r.s[0], r.s[1]), Pair<V>::two(r.s[2], r.s[3])};
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // columns 8 w + 4 h .. + 3
                typename Pair<V>::T p[4], q[4];
                const int pick = h ? 0x7632 : 0x5410;
                Pair<V>::steps(__byte_perm(r.c[0][w], r.c[1][w], pick), r.z[0], r.z[1], p);
                Pair<V>::steps(__byte_perm(r.c[2][w], r.c[3][w], pick), r.z[2], r.z[3], q);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[j] = __hmul2(p[j], s[0]);
                    q[j] = __hmul2(q[j], s[1]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // columns + 2 j and + 2 j + 1
                    const uint32_t a[4] = {raw(p[2 * j]), raw(p[2 * j + 1]), raw(q[2 * j]), raw(q[2 * j + 1])};
                    mma16<V>(d[4 * w + 2 * h + j], a, r.dy.x, r.dy.y);
                }
            }
    };
    Rows r[2];
    int step = from + warp;
    if (step < to) fetch(r[0], step);
    while (step < to) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (step < to) {
                if (step + WARPS < to) fetch(r[j ^ 1], step + WARPS);
                work(r[j]);
            }
            step += WARPS;
        }
    }
    float *mine = parts + warp * WARP_PART;
#pragma unroll
    for (int c = 0; c < 16; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[part_at(2 * quarter + j % 2, 32 * line + 2 * c + j / 2)] = d[c][j];
    if (m.res_ptr) {
        // a lane a row; lanes whose entries meet in a column add one after the other, lower rows first
        __syncwarp();
        const int k1 = (int)min((long long)m.n_cols, (long long)k0 + COLS);
        for (int i0 = from * 16 + 32 * warp; i0 < min(to * 16, m.n_rows); i0 += 32 * WARPS) {
            const int i = i0 + lane;
            int at = 0, end = 0;
            float dy[VEC];
            if (i < min(to * 16, m.n_rows)) {
                res_range(m, i, at, end);
                at = first_at_least(m.res_col, at, end, k0);
            }
#pragma unroll
            for (int t = 0; t < VEC; ++t) dy[t] = at < end && t < g.n_vec ? to_float(g.dy[t * g.ld_dy + i]) : 0.f;
            while (true) {
                const int c = at < end ? m.res_col[at] : INT_MAX;
                const bool hit = c < k1;
                if (!__any_sync(0xffffffffu, hit)) break;
                const float v = hit ? to_float(m.res_val[at]) : 0.f;
                const unsigned same = __match_any_sync(0xffffffffu, hit ? c : -1 - lane);
                const int turn = __popc(same & ((1u << lane) - 1));
                const int turns = __reduce_max_sync(0xffffffffu, turn);
                for (int n = 0; n <= turns; ++n) {
                    if (hit && turn == n && c >= k0)
#pragma unroll
                        for (int t = 0; t < VEC; ++t)
                            if (t < g.n_vec) mine[part_at(t, c - k0)] += v * dy[t];
                    __syncwarp();
                }
                at += hit;
            }
        }
    }
    __syncthreads();
    const int c = threadIdx.x;  // a column
    float s[VEC];
#pragma unroll
    for (int t = 0; t < VEC; ++t) {
        s[t] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s[t] += parts[w * WARP_PART + part_at(t, c)];
    }
    if (g.splits == 1) {
#pragma unroll
        for (int t = 0; t < VEC; ++t)
            if (t < g.n_vec && k0 + c < m.n_cols) g.out[t * g.ld_out + k0 + c] = from_float<V>(s[t]);
        return;
    }
#pragma unroll
    for (int t = 0; t < VEC; ++t) parts[part_at(t, c)] = s[t];  // this thread's own places
    cluster_barrier();
    const int width = COLS / g.splits;
    for (int j = threadIdx.x; j < width * g.n_vec; j += THREADS) {
        const int t = j / width, col = rank * width + j % width;
        float total = 0.f;
        for (int q = 0; q < g.splits; ++q) total += cluster_load(smem_addr(parts + part_at(t, col)), q);
        if (k0 + col < m.n_cols) g.out[t * g.ld_out + k0 + col] = from_float<V>(total);
    }
    __syncwarp();
    cluster_barrier();
}

template <typename V>
bool on_border(const V *p, long long ld, int n_vec, int values) {
    return (uintptr_t)p % (2 * values) == 0 && (ld % values == 0 || n_vec == 1);
}

template <typename V>
cudaError_t run(void (*kernel)(Few<V>), long long blocks, int cluster, size_t smem, const Few<V> &g, cudaStream_t s) {
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1;
    return cudaLaunchKernelEx(&cfg, kernel, g);
}

// as many parts of `pieces` as bring `blocks` to the GPU's 148 SMs, a power of two up to 8, a warp's share not below one
int parts_of(long long blocks, long long pieces) {
    int n = 1;
    while (n < 8 && blocks * n * 2 <= 2 * 148 && pieces >= 2 * n * WARPS) n *= 2;
    return n;
}

template <typename V, int NT>
cudaError_t product_by_width(const Few<V> &g, long long blocks, cudaStream_t s) {
    auto kernel = g.m.group % 128 == 0  ? product_few_kernel<V, 128, NT>
                  : g.m.group % 64 == 0 ? product_few_kernel<V, 64, NT>
                                        : product_few_kernel<V, 32, NT>;
    return run<V>(kernel, blocks * g.splits, g.splits, 0, g, s);
}

template <typename V, int NT>
cudaError_t grad_by_width(const Few<V> &g, long long blocks, cudaStream_t s) {
    auto kernel = g.m.group == 64 ? grad_few_kernel<V, 64, NT> : g.m.group == 32 ? grad_few_kernel<V, 32, NT> : grad_few_kernel<V, 0, NT>;
    return run<V>(kernel, blocks * g.splits, 1, 0, g, s);
}

}  // namespace

template <typename V>
cudaError_t product(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s) {
    if (n_vec > 16) return product_many(m, n_vec, x, ld_x, y, ld_y, s);
    const long long blocks = ((long long)m.n_rows + 15) / 16;
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, ((long long)m.n_cols + 127) / 128);
    g.x = x;
    g.ld_x = ld_x;
    g.wide_x = on_border(x, ld_x, n_vec, 8);
    g.out = y;
    g.ld_out = ld_y;
    return n_vec <= 8 ? product_by_width<V, 1>(g, blocks, s) : product_by_width<V, 2>(g, blocks, s);
}

template <typename V>
cudaError_t product_t(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                      cudaStream_t s) {
    if (n_vec > VEC) return product_t_many(m, n_vec, dy, ld_dy, dx, ld_dx, s);
    const long long blocks = ((long long)m.n_cols + COLS - 1) / COLS;
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, ((long long)m.n_rows + 15) / 16);
    g.dy = dy;
    g.ld_dy = ld_dy;
    g.wide_dy = on_border(dy, ld_dy, n_vec, 4);
    g.out = dx;
    g.ld_out = ld_dx;
    constexpr size_t smem = sizeof(float) * WARPS * WARP_PART;
    const cudaError_t e = allow_smem<V, product_t_few_kernel<V>>(smem);
    return e == cudaSuccess ? run<V>(product_t_few_kernel<V>, blocks * g.splits, g.splits, smem, g, s) : e;
}

template <typename V>
cudaError_t grad(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy, V *d_scales,
                 V *d_res, cudaStream_t s) {
    if (n_vec > 16) return grad_many(m, n_vec, x, ld_x, dy, ld_dy, d_scales, d_res, s);
    const long long blocks = ((long long)m.n_rows + 15) / 16;
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, m.group <= 64 ? (m.n_groups * (long long)m.group + 127) / 128 : m.n_groups);
    g.x = x;
    g.ld_x = ld_x;
    g.wide_x = on_border(x, ld_x, n_vec, 8);
    g.dy = dy;
    g.ld_dy = ld_dy;
    g.out = d_scales;
    g.d_res = m.res_ptr ? d_res : nullptr;
    return n_vec <= 8 ? grad_by_width<V, 1>(g, blocks, s) : grad_by_width<V, 2>(g, blocks, s);
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
