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

// BYTES (8 or 16) into shared memory, of which `size` are read and the others 0
template <int BYTES>
__device__ __forceinline__ void copy(uint32_t to, const void *from, int size) {
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void close_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>  // waits for this thread's copies but those of the LATER last groups
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

// The 32 codes that a lane has of one row of 128 columns.  S is the width that shares a scale: the four lanes of a row
// have neighbouring quarters of every S columns, so that one mma never mixes two groups.  Word w begins at column
// place<S>(w, quarter).
template <int S>
__device__ __forceinline__ int place(int w, int quarter) {
    return S == 128 ? 32 * quarter + 8 * w : S == 64 ? 64 * (w / 2) + 16 * quarter + 8 * (w % 2) : 32 * w + 8 * quarter;
}
// from 64 bytes of the row in shared memory
template <int S>
__device__ __forceinline__ void row_codes(uint32_t (&c)[4], const uint8_t *row, int quarter) {
    if (S == 128) {
        const uint4 v = *reinterpret_cast<const uint4 *>(row + 16 * quarter);
        c[0] = v.x, c[1] = v.y, c[2] = v.z, c[3] = v.w;
    } else if (S == 64) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint2 v = *reinterpret_cast<const uint2 *>(row + 32 * j + 8 * quarter);
            c[2 * j] = v.x, c[2 * j + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const uint32_t *>(row + 16 * j + 4 * quarter);
    }
}

template <typename V>
struct Few {
    Matrix<V> m;
    int n_vec, splits;
    const V *x, *dy;
    long long ld_x, ld_dy;
    V *out;
    long long ld_out;
    V *d_res;
    const int *starts;  // transposed: [block of 256 columns][row] first residual entry not left of the block
};

// A warp's pieces of 32 rows x 128 columns on their way through shared memory, DEPTH at a time: the codes (64 bytes a
// row) and the vectors' values at those columns (256 bytes a vector, the sixteens of bytes in an order that keeps the
// reads below apart).  What bounds the product of one vector is the ALU pipe, which takes the codes apart: every address
// is a lane's constant plus the piece's, and 32 rows share what the vectors cost (with 16 rows and the addresses worked
// out at each use: 470 instructions for 1 KB of codes, 44 us for 16384 x 8192).
template <typename V, int S, int NT, int DEPTH>
struct Pieces {
    const uint8_t *rows[4];  // this lane's 16 bytes of rows `line` + 8 j in a piece at column 0
    const V *x;              // and its 16 bytes of the vectors
    long long ld_x;
    uint32_t ring, to;       // the ring, and where the next piece goes
    const uint8_t *from;     // where the oldest one is
    int lane, n_vec, row_bytes, slot_bytes, place_x[4];
    __device__ __forceinline__ Pieces(const Few<V> &g, int row0, uint8_t *smem, int warp, int lane)
        : x(g.x + lane / 16 * g.ld_x + lane % 16 * 8), ld_x(2 * g.ld_x), lane(lane), n_vec(g.n_vec) {
        const Matrix<V> &m = g.m;
        const int line = lane / 4, quarter = lane % 4;
        row_bytes = (int)(((long long)m.n_cols + 31) / 32 * 16) - 16 * quarter;
#pragma unroll
        for (int j = 0; j < 4; ++j)  // behind the last row the last row again: its results are not used
            rows[j] = m.codes + min(row0 + line + 8 * j, m.n_rows - 1) * m.code_ld + 16 * quarter;
        slot_bytes = bytes(n_vec) / DEPTH;
        from = smem + warp * bytes(n_vec);
        ring = to = smem_addr(from);
        const int t = min(line, n_vec - 1);  // the columns of a product behind the last vector are not used
#pragma unroll
        for (int w = 0; w < 4; ++w) place_x[w] = 2048 + t * 256 + ((place<S>(w, quarter) / 8 ^ t) & 15) * 16;
    }
    static __host__ __device__ int bytes(int n_vec) { return DEPTH * (2048 + 256 * n_vec); }  // of a warp
    // k, k1: the piece's columns, and where they end
    __device__ __forceinline__ void fetch(int k, int k1) {
        const bool inside = k / 2 < row_bytes;
        const int at = inside ? k / 2 : 0, size = inside ? 16 : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) copy<16>(to + 512 * j + lane * 16, rows[j] + at, size);
        const int valid = min(max(k1 - k - lane % 16 * 8, 0), 8) * 2;
        const V *at_x = x + (valid ? k : 0);
#pragma unroll
        for (int j = 0; j < 4 * NT; ++j) {
            const int t = lane / 16 + 2 * j;
            if (t < n_vec) copy<16>(to + 2048 + t * 256 + ((lane ^ t) & 15) * 16, at_x, valid);
            at_x += ld_x;
        }
        to += slot_bytes;
        if (to == ring + DEPTH * slot_bytes) to = ring;
    }
    static __device__ __forceinline__ void arrived() {  // the oldest of DEPTH pieces
        wait_copies<DEPTH - 1>();
        __syncwarp();
    }
    __device__ __forceinline__ void free() {  // the oldest piece is used up
        __syncwarp();
        from += slot_bytes;
        if (smem_addr(from) == ring + DEPTH * slot_bytes) from -= DEPTH * slot_bytes;
    }
    // word w of the oldest piece's columns, of the vectors 8 j + line; codes j and j + 4 of a word share a register, and
    // the vectors' values are paired alike
    __device__ __forceinline__ void values_of(uint32_t (&v)[NT][4], int w) const {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            // 8 vectors on: 2048 bytes, and the other half of the order; behind the last vector anything will do
            const int at = j == 0 || 8 * j + lane / 4 < n_vec ? (place_x[w] ^ 128 * j) + 2048 * j : place_x[w];
            const uint4 u = *reinterpret_cast<const uint4 *>(from + at);
            v[j][0] = __byte_perm(u.x, u.z, 0x5410);
            v[j][1] = __byte_perm(u.x, u.z, 0x7632);
            v[j][2] = __byte_perm(u.y, u.w, 0x5410);
            v[j][3] = __byte_perm(u.y, u.w, 0x7632);
        }
    }
};

// d += 16 rows x 8 columns (a word of the upper and of the lower eight rows) times the vectors' values
template <typename V, int NT>
__device__ __forceinline__ void word_product(float (&d)[NT][4], uint32_t up, uint32_t low, int z_up, int z_low,
                                             const uint32_t (&x)[NT][4]) {
    typename Pair<V>::T p[4], q[4];
    Pair<V>::steps(up, z_up, p);
    Pair<V>::steps(low, z_low, q);
    const uint32_t a0[4] = {raw(p[0]), raw(q[0]), raw(p[1]), raw(q[1])}, a1[4] = {raw(p[2]), raw(q[2]), raw(p[3]), raw(q[3])};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mma16<V>(d[n], a0, x[n][0], x[n][1]);
        mma16<V>(d[n], a1, x[n][2], x[n][3]);
    }
}

// Scales (bits 0-15) and zero points (from bit 16) of a piece's 32 rows, a lane a row, in its SEGMENTS groups.
template <int SEGMENTS>
struct Numbers {
    uint32_t v[SEGMENTS];
};

constexpr int ROWS = 32;

// y = W x for up to 8 NT vectors.  A block has 32 rows; its warps take the 128-column pieces in turn, and the blocks of
// a cluster (where there are too few rows to occupy the GPU) take contiguous parts of them; the parts are added in the
// order of warps and ranks.
template <typename V, int S, int NT, int DEPTH>
__global__ void __launch_bounds__(THREADS, 2) product_few_kernel(const __grid_constant__ Few<V> g) {
    extern __shared__ uint4 smem[];
    __shared__ float part[WARPS][8 * NT][ROWS + 1];
    __shared__ float sum[8 * NT][ROWS];
    const Matrix<V> &m = g.m;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, line = lane / 4, quarter = lane % 4;
    const int rank = g.splits > 1 ? (int)cluster_rank() : 0, row0 = blockIdx.x / g.splits * ROWS;
    const int pieces = (int)(((long long)m.n_cols + 127) / 128);
    const int from = (int)((long long)pieces * rank / g.splits), to = (int)((long long)pieces * (rank + 1) / g.splits);
    constexpr int SEGMENTS = 128 / S;
    Pieces<V, S, NT, DEPTH> ring(g, row0, reinterpret_cast<uint8_t *>(smem), warp, lane);
    int ahead = from + warp;  // the piece to fetch next
#pragma unroll
    for (int n = 0; n < DEPTH - 1; ++n) {
        if (ahead < to) ring.fetch(ahead * 128, m.n_cols);
        close_copies();
        ahead += WARPS;
    }
    GroupOf at((from + warp) * 128, m.group, WARPS * 128);
    const long long my_row = (long long)min(row0 + lane, m.n_rows - 1) * m.n_groups;
    const uint16_t *scales = reinterpret_cast<const uint16_t *>(m.scales) + my_row;
    const uint8_t *zeros = m.zeros + my_row;
    Numbers<SEGMENTS> next;
    auto numbers = [&] {
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) {
            const int gr = j == 0 ? at.g : min(at.after(j * (S / 32)), m.n_groups - 1);
            next.v[j] = scales[gr];
            if (m.zeros) next.v[j] |= (uint32_t)(zeros[gr] & 15) << 16;
        }
        at.move();
    };
    if (from + warp < to) numbers();

    // the residual, while the first pieces are on their way: four rows a warp
    if (m.res_ptr && rank == 0) {
        int begin = 0, end = 0;
        if (lane < 4 && row0 + 4 * warp + lane < m.n_rows) res_range(m, row0 + 4 * warp + lane, begin, end);
        for (int j = 0; j < 4; ++j) {
            const int b = __shfl_sync(0xffffffffu, begin, j), e1 = __shfl_sync(0xffffffffu, end, j);
            float extra[8 * NT] = {};
            for (int e = b + lane; e < e1; e += 32) {
                const int k = m.res_col[e];
                const float v = to_float(m.res_val[e]);
                if (k < 0 || k >= m.n_cols) continue;
#pragma unroll
                for (int t = 0; t < 8 * NT; ++t)
                    if (t < g.n_vec) extra[t] = fmaf(v, to_float(g.x[t * g.ld_x + k]), extra[t]);
            }
            __syncwarp();
#pragma unroll
            for (int t = 0; t < 8 * NT; ++t) {
                if (t >= g.n_vec) break;
                for (int d = 16; d; d /= 2) extra[t] += __shfl_xor_sync(0xffffffffu, extra[t], d);
                if (lane == 0) sum[t][4 * warp + j] = extra[t];
            }
        }
    }

    float total[2][NT][4] = {};
    for (int piece = from + warp; piece < to; piece += WARPS) {
        const Numbers<SEGMENTS> now = next;
        if (ahead < to) ring.fetch(ahead * 128, m.n_cols);
        close_copies();
        ahead += WARPS;
        if (piece + WARPS < to) numbers();
        ring.arrived();
        uint32_t c[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) row_codes<S>(c[j], ring.from + 512 * j + line * 64, quarter);
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) {
            float d[2][NT][4] = {};
            int z[4] = {8, 8, 8, 8};
            float s[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t v = __shfl_sync(0xffffffffu, now.v[j], line + 8 * r);
                const uint16_t bits = (uint16_t)v;
                s[r] = to_float(*reinterpret_cast<const V *>(&bits));
                if (m.zeros) z[r] = v >> 16;
            }
#pragma unroll
            for (int w = j * (S / 32); w < (j + 1) * (S / 32); ++w) {
                uint32_t x[NT][4];
                ring.values_of(x, w);
                word_product<V, NT>(d[0], c[0][w], c[1][w], z[0], z[1], x);
                word_product<V, NT>(d[1], c[2][w], c[3][w], z[2], z[3], x);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < NT; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[h][q][e] = fmaf(s[2 * h + e / 2], d[h][q][e], total[h][q][e]);
        }
        ring.free();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                part[warp][8 * n + 2 * quarter + j % 2][line + 8 * (j / 2) + 16 * h] = total[h][n][j];
    __syncthreads();
    const int row = lane;
    for (int t = warp; t < g.n_vec; t += WARPS) {
        float s = m.res_ptr && rank == 0 ? sum[t][row] : 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += part[w][t][row];
        if (g.splits > 1) {
            sum[t][row] = s;
        } else if (row0 + row < m.n_rows) {
            g.out[t * g.ld_out + row0 + row] = from_float<V>(s);
        }
    }
    if (g.splits > 1) {
        __syncthreads();
        cluster_barrier();
        if (rank == 0) {
            for (int t = warp; t < g.n_vec; t += WARPS) {
                float s = 0.f;
                for (int r = 0; r < g.splits; ++r) s += cluster_load(smem_addr(&sum[t][row]), r);
                if (row0 + row < m.n_rows) g.out[t * g.ld_out + row0 + row] = from_float<V>(s);
            }
        }
        __syncwarp();
        cluster_barrier();
    }
}

// Gradients from up to 8 NT vectors.  A block has 32 rows and a part of the groups, a warp whole groups of them: the
// sums over a group's columns for each vector are the product's, then they are weighed with dy instead of the scale.
// S = 0: one group after the other, in pieces of 128 columns; else a piece has 128 / S groups.
template <typename V, int S, int NT, int DEPTH>
__global__ void __launch_bounds__(THREADS, 2) grad_few_kernel(const __grid_constant__ Few<V> g) {
    extern __shared__ uint4 smem[];
    const Matrix<V> &m = g.m;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, line = lane / 4, quarter = lane % 4;
    const int row0 = blockIdx.x / g.splits * ROWS, rank = blockIdx.x % g.splits;
    constexpr int WIDTH = S ? S : 128, SEGMENTS = 128 / WIDTH;
    const int units = (m.n_groups + SEGMENTS - 1) / SEGMENTS, stride = g.splits * WARPS, width = SEGMENTS * m.group;
    // a place in the warp's order of pieces: its unit, and where its columns begin and end
    struct Place {
        int unit, k, k1;
    };
    auto enter = [&](int unit) {
        const long long k = (long long)unit * width;
        return Place{unit, (int)min(k, (long long)INT_MAX), (int)min((long long)m.n_cols, k + width)};
    };
    auto move = [&](Place &p) {
        p.k += 128;
        if (S || p.k >= p.k1) p = enter(p.unit + stride);
    };
    Place here = enter(g.out ? rank * WARPS + warp : units), ahead = here;
    Pieces<V, WIDTH, NT, DEPTH> ring(g, row0, reinterpret_cast<uint8_t *>(smem), warp, lane);
#pragma unroll
    for (int n = 0; n < DEPTH - 1; ++n) {
        if (ahead.unit < units) {
            ring.fetch(ahead.k, ahead.k1);
            move(ahead);
        }
        close_copies();
    }
    if (g.d_res && rank == 0) {
        for (int r = 4 * warp; r < 4 * warp + 4 && row0 + r < m.n_rows; ++r) {
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
    long long of_row[4];
    float dy[4][NT][2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = min(row0 + line + 8 * r, m.n_rows - 1);
        of_row[r] = (long long)i * m.n_groups;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int t = 8 * n + 2 * quarter + j;
                dy[r][n][j] = t < g.n_vec ? to_float(g.dy[t * g.ld_dy + i]) : 0.f;
            }
    }
    const uint8_t *zeros = m.zeros + (long long)min(row0 + lane, m.n_rows - 1) * m.n_groups;
    float d[SEGMENTS][2][NT][4] = {};
    int next[SEGMENTS];
    auto fetch_zeros = [&](int unit) {
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) next[j] = m.zeros ? zeros[min(unit * SEGMENTS + j, m.n_groups - 1)] & 15 : 8;
    };
    if (here.unit < units) fetch_zeros(here.unit);
    while (here.unit < units) {
        int now[SEGMENTS];
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) now[j] = next[j];
        if (ahead.unit < units) {
            ring.fetch(ahead.k, ahead.k1);
            move(ahead);
        }
        close_copies();
        const Place was = here;
        move(here);
        if (here.unit < units) fetch_zeros(here.unit);
        ring.arrived();
        uint32_t c[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) row_codes<WIDTH>(c[j], ring.from + 512 * j + line * 64, quarter);
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) {
            int z[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] = m.zeros ? __shfl_sync(0xffffffffu, now[j], line + 8 * r) : 8;
#pragma unroll
            for (int w = j * (WIDTH / 32); w < (j + 1) * (WIDTH / 32); ++w) {
                uint32_t x[NT][4];
                ring.values_of(x, w);
                word_product<V, NT>(d[j][0], c[0][w], c[1][w], z[0], z[1], x);
                word_product<V, NT>(d[j][1], c[2][w], c[3][w], z[2], z[3], x);
            }
        }
        ring.free();
        if (here.unit == was.unit) continue;  // more of the group to come
#pragma unroll
        for (int j = 0; j < SEGMENTS; ++j) {
            const int gr = was.unit * SEGMENTS + j;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float e = 0.f;
#pragma unroll
                for (int q = 0; q < NT; ++q)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float &v = d[j][r / 2][q][2 * (r % 2) + t];
                        e = fmaf(dy[r][q][t], 8 * q + 2 * quarter + t < g.n_vec ? v : 0.f, e);
                        v = 0.f;
                    }
                e += __shfl_xor_sync(0xffffffffu, e, 1);
                e += __shfl_xor_sync(0xffffffffu, e, 2);
                if (quarter == 0 && gr < m.n_groups && row0 + line + 8 * r < m.n_rows)
                    g.out[of_row[r] + gr] = from_float<V>(e);
            }
        }
    }
}

// starts[b][i] = first entry of row i with a column not below 256 b, for b = 0 .. blocks; 32 rows and 64 blocks of
// columns at a time, so that both the entries and the results are touched in order.
template <typename V>
__global__ void __launch_bounds__(256) starts_kernel(Matrix<V> m, int blocks, int chunks, int *starts) {
    __shared__ int part[64][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int row0 = blockIdx.x / chunks * 32, b0 = blockIdx.x % chunks * 64;
    for (int r = warp; r < 32 && row0 + r < m.n_rows; r += 8) {
        int begin, end;
        res_range(m, row0 + r, begin, end);
        begin = first_at_least(m.res_col, begin, end, (int)min(b0 * 256ll, (long long)INT_MAX));
        int before = b0 - 1;  // block of the entry in front
        for (int e = begin + lane; before < b0 + 63; e += 32) {
            // behind the last entry everything starts at the end
            const int b = e < end ? min(max(m.res_col[e] / 256, b0 - 1), b0 + 63) : b0 + 63;
            int left = __shfl_up_sync(0xffffffffu, b, 1);
            if (lane == 0) left = before;
            for (int k = left + 1; k <= b; ++k) part[k - b0][r] = min(e, end);
            before = __shfl_sync(0xffffffffu, b, 31);
        }
    }
    __syncthreads();
    for (int k = warp; k < 64 && b0 + k <= blocks; k += 8)
        if (row0 + lane < m.n_rows) starts[(long long)(b0 + k) * m.n_rows + row0 + lane] = part[k][lane];
}

// dx = dy W for up to 8 vectors.  A block has 256 columns, its warps take 16 rows at a time; the contraction runs over
// rows, whose scales differ, so the values are s (c - z), rounded once to the type.  The blocks of a cluster share the
// rows.  A lane holds 32 columns of four rows; two rows' codes of a column are brought into one register.
constexpr int COLS = 256, VEC = 8, VEC_STRIDE = 268, WARP_PART = VEC * VEC_STRIDE;
constexpr int T_DEPTH = 4, T_SLOT = 2048 + 256;  // steps of a warp under way; bytes of one: codes, dy
constexpr int T_SMEM = WARPS * (T_DEPTH * T_SLOT > 4 * WARP_PART ? T_DEPTH * T_SLOT : 4 * WARP_PART);
__device__ __forceinline__ int part_at(int t, int k) { return t * VEC_STRIDE + k + k / 32; }

template <typename V>
__global__ void __launch_bounds__(THREADS, 2) product_t_few_kernel(const __grid_constant__ Few<V> g) {
    extern __shared__ uint4 smem[];
    float *parts = reinterpret_cast<float *>(smem);  // in the end: [warp][vector][column], columns a little apart
    const Matrix<V> &m = g.m;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, line = lane / 4, quarter = lane % 4;
    const int rank = g.splits > 1 ? (int)cluster_rank() : 0, k0 = blockIdx.x / g.splits * COLS;
    const int steps = (int)(((long long)m.n_rows + 15) / 16);
    const int from = (int)((long long)steps * rank / g.splits), to = (int)((long long)steps * (rank + 1) / g.splits);
    const int count = from + warp < to ? (to - from - warp - 1) / WARPS + 1 : 0;
    const int k = k0 + 32 * line, gr = min(k / m.group, m.n_groups - 1);
    const bool inside = k < m.n_cols;
    uint8_t *ring = reinterpret_cast<uint8_t *>(smem) + warp * T_DEPTH * T_SLOT + lane * 16;
    auto rows_of = [&](int n) { return (from + warp + n * WARPS) * 16 + 4 * quarter; };
    auto fetch = [&](int n) {
        const uint32_t slot = smem_addr(ring) + n % T_DEPTH * T_SLOT;
        const int i0 = rows_of(n);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool real = inside && i0 + j < m.n_rows;
            copy<16>(slot + 512 * j, m.codes + (real ? (i0 + j) * m.code_ld + k / 2 : 0), real ? 16 : 0);
        }
        if (line < g.n_vec) {
            const int size = min(max(m.n_rows - i0, 0), 4) * 2;
            copy<8>(slot + 2048 - lane * 8, g.dy + line * g.ld_dy + (size ? i0 : 0), size);
        }
    };
#pragma unroll
    for (int n = 0; n < T_DEPTH - 1; ++n) {
        if (n < count) fetch(n);
        close_copies();
    }
    V scale[4];
    int z[4];
    auto scales = [&](int n) {
        const int i0 = rows_of(n);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool real = inside && i0 + j < m.n_rows;
            scale[j] = real ? m.scales[(long long)(i0 + j) * m.n_groups + gr] : from_float<V>(0.f);
            z[j] = real && m.zeros ? m.zeros[(long long)(i0 + j) * m.n_groups + gr] & 15 : 8;
        }
    };
    if (count > 0) scales(0);
    float d[16][4] = {};
    for (int n = 0; n < count; ++n) {
        const typename Pair<V>::T s0 = Pair<V>::two(scale[0], scale[1]), s1 = Pair<V>::two(scale[2], scale[3]);
        const int z0 = z[0], z1 = z[1], z2 = z[2], z3 = z[3];
        if (n + T_DEPTH - 1 < count) fetch(n + T_DEPTH - 1);
        close_copies();
        if (n + 1 < count) scales(n + 1);
        wait_copies<T_DEPTH - 1>();
        const uint8_t *slot = ring + n % T_DEPTH * T_SLOT;
        // behind the last vector anything will do
        const uint2 dy = *reinterpret_cast<const uint2 *>(slot + 2048 - lane * 8);
        uint32_t c[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 v = *reinterpret_cast<const uint4 *>(slot + 512 * j);
            c[j][0] = v.x, c[j][1] = v.y, c[j][2] = v.z, c[j][3] = v.w;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // columns 8 w + 4 h .. + 3
                typename Pair<V>::T p[4], q[4];
                const int pick = h ? 0x7632 : 0x5410;
                Pair<V>::steps(__byte_perm(c[0][w], c[1][w], pick), z0, z1, p);
                Pair<V>::steps(__byte_perm(c[2][w], c[3][w], pick), z2, z3, q);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[j] = __hmul2(p[j], s0);
                    q[j] = __hmul2(q[j], s1);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // columns + 2 j and + 2 j + 1
                    const uint32_t a[4] = {raw(p[2 * j]), raw(p[2 * j + 1]), raw(q[2 * j]), raw(q[2 * j + 1])};
                    mma16<V>(d[4 * w + 2 * h + j], a, dy.x, dy.y);
                }
            }
    }
    __syncthreads();  // every ring is empty
    float *mine = parts + warp * WARP_PART;
#pragma unroll
    for (int c = 0; c < 16; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[part_at(2 * quarter + j % 2, 32 * line + 2 * c + j / 2)] = d[c][j];
    if (m.res_ptr) {
        // a lane a row; lanes whose entries meet in a column add one after the other, lower rows first
        __syncwarp();
        const int k1 = (int)min((long long)m.n_cols, (long long)k0 + COLS), last = min(to * 16, m.n_rows);
        const int *starts = g.starts + (long long)(k0 / COLS) * m.n_rows;
        for (int i0 = from * 16 + 32 * warp; i0 < last; i0 += 32 * WARPS) {
            const int i = i0 + lane;
            int at = i < last ? starts[i] : 0;
            const int end = i < last ? starts[m.n_rows + i] : 0;
            float dy[VEC];
#pragma unroll
            for (int t = 0; t < VEC; ++t) dy[t] = at < end && t < g.n_vec ? to_float(g.dy[t * g.ld_dy + i]) : 0.f;
            while (__any_sync(0xffffffffu, at < end)) {
                constexpr int TOGETHER = 4;
                int col[TOGETHER];
                V val[TOGETHER];
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) {
                    col[j] = at + j < end ? m.res_col[at + j] : INT_MAX;
                    val[j] = at + j < end ? m.res_val[at + j] : from_float<V>(0.f);
                }
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) {
                    const bool hit = col[j] >= k0 && col[j] < k1;
                    if (!__any_sync(0xffffffffu, hit)) continue;
                    const float v = to_float(val[j]);
                    const unsigned same = __match_any_sync(0xffffffffu, hit ? col[j] : -1 - lane);
                    const int turn = __popc(same & ((1u << lane) - 1));
                    const int turns = __reduce_max_sync(0xffffffffu, turn);
                    for (int n = 0; n <= turns; ++n) {
                        if (hit && turn == n) {
#pragma unroll
                            for (int t = 0; t < VEC; ++t)
                                if (t < g.n_vec) mine[part_at(t, col[j] - k0)] += v * dy[t];
                        }
                        __syncwarp();
                    }
                }
                at += TOGETHER;
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

// sums over no vectors: 0 for every scale and every residual entry that there is
template <typename V>
__global__ void no_gradient_kernel(Matrix<V> m, V *d_scales, V *d_res) {
    const int warp = (blockIdx.x * THREADS + threadIdx.x) / 32, lane = threadIdx.x % 32;
    if (warp >= m.n_rows) return;
    if (d_scales)
        for (int j = lane; j < m.n_groups; j += 32) d_scales[(long long)warp * m.n_groups + j] = from_float<V>(0.f);
    if (!d_res) return;
    int begin, end;
    res_range(m, warp, begin, end);
    for (int e = begin + lane; e < end; e += 32) d_res[e] = from_float<V>(0.f);
}
template <typename V>
cudaError_t no_gradient(const Matrix<V> &m, V *d_scales, V *d_res, cudaStream_t s) {
    no_gradient_kernel<<<(unsigned)ceil_div(m.n_rows, WARPS), THREADS, 0, s>>>(m, d_scales, d_res);
    return cudaGetLastError();
}

template <typename V>
cudaError_t run(void (*kernel)(const Few<V>), long long blocks, int cluster, size_t smem, const Few<V> &g, cudaStream_t s) {
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

template <typename V, auto KERNEL>
cudaError_t run_ring(const Few<V> &g, long long blocks, int cluster, int warp_bytes, cudaStream_t s) {
    const cudaError_t e = allow_smem<V, KERNEL>(WARPS * 3 * (2048 + 256 * 8));
    return e == cudaSuccess ? run<V>(KERNEL, blocks, cluster, WARPS * warp_bytes, g, s) : e;
}

// Pieces under way: four a warp for one or two vectors, three or two for more, whose values take more room, so that two
// blocks fit an SM.
template <typename V, int S>
cudaError_t product_of_width(const Few<V> &g, long long blocks, cudaStream_t s) {
    blocks *= g.splits;
    if (g.n_vec <= 2)
        return run_ring<V, product_few_kernel<V, S, 1, 4>>(g, blocks, g.splits, Pieces<V, S, 1, 4>::bytes(g.n_vec), s);
    if (g.n_vec <= 8)
        return run_ring<V, product_few_kernel<V, S, 1, 3>>(g, blocks, g.splits, Pieces<V, S, 1, 3>::bytes(g.n_vec), s);
    return run_ring<V, product_few_kernel<V, S, 2, 2>>(g, blocks, g.splits, Pieces<V, S, 2, 2>::bytes(g.n_vec), s);
}

template <typename V, int S>
cudaError_t grad_of_width(const Few<V> &g, long long blocks, cudaStream_t s) {
    blocks *= g.splits;
    if (g.n_vec <= 2)
        return run_ring<V, grad_few_kernel<V, S, 1, 4>>(g, blocks, 1, Pieces<V, S, 1, 4>::bytes(g.n_vec), s);
    if (g.n_vec <= 8)
        return run_ring<V, grad_few_kernel<V, S, 1, 3>>(g, blocks, 1, Pieces<V, S, 1, 3>::bytes(g.n_vec), s);
    return run_ring<V, grad_few_kernel<V, S, 2, 2>>(g, blocks, 1, Pieces<V, S, 2, 2>::bytes(g.n_vec), s);
}

}  // namespace

template <typename V>
cudaError_t product(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s) {
    if (n_vec > 16) return product_many(m, n_vec, x, ld_x, y, ld_y, s);
    const long long blocks = ceil_div(m.n_rows, ROWS);
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, ceil_div(m.n_cols, 128));
    g.out = y;
    g.ld_out = ld_y;
    Workspace work(s);
    cudaError_t e = aligned_rows(x, ld_x, m.n_cols, n_vec, work, &g.x, &g.ld_x);
    if (e != cudaSuccess) return e;
    return m.group % 128 == 0  ? product_of_width<V, 128>(g, blocks, s)
           : m.group % 64 == 0 ? product_of_width<V, 64>(g, blocks, s)
                               : product_of_width<V, 32>(g, blocks, s);
}

template <typename V>
cudaError_t product_t(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                      cudaStream_t s) {
    if (n_vec > VEC) return product_t_many(m, n_vec, dy, ld_dy, dx, ld_dx, s);
    const long long blocks = ceil_div(m.n_cols, COLS);
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, ceil_div(m.n_rows, 16));
    g.out = dx;
    g.ld_out = ld_dx;
    Workspace work(s);
    cudaError_t e = aligned_rows(dy, ld_dy, m.n_rows, n_vec, work, &g.dy, &g.ld_dy);
    if (e == cudaSuccess) e = allow_smem<V, product_t_few_kernel<V>>(T_SMEM);
    if (e == cudaSuccess && m.res_ptr && m.n_rows > 0) {
        const long long chunks = ceil_div(blocks + 1, 64), grid = ceil_div(m.n_rows, 32) * chunks;
        int *starts = nullptr;
        if (grid > INT_MAX) return cudaErrorMemoryAllocation;
        if ((e = work.take((void **)&starts, sizeof(int) * (blocks + 1) * m.n_rows)) != cudaSuccess) return e;
        starts_kernel<<<(unsigned)grid, 256, 0, s>>>(m, (int)blocks, (int)chunks, starts);
        e = cudaGetLastError();
        g.starts = starts;
    }
    return e == cudaSuccess ? run<V>(product_t_few_kernel<V>, blocks * g.splits, g.splits, T_SMEM, g, s) : e;
}

template <typename V>
cudaError_t grad(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy, V *d_scales,
                 V *d_res, cudaStream_t s) {
    if (n_vec > 16) return grad_many(m, n_vec, x, ld_x, dy, ld_dy, d_scales, d_res, s);
    if (n_vec == 0) return no_gradient(m, d_scales, m.res_ptr ? d_res : nullptr, s);
    const long long blocks = ceil_div(m.n_rows, ROWS);
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, m.group <= 64 ? ceil_div(m.n_groups * (long long)m.group, 128) : m.n_groups);
    g.dy = dy;
    g.ld_dy = ld_dy;
    g.out = d_scales;
    g.d_res = m.res_ptr ? d_res : nullptr;
    Workspace work(s);
    cudaError_t e = aligned_rows(x, ld_x, m.n_cols, n_vec, work, &g.x, &g.ld_x);
    if (e != cudaSuccess) return e;
    return m.group == 64   ? grad_of_width<V, 64>(g, blocks, s)
           : m.group == 32 ? grad_of_width<V, 32>(g, blocks, s)
                           : grad_of_width<V, 0>(g, blocks, s);
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
