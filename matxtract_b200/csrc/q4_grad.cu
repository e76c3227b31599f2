// Gradients of a 4-bit matrix's own numbers from many vectors, on the fifth-generation tensor cores.
//
//   G[i][k] = sum_t dy[t][i] x[t][k]      A = dy's columns, B = x's columns, both line-major
//   d_scales[i][g] = sum over the group's k of (c - z)[i][k] G[i][k],   d_res[e] = G[row of e][column of e]
//
// G is never stored: it stays in tensor memory and is reduced against the codes from there.  A pair of blocks computes 256
// rows x 256 columns of it: each brings its 128 rows' dy and half of the columns' x into its shared memory, so that a
// step's operands cross the L2 and the shared memories half as often as with a block on its own.  The pairs go on from
// tile to tile, and the tensor memory holds two, so that one is reduced while the next is computed.
//
// Measured, bfloat16: 8192 x 8192, 2048 vectors 169 us, with a residual 173 (1.6 PFLOP/s: the tensor cores and the L2 that
// feeds them bound it); 16384 x 8192, 64 vectors 64 to 78 us (it goes by where the matrix lies): a tile's one step of matrix
// work is followed by 65,536 numbers to weigh, a chain of loads from tensor memory and sums (issue slots 54 %, tensor pipe
// 12 %); with a residual of 0.5 % of the entries 150 to 179: a search for the place of its entries in every row and tile.
// Searched for in front, by a kernel of its own, that was 144 for 167, but 2 to 3 us more for everything smaller.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "q4.h"
#include "q4_gemm.h"
#include "q4_maps.h"
#include "q4_ptx.cuh"
#include "q4_values.cuh"

namespace mx {
namespace q4 {
namespace {

// Warps: 0 and 2 copies, 1 tensor core issue (of block 0), 3 none; then four groups of four that reduce.
constexpr int REDUCE = 4, THREADS = 32 * 20;
constexpr int HALF = 128 * 64 * 2;  // bytes of 128 lines x 64 deep: a block's part of A, and of B
constexpr int STAGE = 2 * HALF, STAGES = 6, COLS = 256;
constexpr int PART = 136, SUMS = 8 * PART;  // parts of the scales' gradients: [32 columns][row], a little apart
constexpr int BARS = 2 * STAGES + 7;
constexpr int SMEM = 1024 + STAGES * STAGE + 2 * SUMS * 4 + BARS * 8;
static_assert(SMEM <= 227 * 1024, "shared memory of one block");

template <typename V>
struct Args {
    Matrix<V> m;
    int n_vec, tiles_m, units, groups_per_unit;
    V *d_scales, *d_res;
};

__device__ int wait_ran_out_grad;

// entries of one row, columns ascending, the next two already loaded
template <typename V>
struct Cursor {
    unsigned at = 0, end = 0;
    int col[2];
    __device__ __forceinline__ void fetch(const Matrix<V> &m, int j) {
        const unsigned p = at + j;
        col[j] = p < end ? m.res_col[p] : 0x7fffffff;
    }
    __device__ __forceinline__ void start(const Matrix<V> &m, int i, int k) {
        at = end = 0;
        if (m.res_ptr && i < m.n_rows) {
            res_range(m, i, at, end);
            at = first_at_least(m.res_col, at, end, k);
        }
        fetch(m, 0);
        fetch(m, 1);
    }
    __device__ __forceinline__ void next(const Matrix<V> &m) {
        ++at;
        col[0] = col[1];
        fetch(m, 1);
    }
};

// Two 32-bit numbers in one operation.
__device__ __forceinline__ uint64_t two(uint32_t low, uint32_t high) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(low), "r"(high));
    return r;
}
__device__ __forceinline__ uint64_t two(float low, float high) { return two(__float_as_uint(low), __float_as_uint(high)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float both(uint64_t v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return __uint_as_float(a) + __uint_as_float(b);
}

// sum of (c - z) v over 32 columns.  A code that begins at bit b of a word becomes the number 2^(23 - b) + c where it
// stands, from which 2^(23 - b) + z is taken, both exact: nine operations for eight codes, and one for two sums each.
__device__ __forceinline__ float weighed(const uint4 &codes, float z, const float (&v)[32]) {
    const float n0 = -8388608.f - z, n1 = -524288.f - z, n2 = -32768.f - z, n3 = -2048.f - z, n4 = -128.f - z;
    const uint64_t n[4] = {two(n0, n1), two(n2, n3), two(n4, n2), two(n3, n4)};
    const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
    uint64_t sum[2] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t w = word[j], h = w >> 12;
        const uint64_t c[4] = {two(pick(w, 0xF, 0x4B000000), pick(w, 0xF0, 0x49000000)),
                               two(pick(w, 0xF00, 0x47000000), pick(w, 0xF000, 0x45000000)),
                               two(pick(w, 0xF0000, 0x43000000), pick(h, 0xF00, 0x47000000)),
                               two(pick(h, 0xF000, 0x45000000), pick(h, 0xF0000, 0x43000000))};
#pragma unroll
        for (int q = 0; q < 4; ++q)
            sum[q % 2] = fma2(add2(c[q], n[q]), two(v[8 * j + 2 * q], v[8 * j + 2 * q + 1]), sum[q % 2]);
    }
    return both(add2(sum[0], sum[1]));
}

template <typename V, bool RES>  // with the residual's gradient
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    gradient_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ Args<V> g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_shared;
    __shared__ volatile int failed;
    uint8_t *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    const uint32_t base = smem_addr(smem);
    float *sums = reinterpret_cast<float *>(smem + STAGES * STAGE);
    const uint32_t bars = smem_addr(sums + 2 * SUMS);
    auto full = [&](int s) { return bars + 8 * s; };               // block 0's: both blocks' parts of a stage are there
    auto empty = [&](int s) { return bars + 8 * (STAGES + s); };   // each block's: the stage is used up
    auto done = [&](int b) { return bars + 8 * (2 * STAGES + b); };         // each block's: D is complete
    auto drained = [&](int b) { return bars + 8 * (2 * STAGES + 2 + b); };  // block 0's: both blocks have taken it
    auto taken = [&](int b) { return bars + 8 * (2 * STAGES + 4 + b); };    // block 1's: its warps have taken it
    const uint32_t together = bars + 8 * (2 * STAGES + 6);                  // the sixteen warps that reduce

    const Matrix<V> &m = g.m;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t rank = cluster_rank();
    const int steps = (g.n_vec + 63) / 64, tiles = g.tiles_m * g.units, pairs = gridDim.x / 2;
    const uint32_t polls = polls_for(steps);
    // A tile: 256 rows, of which this block has 128, and a unit: the columns of a whole number of groups, in turns of 256.
    struct Tile {
        int band, unit;
    };
    const int unit_cols = g.groups_per_unit * m.group;
    auto line0 = [&](Tile t) { return t.band * 256 + 128 * (int)rank; };
    auto col0 = [&](Tile t) { return t.unit * unit_cols; };
    auto col_end = [&](Tile t) { return min(m.n_cols - col0(t), unit_cols) + col0(t); };
    auto turns = [&](Tile t) { return (min(m.n_cols - col0(t), unit_cols) + COLS - 1) / COLS; };
    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(done(b), 1);
            mbar_init(drained(b), 16 + 1);  // block 0's warps, block 1's word
            mbar_init(taken(b), 16);
        }
        mbar_init(together, 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_addr(&tmem_shared), 2 * COLS);
    const Tile first = {(int)(blockIdx.x / 2) % g.tiles_m, (int)(blockIdx.x / 2) / g.tiles_m};
    const int bands_on = pairs % g.tiles_m, units_on = pairs / g.tiles_m;
    auto go_on = [&](Tile &t) {  // to the pair's next tile
        t.band += bands_on;
        t.unit += units_on;
        if (t.band >= g.tiles_m) {
            t.band -= g.tiles_m;
            ++t.unit;
        }
    };
    tc_fence_before();
    __syncthreads();
    cluster_barrier();  // the other block's barriers are there, too
    front_is_done();
    tc_fence_after();
    const uint32_t tmem = tmem_shared;

    if ((warp == 0 || warp == 2) && lane == 0) {  // ---- this block's part of dy, or of x
        // (one thread for both had no time to spare: with its loop a little longer, a step took 550 clocks instead of 500)
        const bool of_dy = warp == 0;
        const CUtensorMap *map = of_dy ? &map_dy : &map_x;
        const uint32_t place = base + (of_dy ? 0 : HALF), bar = in_block(bars, 0);
        int n = 0;
        bool ok = true;
        Tile t = first;
        for (int at = blockIdx.x / 2; at < tiles && ok; at += pairs, go_on(t)) {
            for (int turn = 0; turn < turns(t) && ok; ++turn) {
                const int line = of_dy ? line0(t) : col0(t) + turn * COLS + 128 * (int)rank;
                for (int step = 0; step < steps; ++step, ++n) {
                    const int s = n % STAGES;
                    if (!(ok = mbar_wait(empty(s), (n / STAGES & 1) ^ 1, polls))) break;
                    if (rank == 0 && of_dy) mbar_expect(full(s), 2 * STAGE);
                    const uint32_t to = place + s * STAGE;
                    tma_load_pair(to, map, line, step * 64, bar + 8 * s);
                    tma_load_pair(to + HALF / 2, map, line + 64, step * 64, bar + 8 * s);
                }
            }
        }
        if (!ok) failed = 1;
        // nothing may be on its way to this block when it ends
        if (!ok && rank == 0)
            for (int k = max(0, n - STAGES); k < n; ++k) mbar_wait(full(k % STAGES), k / STAGES & 1, polls);
    } else if (rank == 0 && warp == 1 && elect_one()) {  // ---- tensor cores of both blocks
        constexpr uint32_t idesc = mma_shape(!std::is_same<V, __half>::value, COLS, true, true, 256);
        const uint64_t da0 = operand(base, HALF / 2, 1024), db0 = operand(base + HALF, HALF / 2, 1024);
        int s = 0, all = 0;  // turns of all the pair's tiles
        uint32_t parity = 0;
        bool ok = true;
        Tile t = first;
        for (int at = blockIdx.x / 2; at < tiles; at += pairs, go_on(t)) all += turns(t);
        for (int u = 0; u < all && ok; ++u) {
            const int b = u & 1;
            if (u >= 2) {
                if (!(ok = mbar_wait_cluster(drained(b), (u / 2 - 1) & 1, polls))) break;
                tc_fence_after();
            }
            for (int step = 0; step < steps; ++step) {
                if (!(ok = mbar_wait_cluster(full(s), parity, polls))) break;
                tc_fence_after();
                const uint64_t da = da0 + (uint32_t)(s * STAGE / 16), db = db0 + (uint32_t)(s * STAGE / 16);
#pragma unroll
                for (int j = 0; j < 4; ++j)  // 16 rows of 128 bytes
                    tc_mma_pair(tmem + b * COLS, da + 128 * j, db + 128 * j, idesc, step > 0 || j > 0);
                tc_commit_pair(empty(s));
                if (++s == STAGES) {
                    s = 0;
                    parity ^= 1;
                }
            }
            if (ok) tc_commit_pair(done(b));
        }
        if (!ok) failed = 1;
    } else if (rank == 1 && warp == 3 && lane == 0) {  // ---- tells block 0 what block 1's warps have taken
        // (each of them would wait a thousand clocks for its word to go: 64 vectors, 16384 x 8192: 81 us instead of 64)
        const uint32_t there = in_block(drained(0), 0);
        int all = 0;
        bool ok = true;
        Tile t = first;
        for (int at = blockIdx.x / 2; at < tiles; at += pairs, go_on(t)) all += turns(t);
        for (int u = 0; u < all; ++u) {
            if (!(ok = mbar_wait(taken(u & 1), u / 2 & 1, polls))) break;
            mbar_arrive_at(there + 8 * (u & 1));
        }
        if (!ok) failed = 1;
    } else if (warp >= REDUCE) {
        const int group = (warp - REDUCE) / 4, row = warp % 4 * 32 + lane;
        const uint32_t quarter = tmem + ((uint32_t)(warp % 4 * 32) << 16);
        int u = 0, count = 0;
        bool ok = true;
        // This thread's codes in a turn's columns, 32 at a time, with their zero points: asked for a turn ahead.
        struct Codes {
            uint4 c[2];
            int z;  // the second one's from bit 4 on
        } next;
        // the group of the unit that they belong to: where there are more turns than one, there is only one
        const int of = g.groups_per_unit > 1 ? 64 * group / m.group | (64 * group + 32) / m.group << 4 : 0;
        auto fetch = [&](Tile t, int turn) {
            const int i = line0(t) + row, from = col0(t) + turn * COLS + 64 * group;
            next.z = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = from + 32 * h;
                if (!g.d_scales || i >= m.n_rows || k >= col_end(t)) continue;
                next.c[h] = *reinterpret_cast<const uint4 *>(m.codes + i * m.code_ld + k / 2);
                next.z |= zero_of(m, i, t.unit * g.groups_per_unit + (of >> 4 * h & 15)) << 4 * h;
            }
        };
        const int parts = min(m.group, COLS) / 32;  // of a group
        Tile t = first, after = first;
        if (blockIdx.x / 2 < tiles) fetch(t, 0);
        for (int at = blockIdx.x / 2; at < tiles && ok; at += pairs, ++count, t = after) {
            go_on(after);
            const int i = line0(t) + row;
            const bool real = i < m.n_rows;
            // the parts change places from tile to tile, so that one may still be read while the other is filled
            float *part = sums + (count & 1) * SUMS, sum[2] = {0.f, 0.f};
            Cursor<V> cursor;
            for (int turn = 0; turn < turns(t); ++turn, ++u) {
                const int b = u & 1;
                const int from = col0(t) + turn * COLS + 64 * group, to = min(from + 64, col_end(t));
                const Codes now = next;
                if (turn + 1 < turns(t))
                    fetch(t, turn + 1);
                else if (at + pairs < tiles)
                    fetch(after, 0);
                if (RES) cursor.start(m, i, from);
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(done(b), u / 2 & 1, polls) && !failed))) break;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = from + 32 * h;
                    if (k >= to) break;
                    float v[32];
                    tmem_load32(quarter + b * COLS + (k - col0(t) - turn * COLS), v);
                    // codes behind the last column take part with G = 0
                    if (real && g.d_scales) sum[h] += weighed(now.c[h], (float)(now.z >> 4 * h & 15), v);
                    if (RES && real) {
                        while (cursor.col[0] < min(k + 32, to)) {
                            const int d = cursor.col[0] - k;
                            float e = 0.f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) e = j == d ? v[j] : e;
                            if (d >= 0) g.d_res[cursor.at] = from_float<V>(e);
                            cursor.next(m);
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(rank == 0 ? drained(b) : taken(b));
            }
            if (!ok) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) part[(2 * group + h) * PART + row] = sum[h];
            __syncwarp();
            if (lane == 0) mbar_arrive(together);
            if (!(ok = warp_wait(together, count & 1, polls))) break;
            if (g.d_scales) {  // four threads a row
                const int r = (threadIdx.x - 32 * REDUCE) / 4, i = line0(t) + r;
                const int g0 = t.unit * g.groups_per_unit, n = i < m.n_rows ? min(g.groups_per_unit, m.n_groups - g0) : 0;
                for (int j = threadIdx.x % 4; j < n; j += 4) {
                    float s = 0.f;
                    for (int p = j * parts; p < (j + 1) * parts; ++p) s += part[p * PART + r];
                    g.d_scales[(long long)i * m.n_groups + g0 + j] = from_float<V>(s);
                }
            }
        }
        if (!ok) failed = 1;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_barrier();  // neither block ends while the other may still reach into it
    tc_fence_after();
    if (threadIdx.x == 0 && failed) wait_ran_out_grad = 1;
    if (warp == 1) tmem_free_pair(tmem, 2 * COLS);
}

template <typename V, bool RES>
cudaError_t launch(const CUtensorMap &map_dy, const CUtensorMap &map_x, const Args<V> &g, long long tiles, cudaStream_t s) {
    const cudaError_t e = allow_smem<V, gradient_kernel<V, RES>>(SMEM);
    if (e != cudaSuccess) return e;
    return launch_behind(gradient_kernel<V, RES>, 2 * std::min<long long>(tiles, 74), THREADS, SMEM, 0, s, map_dy, map_x, g);
}

}  // namespace

template <typename V>
cudaError_t grad_many(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy,
                      V *d_scales, V *d_res, cudaStream_t s) {
    Args<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.tiles_m = (int)ceil_div(m.n_rows, 256);
    g.groups_per_unit = std::max(1, COLS / m.group);
    g.units = (int)ceil_div(m.n_groups, g.groups_per_unit);
    g.d_scales = d_scales;
    g.d_res = m.res_ptr ? d_res : nullptr;
    const long long tiles = (long long)g.tiles_m * g.units;
    if (tiles > INT_MAX / 2) return cudaErrorInvalidConfiguration;
    CUtensorMap map_dy = {}, map_x = {};
    Workspace work(s);
    cudaError_t e = map_vectors(&map_dy, dy, m.n_rows, n_vec, ld_dy, 64, work);
    if (e == cudaSuccess) e = map_vectors(&map_x, x, m.n_cols, n_vec, ld_x, 64, work);
    return e != cudaSuccess ? e
           : g.d_res        ? launch<V, true>(map_dy, map_x, g, tiles, s)
                            : launch<V, false>(map_dy, map_x, g, tiles, s);
}

cudaError_t late_flag_grad(int **flag) { return cudaGetSymbolAddress(reinterpret_cast<void **>(flag), wait_ran_out_grad); }

#define INSTANTIATE(V)                                                                                              \
    template cudaError_t grad_many<V>(const Matrix<V> &, int, const V *, long long, const V *, long long, V *, V *, \
                                      cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
