// Products of a 4-bit matrix with many vectors on the fifth-generation tensor cores.
//
// One block computes D[128 x BN] in tensor memory, contraction 64 deep a step:
//   product    D[i][t] = sum_k W[i][k] x[t][k]     A = W's rows, depth-major      B = x's rows, depth-major
//   transposed D[k][t] = sum_i W[i][k] dy[t][i]    A = W's columns, line-major    B = dy's rows, depth-major
// x and dy come through tiled bulk copies.  W is made on the way: its codes come through a ring of their own (128 rows x
// 128 columns = 8 KB each) and four groups of four warps turn them into 16-bit values s * (c - z), rounded once, and store
// them in the operand's swizzled layout, then, on top, W where the tile has entries of the residual (in 32 bits until its one
// rounding, so that every W is what mx_q4_expand gives, bit for bit); in this form a tile of W
// has the same bytes for the product and its transpose, only the operand descriptor differs.
// Where there are fewer tiles than SMs, up to four blocks of a cluster share a tile's contraction and add their parts
// through distributed shared memory, in the order of their ranks; large products are computed by pairs of blocks
// (pair_kernel).
//
// W's rounding to 16 bits is what the tensor cores' operands ask for.  Against 64 bits the results are 1.3 times as far off
// as those of weights in 32 bits; up to 8 vectors (q4_few.cu) no weight is rounded.
//
// Measured, 8192 x 8192 in bfloat16: 16 vectors 23.4 us (the codes at 1.4 TB/s), 128 vectors 28 us, 512 vectors 54 us, 2048
// vectors 192 us (1.43 PFLOP/s; a library's product of these sizes with a dense W takes 181 us), with a residual of 0.5 % of
// the entries 221 us: 13 us for laying it out, the rest for putting it into the tiles.  With few vectors nothing is full
// (16 vectors: ALU pipe 50 %, issue slots 52 %, DRAM a fifth): a code tile takes 800 clocks from its arrival to its values,
// most of them waits, and a block has only 16 of them to hide its beginning and its end behind.
#include <limits.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "q4.h"
#include "q4_gemm.h"
#include "q4_maps.h"
#include "q4_ptx.cuh"
#include "q4_values.cuh"

namespace mx {
namespace q4 {
namespace {

enum { PRODUCT, TRANSPOSED };

// Warps: 0 copies of x and dy, 1 tensor core issue, 2 copies of codes, 3 none; then four groups of four warps that turn
// codes into values and empty the tensor memory.
constexpr int THREADS = 32 * 20;
constexpr int CONVERT = 4;            // first warp of the latter
constexpr int A_BYTES = 128 * 128;    // 128 lines x 64 deep x 2 bytes
// A code tile: 128 rows x 128 columns of codes, then for each thread that converts 64 of its values the residual's entries
// among them in slots of four words, an entry being column << 16 | value.  For pairs of blocks, scales and zero points of
// its two 32s (two words) lie between them.
constexpr int CODE_BYTES = 128 * 64, SLOT_BYTES = 256 * 16, CODE_TILE = CODE_BYTES + SLOT_BYTES;
constexpr int NUMBER_BYTES = 256 * 8, PAIR_TILE = CODE_BYTES + NUMBER_BYTES + SLOT_BYTES;
constexpr uint32_t NO_ENTRY = 0xffffffffu, TOO_MANY = 0xfffffffeu;

// Steps after which a barrier that tells of a step's (or a code tile's) end is used again.  A wait tells a phase from the
// next by one bit, so whoever waits must see every phase: with four groups taking tiles of two steps in turn, a group
// comes back to the same barrier after 8 steps, whatever the number of stages.
constexpr int TURN = 8;

template <int MODE, int BN>
struct Shape {
    static constexpr int STAGE = A_BYTES + BN * 128;
    static constexpr int CODES = BN == 256 ? 2 : BN == 128 ? 5 : 8;
    static constexpr int STAGES = BN == 128 ? 5 : 4;
    static constexpr int BARS = STAGES + 3 * TURN + 1;
    static_assert(STAGES <= TURN && CODES <= TURN, "a barrier is not met again before its last phase was seen");
    static constexpr int SMEM = 1024 + STAGES * STAGE + CODES * CODE_TILE + BARS * 8;
    static_assert(SMEM <= 227 * 1024, "shared memory of one block");
    static_assert(STAGES * STAGE >= 128 * BN * 4, "room for the parts of a split contraction");
};

template <typename V>
struct Args {
    Matrix<V> m;
    int n_vec, tiles_m, splits;
    V *out;
    long long ld_out;
    const uint8_t *sides;  // what follows a code tile's codes, [row / 128][column / 128][side_bytes]; null: nothing
    int side_bytes;
    int wide;  // scales that may be loaded together: 1, 2, 4
    bool slots;  // the residual's entries are among it
};

__device__ int wait_ran_out;  // set when a bounded wait ended without its barrier

// 64 values of a row in the operand's layout, with the residual's entries among them: `a` is the row's 128 bytes in a
// stage, whose sixteens are in an order that goes by the row.  numbers: two scales, and two zero points in a byte each.
// Columns behind the last become 0 before the rounding: what their bytes and scale make may be infinite, and infinity times
// the 0 that stands in the vectors there is no 0.
template <typename V>
__device__ __forceinline__ void convert_row(uint8_t *a, int out_row, uint4 (&c)[2], uint2 numbers, bool slots,
                                            const uint4 &entries, const Matrix<V> &m, int row, int col) {
    if (col + 64 > m.n_cols) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int left = m.n_cols - col - 32 * j;  // columns of these 32 that there are
            if (left <= 0) numbers.x &= ~(0xffffu << 16 * j);
            const uint32_t zeros = 0x11111111u * (numbers.y >> 8 * j & 15);
            uint32_t *w[4] = {&c[j].x, &c[j].y, &c[j].z, &c[j].w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = left - 8 * q;
                const uint32_t there = n >= 8 ? 0xffffffffu : n > 0 ? (1u << 4 * n) - 1 : 0;
                *w[q] = (*w[q] & there) | (zeros & ~there);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const typename Pair<V>::T s = Pair<V>::both(from_bits<V>(numbers.x >> 16 * j));
        const int zero = numbers.y >> 8 * j & 15;
        const uint32_t w[4] = {c[j].x, c[j].y, c[j].z, c[j].w};
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(a + ((4 * j + q ^ out_row & 7) << 4)) = values<V>(w[q], s, zero);
    }
    if (!slots || entries.x == NO_ENTRY) return;
    // W at column k of the 64, exact in 32 bits before the entry
    auto core = [&](int k) {
        const bool second = k & 32, upper = k & 16, odd = k & 8;
        const uint32_t x = second ? c[1].x : c[0].x, y = second ? c[1].y : c[0].y;
        const uint32_t z = second ? c[1].z : c[0].z, w = second ? c[1].w : c[0].w;
        const uint32_t word = odd ? (upper ? w : y) : (upper ? z : x);
        const int code = word >> 4 * (k & 7) & 15, zero = numbers.y >> (second ? 8 : 0) & 15;
        return to_float(from_bits<V>(numbers.x >> (second ? 16 : 0))) * (float)(code - zero);
    };
    auto put = [&](int k, float v) {
        *reinterpret_cast<V *>(a + ((k / 8 ^ out_row & 7) << 4) + k % 8 * 2) = from_float<V>(v);
    };
    if (entries.w != TOO_MANY) {
        const uint32_t entry[4] = {entries.x, entries.y, entries.z, entries.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (entry[j] == NO_ENTRY) break;
            const int k = entry[j] >> 16;
            put(k, core(k) + to_float(from_bits<V>(entry[j])));
        }
    } else {  // this thread looks for its entries itself
        const int k1 = min(col + 64, m.n_cols);
        unsigned b, e;
        res_range(m, row, b, e);
        for (b = first_at_least(m.res_col, b, e, col); b < e;) {
            const int k = m.res_col[b];
            if (k < col || k >= k1) break;
            float v = core(k - col);
            do v += to_float(m.res_val[b]);
            while (++b < e && m.res_col[b] == k);
            put(k - col, v);
        }
    }
}

// A code tile -> 16-bit values in the operand's layout, by the four warps of a group.  A thread has one row of 128 columns:
// of the product's tile 64 columns of each of two stages, of the transposed product's all 128 columns of one stage (rows
// 0-63 or 64-127 of the tile).  `release`: the tile's place may be filled again; free(p), stage(p), arrive(p): of the
// tile's stage p.
template <typename V, int MODE, typename Release, typename Free, typename Stage, typename Arrive>
__device__ __forceinline__ bool convert_tile(const Matrix<V> &m, const uint8_t *from, bool slots, const Scales<V> &now,
                                             int t, int row, int col, Release release, Free free, Stage stage,
                                             Arrive arrive) {
    const int lane = threadIdx.x % 32, out_row = MODE == PRODUCT ? t : t % 64;
    uint4 c[2][2], entries[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j / 2][j % 2] = *reinterpret_cast<const uint4 *>(from + t * 64 + ((j ^ t >> 1 & 3) << 4));
    if (slots) {
        const uint4 *slot = reinterpret_cast<const uint4 *>(from + CODE_BYTES) + (MODE == PRODUCT ? t : t / 64 * 128 + t % 64);
        entries[0] = slot[0];
        entries[1] = slot[MODE == PRODUCT ? 128 : 64];
    }
    // the loads are done before the place is given back: a bulk copy would overtake those still under way
    fence_async_shared();
    __syncwarp();
    if (lane == 0) release();
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // 64 columns
        const int part = MODE == PRODUCT ? half : t / 64;
        if (MODE == PRODUCT || half == 0)
            if (!free(part)) return false;
        convert_row<V>(stage(part) + out_row * 128 + (MODE == PRODUCT ? 0 : half * 8192), out_row, c[half],
                       now.half(half), slots, entries[half], m, row, col + 64 * half);
        if (MODE == PRODUCT || half == 1) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) arrive(part);
        }
    }
    return true;
}

template <typename V, int MODE, int BN>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ Args<V> g) {
    using S = Shape<MODE, BN>;
    constexpr int CODES = S::CODES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_shared;
    __shared__ volatile int failed;
    uint8_t *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    const uint32_t base = smem_addr(smem);
    uint8_t *codes_at = smem + S::STAGES * S::STAGE;
    const uint32_t bars = smem_addr(codes_at + CODES * CODE_TILE);
    auto full = [&](int s) { return bars + 8 * s; };                                   // of a stage
    auto empty = [&](int step) { return bars + 8 * (S::STAGES + step % TURN); };       // of a step
    auto c_full = [&](int n) { return bars + 8 * (S::STAGES + TURN + n % TURN); };     // of a code tile
    auto c_empty = [&](int n) { return bars + 8 * (S::STAGES + 2 * TURN + n % TURN); };
    const uint32_t done = bars + 8 * (S::STAGES + 3 * TURN);
    constexpr uint32_t COLUMNS = BN < 32 ? 32 : BN;

    const Matrix<V> &m = g.m;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const int rank = g.splits > 1 ? (int)cluster_rank() : 0;
    const int tile = blockIdx.x / g.splits;
    const int line0 = tile % g.tiles_m * 128;  // first row of D: a row of W, or a column for the transposed product
    const int col0 = tile / g.tiles_m * BN, col_end = min(g.n_vec, col0 + BN);

    // what is contracted, columns or rows of W, in steps of 64
    const int depth = MODE == PRODUCT ? m.n_cols : m.n_rows;
    const int blocks128 = (int)(((long long)depth + 127) / 128);
    const int block0 = (int)((long long)blocks128 * rank / g.splits);
    const int blocks = (int)((long long)blocks128 * (rank + 1) / g.splits) - block0, steps = 2 * blocks;
    const uint32_t polls = polls_for(steps);

    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < S::STAGES; ++s) mbar_init(full(s), MODE == PRODUCT ? 5 : 3);
        for (int n = 0; n < TURN; ++n) {
            mbar_init(empty(n), 1);
            mbar_init(c_full(n), 1);
            mbar_init(c_empty(n), 4);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_addr(&tmem_shared), COLUMNS);
    tc_fence_before();
    __syncthreads();
    front_is_done();
    tc_fence_after();
    const uint32_t tmem = tmem_shared;
    // the stage of a step is free, the place of a code tile likewise, once what was there before is used up
    auto stage_free = [&](int step) {
        return step < S::STAGES || mbar_wait(empty(step - S::STAGES), (step - S::STAGES) / TURN & 1, polls);
    };
    auto place_free = [&](int n) { return n < CODES || mbar_wait(c_empty(n - CODES), (n - CODES) / TURN & 1, polls); };

    if (warp == 0 && lane == 0) {  // ---- x or dy
        int n = 0;
        bool ok = true;
        for (; n < steps; ++n) {
            const int s = n % S::STAGES;
            if (!(ok = stage_free(n))) break;
            mbar_expect(full(s), BN * 128);
            tma_load(base + s * S::STAGE + A_BYTES, &map_b, block0 * 128 + n * 64, col0, full(s));
        }
        if (!ok) {  // nothing of this block may still be on its way when it ends
            failed = 1;
            for (int k = max(0, n - S::STAGES); k < n; ++k)
                mbar_wait(full(k % S::STAGES), k / S::STAGES & 1, polls);
        }
    } else if (warp == 1 && elect_one()) {  // ---- tensor cores
        constexpr uint32_t idesc = mma_shape(!std::is_same<V, __half>::value, BN, MODE == TRANSPOSED, false);
        const uint64_t da0 = MODE == PRODUCT ? operand(base, 16, 1024) : operand(base, 8192, 1024);
        const uint64_t db0 = operand(base + A_BYTES, 16, 1024);
        // 16 of the depth, in 16 bytes: 32 bytes of each row, or 16 rows of 128 bytes
        constexpr uint32_t NEXT_A = (MODE == PRODUCT ? 32 : 2048) / 16, NEXT_B = 32 / 16;
        int s = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int n = 0; n < steps; ++n) {
            if (!(ok = mbar_wait(full(s), parity, polls))) break;
            tc_fence_after();
            const uint64_t da = da0 + (uint32_t)(s * S::STAGE / 16), db = db0 + (uint32_t)(s * S::STAGE / 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) tc_mma(tmem, da + NEXT_A * j, db + NEXT_B * j, idesc, n > 0 || j > 0);
            tc_commit(empty(n));
            if (++s == S::STAGES) {
                s = 0;
                parity ^= 1;
            }
        }
        if (!ok) failed = 1;
        tc_commit(done);
    } else if (warp == 2 && lane == 0) {  // ---- codes
        int n = 0;
        bool ok = true;
        for (; n < blocks; ++n) {
            const int s = n % CODES;
            if (!(ok = place_free(n))) break;
            const int at = (block0 + n) * 128, row = MODE == PRODUCT ? line0 : at, col = MODE == PRODUCT ? at : line0;
            const uint32_t to = smem_addr(codes_at) + s * CODE_TILE;
            mbar_expect(c_full(n), g.slots ? CODE_TILE : CODE_BYTES);
            tma_load(to, &map_codes, col / 2, row, c_full(n));
            if (g.slots)
                bulk_load(to + CODE_BYTES, g.sides + ((long long)(row / 128) * ((m.n_cols + 127) / 128) + col / 128) * SLOT_BYTES,
                          SLOT_BYTES, c_full(n));
        }
        if (!ok) {
            failed = 1;
            for (int k = max(0, n - CODES); k < n; ++k) mbar_wait(c_full(k), k / TURN & 1, polls);
        }
    } else if (warp >= CONVERT) {  // ---- codes -> 16-bit values
        // the groups take code tiles in turn
        const int group = (warp - CONVERT) / 4, t = threadIdx.x - 32 * CONVERT - 128 * group;
        auto row_at = [&](int n) { return MODE == PRODUCT ? line0 + t : (block0 + n) * 128 + t; };
        auto col_at = [&](int n) { return MODE == PRODUCT ? (block0 + n) * 128 : line0; };
        GroupOf at(col_at(group), m.group, 512);
        Scales<V> next;
        long long numbers = (long long)row_at(group) * m.n_groups;  // of the row
        auto fetch = [&](int n) {
            if (row_at(n) < m.n_rows)
                next.load(m, g.wide, numbers, at.g, [&](int j) { return at.after(j); });
            else
                next = {};  // rows behind the last add nothing
        };
        if (group < blocks) fetch(group);
        bool ok = true;
        for (int n = group; n < blocks && ok; n += 4) {
            const Scales<V> now = next;
            if (n + 4 < blocks) {
                if (MODE == PRODUCT)
                    at.move();
                else
                    numbers += 512ll * m.n_groups;
                fetch(n + 4);
            }
            if (!(ok = warp_wait(c_full(n), n / TURN & 1, polls))) break;
            const int cs = n % CODES;
            ok = convert_tile<V, MODE>(
                m, codes_at + cs * CODE_TILE, g.slots, now, t, row_at(n), col_at(n),
                [&] { mbar_arrive(c_empty(n)); },
                [&](int part) { return __all_sync(0xffffffffu, stage_free(2 * n + part)); },
                [&](int part) { return smem + (2 * n + part) % S::STAGES * S::STAGE; },
                [&](int part) { mbar_arrive(full((2 * n + part) % S::STAGES)); });
        }
        if (!ok) failed = 1;
    }
    __syncwarp();

    // ---- D leaves tensor memory: each group of four warps holds the four quarters of its rows, and every fourth 32 columns
    const int group = (warp - CONVERT) / 4, row = warp % 4 * 32 + lane;
    const bool drains = warp >= CONVERT;
    const uint32_t quarter = tmem + ((uint32_t)(warp % 4 * 32) << 16);
    const int line = line0 + row, lines = MODE == PRODUCT ? m.n_rows : m.n_cols;
    bool ok = false;
    if (drains) {
        ok = __all_sync(0xffffffffu, warp_wait(done, 0, polls) && !failed);
        if (!ok) failed = 1;
        tc_fence_after();
    }
    float v[32];
    if (ok) {
        for (int c = 32 * group; c < BN; c += 128) {
            if (steps > 0) {
                tmem_load32(quarter + c, v);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0.f;
            }
            if (g.splits == 1) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (line < lines && col0 + c + j < col_end)
                        g.out[(col0 + c + j) * g.ld_out + line] = from_float<V>(v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) reinterpret_cast<float *>(smem)[(c + j) * 128 + row] = v[j];
            }
        }
    }
    if (g.splits > 1) {
        __syncwarp();
        cluster_barrier();
        if (ok) {
            const int width = BN / g.splits;
            for (int j = group; j < width; j += 4) {
                const int c = rank * width + j;
                const uint32_t at = base + (c * 128 + row) * 4;
                const float sum = cluster_sum(at, g.splits);
                if (line < lines && col0 + c < col_end) g.out[(col0 + c) * g.ld_out + line] = from_float<V>(sum);
            }
        }
        __syncwarp();
        cluster_barrier();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && failed) wait_ran_out = 1;
    if (warp == 1) tmem_free(tmem, COLUMNS);
}

// The same for large products: a pair of blocks computes 256 lines x 256 vectors.  Each makes its own 128 lines of W and
// brings half of the vectors, so that a step's vectors cross the L2 and the shared memories half as often.  The pairs go on
// from tile to tile; the tensor memory holds two tiles, and four warps more write one while the next is computed.
// What bounds it is shared memory: 64 columns read 32 KB of operands from it, write 16 KB of vectors and 16 KB of values,
// and bring 7 KB of codes, numbers and slots that are read again; 610 clocks for 512 of matrix work, 690 measured.
constexpr int PAIR_THREADS = 32 * 24, WRITE = 20;  // first of the writing warps
struct PairShape {
    static constexpr int STAGE = 2 * A_BYTES, STAGES = 6, CODES = 2, COLS = 256;
    static constexpr int BARS = STAGES + 4 * TURN + 4;
    static constexpr int SMEM = 1024 + STAGES * STAGE + CODES * PAIR_TILE + BARS * 8;
    static_assert(SMEM <= 227 * 1024 && STAGES <= TURN && CODES <= TURN, "as above");
};

template <typename V, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ Args<V> g) {
    using S = PairShape;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_shared;
    __shared__ volatile int failed;
    uint8_t *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    const uint32_t base = smem_addr(smem);
    __shared__ uint4 word;  // block 0's: where block 1's words land
    uint8_t *codes_at = smem + S::STAGES * S::STAGE;
    const uint32_t bars = smem_addr(codes_at + S::CODES * PAIR_TILE);
    auto full = [&](int s) { return bars + 8 * s; };                                // block 0's: of both blocks' stage
    auto empty = [&](int step) { return bars + 8 * (S::STAGES + step % TURN); };    // each block's, of a step
    auto c_full = [&](int n) { return bars + 8 * (S::STAGES + TURN + n % TURN); };  // of a code tile of its own
    auto c_empty = [&](int n) { return bars + 8 * (S::STAGES + 2 * TURN + n % TURN); };
    auto done = [&](int b) { return bars + 8 * (S::STAGES + 3 * TURN + b); };         // each block's: D is complete
    auto drained = [&](int b) { return bars + 8 * (S::STAGES + 3 * TURN + 2 + b); };  // block 0's: both have written it
    auto made = [&](int step) { return bars + 8 * (S::STAGES + 3 * TURN + 4 + step % TURN); };  // block 1's: its W is there

    const Matrix<V> &m = g.m;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t rank = cluster_rank();
    const int pairs = gridDim.x / 2, first = blockIdx.x / 2;
    const int tiles = g.tiles_m * ((g.n_vec + S::COLS - 1) / S::COLS), mine = (tiles - first + pairs - 1) / pairs;
    const int depth = MODE == PRODUCT ? m.n_cols : m.n_rows;
    const int blocks = (int)(((long long)depth + 127) / 128), steps = 2 * blocks;
    auto line_of = [&](int tile) { return tile % g.tiles_m * 256 + 128 * (int)rank; };
    auto vector_of = [&](int tile) { return tile / g.tiles_m * S::COLS; };
    const uint32_t polls = polls_for(steps);

    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < S::STAGES; ++s) mbar_init(full(s), 1 + 4);  // the copies (block 1's word is one), a group's warps
        for (int n = 0; n < TURN; ++n) {
            mbar_init(empty(n), 1);
            mbar_init(c_full(n), 1);
            mbar_init(c_empty(n), 8);
            mbar_init(made(n), 4);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(done(b), 1);
            mbar_init(drained(b), 8);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_addr(&tmem_shared), 2 * S::COLS);
    tc_fence_before();
    __syncthreads();
    cluster_barrier();  // the other block's barriers are there, too
    front_is_done();
    tc_fence_after();
    const uint32_t tmem = tmem_shared;
    // steps and code tiles are numbered on from tile to tile
    auto stage_free = [&](int step) {
        return step < S::STAGES || mbar_wait(empty(step - S::STAGES), (step - S::STAGES) / TURN & 1, polls);
    };
    auto place_free = [&](int n) {
        return n < S::CODES || mbar_wait(c_empty(n - S::CODES), (n - S::CODES) / TURN & 1, polls);
    };

    if (warp == 0 && lane == 0) {  // ---- this block's half of x or dy
        int n = 0;
        bool ok = true;
        for (int at = 0; at < mine && ok; ++at) {
            const int vector = vector_of(first + at * pairs) + 128 * (int)rank;
            for (int step = 0; step < steps; ++step, ++n) {
                const int s = n % S::STAGES;
                if (!(ok = stage_free(n))) break;
                if (rank == 0) mbar_expect(full(s), 2 * A_BYTES + 16);
                tma_load_pair(base + s * S::STAGE + A_BYTES, &map_b, step * 64, vector, in_block(full(s), 0));
            }
        }
        if (!ok) {  // nothing may still be on its way to this block when it ends
            failed = 1;
            for (int k = max(0, n - S::STAGES); k < n && rank == 0; ++k)
                mbar_wait(full(k % S::STAGES), k / S::STAGES & 1, polls);
        }
    } else if (rank == 0 && warp == 1 && elect_one()) {  // ---- tensor cores of both blocks
        constexpr uint32_t idesc = mma_shape(!std::is_same<V, __half>::value, S::COLS, MODE == TRANSPOSED, false, 256);
        const uint64_t da0 = MODE == PRODUCT ? operand(base, 16, 1024) : operand(base, 8192, 1024);
        const uint64_t db0 = operand(base + A_BYTES, 16, 1024);
        constexpr uint32_t NEXT_A = (MODE == PRODUCT ? 32 : 2048) / 16, NEXT_B = 32 / 16;
        int s = 0, n = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int at = 0; at < mine && ok; ++at) {
            const int b = at & 1;
            if (at >= 2) {
                if (!(ok = mbar_wait_cluster(drained(b), (at / 2 - 1) & 1, polls))) break;
                tc_fence_after();
            }
            for (int step = 0; step < steps; ++step, ++n) {
                if (!(ok = mbar_wait_cluster(full(s), parity, polls))) break;
                tc_fence_after();
                const uint64_t da = da0 + (uint32_t)(s * S::STAGE / 16), db = db0 + (uint32_t)(s * S::STAGE / 16);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    tc_mma_pair(tmem + b * S::COLS, da + NEXT_A * j, db + NEXT_B * j, idesc, step > 0 || j > 0);
                tc_commit_pair(empty(n));
                if (++s == S::STAGES) {
                    s = 0;
                    parity ^= 1;
                }
            }
            if (ok) tc_commit_pair(done(b));
        }
        if (!ok) failed = 1;
    } else if (rank == 1 && warp == 3 && lane == 0) {  // ---- tells block 0 what block 1's groups have made
        // The matrix instruction in block 0 reads W in both.  What was made here reaches block 0's barrier by a copy of its
        // first 16 bytes, whose end the barrier counts as it does those of the vectors' copies.  (An arrival that makes sure
        // of this thread's memory in the other block takes 1000 to 2000 clocks: 245 us for 2048 vectors, 8192 x 8192, if
        // the groups' warps make it, 273 if two threads make it for them.)
        const uint32_t there = in_block(bars, 0), to = in_block(smem_addr(&word), 0);
        bool ok = true;
        for (int n = 0; n < mine * steps; ++n) {
            const int s = n % S::STAGES;
            if (!(ok = mbar_wait(made(n), n / TURN & 1, polls))) break;
            bulk_send(to, base + s * S::STAGE, 16, there + 8 * s);
        }
        if (!ok) failed = 1;
    } else if (warp == 2 && lane == 0) {  // ---- codes of this block's lines
        int n = 0;
        bool ok = true;
        for (int at = 0; at < mine && ok; ++at) {
            const int line0 = line_of(first + at * pairs);
            for (int block = 0; block < blocks; ++block, ++n) {
                if (!(ok = place_free(n))) break;
                const int row = MODE == PRODUCT ? line0 : block * 128, col = MODE == PRODUCT ? block * 128 : line0;
                const int tile_rows = (int)(((long long)m.n_rows + 127) / 128);
                const int tile_cols = (int)(((long long)m.n_cols + 127) / 128);
                // the second block of the last pair may lie behind the last line altogether
                const bool sides = row / 128 < tile_rows && col / 128 < tile_cols;
                const uint32_t to = smem_addr(codes_at) + n % S::CODES * PAIR_TILE;
                mbar_expect(c_full(n), CODE_BYTES + (sides ? g.side_bytes : 0));
                tma_load(to, &map_codes, col / 2, row, c_full(n));
                if (sides)
                    bulk_load(to + CODE_BYTES, g.sides + ((long long)(row / 128) * tile_cols + col / 128) * g.side_bytes,
                              g.side_bytes, c_full(n));
            }
        }
        if (!ok) {
            failed = 1;
            for (int k = max(0, n - S::CODES); k < n; ++k) mbar_wait(c_full(k), k / TURN & 1, polls);
        }
    } else if (warp >= CONVERT && warp < WRITE) {  // ---- codes -> 16-bit values
        // Two groups share a code tile, a stage each, so that few stages are being filled at a time: groups 0 and 1 have the
        // even tiles of all, 2 and 3 the odd ones.  (A group with both stages of a tile holds stages that others wait for:
        // 270 us instead of 211 for 2048 vectors, 8192 x 8192, when it was tried.)  A thread has 64 values of a row.
        const int group = (warp - CONVERT) / 4, half = group & 1, t = threadIdx.x - 32 * CONVERT - 128 * group;
        const int tile_row = MODE == PRODUCT ? t : 64 * half + t % 64, part = MODE == PRODUCT ? half : t / 64;
        const int out_row = MODE == PRODUCT ? t : t % 64, out_at = out_row * 128 + (MODE == PRODUCT ? 0 : part * 8192);
        // a group's place: code tile n of all, code tile `block` of the pair's tile `at`
        int at = 0, block = group / 2;
        bool ok = true;
        for (int n = group / 2; ok; n += 2, block += 2) {
            while (block >= blocks && at < mine) {
                block -= blocks;
                ++at;
            }
            if (at >= mine || !(ok = warp_wait(c_full(n), n / TURN & 1, polls))) break;
            const int line0 = line_of(first + at * pairs);
            const uint8_t *from = codes_at + n % S::CODES * PAIR_TILE, *side = from + CODE_BYTES;
            uint4 c[2], entries;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                c[j] = *reinterpret_cast<const uint4 *>(from + tile_row * 64 + ((2 * part + j ^ tile_row >> 1 & 3) << 4));
            const uint2 numbers = reinterpret_cast<const uint2 *>(side)[128 * half + t];
            const bool slots = g.slots && line0 < (MODE == PRODUCT ? m.n_rows : m.n_cols);
            if (slots) entries = reinterpret_cast<const uint4 *>(side + NUMBER_BYTES)[128 * half + t];
            fence_async_shared();  // as in convert_tile
            __syncwarp();
            if (lane == 0) mbar_arrive(c_empty(n));
            const int step = 2 * n + half, s = step % S::STAGES;
            if (!(ok = __all_sync(0xffffffffu, stage_free(step)))) break;
            const int row = (MODE == PRODUCT ? line0 : block * 128) + tile_row;
            const int col = (MODE == PRODUCT ? block * 128 : line0) + 64 * part;
            convert_row<V>(smem + s * S::STAGE + out_at, out_row, c, numbers, slots, entries, m, row, col);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(rank == 0 ? full(s) : made(step));
        }
        if (!ok) failed = 1;
    } else if (warp >= WRITE) {  // ---- D leaves tensor memory
        const int line = warp % 4 * 32 + lane, lines = MODE == PRODUCT ? m.n_rows : m.n_cols;
        const uint32_t quarter = tmem + ((uint32_t)(warp % 4 * 32) << 16);
        bool ok = true;
        for (int at = 0; at < mine; ++at) {
            const int b = at & 1, tile = first + at * pairs, to = line_of(tile) + line, t0 = vector_of(tile);
            if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(done(b), at / 2 & 1, polls) && !failed))) break;
            tc_fence_after();
            for (int c = 0; c < S::COLS && t0 + c < g.n_vec; c += 32) {
                float v[32];
                tmem_load32(quarter + b * S::COLS + c, v);
                V *out = g.out + (long long)(t0 + c) * g.ld_out + to;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    if (to < lines && t0 + c + j < g.n_vec) *out = from_float<V>(v[j]);
                    out += g.ld_out;
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(in_block(drained(b), 0));
        }
        if (!ok) failed = 1;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_barrier();  // neither block ends while the other may still reach into it
    tc_fence_after();
    if (threadIdx.x == 0 && failed) wait_ran_out = 1;
    if (warp == 1) tmem_free_pair(tmem, 2 * S::COLS);
}

// First entry of [begin, end) whose column is at least k, for a whole warp: 32 places are looked at together.
__device__ __forceinline__ unsigned warp_first_at_least(const int *col, unsigned begin, unsigned end, int k) {
    const unsigned lane = threadIdx.x % 32;
    while (end - begin > 32) {
        const unsigned step = (end - begin + 31) / 32, p = min(begin + (lane + 1) * step, end) - 1;  // the last of each part
        const unsigned below = __ballot_sync(0xffffffffu, col[p] < k);
        const unsigned parts = below == 0xffffffffu ? 32 : __ffs(~below) - 1;  // that lie in front of k altogether
        const unsigned from = min(begin + parts * step, end);
        end = min(from + step, end);
        begin = from;
    }
    const bool below = begin + lane < end && col[begin + lane] < k;
    return begin + __popc(__ballot_sync(0xffffffffu, below));
}

// What follows the code tiles' codes: the residual's entries in slots, and scales and zero points (`numbers`) in the order
// in which a tile's threads read them, so that they come with the codes; each block 16 rows (a warp each) x 8192 columns,
// collected in shared memory and written in order.  A segment of 64 columns with more than four entries, or with a
// repeated column, is marked.  It waits for memory, a few loads after one another, so that all rows should be under way at
// once (8192 x 8192: 13 us; by 32 rows x 4096 columns, in two turns, 17; four rows a warp, 13 us more).
constexpr int SIDE_ROWS = 16, SIDE_SEGMENTS = 128;

template <typename V, int MODE>
__global__ void __launch_bounds__(32 * SIDE_ROWS)
    sides_kernel(Matrix<V> m, int chunks, bool numbers, uint8_t *sides, int side_bytes) {
    __shared__ uint4 part[SIDE_SEGMENTS][SIDE_ROWS];
    __shared__ uint2 number[SIDE_SEGMENTS][SIDE_ROWS];  // a segment's rows are in an order that goes by the segment
    next_may_start();
    const int lane = threadIdx.x % 32, r = threadIdx.x / 32;
    const int row0 = blockIdx.x / chunks * SIDE_ROWS, k0 = blockIdx.x % chunks * (64 * SIDE_SEGMENTS);
    const long long tiles = ((long long)m.n_cols + 127) / 128;
    const int segments = (int)min((long long)SIDE_SEGMENTS, 2 * tiles - k0 / 64);  // of whole tiles
    const bool real = row0 + r < m.n_rows;
    unsigned begin = 0, end = 0;
    if (real && m.res_ptr) res_range(m, row0 + r, begin, end);
    if (numbers) {
        const long long from = (real ? row0 + r : 0) * (long long)m.n_groups;
#pragma unroll 4
        for (int j = lane; j < segments; j += 32) {
            uint2 w = make_uint2(0, 0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int g = min((k0 + 64 * j + 32 * h) / m.group, m.n_groups - 1);
                const V scale = real ? m.scales[from + g] : from_float<V>(0.f);  // rows behind the last add nothing
                const uint32_t zero = m.zeros ? m.zeros[from + g] & 15 : 8;
                w.x |= (uint32_t)*reinterpret_cast<const uint16_t *>(&scale) << 16 * h;
                w.y |= zero << 8 * h;
            }
            number[j][(r ^ j) % SIDE_ROWS] = w;
        }
    }
    if (m.res_ptr) {
        for (int j = threadIdx.x; j < SIDE_SEGMENTS * SIDE_ROWS; j += 32 * SIDE_ROWS)
            part[j / SIDE_ROWS][j % SIDE_ROWS] = make_uint4(NO_ENTRY, NO_ENTRY, NO_ENTRY, NO_ENTRY);
        __syncthreads();
        const int k1 = min((long long)m.n_cols, k0 + 64ll * SIDE_SEGMENTS);
        if (k0 > 0) begin = warp_first_at_least(m.res_col, begin, end, k0);
        int segment_before = -1, column_before = -1, run = 0;  // of the entry in front, and how many its segment has
        for (unsigned e0 = begin; e0 < end; e0 += 32) {
            const unsigned e = e0 + lane;
            const int k = e < end ? m.res_col[e] : INT_MAX;
            const V v = e < end ? m.res_val[e] : from_float<V>(0.f);
            const bool mine = k >= k0 && k < k1;
            const int segment = mine ? (k - k0) / 64 : SIDE_SEGMENTS;
            int left = __shfl_up_sync(0xffffffffu, segment, 1), column = __shfl_up_sync(0xffffffffu, k, 1);
            if (lane == 0) {
                left = segment_before;
                column = column_before;
            }
            const unsigned heads = __ballot_sync(0xffffffffu, segment != left) & (0xffffffffu >> (31 - lane));
            const int rank = heads ? lane - (31 - __clz(heads)) : run + lane;
            uint32_t *to = reinterpret_cast<uint32_t *>(&part[segment % SIDE_SEGMENTS][r]);
            if (mine && rank < 4) to[rank] = (uint32_t)(k % 64) << 16 | *reinterpret_cast<const uint16_t *>(&v);
            __syncwarp();
            if (mine && (rank >= 4 || column == k)) to[3] = TOO_MANY;
            __syncwarp();
            segment_before = __shfl_sync(0xffffffffu, segment, 31);
            column_before = __shfl_sync(0xffffffffu, k, 31);
            run = __shfl_sync(0xffffffffu, rank, 31) + 1;
            if (segment_before == SIDE_SEGMENTS) break;
        }
    }
    __syncthreads();
    const int row = threadIdx.x % SIDE_ROWS, i = row0 + row;
    for (int j = threadIdx.x / SIDE_ROWS; j < segments; j += 32) {
        const int in_tile = MODE == PRODUCT ? j % 2 * 128 + i % 128 : i % 128 / 64 * 128 + j % 2 * 64 + i % 64;
        uint8_t *to = sides + ((long long)(i / 128) * tiles + k0 / 128 + j / 2) * side_bytes;
        if (numbers) {
            reinterpret_cast<uint2 *>(to)[in_tile] = number[j][(row ^ j) % SIDE_ROWS];
            to += NUMBER_BYTES;
        }
        if (m.res_ptr) reinterpret_cast<uint4 *>(to)[in_tile] = part[j][row];
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

template <typename V, int MODE, int BN>
cudaError_t launch(const CUtensorMap &codes, const CUtensorMap &b, const Args<V> &g,
                   long long tiles, cudaStream_t s) {
    auto kernel = gemm_kernel<V, MODE, BN>;
    constexpr int bytes = Shape<MODE, BN>::SMEM;
    const cudaError_t e = allow_smem<V, gemm_kernel<V, MODE, BN>>(bytes);
    if (e != cudaSuccess) return e;
    return launch_behind(kernel, tiles * g.splits, THREADS, bytes, g.splits, s, codes, b, g);
}

// Width of a tile and number of blocks that share its contraction: the choice with the least time by a model in clocks.
// Measured on 2048 to 8192 rows and columns, 16 to 2048 vectors: a code tile takes 800 to 1300 clocks (nearly the same
// for 32 to 128 vectors: the conversion bounds it), a block 11,000 to 14,000 to begin and to end, adding up parts through
// the cluster 30 a vector.  A pair of blocks (bn = 0) takes 1060 a code tile and does not pause between its tiles.
// From 1024 to 8192 rows and columns and 128 to 1024 vectors, with and without a residual, the choice between tiles and
// pairs is the faster one to within 4 % (8192 x 8192, 1024 vectors: tiles 112 us, pairs 102; 256 vectors: 39 and 53).
void plan(int lines, int depth, int n_vec, int &bn, int &splits) {
    const long long m_tiles = ceil_div(lines, 128), blocks = std::max<long long>(ceil_div(depth, 128), 1);
    double best = 0;
    for (int w : {32, 64, 128, 256}) {
        for (int s = 1; s <= 4; s *= 2) {
            if (s > blocks) break;
            const double per_block = w == 32 ? 800 : w == 64 ? 850 : w == 128 ? 950 : 1300;
            const double waves = (double)ceil_div(m_tiles * ceil_div(n_vec, w) * s, 148);
            const double cost = waves * (ceil_div(blocks, s) * per_block + 12000 + (s > 1 ? 30 * w : 0));
            if (best == 0 || cost < best) {
                best = cost;
                bn = w;
                splits = s;
            }
        }
    }
    const long long pair_tiles = ceil_div(lines, 256) * ceil_div(n_vec, 256);
    if (ceil_div(pair_tiles, 74) * blocks * 1060.0 + 14000 < best && depth > 0) {
        bn = 0;
        splits = 1;
    }
}

template <typename V, int MODE>
cudaError_t tiles_of(const Matrix<V> &m, int n_vec, const V *b, long long ld_b, V *out, long long ld_out, cudaStream_t s) {
    const int lines = MODE == PRODUCT ? m.n_rows : m.n_cols, depth = MODE == PRODUCT ? m.n_cols : m.n_rows;
    Args<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.out = out;
    g.ld_out = ld_out;
    g.wide = numbers_together(m);
    int bn = 0;
    plan(lines, depth, n_vec, bn, g.splits);
    g.tiles_m = (int)ceil_div(lines, bn ? 128 : 256);
    CUtensorMap codes = {}, vectors = {};
    Workspace work(s);
    if (depth > 0) {
        if (!encode_codes(&codes, m)) return cudaErrorInvalidValue;
        cudaError_t e = map_vectors(&vectors, b, depth, n_vec, ld_b, bn ? bn : 128, work);
        if (e != cudaSuccess) return e;
        g.slots = m.res_ptr != nullptr;
        g.side_bytes = (bn == 0 ? NUMBER_BYTES : 0) + (g.slots ? SLOT_BYTES : 0);
        if (g.side_bytes > 0) {
            // whole tiles of 128 rows: rows behind the last have empty slots
            const long long rows = ceil_div(m.n_rows, 128), cols = ceil_div(m.n_cols, 128);
            const long long grid = rows * (128 / SIDE_ROWS) * ceil_div(m.n_cols, 64 * SIDE_SEGMENTS);
            uint8_t *sides = nullptr;
            if (grid > INT_MAX) return cudaErrorMemoryAllocation;
            if ((e = work.take((void **)&sides, g.side_bytes * rows * cols)) != cudaSuccess) return e;
            sides_kernel<V, MODE><<<(unsigned)grid, 32 * SIDE_ROWS, 0, s>>>(
                m, (int)ceil_div(m.n_cols, 64 * SIDE_SEGMENTS), bn == 0, sides, g.side_bytes);
            if ((e = cudaGetLastError()) != cudaSuccess) return e;
            g.sides = sides;
        }
    }
    if (bn == 0) {
        const long long tiles = g.tiles_m * ceil_div(n_vec, 256);
        if (tiles > INT_MAX / 2) return cudaErrorInvalidConfiguration;
        const cudaError_t e = allow_smem<V, pair_kernel<V, MODE>>(PairShape::SMEM);
        if (e != cudaSuccess) return e;
        return launch_behind(pair_kernel<V, MODE>, 2 * std::min<long long>(tiles, 74), PAIR_THREADS, PairShape::SMEM, 0, s, codes,
                             vectors, g);
    }
    const long long tiles = g.tiles_m * ceil_div(n_vec, bn);
    switch (bn) {
        case 32: return launch<V, MODE, 32>(codes, vectors, g, tiles, s);
        case 64: return launch<V, MODE, 64>(codes, vectors, g, tiles, s);
        case 128: return launch<V, MODE, 128>(codes, vectors, g, tiles, s);
        default: return launch<V, MODE, 256>(codes, vectors, g, tiles, s);
    }
}

}  // namespace

template <typename V>
cudaError_t product_many(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s) {
    return tiles_of<V, PRODUCT>(m, n_vec, x, ld_x, y, ld_y, s);
}

template <typename V>
cudaError_t product_t_many(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                           cudaStream_t s) {
    return tiles_of<V, TRANSPOSED>(m, n_vec, dy, ld_dy, dx, ld_dx, s);
}

cudaError_t late_flag(int **flag) { return cudaGetSymbolAddress(reinterpret_cast<void **>(flag), wait_ran_out); }

#define INSTANTIATE(V)                                                                                             \
    template cudaError_t product_many<V>(const Matrix<V> &, int, const V *, long long, V *, long long, cudaStream_t); \
    template cudaError_t product_t_many<V>(const Matrix<V> &, int, const V *, long long, V *, long long,           \
                                           cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
