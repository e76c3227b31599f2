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
#include "q4_maps.h"
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

// Where a lane's words lie.  S is the width that shares a scale: the four lanes of a row have neighbouring quarters of
// every S columns, so that one mma never mixes two groups.  Word w (eight codes) begins at column place<S>(w, quarter).
template <int S>
__device__ __forceinline__ int place(int w, int quarter) {
    return S == 128 ? 32 * quarter + 8 * w : S == 64 ? 64 * (w / 2) + 16 * quarter + 8 * (w % 2) : 32 * w + 8 * quarter;
}

template <typename V>
struct Few {
    Matrix<V> m;
    int n_vec, splits, wide;
    const V *x, *dy;
    long long ld_x, ld_dy;
    const V *turned;  // x as [column][vector], vectors filled up to 8 or 16; null for up to two vectors
    V *out;
    long long ld_out;
    V *d_res;
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

// sum over the vectors of v times a residual entry's row (product: 1 term each) of the turned vectors
template <typename V, int NT>
__device__ __forceinline__ void turned_values(float (&x)[8 * NT], const V *at) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(at) + n);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint16_t b = (uint16_t)(w[j / 2] >> 16 * (j % 2));
            x[8 * n + j] = to_float(*reinterpret_cast<const V *>(&b));
        }
    }
}

// One kernel for y = W x and for the gradients of W's numbers, for up to 8 NT vectors.  A block has 128 rows; a thread
// of its own brings tiles of 128 rows x 128 columns of codes and the vectors' values at those columns into a ring of
// shared memory; two groups of four warps, 32 rows a warp, take tiles in turn; three more warps see to the residual.
//   product:  the blocks of a cluster take contiguous parts of a row's tiles, the parts are added in the order of groups
//             and ranks.
//   gradient: the sums of whole units (a tile with 128 / S groups, or, S = 0, one group in tiles of 128 columns) for each
//             vector are weighed with dy; the blocks of a row take units in turn.  For S = 0 every warp has 16 rows and
//             takes every tile: with units of several tiles taken in turn, a group of warps would meet a slot's barrier
//             without having seen its last phase, which a wait for a parity cannot tell from the wanted one.
// Taking the codes apart (7 operations for 8 codes and as many again for all the rest) bounded an earlier form, whose
// converting warps fetched tiles themselves, 16 rows a warp: 470 instructions for 2048 codes, 44 us for 16384 x 8192 and one
// vector.  This form takes 25.4 us (the codes at 2.6 TB/s), 8 vectors 26.4, with a residual of 0.5 % of the entries 30.6 and
// 37; the gradients for one vector 25.7, for 16 vectors 34.  Nothing is full any more (one vector with residual: ALU pipe
// 44 %, issue slots 47 %, DRAM a third): a tile is a chain of a wait, loads, the taking apart and products that follow one
// another, with eight warps a block to hide it, and 256 blocks on 148 SMs leave 40 SMs with one of two.
constexpr int STREAM_THREADS = 32 * 12, DEPTH = 8;
constexpr int CODE_BYTES = 128 * 64;
template <int NT>
constexpr int stream_slot = CODE_BYTES + NT * 2048;
template <int NT>
constexpr int stream_smem = 1024 + DEPTH * stream_slot<NT> + 8 * NT * 128 * 4 + DEPTH * 16;
constexpr int PART = 132;  // distance of two vectors' sums over 128 rows

// sums over four neighbouring lanes: lane `quarter` gets that of the value quarter % N
__device__ __forceinline__ float quarters(const float (&e)[1], int) {
    const float s = e[0] + __shfl_xor_sync(0xffffffffu, e[0], 1);
    return s + __shfl_xor_sync(0xffffffffu, s, 2);
}
__device__ __forceinline__ float quarters(const float (&e)[2], int quarter) {
    const bool odd = quarter & 1;
    const float s = (odd ? e[1] : e[0]) + __shfl_xor_sync(0xffffffffu, odd ? e[0] : e[1], 1);
    return s + __shfl_xor_sync(0xffffffffu, s, 2);
}
__device__ __forceinline__ float quarters(const float (&e)[4], int quarter) {
    const bool odd = quarter & 1, high = quarter & 2;
    const float a = (odd ? e[1] : e[0]) + __shfl_xor_sync(0xffffffffu, odd ? e[0] : e[1], 1);
    const float b = (odd ? e[3] : e[2]) + __shfl_xor_sync(0xffffffffu, odd ? e[2] : e[3], 1);
    return (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 2);
}

__device__ int wait_ran_out_few;

template <typename V, int S, int NT, bool GRAD>
__global__ void __launch_bounds__(STREAM_THREADS, NT == 1 ? 2 : 1)
    stream_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ Few<V> g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ volatile int failed;
    constexpr int WIDTH = S ? S : 128, SEGMENTS = 128 / WIDTH, SLOT = stream_slot<NT>;
    constexpr bool ALL = GRAD && S == 0;  // every warp takes every tile
    constexpr int H = ALL ? 1 : 2;        // 16 rows each
    const Matrix<V> &m = g.m;
    uint8_t *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    const uint32_t base = smem_addr(smem);
    float *extra = reinterpret_cast<float *>(smem + DEPTH * SLOT);  // [vector][row]: the residual's part, then sums
    const uint32_t bars = smem_addr(extra + 8 * NT * 128);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (DEPTH + s); };
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const int line = lane / 4, quarter = lane % 4;
    const int rank = blockIdx.x % g.splits, row0 = blockIdx.x / g.splits * 128;

    // the block's tiles; a gradient's unit ends with the columns, whatever its group would have room for
    const int width = SEGMENTS * m.group, per_unit = S ? 1 : (min(m.group, m.n_cols) + 127) / 128;
    const int pieces = (int)(((long long)m.n_cols + 127) / 128), units = (m.n_groups + SEGMENTS - 1) / SEGMENTS;
    const int from = (int)((long long)pieces * rank / g.splits);
    const int my_units = !GRAD || !g.out ? 0 : (units - rank + g.splits - 1) / g.splits;
    const int in_last = S ? 1 : (int)(((long long)m.n_cols - (long long)(units - 1) * width + 127) / 128);
    const int missing = my_units > 0 && (units - 1) % g.splits == rank ? per_unit - in_last : 0;
    const int tiles = GRAD ? my_units * per_unit - missing : (int)((long long)pieces * (rank + 1) / g.splits) - from;
    auto column = [&](int n) {
        return GRAD ? (rank + n / per_unit * g.splits) * width + n % per_unit * 128 : (from + n) * 128;
    };
    const uint32_t polls = polls_for(tiles);

    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < DEPTH; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), ALL ? 8 : 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    float total[2][NT][4] = {};
    if (warp < 8) {  // ---- the codes
        const int group = ALL ? 0 : warp / 4, first_row = 16 * H * (ALL ? warp : warp % 4), lower = row0 + first_row;
        // this lane's places in a slot
        const int swizzle = line >> 1 & 3;
        int code_at[4], x_at[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int byte = place<WIDTH>(w, quarter) / 2, k = place<WIDTH>(w, quarter);
            code_at[w] = (first_row + line) * 64 + ((byte / 16 ^ swizzle) << 4) + byte % 16;
            x_at[w] = CODE_BYTES + k / 64 * (NT * 1024) + line * 128 + ((k % 64 / 8 ^ line) << 4);
        }
        // scales and zero points: a lane a row
        const long long my_row = (long long)min(lower + lane, m.n_rows - 1) * m.n_groups;
        GroupOf at((from + group) * 128, m.group, 256);
        Scales<V> next;
        auto numbers = [&](int n) {
            const int gr = (rank + n / per_unit * g.splits) * SEGMENTS;  // gradient
            if (SEGMENTS == 1) {  // one word: scale, zero point << 16
                next.s.x = GRAD ? 0 : Scales<V>::bits(m.scales[my_row + at.g]);
                if (m.zeros) next.s.x |= (uint32_t)(m.zeros[my_row + (GRAD ? gr : at.g)] & 15) << 16;
                if (!GRAD) at.move();
            } else if (GRAD) {
                if (m.zeros) next.load(m, g.wide, my_row, gr, [&](int j) { return gr + j / (4 / SEGMENTS); });
            } else {
                next.load(m, g.wide, my_row, at.g, [&](int j) { return at.after(j); });
                at.move();
            }
        };
        float dy[2 * H][NT][2];
        if (GRAD) {
#pragma unroll
            for (int r = 0; r < 2 * H; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int t = 8 * n + 2 * quarter + j, i = lower + line + 8 * r;
                        dy[r][n][j] = t < g.n_vec && i < m.n_rows ? to_float(g.dy[t * g.ld_dy + i]) : 0.f;
                    }
        }
        float d[SEGMENTS][H][NT][4] = {};
        int n = group, of_unit = 0;  // the latter: tiles of the unit so far
        if (n < tiles) numbers(n);
        bool ok = true;
        while (n < tiles) {
            const Scales<V> now = next;
            uint32_t two[2 * H], four[2 * H];  // this lane's rows' scales and zero points
            const int was = n;
            n += ALL ? 1 : 2;
            ++of_unit;
            const bool complete = !ALL || of_unit == per_unit || n == tiles;  // the unit's last tile
            if (n < tiles) numbers(n);
            const int slot = was % DEPTH;
            if (!(ok = warp_wait(full(slot), was / DEPTH & 1, polls))) break;
            const uint8_t *tile = smem + slot * SLOT;
            uint32_t c[2 * H][4];
#pragma unroll
            for (int j = 0; j < 2 * H; ++j) {
                if (WIDTH == 128) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(tile + code_at[0] + 512 * j);
                    c[j][0] = v.x, c[j][1] = v.y, c[j][2] = v.z, c[j][3] = v.w;
                } else if (WIDTH == 64) {
#pragma unroll
                    for (int w = 0; w < 4; w += 2) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(tile + code_at[w] + 512 * j);
                        c[j][w] = v.x, c[j][w + 1] = v.y;
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 4; ++w) c[j][w] = *reinterpret_cast<const uint32_t *>(tile + code_at[w] + 512 * j);
                }
            }
            // columns from `left` on belong to the next group (which begins on a multiple of 32)
            const int left = ALL && complete ? m.group - (of_unit - 1) * 128 : 128;
#pragma unroll
            for (int j = 0; j < SEGMENTS; ++j) {
                const int n32 = j * (WIDTH / 32);
                int z[2 * H];
                float s[2 * H];
#pragma unroll
                for (int r = 0; r < 2 * H; ++r) {
                    if (SEGMENTS == 1) {
                        two[r] = !GRAD || m.zeros ? __shfl_sync(0xffffffffu, now.s.x, line + 8 * r) : 0;
                        s[r] = GRAD ? 0.f : to_float(from_bits<V>(two[r]));
                        z[r] = m.zeros ? two[r] >> 16 : 8;
                        continue;
                    }
                    if (!GRAD && n32 % 2 == 0) two[r] = __shfl_sync(0xffffffffu, n32 < 2 ? now.s.x : now.s.y, line + 8 * r);
                    if (j == 0 && m.zeros) four[r] = __shfl_sync(0xffffffffu, now.z, line + 8 * r);
                    s[r] = GRAD ? 0.f : to_float(from_bits<V>(two[r] >> 16 * (n32 % 2)));
                    z[r] = m.zeros ? four[r] >> 8 * n32 & 15 : 8;
                }
                float(&e)[H][NT][4] = d[GRAD ? j : 0];
                if (!GRAD) {
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int q = 0; q < NT; ++q)
#pragma unroll
                            for (int k = 0; k < 4; ++k) e[h][q][k] = 0.f;
                }
#pragma unroll
                for (int w = j * (WIDTH / 32); w < (j + 1) * (WIDTH / 32); ++w) {
                    // codes i and i + 4 of a word share a register; the vectors' values are paired alike
                    uint32_t x[NT][4];
#pragma unroll
                    for (int q = 0; q < NT; ++q) {
                        uint4 u = *reinterpret_cast<const uint4 *>(tile + x_at[w] + 1024 * q);
                        if (ALL && left < 128 && place<WIDTH>(w, quarter) >= left) u = make_uint4(0, 0, 0, 0);
                        x[q][0] = __byte_perm(u.x, u.z, 0x5410);
                        x[q][1] = __byte_perm(u.x, u.z, 0x7632);
                        x[q][2] = __byte_perm(u.y, u.w, 0x5410);
                        x[q][3] = __byte_perm(u.y, u.w, 0x7632);
                    }
                    word_product<V, NT>(e[0], c[0][w], c[1][w], z[0], z[1], x);
                    if (H == 2) word_product<V, NT>(e[H - 1], c[2 * H - 2][w], c[2 * H - 1][w], z[2 * H - 2], z[2 * H - 1], x);
                }
                if (!GRAD) {
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int q = 0; q < NT; ++q)
#pragma unroll
                            for (int k = 0; k < 4; ++k) total[h][q][k] = fmaf(s[2 * h + k / 2], e[h][q][k], total[h][q][k]);
                }
            }
            // the products have used every value from the slot: nothing that a copy could overtake is under way
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(slot));
            if (GRAD && complete) {
                of_unit = 0;
                const int first_group = (rank + was / per_unit * g.splits) * SEGMENTS;
#pragma unroll
                for (int r = 0; r < 2 * H; ++r) {
                    float e[SEGMENTS];
#pragma unroll
                    for (int j = 0; j < SEGMENTS; ++j) {
                        e[j] = 0.f;
#pragma unroll
                        for (int q = 0; q < NT; ++q)
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                float &v = d[j][r / 2][q][2 * (r % 2) + t];
                                e[j] = fmaf(dy[r][q][t], v, e[j]);
                                v = 0.f;
                            }
                    }
                    // over the four lanes of a row, which end with a group each
                    const float sum = quarters(e, quarter);
                    const int i = lower + line + 8 * r, gr = first_group + quarter % SEGMENTS;
                    if (quarter < SEGMENTS && gr < m.n_groups && i < m.n_rows)
                        g.out[(long long)i * m.n_groups + gr] = from_float<V>(sum);
                }
            }
        }
        if (!ok) failed = 1;
    } else if (warp == 8 && lane == 0) {  // ---- copies
        bool ok = true;
        int n = 0;
        for (; n < tiles; ++n) {
            const int slot = n % DEPTH, k = column(n);
            if (!(ok = mbar_wait(empty(slot), (n / DEPTH & 1) ^ 1, polls))) break;
            const uint32_t to = base + slot * SLOT;
            mbar_expect(full(slot), SLOT);
            tma_load(to, &map_codes, k / 2, row0, full(slot));
            tma_load(to + CODE_BYTES, &map_x, k, 0, full(slot));
            tma_load(to + CODE_BYTES + NT * 1024, &map_x, k + 64, 0, full(slot));
        }
        if (!ok) {
            failed = 1;
            for (int k = max(0, n - DEPTH); k < n; ++k) mbar_wait(full(k % DEPTH), k / DEPTH & 1, polls);
        }
    } else if (warp > 8) {  // ---- the residual: eight lanes a row, the ranks share the rows
        const int first = 128 * rank / g.splits, last = 128 * (rank + 1) / g.splits;
        if (!GRAD)
            for (int j = threadIdx.x - 32 * 9; j < 8 * NT * 128; j += 96) extra[j] = 0.f;
        asm volatile("bar.sync 1, 96;" ::: "memory");  // these three warps
        if (m.res_ptr && (!GRAD || g.d_res)) {
            // Everything here waits for memory three times in a row (where the row's entries are, the entries, the
            // vectors), so a warp asks for all its rows' entries' places at once, and for the next four rows' entries
            // while it works on four.
            constexpr int TOGETHER = 6;  // entries a lane asks for at once: 48 of a row
            struct Entries {
                unsigned begin, end;
                int k[TOGETHER];
                V a[TOGETHER];
            };
            auto row_of = [&](int n) { return first + 4 * (warp - 9) + 12 * (n / 4) + n % 4; };  // a warp's n-th row
            unsigned my_begin = 0, my_end = 0;  // of the row that is the lane's number
            if (row_of(lane) < last && row0 + row_of(lane) < m.n_rows) res_range(m, row0 + row_of(lane), my_begin, my_end);
            unsigned their_begin = 0, their_end = 0;  // and 32 rows on
            if (row_of(32 + lane) < last && row0 + row_of(32 + lane) < m.n_rows)
                res_range(m, row0 + row_of(32 + lane), their_begin, their_end);
            auto ask = [&](Entries &n, unsigned from) {
#pragma unroll
                for (int u = 0; u < TOGETHER; ++u) {
                    const unsigned e = from + lane % 8 + 8 * u;
                    n.k[u] = e < n.end ? m.res_col[e] : -1;
                    if (!GRAD) n.a[u] = e < n.end ? m.res_val[e] : from_float<V>(0.f);
                }
            };
            auto rows = [&](Entries &n, int round) {
                const int at = 4 * round + lane / 8;
                const unsigned b0 = __shfl_sync(0xffffffffu, my_begin, at & 31), e0 = __shfl_sync(0xffffffffu, my_end, at & 31);
                const unsigned b1 = __shfl_sync(0xffffffffu, their_begin, at & 31), e1 = __shfl_sync(0xffffffffu, their_end, at & 31);
                n.begin = at < 32 ? b0 : b1;
                n.end = at < 32 ? e0 : e1;
                ask(n, n.begin);
            };
            const int rounds = (last - first + 11) / 12;  // at most 11: 44 rows
            Entries next;
            rows(next, 0);
            for (int round = 0; round < rounds; ++round) {
                Entries now = next;
                if (round + 1 < rounds) rows(next, round + 1);
                const int r = row_of(4 * round + lane / 8), i = row0 + r;
                float v[8 * NT] = {};
                if (GRAD) {
#pragma unroll
                    for (int t = 0; t < 8 * NT; ++t)
                        v[t] = now.begin < now.end && t < g.n_vec ? to_float(g.dy[t * g.ld_dy + i]) : 0.f;
                }
                for (unsigned from = now.begin;;) {
#pragma unroll
                    for (int u = 0; u < TOGETHER; ++u) {
                        const int k = now.k[u];
                        if (k < 0 || k >= m.n_cols) continue;
                        float x[8 * NT];
                        if (g.turned) {
                            turned_values<V, NT>(x, g.turned + (long long)k * (8 * NT));
                        } else {  // one or two vectors
                            x[0] = to_float(g.x[k]);
                            x[1] = g.n_vec > 1 ? to_float(g.x[g.ld_x + k]) : 0.f;
                        }
                        if (GRAD) {
                            float s = fmaf(v[0], x[0], v[1] * x[1]);
                            if (g.turned) {
#pragma unroll
                                for (int t = 2; t < 8 * NT; ++t) s = fmaf(v[t], x[t], s);
                            }
                            g.d_res[from + lane % 8 + 8 * u] = from_float<V>(s);
                        } else {
                            const float a = to_float(now.a[u]);
                            v[0] = fmaf(a, x[0], v[0]);
                            v[1] = fmaf(a, x[1], v[1]);
                            if (g.turned) {
#pragma unroll
                                for (int t = 2; t < 8 * NT; ++t) v[t] = fmaf(a, x[t], v[t]);
                            }
                        }
                    }
                    from += 8 * TOGETHER;
                    if (from >= now.end) break;
                    ask(now, from);
                }
                __syncwarp();
                if (!GRAD) {
#pragma unroll
                    for (int t = 0; t < 8 * NT; ++t) {
                        if (t >= g.n_vec) break;
#pragma unroll
                        for (int x = 1; x < 8; x *= 2) v[t] += __shfl_xor_sync(0xffffffffu, v[t], x);
                        if (lane % 8 == 0 && r < last) extra[t * 128 + r] = v[t];
                    }
                }
            }
        }
    }
    __syncthreads();
    if (!GRAD) {
        // the ring is used up: the two groups' sums go there, [group][vector][row]
        float *part = reinterpret_cast<float *>(smem);
        if (warp < 8) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        part[(warp / 4 * 8 * NT + 8 * n + 2 * quarter + j % 2) * PART + 32 * (warp % 4) + line + 8 * (j / 2) +
                             16 * h] = total[h][n][j];
        }
        __syncthreads();
        const bool ok = !failed;
        for (int j = threadIdx.x; j < 128 * g.n_vec; j += STREAM_THREADS) {
            const int t = j / 128, r = j % 128;
            const float s = extra[j] + part[t * PART + r] + part[(8 * NT + t) * PART + r];
            if (g.splits > 1)
                extra[j] = s;
            else if (ok && row0 + r < m.n_rows)
                g.out[t * g.ld_out + row0 + r] = from_float<V>(s);
        }
        if (g.splits > 1) {
            __syncthreads();
            cluster_barrier();
            const int rows = 128 / g.splits;
            for (int j = threadIdx.x; j < rows * g.n_vec; j += STREAM_THREADS) {
                const int t = j / rows, r = rank * rows + j % rows;
                const float s = cluster_sum(smem_addr(extra + t * 128 + r), g.splits);
                if (ok && row0 + r < m.n_rows) g.out[t * g.ld_out + row0 + r] = from_float<V>(s);
            }
            __syncwarp();
            cluster_barrier();
        }
    }
    if (threadIdx.x == 0 && failed) wait_ran_out_few = 1;
}

// turned[k][t] = x[t][k], 0 for the vectors up to `filled`
template <typename V>
__global__ void turn_kernel(const V *x, long long ld, int n_vec, int n_cols, int filled, V *turned) {
    const int k = blockIdx.x * THREADS + threadIdx.x;
    if (k >= n_cols) return;
    for (int t0 = 0; t0 < filled; t0 += 8) {
        V v[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = t0 + t < n_vec ? x[(t0 + t) * ld + k] : from_float<V>(0.f);
        *reinterpret_cast<uint4 *>(turned + (long long)k * filled + t0) = *reinterpret_cast<uint4 *>(v);
    }
}

// dx = dy W for up to 8 vectors, no residual and matrices of up to 2^22 entries (product_t says why).  A block has 256
// columns, its warps take 16 rows at a time; the contraction runs over rows, whose scales differ, so the values are
// s (c - z), rounded once to the type.  The blocks of a cluster share the rows.  A lane holds 32 columns of four rows; two
// rows' codes of a column are brought into one register.  2048 x 2048, 8 vectors: 7.0 us, most of it the time of the
// launch, of loads that wait for one another and of adding up the warps' parts.
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
        const float total = cluster_sum(smem_addr(parts + part_at(t, col)), g.splits);
        if (k0 + col < m.n_cols) g.out[t * g.ld_out + k0 + col] = from_float<V>(total);
    }
    __syncwarp();
    cluster_barrier();
}

// sums over no vectors: 0 for every scale and every residual entry that there is
template <typename V>
__global__ void no_gradient_kernel(Matrix<V> m, V *d_scales, V *d_res) {
    const long long row = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (row >= m.n_rows) return;
    if (d_scales)
        for (int j = lane; j < m.n_groups; j += 32) d_scales[row * m.n_groups + j] = from_float<V>(0.f);
    if (!d_res) return;
    unsigned begin, end;
    res_range(m, (int)row, begin, end);
    for (unsigned e = begin + lane; e < end; e += 32) d_res[e] = from_float<V>(0.f);
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

// as many parts of `pieces` as bring `blocks` to two on each of the GPU's 148 SMs, a power of two up to 8, a part not
// smaller than `least`
int parts_of(long long blocks, long long pieces, int least) {
    int n = 1;
    while (n < 8 && blocks * n * 2 <= 2 * 148 && pieces >= 2ll * n * least) n *= 2;
    return n;
}

template <typename V, int S, int NT, bool GRAD>
cudaError_t stream(const Few<V> &g, const CUtensorMap &codes, const CUtensorMap &x, cudaStream_t s) {
    auto kernel = stream_kernel<V, S, NT, GRAD>;
    const long long blocks = ceil_div(g.m.n_rows, 128) * g.splits;
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    const cudaError_t e = allow_smem<V, stream_kernel<V, S, NT, GRAD>>(stream_smem<NT>);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(STREAM_THREADS);
    cfg.dynamicSmemBytes = stream_smem<NT>;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = GRAD ? 1 : g.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = attr[0].val.clusterDim.x > 1;
    return cudaLaunchKernelEx(&cfg, kernel, codes, x, g);
}

// x with rows that can be fetched, its tensor map and the codes', and x turned where the residual's gathers want it
template <typename V>
cudaError_t stream_inputs(Few<V> &g, const V *x, long long ld_x, CUtensorMap &codes, CUtensorMap &map_x, bool gathers,
                          Workspace &work) {
    const Matrix<V> &m = g.m;
    cudaError_t e = aligned_rows(x, ld_x, m.n_cols, g.n_vec, work, &g.x, &g.ld_x);
    if (e != cudaSuccess || m.n_cols == 0) return e;
    const int filled = g.n_vec <= 8 ? 8 : 16;
    if (!encode_codes(&codes, m) || !encode_vectors(&map_x, g.x, m.n_cols, g.n_vec, g.ld_x, filled))
        return cudaErrorInvalidValue;
    if (gathers && g.n_vec > 2) {
        V *turned = nullptr;
        if ((e = work.take((void **)&turned, sizeof(V) * filled * m.n_cols)) != cudaSuccess) return e;
        turn_kernel<<<(unsigned)ceil_div(m.n_cols, THREADS), THREADS, 0, work.s>>>(g.x, g.ld_x, g.n_vec, m.n_cols, filled, turned);
        g.turned = turned;
        e = cudaGetLastError();
    }
    return e;
}

}  // namespace

template <typename V>
cudaError_t product(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, V *y, long long ld_y, cudaStream_t s) {
    // 16 vectors, 4096 x 4096: 16.5 us here, 10.2 us there; 8 vectors: 7 and 10.  (The form for 16 was launched for two blocks
    // an SM, as parts_of counts, while its registers leave room for one: two rounds.  One that fits was not measured.)
    if (n_vec > 8) return product_many(m, n_vec, x, ld_x, y, ld_y, s);
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.wide = numbers_together(m);
    g.splits = parts_of(ceil_div(m.n_rows, 128), ceil_div(m.n_cols, 128), 2);
    g.out = y;
    g.ld_out = ld_y;
    Workspace work(s);
    CUtensorMap codes = {}, map_x = {};
    const cudaError_t e = stream_inputs(g, x, ld_x, codes, map_x, m.res_ptr != nullptr, work);
    if (e != cudaSuccess) return e;
    return m.group % 128 == 0  ? stream<V, 128, 1, false>(g, codes, map_x, s)
           : m.group % 64 == 0 ? stream<V, 64, 1, false>(g, codes, map_x, s)
                               : stream<V, 32, 1, false>(g, codes, map_x, s);
}

template <typename V>
cudaError_t product_t(const Matrix<V> &m, int n_vec, const V *dy, long long ld_dy, V *dx, long long ld_dx,
                      cudaStream_t s) {
    // The residual's entries meet in columns: where there are some, the tiles that they are put into are faster even for
    // one vector (4096 x 4096: 15 us there, 28 us with a search and ordered additions here).  Those also take the larger
    // matrices (8 vectors, 2048 x 2048: 7.0 us here, 8.0 there; 4096 x 4096: 13.7 and 10.4, with groups of 32 and zero
    // points 15.5 and 11.3), which few clusters of eight do not spread over the GPU.
    if (n_vec > VEC || m.res_ptr || (long long)m.n_rows * m.n_cols > 1 << 22) return product_t_many(m, n_vec, dy, ld_dy, dx, ld_dx, s);
    const long long blocks = ceil_div(m.n_cols, COLS);
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.splits = parts_of(blocks, ceil_div(m.n_rows, 16), WARPS);
    g.out = dx;
    g.ld_out = ld_dx;
    Workspace work(s);
    cudaError_t e = aligned_rows(dy, ld_dy, m.n_rows, n_vec, work, &g.dy, &g.ld_dy);
    if (e == cudaSuccess) e = allow_smem<V, product_t_few_kernel<V>>(T_SMEM);
    return e == cudaSuccess ? run<V>(product_t_few_kernel<V>, blocks * g.splits, g.splits, T_SMEM, g, s) : e;
}

template <typename V>
cudaError_t grad(const Matrix<V> &m, int n_vec, const V *x, long long ld_x, const V *dy, long long ld_dy, V *d_scales,
                 V *d_res, cudaStream_t s) {
    if (n_vec > 16) return grad_many(m, n_vec, x, ld_x, dy, ld_dy, d_scales, d_res, s);
    if (n_vec == 0) return no_gradient(m, d_scales, m.res_ptr ? d_res : nullptr, s);
    Few<V> g = {};
    g.m = m;
    g.n_vec = n_vec;
    g.wide = numbers_together(m);
    g.splits = parts_of(ceil_div(m.n_rows, 128), m.group == 32 || m.group == 64 ? ceil_div(m.n_cols, 128) : m.n_groups, 2);
    g.dy = dy;
    g.ld_dy = ld_dy;
    g.out = d_scales;
    g.d_res = m.res_ptr ? d_res : nullptr;
    Workspace work(s);
    CUtensorMap codes = {}, map_x = {};
    const cudaError_t e = stream_inputs(g, x, ld_x, codes, map_x, g.d_res != nullptr, work);
    if (e != cudaSuccess) return e;
    const bool one = n_vec <= 8;
    if (m.group == 128) return one ? stream<V, 128, 1, true>(g, codes, map_x, s) : stream<V, 128, 2, true>(g, codes, map_x, s);
    if (m.group == 64) return one ? stream<V, 64, 1, true>(g, codes, map_x, s) : stream<V, 64, 2, true>(g, codes, map_x, s);
    if (m.group == 32) return one ? stream<V, 32, 1, true>(g, codes, map_x, s) : stream<V, 32, 2, true>(g, codes, map_x, s);
    return one ? stream<V, 0, 1, true>(g, codes, map_x, s) : stream<V, 0, 2, true>(g, codes, map_x, s);
}

cudaError_t late_flag_few(int **flag) { return cudaGetSymbolAddress(reinterpret_cast<void **>(flag), wait_ran_out_few); }

#define INSTANTIATE(V)                                                                                                \
    template cudaError_t product<V>(const Matrix<V> &, int, const V *, long long, V *, long long, cudaStream_t);      \
    template cudaError_t product_t<V>(const Matrix<V> &, int, const V *, long long, V *, long long, cudaStream_t);    \
    template cudaError_t grad<V>(const Matrix<V> &, int, const V *, long long, const V *, long long, V *, V *,        \
                                 cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
