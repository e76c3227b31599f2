// 4-bit matrices: dense -> codes + scales + zero points + CSR residual (mx_q4_quantize) and back (mx_q4_expand).
#include <math.h>

#include "q4.h"
#include "q4_gemm.h"
#include "q4_values.cuh"

namespace mx {
namespace q4 {
namespace {

constexpr int WARPS = 8;
// A warp's piece of a row: 4 chunks of 512 columns, 16 neighbouring columns a lane, all asked for at once.  Short pieces
// fill the GPU with few rows too; their entries follow one another in the residual's order.  (With 8 columns a lane the
// work on a group's scale, which all lanes do, was more than that on the codes.)
constexpr int CHUNK = 512, CHUNKS = 4, PIECE = CHUNK * CHUNKS;

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

__device__ __forceinline__ float reciprocal(float v) {  // to a step or two
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// a / b with about = 1 / b to a step or two: the remainder's share corrects the product.  A quotient of few bits, such as
// the border between two codes, comes out exactly.
__device__ __forceinline__ float quotient(float a, float b, float about) {
    const float t = a * about;
    return fmaf(fmaf(-t, b, a), about, t);
}
constexpr float MAGIC = 12582912.f;  // 1.5 * 2^23: adding it rounds to whole numbers, ties to even

// Scale and zero point of a group whose values reach from lo <= 0 to hi >= 0.  `quick`: the scale is an ordinary number
// of the type; one that was rounded to few bits, or is none at all, takes the long way.
template <typename V, bool ZEROS>
struct Scale {
    V stored;
    float s, z, inverse;
    bool usable, quick;
    __device__ __forceinline__ Scale(float lo, float hi, bool nan) {
        // a division by a constant: with the rounded reciprocal and one correction the quotient is correctly rounded
        const float reach = ZEROS ? hi - lo : fmaxf(hi, -lo), steps = ZEROS ? 15.f : 7.f;
        stored = from_float<V>(quotient(reach, steps, 1.f / steps));
        s = to_float(stored);
        quick = !nan && s > 6.2e-5f && s <= 3.4028235e38f;
        usable = quick;
        inverse = reciprocal(s);
        z = ZEROS ? fminf(nearest_from(__fadd_rn(quotient(-lo, s, inverse), MAGIC) - MAGIC, -lo, s), 15.f) : 8.f;
        if (!quick) {
            stored = from_float<V>(nan ? nanf("") : reach / steps);
            s = to_float(stored);
            usable = s > 0.f && s <= 3.4028235e38f;
            z = ZEROS ? (usable ? fminf(nearest_quotient(-lo, s), 15.f) : 0.f) : 8.f;
        }
    }
};

// 8 neighbouring values of a row, 16-bit ones two to a register and worked on two at a time as long as that is exact.
template <typename W>
struct Eight;
template <>
struct Eight<float> {
    float v[8];
    using Limit = float;
    static __device__ __forceinline__ Limit limit(float threshold) { return threshold; }
    __device__ __forceinline__ void load(const float *row, int k, int end, bool wide) {
        if (wide && k + 8 <= end) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(row + k)), b = __ldg(reinterpret_cast<const float4 *>(row + k) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < end ? row[k + j] : 0.f;
        }
    }
    __device__ __forceinline__ unsigned far(Limit t) const {  // a bit for each value above the threshold
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m |= (unsigned)(fabsf(v[j]) > t) << j;
        return m;
    }
    __device__ __forceinline__ int count(Limit t) const { return __popc(far(t)); }
    __device__ __forceinline__ void drop(Limit t) {  // those become 0
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) > t ? 0.f : v[j];
    }
    // lowest and highest value (or only the highest magnitude), a NaN spreading
    struct Range {
        float lo = 0.f, hi = 0.f;
        bool nan = false;
        template <bool ZEROS>
        __device__ __forceinline__ void take(const Eight &e) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (ZEROS) lo = fminf(lo, e.v[j]);
                hi = fmaxf(hi, ZEROS ? e.v[j] : fabsf(e.v[j]));
                nan |= e.v[j] != e.v[j];
            }
        }
        template <bool ZEROS>
        __device__ __forceinline__ void share(int lanes) {
            for (int d = lanes / 2; d; d /= 2) {
                if (ZEROS) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
            }
            const unsigned nans = __ballot_sync(0xffffffffu, nan);
            nan = (nans >> (threadIdx.x % 32 & ~(lanes - 1)) & (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1)) != 0;
        }
        __device__ __forceinline__ float low() const { return lo; }
        __device__ __forceinline__ float high() const { return hi; }
        __device__ __forceinline__ bool is_nan() const { return nan; }
    };
    __device__ __forceinline__ void all(float (&f)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = v[j];
    }
};
template <typename W>
struct Eight {
    using T = typename Pair<W>::T;
    uint32_t u[4];
    using Limit = T;
    // values of the type are above the threshold where they are above the type's last value that is not
    static __device__ __forceinline__ Limit limit(float threshold) { return Pair<W>::both(rounded_down(threshold, W())); }
    static __device__ __forceinline__ __half rounded_down(float v, __half) { return __float2half_rd(v); }
    static __device__ __forceinline__ __nv_bfloat16 rounded_down(float v, __nv_bfloat16) { return __float2bfloat16_rd(v); }
    __device__ __forceinline__ void load(const W *row, int k, int end, bool wide) {
        if (wide && k + 8 <= end) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(row + k));
            u[0] = a.x, u[1] = a.y, u[2] = a.z, u[3] = a.w;
        } else {
            const uint16_t *r = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                u[j] = (k + 2 * j < end ? r[k + 2 * j] : 0u) | (k + 2 * j + 1 < end ? (uint32_t)r[k + 2 * j + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ uint32_t mask(int j, Limit t) const { return __hgt2_mask(__habs2(Pair<W>::bits(u[j])), t); }
    __device__ __forceinline__ unsigned far(Limit t) const {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m |= (mask(j, t) & 0x00020001u) << 2 * j;
        return (m | m >> 16) & 0xff;  // bits 2 j of the low halves, 2 j + 1 of the high ones
    }
    __device__ __forceinline__ int count(Limit t) const { return __popc(far(t)); }
    __device__ __forceinline__ void drop(Limit t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] &= ~mask(j, t);
    }
    struct Range {
        T lo = Pair<W>::bits(0u), hi = Pair<W>::bits(0u);
        template <bool ZEROS>
        __device__ __forceinline__ void take(const Eight &e) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T v = Pair<W>::bits(e.u[j]);
                if (ZEROS) lo = __hmin2_nan(lo, v);
                hi = __hmax2_nan(hi, ZEROS ? v : __habs2(v));
            }
        }
        template <bool ZEROS>
        __device__ __forceinline__ void share(int lanes) {
            for (int d = lanes / 2; d; d /= 2) {
                if (ZEROS) lo = __hmin2_nan(lo, Pair<W>::bits(__shfl_xor_sync(0xffffffffu, raw(lo), d)));
                hi = __hmax2_nan(hi, Pair<W>::bits(__shfl_xor_sync(0xffffffffu, raw(hi), d)));
            }
        }
        __device__ __forceinline__ float low() const { return fminf(to_float(lo.x), to_float(lo.y)); }
        __device__ __forceinline__ float high() const { return fmaxf(to_float(hi.x), to_float(hi.y)); }
        __device__ __forceinline__ bool is_nan() const {
            const float a = to_float(lo.x) + to_float(lo.y), b = to_float(hi.x), c = to_float(hi.y);
            return a != a || b != b || c != c;
        }
    };
    __device__ __forceinline__ void all(float (&f)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const T v = Pair<W>::bits(u[j]);
            f[2 * j] = to_float(v.x);
            f[2 * j + 1] = to_float(v.y);
        }
    }
};

// Where a block's entries begin is only known when all blocks in front of it have counted theirs.  A block takes its
// number when it starts (so that all in front of it have started, too), tells how many entries it has as soon as it has
// its values, works on its codes, and then walks back over the blocks in front: it adds up what they have until it meets
// one that knows its end.  W is read once; a counting pass in front took 31 us of 8192 x 8192 (2 bytes).
// A block's word: entries << 2 | 1 (its own) or 2 (with all in front); it is all that is told, so that it orders nothing else.
__device__ __forceinline__ void tell(unsigned long long *word, long long n, int kind) {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(word), "l"((unsigned long long)n << 2 | kind) : "memory");
}
__device__ int wait_ran_out_quant;
// Entries in front of block `me`, for one warp; -1 when a block in front does not tell in time.  Blocks that run together
// come here together, hundreds of them, before any of them knows its end: 64 words are looked at at a time.
__device__ __forceinline__ long long entries_before(const unsigned long long *words, long long me) {
    constexpr int WORDS = 2;
    const int lane = threadIdx.x % 32;
    long long n = 0;
    for (long long end = me; end > 0; end -= 32 * WORDS) {  // the blocks in front of `end`, the nearest first
        unsigned long long w[WORDS];
        bool all = false;
        for (unsigned polls = 0; polls < 1u << 22 && !all; ++polls) {
            all = true;
#pragma unroll
            for (int u = 0; u < WORDS; ++u) {
                const long long b = end - 1 - lane - 32 * u;
                w[u] = 2;  // in front of the first block: nothing, and that is all
                if (b >= 0) asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(w[u]) : "l"(words + b) : "memory");
                all &= w[u] != 0;
            }
        }
        if (!__all_sync(0xffffffffu, all)) return -1;
        bool found = false;
        long long mine = 0;
#pragma unroll
        for (int u = 0; u < WORDS; ++u) {
            if (found) break;
            const unsigned whole = __ballot_sync(0xffffffffu, (w[u] & 3) == 2);
            mine += whole && lane > __ffs(whole) - 1 ? 0 : (long long)(w[u] >> 2);
            found = whole != 0;
        }
        for (int d = 16; d; d /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, d);
        n += mine;
        if (found) break;
    }
    return n;
}

template <typename V>
struct Out {
    int n_rows, n_cols, group, n_groups, per_row;
    int shift;  // where group is a power of two: its logarithm
    uint8_t *codes;
    long long code_ld;
    V *scales;
    uint8_t *zeros;
    unsigned long long *words;  // residual only: the next block's number, then a word for each block
    int *res_ptr, *res_col;
    V *res_val;
    int res_cap;
};

__device__ __forceinline__ int clamped(long long n) { return (int)min(n, (long long)INT_MAX); }

// Entries among sixteen neighbouring columns a lane, lanes in order: calls put(place, column of the sixteen) for each of
// the bits of `far`; `at` is the warp's place.
template <typename F>
__device__ __forceinline__ void in_order(unsigned far, long long &at, F put) {
    const unsigned some = __ballot_sync(0xffffffffu, far != 0);
    if (!some) return;
    const int n = __popc(far), lane = threadIdx.x % 32;
    int before = __popc(some & ((1u << lane) - 1)), all = __popc(some);
    if (__any_sync(0xffffffffu, n > 1)) {
        before = n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int u = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before += u;
        }
        all = __shfl_sync(0xffffffffu, before, 31);
        before -= n;
    }
    long long e = at + before;
    while (far) {
        put(e++, __ffs(far) - 1);
        far &= far - 1;
    }
    __syncwarp();
    at += all;
}

// What the blocks of a kernel do together to place their entries.
struct Places {
    long long front;
    int counts[WARPS];
    unsigned block;
    // the block's number, in the order in which blocks start
    __device__ __forceinline__ unsigned number(unsigned long long *words) {
        if (threadIdx.x == 0) block = (unsigned)atomicAdd(words, 1ull);
        __syncthreads();
        return block;
    }
    // a warp has n entries
    __device__ __forceinline__ void count(unsigned long long *words, int n) {
        if (threadIdx.x % 32 == 0) counts[threadIdx.x / 32] = n;
        __syncthreads();
        if (threadIdx.x == 0) tell(words + 1 + block, all(), block == 0 ? 2 : 1);
    }
    __device__ __forceinline__ long long all() const {  // eight whole rows may have 2^33
        long long n = 0;
        for (int w = 0; w < WARPS; ++w) n += counts[w];
        return n;
    }
    // where the warp's entries begin; -1 when a block in front did not tell in time
    __device__ __forceinline__ long long mine(unsigned long long *words) {
        const int warp = threadIdx.x / 32;
        if (warp == 0) {
            const long long n = entries_before(words + 1, block);
            if (threadIdx.x == 0) {
                front = n;
                if (n < 0)
                    wait_ran_out_quant = 1;
                else if (block > 0)
                    tell(words + 1 + block, n + all(), 2);
            }
        }
        __syncthreads();
        long long at = front;
        if (at >= 0)
            for (int w = 0; w < warp; ++w) at += counts[w];
        return at;
    }
};

// One warp a piece, for groups of 32, 64, ... 2048 columns: SPAN chunks a group (1: up to 512 columns, lanes of one
// chunk).  Reading W and the ALU are about equally far from bounding it: ranges are taken two values at a time, and a
// quotient is a product with the reciprocal and one step of correction, which is the correctly rounded quotient where
// that has few bits, at a border between two codes above all.
template <typename V, typename W, bool ZEROS, int SPAN>
__global__ void __launch_bounds__(32 * WARPS, sizeof(W) == 2 ? 4 : 2)
    quantize_kernel(const Out<V> o, const W *w, long long ld, bool wide, float threshold) {
    __shared__ Places places;
    constexpr int KEPT = 256;  // entries of a piece whose columns wait for their place here
    __shared__ uint16_t kept[WARPS][KEPT];
    const bool split = o.res_ptr != nullptr;
    const int lane = threadIdx.x % 32;
    const long long pieces = (long long)o.n_rows * o.per_row;
    const unsigned block = split ? places.number(o.words) : blockIdx.x;
    const long long piece = (long long)block * WARPS + threadIdx.x / 32;
    const bool real = piece < pieces;
    if (!real && !split) return;
    const int row = real ? (int)(piece / o.per_row) : 0, start = real ? (int)(piece % o.per_row) * PIECE : o.n_cols;
    const W *from = w + row * ld;
    uint8_t *codes = o.codes + row * o.code_ld + start / 2 + 8 * lane;
    const int lanes = SPAN > 1 ? 32 : o.group / 16;  // that share a group in a chunk
    Eight<W> v[CHUNKS][2];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[c][h].load(from, start + c * CHUNK + 16 * lane + 8 * h, o.n_cols, wide);
    unsigned far[CHUNKS / 2] = {};  // sixteen bits for each chunk
    int mine = 0;                   // entries of the warp
    if (split) {
        const typename Eight<W>::Limit limit = Eight<W>::limit(threshold);
        long long at = 0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int k = start + c * CHUNK + 16 * lane;
            const unsigned f = (v[c][0].far(limit) | v[c][1].far(limit) << 8) &
                               (k + 16 <= o.n_cols ? 0xffffu : (1u << max(o.n_cols - k, 0)) - 1);
            far[c / 2] |= f << 16 * (c % 2);
            in_order(f, at, [&](long long e, int j) {
                if (e < KEPT) kept[threadIdx.x / 32][e] = (uint16_t)(c * CHUNK + 16 * lane + j);
            });
            v[c][0].drop(limit);
            v[c][1].drop(limit);
        }
        mine = (int)at;
        places.count(o.words, mine);
    }
#pragma unroll
    for (int c0 = 0; c0 < CHUNKS; c0 += SPAN) {
        if (start + c0 * CHUNK >= o.n_cols) break;
        typename Eight<W>::Range range;
#pragma unroll
        for (int c = c0; c < c0 + SPAN; ++c) {
            range.template take<ZEROS>(v[c][0]);
            range.template take<ZEROS>(v[c][1]);
        }
        range.template share<ZEROS>(lanes);
        const Scale<V, ZEROS> g(range.low(), range.high(), range.is_nan());
        const int k0 = start + c0 * CHUNK + 16 * lane;
        if (lane % lanes == 0 && k0 < o.n_cols) {
            const long long to = (long long)row * o.n_groups + (k0 >> o.shift);
            o.scales[to] = g.stored;
            if (ZEROS) o.zeros[to] = (uint8_t)g.z;
        }
        const float most = 15.f - g.z;
        // the eight codes are summed up in place: what the sum of the eight MAGICs and zero points comes to
        const uint32_t offset = 0x11111111u * ((uint32_t)g.z - __float_as_uint(MAGIC));
#pragma unroll
        for (int c = c0; c < c0 + SPAN; ++c) {
            const int k = k0 + (c - c0) * CHUNK;
            uint32_t word[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[8];
                v[c][h].all(f);
                word[h] = offset;
                bool border = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float t = quotient(f[j], g.s, g.inverse);
                    if (ZEROS) t = fminf(t, most);
                    const float q = __fadd_rn(t, MAGIC);
                    word[h] += __float_as_uint(q) << 4 * j;
                    if (sizeof(W) == 4) border |= fabsf(t - __fadd_rn(q, -MAGIC)) > 0.4999f;  // 24 bits may lie just beside it
                }
                if (__any_sync(0xffffffffu, border || !g.quick)) {
                    uint32_t exact = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float q = g.usable ? nearest_quotient(f[j], g.s) : 0.f;
                        exact |= (uint32_t)fminf(fmaxf(q + g.z, ZEROS ? 0.f : 1.f), 15.f) << 4 * j;
                    }
                    word[h] = exact;
                }
            }
            uint8_t *to = codes + c * (CHUNK / 2);
            if (k + 16 <= o.n_cols) {
                *reinterpret_cast<uint2 *>(to) = make_uint2(word[0], word[1]);
            } else {
                // the last bytes; a half behind the last column is 0
                for (int j = 0; j < 16 && k + j < o.n_cols; j += 2) {
                    const uint32_t w8 = word[j / 8] >> 4 * (j % 8);
                    to[j / 2] = (uint8_t)(k + j + 1 < o.n_cols ? w8 : w8 & 15);
                }
            }
        }
    }
    if (!split) return;
    // their values are read once more (which takes fewer operations than picking them out of registers), the first ones
    // while the places become known
    __syncwarp();
    const uint16_t *columns = kept[threadIdx.x / 32];
    V first = from_float<V>(0.f);
    if (lane < mine) first = from_float<V>(to_float(from[start + columns[lane]]));
    long long at = places.mine(o.words);
    if (at < 0) return;  // the whole block
    if (real && lane == 0) {
        if (start + PIECE >= o.n_cols) o.res_ptr[row + 1] = clamped(at + mine);
        if (piece == 0) o.res_ptr[0] = 0;
    }
    if (mine <= KEPT) {
        for (int i = lane; i < mine; i += 32)
            if (at + i < o.res_cap) {
                const int k = start + columns[i];
                o.res_col[at + i] = k;
                o.res_val[at + i] = i < 32 ? first : from_float<V>(to_float(from[k]));
            }
    } else {  // more than were kept: their values are read again
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            in_order(far[c / 2] >> 16 * (c % 2) & 0xffff, at, [&](long long e, int j) {
                const int k = start + c * CHUNK + 16 * lane + j;
                if (e < o.res_cap) {
                    o.res_col[e] = k;
                    o.res_val[e] = from_float<V>(to_float(from[k]));
                }
            });
    }
}

// Any other group: one warp a row, 64 columns (2 a lane) at a time; a group is gone through twice, for its range and for
// its codes.
template <typename V, typename W, bool ZEROS>
__global__ void quantize_any_kernel(const Out<V> o, const W *w, long long ld, float threshold) {
    __shared__ Places places;
    const bool split = o.res_ptr != nullptr;
    const unsigned block = split ? places.number(o.words) : blockIdx.x;
    const int row = (int)min((long long)block * WARPS + threadIdx.x / 32, (long long)INT_MAX), lane = threadIdx.x % 32;
    const bool real = row < o.n_rows;
    const W *wr = w + (real ? row : 0) * ld;
    uint8_t *cr = o.codes + (real ? row : 0) * o.code_ld;
    long long at = 0;
    if (split) {
        int n = 0;
        for (int k = lane; real && k < o.n_cols; k += 32) n += fabsf(to_float(wr[k])) > threshold;
        places.count(o.words, __reduce_add_sync(0xffffffffu, n));
        at = places.mine(o.words);
    }
    if (!real || at < 0) return;
    if (split && lane == 0) {
        o.res_ptr[row + 1] = clamped(at + places.counts[threadIdx.x / 32]);
        if (row == 0) o.res_ptr[0] = 0;
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

// One warp a piece, 8 neighbouring columns a lane, so that a warp's stores are one run of 512 bytes: the codes' values
// first, then the entries of the residual on top of them.
template <typename V>
__global__ void __launch_bounds__(32 * WARPS) expand_kernel(Matrix<V> m, int per_row, V *w, long long ld, bool wide) {
    constexpr int STEPS = PIECE / 256;
    const long long piece = (long long)blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (piece >= (long long)m.n_rows * per_row) return;
    const int row = (int)(piece / per_row), start = (int)(piece % per_row) * PIECE;
    const uint8_t *codes = m.codes + row * m.code_ld;
    const V *scales = m.scales + (long long)row * m.n_groups;
    V *to = w + row * ld;
    unsigned begin = 0, end = 0;
    if (m.res_ptr) res_range(m, row, begin, end);
    uint32_t c[STEPS];
    V s[STEPS];
    int z[STEPS];
    GroupOf at(start + 8 * lane, m.group, 256);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
        const int k = start + j * 256 + 8 * lane;
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
    int early[2];  // the first entries' columns are on their way meanwhile
#pragma unroll
    for (int j = 0; j < 2; ++j) early[j] = begin + 32 * j + lane < end ? m.res_col[begin + 32 * j + lane] : -1;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
        const int k = start + j * 256 + 8 * lane;
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
    int n = 0;
    for (unsigned i = begin + lane; i < end; i += 32, ++n) {
        const int k = n == 0 ? early[0] : n == 1 ? early[1] : m.res_col[i];
        if (k < start || k >= stop || (i > begin && m.res_col[i - 1] == k)) continue;
        const int g = k / m.group, code = codes[k / 2] >> 4 * (k & 1) & 15;
        float v = to_float(scales[g]) * (float)(code - zero_of(m, row, g));
        for (unsigned j = i; j < end && m.res_col[j] == k; ++j) v += to_float(m.res_val[j]);
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
        case 256:
        case 512: quantize_kernel<V, W, ZEROS, 1><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
        case 1024: quantize_kernel<V, W, ZEROS, 2><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
        case 2048: quantize_kernel<V, W, ZEROS, 4><<<grid, threads, 0, s>>>(o, w, ld, wide, threshold); break;
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
    while ((1 << o.shift) < m.group) ++o.shift;
    o.codes = static_cast<uint8_t *>(m.codes);
    o.code_ld = m.code_ld;
    o.scales = static_cast<V *>(m.scales);
    o.zeros = static_cast<uint8_t *>(m.zeros);
    const bool wide = (uintptr_t)w % 16 == 0 && (m.n_rows == 1 || ld * sizeof(W) % 16 == 0);
    const long long pieces = (long long)m.n_rows * o.per_row;
    if (ceil_div(pieces, WARPS) > INT_MAX) return cudaErrorInvalidConfiguration;
    Workspace work(s);
    if (m.res_row_ptr) {
        const size_t bytes = sizeof(unsigned long long) * (1 + ceil_div(pieces, WARPS));
        cudaError_t e = work.take((void **)&o.words, bytes);
        if (e == cudaSuccess) e = cudaMemsetAsync(o.words, 0, bytes, s);
        if (e != cudaSuccess) return e;
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

cudaError_t late_flag_quant(int **flag) { return cudaGetSymbolAddress(reinterpret_cast<void **>(flag), wait_ran_out_quant); }

#define INSTANTIATE(V)                                                                                              \
    template cudaError_t quantize<V>(const mx_q4_matrix &, int, const void *, long long, float, cudaStream_t);      \
    template cudaError_t expand<V>(const Matrix<V> &, V *, long long, cudaStream_t);
INSTANTIATE(__half)
INSTANTIATE(__nv_bfloat16)

}  // namespace q4
}  // namespace mx
