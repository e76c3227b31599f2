// Codes -> 16-bit values, and small things that the product kernels share.
#pragma once
#include <limits.h>

#include <algorithm>
#include <atomic>

#include "q4.h"

namespace mx {
namespace q4 {

// (v & mask) | base in one operation: written out, it became two, with a constant each
__device__ __forceinline__ uint32_t pick(uint32_t v, uint32_t mask, uint32_t base) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(base));
    return r;
}

// c - z of a register's codes, two to a register, exact: p[j] holds those in bits 4 j (low half) and 16 + 4 j (high half),
// whose zero points are z0 and z1.
template <typename V>
struct Pair;
template <>
struct Pair<__half> {
    using T = __half2;
    // 1024 + c is exact in the type; so is (1024 + 16 c) / 16
    static __device__ __forceinline__ void steps(uint32_t w, int z0, int z1, T (&p)[4]) {
        const uint32_t both = z0 | z1 << 16;
        const T zz = bits(0x64006400u | both), zl = bits(0xD400D400u | both << 4), sixteenth = bits(0x2C002C00u);
        p[0] = __hsub2(bits(pick(w, 0x000F000Fu, 0x64006400u)), zz);
        p[1] = __hfma2(bits(pick(w, 0x00F000F0u, 0x64006400u)), sixteenth, zl);
        w >>= 8;
        p[2] = __hsub2(bits(pick(w, 0x000F000Fu, 0x64006400u)), zz);
        p[3] = __hfma2(bits(pick(w, 0x00F000F0u, 0x64006400u)), sixteenth, zl);
    }
    static __device__ __forceinline__ T bits(uint32_t v) { return *reinterpret_cast<T *>(&v); }
    static __device__ __forceinline__ void steps(uint32_t w, int z, T (&p)[4]) { steps(w, z, z, p); }
    static __device__ __forceinline__ T two(__half a, __half b) { return __halves2half2(a, b); }
    static __device__ __forceinline__ T both(__half v) { return __half2half2(v); }
};
template <>
struct Pair<__nv_bfloat16> {
    using T = __nv_bfloat162;
    static __device__ __forceinline__ void steps(uint32_t w, int z0, int z1, T (&p)[4]) {  // 128 + c is exact in the type
        const T zz = bits(0x43004300u | z0 | z1 << 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __hsub2(bits(pick(w >> 4 * j, 0x000F000Fu, 0x43004300u)), zz);
    }
    static __device__ __forceinline__ T bits(uint32_t v) { return *reinterpret_cast<T *>(&v); }
    static __device__ __forceinline__ void steps(uint32_t w, int z, T (&p)[4]) { steps(w, z, z, p); }
    static __device__ __forceinline__ T two(__nv_bfloat16 a, __nv_bfloat16 b) { return __halves2bfloat162(a, b); }
    static __device__ __forceinline__ T both(__nv_bfloat16 v) { return __bfloat162bfloat162(v); }
};
template <typename T>
__device__ __forceinline__ uint32_t raw(T v) { return *reinterpret_cast<uint32_t *>(&v); }

// eight codes -> eight values in order; codes j and j + 4 sit in one register until the end
template <typename V>
__device__ __forceinline__ uint4 values(uint32_t w, typename Pair<V>::T s, int z) {
    typename Pair<V>::T p[4];
    Pair<V>::steps(w, z, p);
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = raw(__hmul2(p[j], s));
    return make_uint4(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[2], r[3], 0x5410),
                      __byte_perm(r[0], r[1], 0x7632), __byte_perm(r[2], r[3], 0x7632));
}

// The group of a column that moves on by a fixed number of 32s, without a division at every move.
struct GroupOf {
    int g, r, size, dg, dr;  // group, 32s into it, its 32s; the same of a move
    __device__ __forceinline__ GroupOf(int column, int group, int move) {
        size = group / 32;
        g = column / group;
        r = column / 32 - g * size;
        dg = move / group;
        dr = move / 32 - dg * size;
    }
    __device__ __forceinline__ int second() const { return g + (r + 1 >= size); }  // of the next 32 columns
    // of the 32s that lie `n` < 4 further on
    __device__ __forceinline__ int after(int n) const {
        return g + (size == 1 ? n : size == 2 ? (r + n) / 2 : r + n >= size);
    }
    __device__ __forceinline__ void move() {
        g += dg;
        r += dr;
        if (r >= size) {
            r -= size;
            ++g;
        }
    }
};

template <typename V>
__device__ __forceinline__ V from_bits(uint32_t low) {
    const uint16_t v = (uint16_t)low;
    return *reinterpret_cast<const V *>(&v);
}

// Scales and zero points of 128 columns of a row (from a multiple of 128 on), by 32s.  A warp's lanes look at 32 rows, so
// that each load costs 32 accesses to the L1, whose rate bounds it: neighbouring groups come together where the rows'
// numbers lie on such borders (`wide` of them; groups of 32 with zero points, 8192 x 8192, 16 vectors: 36.5 -> 24.4 us,
// 16384 x 8192, 1 vector: 57.6 -> 32.6).
template <typename V>
struct Scales {
    uint2 s = {0, 0};          // four scales
    uint32_t z = 0x08080808u;  // four zero points, a byte each
    // row: where the row's numbers begin; g: the first column's group, after(n): that of the column 32 n further on
    template <typename F>
    __device__ __forceinline__ void load(const Matrix<V> &m, int wide, long long row, int g, F after) {
        const V *scales = m.scales + row;
        const uint8_t *zeros = m.zeros + row;
        const int last = m.n_groups - 1;  // behind the last column
        g = min(g, last);
        if (m.group % 128 == 0) {
            s.x = s.y = bits(scales[g]) * 0x10001u;
            if (m.zeros) z = zeros[g] * 0x01010101u;
        } else if (m.group == 32 && wide == 4) {
            s = *reinterpret_cast<const uint2 *>(scales + g);
            if (m.zeros) z = *reinterpret_cast<const uint32_t *>(zeros + g);
        } else if (m.group == 32 && wide == 2) {
            const int h = min(g + 2, last - 1);
            s.x = *reinterpret_cast<const uint32_t *>(scales + g);
            s.y = *reinterpret_cast<const uint32_t *>(scales + h);
            if (m.zeros)
                z = *reinterpret_cast<const uint16_t *>(zeros + g) | (uint32_t)*reinterpret_cast<const uint16_t *>(zeros + h) << 16;
        } else if (m.group == 64 && wide >= 2) {
            const uint32_t two = *reinterpret_cast<const uint32_t *>(scales + g);
            s.x = __byte_perm(two, 0, 0x1010);
            s.y = __byte_perm(two, 0, 0x3232);
            if (m.zeros) z = __byte_perm(*reinterpret_cast<const uint16_t *>(zeros + g), 0, 0x1100);
        } else {
            const int g1 = min(after(1), last), g2 = min(after(2), last), g3 = min(after(3), last);
            s.x = bits(scales[g]) | bits(scales[g1]) << 16;
            s.y = bits(scales[g2]) | bits(scales[g3]) << 16;
            if (m.zeros) z = zeros[g] | zeros[g1] << 8 | zeros[g2] << 16 | (uint32_t)zeros[g3] << 24;
        }
    }
    static __device__ __forceinline__ uint32_t bits(V v) { return *reinterpret_cast<const uint16_t *>(&v); }
    __device__ __forceinline__ uint2 half(int h) const { return make_uint2(h ? s.y : s.x, h ? z >> 16 : z); }
};
// how many (1, 2, 4) may be loaded together
template <typename V>
int numbers_together(const Matrix<V> &m) {
    int n = 4;
    while (n > 1 && (m.n_groups % n != 0 || (uintptr_t)m.scales % (2 * n) != 0 || (uintptr_t)m.zeros % n != 0)) n /= 2;
    return n;
}

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// From the device's stream-ordered pool, which keeps what is given back to it (as for the library's handles).
inline cudaError_t pool_memory(void **p, size_t bytes, cudaStream_t s) {
    static std::atomic<uint64_t> kept{0};  // devices whose pool has been told
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device >= 64 || !(kept.load() >> device & 1)) {
        // a process's first call may be one that is captured: this is no part of the graph, and a strict capture would end
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        if ((e = cudaThreadExchangeStreamCaptureMode(&mode)) != cudaSuccess) return e;
        cudaMemPool_t pool;
        uint64_t all = UINT64_MAX;
        e = cudaDeviceGetDefaultMemPool(&pool, device);
        if (e == cudaSuccess) e = cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &all);
        const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess || back != cudaSuccess) return e != cudaSuccess ? e : back;
        if (device < 64) kept.fetch_or(1ull << device);
    }
    return cudaMallocAsync(p, bytes, s);
}

// Buffers of one call, given back to the pool in the stream's order when the call returns.
struct Workspace {
    cudaStream_t s;
    void *held[3] = {};
    int n = 0;
    explicit Workspace(cudaStream_t s) : s(s) {}
    ~Workspace() {
        while (n > 0) cudaFreeAsync(held[--n], s);
    }
    cudaError_t take(void **p, size_t bytes) {
        const cudaError_t e = pool_memory(p, bytes, s);
        if (e == cudaSuccess) held[n++] = *p;
        return e;
    }
};

// A kernel that lays something out for the next one lets it start (`next_may_start`), so that its blocks set themselves up
// meanwhile; they touch no memory of a caller's or of a kernel's in front before `front_is_done` has returned.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void front_is_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that calls front_is_done; cluster: blocks, 0 where the kernel says so itself.
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kernel)(P...), long long blocks, int threads, int smem, int cluster, cudaStream_t s,
                          const A &...args) {
    if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// to[r][c] = from[r][c]
template <typename V>
__global__ void align_kernel(const V *from, long long ld, V *to, long long ld_to, long long rows, int cols) {
    next_may_start();
    const long long stride = (long long)gridDim.y * blockDim.y;
    const long long c = ((long long)blockIdx.x * 32 + threadIdx.x) * 8;
    for (long long r = (long long)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += stride) {
        if (c >= cols) continue;
        V v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? from[r * ld + c + j] : from_float<V>(0.f);
        *reinterpret_cast<uint4 *>(to + r * ld_to + c) = *reinterpret_cast<uint4 *>(v);
    }
}

// Vectors that bulk and 16-byte copies can fetch: rows on 16-byte borders.  Others are copied to such rows first
// (2048 x 8192 values: 13 us; fetching them value by value inside the kernel took several times the product's time).
template <typename V>
cudaError_t aligned_rows(const V *p, long long ld, int cols, int rows, Workspace &work, const V **out, long long *ld_out) {
    if (rows == 1) ld = ceil_div(cols, 8) * 8;
    *out = p;
    *ld_out = ld;
    if (((uintptr_t)p % 16 == 0 && ld % 8 == 0) || rows == 0 || cols == 0) return cudaSuccess;
    V *copy = nullptr;
    const long long ld_copy = ceil_div(cols, 8) * 8;
    const cudaError_t e = work.take((void **)&copy, sizeof(V) * ld_copy * rows);
    if (e != cudaSuccess) return e;
    const dim3 block(32, 8), grid((unsigned)ceil_div(ld_copy, 256), (unsigned)std::min<long long>(ceil_div(rows, 8), 65535));
    align_kernel<<<grid, block, 0, work.s>>>(p, ld, copy, ld_copy, (long long)rows, cols);
    *out = copy;
    *ld_out = ld_copy;
    return cudaGetLastError();
}

// Lets a kernel have `bytes` of dynamic shared memory on the current device; asked once a device.
template <typename V, auto KERNEL>
cudaError_t allow_smem(size_t bytes) {
    static std::atomic<uint64_t> told{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && told.load() >> device & 1)) return e;
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && device < 64) told.fetch_or(1ull << device);
    return e;
}

}  // namespace q4
}  // namespace mx
