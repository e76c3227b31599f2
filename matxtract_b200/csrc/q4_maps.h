// Tensor maps of codes and vectors for tiled bulk copies.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "q4.h"
#include "q4_values.cuh"

namespace mx {
namespace q4 {

using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                            const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline Encode encoder() {
    static const Encode f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<Encode>(p);
    }();
    return f;
}

inline bool encode(CUtensorMap *map, CUtensorMapDataType type, const void *p, uint64_t cols, uint64_t rows, uint64_t ld_bytes,
            uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld_bytes};
    const cuuint32_t box[2] = {box_cols, box_rows}, ones[2] = {1, 1};
    return encoder() && encoder()(map, type, 2, const_cast<void *>(p), dims, strides, box, ones,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows of 64 values in 128-byte swizzle, `box_rows` at a time
template <typename V>
bool encode_vectors(CUtensorMap *map, const V *p, int cols, int rows, long long ld, int box_rows) {
    return encode(map, std::is_same<V, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                  p, cols, rows, 2 * ld, 64, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The tensor map of `rows` vectors.
template <typename V>
cudaError_t map_vectors(CUtensorMap *map, const V *p, int cols, int rows, long long ld, int box_rows, Workspace &work) {
    cudaError_t e = aligned_rows(p, ld, cols, rows, work, &p, &ld);
    if (e != cudaSuccess) return e;
    return encode_vectors(map, p, cols, rows, ld, box_rows) ? cudaSuccess : cudaErrorInvalidValue;
}

// 128 rows x 128 columns of codes (64 bytes a row, in 64-byte swizzle)
template <typename V>
bool encode_codes(CUtensorMap *map, const Matrix<V> &m) {
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, m.codes, ((uint64_t)m.n_cols + 31) / 32 * 16, m.n_rows, m.code_ld, 64,
                  128, CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace q4
}  // namespace mx
