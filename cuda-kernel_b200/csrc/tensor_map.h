// Tensor maps for the TMA copies of matrix tiles.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "host.h"

namespace swb {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library does not link the driver).
inline EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Rows of `pitch` bytes (a multiple of 16) in boxes of `box_rows` by `box_bytes` (64 or 128, swizzled
// over as many bytes); zero beyond the matrix. depth > 0 (box_bytes must divide pitch): a box
// takes `depth` neighbouring pieces of each row, piece after piece in shared memory, and its
// coordinates are (0, row, piece) instead of (byte / 4, row).
inline int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t pitch, int box_bytes, int box_rows,
                    int depth = 0) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(SWB_E_UNSUPPORTED, "the driver has no tensor maps");
    const cuuint32_t words = cuuint32_t(box_bytes / 4), one[3] = {1, 1, 1};
    const cuuint64_t dims[3] = {depth ? words : cuuint64_t(pitch / 4), cuuint64_t(rows), cuuint64_t(pitch / box_bytes)};
    const cuuint64_t strides[2] = {cuuint64_t(pitch), cuuint64_t(box_bytes)};
    const cuuint32_t box[3] = {words, cuuint32_t(box_rows), cuuint32_t(depth)};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, depth ? 3 : 2, const_cast<void*>(base), dims, strides,
                              box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SWB_OK : fail(SWB_E_CUDA, "tensor map");
}

// Rows of `cols` elements, `pitch` bytes apart, in boxes of box_rows by box_cols (128 bytes of shared
// memory, swizzled over as many); zero beyond the matrix.
inline int make_typed_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t cols, int64_t rows,
                          int64_t pitch, int box_cols, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(SWB_E_UNSUPPORTED, "the driver has no tensor maps");
    const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(pitch)};
    const cuuint32_t box[2] = {cuuint32_t(box_cols), cuuint32_t(box_rows)}, one[2] = {1, 1};
    const CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SWB_OK : fail(SWB_E_CUDA, "tensor map");
}

// The maps of a streamed weight tensor (Stream::produce), where its rows allow them.
struct WeightMaps {
    CUtensorMap w, s;
};

// codes or values [rows, pitch bytes], scales [rows, blocks] (null for 16-bit matrices). `fast`
// receives whether every row (and row of scales) starts on 16 bytes; if not, the maps stay unset.
// Rows of whole 128 bytes are copied 1 KB of 16 rows at a time (`deep`), others 128 bytes.
inline int make_weight_maps(WeightMaps* m, const void* w, const void* s, int64_t rows, int64_t pitch, int64_t blocks,
                            bool* fast, bool* deep) {
    *fast = ((reinterpret_cast<uintptr_t>(w) | uintptr_t(pitch)) & 15) == 0 &&
            (!s || ((reinterpret_cast<uintptr_t>(s) | uintptr_t(blocks)) & 15) == 0);
    *deep = pitch % 128 == 0;
    if (!*fast) return SWB_OK;
    if (int rc = make_map(&m->w, w, rows, pitch, 128, 16, *deep ? 8 : 0)) return rc;
    return s ? make_map(&m->s, s, rows, blocks, 64, 16) : SWB_OK;
}

}  // namespace swb
