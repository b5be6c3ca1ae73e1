// MXFP4 matrices: rounding to four bits, reading back, and the product of a four-bit
// weight matrix with 16-bit tokens (declarations: include/swiglu_b200.h).
#include <algorithm>
#include <cstring>

#include "host.h"
#include "project.h"
#include "stream.cuh"

namespace swb {
namespace {

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<float> {
    static __device__ __forceinline__ float load(float v) { return v; }
    static __device__ __forceinline__ float store(float v) { return v; }
};

struct RowMap {
    int64_t rows, cols, blocks, total;  // total = rows * blocks
    int64_t pitch;                      // elements from row to row of the unpacked side
    bool flat;                          // rows of whole blocks without gaps: block id starts at value 32 id
};

// Block id -> (row, block of the row); 32-bit division where the ids allow it.
__device__ __forceinline__ void locate(const RowMap& m, int64_t id, int64_t& row, int64_t& block) {
    if (m.total <= 0x7FFFFFFFll) {
        const uint32_t r = uint32_t(id) / uint32_t(m.blocks);
        row = r;
        block = uint32_t(id) - r * uint32_t(m.blocks);
    } else {
        row = id / m.blocks;
        block = id - row * m.blocks;
    }
}

// The scale byte of a block whose largest magnitude has these bits: floor(log2) - 2,
// so that the largest value lands in [4, 8) and saturates at 6; 255 for NaN and
// infinity, which four bits cannot hold.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    if (top >= 0x7F800000u) return 255u;
    return e > 2u ? e - 2u : 0u;
}
// 2^(127 - byte), the exact inverse of the scale (byte <= 252).
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
    return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}

// Where a quad lane's eight values lie, or -1 beyond the row. (The division of locate is a fifth of
// the kernels' instructions, and they are close to bound by those.)
__device__ __forceinline__ int64_t values_at(const RowMap& m, int64_t id, int q) {
    if (m.flat) return id * kMxBlock + q * 8;
    int64_t row, block;
    locate(m, id, row, block);
    const int64_t k = block * kMxBlock + q * 8;
    return k < m.cols ? row * m.pitch + k : -1;
}

// Eight values, and the bits of the largest magnitude as fp32.
template <typename T>
__device__ __forceinline__ uint32_t load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        return top;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::load(e[i]);
        // magnitudes of 16-bit values order like integers, two at a time
        const uint32_t m = 0x7FFF7FFFu;
        const uint32_t t = __vmaxu2(__vmaxu2(a.x & m, a.y & m), __vmaxu2(a.z & m, a.w & m));
        const unsigned short one = static_cast<unsigned short>(max(t & 0xFFFFu, t >> 16));
        return __float_as_uint(Elem<T>::load(*reinterpret_cast<const T*>(&one)));
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 a;
        T* e = reinterpret_cast<T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = Elem<T>::store(v[i]);
        *reinterpret_cast<uint4*>(p) = a;
    }
}

// Bound by bytes: each value is read once (2 or 4 bytes) and leaves 17/32 of a byte.
// VEC: four lanes share a block, each eight values (16-byte loads, the block's largest
// magnitude by two shuffles, one 4-byte word of codes). Otherwise (rows that do not
// start on 16 bytes, or ragged by less than eight values) a warp takes a block, one
// value a lane, so that its loads stay coalesced whatever the alignment.
// 14336 x 4096 bf16: rounding and reading back take 61 us for 297 MB, 4.9 TB/s (a copy: 6.5). Rounding, 34
// us of it, is held by instructions: issue slots 71 % and the integer pipe 74 % busy, DRAM 48 %. Reading
// back: 57, 56 and 41 %, waiting for its loads.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, RowMap m, unsigned char* codes,
                                                       unsigned char* scales) {
    const int lane = threadIdx.x & 31;
    if constexpr (VEC) {
        const int64_t step = int64_t(gridDim.x) * (blockDim.x / 4);
        const int q = lane & 3;
        // whole warps stay together: the loop runs while any quad of the warp has a block
        for (int64_t id = int64_t(blockIdx.x) * (blockDim.x / 4) + threadIdx.x / 4; id - (lane >> 2) < m.total;
             id += step) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            const bool have = id < m.total;
            uint32_t top = 0u;
            if (have) {
                const int64_t at = values_at(m, id, q);
                if (at >= 0) top = load8(x + at, v);
            }
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t byte = scale_byte(top);
            const float inv = inverse_scale(byte);
            uint32_t w = 0u;
            if (byte != 255u) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w |= mx_encode(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
            }
            if (have) {
                reinterpret_cast<uint32_t*>(codes)[id * 4 + q] = w;
                if (q == 0) scales[id] = static_cast<unsigned char>(byte);
            }
        }
    } else {
        const int64_t step = int64_t(gridDim.x) * (blockDim.x / 32);
        for (int64_t id = int64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32; id < m.total; id += step) {
            int64_t row, block;
            locate(m, id, row, block);
            const int64_t k = block * kMxBlock + lane;
            const float v = k < m.cols ? Elem<T>::load(x[row * m.pitch + k]) : 0.f;
            const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v) & 0x7FFFFFFFu);
            const uint32_t byte = scale_byte(top);
            const float mine = v * inverse_scale(byte);
            const float next = __shfl_down_sync(0xFFFFFFFFu, mine, 1);
            const uint32_t pair = byte == 255u ? 0u : mx_encode(mine, next);
            if ((lane & 1) == 0) codes[id * kMxBlockBytes + lane / 2] = static_cast<unsigned char>(pair);
            if (lane == 0) scales[id] = static_cast<unsigned char>(byte);
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned char* __restrict__ codes,
                                                         const unsigned char* __restrict__ scales, RowMap m, T* out) {
    const int lane = threadIdx.x & 31;
    if constexpr (VEC) {
        const int64_t step = int64_t(gridDim.x) * (blockDim.x / 4);
        const int q = lane & 3;
        for (int64_t id = int64_t(blockIdx.x) * (blockDim.x / 4) + threadIdx.x / 4; id < m.total; id += step) {
            const int64_t at = values_at(m, id, q);
            if (at < 0) continue;
            const float s = mx_scale(scales[id]);
            uint32_t p[4];
            mx_decode_f16(reinterpret_cast<const uint32_t*>(codes)[id * 4 + q], p);
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = half2_bits_to_float2(p[i]);
                v[2 * i] = f.x * s;
                v[2 * i + 1] = f.y * s;
            }
            store8(out + at, v);
        }
    } else {
        const int64_t step = int64_t(gridDim.x) * (blockDim.x / 32);
        for (int64_t id = int64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32; id < m.total; id += step) {
            int64_t row, block;
            locate(m, id, row, block);
            const int64_t k = block * kMxBlock + lane;
            if (k >= m.cols) continue;
            const uint32_t c = (codes[id * kMxBlockBytes + lane / 2] >> (4 * (lane & 1))) & 15u;
            uint32_t p[4];
            mx_decode_f16(c, p);
            out[row * m.pitch + k] = Elem<T>::store(half2_bits_to_float2(p[0]).x * mx_scale(scales[id]));
        }
    }
}

template <typename T, bool BACK>
int launch_convert(const void* from, void* to, void* codes, void* scales, const RowMap& m, cudaStream_t stream) {
    const int sms = sm_count();
    if (sms <= 0) return check_launch();
    const void* side = BACK ? to : from;
    const bool vec = m.cols % 8 == 0 && (m.pitch * int64_t(sizeof(T))) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(side) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0;
    const int64_t per = vec ? 64 : 8;  // blocks of 32 values that a CTA of 256 threads takes at once
    const unsigned grid = unsigned(std::min<int64_t>((m.total + per - 1) / per, int64_t(sms) * 32));
    auto* c = static_cast<unsigned char*>(codes);
    auto* s = static_cast<unsigned char*>(scales);
    if constexpr (BACK) {
        if (vec)
            dequantize_kernel<T, true><<<grid, 256, 0, stream>>>(c, s, m, static_cast<T*>(to));
        else
            dequantize_kernel<T, false><<<grid, 256, 0, stream>>>(c, s, m, static_cast<T*>(to));
    } else {
        if (vec)
            quantize_kernel<T, true><<<grid, 256, 0, stream>>>(static_cast<const T*>(from), m, c, s);
        else
            quantize_kernel<T, false><<<grid, 256, 0, stream>>>(static_cast<const T*>(from), m, c, s);
    }
    return check_launch();
}

size_t elem_size(int type) { return type == SWB_F32 ? 4 : 2; }

template <bool BACK>
int convert(int type, const void* from, void* to, int64_t pitch, const void* codes, const void* scales, int64_t rows,
            int64_t cols, void* stream) {
    if (type != SWB_F16 && type != SWB_BF16 && type != SWB_F32) return fail(SWB_E_TYPE);
    if (rows < 0 || cols < 0 || cols > 0x7FFFFFFF - kMxBlock || pitch < cols) return fail(SWB_E_SHAPE);
    if (rows == 0 || cols == 0) return SWB_OK;
    const void* side = BACK ? to : from;
    if (!side || !codes || !scales) return fail(SWB_E_INPUT);
    if (!aligned(elem_size(type), side)) return fail(SWB_E_ALIGNMENT, "values off their type's size");
    RowMap m;
    m.rows = rows;
    m.cols = cols;
    m.blocks = mx_blocks(cols);
    m.total = rows * m.blocks;
    m.pitch = pitch;
    m.flat = cols % kMxBlock == 0 && (pitch == cols || rows == 1);
    const size_t bytes = (size_t(rows - 1) * pitch + cols) * elem_size(type);
    if (overlaps(side, bytes, codes, size_t(m.total) * kMxBlockBytes) || overlaps(side, bytes, scales, size_t(m.total)))
        return fail(SWB_E_OVERLAP_INPUT);
    if (overlaps(codes, size_t(m.total) * kMxBlockBytes, scales, size_t(m.total))) return fail(SWB_E_OVERLAP_OUTPUT);
    auto s = static_cast<cudaStream_t>(stream);
    auto* c = const_cast<void*>(codes);
    auto* sc = const_cast<void*>(scales);
    switch (type) {
        case SWB_F16: return launch_convert<__half, BACK>(from, to, c, sc, m, s);
        case SWB_BF16: return launch_convert<__nv_bfloat16, BACK>(from, to, c, sc, m, s);
        default: return launch_convert<float, BACK>(from, to, c, sc, m, s);
    }
}

}  // namespace
}  // namespace swb

using namespace swb;

extern "C" {

int swb_mx4_quantize(int type, const void* x, int64_t x_pitch, void* codes, void* scales, int64_t rows, int64_t cols,
                     void* stream) {
    return convert<false>(type, x, nullptr, x_pitch, codes, scales, rows, cols, stream);
}

int swb_mx4_dequantize(int type, const void* codes, const void* scales, void* out, int64_t out_pitch, int64_t rows,
                       int64_t cols, void* stream) {
    return convert<true>(type, nullptr, out, out_pitch, codes, scales, rows, cols, stream);
}

int swb_mx4_project(int type, const void* codes, const void* scales, const void* x, int64_t x_pitch, const void* bias,
                    const void* residual, void* out, int64_t tokens, int64_t rows, int64_t cols, unsigned flags,
                    void* stream) {
    if (type != SWB_F16 && type != SWB_BF16) return fail(SWB_E_TYPE);
    if (flags & ~(SWB_RESIDUAL | SWB_HALF_OUT)) return fail(SWB_E_INPUT, "unknown flags");
    if (tokens < 0 || rows <= 0 || cols <= 0 || rows > SWB_MX4_MAX_DIM || cols > SWB_MX4_MAX_DIM || x_pitch < cols)
        return fail(SWB_E_SHAPE);
    if (tokens == 0) return SWB_OK;
    if (tokens > SWB_MX4_MAX_TOKENS) return fail(SWB_E_SHAPE);
    if (!codes || !scales || !x) return fail(SWB_E_INPUT);
    const bool half = (flags & SWB_HALF_OUT) != 0;
    if (!out) return fail(half ? SWB_E_HALF_OUTPUT : SWB_E_FLOAT_OUTPUT);
    if ((flags & SWB_RESIDUAL) && !residual) return fail(SWB_E_RESIDUAL);
    if (!aligned(16, codes)) return fail(SWB_E_ALIGNMENT, "codes must be 16-byte aligned");
    if (!aligned(2, x, bias, (flags & SWB_RESIDUAL) ? residual : nullptr) || !aligned(half ? 2 : 4, out))
        return fail(SWB_E_ALIGNMENT, "values off their type's size");
    const size_t out_bytes = size_t(tokens) * rows * (half ? 2 : 4);
    const size_t blocks = size_t(rows) * mx_blocks(cols);
    if (overlaps(out, out_bytes, codes, blocks * kMxBlockBytes) || overlaps(out, out_bytes, scales, blocks) ||
        overlaps(out, out_bytes, x, (size_t(tokens - 1) * x_pitch + cols) * 2) ||
        (bias && overlaps(out, out_bytes, bias, size_t(rows) * 2)))
        return fail(SWB_E_OVERLAP_INPUT);
    // the residual may be the output itself: each value is read by the thread that writes it
    if ((flags & SWB_RESIDUAL) && !(half && residual == out) &&
        overlaps(out, out_bytes, residual, size_t(tokens) * rows * 2))
        return fail(SWB_E_OVERLAP_INPUT);
    ProjectParams P;
    std::memset(&P, 0, sizeof P);
    P.w = static_cast<const unsigned char*>(codes);
    P.s = static_cast<const unsigned char*>(scales);
    P.x = x;
    P.bias = bias;
    P.residual = (flags & SWB_RESIDUAL) ? residual : nullptr;
    P.out = out;
    P.x_pitch = x_pitch;
    P.tokens = tokens;
    P.rows = int(rows);
    P.cols = int(cols);
    P.half_out = half;
    P.x_aligned = cols % 8 == 0 && x_pitch % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    auto s = static_cast<cudaStream_t>(stream);
    return project_deep_takes(P) ? project_deep(type, P, s) : project_wide(type, P, s);
}

}  // extern "C"
