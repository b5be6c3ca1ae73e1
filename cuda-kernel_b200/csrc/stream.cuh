// Products of a streamed weight matrix with a few 16-bit tokens, as mma.sync tiles.
//
// A CTA works through items: one or two tiles of 16 weight rows (NM: the gate's and the
// up projection's rows of one expert, or two neighbouring tiles of a matrix) against up
// to NT * 8 tokens over the whole row. Few-token products are bound by the bytes of the
// weights, so the CTA is a pipeline that never drains between items:
//
//   producer   one thread brings the tiles' next 1 or 2 KB of each row, by TMA, into a ring
//              of stages, running ahead across items as far as the ring goes
//   consumers  kWarps warps share each stage by columns; weights are the m16n8k16 A operand,
//              eight tokens the B operand, sums in fp32. The tokens, a few KB that every item
//              reads again, come through L1 into registers. (With the weights on the same
//              path their latency would be the weights': loads return in order.)
//   epilogue   three warps add the consumers' partial sums, kept in shared memory, and finish
//              the item while the consumers are at the next one.
//
// The order of k inside 32 values is free as long as both operands agree, so a lane's four
// registers of A and of B are one 16-byte piece of its row.
//
// MXFP4: codes are decoded in registers, each block of 32 values is summed from zero and
// added to the totals times its scale (both scales are powers of two, so the only
// roundings are the fp32 sums').
//
// Rows that do not start on 16 bytes (16-bit matrices of ragged sizes, scales of ragged
// rows) have no tensor map: each lane of the producer warp copies a row's piece from the 16
// bytes before it (a bulk copy each, about half the rate), and consumers read it shifted.
// Waits are bounded.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "device.cuh"
#include "mx4.cuh"
#include "tensor_map.h"

namespace swb {

constexpr int kTileRows = 16;
constexpr int kUnitBytes = 64;  // of a row: what a consumer warp multiplies at once

template <typename T>
struct Num;
template <>
struct Num<__half> {
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void decode(uint32_t w, uint32_t (&p)[4]) { mx_decode_f16(w, p); }
    // the decoder's order of k within eight consecutive values
    static __device__ __forceinline__ uint4 order(const uint4& v) { return v; }
};
template <>
struct Num<__nv_bfloat16> {
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void decode(uint32_t w, uint32_t (&p)[4]) { mx_decode_bf16(w, p); }
    static __device__ __forceinline__ uint4 order(const uint4& v) {  // pairs (i, i + 4)
        return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                          __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
    }
};

// A row of fp32 values goes through the tensor cores as two values of T: the nearest, and what the
// rounding left, rounded. bf16 has fp32's range, and both are made where the value is. With fp16 the
// row is first divided by a unit, a power of two that brings its largest value to [2^14, 2^15), so
// that fp32's range is kept and only values 2^-28 below the largest meet fp16's subnormals (errors
// within 2^-39 of it); the sums are multiplied by the unit. `top`: the bits of the largest
// magnitude; NaN and infinity stay what they are.
__device__ __forceinline__ float row_unit(uint32_t top) {
    const uint32_t e = top >> 23;
    return __uint_as_float((e > 254u ? 127u : max(e, 15u) - 14u) << 23);
}
__device__ __forceinline__ float unit_inverse(float unit) { return __uint_as_float((254u << 23) - __float_as_uint(unit)); }
// Eight fp32 values times `up` -> both fp16 parts.
__device__ __forceinline__ void split_pairs(const uint4& a, const uint4& b, float up, uint4& hi, uint4& lo) {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = __uint_as_float(w[2 * i]) * up, y = __uint_as_float(w[2 * i + 1]) * up;  // exact
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[i]) : "f"(y), "f"(x));
        const float2 back = half2_bits_to_float2(h[i]);
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(l[i]) : "f"(y - back.y), "f"(x - back.x));
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Shared loads by 32-bit address, left to the compiler to schedule between barriers.
__device__ __forceinline__ const void* smem_ptr(uint32_t a) {
    extern __shared__ __align__(1024) unsigned char smem[];  // keeps the loads in the shared space
    return smem + (a - smem_u32(smem));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) { return *static_cast<const uint4*>(smem_ptr(a)); }
__device__ __forceinline__ uint32_t lds32(uint32_t a) { return *static_cast<const uint32_t*>(smem_ptr(a)); }
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void sts8(uint32_t a, uint32_t v) {
    asm volatile("st.shared.u8 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t a, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// mbar_wait for a whole warp, with one answer for its lanes.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
}
// L2 policy for weights that another item reads again.
__device__ __forceinline__ uint64_t l2_normal_policy() {
    uint64_t pol;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}
// True in one lane of a converged warp. The instructions that one thread issues (copies, tensor-core
// products) take their operands from uniform registers; under this condition the compiler knows
// that one lane runs, under `lane == 0` it emits a loop over the active lanes for each of them
// (about 80 clocks an instruction, measured on bulk copies and on the products' issue).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// TMA tile loads; the barrier counts whole boxes.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// A tensor of row-major matrices of one shape as the copies see it: the codes or values,
// and for MXFP4 the scales.
struct WeightView {
    const unsigned char* begin[2];  // of the whole tensor: values or codes, scales
    const unsigned char* end[2];
    int pitch[2];                   // bytes of a row: values or codes, scales
    int cols;
    int units;                      // kUnitBytes pieces of a row, the last one ragged
    const WeightMaps* maps;         // null: rows (16-bit) or rows of scales (MXFP4) not on 16 bytes
    bool deep;                      // WeightMaps: boxes of 1 KB of a row
};

template <bool MX>
__device__ __forceinline__ WeightView weight_view(const unsigned char* w, const unsigned char* s, int64_t rows, int cols,
                                                  const WeightMaps* maps, bool deep) {
    WeightView v;
    const int blocks = int(mx_blocks(cols));
    v.pitch[0] = MX ? blocks * kMxBlockBytes : cols * 2;
    v.pitch[1] = blocks;
    v.begin[0] = w;
    v.begin[1] = s;
    v.end[0] = w + rows * v.pitch[0];
    v.end[1] = s + (MX ? rows * blocks : 0);
    v.cols = cols;
    v.units = (v.pitch[0] + kUnitBytes - 1) / kUnitBytes;
    v.maps = maps;
    v.deep = deep;
    return v;
}

// Eight values of a token's row from k on, zero beyond `cols`; ALIGNED: 16-byte pieces.
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 load_piece(const T* row, int k, int cols) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (k >= cols) return v;
    if constexpr (ALIGNED) return *reinterpret_cast<const uint4*>(row + k);
    const unsigned short* r = reinterpret_cast<const unsigned short*>(row);
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < cols ? r[k + i] : 0u;
    v.x = e[0] | (e[1] << 16);
    v.y = e[2] | (e[3] << 16);
    v.z = e[4] | (e[5] << 16);
    v.w = e[6] | (e[7] << 16);
    return v;
}

// One item's weights: NM tiles, each the first row's index in its tensor and how many
// of its 16 rows exist.
template <int NM>
struct Tiles {
    int64_t row[NM];
    int rows[NM];
};

constexpr int kEpilogueThreads = 96;
constexpr int kPartPitch = 17;
constexpr int kRingTarget = 160 * 1024;

template <typename T, bool MX, int NT>
struct Stream {
    // Decoding four-bit codes for few tokens keeps the schedulers busy only with four warps each.
    static constexpr int kConsumers = MX ? 16 : 8;
    static constexpr int kThreads = (kConsumers + 4) * 32;  // consumers, producer, epilogue
    // A stage: 2 tiles of 16 rows by 1 KB, or one tile by 2 KB. With maps: 128 bytes of 16 rows
    // after another (kBox), swizzled by the copy; scales 64 bytes of 16 rows after another.
    // Without: row after row, at pitches that leave 16 bytes for a shifted row.
    template <int NM>
    struct Shape {
        static constexpr int kChunk = 2048 / NM;
        static constexpr int kPitch = kChunk + (MX ? 16 : 64);
        static constexpr int kScalePitch = kChunk / kMxBlockBytes + 16;
        static constexpr int kTile = kTileRows * kPitch;
        static constexpr int kScales = NM * kTile;  // offset of the scales in a stage
        static constexpr int kBytes = kScales + (MX ? NM * kTileRows * kScalePitch : 0);
        static constexpr int kBoxes = kChunk / 128;  // of a tile
        static constexpr int kUnits = kChunk / kUnitBytes;
        static constexpr int kPart = NM * NT * 8 * kPartPitch;  // floats of a consumer's partial sums
    };
    static constexpr int kBox = kTileRows * 128, kScaleBox = kTileRows * 64;
    static constexpr int kBoxScales = 32 * 1024;  // offset of the scales in a stage
    static constexpr int kStage = (Shape<2>::kBytes > Shape<1>::kBytes ? Shape<2>::kBytes : Shape<1>::kBytes) / 1024 * 1024 + 1024;
    static_assert(kStage >= kBoxScales + (MX ? 2 * kScaleBox : 0), "a stage holds either layout");
    // The tile's row that is row g of the A operand. 16-bit: eight lanes read 16 bytes of two
    // operand rows at a time; rows four apart have their halves of 128 swizzled bytes apart.
    static __device__ __forceinline__ int tile_row(int g) { return MX ? g : ((g & 1) << 2) | (g >> 1); }
    static constexpr int kPartFloats = kConsumers * Shape<2>::kPart;
    static constexpr int kParts = NT >= 4 ? 1 : 2;  // buffers of partial sums
    static constexpr int kSub = MX ? 4 : 1;         // groups of 32 values in a unit

    // Shared memory: ring (on 1 KB), partial sums, barriers.
    struct Layout {
        uint32_t ring, part, full, empty, part_full, part_empty;
        int stages;
    };
    static constexpr size_t kFixed = size_t(kParts) * kPartFloats * 4 + 2 * kParts * 8;
    __host__ __device__ static constexpr size_t bytes(int stages) { return size_t(stages) * (kStage + 16) + kFixed; }
    // as many stages as fit beside `other` bytes and the ring's share (L1 has the rest)
    __host__ __device__ static constexpr int stages(size_t other) {
        int n = 8;
        while (bytes(n) + other > 232448 - 1024 || n * kStage > kRingTarget) --n;
        return n;
    }

    static __device__ __forceinline__ Layout layout(uint32_t base, int stages) {
        Layout l;
        l.stages = stages;
        l.ring = base;
        l.part = base + stages * kStage;
        l.full = l.part + kParts * kPartFloats * 4;
        l.empty = l.full + stages * 8;
        l.part_full = l.empty + stages * 8;
        l.part_empty = l.part_full + kParts * 8;
        return l;
    }
    // One thread; the CTA synchronises afterwards.
    static __device__ __forceinline__ void init(const Layout& l) {
        for (int i = 0; i < l.stages; ++i) {
            mbar_init(l.full + 8 * i, 1);
            mbar_init(l.empty + 8 * i, kConsumers);
        }
        for (int i = 0; i < kParts; ++i) {
            mbar_init(l.part_full + 8 * i, kConsumers);
            mbar_init(l.part_empty + 8 * i, kEpilogueThreads / 32);
        }
        mbar_fence_init();
    }

    // Where a role stands in the ring and in the buffers of partial sums.
    struct Place {
        int stage = 0, part = 0;
        uint32_t phase = 0, part_phase = 0;
        int64_t issued = 0;
        bool ok = true;
        __device__ __forceinline__ void next_stage(int stages) {
            if (++stage == stages) stage = 0, phase ^= 1u;
        }
        __device__ __forceinline__ void next_part() {
            if (++part == kParts) part = 0, part_phase ^= 1u;
        }
    };

    // Copies [from, from + bytes) of a tensor to dst, from the 16 bytes before `from` on;
    // returns the bytes that complete on the barrier. Where that would leave the tensor, the
    // lane copies them itself.
    static __device__ __forceinline__ uint32_t copy_shifted(uint32_t dst, const unsigned char* from, int bytes,
                                                            const unsigned char* begin, const unsigned char* end,
                                                            uint32_t bar, uint64_t policy) {
        const unsigned char* lo = from - (reinterpret_cast<uintptr_t>(from) & 15);
        const int n = (int(from - lo) + bytes + 15) & ~15;
        if (lo >= begin && lo + n <= end) {
            mbar_expect_tx(bar, n);
            bulk_copy_g2s(dst, lo, n, bar, policy);
            return n;
        }
        const int at = int(from - lo);
        for (int i = 0; i < bytes; ++i) sts8(dst + at + i, from[i]);
        fence_proxy_async_smem();  // before a later bulk copy to the same place
        return 0;
    }

    // Producer warp: the stages of one item. The copies are the only accesses to the weights.
    template <int NM>
    static __device__ __forceinline__ void produce(const Layout& l, Place& p, const Tiles<NM>& t,
                                                   const WeightView (&v)[NM], uint64_t policy) {
        if (!v[0].maps) {
            produce_rows<NM>(l, p, t, v, policy);
            return;
        }
        using S = Shape<NM>;
        const int chunks = (v[0].units + S::kUnits - 1) / S::kUnits;
        for (int c = 0; c < chunks; ++c) {
            if (p.issued >= l.stages && !mbar_wait_warp(l.empty + 8 * p.stage, p.phase ^ 1u)) {
                p.ok = false;
                break;
            }
            const uint32_t bar = l.full + 8 * p.stage, at = l.ring + p.stage * kStage;
            const int left = v[0].pitch[0] - c * S::kChunk;  // bytes of each row from here on
            const int boxes = v[0].deep ? (left + 1023) / 1024 * 8 : (left + 127) / 128, n = min(S::kBoxes, boxes);
            const int scales = MX ? min(S::kChunk / 1024, (left + 1023) / 1024) : 0;
            if (elect_one()) {  // the other lanes keep their place in the ring
                mbar_arrive_expect_tx(bar, NM * (n * kBox + scales * kScaleBox));
#pragma unroll
                for (int m = 0; m < NM; ++m) {
                    const int row = int(t.row[m]);
                    if (v[0].deep) {
                        for (int i = 0; i < n; i += 8)
                            tma_load_3d(at + (m * S::kBoxes + i) * kBox, &v[m].maps->w, 0, row, c * S::kBoxes + i, bar, policy);
                    } else {
                        for (int i = 0; i < n; ++i)
                            tma_load_2d(at + (m * S::kBoxes + i) * kBox, &v[m].maps->w, (c * S::kChunk + i * 128) / 4, row, bar, policy);
                    }
                    for (int i = 0; i < scales; ++i)
                        tma_load_2d(at + kBoxScales + (m + i) * kScaleBox, &v[m].maps->s,
                                    (c * (S::kChunk / kMxBlockBytes) + i * 64) / 4, row, bar, policy);
                }
            }
            __syncwarp();
            ++p.issued;
            p.next_stage(l.stages);
        }
    }

    template <int NM>
    static __device__ __noinline__ void produce_rows(const Layout& l, Place& p, const Tiles<NM>& t,
                                                     const WeightView (&v)[NM], uint64_t policy) {
        using S = Shape<NM>;
        const int lane = threadIdx.x & 31;
        const int m = lane / kTileRows, r = lane % kTileRows;
        const int chunks = (v[0].units + S::kUnits - 1) / S::kUnits;
        const bool mine = NM == 2 ? r < (m ? t.rows[NM - 1] : t.rows[0]) : lane < kTileRows && r < t.rows[0];
        const bool second = NM == 2 && m;  // this lane copies rows of the second tile
        const int64_t row = (second ? t.row[NM - 1] : t.row[0]) + r;
        const unsigned char* wb = second ? v[NM - 1].begin[0] : v[0].begin[0];
        const unsigned char* we = second ? v[NM - 1].end[0] : v[0].end[0];
        const unsigned char* sb = second ? v[NM - 1].begin[1] : v[0].begin[1];
        const unsigned char* se = second ? v[NM - 1].end[1] : v[0].end[1];
        const unsigned char* w = wb + row * v[0].pitch[0];
        const unsigned char* s = sb + row * v[0].pitch[1];
        for (int c = 0; c < chunks && p.ok; ++c) {
            if (p.issued >= l.stages && !mbar_wait_warp(l.empty + 8 * p.stage, p.phase ^ 1u)) {
                p.ok = false;
                break;
            }
            const uint32_t bar = l.full + 8 * p.stage, at = l.ring + p.stage * kStage;
            const int bytes = min(S::kChunk, v[0].pitch[0] - c * S::kChunk);
            if (mine) {
                const uint32_t dst = at + (NM == 2 ? m * S::kTile : 0) + r * S::kPitch;
                if (MX) {  // codes always start on 16 bytes
                    mbar_expect_tx(bar, bytes);
                    bulk_copy_g2s(dst, w + c * S::kChunk, bytes, bar, policy);
                } else {
                    copy_shifted(dst, w + c * S::kChunk, bytes, wb, we, bar, policy);
                }
                if (MX) {
                    const int n = bytes / kMxBlockBytes, off = c * (S::kChunk / kMxBlockBytes);
                    const uint32_t to = at + S::kScales + (NM == 2 ? m * kTileRows + r : r) * S::kScalePitch;
                    copy_shifted(to, s + off, n, sb, se, bar, policy);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);  // the stage is full once every copy has landed
            ++p.issued;
            p.next_stage(l.stages);
        }
    }

    // Producer, at its end: nothing stays in flight into shared memory if it gave up.
    static __device__ __forceinline__ void drain(const Layout& l, const Place& p) {
        if (p.ok) return;
        for (int i = 0; i < l.stages && i < p.issued; ++i) {
            const int64_t idx = p.issued - 1 - i;
            mbar_wait(l.full + 8 * uint32_t(idx % l.stages), uint32_t(idx / l.stages) & 1u);
        }
    }

    // Scales as floats. A byte moved to the exponent field is the scale, but for the bytes 0
    // (2^-127, subnormal) and 255 (NaN); a warp that meets one takes the exact conversion.
    static __device__ __forceinline__ bool special_scale(uint32_t w) {
        return (((w - 0x01010101u) & ~w) | ((~w - 0x01010101u) & w)) & 0x80808080u;
    }
    template <bool SPECIAL>
    static __device__ __forceinline__ float scale_of(uint32_t w, int b) {
        if constexpr (SPECIAL) return mx_scale((w >> (8 * b)) & 255u);
        return __uint_as_float((b < 3 ? w << (23 - 8 * b) : w >> 1) & 0x7F800000u);
    }

    // One group of 32 values of an MXFP4 unit: `a`: this lane's word of row g in the first tile.
    template <int NM, bool SPLIT, bool SPECIAL, bool FAST, int NP>
    static __device__ __forceinline__ void multiply_mx(float (&acc)[NM][NT][4], const uint4 (&x)[NP], uint32_t a,
                                                       const uint32_t (&sc)[NM][2], int b, int count) {
        using S = Shape<NM>;
        constexpr int kTile = FAST ? S::kBoxes * kBox : S::kTile, kHalf = FAST ? 8 * 128 : 8 * S::kPitch;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            uint32_t lo[4], hi[4];
            Num<T>::decode(lds32(a + m * kTile), lo);
            Num<T>::decode(lds32(a + m * kTile + kHalf), hi);
            const float sl = scale_of<SPECIAL>(sc[m][0], b), sh = scale_of<SPECIAL>(sc[m][1], b);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= count) break;
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                Num<T>::mma(d, lo[0], hi[0], lo[1], hi[1], x[n].x, x[n].y);
                Num<T>::mma(d, lo[2], hi[2], lo[3], hi[3], x[n].z, x[n].w);
                if (SPLIT) {
                    Num<T>::mma(d, lo[0], hi[0], lo[1], hi[1], x[NP - NT + n].x, x[NP - NT + n].y);
                    Num<T>::mma(d, lo[2], hi[2], lo[3], hi[3], x[NP - NT + n].z, x[NP - NT + n].w);
                }
                acc[m][n][0] = fmaf(d[0], sl, acc[m][n][0]);
                acc[m][n][1] = fmaf(d[1], sl, acc[m][n][1]);
                acc[m][n][2] = fmaf(d[2], sh, acc[m][n][2]);
                acc[m][n][3] = fmaf(d[3], sh, acc[m][n][3]);
            }
        }
    }

    // The tokens of an item as a consumer lane reads them: its row of each group of eight; with
    // SPLIT, rows of 32 bytes for every eight values, which are multiplied as two values of T: fp32
    // with fp16 (`top`: row_unit), eight first parts and eight second parts with bf16; zero up to a
    // multiple of eight. A warp takes every kConsumers-th unit of a stage and loads its tokens kGroup
    // sub-steps of 32 values ahead, into the next item too: enough that they come from L2 in time.
    template <int NM, bool SPLIT>
    struct Tokens {
        static constexpr int kRows = SPLIT ? 2 * NT : NT;
        static constexpr int kSteps = Shape<NM>::kUnits / kConsumers * kSub;  // sub-steps of a warp in a full stage
        static constexpr int kMost = kConsumers == 16 ? 4 / kRows : 8 / kRows;  // that the registers hold
        static constexpr int kGroup = kMost < 1 ? 1 : kMost > 4 ? (kSteps < 4 ? kSteps : 4) : kMost < kSteps ? kMost : kSteps;
        const std::conditional_t<SPLIT, float, T>* x[NT];  // this lane's rows
        uint32_t top[NT];
        int count;  // tokens; 0: no item
        uint4 ahead[kGroup][kRows];

        // k of this lane's piece in sub-step s of chunk c
        static __device__ __forceinline__ int k_of(int c, int s) {
            const int warp = threadIdx.x >> 5, q = threadIdx.x & 3;
            return ((c * Shape<NM>::kUnits + warp + s / kSub * kConsumers) * kSub + s % kSub) * 32 + q * 8;
        }
        template <bool FAST>
        __device__ __forceinline__ void load(int c, int s, int cols) {
#pragma unroll
            for (int i = 0; i < kGroup; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n * 8 >= count) break;
                    const int k = k_of(c, s + i);
                    if constexpr (SPLIT) {
                        const uint4* p = reinterpret_cast<const uint4*>(x[n] + k);
                        ahead[i][n] = k < cols ? p[0] : make_uint4(0u, 0u, 0u, 0u);
                        ahead[i][NT + n] = k < cols ? p[1] : make_uint4(0u, 0u, 0u, 0u);
                    } else {
                        ahead[i][n] = load_piece<T, FAST>(x[n], k, cols);
                    }
                }
        }
    };

    // Consumer warp: one item. tokens.ahead holds its first values; following(tokens) turns tokens to
    // the next item (count 0: none). FAST: the weights have maps and the rows of x start on 16
    // bytes. Leaves the partial sums in the next buffer.
    template <int NM, bool SPLIT, bool FAST, typename Next>
    static __device__ __forceinline__ void consume(const Layout& l, Place& p, const Tiles<NM>& t,
                                                   const WeightView (&v)[NM], Tokens<NM, SPLIT>& tokens, int x_cols,
                                                   Next&& following) {
        using S = Shape<NM>;
        constexpr int NP = Tokens<NM, SPLIT>::kRows, kSteps = Tokens<NM, SPLIT>::kSteps, kGroup = Tokens<NM, SPLIT>::kGroup;
        const int count = tokens.count;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
        float acc[NM][NT][4];
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[m][n][c] = 0.f;
        float up[NT];
        if constexpr (SPLIT && std::is_same<T, __half>::value) {
#pragma unroll
            for (int n = 0; n < NT; ++n) up[n] = unit_inverse(row_unit(tokens.top[n]));
        }
        const int row = tile_row(g);  // and row + 8
        // how far these rows are shifted in their stage
        uint32_t shift[NM][2];
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                shift[m][h] = FAST ? 0u
                                   : uint32_t(reinterpret_cast<uintptr_t>(v[m].begin[MX ? 1 : 0]) +
                                              (t.row[m] + row + 8 * h) * v[m].pitch[MX ? 1 : 0]) & 15u;
        const int chunks = (v[0].units + S::kUnits - 1) / S::kUnits;
        for (int c = 0; c < chunks; ++c) {
            const int units = min(S::kUnits, v[0].units - c * S::kUnits);
            if (!mbar_wait_warp(l.full + 8 * p.stage, p.phase)) {
                p.ok = false;
                break;
            }
            const uint32_t at = l.ring + p.stage * kStage;
#pragma unroll 1
            for (int s = 0; s < kSteps; s += kGroup) {
                uint4 now[kGroup][NP];
#pragma unroll
                for (int i = 0; i < kGroup; ++i) {
                    constexpr bool kFloat = SPLIT && std::is_same<T, __half>::value;
                    if constexpr (kFloat) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            if (n * 8 < count) split_pairs(tokens.ahead[i][n], tokens.ahead[i][NT + n], up[n], now[i][n], now[i][NT + n]);
                    }
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const uint4& v = kFloat ? now[i][n] : tokens.ahead[i][n];
                        now[i][n] = MX ? Num<T>::order(v) : v;
                    }
                }
                if (s + kGroup < kSteps) {
                    tokens.template load<FAST>(c, s + kGroup, x_cols);
                } else if (c + 1 < chunks) {
                    tokens.template load<FAST>(c + 1, 0, x_cols);
                } else {
                    following(tokens);
                    tokens.template load<FAST>(0, 0, x_cols);
                }
                if constexpr (MX) {
                    const int u = warp + s / kSub * kConsumers;  // a group lies within a unit
                    if (u >= units) continue;
                    uint32_t sc[NM][2];
                    bool special = false;
#pragma unroll
                    for (int m = 0; m < NM; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = row + 8 * h;
                            if (FAST) {
                                sc[m][h] = lds32(at + kBoxScales + (m + u / 16) * kScaleBox + r * 64 +
                                                 (((u >> 2) ^ (r >> 1)) & 3) * 16 + (u & 3) * 4);
                            } else {
                                const uint32_t b = at + S::kScales + (m * kTileRows + r) * S::kScalePitch + u * 4 + shift[m][h];
                                sc[m][h] = __funnelshift_r(lds32(b & ~3u), lds32((b & ~3u) + 4), (b & 3u) * 8);
                            }
                            special |= special_scale(sc[m][h]);
                        }
                    const int subs = v[0].pitch[1] - (c * S::kUnits + u) * kSub;  // blocks left in the row
                    // this lane's word of block b: of its row, q-th in the block
                    const uint32_t a = FAST ? at + (u >> 1) * kBox + row * 128 + q * 4 : at + row * S::kPitch + u * kUnitBytes + q * 4;
                    auto block = [&](int b) { return FAST ? a + ((((u & 1) * 4 + b) ^ row) & 7) * 16 : a + b * 16; };
                    if (__any_sync(0xFFFFFFFFu, special) || subs < kSub) {
#pragma unroll
                        for (int i = 0; i < kGroup; ++i) {
                            const int b = s % kSub + i;
                            if (b < subs) multiply_mx<NM, SPLIT, true, FAST>(acc, now[i], block(b), sc, b, count);
                        }
                    } else if constexpr (kGroup == kSub) {
#pragma unroll
                        for (int i = 0; i < kGroup; ++i)
                            multiply_mx<NM, SPLIT, false, FAST>(acc, now[i], block(i), sc, i, count);
                    } else {
#pragma unroll
                        for (int i = 0; i < kGroup; ++i) {
                            uint32_t shifted[NM][2];  // this sub-step's bytes lowest
#pragma unroll
                            for (int m = 0; m < NM; ++m)
#pragma unroll
                                for (int h = 0; h < 2; ++h) shifted[m][h] = sc[m][h] >> (8 * (s % kSub + i));
                            multiply_mx<NM, SPLIT, false, FAST>(acc, now[i], block(s % kSub + i), shifted, 0, count);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kGroup; ++i) {
                        const int u = warp + (s + i) * kConsumers;
                        if (u >= units) break;
                        const int left = v[0].cols - Tokens<NM, SPLIT>::k_of(c, s + i);  // values of this lane's pieces that the row has
#pragma unroll
                        for (int m = 0; m < NM; ++m) {
                            uint4 a[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (FAST) {
                                    a[h] = lds128(at + (m * S::kBoxes + (u >> 1)) * kBox + (row + 8 * h) * 128 +
                                                  ((((u & 1) * 4 + q) ^ row) & 7) * 16);
                                } else {
                                    const uint32_t b = at + m * S::kTile + (row + 8 * h) * S::kPitch + u * kUnitBytes + q * 16 + shift[m][h];
                                    const uint32_t f = (b & 2u) * 8;
                                    uint32_t w[5];
#pragma unroll
                                    for (int j = 0; j < 5; ++j) w[j] = lds32((b & ~3u) + 4 * j);
#pragma unroll
                                    for (int j = 0; j < 4; ++j) {
                                        w[j] = __funnelshift_r(w[j], w[j + 1], f);
                                        if (2 * j + 1 >= left) w[j] = 2 * j >= left ? 0u : w[j] & 0xFFFFu;
                                    }
                                    a[h] = make_uint4(w[0], w[1], w[2], w[3]);
                                }
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                if (n * 8 >= count) break;
                                Num<T>::mma(acc[m][n], a[0].x, a[1].x, a[0].y, a[1].y, now[i][n].x, now[i][n].y);
                                Num<T>::mma(acc[m][n], a[0].z, a[1].z, a[0].w, a[1].w, now[i][n].z, now[i][n].w);
                                if (SPLIT) {
                                    Num<T>::mma(acc[m][n], a[0].x, a[1].x, a[0].y, a[1].y, now[i][NP - NT + n].x, now[i][NP - NT + n].y);
                                    Num<T>::mma(acc[m][n], a[0].z, a[1].z, a[0].w, a[1].w, now[i][NP - NT + n].z, now[i][NP - NT + n].w);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(l.empty + 8 * p.stage);
            p.next_stage(l.stages);
        }
        if (!p.ok) return;
        // the buffer's last sums are read
        if (p.issued >= kParts && !mbar_wait_warp(l.part_empty + 8 * p.part, p.part_phase ^ 1u)) {
            p.ok = false;
            return;
        }
        const uint32_t part = l.part + (p.part * kPartFloats + warp * S::kPart) * 4;
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= count) break;
                const uint32_t a = part + ((m * NT * 8 + n * 8 + 2 * q) * kPartPitch + row) * 4;
                sts32(a, __float_as_uint(acc[m][n][0]));
                sts32(a + kPartPitch * 4, __float_as_uint(acc[m][n][1]));
                sts32(a + 32, __float_as_uint(acc[m][n][2]));
                sts32(a + (kPartPitch + 8) * 4, __float_as_uint(acc[m][n][3]));
            }
        __syncwarp();
        if (lane == 0) mbar_arrive(l.part_full + 8 * p.part);
        p.issued++;
        p.next_part();
    }

    // Epilogue threads: waits for an item's partial sums; sum(tile, token, row) adds them up;
    // release() frees the buffer.
    static __device__ __forceinline__ bool acquire(const Layout& l, Place& p) {
        if (!mbar_wait_warp(l.part_full + 8 * p.part, p.part_phase)) p.ok = false;
        return p.ok;
    }
    template <int NM>
    static __device__ __forceinline__ float sum(const Layout& l, const Place& p, int m, int token, int row) {
        const uint32_t a = l.part + (p.part * kPartFloats + (m * NT * 8 + token) * kPartPitch + row) * 4;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) s += __uint_as_float(lds32(a + w * Shape<NM>::kPart * 4));
        return s;
    }
    static __device__ __forceinline__ void release(const Layout& l, Place& p) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(l.part_empty + 8 * p.part);
        p.next_part();
    }
};

}  // namespace swb
