// Products of a weight matrix with tokens on the fifth-generation tensor cores, for weights
// that are streamed once: 128 rows of W are the M side, the tokens the N side, so that
// 16-bit weights go from global memory to the tensor core without passing a register.
//
// 16-bit weights: tcgen05.mma kind::f16. Four-bit weights: kind::mxf8f6f4, whose operands may
// differ in type: the codes and their power-of-two scales are the M side as they are; a token is
// the sum of `pieces` e4m3 values, each block of 32 with a scale of its own, five binades apart,
// rounded from what the piece before left. Three pieces hold an fp16 value exactly within 13
// binades of its block's largest, and to 2^-27 of the largest below; two hold a bf16 value to
// 2^-22 of it; an fp32 value, such as an expert's h, is held to 2^-14 of it by three. A piece is a
// column of its own; the epilogue
// adds a token's columns. Every product is exact and the sums are the tensor core's fp32.
//
// Roles of a CTA, through two rings of stages of 128 bytes of every row (one for the weights, one
// for the tokens):
//   copies     one thread, TMA: two halves of 64 rows of W (gate and up rows, or neighbours)
//   spreaders  (four-bit) one or two groups of four warps, stage about. Codes arrive packed in a
//              ring of their own, 16 KB a stage, the bytes in flight, and are spread to the eight
//              bytes of every sixteen that the product reads; their scales go into the 32 x 16-byte
//              blocks that tcgen05.cp spreads over TMEM. (The copy engine can spread codes too, at
//              about the same rate.)
//   splitters  tokens from their rows, gathered and split into pieces, or copied where they lie
//              prepared. A stage's chain of conversions takes 0.5 to 1 us whatever its size, so
//              groups of warps each take stages of their own: that chain, done by all warps
//              together stage after stage, held the kernel to a sixth of the memory's rate.
//   products   one thread
//   epilogue   four warps, a TMEM quadrant each
#pragma once

#include "stream.cuh"
#include "tcgen05.cuh"

namespace swb {

constexpr int kWideM = 128, kWideHalf = 64;
constexpr int kWideRowBytes = 128;                     // of a row in a stage, in shared memory
constexpr int kWideA = kWideM * kWideRowBytes;
constexpr int kWideEpilogue = 4;                       // warps
constexpr int kWidePartPitch = kWideM + 1;             // floats of a token's column

// ------------------------------------------------------------ tokens in e4m3 pieces
// The scale byte of the first piece of a block whose largest magnitude has these bits: it brings
// the largest value to [128, 256); pieces 1 and 2 are 5 and 10 less.
__device__ __forceinline__ uint32_t piece_scale(uint32_t top) {
    const uint32_t e = top >> 23;
    return e > 254u ? 127u : e > 17u ? e - 7u : 10u;
}
// Eight values -> PIECES times eight e4m3 bytes. A NaN or an infinity becomes NaN.
template <int PIECES>
__device__ __forceinline__ void split_pieces(float (&f)[8], uint32_t scale, uint2 (&out)[PIECES]) {
    const float inv = __uint_as_float((254u - scale) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] *= inv;
        if (!(fabsf(f[i]) < 1024.f)) f[i] = __uint_as_float(0x7FC00000u);
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        uint32_t pair[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint16_t b;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
            pair[i] = b;
            if (p + 1 < PIECES) {
                uint32_t h;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(b));
                const float2 v = half2_bits_to_float2(h);
                f[2 * i] = (f[2 * i] - v.x) * 32.f;  // exact
                f[2 * i + 1] = (f[2 * i + 1] - v.y) * 32.f;
            }
        }
        out[p] = make_uint2(pair[0] | (pair[1] << 16), pair[2] | (pair[3] << 16));
    }
}

// Eight values of a token (`raw`) -> pieces; the four lanes of a quad hold a block and agree on
// the scale byte, which is returned. bf16 goes through fp32. fp16 stays packed: what a piece leaves
// is exact in fp16 (at most 11 bits), and so are the scalings but for values 2^-32 below the
// block's largest; the first factor is at most 2^15, which holds every bit of smaller blocks too.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
    return max(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
}
template <int PIECES>
__device__ __forceinline__ uint32_t split_token(const uint4& raw, uint2 (&out)[PIECES], __nv_bfloat16) {
    float f[8];
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f[e] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&raw)[e]);
        top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
    }
    const uint32_t scale = piece_scale(quad_max(top));
    split_pieces<PIECES>(f, scale, out);
    return scale;
}
template <int PIECES>
__device__ __forceinline__ uint32_t split_token(const uint4& raw, uint2 (&out)[PIECES], __half) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    // magnitudes as integers order like the values; NaN and infinity lie above all
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
    top = quad_max(max(top & 0xFFFFu, top >> 16));
    const int e = int(top >> 10) - 15;                    // floor(log2) of the largest (or less: subnormal)
    const int up = top >= 0x7C00u ? 0 : min(7 - e, 15);   // it goes to [2^7, 2^8)
    const uint32_t factor = uint32_t(up + 15) << 10 | uint32_t(up + 15) << 26;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(w[i]), "r"(factor));
    if (top >= 0x7C00u) {  // a block with a NaN or an infinity: those become NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((v[i] & 0x7C00u) == 0x7C00u) v[i] |= 0x7FFFu;
            if ((v[i] & 0x7C000000u) == 0x7C000000u) v[i] |= 0x7FFF0000u;
        }
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        uint16_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(b[i]) : "r"(v[i]));
            if (p + 1 < PIECES) {
                uint32_t back;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(b[i]));
                asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(v[i]) : "r"(back));
                asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(v[i]) : "r"(0x50005000u));  // times 32
            }
        }
        out[p] = make_uint2(uint32_t(b[0]) | uint32_t(b[1]) << 16, uint32_t(b[2]) | uint32_t(b[3]) << 16);
    }
    return uint32_t(127 - up);
}

// Where row r's 16-byte piece c lies in a tile of 128-byte rows as the 128-byte swizzle has it.
__device__ __forceinline__ uint32_t swizzled(int r, int c) { return uint32_t(r * 128 + ((c ^ r) & 7) * 16); }
// Byte of row r, block b of 128 values, in its 512-byte block of scales.
__device__ __forceinline__ uint32_t scale_place(int r) {
    return uint32_t((r >> 7) * kScaleBlock + (r & 31) * 16 + ((r >> 5) & 3) * 4);
}

// Whether a phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

// One piece of work: 128 rows of W (two halves of 64) by `count` tokens over stages [s0, s1).
struct WideItem {
    int64_t row[2];  // first row of each half in its tensor
    int s0, s1;
    int count;
    int first;       // the tokens' first index, as the work counts them
};

// W describes the work:
//   types      T; kMx; kPieces; kTok (tokens of an item, a multiple of 16); kLoad (tokens by the
//              splitters; kFloat: rows of fp32 on 16 bytes, `cols` a multiple of eight, times
//              up(it, n), as two 16-bit pieces; else rows `first * kPieces` on of a tensor map, or with kGather rows
//              place(it, n) * kPieces on of `pieces`, `pitch` bytes apart, and for four-bit
//              weights scales `sb`, `pitch_b` apart); kAccs; kStages and kTokenStages (of the
//              rings); kRaw (stages of packed codes); kSpreadGroups; kSplitters (warps) in groups
//              of kGroupWarps; kPerSm
//   item(i, it) -> false past the last one;  token(it, n): row of token n (kLoad)
//   halves: 1 or 2 of 64 rows;  scales of W: sa[2], blocks, rows_a;  x_aligned, cols
//   begin(it) / value(it, n, row, v) / end(it): epilogue threads, by their row
template <typename W>
struct Wide {
    using T = typename W::T;
    static constexpr bool kMx = W::kMx;
    static constexpr int kN = W::kPieces * W::kTok;
    static constexpr int kBytesB = kN * kWideRowBytes;
    static constexpr int kBlocksB = kMx ? (kN + 127) / 128 : 0;
    // A stage of weights: tile, block of scales. A stage of tokens: tile, blocks of scales.
    static constexpr int kStageA = kWideA, kStageB = kBytesB;
    static constexpr int kScaleColumnsA = kMx ? 4 : 0, kScaleColumnsB = 4 * kBlocksB;
    static constexpr int kUsed = W::kAccs * kN + W::kStages * kScaleColumnsA + W::kTokenStages * kScaleColumnsB;
    static constexpr int kColumns = kUsed <= 32 ? 32 : kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static constexpr int kValues = kMx ? 128 : 64;   // of a row in a stage
    static constexpr int kRawStage = kMx ? kWideM * 128 : 0, kRaw = kMx ? W::kRaw : 0;
    static constexpr int kSpreadGroups = kMx ? W::kSpreadGroups : 0, kSpreaders = 4 * kSpreadGroups;
    static constexpr int kSplitters = W::kSplitters, kGroupWarps = W::kGroupWarps;
    static constexpr int kGroups = kSplitters / kGroupWarps;
    static constexpr int kWarps = kWideEpilogue + kSpreaders + kSplitters + 2, kThreads = kWarps * 32;
    static_assert(kUsed <= 512 && kColumns * W::kPerSm <= 512, "TMEM columns");
    static_assert(W::kLoad || kGroupWarps == 1, "a warp brings prepared tokens");
    static_assert(!W::kGather || kMx, "gathered rows are pieces");
    static_assert(!W::kFloat || (W::kLoad && !kMx && W::kPieces == 2), "fp32 rows are split in two");
    // a group that waits for a stage of tokens is at most one round of the ring ahead of its readers
    static_assert(kGroups <= W::kTokenStages, "groups do not overtake the ring");

    // Offsets from the base of the dynamic shared memory (on 1 KB).
    static constexpr uint32_t kAtB = W::kStages * kStageA, kAtRaw = kAtB + W::kTokenStages * kStageB;
    static constexpr uint32_t kAtScalesA = kAtRaw + kRaw * kRawStage;
    static constexpr uint32_t kAtScalesB = kAtScalesA + (kMx ? W::kStages * kScaleBlock : 0);
    static constexpr uint32_t kRing = (kAtScalesB + W::kTokenStages * kBlocksB * kScaleBlock + 1023) / 1024 * 1024;
    static_assert(kStageB % 1024 == 0, "tiles keep the swizzle's alignment");

    struct Shared {
        uint64_t full[W::kStages], empty[W::kStages], acc_full[2], acc_empty[2];
        uint64_t tokens_full[W::kTokenStages], tokens_empty[W::kTokenStages];
        uint64_t raw_full[kRaw + 1], raw_empty[kRaw + 1];
        uint32_t tmem;
        int failed;
    };

    // A place in a ring.
    template <int STAGES>
    struct Ring {
        int s = 0;
        uint32_t ph = 0;
        int64_t issued = 0;
        __device__ __forceinline__ void next() {
            ++issued;
            if (++s == STAGES) s = 0, ph ^= 1u;
        }
        // The stage is free again (a producer's wait).
        __device__ __forceinline__ bool free(uint64_t* empty) const {
            return issued < STAGES || mbar_wait(smem_u32(empty + s), ph ^ 1u);
        }
        // Nothing stays in flight into shared memory when a copier gives up.
        __device__ __forceinline__ void drain(uint64_t* full) const {
            for (int i = 0; i < STAGES && i < issued; ++i) {
                const int64_t idx = issued - 1 - i;
                mbar_wait(smem_u32(full + idx % STAGES), uint32_t(idx / STAGES) & 1u);
            }
        }
    };

    // Groups of warps take the stages of the sequence (item after item) in turn, each its own only:
    // passing over the others' stages one by one cost more than the work on its own. Stage q of
    // the sequence is in slot q % STAGES for the (q / STAGES)-th time.
    template <int STAGES>
    static __device__ __forceinline__ bool slot_free(uint64_t* empty, uint32_t q) {
        const uint32_t use = q / STAGES;
        return use == 0 || mbar_wait(smem_u32(empty + q % STAGES), (use & 1u) ^ 1u);
    }
    // The first stage from s0 on of an item that starts at q0 of the sequence which is `group`'s.
    template <int GROUPS>
    static __device__ __forceinline__ int first_of(int group, uint32_t q0, int s0) {
        return s0 + int((uint32_t(group) + GROUPS - q0 % GROUPS) % GROUPS);
    }

    // Every thread of the CTA, before run(); the CTA synchronises in between.
    static __device__ __forceinline__ void init(Shared& s) {
        if (threadIdx.x == 0) {
            s.failed = 0;
            for (int i = 0; i < W::kStages; ++i) {
                mbar_init(smem_u32(s.full + i), kMx ? 4 : 1);
                mbar_init(smem_u32(s.empty + i), 1);
            }
            for (int i = 0; i < W::kTokenStages; ++i) {
                mbar_init(smem_u32(s.tokens_full + i), kGroupWarps);
                mbar_init(smem_u32(s.tokens_empty + i), 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(smem_u32(s.acc_full + i), 1);
                mbar_init(smem_u32(s.acc_empty + i), kWideEpilogue * 32);
            }
            for (int i = 0; i < kRaw; ++i) {
                mbar_init(smem_u32(s.raw_full + i), 1);
                mbar_init(smem_u32(s.raw_empty + i), 8);  // two stages, four warps each
            }
            mbar_fence_init();
        }
        if (threadIdx.x < 32) tmem_alloc(smem_u32(&s.tmem), kColumns);
        fence_before();
    }
    // Every thread, after run() and a CTA barrier.
    static __device__ __forceinline__ void finish(Shared& s) {
        if (threadIdx.x < 32) {
            fence_after();
            tmem_free(s.tmem, kColumns);
        }
    }
    // Columns of an item.
    static __device__ __forceinline__ int columns(int count) { return (count * W::kPieces + 15) / 16 * 16; }

    // maps: W's two tensors, the prepared tokens.
    static __device__ __forceinline__ void run(W& work, Shared& sh, uint32_t base, const CUtensorMap* map0,
                                               const CUtensorMap* map1, const CUtensorMap* map_b, uint64_t policy) {
        fence_after();
        const int warp = threadIdx.x >> 5;
        bool ok = true;
        if (warp < kWideEpilogue) {
            ok = epilogue(work, sh);
        } else if (warp < kWideEpilogue + kSpreaders) {
            if constexpr (kMx) ok = spread(work, sh, base);
        } else if (warp < kWideEpilogue + kSpreaders + kSplitters) {
            if constexpr (W::kLoad)
                ok = split(work, sh, base);
            else
                ok = bring(work, sh, base, map_b);
        } else if (warp == kWarps - 2) {
            if (elect_one()) ok = copy(work, sh, base, map0, map1, policy);
        } else {
            if (elect_one()) ok = multiply(work, sh, base);
        }
        if (!ok) sh.failed = 1;
        __syncwarp();
        fence_before();
    }

    // Copies of W: 16-bit tiles straight into the products' stages, codes into the raw ring.
    static __device__ __forceinline__ bool copy(W& work, Shared& sh, uint32_t base, const CUtensorMap* map0,
                                                const CUtensorMap* map1, uint64_t policy) {
        constexpr int kStages = kMx ? kRaw : W::kStages, kBytes = kMx ? kRawStage : kStageA;
        uint64_t* full = kMx ? sh.raw_full : sh.full;
        uint64_t* empty = kMx ? sh.raw_empty : sh.empty;
        Ring<kStages> ring;
        WideItem it;
        for (int i = 0; work.item(i, it); ++i) {
            // a raw stage holds two of the products' stages
            const int k0 = kMx ? it.s0 / 2 : it.s0, k1 = kMx ? (it.s1 + 1) / 2 : it.s1;
            for (int k = k0; k < k1; ++k) {
                if (!ring.free(empty)) {
                    ring.drain(full);
                    return false;
                }
                const uint32_t bar = smem_u32(full + ring.s), at = base + (kMx ? kAtRaw : 0u) + ring.s * kBytes;
                mbar_arrive_expect_tx(bar, work.halves * (kBytes / 2));
                const int x = k * (kMx ? 32 : 64);  // elements of four bytes (codes), or of two
                tma_load_2d(at, map0, x, int(it.row[0]), bar, policy);
                if (work.halves == 2) tma_load_2d(at + kBytes / 2, map1, x, int(it.row[1]), bar, policy);
                ring.next();
            }
        }
        return true;
    }

    static __device__ __forceinline__ bool multiply(W& work, Shared& sh, uint32_t base) {
        const uint32_t tmem = sh.tmem, columns_a = tmem + W::kAccs * kN, columns_b = columns_a + W::kStages * kScaleColumnsA;
        Ring<W::kStages> a;
        Ring<W::kTokenStages> b;
        Ring<W::kAccs> acc;
        WideItem it;
        // a stage's barriers are asked for while the stage before is being issued
        bool have_a = false, have_b = false;
        for (int i = 0; work.item(i, it); ++i) {
            const int n = columns(it.count);
            if (!acc.free(sh.acc_empty)) return false;  // the accumulator's last item has been read
            for (int k = it.s0; k < it.s1; ++k) {
                if (!have_a && !mbar_wait(smem_u32(sh.full + a.s), a.ph)) return false;
                if (!have_b && !mbar_wait(smem_u32(sh.tokens_full + b.s), b.ph)) return false;
                const int as = a.s, bs = b.s;
                a.next();
                b.next();
                have_a = mbar_test(smem_u32(sh.full + a.s), a.ph);
                have_b = mbar_test(smem_u32(sh.tokens_full + b.s), b.ph);
                fence_after();
                const uint32_t ca = columns_a + as * kScaleColumnsA, cb = columns_b + bs * kScaleColumnsB;
                if constexpr (kMx) {
                    scale_copy(ca, scale_desc(base + kAtScalesA + as * kScaleBlock));
#pragma unroll
                    for (int j = 0; j < kBlocksB; ++j)
                        scale_copy(cb + 4 * j, scale_desc(base + kAtScalesB + (bs * kBlocksB + j) * kScaleBlock));
                }
                const uint64_t da = operand_desc(base + as * kStageA), db = operand_desc(base + kAtB + bs * kStageB);
                const uint32_t d = tmem + acc.s * kN;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (kMx)
                        mma_mxf8f6f4(d, da + 2 * j, db + 2 * j, mxf8f6f4_desc(kWideM, n, j), ca, cb, k > it.s0 || j > 0);
                    else
                        mma_f16(d, da + 2 * j, db + 2 * j, f16_desc<T>(kWideM, n), k > it.s0 || j > 0);
                }
                mma_commit(smem_u32(sh.empty + as));
                mma_commit(smem_u32(sh.tokens_empty + bs));
                if (k == it.s1 - 1) mma_commit(smem_u32(sh.acc_full + acc.s));
            }
            acc.next();
        }
        return true;
    }

    static __device__ __forceinline__ bool epilogue(W& work, Shared& sh) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const uint32_t quadrant = sh.tmem + (uint32_t(warp * 32) << 16);
        Ring<W::kAccs> acc;
        WideItem it;
        bool ok = true;
        for (int i = 0; work.item(i, it); ++i) {
            // a warp that gives up still comes to the others' barriers
            ok = ok && mbar_wait_warp(smem_u32(sh.acc_full + acc.s), acc.ph);
            fence_after();
            work.begin(it);
#pragma unroll 1
            for (int c = 0; c < it.count && ok; c += 16) {  // 16 tokens, kPieces columns each
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll
                for (int part = 0; part < W::kPieces; ++part) {
                    uint32_t r[16];
                    __syncwarp();
                    tmem_load16(quadrant + acc.s * kN + c * W::kPieces + part * 16, r);
                    tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[(part * 16 + j) / W::kPieces] += __uint_as_float(r[j]);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c + j < it.count) work.value(it, c + j, warp * 32 + lane, v[j]);
            }
            fence_before();
            if (ok) mbar_arrive(smem_u32(sh.acc_empty + acc.s));
            work.end(it);
            acc.next();
        }
        return ok;
    }

    // Spreaders: codes and scales of W. Scale words are loaded four of the group's stages ahead, since
    // they come from DRAM.
    static __device__ __forceinline__ bool spread(W& work, Shared& sh, uint32_t base) {
        constexpr int kGroupsA = kSpreadGroups > 0 ? kSpreadGroups : 1;
        const int group = threadIdx.x / 128 - kWideEpilogue / 4, t = threadIdx.x % 128, lane = t & 31;
        // the thread's row for scales: a warp's words lie side by side in their block
        const int row_a = t / 32 * 8 + (t & 7) + (t >> 3 & 3) * 32, half = row_a / kWideHalf;
        uint32_t q0 = 0, raw0 = 0;
        WideItem it;
        for (int i = 0; work.item(i, it); ++i) {
            const int64_t r = (half ? it.row[1] : it.row[0]) + row_a % kWideHalf;
            const unsigned char* row =
                r < work.rows_a && half < work.halves ? (half ? work.sa[1] : work.sa[0]) + r * work.blocks : nullptr;
            int k = first_of<kGroupsA>(group, q0, it.s0);
            uint32_t word[5];
#pragma unroll
            for (int w = 0; w < 4; ++w) word[w] = scale_word<false>(row, k + w * kGroupsA, it.s1, work.blocks);
            for (; k < it.s1; k += kGroupsA) {
                word[4] = scale_word<false>(row, k + 4 * kGroupsA, it.s1, work.blocks);
                const uint32_t q = q0 + uint32_t(k - it.s0), s = q % W::kStages;
                const uint32_t raw = raw0 + uint32_t(k / 2 - it.s0 / 2), rs = raw % kRaw;
                const bool ready = mbar_wait(smem_u32(sh.raw_full + rs), raw / kRaw & 1u) && slot_free<W::kStages>(sh.empty, q);
                if (!__all_sync(0xFFFFFFFFu, ready)) return false;
                // a warp takes eight rows, four blocks of 16 bytes each, at a time
                const uint32_t from = base + kAtRaw + rs * kRawStage, to = base + s * kStageA;
                const int block = lane >> 3;
                uint4 c[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) c[u] = lds128(from + swizzled((t / 32 + u * 4) * 8 + (lane & 7), k % 2 * 4 + block));
                sts32(base + kAtScalesA + s * kScaleBlock + scale_place(row_a), word[0]);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int n = (t / 32 + u * 4) * 8 + (lane & 7);
                    sts64(to + swizzled(n, 2 * block), c[u].x, c[u].y);
                    sts64(to + swizzled(n, 2 * block + 1), c[u].z, c[u].w);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(sh.full + s));
                    mbar_arrive(smem_u32(sh.raw_empty + rs));
                    // a raw stage of which the item takes one half only
                    if ((k == it.s0 && k % 2 == 1) || (k == it.s1 - 1 && k % 2 == 0)) mbar_arrive(smem_u32(sh.raw_empty + rs));
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) word[w] = word[w + 1];
            }
            q0 += uint32_t(it.s1 - it.s0);
            raw0 += uint32_t((it.s1 + 1) / 2 - it.s0 / 2);
        }
        return true;
    }
    // The four scale bytes of stage k of a row, zero beyond it. The non-coherent load is for W's, which
    // nothing writes while the kernel runs. A token's (WRITTEN) come from the workspace, where other
    // CTAs of this launch, or the launch before while this one is already resident, put them.
    template <bool WRITTEN>
    static __device__ __forceinline__ uint32_t scale_word(const unsigned char* row, int k, int end, int blocks) {
        if (!row || k >= end) return 0u;
        if ((blocks & 3) == 0 && (reinterpret_cast<uintptr_t>(row) & 3) == 0) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(row) + k;
            return WRITTEN ? __ldcg(p) : __ldg(p);
        }
        uint32_t w = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k * 4 + e < blocks) w |= uint32_t(WRITTEN ? __ldcg(row + k * 4 + e) : __ldg(row + k * 4 + e)) << (8 * e);
        return w;
    }

    // Splitters: tokens from their rows.
    static __device__ __forceinline__ bool split(W& work, Shared& sh, uint32_t base) {
        constexpr int kPer = kMx ? 16 : 8;                    // eight-value parts of a row in a stage
        constexpr int kStride = kGroupWarps * 32 / kPer;      // tokens taken at once
        constexpr int kTurns = (W::kTok + kStride - 1) / kStride, kBatch = kTurns < 4 ? kTurns : 4;
        const int warp = threadIdx.x / 32 - kWideEpilogue - kSpreaders, group = warp / kGroupWarps;
        const int t = threadIdx.x - (kWideEpilogue + kSpreaders + group * kGroupWarps) * 32, j = t % kPer, n0 = t / kPer;
        uint32_t q0 = 0;
        WideItem it;
        uint4 x[kTurns], second[W::kFloat ? kTurns : 1];
        for (int i = 0; work.item(i, it); ++i) {
            auto load = [&](int k) {
                if (k >= it.s1) return;
#pragma unroll
                for (int u = 0; u < kTurns; ++u) {
                    if (u * kStride >= it.count) break;
                    const auto* row = work.token(it, min(n0 + u * kStride, it.count - 1));
                    const int at = k * kValues + j * 8;
                    if constexpr (W::kFloat) {
                        const uint4* p = reinterpret_cast<const uint4*>(row + at);
                        x[u] = at < work.cols ? __ldcg(p) : make_uint4(0u, 0u, 0u, 0u);
                        second[u] = at < work.cols ? __ldcg(p + 1) : make_uint4(0u, 0u, 0u, 0u);
                    } else
                        x[u] = work.x_aligned ? load_piece<T, true>(row, at, work.cols) : load_piece<T, false>(row, at, work.cols);
                }
            };
            int k = first_of<kGroups>(group, q0, it.s0);
            load(k);
            for (; k < it.s1; k += kGroups) {
                const uint32_t q = q0 + uint32_t(k - it.s0), s = q % W::kTokenStages;
                if (!__all_sync(0xFFFFFFFFu, slot_free<W::kTokenStages>(sh.tokens_empty, q))) return false;
                const uint32_t b = base + kAtB + s * kStageB, sc = base + kAtScalesB + s * kBlocksB * kScaleBlock;
#pragma unroll
                for (int u0 = 0; u0 < kTurns; u0 += kBatch) {
                    if (u0 * kStride >= it.count) break;  // whole groups: the shuffles stay together
                    if constexpr (!kMx) {
#pragma unroll
                        for (int u = u0; u < u0 + kBatch && u < kTurns; ++u) {
                            const int n = n0 + u * kStride;
                            if constexpr (W::kFloat) {
                                if (n >= it.count) continue;
                                uint4 hi, lo;
                                split_pairs(x[u], second[u], work.up(it, n), hi, lo);
                                sts128(b + swizzled(2 * n, j), hi.x, hi.y, hi.z, hi.w);
                                sts128(b + swizzled(2 * n + 1, j), lo.x, lo.y, lo.z, lo.w);
                            } else if (n < it.count)
                                sts128(b + swizzled(n, j), x[u].x, x[u].y, x[u].z, x[u].w);
                        }
                    } else {
                        uint2 piece[kBatch][W::kPieces];
                        uint32_t scale[kBatch];
#pragma unroll
                        for (int u = 0; u < kBatch; ++u)
                            scale[u] = split_token<W::kPieces>(x[u0 + u < kTurns ? u0 + u : kTurns - 1], piece[u], T());
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            const int n = n0 + (u0 + u) * kStride;
                            if (n >= it.count) continue;
#pragma unroll
                            for (int p = 0; p < W::kPieces; ++p) {
                                const int r = n * W::kPieces + p;
                                sts64(b + swizzled(r, j / 2) + (j & 1) * 8, piece[u][p].x, piece[u][p].y);
                                if ((j & 3) == 0) sts8(sc + scale_place(r) + j / 4, scale[u] - 5u * p);
                            }
                        }
                    }
                }
                load(k + kGroups);
                fence_proxy_async_smem();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(sh.tokens_full + s));
            }
            q0 += uint32_t(it.s1 - it.s0);
        }
        return true;
    }

    // Prepared tokens: a warp brings a stage's rows, by TMA or (gathered) by asynchronous copies, and
    // their scale words by plain loads.
    static __device__ __forceinline__ bool bring(W& work, Shared& sh, uint32_t base, const CUtensorMap* map_b) {
        const int lane = threadIdx.x & 31, group = threadIdx.x / 32 - kWideEpilogue - kSpreaders;
        uint32_t q0 = 0;
        WideItem it;
        for (int i = 0; work.item(i, it); ++i) {
            const int n = columns(it.count), rows = it.count * W::kPieces;
            for (int k = first_of<kGroups>(group, q0, it.s0); k < it.s1; k += kGroups) {
                const uint32_t q = q0 + uint32_t(k - it.s0), s = q % W::kTokenStages;
                const uint32_t bar = smem_u32(sh.tokens_full + s), b = base + kAtB + s * kStageB;
                if (!__all_sync(0xFFFFFFFFu, slot_free<W::kTokenStages>(sh.tokens_empty, q))) {
                    // this warp's copies have landed where its earlier stages were read; the last ones may not
                    if (!W::kGather && lane == 0 && q >= kGroups)
                        mbar_wait(smem_u32(sh.tokens_full + (q - kGroups) % W::kTokenStages), (q - kGroups) / W::kTokenStages & 1u);
                    return false;
                }
                if constexpr (W::kGather) {  // eight lanes a row
                    for (int r = lane / 8; r < rows; r += 4) {
                        const int64_t from = int64_t(work.place(it, r / W::kPieces)) * W::kPieces + r % W::kPieces;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(b + swizzled(r, lane & 7)),
                                     "l"(work.pieces + from * work.pitch + k * kWideRowBytes + (lane & 7) * 16) : "memory");
                    }
                } else if (elect_one()) {
                    mbar_expect_tx(bar, n * kWideRowBytes);
                    for (int r = 0; r < n; r += 16)
                        tma_load_2d(b + r * kWideRowBytes, map_b, k * kValues, it.first * W::kPieces + r, bar);
                }
                if constexpr (kMx) {
                    const uint32_t sc = base + kAtScalesB + s * kBlocksB * kScaleBlock;
                    uint32_t word[(kN + 31) / 32];
#pragma unroll
                    for (int u = 0; u < (kN + 31) / 32; ++u) {
                        const int r = lane + 32 * u;
                        const unsigned char* row = nullptr;
                        if (r < rows) {
                            const int n = r / W::kPieces, token = W::kGather ? work.place(it, n) : it.first + n;
                            row = work.sb + (int64_t(token) * W::kPieces + r % W::kPieces) * work.pitch_b;
                        }
                        word[u] = scale_word<true>(row, k, it.s1, work.pitch_b);
                    }
#pragma unroll
                    for (int u = 0; u < (kN + 31) / 32; ++u)
                        if (lane + 32 * u < rows) sts32(sc + scale_place(lane + 32 * u), word[u]);
                    if (W::kGather) asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            }
            q0 += uint32_t(it.s1 - it.s0);
        }
        return true;
    }
};

// ------------------------------------------------------------ host
// Whether W's rows can be copied: whole 16-byte rows (of codes: always, and the calls require it).
inline bool wide_rows(const void* w, int64_t cols, bool mx) {
    return mx || (cols % 8 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0);
}
// Map of W [rows, cols] in boxes of 64 rows by 128 bytes.
inline int make_wide_map(CUtensorMap* map, const void* w, int64_t rows, int64_t cols, bool mx) {
    return mx ? make_map(map, w, rows, mx_blocks(cols) * kMxBlockBytes, 128, kWideHalf)
              : make_typed_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, w, cols, rows, cols * 2, 64, kWideHalf);
}

}  // namespace swb
