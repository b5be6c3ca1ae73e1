// Products of a weight matrix with tokens on the fifth-generation tensor cores, for weights
// that are streamed once: 128 rows of W are the M side, the tokens the N side, so that the
// weights go from global memory to the tensor core without passing a register.
//
// 16-bit weights: tcgen05.mma kind::f16. Four-bit weights: kind::mxf8f6f4, whose operands may
// differ in type: the codes (spread to a byte each by the copy) and their power-of-two scales
// are the M side as they are; a token is the sum of `pieces` e4m3 values, each block of 32 with
// a scale of its own, five binades apart, rounded from what the piece before left. Three pieces
// hold 15 bits below a block's largest value (all of an fp16 value within 13 binades of it, and
// 2^-27 of the largest beyond), two hold 9 (bf16). A piece is a column of its own; the epilogue
// adds a token's columns. Every product is exact and the sums are the tensor core's fp32.
//
// Roles of a CTA (10 or 14 warps), through a ring of stages of 128 bytes of every row:
//   copies     one thread, TMA: two halves of 64 rows of W (gate and up rows, or neighbours), and
//              the tokens where they lie prepared in memory
//   loaders    four warps, or eight that split tokens: tokens from their rows (gathered, split into pieces), scale bytes of
//              both sides into the 32 x 16-byte blocks that tcgen05.cp spreads over TMEM
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

// One piece of work: 128 rows of W (two halves of 64) by `count` tokens over stages [s0, s1).
struct WideItem {
    int64_t row[2];  // first row of each half in its tensor
    int s0, s1;
    int count;
    int first;       // the tokens' first index, as the work counts them
};

// W describes the work:
//   types      T; kMx; kPieces; kTok (tokens of an item, a multiple of 16); kLoad (tokens by the
//              loaders; else rows `first * kPieces` on of a tensor map); kAccs; kStages; kPerSm
//   item(i, it) -> false past the last one;  token(it, n): row of token n (kLoad)
//   halves: 1 or 2 of 64 rows;  scales of W: sa[2], blocks, rows_a;  of tokens that lie prepared: sb
//   begin(it) / value(it, n, row, v) / end(it): epilogue threads, by their row
template <typename W>
struct Wide {
    using T = typename W::T;
    static constexpr bool kMx = W::kMx;
    static constexpr int kN = W::kPieces * W::kTok;
    static constexpr int kBytesB = kN * kWideRowBytes;
    static constexpr int kBlocksB = kMx ? (kN + 127) / 128 : 0;
    static constexpr int kScales = kMx ? (1 + kBlocksB) * kScaleBlock : 0;
    static constexpr int kStage = (kWideA + kBytesB + kScales + 1023) / 1024 * 1024;
    static constexpr int kScaleColumns = kMx ? 4 * (1 + kBlocksB) : 0;
    static constexpr int kUsed = W::kAccs * kN + W::kStages * kScaleColumns;
    static constexpr int kColumns = kUsed <= 32 ? 32 : kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static constexpr int kValues = kMx ? 128 : 64;   // of a row in a stage
    static constexpr int kRowSource = kMx ? 64 : 128;  // their bytes in W
    static constexpr bool kLoaders = W::kLoad || kMx;
    static constexpr int kWideLoaders = kMx && W::kLoad ? 8 : 4;  // warps
    static constexpr int kThreads = (kWideEpilogue + kWideLoaders + 2) * 32;
    static_assert(kUsed <= 512 && kColumns * W::kPerSm <= 512, "TMEM columns");
    static constexpr size_t kRing = size_t(W::kStages) * kStage;

    struct Shared {
        uint64_t full[W::kStages], loaded[W::kStages], empty[W::kStages], acc_full[2], acc_empty[2];
        uint32_t tmem;
        int failed;
    };

    // Every thread of the CTA, before run(); the CTA synchronises in between.
    static __device__ __forceinline__ void init(Shared& s) {
        if (threadIdx.x == 0) {
            s.failed = 0;
            for (int i = 0; i < W::kStages; ++i) {
                mbar_init(smem_u32(s.full + i), 1);
                mbar_init(smem_u32(s.loaded + i), kWideLoaders * 32);
                mbar_init(smem_u32(s.empty + i), 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(smem_u32(s.acc_full + i), 1);
                mbar_init(smem_u32(s.acc_empty + i), kWideEpilogue * 32);
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
    // Columns of an item: whole groups of 16 tokens.
    static __device__ __forceinline__ int columns(int count) { return (count + 15) / 16 * 16 * W::kPieces; }

    // base: the ring, on 1 KB. maps: W's two tensors, the prepared tokens.
    static __device__ __forceinline__ void run(W& work, Shared& sh, uint32_t base, const CUtensorMap* map0,
                                               const CUtensorMap* map1, const CUtensorMap* map_b, uint64_t policy) {
        fence_after();
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const uint32_t tmem = sh.tmem, scale_columns = tmem + W::kAccs * kN;
        int s = 0;
        uint32_t ph = 0;
        int64_t issued = 0;
        bool ok = true;
        auto next_stage = [&] {
            ++issued;
            if (++s == W::kStages) s = 0, ph ^= 1u;
        };
        WideItem it;

        if (warp == kWideEpilogue + kWideLoaders) {
            if (lane == 0) {
                for (int i = 0; ok && work.item(i, it); ++i) {
                    const int n = columns(it.count);
                    for (int k = it.s0; k < it.s1; ++k) {
                        if (issued >= W::kStages && !mbar_wait(smem_u32(sh.empty + s), ph ^ 1u)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bar = smem_u32(sh.full + s), at = base + s * kStage;
                        mbar_arrive_expect_tx(bar, work.halves * kWideHalf * kRowSource + (W::kLoad ? 0 : n * kWideRowBytes));
                        tma_load_2d(at, map0, k * kValues, int(it.row[0]), bar, policy);
                        if (work.halves == 2) tma_load_2d(at + kWideA / 2, map1, k * kValues, int(it.row[1]), bar, policy);
                        if (!W::kLoad) {
                            for (int r = 0; r < n; r += 16)
                                tma_load_2d(at + kWideA + r * kWideRowBytes, map_b, k * kValues, it.first * W::kPieces + r, bar);
                        }
                        next_stage();
                    }
                }
                if (!ok) {  // nothing stays in flight into shared memory
                    for (int i = 0; i < W::kStages && i < issued; ++i) {
                        const int64_t idx = issued - 1 - i;
                        mbar_wait(smem_u32(sh.full + idx % W::kStages), uint32_t(idx / W::kStages) & 1u);
                    }
                    sh.failed = 1;
                }
            }
        } else if (warp == kWideEpilogue + kWideLoaders + 1) {
            if (lane == 0) {
                int acc = 0, done = 0;
                uint32_t aph = 0;
                for (int i = 0; ok && work.item(i, it); ++i, ++done) {
                    const int n = columns(it.count);
                    if (done >= W::kAccs) {  // the accumulator's last item has been read
                        ok = mbar_wait(smem_u32(sh.acc_empty + acc), aph ^ 1u);
                        if (!ok) break;
                    }
                    for (int k = it.s0; k < it.s1; ++k) {
                        ok = mbar_wait(smem_u32(sh.full + s), ph) && (!kLoaders || mbar_wait(smem_u32(sh.loaded + s), ph));
                        if (!ok) break;
                        fence_after();
                        const uint32_t at = base + s * kStage, col = scale_columns + s * kScaleColumns;
                        if constexpr (kMx) {
#pragma unroll
                            for (int j = 0; j < 1 + kBlocksB; ++j)
                                scale_copy(col + 4 * j, scale_desc(at + kWideA + kBytesB + j * kScaleBlock));
                        }
                        const uint64_t da = operand_desc(at), db = operand_desc(at + kWideA);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (kMx)
                                mma_mxf8f6f4(tmem + acc * kN, da + 2 * j, db + 2 * j, mxf8f6f4_desc(kWideM, n, j), col, col + 4,
                                             k > it.s0 || j > 0);
                            else
                                mma_f16(tmem + acc * kN, da + 2 * j, db + 2 * j, f16_desc<T>(kWideM, n), k > it.s0 || j > 0);
                        }
                        mma_commit(smem_u32(sh.empty + s));
                        if (k == it.s1 - 1) mma_commit(smem_u32(sh.acc_full + acc));
                        next_stage();
                    }
                    if (++acc == W::kAccs) acc = 0, aph ^= 1u;
                }
                if (!ok) sh.failed = 1;
            }
        } else if (warp >= kWideEpilogue) {
            if constexpr (kLoaders) ok = load(work, sh, base);
            if (!ok) sh.failed = 1;
        } else {
            int acc = 0;
            uint32_t aph = 0;
            const uint32_t quadrant = uint32_t(warp * 32) << 16;
            for (int i = 0; work.item(i, it); ++i) {
                ok = mbar_wait_warp(smem_u32(sh.acc_full + acc), aph);
                if (!ok) break;
                fence_after();
                work.begin(it);
#pragma unroll 1
                for (int c = 0; c < it.count; c += 16) {  // 16 tokens, kPieces columns each
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll
                    for (int part = 0; part < W::kPieces; ++part) {
                        uint32_t r[16];
                        __syncwarp();
                        tmem_load16(tmem + quadrant + acc * kN + c * W::kPieces + part * 16, r);
                        tmem_load_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[(part * 16 + j) / W::kPieces] += __uint_as_float(r[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (c + j < it.count) work.value(it, c + j, warp * 32 + lane, v[j]);
                }
                fence_before();
                mbar_arrive(smem_u32(sh.acc_empty + acc));
                work.end(it);
                if (++acc == W::kAccs) acc = 0, aph ^= 1u;
            }
            if (!ok) sh.failed = 1;
        }
        __syncwarp();
        fence_before();
    }

    // Loader warps: tokens and scale bytes of every stage, the next stage's on their way meanwhile.
    static __device__ __forceinline__ bool load(W& work, Shared& sh, uint32_t base) {
        constexpr int kPer = kMx ? 16 : 8;                       // 8-value parts of a row in a stage
        constexpr int kStride = kWideLoaders * 32 / kPer;        // tokens taken at once
        constexpr int kTurns = W::kLoad ? (W::kTok + kStride - 1) / kStride : 1;
        constexpr int kRowsB = W::kLoad ? 1 : (kN + 127) / 128;  // rows of prepared scales of a thread
        const int t = threadIdx.x - kWideEpilogue * 32, j = t % kPer, n0 = t / kPer;
        int s = 0;
        uint32_t ph = 0;
        int64_t issued = 0;
        WideItem it;
        for (int i = 0; work.item(i, it); ++i) {
            const typename W::T* x[kTurns];
            const unsigned char *row_a = nullptr, *row_b[kRowsB];
            if constexpr (W::kLoad) {
#pragma unroll
                for (int u = 0; u < kTurns; ++u) x[u] = work.token(it, min(n0 + u * kStride, it.count - 1));
            }
            if (kMx && t < kWideM) {
                const int half = t / kWideHalf;
                const int64_t r = (half ? it.row[1] : it.row[0]) + t % kWideHalf;
                if (r < work.rows_a && half < work.halves) row_a = (half ? work.sa[1] : work.sa[0]) + r * work.blocks;
#pragma unroll
                for (int u = 0; u < kRowsB; ++u) {
                    const int b = t + 128 * u;
                    row_b[u] = !W::kLoad && b < it.count * W::kPieces ? work.sb + int64_t(it.first * W::kPieces + b) * work.blocks : nullptr;
                }
            }
            uint4 xv[kTurns];
            auto load_x = [&](int k) {
                if constexpr (W::kLoad) {
#pragma unroll
                    for (int u = 0; u < kTurns; ++u) {
                        if (u * kStride >= it.count) break;
                        const int at = k * kValues + j * 8;
                        xv[u] = work.x_aligned ? load_piece<T, true>(x[u], at, work.cols) : load_piece<T, false>(x[u], at, work.cols);
                    }
                }
            };
            // Windows of 16 scale bytes, four stages each, two windows ahead: W's come from DRAM.
            uint4 win_a[3] = {}, win_b[3][kRowsB] = {};
            auto load_windows = [&](int w, int k) {
                if constexpr (kMx) {
                    const bool have = k < it.s1;
                    win_a[w] = row_a && have ? load_scales(row_a, k / 4 * 16, work.blocks) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                    for (int u = 0; u < kRowsB; ++u)
                        win_b[w][u] = row_b[u] && have ? load_scales(row_b[u], k / 4 * 16, work.blocks) : make_uint4(0u, 0u, 0u, 0u);
                }
            };
            load_x(it.s0);
            load_windows(0, it.s0);
            load_windows(1, (it.s0 | 3) + 1);
            load_windows(2, (it.s0 | 3) + 5);
            for (int k = it.s0; k < it.s1; ++k) {
                uint4 now[kTurns];
#pragma unroll
                for (int u = 0; u < kTurns; ++u) now[u] = xv[u];
                if (kMx && k > it.s0 && k % 4 == 0) {
                    win_a[0] = win_a[1], win_a[1] = win_a[2];
#pragma unroll
                    for (int u = 0; u < kRowsB; ++u) win_b[0][u] = win_b[1][u], win_b[1][u] = win_b[2][u];
                    load_windows(2, k + 8);
                }
                if (k + 1 < it.s1) load_x(k + 1);
                if (issued >= W::kStages && !mbar_wait_warp(smem_u32(sh.empty + s), ph ^ 1u)) return false;
                const uint32_t b = base + s * kStage + kWideA, sc = b + kBytesB;
                if (kMx && t < kWideM) sts32(sc + scale_place(t), word_of(win_a[0], k));
                if constexpr (kMx && !W::kLoad) {
#pragma unroll
                    for (int u = 0; u < kRowsB; ++u)
                        if (t + 128 * u < kN) sts32(sc + kScaleBlock + scale_place(t + 128 * u), word_of(win_b[0][u], k));
                }
                if constexpr (W::kLoad) {
#pragma unroll
                    for (int u = 0; u < kTurns; ++u) {
                        if (u * kStride >= it.count) break;  // whole warps: the shuffles below stay together
                        const int n = n0 + u * kStride;
                        if constexpr (!kMx) {
                            if (n < it.count)
                                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(b + swizzled(n, j)), "r"(now[u].x), "r"(now[u].y), "r"(now[u].z), "r"(now[u].w) : "memory");
                        } else {
                            uint2 piece[W::kPieces];
                            const uint32_t scale = split_token<W::kPieces>(now[u], piece, T());
                            if (n < it.count) {
#pragma unroll
                                for (int p = 0; p < W::kPieces; ++p) {
                                    const int r = n * W::kPieces + p;
                                    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(b + swizzled(r, j / 2) + (j & 1) * 8), "r"(piece[p].x), "r"(piece[p].y) : "memory");
                                    if ((j & 3) == 0) sts8(sc + kScaleBlock + scale_place(r) + j / 4, scale - 5u * p);
                                }
                            }
                        }
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(smem_u32(sh.loaded + s));
                ++issued;
                if (++s == W::kStages) s = 0, ph ^= 1u;
            }
        }
        return true;
    }
    static __device__ __forceinline__ uint32_t word_of(const uint4& w, int k) {
        return k & 2 ? (k & 1 ? w.w : w.z) : (k & 1 ? w.y : w.x);
    }
};

// ------------------------------------------------------------ host
// Whether W's rows can be copied for the tensor core: whole 16-byte rows, or codes in pairs of
// 32-byte pieces of 128 values.
inline bool wide_rows(const void* w, int64_t cols, bool mx) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(w);
    return mx ? mx_blocks(cols) % 4 == 0 && a % 32 == 0 : cols % 8 == 0 && a % 16 == 0;
}
// Map of W [rows, cols] in boxes of 64 rows by 128 bytes of shared memory.
inline int make_wide_map(CUtensorMap* map, const void* w, int64_t rows, int64_t cols, bool mx) {
    const int64_t padded = mx_blocks(cols) * kMxBlock;
    return mx ? make_typed_map(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, w, padded, rows, padded / 2, 128, kWideHalf)
              : make_typed_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, w, cols, rows, cols * 2, 64, kWideHalf);
}

}  // namespace swb
