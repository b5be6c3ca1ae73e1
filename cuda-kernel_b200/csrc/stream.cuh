// Products of a streamed weight matrix with a few 16-bit tokens, as mma.sync tiles.
//
// A warp takes 16 rows of a matrix (or of NM matrices, or NM such tiles) and a range
// of steps along the row; a step is 64 bytes of every row: 32 values of a 16-bit
// matrix, 128 of an MXFP4 one. The weights are the m16n8k16 A operand, eight tokens
// per N tile the B operand, sums in fp32. The order of k inside a step is free as
// long as both operands agree, so each lane keeps the 16 bytes of its row that it
// loaded itself (16-bit matrices) and reads B as one 16-byte piece of a token's row.
//
// Batch-one and few-token products are bound by the bytes of the weights: every warp
// keeps STAGES - 1 steps in flight through its own ring of asynchronous copies (no
// barrier between warps), while the tokens, a few KB that every tile reads again,
// come through L1 into registers one sub-step ahead.
//
// MXFP4: a step's codes are decoded in registers, each block of 32 values is summed
// from zero and added to the totals times its scale (both scales are powers of two,
// so the only roundings are the fp32 sums'). The copies swap pieces between lanes of
// a quad through the ring, hence the warp barrier after each wait.
#pragma once

#include "device.cuh"
#include "mx4.cuh"

namespace swb {

constexpr int kTileRows = 16;
constexpr int kStepBytes = 64;  // of each row

template <typename T>
struct Num;
template <>
struct Num<__half> {
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
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
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
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

// Global -> shared, 16 bytes, of which the first `valid` are read and the rest zeroed.
// Weights are read once: past L1.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// A row-major weight matrix as the copies see it.
struct WeightView {
    int64_t pitch;   // bytes from row to row
    int row_bytes;   // bytes of one row
    int blocks;      // MXFP4: scale bytes of one row
    int steps;       // kStepBytes pieces of one row, the last one filled up with zeros
    bool aligned;    // 16-byte rows (16-bit matrices) / 4-byte rows of scales (MXFP4)
};

// A token's row as B pieces: `cols` values, `aligned` when every piece is 16 aligned bytes.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* row, int k, int cols, bool aligned) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (k >= cols) return v;
    if (aligned) return *reinterpret_cast<const uint4*>(row + k);
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

// One warp's piece of work: NM tiles of 16 rows (`rows` of them exist), steps [s0, s1),
// `count` tokens whose rows each lane's `x` names.
template <typename T, int NM, int NT>
struct Piece {
    const unsigned char* w[NM];  // first byte of the tile's first row
    const unsigned char* s[NM];  // MXFP4: its first scale byte
    int rows[NM];
    int s0, s1;
    int count;
    const T* x[NT];
};

template <typename T, bool MX, int NM, int NT, int STAGES>
struct WarpStream {
    static constexpr int kTileBytes = kTileRows * kStepBytes;
    static constexpr int kScaleBytes = MX ? kTileRows * 4 : 0;
    static constexpr int kStage = NM * (kTileBytes + kScaleBytes);
    static constexpr int kRing = kStage * STAGES;
    static constexpr int kSub = MX ? 4 : 1;  // groups of 32 values in a step

    // Where in the ring lane 4g + q's 16 bytes of half a tile go. MXFP4: a quad's lanes
    // read each other's pieces a word at a time; the rotation keeps those reads free of
    // bank conflicts.
    static __device__ __forceinline__ uint32_t slot(int g, int q) {
        return uint32_t(g * 4 + (MX ? ((q + (g >> 1)) & 3) : q)) * 16u;
    }

    static __device__ __forceinline__ void fetch(const Piece<T, NM, NT>& p, int step, uint32_t stage,
                                                 const WeightView& v, int lane) {
        const int g = lane >> 2, q = lane & 3;
        const int off = step * kStepBytes + q * 16;
        const int left = min(16, v.row_bytes - off);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = g + 8 * half;
                const int valid = row < p.rows[m] ? max(left, 0) : 0;
                const unsigned char* src = valid > 0 ? p.w[m] + row * v.pitch + off : p.w[m];
                const uint32_t dst = stage + m * kTileBytes + half * (kTileBytes / 2) + slot(g, q);
                if (MX || v.aligned) {
                    copy16(dst, src, valid);
                } else {
                    const unsigned short* r = reinterpret_cast<const unsigned short*>(src);
                    uint32_t e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[i] = 2 * i < valid ? r[i] : 0u;
                    sts128(dst, make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16),
                                           e[6] | (e[7] << 16)));
                }
            }
            if (MX && lane < kTileRows) {
                const int b0 = step * 4;
                const bool have = lane < p.rows[m];
                const unsigned char* src = have ? p.s[m] + int64_t(lane) * v.blocks + b0 : p.s[m];
                const uint32_t dst = stage + NM * kTileBytes + (m * kTileRows + lane) * 4;
                if (v.aligned) {
                    copy4(dst, src, have ? 4 : 0);
                } else {
                    uint32_t w = 0u;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (have && b0 + i < v.blocks) w |= uint32_t(src[i]) << (8 * i);
                    sts32(dst, w);
                }
            }
        }
    }

    static __device__ __forceinline__ void load_tokens(const Piece<T, NM, NT>& p, int sub, int cols, bool aligned,
                                                       int lane, uint4 (&x)[NT]) {
        const int k = sub * 32 + (lane & 3) * 8;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n * 8 < p.count) x[n] = load_piece<T>(p.x[n], k, cols, aligned);
    }

    static __device__ __forceinline__ void multiply(float (&acc)[NM][NT][4], const uint4 (&x)[NT], uint32_t stage,
                                                    int sub, int count, int lane) {
        const int g = lane >> 2, q = lane & 3;
        if constexpr (!MX) {
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const uint4 lo = lds128(stage + m * kTileBytes + slot(g, q));
                const uint4 hi = lds128(stage + m * kTileBytes + kTileBytes / 2 + slot(g, q));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n * 8 >= count) break;
                    Num<T>::mma(acc[m][n], lo.x, hi.x, lo.y, hi.y, x[n].x, x[n].y);
                    Num<T>::mma(acc[m][n], lo.z, hi.z, lo.w, hi.w, x[n].z, x[n].w);
                }
            }
        } else {
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const uint32_t at = stage + m * kTileBytes + slot(g, sub) + q * 4;
                uint32_t lo[4], hi[4];
                Num<T>::decode(lds32(at), lo);
                Num<T>::decode(lds32(at + kTileBytes / 2), hi);
                const uint32_t sc = stage + NM * kTileBytes + (m * kTileRows + g) * 4;
                const float sl = mx_scale((lds32(sc) >> (8 * sub)) & 255u);
                const float sh = mx_scale((lds32(sc + 32) >> (8 * sub)) & 255u);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n * 8 >= count) break;
                    const uint4 b = Num<T>::order(x[n]);
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                    Num<T>::mma(c, lo[0], hi[0], lo[1], hi[1], b.x, b.y);
                    Num<T>::mma(c, lo[2], hi[2], lo[3], hi[3], b.z, b.w);
                    acc[m][n][0] = fmaf(c[0], sl, acc[m][n][0]);
                    acc[m][n][1] = fmaf(c[1], sl, acc[m][n][1]);
                    acc[m][n][2] = fmaf(c[2], sh, acc[m][n][2]);
                    acc[m][n][3] = fmaf(c[3], sh, acc[m][n][3]);
                }
            }
        }
    }

    // Runs pieces 0, 1, ... of a warp: get(i, piece) -> false past the last one;
    // done(i, piece, acc) after each, in order, with the piece's sums.
    template <typename Get, typename Done>
    static __device__ __forceinline__ void run(uint32_t ring, const WeightView& v, int cols, bool x_aligned,
                                               Get&& get, Done&& done) {
        const int lane = threadIdx.x & 31;
        Piece<T, NM, NT> f;
        int fi = 0;
        bool more = get(fi, f);
        int fs = more ? f.s0 : 0;
        auto feed = [&](int stage) {
            while (more && fs >= f.s1) {
                more = get(++fi, f);
                if (more) fs = f.s0;
            }
            if (more) {
                fetch(f, fs, ring + stage * kStage, v, lane);
                ++fs;
            }
            copy_commit();
        };
#pragma unroll 1
        for (int s = 0; s < STAGES - 1; ++s) feed(s);
        int stage = 0;
        Piece<T, NM, NT> p;
        for (int i = 0; get(i, p); ++i) {
            float acc[NM][NT][4];
#pragma unroll
            for (int m = 0; m < NM; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[m][n][c] = 0.f;
            uint4 x[NT];
            if (p.s0 < p.s1) load_tokens(p, p.s0 * kSub, cols, x_aligned, lane, x);
#pragma unroll 1
            for (int s = p.s0; s < p.s1; ++s) {
                copy_wait<STAGES - 2>();
                __syncwarp();  // the step's copies by every lane have landed; the stage to refill is read
                feed(stage == 0 ? STAGES - 1 : stage - 1);
                const uint32_t at = ring + stage * kStage;
#pragma unroll
                for (int b = 0; b < kSub; ++b) {
                    uint4 now[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) now[n] = x[n];
                    if (b + 1 < kSub || s + 1 < p.s1) load_tokens(p, s * kSub + b + 1, cols, x_aligned, lane, x);
                    multiply(acc, now, at, b, p.count, lane);
                }
                stage = stage + 1 == STAGES ? 0 : stage + 1;
            }
            done(i, p, acc);
        }
        copy_wait<0>();
        __syncwarp();
    }
};

// ------------------------------------------------------------ a CTA's share
//
// A CTA takes its items (16-row tiles) in rounds of W, W/2, ..., 1 so that W warps
// share a round's items evenly, each item's steps split over the W / r warps that
// share it. Partial sums meet in shared memory: part[warp][tile][token][17 rows].
constexpr int kPartPitch = 17;

struct Round {
    int first, items;  // items [first, first + items) of the list
};

__device__ __forceinline__ int round_count(int items, int warps) {
    return items / warps + __popc(items & (warps - 1));
}

__device__ __forceinline__ Round round_at(int i, int items, int warps) {  // warps: a power of two
    const int full = items / warps;
    if (i < full) return {i * warps, warps};
    int first = full * warps, rest = items & (warps - 1), skip = i - full;
    for (int bit = warps >> 1;; bit >>= 1) {
        if (rest & bit) {
            if (skip == 0) return {first, bit};
            --skip;
            first += bit;
        }
    }
}

template <int NM, int NT>
__device__ __forceinline__ void store_partial(float* part, const float (&acc)[NM][NT][4], int count, int lane) {
    const int g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n * 8 >= count) break;
            float* p = part + (m * NT * 8 + n * 8 + 2 * q) * kPartPitch + g;
            p[0] = acc[m][n][0];
            p[kPartPitch] = acc[m][n][1];
            p[8] = acc[m][n][2];
            p[kPartPitch + 8] = acc[m][n][3];
        }
}

}  // namespace swb
