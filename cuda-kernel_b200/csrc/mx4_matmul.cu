// Product of two MXFP4 matrices on the fifth-generation tensor cores
// (declaration: include/swiglu_b200.h).
//
//   out[t][r] = sum_k X[t][k] W[r][k] (+ bias[r]) (+ residual[t][r])
//
// tcgen05.mma kind::mxf4 multiplies 64 four-bit values a step and applies the two
// blocks' power-of-two scales itself, so codes go from global memory to the tensor
// core untouched: TMA brings 256 values (128 bytes) of every row of both tiles into a
// 128-byte swizzled stage; four warps bring the scale bytes of the same rows into
// the 32 x 16-byte blocks that tcgen05.cp spreads over TMEM; a thread each issues the
// copies and the products; eight warps drain the accumulators.
//
// Long batches (tokens on the M side, 128 of them by N = 192 rows of W): two
// accumulators of 192 columns and the stages' scales fill TMEM. Without sharing a
// tile between CTAs the bytes that L2 hands out bound this kernel (0.5 B per value at
// 4x the rate of 16-bit products), hence the large tile.
// Few tokens (W on the M side, N = 16 to 128 tokens): bound by the bytes of W. The
// CTAs of a cluster split K, so that every SM streams, and add their parts through
// each other's shared memory in a fixed order.
// 4096 tokens by 14336 x 4096 with a residual: 169 us, 2.85 PFLOP/s, a few launches at a time; 195 us,
// 2.5, launched without a pause (the power cap lowers the clocks). 16 tokens: 13 us for 31 MB, 11 with W in L2.
#include <algorithm>
#include <cstring>

#include "device.cuh"
#include "host.h"
#include "stream.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace swb {

int mx4_matmul_device_error(int clear, int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_device_error, sizeof v);
    if (e == cudaSuccess && clear) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof zero);
    }
    if (e != cudaSuccess) return fail(SWB_E_CUDA, cudaGetErrorString(e));
    *out = v;
    return SWB_OK;
}

namespace {

constexpr int kMmaM = 128;
constexpr int kRowBytes = 128;     // of a row in a stage: 256 values, 8 scales
constexpr int kWindow = 16;        // scale bytes of a row that a thread loads at once: two stages
constexpr int kEpilogueWarps = 8, kScaleWarps = 4;  // epilogue: two warps a TMEM quadrant
constexpr int kTurnColumns = 32, kTurnPitch = kTurnColumns + 2;  // floats of a row in the epilogue
constexpr int kThreads = (kEpilogueWarps + kScaleWarps + 2) * 32;

struct MatmulParams {
    const unsigned char* sa;  // scales of the M side, [rows_a, blocks]
    const unsigned char* sb;  // of the N side
    const void* bias;
    const void* residual;
    void* out;
    int64_t rows_a, rows_b;   // rows of the M and N side
    int64_t tokens, rows;     // of the output
    int tiles_a, tiles_b;     // M tiles, N tiles
    int64_t tiles;
    int blocks;               // scales of a row
    int stages_k;             // stages that cover K
    int splits;               // CTAs of a cluster that share a tile's K
};

template <int N, bool TOKENS_M>
struct MatmulShape {
    static constexpr int kStages = TOKENS_M || N > 32 ? 4 : 5;
    static constexpr int kPerSm = TOKENS_M || N > 64 ? 1 : 2;
    static constexpr int kBytesA = kMmaM * kRowBytes, kBytesB = N * kRowBytes;
    static constexpr int kBlocksB = (N + kMmaM - 1) / kMmaM;   // 128-row blocks of scales of the N side
    static constexpr int kScales = 2 * (1 + kBlocksB) * kScaleBlock;
    static constexpr int kStage = kBytesA + kBytesB + kScales;
    static_assert(!TOKENS_M || N % kTurnColumns == 0, "whole turns");
    static_assert(kStage % 1024 == 0, "stages keep the swizzle's alignment");
    static constexpr int kAccs = TOKENS_M ? 2 : 1;             // accumulators of N columns
    static constexpr int kScaleColumns = 2 * (1 + kBlocksB) * 4;
    static constexpr int kUsed = kAccs * N + kStages * kScaleColumns;
    static constexpr int kColumns = kUsed <= 32 ? 32 : kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static_assert(kUsed <= 512, "TMEM columns");
    static constexpr int kPartPitch = kMmaM + 1;               // floats of a token's column in the exchange
    static constexpr int kExchange = TOKENS_M ? 0 : N * kPartPitch * 4;
    static constexpr int kTurn = TOKENS_M ? kEpilogueWarps * 32 * kTurnPitch * 4 : 0;  // the epilogue's tiles
    static constexpr size_t kSmem = size_t(kStages) * kStage + kTurn + 1024;  // the exchange reuses the stages
    static_assert(kExchange <= kStages * kStage, "exchange fits the stages");
    static_assert(kColumns * kPerSm <= 512, "CTAs of an SM share TMEM");
    static_assert((kSmem + 2048) * kPerSm <= kSmemPerSm, "CTAs of an SM share its shared memory");
};

template <typename T>
__device__ __forceinline__ float load_value(const void* p, int64_t i) {
    return Num<T>::to_float(static_cast<const T*>(p)[i]);
}

template <typename T, int N, bool TOKENS_M>
__global__ void __launch_bounds__(kThreads, MatmulShape<N, TOKENS_M>::kPerSm)
    matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const MatmulParams P) {
    using S = MatmulShape<N, TOKENS_M>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::kStages], scaled[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // this CTA's tiles [first, last) by `step`, and its share of K
    const int rank = P.splits > 1 ? int(blockIdx.x % P.splits) : 0;
    const int64_t step = gridDim.x / P.splits, first = blockIdx.x / P.splits;
    const int k0 = int(int64_t(P.stages_k) * rank / P.splits), k1 = int(int64_t(P.stages_k) * (rank + 1) / P.splits);

    if (threadIdx.x == 0) {
        s_failed = 0;
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(smem_u32(full + i), 1);
            mbar_init(smem_u32(scaled + i), kScaleWarps * 32);
            mbar_init(smem_u32(empty + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(acc_full + i), 1);
            mbar_init(smem_u32(acc_empty + i), kEpilogueWarps * 32);
        }
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), S::kColumns);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t scale_columns = tmem + S::kAccs * N;

    if (warp == kEpilogueWarps + kScaleWarps) {
        // ------------------------------------------------------- codes, by TMA
        if (elect_one()) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int64_t tile = first; tile < P.tiles && ok; tile += step) {
                const int a = int(tile % P.tiles_a), b = int(tile / P.tiles_a);
                for (int k = k0; k < k1; ++k) {
                    if (issued >= S::kStages && !mbar_wait(smem_u32(empty + s), ph ^ 1u)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(full + s), at = base + s * S::kStage;
                    mbar_arrive_expect_tx(bar, S::kBytesA + S::kBytesB);
                    tma_load_2d(at, &map_a, k * (kRowBytes / 4), a * kMmaM, bar);
                    tma_load_2d(at + S::kBytesA, &map_b, k * (kRowBytes / 4), b * N, bar);
                    ++issued;
                    if (++s == S::kStages) s = 0, ph ^= 1u;
                }
            }
            // nothing stays in flight into shared memory when the CTA leaves early
            if (!ok) {
                for (int i = 0; i < S::kStages && i < issued; ++i) {
                    const int idx = issued - 1 - i;
                    mbar_wait(smem_u32(full + idx % S::kStages), uint32_t(idx / S::kStages) & 1u);
                }
                s_failed = 1;
            }
        }
    } else if (warp == kEpilogueWarps + kScaleWarps + 1) {
        // ------------------------------------------------------- products
        if (elect_one()) {
            int s = 0, acc = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            int64_t done = 0;
            for (int64_t tile = first; tile < P.tiles && ok; tile += step, ++done) {
                for (int k = k0; k < k1 && ok; ++k) {
                    ok = mbar_wait(smem_u32(full + s), ph) && mbar_wait(smem_u32(scaled + s), ph);
                    if (!ok) break;
                    fence_after();
                    const uint32_t at = base + s * S::kStage, sc = at + S::kBytesA + S::kBytesB;
                    const uint32_t col = scale_columns + s * S::kScaleColumns;
#pragma unroll
                    for (int i = 0; i < 2 * (1 + S::kBlocksB); ++i)
                        scale_copy(col + 4 * i, scale_desc(sc + i * kScaleBlock));
                    // the accumulator's last tile has been read
                    if (k == k0 && done >= S::kAccs) {
                        ok = mbar_wait(smem_u32(acc_empty + acc), aph ^ 1u);
                        if (!ok) break;
                        fence_after();
                    }
                    const uint64_t da = operand_desc(at), db = operand_desc(at + S::kBytesA);
#pragma unroll
                    for (int i = 0; i < 4; ++i)  // 64 values a step; scales: blocks of 128 values, then rows
                        mma_mxf4(tmem + acc * N, da + 2 * i, db + 2 * i, mxf4_desc(kMmaM, N, (i & 1) * 2),
                                 col + (i >> 1) * 4, col + (2 + (i >> 1) * S::kBlocksB) * 4, k > k0 || i > 0);
                    mma_commit(smem_u32(empty + s));
                    if (k == k1 - 1) mma_commit(smem_u32(acc_full + acc));
                    if (++s == S::kStages) s = 0, ph ^= 1u;
                }
                if (++acc == S::kAccs) {
                    acc = 0;
                    aph ^= 1u;
                }
            }
            if (!ok) s_failed = 1;
        }
    } else if (warp >= kEpilogueWarps) {
        // ------------------------------------------------------- scales
        constexpr int kRows = kMmaM + N, kPer = (kRows + 127) / 128;
        // A warp's lanes take rows 8 apart in four quarters of 128: their words lie side by side.
        const int lt = threadIdx.x - kEpilogueWarps * 32, t = lt / 32 * 8 + (lt & 7) + (lt >> 3 & 3) * 32;
        int s = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int64_t tile = first; tile < P.tiles && ok; tile += step) {
            const int64_t a0 = tile % P.tiles_a * kMmaM, b0 = tile / P.tiles_a * N;
            const unsigned char* row[kPer];
            uint32_t dst[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int r = t + 128 * i;
                row[i] = nullptr;
                const bool in_a = r < kMmaM;
                const int q = in_a ? r : r - kMmaM, in = q & 127;
                const int64_t global = in_a ? a0 + q : b0 + q;
                if (r < kRows && global < (in_a ? P.rows_a : P.rows_b))
                    row[i] = (in_a ? P.sa : P.sb) + global * P.blocks;
                // blocks of the M side: [128 values][128 rows], then the N side's
                dst[i] = (in_a ? q >> 7 : 2 + (q >> 7)) * kScaleBlock + (in & 31) * 16 + (in >> 5) * 4;
            }
            // two windows ahead: scales of long rows come from L2 or DRAM
            uint4 window[3][kPer];
            auto load = [&](int w, int k) {  // the window that holds stage k's scales
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    window[w][i] = row[i] && k < k1 ? load_scales(row[i], k * 8 & ~(kWindow - 1), P.blocks) : make_uint4(0u, 0u, 0u, 0u);
            };
            load(0, k0);
            load(1, (k0 | 1) + 1);
            load(2, (k0 | 1) + 3);
            for (int k = k0; k < k1; ++k) {
                if (k > k0 && (k & 1) == 0) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) window[0][i] = window[1][i], window[1][i] = window[2][i];
                    load(2, k + 4);
                }
                if (issued >= S::kStages && !mbar_wait(smem_u32(empty + s), ph ^ 1u)) {
                    ok = false;
                    break;
                }
                const uint32_t sc = base + s * S::kStage + S::kBytesA + S::kBytesB;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const int r = t + 128 * i;
                    if (r < kRows) {
                        const uint32_t next_block = (r < kMmaM ? 1 : S::kBlocksB) * kScaleBlock;
                        sts32(sc + dst[i], k & 1 ? window[0][i].z : window[0][i].x);
                        sts32(sc + dst[i] + next_block, k & 1 ? window[0][i].w : window[0][i].y);
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(smem_u32(scaled + s));
                ++issued;
                if (++s == S::kStages) s = 0, ph ^= 1u;
            }
        }
        if (!ok) s_failed = 1;
    } else {
        // ------------------------------------------------------- epilogue
        int acc = 0;
        uint32_t ph = 0;
        bool ok = true;
        const int quarter = warp % 4, share = warp / 4;  // this warp takes every other group of columns
        const uint32_t quadrant = uint32_t(quarter * 32) << 16;
        for (int64_t tile = first; tile < P.tiles && ok; tile += step) {
            const int64_t a0 = tile % P.tiles_a * kMmaM, b0 = tile / P.tiles_a * N;
            // The residual's values for 32 columns of this warp's tokens (a lane: two columns of every
            // other token), on their way before the accumulator is waited for, the next
            // ones before these are written.
            uint32_t residual[16], ahead[16];
            const int64_t token0 = a0 + quarter * 32 + lane / 16;
            const int tokens = int(min(int64_t(32), P.tokens - token0));
            auto load_residual = [&](int c) {
                if (!TOKENS_M || !P.residual) return;
                const int64_t row = b0 + c + lane % 16 * 2;
                const T* r = static_cast<const T*>(P.residual) + token0 * P.rows + row;
                const bool have0 = row < P.rows, have1 = row + 1 < P.rows;
#pragma unroll
                for (int u = 0; u < 16; ++u, r += 2 * P.rows) {
                    ahead[u] = 0u;
                    if (2 * u < tokens && have0) {
                        if (have1 && (reinterpret_cast<uintptr_t>(r) & 3) == 0) {
                            ahead[u] = *reinterpret_cast<const uint32_t*>(r);
                        } else {
                            ahead[u] = *reinterpret_cast<const unsigned short*>(r);
                            if (have1) ahead[u] |= uint32_t(reinterpret_cast<const unsigned short*>(r)[1]) << 16;
                        }
                    }
                }
            };
            load_residual(share * kTurnColumns);
            ok = mbar_wait_warp(smem_u32(acc_full + acc), ph);
            if (!ok) break;
            fence_after();
            const int in_tile = quarter * 32 + lane;
            if constexpr (TOKENS_M) {
                // A lane holds a token's columns; through shared memory, so that half a warp writes 32
                // neighbouring values of one token at a time (a lane storing its own token's 16
                // bytes took 40 % of the kernel, single values of ragged rows 80 %).
                float* turn = reinterpret_cast<float*>(raw + (base - smem_u32(raw)) + S::kStages * S::kStage) + warp * 32 * kTurnPitch;
#pragma unroll 1
                for (int c = share * kTurnColumns; c < N; c += 2 * kTurnColumns) {
                    if (P.residual) {
#pragma unroll
                        for (int u = 0; u < 16; ++u) residual[u] = ahead[u];
                        if (c + 2 * kTurnColumns < N) load_residual(c + 2 * kTurnColumns);
                    }
                    uint32_t v[32];
                    __syncwarp();  // the last columns are read
                    tmem_load32(tmem + quadrant + acc * N + c, v);
                    tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 32; j += 2)
                        *reinterpret_cast<float2*>(turn + lane * kTurnPitch + j) =
                            make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                    __syncwarp();
                    const int64_t row = b0 + c + lane % 16 * 2;  // this lane's two columns
                    const bool have0 = row < P.rows, have1 = row + 1 < P.rows;
                    float2 bias = make_float2(0.f, 0.f);
                    if (P.bias) {
                        if (have0) bias.x = load_value<T>(P.bias, row);
                        if (have1) bias.y = load_value<T>(P.bias, row + 1);
                    }
                    T* o = static_cast<T*>(P.out) + token0 * P.rows + row;
                    const float* from = turn + lane / 16 * kTurnPitch + lane % 16 * 2;
#pragma unroll
                    for (int u = 0; u < 16; ++u, o += 2 * P.rows) {
                        if (2 * u >= tokens) break;
                        float2 f = *reinterpret_cast<const float2*>(from + 2 * u * kTurnPitch);
                        T two[2];
                        f.x += bias.x;
                        f.y += bias.y;
                        if (P.residual) {
                            *reinterpret_cast<uint32_t*>(two) = residual[u];
                            f.x += Num<T>::to_float(two[0]);
                            f.y += Num<T>::to_float(two[1]);
                        }
                        two[0] = Num<T>::from_float(f.x);
                        two[1] = Num<T>::from_float(f.y);
                        if (have1 && (reinterpret_cast<uintptr_t>(o) & 3) == 0) {
                            *reinterpret_cast<uint32_t*>(o) = *reinterpret_cast<const uint32_t*>(two);
                        } else {
                            if (have0) o[0] = two[0];
                            if (have1) o[1] = two[1];
                        }
                    }
                }
            } else {
                // a column is a token, a lane a row of W: to shared memory, [token][row]
                float* part = reinterpret_cast<float*>(raw + (base - smem_u32(raw)));
#pragma unroll 1
                for (int c = share * 16; c < N; c += 32) {
                    uint32_t v[16];
                    __syncwarp();
                    tmem_load16(tmem + quadrant + acc * N + c, v);
                    tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(c + j) * S::kPartPitch + in_tile] = __uint_as_float(v[j]);
                }
            }
            fence_before();
            mbar_arrive(smem_u32(acc_empty + acc));
            if (++acc == S::kAccs) {
                acc = 0;
                ph ^= 1u;
            }
        }
        if (!ok) s_failed = 1;
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        tmem_free(tmem, S::kColumns);
    }
    if constexpr (!TOKENS_M) {
        // The cluster's parts, added in rank order; each CTA takes its share of the tile's outputs.
        // A CTA that failed writes nothing, and its peers keep what they could add.
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        const int64_t w0 = first % P.tiles_a * kMmaM, t0 = first / P.tiles_a * N;
        const int count = int(min(int64_t(N), P.tokens - t0)) * kMmaM;
        if (!s_failed) {
            for (int i = rank * kThreads + threadIdx.x; i < count; i += P.splits * kThreads) {
                const int t = i / kMmaM, r = i % kMmaM;
                if (w0 + r >= P.rows) continue;
                float v = 0.f;
                for (int j = 0; j < P.splits; ++j) {
                    uint32_t remote;
                    float f;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(base + (t * S::kPartPitch + r) * 4), "r"(j));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(remote) : "memory");
                    v += f;
                }
                const int64_t row = w0 + r, at = (t0 + t) * P.rows + row;
                if (P.bias) v += load_value<T>(P.bias, row);
                if (P.residual) v += load_value<T>(P.residual, at);
                static_cast<T*>(P.out)[at] = Num<T>::from_float(v);
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    }
}

// ------------------------------------------------------------ host
struct Side {
    const void* codes;
    const unsigned char* scales;
    int64_t rows;
};

template <typename T, int N, bool TOKENS_M>
int launch_matmul(const Side& x, const Side& w, MatmulParams P, cudaStream_t stream) {
    using S = MatmulShape<N, TOKENS_M>;
    static std::atomic<uint64_t> smem_set{0};
    const int sms = sm_count();
    if (sms <= 0) return check_launch();
    auto kernel = matmul_kernel<T, N, TOKENS_M>;
    if (int rc = allow_smem(kernel, smem_set, S::kSmem)) return rc;
    const Side& a = TOKENS_M ? x : w;
    const Side& b = TOKENS_M ? w : x;
    CUtensorMap map_a, map_b;
    if (int rc = make_map(&map_a, a.codes, a.rows, int64_t(P.blocks) * kMxBlockBytes, kRowBytes, kMmaM)) return rc;
    if (int rc = make_map(&map_b, b.codes, b.rows, int64_t(P.blocks) * kMxBlockBytes, kRowBytes, N)) return rc;
    P.sa = a.scales;
    P.sb = b.scales;
    P.rows_a = a.rows;
    P.rows_b = b.rows;
    P.tiles_a = int((a.rows + kMmaM - 1) / kMmaM);
    P.tiles_b = int((b.rows + N - 1) / N);
    P.tiles = int64_t(P.tiles_a) * P.tiles_b;
    P.stages_k = (P.blocks + 7) / 8;
    P.splits = 1;
    int64_t grid = std::min<int64_t>(P.tiles, sms);
    if (!TOKENS_M) {
        // every SM streams: split K until the CTAs fill the GPU, down to two stages each
        while (P.splits < 8 && P.tiles * P.splits * 2 <= int64_t(sms) * S::kPerSm && P.stages_k / (P.splits * 2) >= 2)
            P.splits *= 2;
        grid = P.tiles * P.splits;
        if (grid > 0x7FFFFFFF) return fail(SWB_E_SHAPE);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(P.splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, P);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(SWB_E_CUDA, cudaGetErrorString(e));
    }
    return SWB_OK;
}

template <typename T>
int dispatch_matmul(const Side& x, const Side& w, const MatmulParams& P, cudaStream_t stream) {
    if (P.tokens <= 16) return launch_matmul<T, 16, false>(x, w, P, stream);
    if (P.tokens <= 32) return launch_matmul<T, 32, false>(x, w, P, stream);
    if (P.tokens <= 64) return launch_matmul<T, 64, false>(x, w, P, stream);
    // 65 to 128 tokens: a tile of tokens by 192 rows where that gives half the SMs one (W in L2, us, fp16;
    // bf16 within 0.4: 14336 x 4096, 65 tokens 16.8 against 17.4, 128 17.6 against 21.5), else W on the M side
    // (4096 x 14336, 65 tokens 15.3 against 37.5, 128 17.7 against 39.1; 5632 x 2048, 65 tokens 10.8 against
    // 11.3, but 128 13.3 against 11.3). 64 tokens by 14336 x 4096: W's side 16.3 against 16.7.
    if (P.tokens <= 128 && (P.rows + 191) / 192 * 2 < sm_count()) return launch_matmul<T, 128, false>(x, w, P, stream);
    return launch_matmul<T, 192, true>(x, w, P, stream);
}

}  // namespace
}  // namespace swb

using namespace swb;

extern "C" int swb_mx4_matmul(int type, const void* x_codes, const void* x_scales, const void* w_codes,
                              const void* w_scales, const void* bias, const void* residual, void* out, int64_t tokens,
                              int64_t rows, int64_t cols, unsigned flags, void* stream) {
    if (type != SWB_F16 && type != SWB_BF16) return fail(SWB_E_TYPE);
    if (flags & ~SWB_RESIDUAL) return fail(SWB_E_INPUT, "unknown flags");
    if (tokens < 0 || tokens > SWB_MX4_MAX_TOKENS || rows <= 0 || cols <= 0 || rows > SWB_MX4_MAX_DIM ||
        cols > SWB_MX4_MAX_DIM)
        return fail(SWB_E_SHAPE);
    if (tokens == 0) return SWB_OK;
    if (!x_codes || !x_scales || !w_codes || !w_scales) return fail(SWB_E_INPUT);
    if (!out) return fail(SWB_E_HALF_OUTPUT);
    if ((flags & SWB_RESIDUAL) && !residual) return fail(SWB_E_RESIDUAL);
    if (!aligned(16, x_codes, w_codes)) return fail(SWB_E_ALIGNMENT, "codes must be 16-byte aligned");
    if (!aligned(2, out, bias, (flags & SWB_RESIDUAL) ? residual : nullptr))
        return fail(SWB_E_ALIGNMENT, "values off their type's size");
    const int64_t blocks = mx_blocks(cols);
    const size_t out_bytes = size_t(tokens) * rows * 2;
    if (overlaps(out, out_bytes, x_codes, size_t(tokens) * blocks * kMxBlockBytes) ||
        overlaps(out, out_bytes, x_scales, size_t(tokens) * blocks) ||
        overlaps(out, out_bytes, w_codes, size_t(rows) * blocks * kMxBlockBytes) ||
        overlaps(out, out_bytes, w_scales, size_t(rows) * blocks) ||
        (bias && overlaps(out, out_bytes, bias, size_t(rows) * 2)))
        return fail(SWB_E_OVERLAP_INPUT);
    // the residual may be the output itself: each value is read by the thread that writes it
    if ((flags & SWB_RESIDUAL) && residual != out && overlaps(out, out_bytes, residual, out_bytes))
        return fail(SWB_E_OVERLAP_INPUT);
    MatmulParams P;
    std::memset(&P, 0, sizeof P);
    P.bias = bias;
    P.residual = (flags & SWB_RESIDUAL) ? residual : nullptr;
    P.out = out;
    P.tokens = tokens;
    P.rows = rows;
    P.blocks = int(blocks);
    const Side x{x_codes, static_cast<const unsigned char*>(x_scales), tokens};
    const Side w{w_codes, static_cast<const unsigned char*>(w_scales), rows};
    auto s = static_cast<cudaStream_t>(stream);
    return type == SWB_F16 ? dispatch_matmul<__half>(x, w, P, s) : dispatch_matmul<__nv_bfloat16>(x, w, P, s);
}
