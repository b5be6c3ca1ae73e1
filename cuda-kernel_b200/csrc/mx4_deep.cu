// The product of a four-bit matrix with many 16-bit tokens on the tensor cores.
//
// Splitting tokens into pieces (wide.cuh) costs conversions for every 128 rows of W, which bound
// that kernel from a few dozen tokens on (113 us for 512 tokens by 5632 x 2048). Here the
// tokens go to tcgen05.mma kind::f16 as they are, 128 on the M side, and the codes of N rows
// of W are decoded into a 16-bit tile on the way:
//
//   bf16   code times scale is exact
//   fp16   code times 2^(scale - largest scale of the row + 13); the epilogue multiplies a row's
//          column by what is left. Exact for blocks whose scale is within 2^36 of the row's
//          largest; a smaller value is off by at most 6 2^-38 of that scale (fp16's subnormals
//          end there), 2^-37 of the largest value of a row that was rounded from 16 bits.
//
// 512 tokens by 5632 x 2048: 24.4 us, 480 TFLOP/s (22 with W in L2); one tile an SM, so that decoding
// its first stages and its epilogue overlap with nothing.
//
// Roles: copies (TMA: 64 values of the tokens a stage, 256 of W's packed rows), decoding
// warps in groups, stage about, products, eight epilogue warps. Where a CTA takes several tiles,
// two accumulators, so that a tile's epilogue runs beside the next tile's products.
#include <algorithm>
#include <cstring>

#include "host.h"
#include "project.h"
#include "wide.cuh"

namespace swb {

int mx4_deep_device_error(int clear, int* out) {
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

constexpr int kDeepM = 128, kDeepEpilogue = 8;  // rows; warps
constexpr int kDeepTurn = 32, kDeepPitch = kDeepTurn + 2;  // columns of the epilogue's tiles

template <int N>
struct DeepShape {
    // A stage's decoding is a chain of about a microsecond: groups of warps take stages of their own.
    static constexpr int kGroups = N == 192 ? 3 : 8, kGroupWarps = N == 192 ? 4 : 1, kDecoders = kGroups * kGroupWarps;
    static constexpr int kThreads = (kDeepEpilogue + kDecoders + 2) * 32;
    static constexpr int kStagesA = N == 192 ? 4 : 5, kStagesB = N == 192 ? 3 : 8, kRaw = N == 192 ? 2 : 4;
    static_assert(kGroups <= kStagesB, "groups do not overtake the ring");
    // 64 rows are taken while every CTA gets one tile at most (dispatch_deep).
    static constexpr bool kOneTile = N == 64;
    static constexpr int kAccs = kOneTile ? 1 : 2;
    // Tiles whose row factors are kept. Decoders that begin tile t have filled the ring with stages before
    // it, of which the products have finished all but the last kStagesB, tile t - 1 - kStagesB at least
    // (one stage a tile); those began when the epilogue had read two tiles before.
    static constexpr int kFactors = kOneTile ? 1 : kStagesB + 3;
    static constexpr int kStageA = kDeepM * 128, kStageB = N * 128, kRawStage = N * 128;
    static constexpr uint32_t kAtB = kStagesA * kStageA, kAtRaw = kAtB + kStagesB * kStageB;
    static constexpr uint32_t kAtTurn = kAtRaw + kRaw * kRawStage;
    static constexpr uint32_t kAtFactors = kAtTurn + kDeepEpilogue * 32 * kDeepPitch * 4;
    static constexpr size_t kSmem = kAtFactors + (kFactors + 1) * N * 4 + 1024;  // factors, and the current tile's largest scales
    static constexpr int kColumns = N == 192 ? 512 : 64;
    static_assert(kSmem + 1024 <= kSmemPerCtaMax && kAccs * N <= kColumns, "fits");
};

// The factor of a block in fp16: 2^(scale - top + 13), NaN for 255.
__device__ __forceinline__ uint32_t deep_factor_f16(uint32_t scale, uint32_t top) {
    const int e = int(scale) - int(top) + 13;
    uint32_t h = e >= -14 ? uint32_t(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
    if (scale == 255u) h = 0x7E00u;
    return h | h << 16;
}

// Sixteen bytes of codes -> 32 values as 16-bit words in order, times the block's scale.
template <typename T>
__device__ __forceinline__ void deep_decode(const uint4& codes, uint32_t scale, uint32_t top, uint32_t (&w)[16]) {
    const uint32_t c[4] = {codes.x, codes.y, codes.z, codes.w};
    if constexpr (std::is_same<T, __half>::value) {
        const uint32_t f = deep_factor_f16(scale, top);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t p[4];
            mx_decode_f16(c[i], p);
#pragma unroll
            for (int j = 0; j < 4; ++j) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(w[4 * i + j]) : "r"(p[j]), "r"(f));
        }
    } else {
        uint32_t b = scale << 7;  // 2^(scale - 127) in bf16
        if (scale == 0u) b = 0x0040u;
        if (scale == 255u) b = 0x7FC0u;
        b |= b << 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t p[4];
            mx_decode_bf16(c[i], p);
#pragma unroll
            for (int j = 0; j < 4; ++j) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(p[j]) : "r"(p[j]), "r"(b));
            w[4 * i] = __byte_perm(p[0], p[1], 0x5410);
            w[4 * i + 1] = __byte_perm(p[2], p[3], 0x5410);
            w[4 * i + 2] = __byte_perm(p[0], p[1], 0x7632);
            w[4 * i + 3] = __byte_perm(p[2], p[3], 0x7632);
        }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(DeepShape<N>::kThreads, 1)
    project_deep_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                        const ProjectParams P, int tiles_x, int stages) {
    using S = DeepShape<N>;
    constexpr int kDeepDecoders = S::kDecoders;
    extern __shared__ unsigned char raw_smem[];
    __shared__ uint64_t a_full[S::kStagesA], a_empty[S::kStagesA], b_full[S::kStagesB], b_empty[S::kStagesB];
    __shared__ uint64_t raw_full[S::kRaw], raw_empty[S::kRaw], acc_full[S::kAccs], acc_empty[S::kAccs];
    __shared__ uint32_t s_tmem;
    const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStagesA; ++i) mbar_init(smem_u32(a_full + i), 1), mbar_init(smem_u32(a_empty + i), 1);
        for (int i = 0; i < S::kStagesB; ++i) mbar_init(smem_u32(b_full + i), S::kGroupWarps), mbar_init(smem_u32(b_empty + i), 1);
        for (int i = 0; i < S::kRaw; ++i) mbar_init(smem_u32(raw_full + i), 1), mbar_init(smem_u32(raw_empty + i), 4 * S::kGroupWarps);
        for (int i = 0; i < S::kAccs; ++i) mbar_init(smem_u32(acc_full + i), 1), mbar_init(smem_u32(acc_empty + i), kDeepEpilogue);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), S::kColumns);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    const int blocks = int(mx_blocks(P.cols));
    float* factors = reinterpret_cast<float*>(raw_smem + (base - smem_u32(raw_smem)) + S::kAtFactors);

    if (warp == kDeepEpilogue + kDeepDecoders) {
        // ---------------------------------------------------- copies
        if (elect_one()) {
            int a = 0, r = 0;
            uint32_t pa = 0, pr = 0;
            int64_t na = 0, nr = 0;
            bool ok = true;
            for (int64_t tile = blockIdx.x; tile < P.items && ok; tile += gridDim.x) {
                const int x0 = int(tile % tiles_x) * kDeepM, w0 = int(tile / tiles_x) * N;
                for (int k = 0; k < stages && ok; ++k) {
                    if (k % 4 == 0) {
                        ok = nr < S::kRaw || mbar_wait(smem_u32(raw_empty + r), pr ^ 1u);
                        if (!ok) break;
                        mbar_arrive_expect_tx(smem_u32(raw_full + r), S::kRawStage);
                        tma_load_2d(base + S::kAtRaw + r * S::kRawStage, &map_w, k / 4 * 32, w0, smem_u32(raw_full + r));
                        ++nr;
                        if (++r == S::kRaw) r = 0, pr ^= 1u;
                    }
                    ok = na < S::kStagesA || mbar_wait(smem_u32(a_empty + a), pa ^ 1u);
                    if (!ok) break;
                    mbar_arrive_expect_tx(smem_u32(a_full + a), S::kStageA);
                    tma_load_2d(base + a * S::kStageA, &map_x, k * 64, x0, smem_u32(a_full + a));
                    ++na;
                    if (++a == S::kStagesA) a = 0, pa ^= 1u;
                }
            }
            if (!ok) {  // nothing stays in flight into shared memory
                for (int64_t i = max(int64_t(0), na - S::kStagesA); i < na; ++i)
                    mbar_wait(smem_u32(a_full + i % S::kStagesA), uint32_t(i / S::kStagesA) & 1u);
                for (int64_t i = max(int64_t(0), nr - S::kRaw); i < nr; ++i)
                    mbar_wait(smem_u32(raw_full + i % S::kRaw), uint32_t(i / S::kRaw) & 1u);
            }
        }
    } else if (warp == kDeepEpilogue + kDeepDecoders + 1) {
        // ---------------------------------------------------- products
        if (elect_one()) {
            int a = 0, b = 0, acc = 0, done = 0;
            uint32_t pa = 0, pb = 0, pacc = 0;
            bool ok = true, have_a = false, have_b = false;
            for (int64_t tile = blockIdx.x; tile < P.items && ok; tile += gridDim.x, ++done) {
                ok = done < S::kAccs || mbar_wait(smem_u32(acc_empty + acc), pacc ^ 1u);
                for (int k = 0; k < stages && ok; ++k) {
                    ok = (have_a || mbar_wait(smem_u32(a_full + a), pa)) && (have_b || mbar_wait(smem_u32(b_full + b), pb));
                    if (!ok) break;
                    const int as = a, bs = b;
                    if (++a == S::kStagesA) a = 0, pa ^= 1u;
                    if (++b == S::kStagesB) b = 0, pb ^= 1u;
                    have_a = mbar_test(smem_u32(a_full + a), pa);
                    have_b = mbar_test(smem_u32(b_full + b), pb);
                    fence_after();
                    const uint64_t da = operand_desc(base + as * S::kStageA), db = operand_desc(base + S::kAtB + bs * S::kStageB);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_f16(tmem + acc * N, da + 2 * j, db + 2 * j, f16_desc<T>(kDeepM, N), k > 0 || j > 0);
                    mma_commit(smem_u32(a_empty + as));
                    mma_commit(smem_u32(b_empty + bs));
                    if (k == stages - 1) mma_commit(smem_u32(acc_full + acc));
                }
                if (++acc == S::kAccs) acc = 0, pacc ^= 1u;
            }
        }
    } else if (warp >= kDeepEpilogue) {
        // ---------------------------------------------------- decoders
        // Group g takes the stages g, g + kGroups, ... of the sequence, and nothing else: passing
        // over the others' stages one by one cost more than decoding its own.
        constexpr int kGroupThreads = S::kGroupWarps * 32, kAll = S::kDecoders * 32;
        constexpr int kTasks = N * 2 / kGroupThreads;  // blocks of a stage's 64 values that a thread decodes
        const int thread = threadIdx.x - kDeepEpilogue * 32, group = thread / kGroupThreads, t = thread % kGroupThreads;
        const int raws = (stages + 3) / 4;
        uint32_t* tops = reinterpret_cast<uint32_t*>(factors) + S::kFactors * N;
        int slot = 0, tiles = 0;
        bool ok = true;
        for (int64_t tile = blockIdx.x; tile < P.items; tile += gridDim.x, ++tiles) {
            const int64_t w0 = tile / tiles_x * N;
            // The groups begin a tile together: a group that went on past stages of others could come to a
            // raw stage two rounds ahead of what has landed, where the barrier's parity says that it has.
            // (Within a tile the ring of decoded stages holds them close enough.)
            named_barrier_sync(1, kAll);
            if (!ok) {  // a group that gave up still comes to the others' barriers
                if constexpr (std::is_same<T, __half>::value) named_barrier_sync(1, kAll);
                continue;
            }
            if constexpr (std::is_same<T, __half>::value) {  // the rows' largest scales; the last tile's are read
                for (int q = thread; q < N; q += kAll) {
                    uint32_t m = 0u;
                    if (w0 + q < P.rows) {
#pragma unroll 4
                        for (int i = 0; i < blocks; i += 16) {
                            const uint4 v = load_scales(P.s + (w0 + q) * blocks, i, blocks);
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) m = __vmaxu4(m, w[e] & ~__vcmpeq4(w[e], 0xFFFFFFFFu));
                        }
                    }
                    m = max(max(m & 255u, m >> 8 & 255u), max(m >> 16 & 255u, m >> 24));
                    tops[q] = m;
                    factors[slot * N + q] = mx_scale(m);
                }
                named_barrier_sync(1, kAll);
            }
            const unsigned char* row[kTasks];
            uint32_t top[kTasks], scale[kTasks];
#pragma unroll
            for (int u = 0; u < kTasks; ++u) {
                const int q = (t + kGroupThreads * u) % N;
                row[u] = w0 + q < P.rows ? P.s + (w0 + q) * blocks + (t + kGroupThreads * u) / N : nullptr;
                top[u] = std::is_same<T, __half>::value ? tops[q] : 0u;
            }
            auto load = [&](int k) {
#pragma unroll
                for (int u = 0; u < kTasks; ++u) {
                    const int byte = k * 2 + (t + kGroupThreads * u) / N;
                    scale[u] = row[u] && byte < blocks ? row[u][k * 2] : 0u;
                }
            };
            const uint32_t q0 = uint32_t(tiles) * uint32_t(stages);  // of the sequence
            int k = int((uint32_t(group) + uint32_t(S::kGroups) - q0 % S::kGroups) % S::kGroups);
            if (k < stages) load(k);
            for (; k < stages; k += S::kGroups) {
                const uint32_t q = q0 + uint32_t(k), b = q % S::kStagesB, use = q / S::kStagesB;
                const uint32_t rq = uint32_t(tiles) * uint32_t(raws) + uint32_t(k / 4), r = rq % S::kRaw;
                ok = mbar_wait_warp(smem_u32(raw_full + r), rq / S::kRaw & 1u) &&
                     (use == 0 || mbar_wait_warp(smem_u32(b_empty + b), (use & 1u) ^ 1u));
                if (!ok) break;
                const uint32_t from = base + S::kAtRaw + r * S::kRawStage, to = base + S::kAtB + b * S::kStageB;
                uint32_t now[kTasks];
#pragma unroll
                for (int u = 0; u < kTasks; ++u) now[u] = scale[u];
                if (k + S::kGroups < stages) load(k + S::kGroups);
#pragma unroll
                for (int u = 0; u < kTasks; ++u) {
                    const int row16 = (t + kGroupThreads * u) % N, block = (t + kGroupThreads * u) / N;
                    const uint4 codes = lds128(from + swizzled(row16, k % 4 * 2 + block));
                    uint32_t w[16];
                    deep_decode<T>(codes, now[u], top[u], w);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sts128(to + swizzled(row16, block * 4 + i), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(b_full + b));
                    // a raw stage is free after its four; the last one's missing stages count here
                    for (int n = k == stages - 1 ? 4 - k % 4 : 1; n > 0; --n) mbar_arrive(smem_u32(raw_empty + r));
                }
            }
            if (++slot == S::kFactors) slot = 0;
        }
    } else {
        // ---------------------------------------------------- epilogue
        const int quarter = warp % 4, share = warp / 4;  // this warp takes every other group of columns
        const uint32_t quadrant = uint32_t(quarter * 32) << 16;
        float* turn = reinterpret_cast<float*>(raw_smem + (base - smem_u32(raw_smem)) + S::kAtTurn) + warp * 32 * kDeepPitch;
        int acc = 0, slot = 0;
        uint32_t pacc = 0;
        for (int64_t tile = blockIdx.x; tile < P.items; tile += gridDim.x) {
            const int64_t w0 = tile / tiles_x * N, token0 = tile % tiles_x * kDeepM + quarter * 32 + lane / 16;
            const int tokens = int(min(int64_t(32), P.tokens - token0));
            if (!mbar_wait_warp(smem_u32(acc_full + acc), pacc)) break;
            fence_after();
#pragma unroll 1
            for (int c = share * kDeepTurn; c < N; c += 2 * kDeepTurn) {
                const int64_t row = w0 + c + lane % 16 * 2;  // this lane's two columns
                const bool have0 = row < P.rows, have1 = row + 1 < P.rows;
                uint32_t v[32];
                __syncwarp();  // the last columns are read
                tmem_load32(tmem + quadrant + acc * N + c, v);
                tmem_load_wait();
#pragma unroll
                for (int j = 0; j < 32; j += 2)
                    *reinterpret_cast<float2*>(turn + lane * kDeepPitch + j) =
                        make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                __syncwarp();
                float2 bias = make_float2(0.f, 0.f), f = make_float2(1.f, 1.f);
                if constexpr (std::is_same<T, __half>::value) {
                    f.x = factors[slot * N + c + lane % 16 * 2];
                    f.y = factors[slot * N + c + lane % 16 * 2 + 1];
                }
                if (P.bias) {
                    if (have0) bias.x = Num<T>::to_float(static_cast<const T*>(P.bias)[row]);
                    if (have1) bias.y = Num<T>::to_float(static_cast<const T*>(P.bias)[row + 1]);
                }
#pragma unroll 4
                for (int u = 0; u < 16; ++u) {
                    if (2 * u >= tokens) break;
                    const int64_t at = (token0 + 2 * u) * P.rows + row;
                    float2 o = *reinterpret_cast<const float2*>(turn + (2 * u + lane / 16) * kDeepPitch + lane % 16 * 2);
                    if constexpr (std::is_same<T, __half>::value) {
                        o.x = o.x * 0x1p-13f * f.x;
                        o.y = o.y * 0x1p-13f * f.y;
                    }
                    o.x += bias.x;
                    o.y += bias.y;
                    if (P.residual) {
                        const T* p = static_cast<const T*>(P.residual) + at;
                        if (have0) o.x += Num<T>::to_float(p[0]);
                        if (have1) o.y += Num<T>::to_float(p[1]);
                    }
                    if (P.half_out) {
                        T two[2] = {Num<T>::from_float(o.x), Num<T>::from_float(o.y)};
                        T* p = static_cast<T*>(P.out) + at;
                        if (have1 && (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
                            *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(two);
                        } else {
                            if (have0) p[0] = two[0];
                            if (have1) p[1] = two[1];
                        }
                    } else {
                        float* p = static_cast<float*>(P.out) + at;
                        if (have0) p[0] = o.x;
                        if (have1) p[1] = o.y;
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(acc_empty + acc));
            if (++acc == S::kAccs) acc = 0, pacc ^= 1u;
            if (++slot == S::kFactors) slot = 0;
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        tmem_free(tmem, S::kColumns);
    }
}

template <typename T, int N>
int launch_deep(ProjectParams P, cudaStream_t stream) {
    using S = DeepShape<N>;
    static std::atomic<uint64_t> smem_set{0};
    const int sms = sm_count();
    if (sms <= 0) return check_launch();
    auto kernel = project_deep_kernel<T, N>;
    if (int rc = allow_smem(kernel, smem_set, S::kSmem)) return rc;
    CUtensorMap map_x, map_w;
    if (int rc = make_typed_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, P.x, P.cols, P.tokens, P.x_pitch * 2, 64, kDeepM)) return rc;
    if (int rc = make_map(&map_w, P.w, P.rows, mx_blocks(P.cols) * kMxBlockBytes, 128, N)) return rc;
    const int tiles_x = int((P.tokens + kDeepM - 1) / kDeepM), stages = (P.cols + 63) / 64;
    P.tiles = (P.rows + N - 1) / N;
    P.items = int64_t(P.tiles) * tiles_x;
    return launch_ex(kernel, unsigned(std::min<int64_t>(P.items, sms)), S::kThreads, S::kSmem, stream, false, map_x, map_w, P,
                     tiles_x, stages);
}

template <typename T>
int dispatch_deep(const ProjectParams& P, cudaStream_t stream) {
    // 64 rows a tile while every SM gets one at most, else 192: 44.7 us against 51.2 with 224 tiles of 64
    // (64 tokens by 14336 x 4096), 21.8 against 24.6 with 264 (384 tokens by 5632 x 2048).
    const int64_t tiles = int64_t((P.rows + 63) / 64) * ((P.tokens + kDeepM - 1) / kDeepM);
    if (tiles > sm_count()) return launch_deep<T, 192>(P, stream);
    return launch_deep<T, 64>(P, stream);
}

}  // namespace

// Pieces up to 32 tokens, decoding W from 33 on. Both ways, us, pieces first:
//                        24 tokens      32             33             64             128
//   14336 x 4096  fp16   33.0  45.7     40.2  46.4     66.5  46.4     77.8  46.5    150.4  47.2
//                 bf16   30.3  43.0     37.3  44.0     49.7  43.7     55.1  44.1    107.3  44.2
//   5632 x 2048   fp16   14.4  19.4     17.0  14.8     20.9  15.0     24.5  14.8     42.0  15.1
//                 bf16   13.7  17.7     16.1  14.4     17.6  14.7     19.8  14.5     31.6  14.7
//   4096 x 14336  fp16   29.1  80.9     35.0  81.2     58.2  81.2     67.6  81.6    129.7  81.5
//                 bf16   27.3  79.9     33.2  80.3     44.0  80.2     48.4  80.4     88.4  80.3
// The border suits the first two; long rows in few tiles (64 CTAs of 224 stages, K is not split) would
// gain from pieces to about 64 tokens.
bool project_deep_takes(const ProjectParams& P) { return P.tokens > 32 && P.x_aligned; }

int project_deep(int type, const ProjectParams& P, cudaStream_t stream) {
    return type == SWB_F16 ? dispatch_deep<__half>(P, stream) : dispatch_deep<__nv_bfloat16>(P, stream);
}

}  // namespace swb
