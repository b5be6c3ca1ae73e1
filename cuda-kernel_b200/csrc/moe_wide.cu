// The mixture-of-experts layer on the tensor cores (wide.cuh), for more tokens than the
// register path of moe.cuh likes: two kernels, both bound by the bytes of the weights.
//
//   gate   router and selection as in moe.cuh, then items (expert's group of tokens, 64 rows of Wg
//          and of Wu): gate rows in lanes 0 to 63 of the accumulator, up rows in 64 to 127. h goes
//          to the workspace as the second kernel reads it: fp16 layers in fp32, with the largest
//          magnitude of each row, from which that kernel splits it (split_pairs: within 2^-22); bf16
//          as two values (rounded, and what the rounding left: within 2^-16) that its copies bring;
//          four-bit experts' as three e4m3 pieces with block scales (within 2^-14 of the block's
//          largest value).
//   down   a cluster owns 128 rows of y; its CTAs take equal shares of the experts' steps along
//          the intermediate dimension, keep y's sums in shared memory and add them in rank order.
//
// 16 tokens, 8 of 64 experts of 1376 x 2048: bf16 190 us, fp16 193 for 955 MB (146 at the copy rate); 2 of 8
// of 8192 x 4096, bf16: 256 us, 95 % of it. Four bits, 32 tokens, 2 of 8 of 14336 x 4096: 251 us for
// 749 MB (114): spreading codes and bringing tokens take turns with the products at each stage.
#include <algorithm>
#include <cstring>

#include "host.h"
#include "moe.cuh"
#include "moe_wide.h"
#include "wide.cuh"

namespace swb {

int moe_wide_device_error(int clear, int* out) {
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

// Rows of h: token by token of its expert, `pieces` rows each.
__host__ __device__ constexpr int h_pieces(bool mx) { return mx ? 3 : 2; }

struct WideMaps {
    CUtensorMap gate, up;
};

// SPLIT: tokens are split into pieces at each use; else once, ahead of the items, into the
// workspace, which holds the pieces of kMoePieceDim values a token.
template <typename T_, bool MX, bool SPLIT, int TOK>
struct GateWork {
    using T = T_;
    static constexpr bool kMx = MX, kLoad = SPLIT || !MX, kFloat = false, kGather = MX && !SPLIT;
    static constexpr int kPieces = MX ? (std::is_same<T, __half>::value ? 3 : 2) : 1;
    static constexpr int kTok = TOK, kAccs = 2, kPerSm = 1;
    static constexpr int kStages = MX ? 3 : 8, kRaw = 4, kTokenStages = MX ? (TOK == 16 ? 10 : 5) : 6;
    static constexpr int kSpreadGroups = 2, kSplitters = kTokenStages, kGroupWarps = 1;

    const unsigned char* sa[2];
    const unsigned char *sb, *pieces;
    int pitch, pitch_b;
    int blocks, cols;
    int64_t rows_a;
    bool x_aligned;
    int halves;
    const MoeParams* P;
    const MoeRoute* R;
    int tiles, steps, g0, g1;
    uint32_t part;  // [token][kWidePartPitch]: gate rows, then up rows

    __device__ __forceinline__ bool item(int i, WideItem& it) const {
        if (g0 + i >= g1) return false;
        const int a = (g0 + i) / tiles, f = R->first[a], k = R->of_expert[a], j = g0 + i - f * tiles;
        const int group = f + j % k;
        it.row[0] = it.row[1] = int64_t(R->expert[group]) * P->inter + j / k * kWideHalf;
        it.s0 = 0;
        it.s1 = steps;
        it.first = R->start[group];
        it.count = R->start[group + 1] - it.first;
        return true;
    }
    __device__ __forceinline__ int place(const WideItem& it, int n) const { return R->token[it.first + n]; }
    __device__ __forceinline__ const T* token(const WideItem& it, int n) const {
        return static_cast<const T*>(P->x) + R->token[it.first + n] * P->x_pitch;
    }
    __device__ __forceinline__ void begin(const WideItem&) const {
        named_barrier_sync(4, kWideEpilogue * 32);  // the last item's sums are read
    }
    __device__ __forceinline__ void value(const WideItem&, int n, int row, float v) const {
        sts32(part + (n * kWidePartPitch + row) * 4, __float_as_uint(v));
    }
    __device__ __forceinline__ void end(const WideItem& it) const {
        named_barrier_sync(4, kWideEpilogue * 32);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int row0 = int(it.row[0] % P->inter);
        unsigned char* h = static_cast<unsigned char*>(P->h);
        // a warp takes 32 consecutive rows of a token, a block of h
        for (int c = warp; c < it.count * 2; c += kWideEpilogue) {
            const int n = c >> 1, r = (c & 1) * 32 + lane, i = row0 + r;
            if (row0 + (c & 1) * 32 >= P->inter) continue;
            const uint32_t at = part + (n * kWidePartPitch + r) * 4;
            const float g = __uint_as_float(lds32(at)), u = __uint_as_float(lds32(at + kWideHalf * 4));
            const float v = i < P->inter ? silu(g) * u : 0.f;
            const int64_t row = it.first + n;
            if constexpr (MX) {
                uint32_t top = __float_as_uint(v) & 0x7FFFFFFFu;
                top = __reduce_max_sync(0xFFFFFFFFu, top);
                const uint32_t scale = piece_scale(top);
                float f = v * __uint_as_float((254u - scale) << 23);
                if (!(fabsf(f) < 1024.f)) f = __uint_as_float(0x7FC00000u);
                unsigned char* s = h + int64_t(P->tokens) * P->topk * 3 * P->h_pitch;
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    uint16_t b;
                    uint32_t back;
                    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(b) : "f"(f));
                    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(b));
                    f = (f - half2_bits_to_float2(back).x) * 32.f;
                    if (i < P->inter) h[(row * 3 + p) * P->h_pitch + i] = static_cast<unsigned char>(b);
                    if (lane == 0) s[(row * 3 + p) * mx_blocks(P->inter) + i / kMxBlock] = static_cast<unsigned char>(scale - 5u * p);
                }
            } else if constexpr (std::is_same<T, __half>::value) {
                const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v) & 0x7FFFFFFFu);
                if (lane == 0) atomicMax(P->tops + kTopsWide * kMoeMaxRows + row, top);
                if (i < P->inter) reinterpret_cast<float*>(h)[row * P->h_pitch + i] = v;
            } else if (i < P->inter) {
                T* to = reinterpret_cast<T*>(h) + row * 2 * P->h_pitch + i;
                const T hi = Num<T>::from_float(v);
                to[0] = hi;
                to[P->h_pitch] = Num<T>::from_float(v - Num<T>::to_float(hi));
            }
        }
    }
};

template <typename T_, bool MX, int TOK>
struct DownWork {
    using T = T_;
    static constexpr bool kFloat = !MX && std::is_same<T, __half>::value;
    static constexpr bool kMx = MX, kLoad = kFloat, kGather = false;
    static constexpr int kPieces = h_pieces(MX);
    static constexpr int kTok = TOK, kAccs = 2, kPerSm = 1;
    static constexpr int kStages = MX ? 3 : 7, kRaw = 4, kTokenStages = MX ? (TOK == 16 ? 8 : 4) : 6;
    static constexpr int kSpreadGroups = 2, kSplitters = MX || kFloat ? kTokenStages : 4, kGroupWarps = 1;

    const unsigned char* sa[2];
    const unsigned char *sb, *pieces;
    int pitch, pitch_b;
    int blocks, cols;
    int64_t rows_a;
    bool x_aligned;
    int halves;
    const MoeParams* P;
    const MoeRoute* R;
    int64_t row0;    // of y
    int steps, f0, f1;  // this CTA's share [f0, f1) of groups x steps
    uint32_t total;  // [token][128]

    __device__ __forceinline__ bool item(int i, WideItem& it) const {
        const int group = f0 / steps + i, at = group * steps;
        if (at >= f1 || f0 >= f1) return false;
        it.row[0] = int64_t(R->expert[group]) * P->hidden + row0;
        it.row[1] = it.row[0] + kWideHalf;
        it.s0 = max(f0 - at, 0);
        it.s1 = min(f1 - at, steps);
        it.first = R->start[group];
        it.count = R->start[group + 1] - it.first;
        return true;
    }
    __device__ __forceinline__ int place(const WideItem&, int) const { return 0; }
    __device__ __forceinline__ const float* token(const WideItem& it, int n) const {
        return static_cast<const float*>(P->h) + int64_t(it.first + n) * P->h_pitch;
    }
    __device__ __forceinline__ float up(const WideItem& it, int n) const { return unit_inverse(R->unit[it.first + n]); }
    __device__ __forceinline__ void begin(const WideItem&) const {}
    // a thread owns a row of y; items come in the order of their experts
    __device__ __forceinline__ void value(const WideItem& it, int n, int row, float v) const {
        if constexpr (kFloat) v *= R->unit[it.first + n];
        const uint32_t at = total + (R->token[it.first + n] * kWideM + row) * 4;
        sts32(at, __float_as_uint(fmaf(R->share[it.first + n], v, __uint_as_float(lds32(at)))));
    }
    __device__ __forceinline__ void end(const WideItem&) const {}
};

// Every token's pieces, whole stages of them: [token * PIECES + piece][piece_pitch] and their scales.
__host__ __device__ inline int piece_pitch(int hidden) { return (hidden + 127) / 128 * 128; }
template <typename T, int PIECES>
__device__ void split_tokens(const MoeParams& P) {
    const int pitch = piece_pitch(P.hidden), parts = pitch / 8, all = P.tokens * parts;
    unsigned char* to = static_cast<unsigned char*>(P.pieces);
    unsigned char* scales = to + int64_t(P.tokens) * PIECES * pitch;
    // whole quads: a block's four lanes stay together (parts is a multiple of 16)
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i - int(threadIdx.x & 31) < all; i += gridDim.x * blockDim.x) {
        const int token = min(i, all - 1) / parts, part = min(i, all - 1) % parts;
        const T* row = static_cast<const T*>(P.x) + token * P.x_pitch;
        const uint4 v = P.x_aligned ? load_piece<T, true>(row, part * 8, P.hidden) : load_piece<T, false>(row, part * 8, P.hidden);
        uint2 piece[PIECES];
        const uint32_t scale = split_token<PIECES>(v, piece, T());
        if (i >= all) continue;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int64_t r = int64_t(token) * PIECES + p;
            *reinterpret_cast<uint2*>(to + r * pitch + part * 8) = piece[p];
            if (part % 4 == 0) scales[r * (pitch / kMxBlock) + part / 4] = static_cast<unsigned char>(scale - 5u * p);
        }
    }
}

template <typename T, bool MX, bool SPLIT, int TOK>
struct GateShape {
    using Pipe = Wide<GateWork<T, MX, SPLIT, TOK>>;
    static constexpr size_t kPart = Pipe::kRing;
    static constexpr size_t kRoute = (kPart + TOK * kWidePartPitch * 4 + 15) / 16 * 16;
    static constexpr size_t kSmem = kRoute + sizeof(MoeRoute) + 1024;
    static_assert(kSmem + 2048 <= kSmemPerCtaMax, "shared memory");
};
template <typename T, bool MX, int TOK>
struct DownShape {
    using Pipe = Wide<DownWork<T, MX, TOK>>;
    static constexpr size_t kTotal = Pipe::kRing;
    static constexpr size_t kRoute = kTotal + kMoeMaxTokens * kWideM * 4;
    static constexpr size_t kSmem = kRoute + sizeof(MoeRoute) + 1024;
    static_assert(kSmem + 1024 <= kSmemPerCtaMax, "shared memory");
};

template <typename T, bool MX, bool SPLIT, int TOK>
__global__ void __launch_bounds__(Wide<GateWork<T, MX, SPLIT, TOK>>::kThreads, 1)
    moe_gate_kernel(const __grid_constant__ WideMaps maps, const __grid_constant__ MoeParams P) {
    using S = GateShape<T, MX, SPLIT, TOK>;
    using Work = GateWork<T, MX, SPLIT, TOK>;
    constexpr int kWideThreads = S::Pipe::kThreads;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ typename S::Pipe::Shared sh;
    __shared__ double scratch[kRouteExperts * kRouteTokens * kRouteWarps];
    __shared__ int flag;
    MoeRoute& R = *reinterpret_cast<MoeRoute*>(smem + S::kRoute);
    S::Pipe::init(sh);
    if constexpr (!MX && std::is_same<T, __half>::value) {  // before the router's barrier
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < P.tokens * P.topk; i += kWideThreads) P.tops[kTopsWide * kMoeMaxRows + i] = 0u;
    }
    if constexpr (Work::kGather) split_tokens<T, Work::kPieces>(P);
    if (threadIdx.x < kRouteThreads) moe_router<T>(P, scratch, &flag);
    const bool routed = moe_grid_barrier(P.sync, &flag);
    griddep_launch_dependents();
    if (routed) {
        for (int i = threadIdx.x; i < P.tokens * P.topk; i += kWideThreads) {
            R.pick[i] = __ldcg(P.picks + i);
            R.shares[i] = __ldcg(P.shares + i);
        }
        __syncthreads();
        moe_lists(P, R);
        Work work;
        work.sa[0] = P.s[0];
        work.sa[1] = P.s[1];
        work.pitch = piece_pitch(P.hidden);
        work.pitch_b = work.pitch / kMxBlock;
        work.pieces = static_cast<const unsigned char*>(P.pieces);
        work.sb = work.pieces + int64_t(P.tokens) * Work::kPieces * work.pitch;
        work.blocks = int(mx_blocks(P.hidden));
        work.cols = P.hidden;
        work.rows_a = int64_t(P.experts) * P.inter;
        work.x_aligned = P.x_aligned != 0;
        work.halves = 2;
        work.P = &P;
        work.R = &R;
        work.tiles = (P.inter + kWideHalf - 1) / kWideHalf;
        work.steps = (P.hidden + S::Pipe::kValues - 1) / S::Pipe::kValues;
        const long long items = (long long)R.groups * work.tiles;
        work.g0 = int(blockIdx.x * items / gridDim.x);
        work.g1 = int((blockIdx.x + 1) * items / gridDim.x);
        work.part = smem_u32(smem + S::kPart);
        S::Pipe::run(work, sh, smem_u32(smem), &maps.gate, &maps.up, nullptr, l2_evict_first_policy());
    }
    __syncthreads();
    S::Pipe::finish(sh);
}

template <typename T, bool MX, int TOK>
__global__ void __launch_bounds__(Wide<DownWork<T, MX, TOK>>::kThreads, 1)
    moe_down_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_h,
                    const __grid_constant__ MoeParams P, int splits, int halves) {
    using S = DownShape<T, MX, TOK>;
    using Work = DownWork<T, MX, TOK>;
    constexpr int kWideThreads = S::Pipe::kThreads;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ typename S::Pipe::Shared sh;
    MoeRoute& R = *reinterpret_cast<MoeRoute*>(smem + S::kRoute);
    const uint32_t total = smem_u32(smem + S::kTotal);
    S::Pipe::init(sh);
    for (int i = threadIdx.x; i < P.tokens * kWideM; i += kWideThreads) sts32(total + i * 4, 0u);
    griddep_wait();  // the gate kernel's selection and h
    for (int i = threadIdx.x; i < P.tokens * P.topk; i += kWideThreads) {
        R.pick[i] = min(max(__ldcg(P.picks + i), 0), P.experts - 1);
        R.shares[i] = __ldcg(P.shares + i);
    }
    __syncthreads();
    moe_lists(P, R);
    if constexpr (Work::kFloat) {
        for (int i = threadIdx.x; i < P.tokens * P.topk; i += kWideThreads)
            R.unit[i] = row_unit(__ldcg(P.tops + kTopsWide * kMoeMaxRows + i));
        __syncthreads();
    }
    const int rank = int(blockIdx.x % splits);
    Work work;
    work.sa[0] = work.sa[1] = P.s[2];
    work.sb = static_cast<const unsigned char*>(P.h) + int64_t(P.tokens) * P.topk * 3 * P.h_pitch;
    work.blocks = work.pitch_b = int(mx_blocks(P.inter));
    work.pitch = 0;
    work.pieces = nullptr;
    work.cols = P.inter;
    work.rows_a = int64_t(P.experts) * P.hidden;
    work.x_aligned = true;
    work.halves = halves;
    work.P = &P;
    work.R = &R;
    const int tile_rows = halves * kWideHalf;
    work.row0 = int64_t(blockIdx.x / splits) * tile_rows;
    work.steps = (P.inter + S::Pipe::kValues - 1) / S::Pipe::kValues;
    const long long all = (long long)R.groups * work.steps;
    work.f0 = int(rank * all / splits);
    work.f1 = int((rank + 1) * all / splits);
    work.total = total;
    S::Pipe::run(work, sh, smem_u32(smem), &map_w, &map_w, &map_h, l2_evict_first_policy());
    __syncthreads();
    S::Pipe::finish(sh);

    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    if (!sh.failed) {
        for (int i = rank * kWideThreads + threadIdx.x; i < P.tokens * kWideM; i += splits * kWideThreads) {
            const int64_t row = work.row0 + i % kWideM;
            if (i % kWideM >= tile_rows || row >= P.hidden) continue;
            float v = 0.f;
            for (int j = 0; j < splits; ++j) {
                uint32_t remote;
                float f;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(total + i * 4), "r"(j));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(remote) : "memory");
                v += f;
            }
            static_cast<T*>(P.y)[int64_t(i / kWideM) * P.hidden + row] = Num<T>::from_float(v);
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, bool MX, bool SPLIT, int TOK>
int launch_moe_wide(const MoeParams& P, cudaStream_t stream) {
    static std::atomic<uint64_t> gate_set{0}, down_set{0};
    const int sms = sm_count();
    if (sms <= 0) return check_launch();
    using G = GateShape<T, MX, SPLIT, TOK>;
    using D = DownShape<T, MX, TOK>;
    auto gate = moe_gate_kernel<T, MX, SPLIT, TOK>;
    auto down = moe_down_kernel<T, MX, TOK>;
    if (int rc = allow_smem(gate, gate_set, G::kSmem)) return rc;
    if (int rc = allow_smem(down, down_set, D::kSmem)) return rc;
    WideMaps maps;
    CUtensorMap map_w, map_h;
    const int64_t gate_rows = int64_t(P.experts) * P.inter, rows = int64_t(P.tokens) * P.topk * h_pieces(MX);
    if (int rc = make_wide_map(&maps.gate, P.w[0], gate_rows, P.hidden, MX)) return rc;
    if (int rc = make_wide_map(&maps.up, P.w[1], gate_rows, P.hidden, MX)) return rc;
    if (int rc = make_wide_map(&map_w, P.w[2], int64_t(P.experts) * P.hidden, P.inter, MX)) return rc;
    if (DownWork<T, MX, TOK>::kFloat)
        map_h = map_w;  // its kernel loads h itself
    else if (int rc = make_typed_map(&map_h, MX ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, P.h, P.inter,
                                rows, int64_t(P.h_pitch) * (MX ? 1 : 2), MX ? 128 : 64, 16))
        return rc;
    // every CTA resident at once: the cooperative launch makes the runtime check it
    if (int rc = launch_ex(gate, unsigned(sms), G::Pipe::kThreads, G::kSmem, stream, true, maps, P)) return rc;

    // 128 rows of y a cluster, or 64 where that leaves SMs without work. Clusters of four: the SMs
    // of a GPC hold few of eight (16 clusters of eight took two waves, 113 us for 309 MB).
    constexpr int kMostSplits = 4;
    const int halves = (P.hidden + kWideM - 1) / kWideM * kMostSplits > sms / 2 ? 2 : 1;
    const int tiles = (P.hidden + halves * kWideHalf - 1) / (halves * kWideHalf);
    int splits = 1;
    while (splits < kMostSplits && tiles * splits * 2 <= sms) splits *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(tiles * splits));
    cfg.blockDim = dim3(D::Pipe::kThreads);
    cfg.dynamicSmemBytes = D::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, down, map_w, map_h, P, splits, halves);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(SWB_E_CUDA, cudaGetErrorString(e));
    }
    return SWB_OK;
}

}  // namespace

// Up to eight tokens the register path's 16-row items spread better over the SMs and its one
// kernel starts sooner.
bool moe_wide_takes(const MoeParams& P, bool mx) {
    return P.tokens > 8 && wide_rows(P.w[0], P.hidden, mx) && wide_rows(P.w[1], P.hidden, mx) &&
           wide_rows(P.w[2], P.inter, mx);
}

namespace {
template <typename T>
int dispatch_moe_wide(bool mx, MoeParams P, cudaStream_t stream) {
    if (!mx) return launch_moe_wide<T, false, false, kMoeGroup>(P, stream);
    // longer tokens than the workspace's pieces are split at each use: every item of an expert repeats
    // the conversions (four-bit experts of 14336 x 4096, 32 tokens: 330 us of gate against 190)
    const bool split = P.hidden > kMoePieceDim;
    // Four-bit items of 16 tokens leave shared memory for twice the stages of tokens: 247 us against
    // 273 (32 tokens, 2 of 8 experts of 14336 x 4096). An expert with more tokens is then read twice:
    // 118 us against 101 (64 tokens, 2 of 8 experts of 5632 x 2048, 16 each on average).
    if (P.tokens * P.topk <= 8 * P.experts) {
        P.group = kMoeFewGroup;
        return split ? launch_moe_wide<T, true, true, kMoeFewGroup>(P, stream) : launch_moe_wide<T, true, false, kMoeFewGroup>(P, stream);
    }
    return split ? launch_moe_wide<T, true, true, kMoeGroup>(P, stream) : launch_moe_wide<T, true, false, kMoeGroup>(P, stream);
}
}  // namespace

int moe_wide(int type, bool mx, const MoeParams& P, cudaStream_t stream) {
    return type == SWB_F16 ? dispatch_moe_wide<__half>(mx, P, stream) : dispatch_moe_wide<__nv_bfloat16>(mx, P, stream);
}

}  // namespace swb
