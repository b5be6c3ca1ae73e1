// A whole mixture-of-experts SwiGLU layer in one kernel: up to eight tokens, and 16-bit matrices
// whose rows do not start on 16 bytes (moe_wide.cu takes the others).
//
//   logits = Wr x;  experts = the topk largest (ties: lowest index, NaN first);
//   w = softmax over the selected (or over all) logits
//   y_t = sum_j w_tj Wd_e (SiLU(Wg_e x_t) * (Wu_e x_t)),  e = experts_tj
//
// Bound by bytes: every expert that a token selects is read once, 6 HI bytes at 16
// bits or 51/32 HI at four. One persistent cooperative kernel, so that a call costs one
// launch and the three phases are separated by a grid barrier (about a microsecond)
// instead of a kernel boundary each:
//
//   router  a CTA takes four experts by four tokens, its warps splitting H; products
//           and sums in 64 bits, so that the selection does not depend on the order of
//           a sum. The CTA that completes a group of four tokens selects their experts.
//   gate    items (expert, 16 rows of Wg and Wu) spread over the CTAs; h goes to the
//           workspace with an expert's tokens side by side: fp16 layers in fp32, with the largest
//           magnitude of each row, bf16 as two values (rounded, and what the rounding left).
//   down    a CTA owns 16 rows of y at a time and takes every expert's product for
//           them in expert order, so y needs no atomics and repeats bit for bit. Its
//           weights are on their way while the grid waits for h. h is multiplied as two values of
//           the layer's type (row_unit): 2^-22 of it is lost with fp16, 2^-16 with bf16.
//
// An expert with more than 32 tokens is taken in groups of 32, each group of a tile right
// after the other, so that the second finds the weights in L2 (64 tokens through two experts read 147
// MB from DRAM, 32 tokens 139).
//
// 40 us for the two experts that one token selects of 5632 x 2048 (fp16, 138 MB: 3.4 TB/s of the
// 6.5 that a copy reaches); the router, its lists and the grid barrier take about 7 us of it, the
// first and last stages of the two streams most of the rest. Four-bit experts, one token: 37 us for 37 MB
// (5632 x 2048; issue slots 32 % busy, DRAM 9 %, most stalls at barriers and waits) and 104 us for 187 MB
// (14336 x 4096).
#pragma once

#include <type_traits>

#include "stream.cuh"

namespace swb {

constexpr int kMoeMaxTokens = 64;
constexpr int kMoeMaxExperts = 256;
constexpr int kMoeMaxTopk = 16;
constexpr int kMoeGroup = 32, kMoeFewGroup = 16;  // most tokens of an item; where experts get few (moe_wide.cu)
constexpr int kMoeMaxGroups = kMoeMaxExperts + kMoeMaxTokens * kMoeMaxTopk / kMoeFewGroup;
constexpr int kMoeMaxRows = kMoeMaxTokens * kMoeMaxTopk;  // of h
// The largest magnitudes start a call at zero. moe_kernel may have no barrier before the first of
// them, so its calls use two sets in turn (sync word kSyncTurn: which) and clear the other; the third
// is moe_wide.cu's, cleared before its router's barrier.
constexpr int kSyncTurn = 63, kTopsWide = 2;
constexpr int kRouteExperts = 4, kRouteTokens = 4;  // of a router unit
constexpr int kRouteWarps = 8, kRouteThreads = kRouteWarps * 32;  // that compute logits

struct MoeMaps {
    WeightMaps m[3];  // gate, up, down
};

struct MoeParams {
    const void* x;
    const void* router;
    const unsigned char* w[3];  // gate, up, down
    const unsigned char* s[3];  // their scales (MXFP4)
    void* y;
    int* ids;        // [tokens, topk] or null
    float* weights;  // [tokens, topk] or null
    uint32_t* sync;  // [0] grid barrier, [1 + group] finished router units of a group of tokens, [kSyncTurn]
    uint32_t* tops;  // [3][kMoeMaxRows]: the largest magnitude of each row of h (fp16 layers)
    double* logits;  // [tokens, experts]
    int* picks;      // [tokens, topk]
    float* shares;   // [tokens, topk]
    void* h;         // [tokens * topk, h_pitch], four bytes a value: fp32, or two parts of eight values after
                     // another (bf16); moe_wide.cu: or what its second kernel's copies bring
    void* pieces;    // tokens split into e4m3 values (moe_wide.cu)
    int64_t x_pitch;
    int tokens, hidden, inter, experts, topk, h_pitch;
    int group;  // tokens of an item
    int renormalize;
    int x_aligned, router_aligned;  // 16-byte pieces of the rows of x, of Wr
    bool fast[2], deep[2];          // make_weight_maps of gate and up, of down
};

// Offsets of the workspace's parts.
struct MoeWorkspace {
    size_t tops, logits, picks, shares, h, pieces, total;
};
constexpr int kMoePieceDim = 8192;  // values of a token whose pieces the workspace holds
__host__ __device__ inline int moe_h_pitch(int inter) { return (inter + kTileRows - 1) / kTileRows * kTileRows; }
__host__ __device__ inline MoeWorkspace moe_workspace(int tokens, int experts, int topk, int inter) {
    MoeWorkspace m;
    m.tops = 256;  // the sync words before it; these two stand where every size of call finds them
    m.logits = m.tops + 3 * kMoeMaxRows * 4;
    m.picks = m.logits + size_t(tokens) * experts * 8;
    m.shares = m.picks + size_t(tokens) * topk * 4;
    m.h = (m.shares + size_t(tokens) * topk * 4 + 255) / 256 * 256;
    m.pieces = (m.h + size_t(tokens) * topk * moe_h_pitch(inter) * 4 + 255) / 256 * 256;
    m.total = m.pieces + (tokens > 8 ? size_t(tokens) * 3 * (kMoePieceDim + kMoePieceDim / 32) : 0);
    return m;
}

// What every CTA derives from the selection. Rows of h stand in the order of their experts,
// then tokens; a group is up to P.group of an expert's rows.
struct MoeRoute {
    unsigned long long taken[kMoeMaxExperts];          // an expert's tokens, a bit each
    float share[kMoeMaxTokens * kMoeMaxTopk];          // of each row of h: its expert's weight
    union {
        float shares[kMoeMaxTokens * kMoeMaxTopk];     // [token, place]: the same, until the lists are made
        float unit[kMoeMaxTokens * kMoeMaxTopk];       // of each row of h (row_unit), once h is complete
    };
    int pick[kMoeMaxTokens * kMoeMaxTopk];             // [token, place]: the expert
    int groups;
    short row[kMoeMaxExperts];                         // an expert's first row of h
    short expert[kMoeMaxGroups];                       // of each group
    short start[kMoeMaxGroups + 1];                    // its first row of h, and the end
    short first[kMoeMaxGroups];                        // the expert's first group
    short of_expert[kMoeMaxGroups];                    // and how many it has
    unsigned char token[kMoeMaxTokens * kMoeMaxTopk];  // of each row of h
};

template <typename T, bool MX, int NT>
struct MoeShape {
    using Pipe = Stream<T, MX, NT>;
    static constexpr size_t kOther = (sizeof(MoeRoute) + 15) / 16 * 16 + kMoeMaxTokens * kTileRows * 4 + 1280;
    static constexpr int kStages = Pipe::stages(kOther);
    static constexpr size_t kRoute = (Pipe::bytes(kStages) + 15) / 16 * 16;   // offset of MoeRoute
    static constexpr size_t kTotal = kRoute + (sizeof(MoeRoute) + 15) / 16 * 16;  // of y's sums
    static constexpr size_t kSmem = kTotal + kMoeMaxTokens * kTileRows * 4;
};

__device__ __forceinline__ uint32_t moe_ld_acquire(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// One thread's part of a grid barrier over a word whose low 31 bits are zero between
// barriers: CTA 0 adds what the others' ones leave to 2^31, so the top bit flips once
// everybody arrived. Waits at most kWaitLimitNs; false when it gave up. What the CTA wrote
// before (ordered by a barrier among its threads) is visible to every CTA afterwards.
__device__ __forceinline__ bool moe_grid_arrive_wait(uint32_t* word) {
    __threadfence();
    const uint32_t add = blockIdx.x == 0 ? 0x80000000u - uint32_t(gridDim.x - 1) : 1u;
    const uint32_t seen = atomicAdd(word, add) & 0x80000000u;
    const uint64_t t0 = global_timer_ns();
    while ((moe_ld_acquire(word) & 0x80000000u) == seen) {
        if (global_timer_ns() - t0 > kWaitLimitNs) {
            atomicOr(&g_device_error, 1);
            return false;
        }
    }
    __threadfence();
    return true;
}

// The barrier for every thread of the CTA; false in all of them when it gave up.
__device__ __forceinline__ bool moe_grid_barrier(uint32_t* word, int* ok) {
    __syncthreads();
    if (threadIdx.x == 0) *ok = moe_grid_arrive_wait(word);
    __syncthreads();
    return *ok != 0;
}

// Order of selection: NaN above everything, then the value.
__device__ __forceinline__ bool moe_above(double a, int ia, double b, int ib) {
    const bool na = a != a, nb = b != b;
    if (na != nb) return na;
    if (na || a == b) return ia < ib;
    return a > b;
}

// One warp selects a token's experts from its logits `l` into picks and shares [topk].
__device__ inline void moe_select(const MoeParams& P, const double* l, int* picks, float* shares, int lane) {
    constexpr int kPer = kMoeMaxExperts / 32;
    double v[kPer];
    uint32_t left = 0;  // which of this lane's logits are still in play
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        v[i] = 0.0;
        if (e < P.experts) {
            v[i] = *reinterpret_cast<const volatile double*>(l + e);
            left |= 1u << i;
        }
    }
    const uint32_t all = left;
    double top = 0.0, mine = 0.0;
    int pick = 0;
    for (int j = 0; j < P.topk; ++j) {
        double best = 0.0;
        int at = -1;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if ((left >> i) & 1u)
                if (at < 0 || moe_above(v[i], lane + 32 * i, best, at)) best = v[i], at = lane + 32 * i;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const double ob = __shfl_xor_sync(0xFFFFFFFFu, best, d);
            const int oa = __shfl_xor_sync(0xFFFFFFFFu, at, d);
            if (oa >= 0 && (at < 0 || moe_above(ob, oa, best, at))) best = ob, at = oa;
        }
        if (j == 0) top = best;
        if (lane == j) mine = best, pick = at;
        if ((at & 31) == lane) left &= ~(1u << (at >> 5));
    }
    float e = lane < P.topk ? expf(float(mine - top)) : 0.f;
    float sum = 0.f;
    if (P.renormalize) {
        sum = e;
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if ((all >> i) & 1u) sum += expf(float(v[i] - top));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane < P.topk) {
        picks[lane] = pick;
        shares[lane] = e / sum;
    }
}

template <typename T>
__device__ __forceinline__ uint4 route_piece(const T* row, int k, int cols, int aligned) {
    return aligned ? load_piece<T, true>(row, k, cols) : load_piece<T, false>(row, k, cols);
}

// Router of a few (token, expert) pairs: every CTA takes all of them, a warp a pair at a time, and
// selects for itself, which costs less than telling the others. Logits in 64 bits as above.
constexpr int kRouteAlone = 32;  // pairs; 148 CTAs reading the router's rows from L2 is about a barrier's time
template <typename T>
__device__ void moe_router_alone(const MoeParams& P, double* logits, int* picks, float* shares) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(P.x);
    const T* r = static_cast<const T*>(P.router);
    for (int pair = warp; pair < P.tokens * P.experts; pair += kRouteWarps) {
        const int t = pair / P.experts, e = pair % P.experts;
        double sum[8] = {0., 0., 0., 0., 0., 0., 0., 0.};
#pragma unroll 4
        for (int k = lane * 8; k < P.hidden; k += 256) {
            const uint4 wv = route_piece(r + size_t(e) * P.hidden, k, P.hidden, P.router_aligned);
            const uint4 xv = route_piece(x + t * P.x_pitch, k, P.hidden, P.x_aligned);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sum[i] = fma(double(Num<T>::to_float(reinterpret_cast<const T*>(&wv)[i])),
                             double(Num<T>::to_float(reinterpret_cast<const T*>(&xv)[i])), sum[i]);
        }
        double s = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        if (lane == 0) logits[pair] = s;
    }
    named_barrier_sync(1, kRouteThreads);
    for (int t = warp; t < P.tokens; t += kRouteWarps)
        moe_select(P, logits + t * P.experts, picks + t * P.topk, shares + t * P.topk, lane);
}

// The first kRouteThreads threads of the CTA.
template <typename T>
__device__ void moe_router(const MoeParams& P, double* scratch, int* flag) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int expert_units = (P.experts + kRouteExperts - 1) / kRouteExperts;
    const int groups = (P.tokens + kRouteTokens - 1) / kRouteTokens;
    const T* x = static_cast<const T*>(P.x);
    const T* r = static_cast<const T*>(P.router);
    for (int unit = blockIdx.x; unit < expert_units * groups; unit += gridDim.x) {
        const int group = unit / expert_units, e0 = unit % expert_units * kRouteExperts, t0 = group * kRouteTokens;
        double sum[kRouteExperts][kRouteTokens];
#pragma unroll
        for (int a = 0; a < kRouteExperts; ++a)
#pragma unroll
            for (int b = 0; b < kRouteTokens; ++b) sum[a][b] = 0.0;
        const int nt = min(kRouteTokens, P.tokens - t0);
        for (int k = threadIdx.x * 8; k < P.hidden; k += kRouteThreads * 8) {
            uint4 wv[kRouteExperts], xv[kRouteTokens];
#pragma unroll
            for (int a = 0; a < kRouteExperts; ++a)
                wv[a] = route_piece(r + size_t(min(e0 + a, P.experts - 1)) * P.hidden, k, P.hidden, P.router_aligned);
#pragma unroll
            for (int b = 0; b < kRouteTokens; ++b)
                xv[b] = route_piece(x + (t0 + min(b, nt - 1)) * P.x_pitch, k, P.hidden, P.x_aligned);
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // zero beyond the row
                double wd[kRouteExperts];
#pragma unroll
                for (int a = 0; a < kRouteExperts; ++a) wd[a] = Num<T>::to_float(reinterpret_cast<const T*>(wv + a)[i]);
#pragma unroll
                for (int b = 0; b < kRouteTokens; ++b) {
                    if (b >= nt) break;
                    const double xd = Num<T>::to_float(reinterpret_cast<const T*>(xv + b)[i]);
#pragma unroll
                    for (int a = 0; a < kRouteExperts; ++a) sum[a][b] = fma(wd[a], xd, sum[a][b]);
                }
            }
        }
#pragma unroll
        for (int a = 0; a < kRouteExperts; ++a)
#pragma unroll
            for (int b = 0; b < kRouteTokens; ++b) {
                if (b >= nt) break;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) sum[a][b] += __shfl_xor_sync(0xFFFFFFFFu, sum[a][b], d);
                if (lane == 0) scratch[(a * kRouteTokens + b) * kRouteWarps + warp] = sum[a][b];
            }
        named_barrier_sync(1, kRouteThreads);
        if (threadIdx.x < kRouteExperts * kRouteTokens) {
            const int a = threadIdx.x / kRouteTokens, b = threadIdx.x % kRouteTokens;
            if (e0 + a < P.experts && b < nt) {
                double s = 0.0;
                for (int j = 0; j < kRouteWarps; ++j) s += scratch[(a * kRouteTokens + b) * kRouteWarps + j];
                P.logits[size_t(t0 + b) * P.experts + e0 + a] = s;
            }
            __threadfence();
        }
        named_barrier_sync(1, kRouteThreads);
        if (threadIdx.x == 0) {
            *flag = atomicAdd(P.sync + 1 + group, 1u) == uint32_t(expert_units - 1);
            if (*flag) {
                P.sync[1 + group] = 0u;  // for the next call
                __threadfence();
            }
        }
        named_barrier_sync(1, kRouteThreads);
        if (*flag && warp < nt) {
            const int t = t0 + warp;
            moe_select(P, P.logits + size_t(t) * P.experts, P.picks + t * P.topk, P.shares + t * P.topk, lane);
        }
        named_barrier_sync(1, kRouteThreads);
    }
}

// Groups of each expert's tokens, in token order, the same in every CTA; R.pick and R.shares
// are set. One CTA hands the selection to the caller.
__device__ inline void moe_lists(const MoeParams& P, MoeRoute& R) {
    const int n = P.tokens * P.topk, t = threadIdx.x;
    if (t < kMoeMaxExperts) R.taken[t] = 0ull;
    __syncthreads();
    for (int i = t; i < n; i += blockDim.x) {
        atomicOr(&R.taken[R.pick[i]], 1ull << (i / P.topk));  // a token takes an expert once: the bits are its rows
        if (blockIdx.x == 0) {
            if (P.ids) P.ids[i] = R.pick[i];
            if (P.weights) P.weights[i] = R.shares[i];
        }
    }
    __syncthreads();
    if (t < 32) {  // eight experts a lane: rows and groups before them
        constexpr int kPer = kMoeMaxExperts / 32;
        int count[kPer], rows = 0, groups = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            count[i] = __popcll(R.taken[t * kPer + i]);
            rows += count[i];
            groups += (count[i] + P.group - 1) / P.group;
        }
        int row = rows, a = groups;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int r = __shfl_up_sync(0xFFFFFFFFu, row, d), b = __shfl_up_sync(0xFFFFFFFFu, a, d);
            if (t >= d) row += r, a += b;
        }
        if (t == 31) {
            R.groups = a;
            R.start[a] = short(row);
        }
        row -= rows;
        a -= groups;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = t * kPer + i, k = (count[i] + P.group - 1) / P.group;
            R.row[e] = short(row);
            for (int j = 0; j < k; ++j) {
                R.expert[a + j] = short(e);
                R.start[a + j] = short(row + j * P.group);
                R.first[a + j] = short(a);
                R.of_expert[a + j] = short(k);
            }
            a += k;
            row += count[i];
        }
    }
    __syncthreads();
    for (int i = t; i < n; i += blockDim.x) {
        const int e = R.pick[i], token = i / P.topk;
        const int row = R.row[e] + __popcll(R.taken[e] & ((1ull << token) - 1ull));
        R.token[row] = static_cast<unsigned char>(token);
        R.share[row] = R.shares[i];
    }
    __syncthreads();
}

template <typename T, bool MX, int NT>
__global__ void __launch_bounds__(Stream<T, MX, NT>::kThreads, 1)
    moe_kernel(const __grid_constant__ MoeMaps maps, const MoeParams P) {
    using S = MoeShape<T, MX, NT>;
    using Pipe = typename S::Pipe;
    constexpr int kConsumers = Pipe::kConsumers, kThreads = Pipe::kThreads;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ double scratch[kRouteExperts * kRouteTokens * kRouteWarps];
    __shared__ int flag, sums_ok;
    MoeRoute& R = *reinterpret_cast<MoeRoute*>(smem + S::kRoute);
    float* total = reinterpret_cast<float*>(smem + S::kTotal);  // [token][16 rows of y]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = gridDim.x, b = blockIdx.x;
    const auto l = Pipe::layout(smem_u32(smem), S::kStages);
    if (threadIdx.x == kThreads - 1) Pipe::init(l);
    constexpr bool kHalf = std::is_same<T, __half>::value;
    // read before this CTA comes to a barrier, after which CTA 0 turns it
    const uint32_t turn = kHalf ? *reinterpret_cast<volatile uint32_t*>(P.sync + kSyncTurn) & 1u : 0u;
    uint32_t* tops = P.tops + turn * kMoeMaxRows;
    if (kHalf && b == G - 1)
        for (int i = threadIdx.x; i < kMoeMaxRows; i += kThreads) P.tops[(turn ^ 1u) * kMoeMaxRows + i] = 0u;

    if (P.tokens * P.experts <= kRouteAlone) {
        if (warp < kRouteWarps) moe_router_alone<T>(P, scratch, R.pick, R.shares);
        __syncthreads();
    } else {
        if (warp < kRouteWarps) moe_router<T>(P, scratch, &flag);
        if (!moe_grid_barrier(P.sync, &flag)) return;
        for (int i = threadIdx.x; i < P.tokens * P.topk; i += kThreads) {
            R.pick[i] = __ldcg(P.picks + i);
            R.shares[i] = __ldcg(P.shares + i);
        }
        __syncthreads();
    }
    moe_lists(P, R);

    // gate: items [g0, g1) are (expert, tile, group); down: tiles [d0, d1) times every group
    const int gate_tiles = (P.inter + kTileRows - 1) / kTileRows, down_tiles = (P.hidden + kTileRows - 1) / kTileRows;
    const long long gate_items = (long long)R.groups * gate_tiles;
    const int g0 = int(b * gate_items / G), g1 = int((b + 1) * gate_items / G);
    const int d0 = int((long long)b * down_tiles / G), d1 = int((long long)(b + 1) * down_tiles / G);
    auto gate_item = [&](int item, int& group, int& row) {
        const int a = item / gate_tiles, f = R.first[a], k = R.of_expert[a], j = item - f * gate_tiles;
        group = f + j % k;
        row = j / k * kTileRows;
    };
    const WeightMaps* gm = P.fast[0] ? &maps.m[0] : nullptr;
    const WeightView gv[2] = {
        weight_view<MX>(P.w[0], P.s[0], int64_t(P.experts) * P.inter, P.hidden, gm, P.deep[0]),
        weight_view<MX>(P.w[1], P.s[1], int64_t(P.experts) * P.inter, P.hidden, gm ? &maps.m[1] : nullptr, P.deep[0])};
    const WeightView dv[1] = {weight_view<MX>(P.w[2], P.s[2], int64_t(P.experts) * P.hidden, P.inter,
                                              P.fast[1] ? &maps.m[2] : nullptr, P.deep[1])};
    auto gate_rows = [&](int group, int row) {
        Tiles<2> t;
        t.row[0] = t.row[1] = int64_t(R.expert[group]) * P.inter + row;
        t.rows[0] = t.rows[1] = min(kTileRows, P.inter - row);
        return t;
    };
    auto down_rows = [&](int group, int tile) {
        Tiles<1> t;
        t.row[0] = int64_t(R.expert[group]) * P.hidden + tile * kTileRows;
        t.rows[0] = min(kTileRows, P.hidden - tile * kTileRows);
        return t;
    };
    float* h = static_cast<float*>(P.h);
    typename Pipe::Place place;

    if (warp == kConsumers) {
        const uint64_t policy = l2_evict_first_policy();
        for (int i = g0; i < g1 && place.ok; ++i) {
            int group, row;
            gate_item(i, group, row);
            Pipe::template produce<2>(l, place, gate_rows(group, row), gv, policy);
        }
        for (int d = d0; d < d1; ++d)
            for (int a = 0; a < R.groups && place.ok; ++a)
                Pipe::template produce<1>(l, place, down_rows(a, d), dv, policy);
        Pipe::drain(l, place);
    } else if (warp < kConsumers) {
        auto gate = [&](auto fast) {
            typename Pipe::template Tokens<2, false> tokens;
            auto turn_to = [&](int i) {
                tokens.count = 0;
                if (i >= g1) return;
                int group, row;
                gate_item(i, group, row);
                const int start = R.start[group];
                tokens.count = R.start[group + 1] - start;
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    tokens.x[n] = static_cast<const T*>(P.x) + R.token[start + min(n * 8 + (lane >> 2), tokens.count - 1)] * P.x_pitch;
            };
            turn_to(g0);
            tokens.template load<decltype(fast)::value>(0, 0, P.hidden);
            for (int i = g0; i < g1 && place.ok; ++i) {
                int group, row;
                gate_item(i, group, row);
                Pipe::template consume<2, false, decltype(fast)::value>(l, place, gate_rows(group, row), gv, tokens, P.hidden,
                                                                        [&](auto&) { turn_to(i + 1); });
            }
        };
        if (gv[0].maps)
            gate(std::true_type{});
        else
            gate(std::false_type{});
        named_barrier_sync(2, kThreads - 32);  // h is complete, or flag says that it will not be
        auto down = [&](auto fast) {
            typename Pipe::template Tokens<1, true> tokens;
            auto turn_to = [&](int d, int a) {
                if (a == R.groups) ++d, a = 0;
                tokens.count = 0;
                if (d >= d1) return;
                const int start = R.start[a];
                tokens.count = R.start[a + 1] - start;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int row = start + min(n * 8 + (lane >> 2), tokens.count - 1);
                    tokens.x[n] = h + int64_t(row) * P.h_pitch;
                    if constexpr (kHalf) tokens.top[n] = __ldcg(tops + row);
                }
            };
            turn_to(d0, 0);
            tokens.template load<decltype(fast)::value>(0, 0, P.h_pitch);
            for (int d = d0; d < d1; ++d)
                for (int a = 0; a < R.groups && place.ok; ++a)
                    Pipe::template consume<1, true, decltype(fast)::value>(l, place, down_rows(a, d), dv, tokens, P.h_pitch,
                                                                           [&](auto&) { turn_to(d, a + 1); });
        };
        if (flag) {
            if (dv[0].maps)
                down(std::true_type{});
            else
                down(std::false_type{});
        }
    } else {
        const int thread = threadIdx.x - (kConsumers + 1) * 32;
        for (int i = g0; i < g1 && Pipe::acquire(l, place); ++i) {
            int group, row;
            gate_item(i, group, row);
            const int start = R.start[group], count = R.start[group + 1] - start;
            for (int c = thread; c - lane < count * kTileRows; c += kEpilogueThreads) {  // whole warps
                const int n = c >> 4, r = c & 15;
                float v = 0.f;
                if (c < count * kTileRows) {
                    const float g = Pipe::template sum<2>(l, place, 0, n, r), u = Pipe::template sum<2>(l, place, 1, n, r);
                    // rows up to the pitch of h are zero, so that a whole piece of h may be read
                    if (row + r < P.inter) v = silu(g) * u;
                    float* to = h + int64_t(start + n) * P.h_pitch + row;
                    if constexpr (kHalf) {
                        to[r] = v;
                    } else {
                        T* parts = reinterpret_cast<T*>(to + (r & 8)) + (r & 7);
                        const T hi = Num<T>::from_float(v);
                        parts[0] = hi;
                        parts[8] = Num<T>::from_float(v - Num<T>::to_float(hi));
                    }
                }
                if constexpr (kHalf) {  // 16 lanes hold 16 places of a row
                    uint32_t top = __float_as_uint(v) & 0x7FFFFFFFu;
#pragma unroll
                    for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                    if (r == 0 && c < count * kTileRows) atomicMax(tops + start + n, top);
                }
            }
            Pipe::release(l, place);
        }
        named_barrier_sync(3, kEpilogueThreads);
        if (thread == 0) {
            flag = place.ok && moe_grid_arrive_wait(P.sync);
            if (kHalf && b == 0 && flag) P.sync[kSyncTurn] = turn ^ 1u;
            __threadfence();
        }
        named_barrier_sync(2, kThreads - 32);
        if constexpr (kHalf)  // before the barrier that precedes the first sums
            for (int i = thread; i < P.tokens * P.topk; i += kEpilogueThreads) R.unit[i] = row_unit(__ldcg(tops + i));
        T* y = static_cast<T*>(P.y);
        for (int d = d0; d < d1 && flag; ++d) {
            for (int c = thread; c < P.tokens * kTileRows; c += kEpilogueThreads) total[c] = 0.f;
            for (int a = 0; a < R.groups; ++a) {
                if (thread < 32) {
                    Pipe::acquire(l, place);
                    if (thread == 0) sums_ok = place.ok;
                }
                named_barrier_sync(3, kEpilogueThreads);  // the sums are there, the last group's additions done
                place.ok = sums_ok != 0;
                if (!place.ok) break;
                const int start = R.start[a], count = R.start[a + 1] - start;
                for (int c = thread; c < count * kTileRows; c += kEpilogueThreads) {
                    const int n = c >> 4, r = c & 15;  // a token takes an expert once: no two threads meet
                    float& sum = total[R.token[start + n] * kTileRows + r];
                    float v = Pipe::template sum<1>(l, place, 0, n, r);
                    if constexpr (kHalf) v *= R.unit[start + n];
                    sum = fmaf(R.share[start + n], v, sum);
                }
                Pipe::release(l, place);
            }
            if (!place.ok) break;
            named_barrier_sync(3, kEpilogueThreads);
            for (int c = thread; c < P.tokens * kTileRows; c += kEpilogueThreads) {
                const int row = d * kTileRows + (c & 15);
                if (row < P.hidden) y[int64_t(c >> 4) * P.hidden + row] = Num<T>::from_float(total[c]);
            }
            named_barrier_sync(3, kEpilogueThreads);
        }
    }
}

}  // namespace swb
