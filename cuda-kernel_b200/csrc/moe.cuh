// A whole mixture-of-experts SwiGLU layer for a few tokens in one kernel.
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
//   gate    items (expert, 16 rows of Wg and Wu) spread over the CTAs; h, rounded to
//           the layer's type (the operand of the next product), goes to the workspace
//           with an expert's tokens side by side.
//   down    a CTA owns 16 rows of y at a time and takes every expert's product for
//           them in expert order, so y needs no atomics and repeats bit for bit.
#pragma once

#include "stream.cuh"

namespace swb {

constexpr int kMoeWarps = 8;
constexpr int kMoeThreads = kMoeWarps * 32;
constexpr int kMoeMaxTokens = 64;
constexpr int kMoeMaxExperts = 256;
constexpr int kMoeMaxTopk = 16;
constexpr int kRouteExperts = 4, kRouteTokens = 4;  // of a router unit

struct MoeParams {
    const void* x;
    const void* router;
    const unsigned char* w[3];  // gate, up, down
    const unsigned char* s[3];  // their scales (MXFP4)
    void* y;
    int* ids;        // [tokens, topk] or null
    float* weights;  // [tokens, topk] or null
    uint32_t* sync;  // [0] grid barrier, [1 + group] finished router units of a group of tokens
    double* logits;  // [tokens, experts]
    int* picks;      // [tokens, topk]
    float* shares;   // [tokens, topk]
    void* h;         // [tokens * topk, h_pitch]
    int64_t x_pitch;
    int tokens, hidden, inter, experts, topk, h_pitch;
    int renormalize;
    int x_aligned, router_aligned;   // 16-byte pieces of the rows of x, of Wr
    int gate_aligned, down_aligned;  // copies of Wg and Wu, of Wd (WeightView::aligned)
};

// Offsets of the workspace's parts.
struct MoeWorkspace {
    size_t logits, picks, shares, h, total;
};
__host__ __device__ inline int moe_h_pitch(int inter) { return (inter + kTileRows - 1) / kTileRows * kTileRows; }
__host__ __device__ inline MoeWorkspace moe_workspace(int tokens, int experts, int topk, int inter) {
    MoeWorkspace m;
    m.logits = 256;  // the sync words before it
    m.picks = m.logits + size_t(tokens) * experts * 8;
    m.shares = m.picks + size_t(tokens) * topk * 4;
    m.h = (m.shares + size_t(tokens) * topk * 4 + 255) / 256 * 256;
    m.total = m.h + size_t(tokens) * topk * moe_h_pitch(inter) * 2;
    return m;
}

// What every CTA derives from the selection.
struct MoeRoute {
    int active;                                // experts with a token
    float share[kMoeMaxTokens * kMoeMaxTopk];  // [token, place]: the expert's weight
    short pick[kMoeMaxTokens * kMoeMaxTopk];   // [token, place]: the expert
    short act[kMoeMaxTokens * kMoeMaxTopk];    // [token, place]: its index among the active
    short row[kMoeMaxTokens * kMoeMaxTopk];    // [token, place]: its row of h
    short count[kMoeMaxExperts];               // tokens of each expert
    short expert[kMoeMaxExperts];              // active experts, ascending
    short start[kMoeMaxExperts + 1];           // first row of h of each active expert, and the end
    unsigned char token[kMoeMaxTokens * kMoeMaxTopk];  // token of each row of h
};

template <typename T, bool MX, int NT>
struct MoeShape {
    static constexpr int kPerSm = NT <= 2 ? 2 : 1;  // CTAs of an SM
    static constexpr int kGateStages = NT <= 2 ? 4 : 6;
    using Gate = WarpStream<T, MX, 2, NT, kGateStages>;
    using Down = WarpStream<T, MX, 1, NT, 2 * kGateStages>;
    static constexpr size_t kRing = size_t(Gate::kRing) * kMoeWarps;
    static constexpr int kPart = 2 * NT * 8 * kPartPitch;  // floats of a warp
    static constexpr size_t kPartBytes = size_t(kMoeWarps) * kPart * 4;
    static constexpr size_t kSmem = kRing + kPartBytes + (sizeof(MoeRoute) + 15) / 16 * 16;
    static_assert(int(Down::kRing) <= int(Gate::kRing), "one ring serves both phases");
    static_assert(kSmem + 1024 <= 233472 / kPerSm && kSmem <= 232448 - 1024, "shared memory");
};

__device__ __forceinline__ uint32_t moe_ld_acquire(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// Grid barrier over one word whose low 31 bits are zero between barriers: CTA 0 adds
// what the others' ones leave to 2^31, so the top bit flips once everybody arrived.
// Waits at most kWaitLimitNs; false (in every thread of the CTA) when it gave up.
__device__ __forceinline__ bool moe_grid_barrier(uint32_t* word, int* ok) {
    __syncthreads();
    if (threadIdx.x == 0) {
        *ok = 1;
        __threadfence();
        const uint32_t add = blockIdx.x == 0 ? 0x80000000u - uint32_t(gridDim.x - 1) : 1u;
        const uint32_t seen = atomicAdd(word, add) & 0x80000000u;
        const uint64_t t0 = global_timer_ns();
        while ((moe_ld_acquire(word) & 0x80000000u) == seen) {
            if (global_timer_ns() - t0 > kWaitLimitNs) {
                atomicOr(&g_device_error, 1);
                *ok = 0;
                break;
            }
        }
        __threadfence();
    }
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

// One warp selects a token's experts from its logits.
template <typename T>
__device__ void moe_select(const MoeParams& P, int token, int lane) {
    const double* l = P.logits + size_t(token) * P.experts;
    constexpr int kPer = kMoeMaxExperts / 32;
    double v[kPer];
    uint32_t left = 0;  // which of this lane's logits are still in play
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        v[i] = 0.0;
        if (e < P.experts) {
            v[i] = __ldcg(l + e);
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
        const int at = token * P.topk + lane;
        const float share = e / sum;
        P.picks[at] = pick;
        P.shares[at] = share;
        if (P.ids) P.ids[at] = pick;
        if (P.weights) P.weights[at] = share;
    }
}

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
        for (int k = threadIdx.x * 8; k < P.hidden; k += kMoeThreads * 8) {
            uint4 wv[kRouteExperts], xv[kRouteTokens];
#pragma unroll
            for (int a = 0; a < kRouteExperts; ++a)
                wv[a] = load_piece<T>(r + size_t(min(e0 + a, P.experts - 1)) * P.hidden, k, P.hidden, P.router_aligned);
#pragma unroll
            for (int b = 0; b < kRouteTokens; ++b)
                xv[b] = load_piece<T>(x + (t0 + min(b, nt - 1)) * P.x_pitch, k, P.hidden, P.x_aligned);
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
                if (lane == 0) scratch[(a * kRouteTokens + b) * kMoeWarps + warp] = sum[a][b];
            }
        __syncthreads();
        if (threadIdx.x < kRouteExperts * kRouteTokens) {
            const int a = threadIdx.x / kRouteTokens, b = threadIdx.x % kRouteTokens;
            if (e0 + a < P.experts && b < nt) {
                double s = 0.0;
                for (int j = 0; j < kMoeWarps; ++j) s += scratch[(a * kRouteTokens + b) * kMoeWarps + j];
                P.logits[size_t(t0 + b) * P.experts + e0 + a] = s;
            }
            __threadfence();
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            *flag = atomicAdd(P.sync + 1 + group, 1u) == uint32_t(expert_units - 1);
            if (*flag) {
                P.sync[1 + group] = 0u;  // for the next call
                __threadfence();
            }
        }
        __syncthreads();
        if (*flag && warp < nt) moe_select<T>(P, t0 + warp, lane);
        __syncthreads();
    }
}

// Lists of each expert's tokens, in token order, the same in every CTA.
__device__ inline void moe_lists(const MoeParams& P, MoeRoute& R) {
    const int n = P.tokens * P.topk, t = threadIdx.x;
    for (int i = t; i < n; i += kMoeThreads) {
        R.pick[i] = short(__ldcg(P.picks + i));
        R.share[i] = __ldcg(P.shares + i);
    }
    __syncthreads();
    int mine = 0;
    if (t < P.experts)
        for (int i = 0; i < n; ++i) mine += R.pick[i] == t;
    R.count[t] = mine;
    __syncthreads();
    if (t < 32) {  // eight experts a lane: sums of tokens and of active experts before them
        constexpr int kPer = kMoeMaxExperts / 32;
        int rows = 0, act = 0;
        for (int i = 0; i < kPer; ++i) {
            rows += R.count[t * kPer + i];
            act += R.count[t * kPer + i] > 0;
        }
        int row = rows, a = act;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int r = __shfl_up_sync(0xFFFFFFFFu, row, d), b = __shfl_up_sync(0xFFFFFFFFu, a, d);
            if (t >= d) row += r, a += b;
        }
        if (t == 31) {
            R.active = a;
            R.start[a] = row;
        }
        row -= rows;
        a -= act;
        for (int i = 0; i < kPer; ++i) {
            const int e = t * kPer + i;
            if (R.count[e] > 0) {
                R.expert[a] = short(e);
                R.start[a++] = short(row);
            }
            row += R.count[e];
        }
    }
    __syncthreads();
    if (t < R.active) {
        const int e = R.expert[t];
        int row = R.start[t];
        for (int i = 0; i < n; ++i)
            if (R.pick[i] == e) {
                R.token[row] = static_cast<unsigned char>(i / P.topk);
                R.act[i] = short(t);
                R.row[i] = short(row++);
            }
    }
    __syncthreads();
}

// A tensor of experts' matrices [experts, rows, cols] as the copies see one of them.
template <bool MX>
__device__ __forceinline__ WeightView moe_view(int cols, int aligned) {
    WeightView v;
    v.blocks = MX ? int(mx_blocks(cols)) : 0;
    v.row_bytes = MX ? v.blocks * kMxBlockBytes : cols * 2;
    v.pitch = v.row_bytes;
    v.steps = (v.row_bytes + kStepBytes - 1) / kStepBytes;
    v.aligned = aligned != 0;
    return v;
}

template <typename T, bool MX, int NT>
__global__ void __launch_bounds__(kMoeThreads, MoeShape<T, MX, NT>::kPerSm) moe_kernel(const MoeParams P) {
    using S = MoeShape<T, MX, NT>;
    using Gate = typename S::Gate;
    using Down = typename S::Down;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ double scratch[kRouteExperts * kRouteTokens * kMoeWarps];
    __shared__ int flag;
    float* part = reinterpret_cast<float*>(smem + S::kRing);
    MoeRoute& R = *reinterpret_cast<MoeRoute*>(smem + S::kRing + S::kPartBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = gridDim.x, b = blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * Gate::kRing;

    moe_router<T>(P, scratch, &flag);
    if (!moe_grid_barrier(P.sync, &flag)) return;
    moe_lists(P, R);

    T* h = static_cast<T*>(P.h);
    {
        const WeightView v = moe_view<MX>(P.hidden, P.gate_aligned);
        const int tiles = (P.inter + kTileRows - 1) / kTileRows;
        const int all = R.active * tiles;
        const int first = int((long long)b * all / G), mine = int((long long)(b + 1) * all / G) - first;
        const int rounds = round_count(mine, kMoeWarps);
        const T* x = static_cast<const T*>(P.x);
        auto get = [&](int i, Piece<T, 2, NT>& p) {
            if (i >= rounds) return false;
            const Round r = round_at(i, mine, kMoeWarps);
            const int share = kMoeWarps / r.items, part_of = warp % share;
            const int item = first + r.first + warp / share;
            const int a = item / tiles, row = item % tiles * kTileRows;
            const int e = R.expert[a], start = R.start[a];
            p.count = R.start[a + 1] - start;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                p.x[n] = x + R.token[start + min(n * 8 + (lane >> 2), p.count - 1)] * P.x_pitch;
            const int64_t base = int64_t(e) * P.inter + row;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                p.rows[m] = P.inter - row;
                p.w[m] = P.w[m] + base * v.pitch;
                p.s[m] = P.s[m] + base * v.blocks;
            }
            p.s0 = v.steps * part_of / share;
            p.s1 = v.steps * (part_of + 1) / share;
            return true;
        };
        auto done = [&](int i, const Piece<T, 2, NT>& p, const float (&acc)[2][NT][4]) {
            const Round r = round_at(i, mine, kMoeWarps);
            const int share = kMoeWarps / r.items;
            __syncthreads();  // the last round's sums are read
            store_partial<2, NT>(part + warp * S::kPart, acc, p.count, lane);
            __syncthreads();
            for (int c = threadIdx.x; c < r.items * kTileRows * NT * 8; c += kMoeThreads) {
                const int row16 = c & 15, n = (c >> 4) % (NT * 8), idx = (c >> 4) / (NT * 8);
                const int item = first + r.first + idx;
                const int a = item / tiles, row = item % tiles * kTileRows + row16;
                const int start = R.start[a];
                if (n >= R.start[a + 1] - start) continue;
                const float* q = part + idx * share * S::kPart + n * kPartPitch + row16;
                float g = 0.f, u = 0.f;
                for (int j = 0; j < share; ++j) {
                    g += q[j * S::kPart];
                    u += q[j * S::kPart + NT * 8 * kPartPitch];
                }
                // rows up to the pitch of h are zero, so that a whole piece of h may be read
                h[int64_t(start + n) * P.h_pitch + row] = Num<T>::from_float(row < P.inter ? silu(g) * u : 0.f);
            }
        };
        Gate::run(ring, v, P.hidden, P.x_aligned != 0, get, done);
    }
    if (!moe_grid_barrier(P.sync, &flag)) return;

    {
        const WeightView v = moe_view<MX>(P.inter, P.down_aligned);
        const int tiles = (P.hidden + kTileRows - 1) / kTileRows;
        const int first = int((long long)b * tiles / G), mine = int((long long)(b + 1) * tiles / G) - first;
        const int per_tile = round_count(R.active, kMoeWarps), rounds = mine * per_tile;
        T* y = static_cast<T*>(P.y);
        float* total = reinterpret_cast<float*>(part) + kMoeWarps * (NT * 8 * kPartPitch);  // [tokens][16]
        auto get = [&](int i, Piece<T, 1, NT>& p) {
            if (i >= rounds) return false;
            const Round r = round_at(i % per_tile, R.active, kMoeWarps);
            const int share = kMoeWarps / r.items, part_of = warp % share;
            const int a = r.first + warp / share, row = (first + i / per_tile) * kTileRows;
            const int start = R.start[a];
            p.count = R.start[a + 1] - start;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                p.x[n] = h + int64_t(start + min(n * 8 + (lane >> 2), p.count - 1)) * P.h_pitch;
            const int64_t base = int64_t(R.expert[a]) * P.hidden + row;
            p.rows[0] = P.hidden - row;
            p.w[0] = P.w[2] + base * v.pitch;
            p.s[0] = P.s[2] + base * v.blocks;
            p.s0 = v.steps * part_of / share;
            p.s1 = v.steps * (part_of + 1) / share;
            return true;
        };
        auto done = [&](int i, const Piece<T, 1, NT>& p, const float (&acc)[1][NT][4]) {
            constexpr int kPart = NT * 8 * kPartPitch;
            const int turn = i % per_tile;
            const Round r = round_at(turn, R.active, kMoeWarps);
            const int share = kMoeWarps / r.items;
            __syncthreads();  // the last round's sums are read
            store_partial<1, NT>(part + warp * kPart, acc, p.count, lane);
            __syncthreads();
            for (int c = threadIdx.x; c < P.tokens * kTileRows; c += kMoeThreads) {
                const int row16 = c & 15, t = c >> 4;
                float sum = turn == 0 ? 0.f : total[c];
                for (int j = 0; j < P.topk; ++j) {
                    const int at = t * P.topk + j, idx = R.act[at] - r.first;
                    if (idx < 0 || idx >= r.items) continue;
                    const int n = R.row[at] - R.start[R.act[at]];
                    const float* q = part + idx * share * kPart + n * kPartPitch + row16;
                    float d = 0.f;
                    for (int w = 0; w < share; ++w) d += q[w * kPart];
                    sum = fmaf(R.share[at], d, sum);
                }
                total[c] = sum;
                const int row = (first + i / per_tile) * kTileRows + row16;
                if (turn == per_tile - 1 && row < P.hidden) y[int64_t(t) * P.hidden + row] = Num<T>::from_float(sum);
            }
        };
        Down::run(ring, v, P.h_pitch, true, get, done);
    }
}

}  // namespace swb
