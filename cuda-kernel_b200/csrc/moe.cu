// C entry points of the mixture-of-experts layer (declarations: include/swiglu_b200.h).
#include "moe.cuh"

#include <algorithm>
#include <cstring>

#include "host.h"
#include "moe_wide.h"

namespace swb {

int moe_device_error(int clear, int* out) {
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

static_assert(SWB_MOE_MAX_TOKENS == kMoeMaxTokens && SWB_MOE_MAX_EXPERTS == kMoeMaxExperts &&
                  SWB_MOE_MAX_TOPK == kMoeMaxTopk,
              "the header's limits");
static_assert(1 + (kMoeMaxTokens + kRouteTokens - 1) / kRouteTokens <= kSyncTurn && kSyncTurn < 64, "sync words fit");

template <typename T, bool MX, int NT>
int launch_moe(MoeParams P, cudaStream_t stream) {
    using S = MoeShape<T, MX, NT>;
    static std::atomic<uint64_t> smem_set{0};
    const int sms = sm_count();
    if (sms <= 0) return check_launch();
    auto kernel = moe_kernel<T, MX, NT>;
    if (int rc = allow_smem(kernel, smem_set, S::kSmem)) return rc;
    static_assert(S::kStages >= 3, "a ring");
    MoeMaps maps;
    bool fast[3], deep[3];
    for (int i = 0; i < 3; ++i) {
        const int64_t rows = int64_t(P.experts) * (i < 2 ? P.inter : P.hidden), cols = i < 2 ? P.hidden : P.inter;
        const int64_t blocks = mx_blocks(cols), pitch = MX ? blocks * kMxBlockBytes : cols * 2;
        if (int rc = make_weight_maps(&maps.m[i], P.w[i], MX ? P.s[i] : nullptr, rows, pitch, blocks, &fast[i], &deep[i]))
            return rc;
    }
    // one way of reading for the copies and the consumers of a phase
    P.fast[0] = fast[0] && fast[1] && P.x_aligned;
    P.fast[1] = fast[2];
    P.deep[0] = deep[0];
    P.deep[1] = deep[2];
    // every CTA resident at once: the cooperative launch makes the runtime check it
    return launch_ex(kernel, unsigned(sms), S::Pipe::kThreads, S::kSmem, stream, true, maps, P);
}

template <typename T>
int dispatch_moe(bool mx, const MoeParams& P, cudaStream_t stream) {
    // four-bit experts come here with up to eight tokens only (moe_wide_takes)
    if (mx) return launch_moe<T, true, 1>(P, stream);
    // an expert can be given every token; beyond 32 in groups of 32
    if (P.tokens <= 8) return launch_moe<T, false, 1>(P, stream);
    if (P.tokens <= 16) return launch_moe<T, false, 2>(P, stream);
    return launch_moe<T, false, 4>(P, stream);
}

}  // namespace
}  // namespace swb

using namespace swb;

extern "C" {

size_t swb_moe_workspace_bytes(int tokens, int experts, int topk, int inter) {
    if (tokens < 0 || tokens > SWB_MOE_MAX_TOKENS || experts <= 0 || experts > SWB_MOE_MAX_EXPERTS || topk <= 0 ||
        topk > SWB_MOE_MAX_TOPK || topk > experts || inter <= 0 || inter > SWB_MOE_MAX_DIM)
        return 0;
    return moe_workspace(tokens, experts, topk, inter).total;
}

int swb_moe(int type, unsigned flags, const void* x, int64_t x_pitch, const void* router, const void* gate,
            const void* up, const void* down, const void* gate_scales, const void* up_scales, const void* down_scales,
            void* y, int* ids, float* weights, int tokens, int hidden, int inter, int experts, int topk,
            void* workspace, size_t workspace_bytes, void* stream) {
    if (type != SWB_F16 && type != SWB_BF16) return fail(SWB_E_TYPE);
    if (flags & ~(SWB_MOE_MX4 | SWB_MOE_RENORMALIZE)) return fail(SWB_E_INPUT, "unknown flags");
    const bool mx = (flags & SWB_MOE_MX4) != 0;
    if (tokens < 0 || tokens > SWB_MOE_MAX_TOKENS || hidden <= 0 || hidden > SWB_MOE_MAX_DIM || inter <= 0 ||
        inter > SWB_MOE_MAX_DIM || experts <= 0 || experts > SWB_MOE_MAX_EXPERTS || topk <= 0 ||
        topk > SWB_MOE_MAX_TOPK || topk > experts || x_pitch < hidden)
        return fail(SWB_E_SHAPE);
    if (tokens == 0) return SWB_OK;
    if (!x || !router || !gate || !up || !down) return fail(SWB_E_INPUT);
    if (mx && (!gate_scales || !up_scales || !down_scales)) return fail(SWB_E_INPUT, "missing scales");
    if (!y) return fail(SWB_E_HALF_OUTPUT);
    const MoeWorkspace w = moe_workspace(tokens, experts, topk, inter);
    if (!workspace || workspace_bytes < w.total) return fail(SWB_E_WORKSPACE, "swb_moe workspace too small");
    if (!aligned(256, workspace)) return fail(SWB_E_ALIGNMENT, "workspace must be 256-byte aligned");
    if (!aligned(mx ? 16 : 2, gate, up, down))
        return fail(SWB_E_ALIGNMENT, mx ? "codes must be 16-byte aligned" : "values off their type's size");
    if (!aligned(2, x, router, y) || !aligned(4, ids, weights)) return fail(SWB_E_ALIGNMENT, "values off their type's size");
    // what the call writes may not overlap what it reads, nor each other
    const size_t n = size_t(experts) * hidden * inter;
    const size_t gate_blocks = size_t(experts) * inter * mx_blocks(hidden);
    const size_t down_blocks = size_t(experts) * hidden * mx_blocks(inter);
    const struct { const void* p; size_t bytes; } in[] = {
        {x, (size_t(tokens - 1) * x_pitch + hidden) * 2},
        {router, size_t(experts) * hidden * 2},
        {gate, mx ? gate_blocks * kMxBlockBytes : n * 2},
        {up, mx ? gate_blocks * kMxBlockBytes : n * 2},
        {down, mx ? down_blocks * kMxBlockBytes : n * 2},
        {mx ? gate_scales : nullptr, gate_blocks},
        {mx ? up_scales : nullptr, gate_blocks},
        {mx ? down_scales : nullptr, down_blocks},
    };
    const size_t picks = size_t(tokens) * topk * 4;
    const struct { const void* p; size_t bytes; } out[] = {
        {workspace, w.total}, {y, size_t(tokens) * hidden * 2}, {ids, picks}, {weights, picks}};
    for (int i = 0; i < 4; ++i) {
        if (!out[i].p) continue;
        for (const auto& a : in)
            if (a.p && overlaps(out[i].p, out[i].bytes, a.p, a.bytes)) return fail(SWB_E_OVERLAP_INPUT);
        for (int j = 0; j < i; ++j)
            if (out[j].p && overlaps(out[i].p, out[i].bytes, out[j].p, out[j].bytes)) return fail(SWB_E_OVERLAP_OUTPUT);
    }
    MoeParams P;
    std::memset(&P, 0, sizeof P);
    auto* base = static_cast<unsigned char*>(workspace);
    P.x = x;
    P.router = router;
    const void* ws[3] = {gate, up, down};
    const void* ss[3] = {gate_scales, up_scales, down_scales};
    for (int i = 0; i < 3; ++i) {
        P.w[i] = static_cast<const unsigned char*>(ws[i]);
        P.s[i] = static_cast<const unsigned char*>(ss[i]);
    }
    P.y = y;
    P.ids = ids;
    P.weights = weights;
    P.sync = reinterpret_cast<uint32_t*>(base);
    P.tops = reinterpret_cast<uint32_t*>(base + w.tops);
    P.logits = reinterpret_cast<double*>(base + w.logits);
    P.picks = reinterpret_cast<int*>(base + w.picks);
    P.shares = reinterpret_cast<float*>(base + w.shares);
    P.h = base + w.h;
    P.pieces = base + w.pieces;
    P.x_pitch = x_pitch;
    P.tokens = tokens;
    P.hidden = hidden;
    P.inter = inter;
    P.experts = experts;
    P.topk = topk;
    P.group = kMoeGroup;
    P.h_pitch = moe_h_pitch(inter);
    P.renormalize = (flags & SWB_MOE_RENORMALIZE) != 0;
    P.x_aligned = hidden % 8 == 0 && x_pitch % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    P.router_aligned = hidden % 8 == 0 && reinterpret_cast<uintptr_t>(router) % 16 == 0;
    auto s = static_cast<cudaStream_t>(stream);
    if (moe_wide_takes(P, mx)) return moe_wide(type, mx, P, s);
    return type == SWB_F16 ? dispatch_moe<__half>(mx, P, s) : dispatch_moe<__nv_bfloat16>(mx, P, s);
}

}  // extern "C"
