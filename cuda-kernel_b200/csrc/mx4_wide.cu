// The product of a four-bit matrix with 16-bit tokens on the tensor cores (wide.cuh).
//
// Bound by the bytes of W for few tokens. A CTA takes 128 rows by up to 64 tokens; where that
// leaves SMs without work the CTAs of a cluster split K and add their parts through each other's
// shared memory in rank order. Up to 16 tokens two CTAs share an SM, so that one's first bytes and
// exchange run beside the other's stream.
// 14336 x 4096, one token: 16.6 us for 31 MB, 4.8 at the copy rate; about half is launch, first
// bytes and exchange, the rest 16 stages a CTA, each a chain of waits, spreading and a product.
#include <algorithm>
#include <cstring>

#include "host.h"
#include "project.h"
#include "wide.cuh"

namespace swb {

int mx4_wide_device_error(int clear, int* out) {
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

template <typename T_, int TOK>
struct ProjectWork {
    using T = T_;
    static constexpr bool kMx = true, kLoad = true, kFloat = false, kGather = false;
    static constexpr int kPieces = std::is_same<T, __half>::value ? 3 : 2;
    static constexpr int kTok = TOK, kAccs = 1;
    static constexpr int kPerSm = TOK == 16 ? 2 : 1;
    static constexpr int kStages = TOK == 16 ? 2 : 4, kRaw = TOK == 16 ? 3 : 4;
    static constexpr int kSpreadGroups = 1, kTokenStages = TOK == 16 ? 4 : TOK == 32 ? 6 : 2;
    static constexpr int kSplitters = TOK == 16 ? 4 : TOK == 32 ? 6 : 8, kGroupWarps = TOK == 64 ? 4 : 1;

    const unsigned char* sa[2];
    int blocks, cols;
    int64_t rows_a;
    bool x_aligned;
    const T* x;
    int64_t x_pitch;
    int halves;
    WideItem only;
    int64_t token0;
    uint32_t part;  // [token][kWidePartPitch]

    __device__ __forceinline__ bool item(int i, WideItem& it) const {
        it = only;
        return i == 0;
    }
    __device__ __forceinline__ const T* token(const WideItem&, int n) const { return x + (token0 + n) * x_pitch; }
    __device__ __forceinline__ void begin(const WideItem&) const {}
    __device__ __forceinline__ void value(const WideItem&, int n, int row, float v) const {
        sts32(part + (n * kWidePartPitch + row) * 4, __float_as_uint(v));
    }
    __device__ __forceinline__ void end(const WideItem&) const {}
};

template <typename T, int TOK>
struct ProjectWide {
    using Pipe = Wide<ProjectWork<T, TOK>>;
    static constexpr size_t kSmem = Pipe::kRing + 1024;  // the parts reuse the ring
    static_assert(TOK * kWidePartPitch * 4 <= Pipe::kRing, "the parts fit the ring");
    static_assert((kSmem + 2048) * ProjectWork<T, TOK>::kPerSm <= kSmemPerSm, "CTAs of an SM share its memory");
};

template <typename T, int TOK>
__global__ void __launch_bounds__(Wide<ProjectWork<T, TOK>>::kThreads, ProjectWork<T, TOK>::kPerSm)
    project_wide_kernel(const __grid_constant__ CUtensorMap map, const ProjectParams P, int splits, int steps) {
    using Work = ProjectWork<T, TOK>;
    using Pipe = Wide<Work>;
    constexpr int kWideThreads = Pipe::kThreads;
    extern __shared__ unsigned char raw[];
    __shared__ typename Pipe::Shared sh;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const int rank = int(blockIdx.x % splits);
    const int64_t item = blockIdx.x / splits;
    const int64_t row0 = item % P.tiles * kWideM, token0 = item / P.tiles * TOK;

    Work work;
    work.sa[0] = work.sa[1] = P.s;
    work.halves = 2;
    work.blocks = int(mx_blocks(P.cols));
    work.cols = P.cols;
    work.rows_a = P.rows;
    work.x_aligned = P.x_aligned;
    work.x = static_cast<const T*>(P.x);
    work.x_pitch = P.x_pitch;
    work.token0 = token0;
    work.part = base;
    work.only.row[0] = row0;
    work.only.row[1] = row0 + kWideHalf;
    work.only.s0 = int(int64_t(steps) * rank / splits);
    work.only.s1 = int(int64_t(steps) * (rank + 1) / splits);
    work.only.count = int(min(int64_t(TOK), P.tokens - token0));
    work.only.first = 0;

    Pipe::init(sh);
    __syncthreads();
    // W is read once unless more tokens follow
    const uint64_t policy = P.tokens > TOK ? l2_normal_policy() : l2_evict_first_policy();
    Pipe::run(work, sh, base, &map, &map, &map, policy);
    __syncthreads();
    Pipe::finish(sh);

    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    if (!sh.failed) {
        const int count = work.only.count * kWideM;
        for (int i = rank * kWideThreads + threadIdx.x; i < count; i += splits * kWideThreads) {
            const int t = i / kWideM, r = i % kWideM;
            const int64_t row = row0 + r, at = (token0 + t) * P.rows + row;
            if (row >= P.rows) continue;
            float v = 0.f;
            for (int j = 0; j < splits; ++j) {
                uint32_t remote;
                float f;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(base + (t * kWidePartPitch + r) * 4), "r"(j));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(remote) : "memory");
                v += f;
            }
            if (P.bias) v += Num<T>::to_float(static_cast<const T*>(P.bias)[row]);
            if (P.residual) v += Num<T>::to_float(static_cast<const T*>(P.residual)[at]);
            if (P.half_out)
                static_cast<T*>(P.out)[at] = Num<T>::from_float(v);
            else
                static_cast<float*>(P.out)[at] = v;
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, int TOK>
int launch_wide(ProjectParams P, cudaStream_t stream) {
    using Shape = ProjectWide<T, TOK>;
    static std::atomic<uint64_t> smem_set{0};
    const int sms = sm_count();
    if (sms <= 0) return check_launch();
    auto kernel = project_wide_kernel<T, TOK>;
    if (int rc = allow_smem(kernel, smem_set, Shape::kSmem)) return rc;
    CUtensorMap map;
    if (int rc = make_wide_map(&map, P.w, P.rows, P.cols, true)) return rc;
    P.tiles = (P.rows + kWideM - 1) / kWideM;
    P.items = int64_t(P.tiles) * ((P.tokens + TOK - 1) / TOK);
    const int steps = int((mx_blocks(P.cols) + 3) / 4), slots = sms * ProjectWork<T, TOK>::kPerSm;
    // every SM streams: split K until the CTAs fill the GPU, down to four steps each
    int splits = 1;
    while (splits < 8 && P.items * splits * 2 <= slots && steps / (splits * 2) >= 4) splits *= 2;
    if (P.items * splits > 0x7FFFFFFF) return fail(SWB_E_SHAPE);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(P.items * splits));
    cfg.blockDim = dim3(Shape::Pipe::kThreads);
    cfg.dynamicSmemBytes = Shape::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map, P, splits, steps);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(SWB_E_CUDA, cudaGetErrorString(e));
    }
    return SWB_OK;
}

template <typename T>
int dispatch_wide(const ProjectParams& P, cudaStream_t stream) {
    if (P.tokens <= 16) return launch_wide<T, 16>(P, stream);
    if (P.tokens <= 32) return launch_wide<T, 32>(P, stream);
    return launch_wide<T, 64>(P, stream);
}

}  // namespace

int project_wide(int type, ProjectParams P, cudaStream_t stream) {
    return type == SWB_F16 ? dispatch_wide<__half>(P, stream) : dispatch_wide<__nv_bfloat16>(P, stream);
}

}  // namespace swb
