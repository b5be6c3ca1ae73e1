// The mixture-of-experts layer's tensor-core kernels (moe_wide.cu).
#pragma once

#include <cuda_runtime.h>

namespace swb {

struct MoeParams;

// Whether those kernels take the call: more than a few tokens, rows that their copies can bring.
bool moe_wide_takes(const MoeParams& P, bool mx);
int moe_wide(int type, bool mx, const MoeParams& P, cudaStream_t stream);

}  // namespace swb
