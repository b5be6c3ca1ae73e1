// Arguments of the product of a four-bit matrix with 16-bit tokens, shared by its kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace swb {

struct ProjectParams {
    const unsigned char* w;
    const unsigned char* s;
    const void* x;
    const void* bias;
    const void* residual;
    void* out;
    int64_t x_pitch, tokens;
    int rows, cols;
    int tiles;       // of rows
    int64_t items;   // tiles x groups of tokens
    bool x_aligned;  // 16-byte pieces of x
    bool half_out;
};

// Few tokens, split into e4m3 pieces (mx4_wide.cu).
int project_wide(int type, ProjectParams P, cudaStream_t stream);
// More tokens, W decoded into 16-bit tiles (mx4_deep.cu): takes tokens on 16 bytes.
bool project_deep_takes(const ProjectParams& P);
int project_deep(int type, const ProjectParams& P, cudaStream_t stream);

}  // namespace swb
