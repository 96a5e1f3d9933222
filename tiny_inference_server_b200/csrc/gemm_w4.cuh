// What the kernels of products with weights of four bits share.
#pragma once
#include "common.cuh"

constexpr int W4_STRIP = 16, W4_CHUNK = 64;

struct W4Params {
    const uint4* words; const unsigned* scales; const unsigned short* zeros;
    const void* x; long long ldx;
    void* out; long long ldo;
    int rows, slab, K, N, chunks, strips, groups, group_shift;      // group_shift: log2 of the halves of a chunk in a group
    int ws, wk, stage_chunks, stages;
    bool f32, vectors;
};

// two codes (bits 0-3 and 16-19 of w) less their zero point; `base` is 128 + zero in both halves
__device__ __forceinline__ unsigned w4_pair(unsigned w, unsigned base) {
    const unsigned v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&base));
    return *reinterpret_cast<const unsigned*>(&d);
}
// gemm_w4_tc.cu: x in bfloat16 (`x_rows` rows; for float32 three of them, one after another, are a row), rows that start on 16 bytes
int w4_tc_launch(const W4Params& p, const void* x, int x_rows, long long ldx, int* fault, cudaStream_t stream);
