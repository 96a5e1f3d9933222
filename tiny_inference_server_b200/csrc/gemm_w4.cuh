// What the kernels of products with weights of four bits share.
#pragma once
#include "common.cuh"

constexpr int W4_STRIP = 16, W4_CHUNK = 64;

struct W4Params {
    const uint4* words; const unsigned* scales; const unsigned short* zeros;
    const void* x; long long ldx;
    void* out; long long ldo;
    int rows, K, N, chunks, strips, groups, group_shift;      // group_shift: log2 of the halves of a chunk in a group
    int ws, wk, stage_chunks, stages;
    bool f32, vectors;
};

// two codes (bits 0-3 and 16-19 of w) less their zero point; `base` is 128 + zero in both halves
__device__ __forceinline__ unsigned w4_pair(unsigned w, unsigned base) {
    const unsigned v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&base));
    return *reinterpret_cast<const unsigned*>(&d);
}
// One float as three bfloat16 numbers, x = v0 + 2^-8 v1 + 2^-16 v2, exactly: its top eight bits, the next eight and the last eight.  The lower two are
// kept 2^8 and 2^16 times as large (at most twice x): as they are, those of a number below 2^-110 would reach under bfloat16's smallest, 2^-133.
__device__ __forceinline__ void three(float x, unsigned short (&v)[3]) {
    const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    const float rest = fabsf(x) < INFINITY ? (x - hi) * 256.f : 0.f;
    const float mid = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
    v[0] = x != x ? 0x7fc0 : (unsigned short)(__float_as_uint(hi) >> 16);
    v[1] = (unsigned short)(__float_as_uint(mid) >> 16);
    v[2] = (unsigned short)(__float_as_uint((rest - mid) * 256.f) >> 16);
}
// and the sums of their products back in one, the small ones first
__device__ __forceinline__ float of_three(float v0, float v1, float v2) { return fmaf(fmaf(v2, 0x1p-8f, v1), 0x1p-8f, v0); }

// gemm_w4_tc.cu.  `copy` (null: x is bfloat16 in rows that start on 16 bytes): room for x's rows in bfloat16, (K + 7) / 8 * 8 entries each, three for
// one of float32.
constexpr int W4_TC_ROWS = 64, W4_TC_ROWS_F32 = 21;      // of a launch
int w4_tc_launch(const W4Params& p, void* copy, int* fault, cudaStream_t stream);
