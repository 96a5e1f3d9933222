// Attention of rows whose requests share the first keys and values of the paged cache.
//
// A tile is up to 16 (or 64, or 128) "row heads" (row, query head) of one kv head, counted row by row, the G heads of a row one after
// another, and a range of keys:
//   shared tiles  row heads of all requests of a group, keys [0, shared): read once for all of them, through the table of one;
//   own tiles     row heads of one request, keys [shared, position] of its own, each row up to its position.
// A tile's keys are split into parts; a part leaves its share of the softmax, in 32 bits: m, the largest score (in units of log2), l, the
// sum of 2^(score - m), and o, the sum of 2^(score - m) v.  With M the largest m of a row's parts, its result is
// sum 2^(m - M) o / sum 2^(m - M) l, parts in a fixed order.
#pragma once
#include "common.cuh"

// rh0, count: its row heads; slot: whose table; prefix: the group's shared keys (not yet cut to whole pages)
struct SharedTile { int rh0, count, slot, prefix; };

struct SharedParams {
    const void* q; long long ldq;                 // (rows, >= H * hd), queries first
    const void* plane;                            // [pages, 2, KVH, page, hd]
    const int* table; int table_stride, table_width, num_pages;
    const int* positions;
    float* part_o;                                // [parts][rows][H][hd]
    float2* part_ml;                              // [parts][rows][H]
    int rows, H, KVH, page, own_parts, shared_parts;
    void* out; long long ldo; bool out_vectors;   // results; whether their rows start on 16 bytes
    float scale_log2;
    int* fault;
};

namespace shared_attention {

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// Whole pages of the group's shared keys.
__device__ __forceinline__ int shared_keys(const SharedParams& p, const SharedTile& t) { return t.prefix / p.page * p.page; }

// The page of a logical page of a request; one that is not there is marked, and read as page 0.
__device__ __forceinline__ int page_at(const SharedParams& p, int slot, int index) {
    int page = index < p.table_width ? p.table[(size_t)slot * p.table_stride + index] : -1;
    if (page < 0 || page >= p.num_pages) {
        atomicExch(p.fault, 3);
        page = 0;
    }
    return page;
}

// Keys [lo, hi) of part `part` of `parts`, cut at multiples of `step` counted from `base` (a multiple of it at or below the first key).
struct Range { int lo, hi; };
__device__ __forceinline__ Range part_range(int first, int last, int base, int part, int parts, int step) {
    const int steps = last > base ? (last - base + step - 1) / step : 0;
    const int per = (steps + parts - 1) / parts;
    Range r;
    r.lo = max(first, base + part * per * step);
    r.hi = min(last, base + (part + 1) * per * step);
    return r;
}

}  // namespace shared_attention
