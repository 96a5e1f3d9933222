// Attention over a shared prefix (shared_attention.cuh): the kernel of the requests' own keys, also of shared keys at head sizes
// and pages that the tcgen05 kernel does not take; the float32 kernel; and the kernel that joins the parts.
//
// The first is bound by the keys' and values' bytes (a request's own keys serve its own few row heads only) or, with few of them, by the
// chain position -> page -> row -> product.  Rows of the cache come by cp.async, 64 keys a tile, STAGES tiles ahead, into shared
// memory as they are stored (their permuted chunks are free of bank conflicts for ldmatrix).  Four warps: with at most 16 row heads each
// takes a quarter of every tile's keys and they merge at the end; with up to 64 each takes 16 row heads and all keys.
#include "shared_attention.cuh"

#ifndef TIS_HD
#define TIS_HD 128
#endif

namespace {

using namespace shared_attention;

constexpr int HD = TIS_HD;
constexpr unsigned ALL = 0xffffffffu;

__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], const void* smem) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((unsigned)__cvta_generic_to_shared(smem)));
}
__device__ __forceinline__ void ldmatrix4_trans(unsigned (&r)[4], const void* smem) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((unsigned)__cvta_generic_to_shared(smem)));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}

constexpr int KT = 64;                       // keys of a tile
constexpr int CHUNKS = HD / 8;               // 16-byte pieces of a row
constexpr int TILE_ELEMENTS = KT * HD;       // keys, or values
constexpr int STAGES = HD <= 64 ? 4 : (HD <= 128 ? 3 : 2);
constexpr int MMA_THREADS = 128;

// A tile's rows: position of row head rh0 + i (-1: beyond the tile, or before the end of the shared keys: it sees nothing)
__device__ __forceinline__ int position_of(const SharedParams& p, const SharedTile& t, int i) {
    if (i >= t.count) return -1;
    const int pos = p.positions[(t.rh0 + i) / (p.H / p.KVH)];
    return pos >= t.prefix ? pos : -1;
}

// Q row heads rh0 .. rh0 + n - 1 of kv head `kvh` into shared memory, rows of HD, chunk c of row i at c XOR / + i as a cache row
// of position i; zero beyond the tile.
__device__ __forceinline__ void load_queries(const SharedParams& p, const SharedTile& t, int kvh, int n, bf16* to) {
    const int G = p.H / p.KVH;
    for (int j = threadIdx.x; j < n * CHUNKS; j += MMA_THREADS) {
        const int i = j / CHUNKS, c = j % CHUNKS;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (i < t.count) {
            const int rh = t.rh0 + i, row = rh / G;
            v = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (long long)row * p.ldq + (kvh * G + rh % G) * HD + c * 8);
        }
        *reinterpret_cast<uint4*>(to + i * HD + cache_chunk(c, i, CHUNKS) * 8) = v;
    }
}

// OWN: own tiles (rows end at their positions), else shared ones.  WIDE: 64 row heads, 16 a warp; else 16, a quarter of the keys a warp.
template <bool OWN, bool WIDE>
__global__ void __launch_bounds__(MMA_THREADS)
shared_mma_kernel(const SharedParams p, const SharedTile* tiles, int parts, int part0) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    bf16* q_smem = reinterpret_cast<bf16*>(smem_raw);
    bf16* ring = q_smem + (WIDE ? 64 : 16) * HD;
    __shared__ int row_pos[64];
    __shared__ float merge_m[4][16], merge_l[4][16];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int kvh = blockIdx.x % p.KVH, part = blockIdx.x / p.KVH % parts;
    const SharedTile t = tiles[blockIdx.x / p.KVH / parts];
    const int G = p.H / p.KVH;
    pdl_wait();

    const int shared = shared_keys(p, t);
    int last = shared;                                      // keys [.., last) are seen by some row
    if (threadIdx.x < (WIDE ? 64 : 32)) {
        const int pos = threadIdx.x < (WIDE ? 64 : 16) ? position_of(p, t, threadIdx.x) : -1;
        row_pos[threadIdx.x] = pos;
    }
    __syncthreads();
    int least = 0x7fffffff;                                 // the smallest position of a row that sees anything
    bool any = false;
    for (int i = 0; i < (WIDE ? 64 : 16); ++i) {
        const int pos = row_pos[i];
        if (pos >= 0) { any = true; least = min(least, pos); if (OWN) last = max(last, pos + 1); }
    }
    const int base = OWN ? shared & ~(KT - 1) : 0;
    Range keys = part_range(OWN ? shared : 0, last, base, part, parts, KT);
    if (!any) keys.hi = keys.lo;
    const int kt0 = keys.lo & ~(KT - 1), count = keys.hi > keys.lo ? (keys.hi - kt0 + KT - 1) / KT : 0;

    load_queries(p, t, kvh, WIDE ? 64 : 16, q_smem);
    // keys and values of tile j: rows in [lo, hi), zero elsewhere
    auto stage = [&](int j) {
        if (j < count) {
            bf16* to = ring + (size_t)(j % STAGES) * 2 * TILE_ELEMENTS;
            for (int i = threadIdx.x; i < KT * CHUNKS; i += MMA_THREADS) {
                const int r = i / CHUNKS, c = i % CHUNKS, key = kt0 + j * KT + r;
                const bool in = key >= keys.lo && key < keys.hi;
                size_t at = 0;
                if (in) at = (((size_t)page_at(p, t.slot, key / p.page) * 2 * p.KVH + kvh) * p.page + key % p.page) * HD + c * 8;
                const bf16* k = static_cast<const bf16*>(p.plane) + at;
                const bf16* v = k + (in ? (size_t)p.KVH * p.page * HD : 0);
                const int bytes = in ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                             ::"r"((unsigned)__cvta_generic_to_shared(to + r * HD + c * 8)), "l"(k), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                             ::"r"((unsigned)__cvta_generic_to_shared(to + TILE_ELEMENTS + r * HD + c * 8)), "l"(v), "r"(bytes) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
#pragma unroll
    for (int j = 0; j < STAGES - 1; ++j) stage(j);

    // this lane's two row heads
    const int i0 = (WIDE ? warp * 16 : 0) + g, i1 = i0 + 8;
    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    for (int j = 0; j < count; ++j) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
        __syncthreads();                                    // tile j is here, tile j - 1's place is free
        stage(j + STAGES - 1);
        const bf16* ks = ring + (size_t)(j % STAGES) * 2 * TILE_ELEMENTS;
        bf16* vs = const_cast<bf16*>(ks) + TILE_ELEMENTS;
        const int kt = kt0 + j * KT;
        const int pos0 = row_pos[i0], pos1 = row_pos[i1];
        if (OWN && kt + KT - 1 > least) {
            // Behind the first row's position a key is seen by some rows and not by others, whose probability of 0 does not take away a
            // value that is not finite: such values go apart, and zeros into the products.  (Uniform in the CTA.)
            __shared__ int odd[KT];
            if (threadIdx.x < KT) odd[threadIdx.x] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < KT * CHUNKS; i += MMA_THREADS) {
                const int r = i / CHUNKS, key = kt + r;
                if (key > least && key < keys.hi) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vs + r * HD + i % CHUNKS * 8);
                    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u) odd[r] = 1;
                }
            }
            __syncthreads();
            for (int r = 0; r < KT; ++r) {
                if (!odd[r]) continue;
                // rows that see it have a result that is not finite there, whatever its probability (a positive number, or 0): the
                // products of a positive probability say so; a row that does not see it is left alone
                for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = n * 8 + t4 * 2 + (e & 1);
                        const float v = __bfloat162float(vs[r * HD + cache_chunk(d / 8, kt + r, CHUNKS) * 8 + d % 8]);
                        const bool sees = kt + r <= (e < 2 ? pos0 : pos1) && (WIDE || warp == 0);
                        if (sees && !(fabsf(v) < INFINITY)) o[n][e] += v;
                    }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < KT * CHUNKS; i += MMA_THREADS) {
                if (!odd[i / CHUNKS]) continue;
                unsigned short* w = reinterpret_cast<unsigned short*>(vs + i * 8);
                for (int e = 0; e < 8; ++e)
                    if ((w[e] & 0x7f80u) == 0x7f80u) w[e] = 0;
            }
            __syncthreads();
        }
#pragma unroll
        for (int b = 0; b < (WIDE ? KT / 16 : 1); ++b) {
            const int kb = (WIDE ? b : warp) * 16;          // 16 keys of the tile
            if (kt + kb >= keys.hi || kt + kb + 15 < keys.lo) continue;
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                unsigned a[4], bk[4];
                const int qr = (WIDE ? warp * 16 : 0) + (lane & 15);
                ldmatrix4(a, q_smem + qr * HD + cache_chunk(2 * k + (lane >> 4), qr, CHUNKS) * 8);
                const int kr = kb + (lane & 7) + (lane >> 4) * 8;
                ldmatrix4(bk, ks + kr * HD + cache_chunk(2 * k + ((lane >> 3) & 1), kt + kr, CHUNKS) * 8);
                mma(s[0], a, bk[0], bk[1]);
                mma(s[1], a, bk[2], bk[3]);
            }
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = kt + kb + n * 8 + t4 * 2 + e;
                    const bool in = key >= keys.lo && key < keys.hi;
                    s[n][e] = in && (OWN ? key <= pos0 : pos0 >= 0) ? s[n][e] * p.scale_log2 : -INFINITY;
                    s[n][2 + e] = in && (OWN ? key <= pos1 : pos1 >= 0) ? s[n][2 + e] * p.scale_log2 : -INFINITY;
                    x0 = fmaxf(x0, s[n][e]);
                    x1 = fmaxf(x1, s[n][2 + e]);
                }
            x0 = fmaxf(x0, __shfl_xor_sync(ALL, x0, 1)); x0 = fmaxf(x0, __shfl_xor_sync(ALL, x0, 2));
            x1 = fmaxf(x1, __shfl_xor_sync(ALL, x1, 1)); x1 = fmaxf(x1, __shfl_xor_sync(ALL, x1, 2));
            if (__any_sync(ALL, x0 > m0 || x1 > m1)) {
                const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
                const float f0 = m0 == -INFINITY ? 0.f : exp2_fast(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2_fast(m1 - n1);
                // (a row without a maximum has no sums yet but what is not finite: that stays)
                const float r0 = m0 == -INFINITY ? 1.f : f0, r1 = m1 == -INFINITY ? 1.f : f1;
                l0 *= f0; l1 *= f1;
#pragma unroll
                for (int n = 0; n < HD / 8; ++n) { o[n][0] *= r0; o[n][1] *= r0; o[n][2] *= r1; o[n][3] *= r1; }
                m0 = n0; m1 = n1;
            }
            const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[n][e] = exp2_fast(s[n][e] - b0);
                    s[n][2 + e] = exp2_fast(s[n][2 + e] - b1);
                    l0 += s[n][e];
                    l1 += s[n][2 + e];
                }
            // probabilities in bfloat16 (half a step, 2^-9 of each, at random): the tensor cores' operand; their sum stays in 32 bits
            const unsigned a[4] = {pack(s[0][0], s[0][1]), pack(s[0][2], s[0][3]), pack(s[1][0], s[1][1]), pack(s[1][2], s[1][3])};
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                unsigned bv[4];
                const int vr = kb + (lane & 15);
                ldmatrix4_trans(bv, vs + vr * HD + cache_chunk(2 * n + (lane >> 4), kt + vr, CHUNKS) * 8);
                mma(o[2 * n], a, bv[0], bv[1]);
                mma(o[2 * n + 1], a, bv[2], bv[3]);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    l0 += __shfl_xor_sync(ALL, l0, 1); l0 += __shfl_xor_sync(ALL, l0, 2);
    l1 += __shfl_xor_sync(ALL, l1, 1); l1 += __shfl_xor_sync(ALL, l1, 2);

    auto place = [&](int i) { const int rh = t.rh0 + i; return ((size_t)(part0 + part) * p.rows + rh / G) * p.H + kvh * G + rh % G; };
    if (WIDE) {
        if (i0 < t.count) {
            const size_t at = place(i0);
            if (t4 == 0) p.part_ml[at] = make_float2(m0, l0);
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(p.part_o + at * HD + n * 8 + t4 * 2) = make_float2(o[n][0], o[n][1]);
        }
        if (i1 < t.count) {
            const size_t at = place(i1);
            if (t4 == 0) p.part_ml[at] = make_float2(m1, l1);
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(p.part_o + at * HD + n * 8 + t4 * 2) = make_float2(o[n][2], o[n][3]);
        }
    } else {
        // the four warps' shares: sums relative to the largest maximum, added up in the order of the warps
        if (t4 == 0) { merge_m[warp][g] = m0; merge_m[warp][g + 8] = m1; merge_l[warp][g] = l0; merge_l[warp][g + 8] = l1; }
        __syncthreads();                                    // (the last tile has been read, too)
        float* merge_o = reinterpret_cast<float*>(ring);    // [warp][row][HD]
        const float M0 = fmaxf(fmaxf(merge_m[0][g], merge_m[1][g]), fmaxf(merge_m[2][g], merge_m[3][g]));
        const float M1 = fmaxf(fmaxf(merge_m[0][g + 8], merge_m[1][g + 8]), fmaxf(merge_m[2][g + 8], merge_m[3][g + 8]));
        const float w0 = m0 == -INFINITY ? 1.f : exp2_fast(m0 - M0), w1 = m1 == -INFINITY ? 1.f : exp2_fast(m1 - M1);
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
            *reinterpret_cast<float2*>(merge_o + (size_t)(warp * 16 + g) * HD + n * 8 + t4 * 2) = make_float2(o[n][0] * w0, o[n][1] * w0);
            *reinterpret_cast<float2*>(merge_o + (size_t)(warp * 16 + g + 8) * HD + n * 8 + t4 * 2) = make_float2(o[n][2] * w1, o[n][3] * w1);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * HD; i += MMA_THREADS) {
            const int r = i / HD;
            if (r >= t.count) break;
            p.part_o[place(r) * HD + i % HD] = ((merge_o[i] + merge_o[16 * HD + i]) + merge_o[32 * HD + i]) + merge_o[48 * HD + i];
        }
        if (threadIdx.x < 16 && (int)threadIdx.x < t.count) {
            const int r = threadIdx.x;
            const float M = fmaxf(fmaxf(merge_m[0][r], merge_m[1][r]), fmaxf(merge_m[2][r], merge_m[3][r]));
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) l += merge_m[w][r] == -INFINITY ? merge_l[w][r] : merge_l[w][r] * exp2_fast(merge_m[w][r] - M);
            p.part_ml[place(r)] = make_float2(M, l);
        }
    }
}

// ---- float32: dot products on the CUDA cores, everything in 32 bits ---------------------------------------------------------
// A CTA has up to 16 row heads; a warp takes every fourth key of the part, a lane's share of the head a stride of 32, and keeps sums of its own for
// four row heads at a time.
constexpr int F32_ROWS = 4, F32_LANES = (HD + 31) / 32;

template <bool OWN>
__global__ void __launch_bounds__(MMA_THREADS)
shared_f32_kernel(const SharedParams p, const SharedTile* tiles, int parts, int part0) {
    __shared__ float merge_o[4][F32_ROWS][HD];
    __shared__ float merge_m[4][F32_ROWS], merge_l[4][F32_ROWS];
    __shared__ int row_pos[16];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % p.KVH, part = blockIdx.x / p.KVH % parts;
    const SharedTile t = tiles[blockIdx.x / p.KVH / parts];
    const int G = p.H / p.KVH;
    constexpr int NCH = HD / 4;
    pdl_wait();
    if (threadIdx.x < 16) {
        const int i = threadIdx.x;
        const int pos = i < t.count ? p.positions[(t.rh0 + i) / G] : -1;
        row_pos[i] = pos >= t.prefix ? pos : -1;
    }
    __syncthreads();
    const int shared = shared_keys(p, t);
    for (int i0 = 0; i0 < t.count; i0 += F32_ROWS) {
        int last = shared, pos[F32_ROWS];
        bool any = false;
        float q[F32_ROWS][F32_LANES], o[F32_ROWS][F32_LANES], m[F32_ROWS], l[F32_ROWS];
#pragma unroll
        for (int r = 0; r < F32_ROWS; ++r) {
            pos[r] = i0 + r < t.count ? row_pos[i0 + r] : -1;
            any |= pos[r] >= 0;
            if (OWN) last = max(last, pos[r] + 1);
            m[r] = -INFINITY;
            l[r] = 0.f;
            const int rh = t.rh0 + min(i0 + r, t.count - 1);
            const float* src = static_cast<const float*>(p.q) + (long long)(rh / G) * p.ldq + (kvh * G + rh % G) * HD;
#pragma unroll
            for (int e = 0; e < F32_LANES; ++e) {
                q[r][e] = lane + e * 32 < HD ? src[lane + e * 32] : 0.f;
                o[r][e] = 0.f;
            }
        }
        // (rows of a tile may end at different keys: the part is one of the tile's keys, the same for all)
        int tile_last = shared;
        if (OWN)
            for (int i = 0; i < t.count; ++i) tile_last = max(tile_last, row_pos[i] + 1);
        const Range keys = part_range(OWN ? shared : 0, tile_last, OWN ? shared & ~63 : 0, part, parts, 64);
        const int hi = any ? min(keys.hi, last) : keys.lo;
        for (int key = keys.lo + warp; key < hi; key += 4) {
            const size_t at = (((size_t)page_at(p, t.slot, key / p.page) * 2 * p.KVH + kvh) * p.page + key % p.page) * HD;
            const float* k = static_cast<const float*>(p.plane) + at;
            const float* v = k + (size_t)p.KVH * p.page * HD;
            float kx[F32_LANES], vx[F32_LANES], s[F32_ROWS];
#pragma unroll
            for (int e = 0; e < F32_LANES; ++e) {
                const int d = lane + e * 32;
                const int from = d < HD ? cache_chunk(d / 4, key, NCH) * 4 + d % 4 : 0;
                kx[e] = d < HD ? k[from] : 0.f;
                vx[e] = d < HD ? v[from] : 0.f;
            }
#pragma unroll
            for (int r = 0; r < F32_ROWS; ++r) {
                s[r] = 0.f;
#pragma unroll
                for (int e = 0; e < F32_LANES; ++e) s[r] = fmaf(q[r][e], kx[e], s[r]);
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1)
#pragma unroll
                for (int r = 0; r < F32_ROWS; ++r) s[r] += __shfl_xor_sync(ALL, s[r], w);
#pragma unroll
            for (int r = 0; r < F32_ROWS; ++r) {
                if (OWN ? key > pos[r] : pos[r] < 0) continue;          // (uniform in the warp)
                const float x = s[r] * p.scale_log2;
                if (x > m[r]) {
                    const float f = exp2f(m[r] - x);                    // (of minus infinity: 0)
                    l[r] *= f;
#pragma unroll
                    for (int e = 0; e < F32_LANES; ++e) o[r][e] *= f;
                    m[r] = x;
                }
                const float w = exp2f(x - (m[r] == -INFINITY ? 0.f : m[r]));
                l[r] += w;
#pragma unroll
                for (int e = 0; e < F32_LANES; ++e) o[r][e] = fmaf(w, vx[e], o[r][e]);
            }
        }
        __syncthreads();                                    // (the merge of the rows before has been read)
#pragma unroll
        for (int r = 0; r < F32_ROWS; ++r) {
            if (lane == 0) { merge_m[warp][r] = m[r]; merge_l[warp][r] = l[r]; }
#pragma unroll
            for (int e = 0; e < F32_LANES; ++e)
                if (lane + e * 32 < HD) merge_o[warp][r][lane + e * 32] = o[r][e];
        }
        __syncthreads();
        const int r = warp;                                 // a warp a row head
        if (i0 + r < t.count) {
            const float M = fmaxf(fmaxf(merge_m[0][r], merge_m[1][r]), fmaxf(merge_m[2][r], merge_m[3][r]));
            float f[4], sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                f[w] = merge_m[w][r] == -INFINITY ? 1.f : exp2f(merge_m[w][r] - M);      // (no keys, or scores that are no numbers: as they are)
                sum += merge_l[w][r] * f[w];
            }
            const int rh = t.rh0 + i0 + r;
            const size_t at = ((size_t)(part0 + part) * p.rows + rh / G) * p.H + kvh * G + rh % G;
            if (lane == 0) p.part_ml[at] = make_float2(M, sum);
            for (int d = lane; d < HD; d += 32) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) x += merge_o[w][r][d] * f[w];
                p.part_o[at * HD + d] = x;
            }
        }
    }
}

// ---- the parts of a row head joined: a warp each -------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
shared_join_kernel(const SharedParams p, T* out, long long ldo, int row_heads, int parts) {
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5);      // row, head
    pdl_wait();
    if (i >= row_heads) return;
    const int row = i / p.H, head = i % p.H;
    float M = -INFINITY;
    for (int q = 0; q < parts; ++q) M = fmaxf(M, p.part_ml[(size_t)q * row_heads + i].x);
    float l = 0.f, o[F32_LANES];
#pragma unroll
    for (int e = 0; e < F32_LANES; ++e) o[e] = 0.f;
    for (int q = 0; q < parts; ++q) {
        const float2 ml = p.part_ml[(size_t)q * row_heads + i];
        if (ml.x == -INFINITY && ml.y == 0.f) continue;     // no keys
        const float f = ml.x == -INFINITY ? 1.f : exp2f(ml.x - M);
        l += ml.y * f;
        const float* src = p.part_o + ((size_t)q * row_heads + i) * HD;
#pragma unroll
        for (int e = 0; e < F32_LANES; ++e)
            if (lane + e * 32 < HD) o[e] = fmaf(src[lane + e * 32], f, o[e]);
    }
    T* dst = out + (long long)row * ldo + head * HD;
#pragma unroll
    for (int e = 0; e < F32_LANES; ++e)
        if (lane + e * 32 < HD) dst[lane + e * 32] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
}

template <bool OWN, bool WIDE> int launch_mma(const SharedParams& p, const SharedTile* tiles, int count, int parts, int part0, cudaStream_t stream) {
    const int ring = STAGES * 2 * TILE_ELEMENTS * 2, merge = 4 * 16 * HD * 4;
    const size_t smem = (size_t)(WIDE ? 64 : 16) * HD * 2 + (ring > merge ? ring : merge);
    static DeviceOnce configured;
    if (configured.first() && cudaFuncSetAttribute(shared_mma_kernel<OWN, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return tis_check_launch("shared_prefix_attention (shared memory)");
    tis_launch(shared_mma_kernel<OWN, WIDE>, dim3((unsigned)(count * parts * p.KVH)), dim3(MMA_THREADS), smem, stream, p, tiles, parts, part0);
    return tis_check_launch("shared_prefix_attention");
}

}  // namespace

TIS_API int tis_shared_attn_head_dim() { return HD; }

// `own`, `wide`: tiles on the device, own ones of up to 16 row heads, shared ones of up to 64 (bfloat16) or 16 (float32) row heads.
// The first `shared_parts` parts of the scratch are the shared tiles', the `own_parts` behind them the own ones'; rows of groups
// without shared keys have empty ones.  `rows`: the rows of the plan, all of which are written.
TIS_API int tis_shared_attention(int dtype, const void* q, long long ldq, void* out, long long ldo, const void* plane, const int* table,
                                 int table_stride, int table_width, int num_pages, const int* positions, const void* own, int own_count,
                                 const void* wide, int wide_count, int own_parts, int shared_parts, int rows, int H, int KVH, int page,
                                 float scale, float* part_o, void* part_ml, int* fault, cudaStream_t stream) {
    if (rows <= 0) return TIS_OK;
    SharedParams p;
    p.q = q; p.ldq = ldq; p.plane = plane;
    p.table = table; p.table_stride = table_stride; p.table_width = table_width; p.num_pages = num_pages;
    p.positions = positions;
    p.part_o = part_o; p.part_ml = static_cast<float2*>(part_ml);
    p.rows = rows; p.H = H; p.KVH = KVH; p.page = page; p.own_parts = own_parts; p.shared_parts = shared_parts;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.fault = fault;
    const SharedTile* o = static_cast<const SharedTile*>(own);
    const SharedTile* w = static_cast<const SharedTile*>(wide);
    const int parts = own_parts + shared_parts, row_heads = rows * H;
    int status = TIS_OK;
    if (dtype == TIS_F32) {
        if (shared_parts > 0) {
            tis_launch(shared_f32_kernel<false>, dim3((unsigned)(wide_count * shared_parts * KVH)), dim3(MMA_THREADS), 0, stream, p, w, shared_parts, 0);
            status = tis_check_launch("shared_prefix_attention");
        }
        if (status == TIS_OK) {
            tis_launch(shared_f32_kernel<true>, dim3((unsigned)(own_count * own_parts * KVH)), dim3(MMA_THREADS), 0, stream, p, o, own_parts, shared_parts);
            status = tis_check_launch("shared_prefix_attention");
        }
    } else if (dtype == TIS_BF16) {
        if (shared_parts > 0) status = launch_mma<false, true>(p, w, wide_count, shared_parts, 0, stream);
        if (status == TIS_OK) status = launch_mma<true, false>(p, o, own_count, own_parts, shared_parts, stream);
    } else {
        tis_set_error("shared_prefix_attention: dtype code %d", dtype);
        return TIS_BAD_DTYPE;
    }
    if (status != TIS_OK) return status;
    if (dtype == TIS_F32) tis_launch(shared_join_kernel<float>, dim3((unsigned)((row_heads + 7) / 8)), dim3(256), 0, stream, p, static_cast<float*>(out), ldo, row_heads, parts);
    else tis_launch(shared_join_kernel<bf16>, dim3((unsigned)((row_heads + 7) / 8)), dim3(256), 0, stream, p, static_cast<bf16*>(out), ldo, row_heads, parts);
    return tis_check_launch("shared_prefix_attention");
}
