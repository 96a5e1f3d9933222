// Products with weights of four bits on the fifth-generation tensor cores: up to 64 rows, many columns (gemm_w4.cu has the formula and the
// exactness of the parts, weights/w4.py the layout).
//
// mma.sync asks for a warp's instruction per 16 columns, 8 rows and 16 entries of the sum, and for the rows' operands from shared memory once a
// strip: from some 8 rows on that costs more than the weights' bytes.  Here a CTA has 128 columns as the rows of the tile and the rows of x
// as its narrow side.  Codes come by bulk copies into a ring in shared memory; four warps turn them into bfloat16 (a shift, a mask, a difference
// for two) and store them into tensor memory as the first operand, 64 entries of the sum at a time; one thread issues the products with x's
// rows, which TMA boxes bring beside the codes; and four other warps take a group's sums out of tensor memory and add them up, times the group's
// scale, in 32 bits.  Sums have two places, operands four, so that all of it runs at once.  Two CTAs an SM.
// Few columns leave SMs to share the sum out: a cluster of up to eight CTAs then has a tile, each a run of chunks, and its CTAs add up
// through one another's shared memory, in the order of the ranks.
// Bound by the weights' bytes, and by the instructions that unpack them: about 100 of a thread for 64 codes, 4 KB of a warp group.
// All waits are bounded; one that runs out sets the fault word, and every role leaves.
#include "tc_common.cuh"
#include "cluster_reduce.cuh"
#include "gemm_w4.cuh"

namespace {

using namespace tc;

constexpr int TILE = 128, TILE_STRIPS = TILE / W4_STRIP;
constexpr int STAGE_CHUNKS = 2, STAGE_WORDS = TILE_STRIPS * STAGE_CHUNKS * 512;          // bytes of codes of a stage
constexpr int A_STAGES = 4, A_COLS = 32;    // tensor memory: operands of 64 entries, two a column
constexpr unsigned COL_D = 0, COL_A = 128, TMEM_COLS = 256;
constexpr int NTH = 384;                    // warps 0-3 unpack, 4-7 add up, 8 orders copies, 9 issues products, 10 and 11 fill the group

template <int NB> struct Ring {
    static constexpr int X_BYTES = NB * 128 * STAGE_CHUNKS, BYTES = STAGE_WORDS + X_BYTES;
    static constexpr int STAGES = 100 * 1024 / BYTES < 8 ? 100 * 1024 / BYTES : 8;
};

struct W4TcParams {
    const unsigned char* words; const unsigned short* scales; const unsigned short* zeros;
    void* out; long long ldo;
    int rows, N, chunks, strips, groups, group_shift, tiles, slice;     // slice: chunks of a CTA of the cluster
    bool f32;
    int* fault;
};

__device__ __forceinline__ void bulk_copy(void* to, const void* from, int bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(smem_u32(to)), "l"(from), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// the product with its first operand in tensor memory
__device__ __forceinline__ void umma_ts(unsigned d, unsigned a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// 16 lanes of 32 columns of tensor memory: four blocks of eight columns, of which a thread (g, t) has columns 2 t and 2 t + 1 of lane g, then of lane g + 8
__device__ __forceinline__ void tmem_st_16x256b_x4(unsigned at, const unsigned (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                   "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned at, float* v) {
    unsigned* r = reinterpret_cast<unsigned*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(at));
}
__device__ __forceinline__ float load_rank(const float* local, unsigned rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(cluster_reduce::map_to_rank(smem_u32(local), rank)) : "memory");
    return v;
}

// NB: rows of x in the product (16, 32, 48, 64).  HALVES: groups of 32, two a chunk.  F32: the rows of x are three parts of a float's each, one
// after another, and out is in float32.
template <int NB, bool HALVES, bool F32>
__global__ void __launch_bounds__(NTH, 2)
w4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const W4TcParams p) {
    constexpr int STAGES = Ring<NB>::STAGES, BYTES = Ring<NB>::BYTES;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ unsigned long long full[STAGES], empty[STAGES], a_full[A_STAGES], a_empty[A_STAGES], d_full[2], d_empty[2];
    __shared__ unsigned tmem_base_slot;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned ranks, rank;
    asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(ranks));
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
    const int first_tile = blockIdx.x / ranks, tile_step = gridDim.x / ranks;
    const int c0 = (int)rank * p.slice, c1 = min(c0 + p.slice, p.chunks);               // (no rank is without chunks)

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 5); }
        for (int s = 0; s < A_STAGES; ++s) { mbar_init(&a_full[s], 4); mbar_init(&a_empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&d_full[s], 1); mbar_init(&d_empty[s], 4); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_map(&map_x);
    }
    __syncthreads();
    volatile int* abort = &abort_flag;
    unsigned tmem = 0;
    if (warp != 8) {
        // Tensor memory only when the kernel before is done: one that has begun to let this one in may still have to ask for its own.
        if (warp == 9) {
            pdl_wait();
            tmem_alloc(&tmem_base_slot, TMEM_COLS);
            pdl_launch_dependents();
        }
        fence_before();
        asm volatile("bar.sync 1, 352;\n" ::: "memory");
        fence_after();
        tmem = tmem_base_slot;
    }

    // 384 threads are launched with 80 registers each at the least, 30720 in all: 128 x 104 + 128 x 104 + 128 x 32
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;\n" ::);
        if (warp == 8) {
            // ---- codes (eight copies a stage, a lane a strip) and x (a box a chunk); weights do not come from the kernel before, x does ----
            int stage = 0;
            bool waited = false, ok = true;
            for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
                const int strip = min(tile * TILE_STRIPS + (lane & 7), p.strips - 1);
                const unsigned char* src = p.words + (size_t)strip * p.chunks * 512;
                for (int c = c0; c < c1; c += STAGE_CHUNKS, ++stage) {
                    const int s = stage % STAGES, n = min(STAGE_CHUNKS, c1 - c);
                    ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((stage / STAGES) & 1) ^ 1, abort, p.fault, 6));
                    if (!ok) break;
                    unsigned char* at = ring + (size_t)s * BYTES;
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], n * (TILE_STRIPS * 512 + NB * 128));
                    __syncwarp();
                    if (lane < TILE_STRIPS) bulk_copy(at + lane * (STAGE_CHUNKS * 512), src + (size_t)c * 512, n * 512, &full[s]);
                    if (!waited) { pdl_wait(); waited = true; }
                    if (lane < n) tma_load_2d(at + STAGE_WORDS + lane * (NB * 128), &map_x, (c + lane) * W4_CHUNK, 0, &full[s]);
                }
            }
            if (!waited) pdl_wait();
        } else if (warp == 9) {
            // ---- products: a chunk is four steps of 16 entries; a group's first step starts its sum ----
            constexpr unsigned IDESC = instr_desc(TILE, NB, false);
            const unsigned long long x_desc0 = smem_desc(smem_u32(ring + STAGE_WORDS), 16, 1024);
            int stage = 0, a = 0, d = 0;                    // stages, operands and sums so far
            bool ok = true;
            for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
                bool open = false;                          // a group's sum has begun
                for (int c = c0; c < c1 && ok; c += STAGE_CHUNKS, ++stage) {
                    const int s = stage % STAGES, n = min(STAGE_CHUNKS, c1 - c);
                    ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (stage / STAGES) & 1, abort, p.fault, 6));
                    for (int u = 0; u < n && ok; ++u, ++a) {
                        const int as = a % A_STAGES;
                        ok = __all_sync(0xffffffffu, mbar_wait(&a_full[as], (a / A_STAGES) & 1, abort, p.fault, 6));
                        if (!ok) break;
                        const bool ends = ((2 * (c + u)) >> p.group_shift) != ((2 * (c + u + 1)) >> p.group_shift) || c + u + 1 == c1;
                        const unsigned long long xd = x_desc0 + (unsigned long long)((s * BYTES + u * NB * 128) >> 4);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (!open) {
                                ok = ok && __all_sync(0xffffffffu, mbar_wait(&d_empty[d & 1], ((d >> 1) & 1) ^ 1, abort, p.fault, 6));
                                if (!ok) break;
                            }
                            fence_after();
                            if (elect_one()) {
                                const unsigned dst = tmem + COL_D + (d & 1) * 64;
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const int k = 2 * h + j;
                                    umma_ts(dst, tmem + COL_A + as * A_COLS + k * 8, xd + (unsigned long long)(k * 2), IDESC, open || j > 0);
                                }
                                if (h == 1) umma_commit(&a_empty[as]);
                                if (h == 1 && u == n - 1) umma_commit(&empty[s]);
                                if (HALVES || (h == 1 && ends)) umma_commit(&d_full[d & 1]);
                            }
                            __syncwarp();
                            open = true;
                            if (HALVES || (h == 1 && ends)) { open = false; ++d; }
                        }
                    }
                }
            }
        }
    } else if (warp < 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::);
        // ---- codes to bfloat16: a warp has two strips, 32 lanes of tensor memory ----
        int stage = 0, a = 0;
        bool ok = true;
        const int g = lane >> 2;
        for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
            const unsigned short* zeros[2];
            int seen = -1;                                  // the group whose zero points are here
            unsigned low[2] = {0x43084308u, 0x43084308u}, high[2] = {0x43084308u, 0x43084308u};     // 128 + zero of the columns g and g + 8
            unsigned next[2] = {0u, 0u};                    // and those of the group behind it
#pragma unroll
            for (int q = 0; q < 2; ++q)
                zeros[q] = p.zeros + (size_t)min(tile * TILE_STRIPS + warp * 2 + q, p.strips - 1) * p.groups * 8 + g;
            if (p.zeros != nullptr) {
#pragma unroll
                for (int q = 0; q < 2; ++q) next[q] = __ldg(zeros[q] + ((2 * c0) >> p.group_shift) * 8);
            }
            for (int c = c0; c < c1 && ok; c += STAGE_CHUNKS, ++stage) {
                const int s = stage % STAGES, n = min(STAGE_CHUNKS, c1 - c);
                ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (stage / STAGES) & 1, abort, p.fault, 6));
                if (!ok) break;
                for (int u = 0; u < n; ++u, ++a) {
                    const int as = a % A_STAGES;
                    uint4 w[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        w[q] = *reinterpret_cast<const uint4*>(ring + (size_t)s * BYTES + (warp * 2 + q) * (STAGE_CHUNKS * 512) + u * 512 + lane * 16);
                    unsigned r[2][16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (p.zeros != nullptr && (h == 0 || HALVES)) {
                            const int group = (2 * (c + u) + h) >> p.group_shift;
                            if (group != seen) {            // (uniform in the CTA)
                                seen = group;
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    low[q] = 0x43004300u | (next[q] & 0xffu) * 0x00010001u;
                                    high[q] = 0x43004300u | (next[q] >> 8) * 0x00010001u;
                                    next[q] = __ldg(zeros[q] + min(group + 1, p.groups - 1) * 8);
                                }
                            }
                        }
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const unsigned v = h ? (j ? w[q].w : w[q].z) : (j ? w[q].y : w[q].x);
                                unsigned* to = r[q] + (2 * h + j) * 4;
                                to[0] = w4_pair(v, low[q]);
                                to[2] = w4_pair(v >> 4, high[q]);
                                to[1] = w4_pair(v >> 8, low[q]);
                                to[3] = w4_pair(v >> 12, high[q]);
                            }
                    }
                    ok = __all_sync(0xffffffffu, mbar_wait(&a_empty[as], ((a / A_STAGES) & 1) ^ 1, abort, p.fault, 6));
                    if (!ok) break;
                    fence_after();
#pragma unroll
                    for (int q = 0; q < 2; ++q) tmem_st_16x256b_x4(tmem + ((unsigned)(warp * 32 + q * 16) << 16) + COL_A + as * A_COLS, r[q]);
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&a_full[as]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);      // the stage's codes have been read
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::);
        // ---- a thread a column: the groups' sums, times their scales, added up ----
        const int quarter = warp & 3, column = quarter * 32 + lane;
        const unsigned from = tmem + ((unsigned)(quarter * 32) << 16) + COL_D;
        int d = 0;
        bool ok = true;
        for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
            const int strip = min(tile * TILE_STRIPS + column / W4_STRIP, p.strips - 1), in = column % W4_STRIP;
            const unsigned short* scales = p.scales + ((size_t)strip * p.groups * 8 + (in & 7)) * 2 + (in >> 3);
            float total[NB];
#pragma unroll
            for (int r = 0; r < NB; ++r) total[r] = 0.f;
            const int h0 = HALVES ? 2 * c0 : (2 * c0) >> p.group_shift, h1 = min(HALVES ? 2 * c1 : ((2 * c1 - 1) >> p.group_shift) + 1, HALVES ? 2 * c1 : p.groups);
            unsigned short scale = __ldg(scales + min(h0, p.groups - 1) * 16);
            for (int group = h0; group < h1; ++group, ++d) {
                const float f = __uint_as_float((unsigned)scale << 16);
                scale = __ldg(scales + min(group + 1, p.groups - 1) * 16);
                ok = __all_sync(0xffffffffu, mbar_wait(&d_full[d & 1], (d >> 1) & 1, abort, p.fault, 6));
                if (!ok) break;
                fence_after();
                constexpr int STEP = NB % 32 == 0 ? 32 : 16;
#pragma unroll
                for (int b = 0; b < NB; b += STEP) {
                    float v[STEP];
#pragma unroll
                    for (int e = 0; e < STEP; e += 16) tmem_ld16(from + (d & 1) * 64 + b + e, v + e);
                    tmem_ld_wait();
                    tmem_ld_arrived(v);
                    if (b + STEP == NB) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&d_empty[d & 1]);
                    }
#pragma unroll
                    for (int e = 0; e < STEP; ++e) total[b + e] = fmaf(v[e], f, total[b + e]);
                }
            }
            if (!ok) break;
            if (ranks == 1) {
                const int n = tile * TILE + column;
                if (n < p.N) {
                    if (F32) {
#pragma unroll
                        for (int r = 0; r < NB / 3; ++r)    // the small parts first
                            if (r < p.rows) static_cast<float*>(p.out)[r * p.ldo + n] = (total[3 * r + 2] + total[3 * r + 1]) + total[3 * r];
                    } else {
#pragma unroll
                        for (int r = 0; r < NB; ++r)
                            if (r < p.rows) static_cast<bf16*>(p.out)[r * p.ldo + n] = __float2bfloat16_rn(total[r]);
                    }
                }
            } else {
                // the ring has no more to come: it takes the CTA's sums, [row][column]
                float* part = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int r = 0; r < NB; ++r) part[r * TILE + column] = total[r];
            }
        }
    }
    if (*abort) {
        // a wait ran out: copies that may still be on their way get time to land before the shared memory is given up
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    fence_before();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
    if (ranks > 1) {
        cluster_reduce::cluster_arrive();
        cluster_reduce::cluster_wait();
        const float* part = reinterpret_cast<const float*>(ring);
        const int n = first_tile * TILE + (int)(threadIdx.x & 127);
        // rows rank, rank + ranks, ..: three at a time, the ranks' sums in their order
        for (int r = (int)rank + (int)(threadIdx.x >> 7) * (int)ranks; r < p.rows; r += 3 * (int)ranks) {
            float v[3] = {0.f, 0.f, 0.f};
            for (unsigned q = 0; q < ranks; ++q)
#pragma unroll
                for (int e = 0; e < (F32 ? 3 : 1); ++e) v[e] += load_rank(part + ((F32 ? 3 : 1) * r + e) * TILE + (threadIdx.x & 127), q);
            if (n < p.N) {
                if (F32) static_cast<float*>(p.out)[r * p.ldo + n] = (v[2] + v[1]) + v[0];
                else static_cast<bf16*>(p.out)[r * p.ldo + n] = __float2bfloat16_rn(v[0]);
            }
        }
        cluster_reduce::cluster_arrive();                   // (read before its owner leaves)
        cluster_reduce::cluster_wait();
    }
}

template <int NB, bool HALVES, bool F32> int launch(const CUtensorMap& map, const W4TcParams& p, int ranks, cudaStream_t stream) {
    const int smem = Ring<NB>::STAGES * Ring<NB>::BYTES + 1024;
    static_assert(Ring<NB>::STAGES * Ring<NB>::BYTES >= NB * TILE * 4, "a CTA's sums fit the ring");
    static DeviceOnce configured;
    if (configured.first() && cudaFuncSetAttribute(w4_tc_kernel<NB, HALVES, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return tis_check_launch("gemm_w4 (shared memory)");
    const int most = 2 * sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ranks > 1 ? p.tiles * ranks : (p.tiles < most ? p.tiles : most)));
    cfg.blockDim = dim3(NTH);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = (unsigned)ranks;
    attrs[0].val.clusterDim.y = 1;
    attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = tis_pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, w4_tc_kernel<NB, HALVES, F32>, map, p);
    return tis_check_launch("gemm_w4");
}
template <int NB> int launch_form(const CUtensorMap& map, const W4TcParams& p, int ranks, cudaStream_t stream) {
    if (p.f32) return p.group_shift == 0 ? launch<NB, true, true>(map, p, ranks, stream) : launch<NB, false, true>(map, p, ranks, stream);
    return p.group_shift == 0 ? launch<NB, true, false>(map, p, ranks, stream) : launch<NB, false, false>(map, p, ranks, stream);
}

}  // namespace

int w4_tc_launch(const W4Params& w, const void* x, int x_rows, long long ldx, int* fault, cudaStream_t stream) {
    const int nb = x_rows <= 16 ? 16 : (x_rows <= 32 ? 32 : (x_rows <= 48 ? 48 : 64));
    CUtensorMap map;
    if (!tensor_map(x, w.K, x_rows, ldx, nb, true, &map)) return TIS_CUDA_ERROR;
    W4TcParams p;
    p.words = reinterpret_cast<const unsigned char*>(w.words);
    p.scales = reinterpret_cast<const unsigned short*>(w.scales);
    p.zeros = w.zeros;
    p.out = w.out; p.ldo = w.ldo;
    p.rows = w.rows; p.N = w.N; p.chunks = w.chunks; p.strips = w.strips; p.groups = w.groups; p.group_shift = w.group_shift;
    p.tiles = (w.N + TILE - 1) / TILE;
    p.f32 = w.f32;
    p.fault = fault;
    // CTAs of a tile: as many as are all resident, with four chunks each at the least, none of them empty
    int ranks = 1;
    while (ranks < 8 && p.tiles * ranks * 2 <= 2 * sm_count() && p.chunks >= 2 * ranks * 4) ranks *= 2;
    while (ranks > 1 && ((p.chunks + ranks - 1) / ranks) * (ranks - 1) >= p.chunks) ranks /= 2;
    p.slice = (p.chunks + ranks - 1) / ranks;
    switch (nb) {
        case 16: return launch_form<16>(map, p, ranks, stream);
        case 32: return launch_form<32>(map, p, ranks, stream);
        case 48: return launch_form<48>(map, p, ranks, stream);
        default: return launch_form<64>(map, p, ranks, stream);
    }
}
