// Products with weights of four bits on the fifth-generation tensor cores: up to 64 rows, many columns (gemm_w4.cu has the formula and the
// exactness of the parts, weights/w4.py the layout).
//
// mma.sync asks for a warp's instruction per 16 columns, 8 rows and 16 entries of the sum, and for the rows' operands from shared memory once a
// strip: from some 8 rows on that costs more than the weights' bytes.  Here a CTA has 128 columns as the rows of the tile and the rows of x
// as its narrow side.  Codes come by bulk copies into a ring in shared memory; eight warps turn them into bfloat16 (a shift, a mask, a difference
// for two) and store them into tensor memory as the first operand, 64 entries of the sum a half; one thread issues the products with x's
// rows, which TMA boxes bring beside the codes; and four more warps take a group's sums out of tensor memory and add them up, times the group's
// scale, in 32 bits.  Sums and operands have two places each, an operand's being a stage of 128 entries with one hand-over, so that all of it runs at once.
// Two CTAs an SM.
// Few columns leave SMs to share the sum out: a cluster of up to eight CTAs then has a tile, each a run of chunks, and its CTAs add up
// through one another's shared memory, in the order of the ranks.
// Bound by the weights' bytes, and by the instructions that unpack them: about 100 of a thread for 64 codes; now by
// the hand-overs between the roles (1900 cycles for 128 entries of 128 columns, the same with the work between them left out).  The schedulers issue in
// 67 % of the cycles; of 11.3 cycles from one of a warp's instructions to its next it waits 3.1 for loads and tensor memory, 1.6 at barriers, 1.1 for the units.
// Measured: 40 rows x 4096 x 131072, groups of 64 with zero points (302 MB): 159 us, 1.9 TB/s (1024 tiles on 296 CTAs, 3.46 each: four turns).
// With 33 to 48 rows the adding warps keep 28 to 32 bytes of their registers in local memory.
// All waits are bounded; one that runs out sets the fault word, and every role leaves.
#include "tc_common.cuh"
#include "cluster_reduce.cuh"
#include "gemm_w4.cuh"

namespace {

using namespace tc;

constexpr int TILE = 128, TILE_STRIPS = TILE / W4_STRIP;
constexpr int STAGE_CHUNKS = 2, STAGE_WORDS = TILE_STRIPS * STAGE_CHUNKS * 512;          // bytes of codes of a stage
constexpr int A_STAGES = 2, A_COLS = 32;    // tensor memory: operands of a stage of the ring, a chunk's 64 entries in 32 columns
constexpr unsigned COL_D = 0, COL_A = 128, TMEM_COLS = 256;
constexpr int NTH = 512;                    // warps 0-7 unpack, 8-11 add up, 12 orders copies, 13 issues products, 14 and 15 fill the group

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

// NB: rows of x in the product (16, 32, 48, 64).  SPAN: entries of a group, 128 for all from there on.  F32: the rows of x are three parts of a float's each, one
// after another, and out is in float32.
template <int NB, int SPAN, bool F32>
__global__ void __launch_bounds__(NTH, 2)
w4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const W4TcParams p) {
    constexpr int STAGES = Ring<NB>::STAGES, BYTES = Ring<NB>::BYTES;
    constexpr bool HALVES = SPAN == 32;
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
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 8); }
        for (int s = 0; s < A_STAGES; ++s) { mbar_init(&a_full[s], 8); mbar_init(&a_empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&d_full[s], 1); mbar_init(&d_empty[s], 4); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_map(&map_x);
    }
    __syncthreads();
    volatile int* abort = &abort_flag;
    unsigned tmem = 0;
    if (warp != 12) {
        // Tensor memory only when the kernel before is done: one that has begun to let this one in may still have to ask for its own.
        if (warp == 13) {
            pdl_wait();
            tmem_alloc(&tmem_base_slot, TMEM_COLS);
            pdl_launch_dependents();
        }
        fence_before();
        asm volatile("bar.sync 1, 480;\n" ::: "memory");
        fence_after();
        tmem = tmem_base_slot;
    }

    // 512 threads are launched with 64 registers each, 32768 in all: 256 x 64 + 128 x 96 + 128 x 32
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;\n" ::);
        if (warp == 12) {
            // ---- codes (a copy a stage) and x (a box a chunk), by one thread; weights do not come from the kernel before, x does ----
            if (elect_one()) {
                int stage = 0;
                bool waited = false, ok = true;
                for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
                    const unsigned char* src = p.words + (size_t)tile * p.chunks * (TILE_STRIPS * 512);
                    for (int c = c0; c < c1; c += STAGE_CHUNKS, ++stage) {
                        const int s = stage % STAGES, n = min(STAGE_CHUNKS, c1 - c);
                        ok = mbar_wait(&empty[s], ((stage / STAGES) & 1) ^ 1, abort, p.fault, 6);
                        if (!ok) break;
                        unsigned char* at = ring + (size_t)s * BYTES;
                        mbar_arrive_expect_tx(&full[s], n * (TILE_STRIPS * 512 + NB * 128));
                        bulk_copy(at, src + (size_t)c * (TILE_STRIPS * 512), n * (TILE_STRIPS * 512), &full[s]);
                        if (!waited) { pdl_wait(); waited = true; }
                        for (int u = 0; u < n; ++u) tma_load_2d(at + STAGE_WORDS + u * (NB * 128), &map_x, (c + u) * W4_CHUNK, 0, &full[s]);
                    }
                }
                if (!waited) pdl_wait();
            }
            __syncwarp();
        } else if (warp == 13) {
            // ---- products: a chunk is four steps of 16 entries; a group's first step starts its sum.  One hand-over a stage; that its rows of x
            // have landed the unpacking warps have seen.  (The warp walks together and one lane issues what a stage has in one go, so that
            // operands come from uniform registers: alone in its branch a thread takes 100 cycles a product, this way 25.) ----
            constexpr unsigned IDESC = instr_desc(TILE, NB, false);
            // (groups of 32 and 64: a chunk a round, with its two groups or its one, so that a round waits for places of its own sums only)
            constexpr int ROUNDS = SPAN == 128 ? 1 : STAGE_CHUNKS, SUMS = HALVES ? 2 : 1;
            const unsigned long long x_desc0 = smem_desc(smem_u32(ring + STAGE_WORDS), 16, 1024);
            int stage = 0, d = 0;                           // stages and sums so far
            bool ok = true;
            for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
                bool open = false;                          // a group's sum has begun (SPAN 128: it may go over several stages)
                for (int c = c0; c < c1 && ok; c += STAGE_CHUNKS, ++stage) {
                    const int s = stage % STAGES, as = stage % A_STAGES, n = min(STAGE_CHUNKS, c1 - c);
                    ok = __all_sync(0xffffffffu, mbar_wait(&a_full[as], (stage / A_STAGES) & 1, abort, p.fault, 6));
                    if (!ok) break;
                    const bool ends = SPAN != 128 || c + n == c1 || ((2 * c) >> p.group_shift) != ((2 * (c + n)) >> p.group_shift);
#pragma unroll
                    for (int round = 0; round < ROUNDS; ++round) {
                        if (round == 1 && n == 1) break;
                        if (!open) {
#pragma unroll
                            for (int q = 0; q < SUMS; ++q)
                                ok = ok && __all_sync(0xffffffffu, mbar_wait(&d_empty[(d + q) & 1], (((d + q) >> 1) & 1) ^ 1, abort, p.fault, 6));
                            if (!ok) break;
                        }
                        fence_after();
                        if (elect_one()) {
                            const unsigned a0 = tmem + COL_A + as * (STAGE_CHUNKS * A_COLS);
                            const unsigned long long x0 = x_desc0 + (unsigned long long)((s * BYTES) >> 4);
#pragma unroll
                            for (int u = SPAN == 128 ? 0 : round; u < (SPAN == 128 ? STAGE_CHUNKS : round + 1); ++u) {
                                if (u == 1 && n == 1) break;
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const unsigned dst = tmem + COL_D + ((d + (HALVES ? k / 2 : 0)) & 1) * 64;
                                    const unsigned going = SPAN == 128 ? (open || u > 0 || k > 0) : (SPAN == 64 ? k > 0 : (k & 1));
                                    umma_ts(dst, a0 + u * A_COLS + k * 8, x0 + (unsigned long long)((u * NB * 128 + k * 32) >> 4), IDESC, going);
                                    if (HALVES && (k & 1)) umma_commit(&d_full[(d + k / 2) & 1]);
                                }
                                if (SPAN == 64) umma_commit(&d_full[d & 1]);
                            }
                            if (SPAN == 128 && ends) umma_commit(&d_full[d & 1]);
                            if (round == ROUNDS - 1 || n == 1) umma_commit(&a_empty[as]);
                        }
                        __syncwarp();
                        if (SPAN == 128) { open = !ends; d += ends; }
                        else d += SUMS;
                    }
                }
            }
        }
    } else if (warp < 8) {
        // ---- codes to bfloat16: a warp has two strips, 32 lanes of tensor memory, of every other chunk: the two of a stage are two warps' ----
        static_assert(STAGE_CHUNKS == 2, "a chunk of a stage each");
        const int quarter = warp & 3, u = warp >> 2;
        int stage = 0;
        bool ok = true;
        const int g = lane >> 2;
        for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
            const unsigned short* zeros[2];
            int seen = -1;                                  // the group whose zero points are here
            unsigned low[2] = {0x43084308u, 0x43084308u}, high[2] = {0x43084308u, 0x43084308u};     // 128 + zero of the columns g and g + 8
#pragma unroll
            for (int q = 0; q < 2; ++q)
                zeros[q] = p.zeros + (size_t)min(tile * TILE_STRIPS + quarter * 2 + q, p.strips - 1) * p.groups * 8 + g;
            for (int c = c0; c < c1 && ok; c += STAGE_CHUNKS, ++stage) {
                const int s = stage % STAGES, n = min(STAGE_CHUNKS, c1 - c);
                // zero points are asked for before the codes are waited for
                unsigned short z[2][2] = {{0, 0}, {0, 0}};
                const int group = min((2 * (c + u)) >> p.group_shift, p.groups - 1);
                const bool fresh = p.zeros != nullptr && group != seen;         // (uniform in the warp)
                if (fresh) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        z[q][0] = __ldg(zeros[q] + group * 8);
                        if (HALVES) z[q][1] = __ldg(zeros[q] + min(group + 1, p.groups - 1) * 8);
                    }
                    seen = group;
                }
                const int as = stage % A_STAGES;
                ok = __all_sync(0xffffffffu, mbar_wait_both(&full[s], (stage / STAGES) & 1, &a_empty[as], ((stage / A_STAGES) & 1) ^ 1, abort, p.fault, 6));
                if (!ok) break;
                // the products of the stage before the one before are done: its place in the ring is free, codes and rows of x
                if (stage >= A_STAGES && lane == 0) mbar_arrive(&empty[(stage - A_STAGES) % STAGES]);
                fence_after();
                unsigned r[2][16];
#pragma unroll
                for (int q = 0; q < 2; ++q) {               // (of a chunk beyond the last: what lies there, for an operand that no product takes)
                    const uint4 w = *reinterpret_cast<const uint4*>(ring + (size_t)s * BYTES + (u * TILE_STRIPS + quarter * 2 + q) * 512 + lane * 16);
                    if (fresh) {
                        low[q] = 0x43004300u | (z[q][0] & 0xffu) * 0x00010001u;
                        high[q] = 0x43004300u | (unsigned)(z[q][0] >> 8) * 0x00010001u;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const unsigned v = k == 0 ? w.x : (k == 1 ? w.y : (k == 2 ? w.z : w.w));
                        unsigned lo = low[q], hi = high[q];
                        if (HALVES && k >= 2 && p.zeros != nullptr) {
                            lo = 0x43004300u | (z[q][1] & 0xffu) * 0x00010001u;
                            hi = 0x43004300u | (unsigned)(z[q][1] >> 8) * 0x00010001u;
                        }
                        r[q][4 * k] = w4_pair(v, lo);
                        r[q][4 * k + 2] = w4_pair(v >> 4, hi);
                        r[q][4 * k + 1] = w4_pair(v >> 8, lo);
                        r[q][4 * k + 3] = w4_pair(v >> 12, hi);
                    }
                }
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    tmem_st_16x256b_x4(tmem + ((unsigned)(quarter * 32 + q * 16) << 16) + COL_A + (as * STAGE_CHUNKS + u) * A_COLS, r[q]);
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[as]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;\n" ::);
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
#pragma unroll
                for (int b = 0; b < NB; b += 32) {
                    constexpr int STEP = 32;
                    float v[STEP];
#pragma unroll
                    for (int e = 0; e < STEP; e += 16)
                        if (b + e < NB) tmem_ld16(from + (d & 1) * 64 + b + e, v + e);
                    tmem_ld_wait();
                    tmem_ld_arrived(v);
                    if (b + STEP >= NB) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&d_empty[d & 1]);
                    }
#pragma unroll
                    for (int e = 0; e < STEP; ++e)
                        if (b + e < NB) total[b + e] = fmaf(v[e], f, total[b + e]);
                }
            }
            if (!ok) break;
            if (ranks == 1) {
                const int n = tile * TILE + column;
                if (n < p.N) {
                    if (F32) {
#pragma unroll
                        for (int r = 0; r < NB / 3; ++r)
                            if (r < p.rows) static_cast<float*>(p.out)[r * p.ldo + n] = of_three(total[3 * r], total[3 * r + 1], total[3 * r + 2]);
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
    if (warp == 13) {
        fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
    if (ranks > 1) {
        cluster_reduce::cluster_arrive();
        cluster_reduce::cluster_wait();
        const float* part = reinterpret_cast<const float*>(ring);
        const int n = first_tile * TILE + (int)(threadIdx.x & 127);
        // rows rank, rank + ranks, ..: four at a time, the ranks' sums in their order
        for (int r = (int)rank + (int)(threadIdx.x >> 7) * (int)ranks; r < p.rows; r += 4 * (int)ranks) {
            float v[3] = {0.f, 0.f, 0.f};
            for (unsigned q = 0; q < ranks; ++q)
#pragma unroll
                for (int e = 0; e < (F32 ? 3 : 1); ++e) v[e] += load_rank(part + ((F32 ? 3 : 1) * r + e) * TILE + (threadIdx.x & 127), q);
            if (n < p.N) {
                if (F32) static_cast<float*>(p.out)[r * p.ldo + n] = of_three(v[0], v[1], v[2]);
                else static_cast<bf16*>(p.out)[r * p.ldo + n] = __float2bfloat16_rn(v[0]);
            }
        }
        cluster_reduce::cluster_arrive();                   // (read before its owner leaves)
        cluster_reduce::cluster_wait();
    }
}

// x's rows as the products take them: bfloat16 in rows that start on 16 bytes; a row of float32 is three (`three`).
template <typename T>
__global__ void __launch_bounds__(256) w4_copy_kernel(const T* x, long long ldx, bf16* to, long long ldt, int rows, int K) {
    pdl_launch_dependents();
    pdl_wait();
    const int k = blockIdx.x * 256 + threadIdx.x;
    if (k >= K) return;
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        if (sizeof(T) == 2) {
            to[r * ldt + k] = *reinterpret_cast<const bf16*>(x + r * ldx + k);
        } else {
            unsigned short v[3];
            three(*reinterpret_cast<const float*>(x + r * ldx + k), v);
#pragma unroll
            for (int q = 0; q < 3; ++q) reinterpret_cast<unsigned short*>(to)[(3ll * r + q) * ldt + k] = v[q];
        }
    }
}

template <int NB, int SPAN, bool F32> int launch(const CUtensorMap& map, const W4TcParams& p, int ranks, cudaStream_t stream) {
    const int smem = Ring<NB>::STAGES * Ring<NB>::BYTES + 1024;
    static_assert(Ring<NB>::STAGES > A_STAGES, "the ring is ahead of the operands");
    static_assert(Ring<NB>::STAGES * Ring<NB>::BYTES >= NB * TILE * 4, "a CTA's sums fit the ring");
    static DeviceOnce configured;
    if (configured([&] { return cudaFuncSetAttribute(w4_tc_kernel<NB, SPAN, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }) != cudaSuccess)
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
    cudaLaunchKernelEx(&cfg, w4_tc_kernel<NB, SPAN, F32>, map, p);
    return tis_check_launch("gemm_w4");
}
template <int NB, bool F32> int launch_span(const CUtensorMap& map, const W4TcParams& p, int ranks, cudaStream_t stream) {
    if (p.group_shift == 0) return launch<NB, 32, F32>(map, p, ranks, stream);
    if (p.group_shift == 1) return launch<NB, 64, F32>(map, p, ranks, stream);
    return launch<NB, 128, F32>(map, p, ranks, stream);
}
template <int NB> int launch_form(const CUtensorMap& map, const W4TcParams& p, int ranks, cudaStream_t stream) {
    return p.f32 ? launch_span<NB, true>(map, p, ranks, stream) : launch_span<NB, false>(map, p, ranks, stream);
}

}  // namespace

int w4_tc_launch(const W4Params& w, void* copy, int* fault, cudaStream_t stream) {
    const bf16* x = static_cast<const bf16*>(w.x);
    long long ldx = w.ldx;
    const int times = w.f32 ? 3 : 1;
    if (copy != nullptr) {
        ldx = (w.K + 7) / 8 * 8;
        x = static_cast<const bf16*>(copy);
        const dim3 grid((unsigned)((w.K + 255) / 256), (unsigned)(w.rows < 65535 ? w.rows : 65535));
        if (w.f32) tis_launch(w4_copy_kernel<float>, grid, dim3(256), 0, stream, static_cast<const float*>(w.x), w.ldx, static_cast<bf16*>(copy), ldx, w.rows, w.K);
        else tis_launch(w4_copy_kernel<bf16>, grid, dim3(256), 0, stream, static_cast<const bf16*>(w.x), w.ldx, static_cast<bf16*>(copy), ldx, w.rows, w.K);
        const int status = tis_check_launch("gemm_w4 (copy)");
        if (status != TIS_OK) return status;
    }
    W4TcParams p;
    p.words = reinterpret_cast<const unsigned char*>(w.words);
    p.scales = reinterpret_cast<const unsigned short*>(w.scales);
    p.zeros = w.zeros;
    p.ldo = w.ldo;
    p.N = w.N; p.chunks = w.chunks; p.strips = w.strips; p.groups = w.groups; p.group_shift = w.group_shift;
    p.tiles = (w.N + TILE - 1) / TILE;
    p.f32 = w.f32;
    p.fault = fault;
    // CTAs of a tile: as many as are all resident, with four chunks each at the least, none of them empty
    int ranks = 1;
    while (ranks < 8 && p.tiles * ranks * 2 <= 2 * sm_count() && p.chunks >= 2 * ranks * 4) ranks *= 2;
    // (whole stages each, so that a stage has whole groups)
    auto slice = [&](int r) { return ((p.chunks + r - 1) / r + STAGE_CHUNKS - 1) / STAGE_CHUNKS * STAGE_CHUNKS; };
    while (ranks > 1 && slice(ranks) * (ranks - 1) >= p.chunks) ranks /= 2;
    p.slice = slice(ranks);
    // rows in slabs of about the same size
    const int most = w.f32 ? W4_TC_ROWS_F32 : W4_TC_ROWS, slabs = (w.rows + most - 1) / most, slab = (w.rows + slabs - 1) / slabs;
    for (int row = 0; row < w.rows; row += slab) {
        p.rows = w.rows - row < slab ? w.rows - row : slab;
        p.out = static_cast<char*>(w.out) + (long long)row * w.ldo * (w.f32 ? 4 : 2);
        const int x_rows = times * p.rows, nb = x_rows <= 16 ? 16 : (x_rows <= 32 ? 32 : (x_rows <= 48 ? 48 : 64));
        CUtensorMap map;
        if (!tensor_map(x + (long long)times * row * ldx, w.K, x_rows, ldx, nb, true, &map)) return TIS_CUDA_ERROR;
        const int status = nb == 16 ? launch_form<16>(map, p, ranks, stream) : nb == 32 ? launch_form<32>(map, p, ranks, stream)
                         : nb == 48 ? launch_form<48>(map, p, ranks, stream) : launch_form<64>(map, p, ranks, stream);
        if (status != TIS_OK) return status;
    }
    return TIS_OK;
}
