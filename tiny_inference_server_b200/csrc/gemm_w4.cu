// Products of few rows with weights of four bits: out[r][n] = sum over k of x[r][k] (code[k][n] - zero[k / group][n]) scale[k / group][n].
//
// Bound by the weights' bytes: half a byte a weight, and two or three a group for its scale and zero point.  Every weight is read
// once, by a 16-byte load of a lane straight into registers, several of them under way at a time; a lane's 16 bytes are its parts
// of four 16 x 16 operands of mma.sync (16 columns of the matrix as the operand's rows, the rows of x as its narrow side), laid out so
// beforehand (weights/w4.py has the layout).  A shift, a mask and a difference make two of them bfloat16 numbers: 0x4300 | code is 128 + code,
// exactly, and so is (128 + code) - (128 + zero).  So the products are of whole numbers up to 15, exact in 32 bits, and a group's sum is
// multiplied by its scale once, in 32 bits: weights are never rounded.
//
// x in float32 goes through the same products as three bfloat16 numbers each, cut off and not rounded: 8 + 8 + 8 bits hold all 24
// of a float, and the lower ones are scaled (`three`) so that those of the smallest floats are held too: nothing is lost there either.
// A group's sum of whole numbers is formed before its scale, in 32 bits: 15 times the sum of a group's |x|, in float32 twice that, has to stay below
// 2^128, or a result comes out as infinite that with the scale would not be.
//
// A CTA of eight warps takes a few strips of 16 columns; its warps share them out (`ws` of them side by side) and the chunks of
// 64 entries of the sum (`wk` of them take turns), and add up in shared memory, in a fixed order.  x waits in shared memory, whole or in
// stages; its rows lie 32 bytes off a multiple of 128 apart, so that the four rows x four pieces of 8 bytes that half a warp reads at a time
// are free of bank conflicts.
// Measured: 8 rows x 4096 x 28672, groups of 128 (61 MB): 26.3 us, 2.3 TB/s; 1 row x 1536 x 2304: 2.4 us; 3 float32 rows x 2005 x 5501, groups of 32: 8.3 us.
// The first without its loads 21.4 us, with nothing but its loads 8.0: some 120 instructions of a warp for 1024 codes, and what each waits for, count for more
// than the bytes.  The schedulers issue in 53 % of the cycles; of 7.2 cycles from one of a warp's instructions to its next it waits 2.6 for loads, 1.3
// for a result and 0.6 for the arithmetic units.  896 tiles on 296 CTAs are 3.03 each: eight CTAs have a fourth turn, the others none.
// With few tiles (x in several pieces) a CTA has a tile at most and walks K by two warps' turns, which is why the choice between the two kernels
// (kernels/ops.py) asks for the tiles.
#include "gemm_w4.cuh"

namespace {

constexpr int W4_THREADS = 256, W4_WARPS = 8;
constexpr int W4_PAD = 16;                  // elements behind a staged row
constexpr int W4_STAGED = 24;                // most staged rows: those of bfloat16, three of each of float32

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float low_half(unsigned v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_half(unsigned v) { return __uint_as_float(v & 0xffff0000u); }

// Entries [k0, k0 + count) of the rows of x into shared memory, zero beyond K.  In float32 the rows stand three times, the
// high parts, the middle ones, the low ones.
__device__ __forceinline__ void stage_rows(const W4Params& p, bf16* to, int stride, int rows, int k0, int count) {
    const int pieces = count / 8;
    for (int i = threadIdx.x; i < rows * pieces; i += W4_THREADS) {
        const int r = i / pieces, k = k0 + (i - r * pieces) * 8;
        bf16* dst = to + (size_t)r * stride + (k - k0);
        if (!p.f32) {
            const bf16* src = static_cast<const bf16*>(p.x) + (long long)r * p.ldx + k;
            if (p.vectors) {
                const int bytes = k < p.K ? 16 : 0;         // (whole pieces: K is a multiple of 8 here)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                             ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(bytes ? src : static_cast<const bf16*>(p.x)), "r"(bytes) : "memory");
            } else {
                unsigned short v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = k + e < p.K ? reinterpret_cast<const unsigned short*>(src)[e] : (unsigned short)0;
                *reinterpret_cast<uint4*>(dst) = make_uint4(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16,
                                                            v[4] | (unsigned)v[5] << 16, v[6] | (unsigned)v[7] << 16);
            }
        } else {
            const float* src = static_cast<const float*>(p.x) + (long long)r * p.ldx + k;
            float f[8];
            if (p.vectors && k < p.K) {
                const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
                f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = k + e < p.K ? src[e] : 0.f;
            }
            unsigned short v[8][3];
#pragma unroll
            for (int e = 0; e < 8; ++e) three(f[e], v[e]);
#pragma unroll
            for (int q = 0; q < 3; ++q)
                *reinterpret_cast<uint4*>(dst + (size_t)q * rows * stride) =
                    make_uint4(v[0][q] | (unsigned)v[1][q] << 16, v[2][q] | (unsigned)v[3][q] << 16,
                               v[4][q] | (unsigned)v[5][q] << 16, v[6][q] | (unsigned)v[7][q] << 16);
        }
    }
}

// NT: eights of staged rows; SP: strips of a warp; AHEAD: chunks that it has under way; HALVES: groups of 32, two a chunk.
template <int NT, int SP, int AHEAD, int CTAS, bool HALVES, bool ZEROS>
__global__ void __launch_bounds__(W4_THREADS, CTAS)
w4_kernel(const W4Params p) {
    extern __shared__ __align__(16) unsigned char w4_smem[];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int side = warp % p.ws, turn = warp / p.ws;
    const int rows = p.rows;
    constexpr int GROUPS = HALVES ? 2 : 1;                  // of a chunk
    const int strips_of_tile = p.ws * SP, tiles = (p.strips + strips_of_tile - 1) / strips_of_tile;
    const int mine = turn < p.chunks ? (p.chunks - turn + p.wk - 1) / p.wk : 0;         // this warp's chunks of a tile

    struct Item { uint4 w[SP]; unsigned s[SP][GROUPS]; unsigned z[ZEROS ? SP : 1][GROUPS]; };
    // ---- the loads: chunks one after another, tile after tile.  (Places in 32 bits: of 16 bytes, of pairs of scales.) ----
    int load_tile = blockIdx.x, load_i = 0;
    unsigned words[SP], groups[SP];
    auto aim = [&]() {
#pragma unroll
        for (int s = 0; s < SP; ++s) {
            const unsigned strip = (unsigned)min(load_tile * strips_of_tile + side * SP + s, p.strips - 1);
            words[s] = ((strip / 8 * (unsigned)p.chunks + turn) * 8 + strip % 8) * 32 + lane;
            groups[s] = strip * (unsigned)p.groups * 8 + g;
        }
    };
    auto load = [&](Item& it, int i) {
        if (load_tile < tiles && i < mine) {
            const int c = turn + p.wk * i;
#pragma unroll
            for (int s = 0; s < SP; ++s) {
                it.w[s] = load_stream(p.words + words[s]);
                words[s] += p.wk * (8 * 32);
#pragma unroll
                for (int h = 0; h < GROUPS; ++h) {
                    const unsigned a = groups[s] + 8 * (HALVES ? min(2 * c + h, p.groups - 1) : (2 * c) >> p.group_shift);
                    it.s[s][h] = __ldg(p.scales + a);
                    if (ZEROS) it.z[s][h] = __ldg(p.zeros + a);
                }
            }
        }
    };
    // behind AHEAD loads: the chunks of a tile are taken AHEAD at a time, and the next tile's follow
    auto advance = [&]() {
        load_i += AHEAD;
        if (load_i >= mine) {
            load_i = 0;
            load_tile += gridDim.x;
            if (load_tile < tiles) aim();
        }
    };
    Item ring[AHEAD];
    aim();
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load(ring[u], u);       // (weights do not come from the kernel before)
    advance();
    pdl_wait();

    const int count = p.stage_chunks * W4_CHUNK, stride = count + W4_PAD;
    bf16* x_smem = reinterpret_cast<bf16*>(w4_smem);
    const size_t buffer = (size_t)NT * 8 * stride;          // elements
    const int buffers = p.stages > 1 ? 2 : 1;
    const int cols = strips_of_tile * W4_STRIP, pitch = cols + 1;
    float* part = reinterpret_cast<float*>(x_smem + buffers * buffer);          // [two][turn][staged row][column]
    const int part_floats = p.wk * NT * 8 * pitch;

    stage_rows(p, x_smem, stride, rows, 0, count);
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    const int per_stage = p.stage_chunks / p.wk;
    bool staged = false;                                    // (x in one stage: it stays)
    int stages_done = 0, flip = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, flip ^= 1) {
        float total[SP][NT][4];
#pragma unroll
        for (int s = 0; s < SP; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) total[s][n][e] = 0.f;
        for (int stage = 0; stage < p.stages; ++stage) {
            const int now = p.stages > 1 ? stages_done & 1 : 0;
            if (!staged) {
                // the stage that was ordered last is here; the next one, of the next tile's behind this tile's last, is ordered
                asm volatile("cp.async.wait_group 0;\n" ::: "memory");
                __syncthreads();
                if (p.stages > 1) {
                    if (stage + 1 < p.stages || tile + (int)gridDim.x < tiles)
                        stage_rows(p, x_smem + (now ^ 1) * buffer, stride, rows, (stage + 1 < p.stages ? stage + 1 : 0) * count, count);
                    asm volatile("cp.async.commit_group;\n" ::: "memory");
                    ++stages_done;
                }
                staged = p.stages == 1;
            }
            const bf16* x_lane = x_smem + now * buffer + (size_t)g * stride + t * 4 + turn * W4_CHUNK;
            // (chunks of the stage: per_stage of this warp's, in steps of AHEAD, per_stage being a multiple of that where there are several stages)
            for (int i = stage * per_stage; i < min(mine, (stage + 1) * per_stage); i += AHEAD) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    Item& it = ring[u];
                    if (i + u < mine) {                     // (uniform in the warp)
                    const int local = (i + u - stage * per_stage) * p.wk;
                    const bf16* xc = x_lane + local * W4_CHUNK;
                    float sum[SP][NT][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint2 x[NT][2];
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < 2; ++j) x[n][j] = *reinterpret_cast<const uint2*>(xc + (size_t)n * 8 * stride + 32 * h + 16 * j);
                        if (h == 0 || HALVES) {
#pragma unroll
                            for (int s = 0; s < SP; ++s)
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) sum[s][n][e] = 0.f;
                        }
#pragma unroll
                        for (int s = 0; s < SP; ++s) {
                            // 128 + zero of the columns g and g + 8
                            const unsigned z = ZEROS ? it.z[ZEROS ? s : 0][HALVES ? h : 0] : 0x0808u;
                            const unsigned low = 0x43004300u | (z & 0xffu) * 0x00010001u, high = 0x43004300u | (z >> 8) * 0x00010001u;
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const unsigned w = h ? (j ? it.w[s].w : it.w[s].z) : (j ? it.w[s].y : it.w[s].x);
                                const unsigned a[4] = {w4_pair(w, low), w4_pair(w >> 4, high),
                                                       w4_pair(w >> 8, low), w4_pair(w >> 12, high)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma_bf16(sum[s][n], a, x[n][j].x, x[n][j].y);
                            }
                            if (h == 1 || HALVES) {
                                const unsigned sc = it.s[s][HALVES ? h : 0];
                                const float s0 = low_half(sc), s1 = high_half(sc);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    total[s][n][0] = fmaf(sum[s][n][0], s0, total[s][n][0]);
                                    total[s][n][1] = fmaf(sum[s][n][1], s0, total[s][n][1]);
                                    total[s][n][2] = fmaf(sum[s][n][2], s1, total[s][n][2]);
                                    total[s][n][3] = fmaf(sum[s][n][3], s1, total[s][n][3]);
                                }
                            }
                        }
                    }
                    }
                    load(it, load_i + u);                   // its place is free: the chunk AHEAD further
                }
                advance();
            }
        }
        // ---- the warps' turns added up, float32's three parts too, and stored.  Two tiles' sums lie side by
        // side: a warp may be a tile ahead of the slowest, not two ----
        float* here = part + flip * part_floats;
#pragma unroll
        for (int s = 0; s < SP; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    here[((size_t)turn * NT * 8 + n * 8 + t * 2 + (e & 1)) * pitch + (side * SP + s) * W4_STRIP + g + (e >> 1) * 8] = total[s][n][e];
        __syncthreads();
        const int first = tile * cols;
        for (int i = threadIdx.x; i < rows * cols; i += W4_THREADS) {
            const int r = i / cols, c = i - r * cols;
            if (first + c >= p.N) continue;
            float v[3] = {0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < 3; ++q)
                for (int w = 0; w < (q == 0 || p.f32 ? p.wk : 0); ++w) v[q] += here[((size_t)w * NT * 8 + q * rows + r) * pitch + c];
            const long long at = (long long)r * p.ldo + first + c;
            if (p.f32) static_cast<float*>(p.out)[at] = of_three(v[0], v[1], v[2]);
            else static_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(v[0]);
        }
    }
}

// Shared memory of a CTA: `eights` of staged rows, strips of a warp, warps side by side and in turns, chunks of a stage; and what two CTAs of an SM have.
constexpr size_t W4_SMEM = 224 * 1024 / 2;
constexpr size_t w4_bytes(int eights, int sp, int ws, int wk, int stage_chunks, int buffers) {
    return (size_t)eights * 8 * ((size_t)stage_chunks * W4_CHUNK + W4_PAD) * 2 * buffers + (size_t)2 * wk * eights * 8 * (ws * sp * W4_STRIP + 1) * 4;
}
// Strips of a warp: two where that leaves all CTAs some, and the registers take it.
constexpr int w4_side(int eights, int strips) { return eights == 2 || (eights == 1 && strips > 2 * 148) ? 2 : 1; }
// Chunks of x in one piece: every warp has as many turns.
constexpr int w4_whole(int chunks) { return (chunks + W4_WARPS - 1) / W4_WARPS * W4_WARPS; }
constexpr bool w4_one_piece(int eights, int sp, int chunks) { return w4_bytes(eights, sp, 1, W4_WARPS, w4_whole(chunks), 1) <= W4_SMEM; }

template <int NT, int SP, int AHEAD, int CTAS, bool HALVES, bool ZEROS> int w4_launch(W4Params p, cudaStream_t stream) {
    // x in one stage where it fits: all warps share out the sum.  Else four of them stand side by side, for fewer passes over x.
    p.ws = 1;
    p.wk = W4_WARPS;
    p.stages = 1;
    p.stage_chunks = w4_whole(p.chunks);
    if (!w4_one_piece(NT, SP, p.chunks)) {
        p.ws = 4;
        p.wk = W4_WARPS / p.ws;
        const int unit = p.wk * AHEAD;
        p.stage_chunks = unit;
        while (w4_bytes(NT, SP, p.ws, p.wk, p.stage_chunks + unit, 2) <= W4_SMEM) p.stage_chunks += unit;
        p.stages = (p.chunks + p.stage_chunks - 1) / p.stage_chunks;
    }
    const size_t smem = w4_bytes(NT, SP, p.ws, p.wk, p.stage_chunks, p.stages > 1 ? 2 : 1);
    static DeviceOnce configured;
    if (configured([&] { return cudaFuncSetAttribute(w4_kernel<NT, SP, AHEAD, CTAS, HALVES, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024); }) != cudaSuccess)
        return tis_check_launch("gemm_w4 (shared memory)");
    if (smem > 227 * 1024) {
        tis_set_error("gemm_w4: %zu bytes of shared memory", smem);
        return TIS_BAD_SIZE;
    }
    const int tiles = (p.strips + p.ws * SP - 1) / (p.ws * SP);
    const int most = CTAS * 148;
    tis_launch(w4_kernel<NT, SP, AHEAD, CTAS, HALVES, ZEROS>, dim3((unsigned)(tiles < most ? tiles : most)), dim3(W4_THREADS), smem, stream, p);
    return tis_check_launch("gemm_w4");
}

template <int NT, int SP, int AHEAD, int CTAS, bool HALVES> int w4_zeros(const W4Params& p, cudaStream_t stream) {
    return p.zeros != nullptr ? w4_launch<NT, SP, AHEAD, CTAS, HALVES, true>(p, stream) : w4_launch<NT, SP, AHEAD, CTAS, HALVES, false>(p, stream);
}
template <int NT, int SP, int AHEAD, int CTAS> int w4_forms(const W4Params& p, cudaStream_t stream) {
    return p.group_shift == 0 ? w4_zeros<NT, SP, AHEAD, CTAS, true>(p, stream) : w4_zeros<NT, SP, AHEAD, CTAS, false>(p, stream);
}

}  // namespace

// Whether the mma.sync kernel holds `staged` rows of x (a row of float32 is three) in one piece, for the choice between the two.
TIS_API int tis_gemm_w4_one_piece(int staged, int K, int N) {
    const int eights = (staged + 7) / 8, strips = (N + W4_STRIP - 1) / W4_STRIP;
    return w4_one_piece(eights, w4_side(eights, strips), (K + W4_CHUNK - 1) / W4_CHUNK);
}

// out (rows, N) = x (rows, K) times the packed weights; dtype is that of x and out, rows of both contiguous, row strides free.
struct W4Args { long long dtype, x, ldx, words, scales, zeros, out, ldo, rows, K, N, group, tensor, copy, fault, stream; };
TIS_API int tis_gemm_w4(const W4Args* a) {
    if (a->K <= 0 || a->K > (1 << 30) || a->N > (1 << 30) || a->rows > (1 << 30) || a->group < 32 || a->group > (1 << 30) ||
        (a->group & (a->group - 1)) != 0 || a->K * a->N > (1ll << 36)) {
        tis_set_error("gemm_w4: %lld rows, %lld x %lld in groups of %lld", a->rows, a->K, a->N, a->group);
        return TIS_BAD_SIZE;
    }
    const int dtype = (int)a->dtype, rows = (int)a->rows, K = (int)a->K, N = (int)a->N, group = (int)a->group;
    const void* x = reinterpret_cast<const void*>(a->x);
    const long long ldx = a->ldx;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
    if (rows <= 0 || N <= 0) return TIS_OK;
    if (dtype != TIS_F32 && dtype != TIS_BF16) {
        tis_set_error("gemm_w4: dtype code %d", dtype);
        return TIS_BAD_DTYPE;
    }
    W4Params p = {};
    p.words = reinterpret_cast<const uint4*>(a->words);
    p.scales = reinterpret_cast<const unsigned*>(a->scales);
    p.zeros = reinterpret_cast<const unsigned short*>(a->zeros);
    p.x = x; p.ldx = ldx; p.out = reinterpret_cast<void*>(a->out); p.ldo = a->ldo;
    p.rows = rows; p.K = K; p.N = N;
    p.chunks = (K + W4_CHUNK - 1) / W4_CHUNK;
    p.strips = (N + W4_STRIP - 1) / W4_STRIP;
    p.groups = (int)(((long long)K + group - 1) / group);
    for (int h = group / 32; h > 1; h >>= 1) ++p.group_shift;
    p.f32 = dtype == TIS_F32;
    p.vectors = K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % (p.f32 ? 4 : 8) == 0;
    if (a->tensor) {
        if (a->copy == 0 && (p.f32 || !p.vectors)) {
            tis_set_error("gemm_w4: the tcgen05 kernel takes bfloat16 rows that start on 16 bytes, or room to copy them to");
            return TIS_BAD_SIZE;
        }
        return w4_tc_launch(p, reinterpret_cast<void*>(a->copy), reinterpret_cast<int*>(a->fault), stream);
    }
    if ((p.f32 ? 3ll : 1ll) * rows > W4_STAGED) {
        tis_set_error("gemm_w4: %d rows, of which the mma.sync kernel takes %d", rows, p.f32 ? W4_STAGED / 3 : W4_STAGED);
        return TIS_BAD_SIZE;
    }
    const int eights = ((p.f32 ? 3 : 1) * rows + 7) / 8;
    switch (eights) {
        case 1: return w4_side(1, p.strips) == 1 ? w4_forms<1, 1, 4, 2>(p, stream) : w4_forms<1, 2, 4, 2>(p, stream);
        case 2: return w4_forms<2, 2, 2, 2>(p, stream);
        default: return w4_forms<3, 1, 4, 2>(p, stream);
    }
}
