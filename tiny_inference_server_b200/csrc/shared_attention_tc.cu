// Shared tiles of attention over a shared prefix (shared_attention.cuh) on the fifth-generation tensor cores: head sizes 64 and
// 128, pages of 16, 32, 64 or 128 keys, bfloat16.
//
// A CTA has up to 128 row heads of one kv head (rows of different requests, and the heads of a row, side by side: they all see the same
// keys) and a part of the shared keys, 128 at a time.  The roles are those of attention_tc.cu, which walks a prompt's rows: two pairs
// of loading warps (keys, values; boxes of 64 elements x a page's rows, which the cache's permutation makes swizzled operand tiles), two
// warps that issue the products, two groups of four softmax warps with a score buffer, a probability buffer and an output accumulator each
// that take tiles in turns.  Different here: the row heads are gathered by the softmax warps, since a tile's rows are no box of the
// queries; no key is masked but those behind the part's end in its last tile, since every row sees all shared keys; and the part leaves its
// sums in 32 bits for the join instead of a result.
// Bound, with 128 row heads a tile, by the chain of a tile, scores to maximum to exponentials to products: about 1800 cycles for 128 x 128 scores, of which
// the products alone take 1050 and the exponentials, 16 a cycle, 1024.  (The schedulers issue in 46 % of the cycles; a warp waits 1.8 cycles an instruction at barriers,
// 1.8 for a result, 1.7 for tensor memory.)  With few row heads by the bytes, or by code that runs once: with 16 requests behind 4096 keys, a tile or two a CTA,
// a warp waits 4.8 of 23 cycles for instructions and 8.8 at barriers.
// Measured: 64 rows of 32 heads on 8 of 128 behind 32768 keys (34 GFLOP) some 42 us, 0.8 PFLOP/s, and with the requests' own keys beside it 96 us;
// the same on mma.sync 326 us.
// All hand-offs are mbarriers with bounded waits; a wait that runs out sets the fault word and every role leaves; tensor memory is
// freed on every path.
#include "tc_common.cuh"
#include "shared_attention.cuh"

#ifndef TIS_HD
#define TIS_HD 128
#endif

#if TIS_HD == 64 || TIS_HD == 128

namespace {

using namespace tc;
using namespace shared_attention;

constexpr int HD = TIS_HD;
constexpr int HALVES = HD / 64;             // 128-byte column blocks of a row
constexpr int BM = 128;                     // row heads of a CTA
constexpr int BN = 128;                     // keys of a tile
constexpr int NTH = 512;
constexpr int HALF_BYTES = 128 * 128;       // 128 rows x 128 bytes: one swizzled column block
constexpr int Q_BYTES = HALVES * HALF_BYTES;
constexpr int P_BYTES = 2 * HALF_BYTES;     // 128 rows x 128 keys, bfloat16 (one per softmax group)
constexpr int SLOT_BYTES = HALVES * HALF_BYTES;   // keys or values of one tile
constexpr int SLOTS = HD == 128 ? 2 : 4;    // per ring (keys, values)
constexpr int PAGES_AHEAD = 3;
constexpr unsigned TMEM_COLS = 512;
constexpr unsigned COL_S = 0;               // two score buffers of 128 columns
constexpr unsigned COL_O = 256;             // two output accumulators of up to 128 columns
constexpr float RESCALE_STEP = 8.f;         // in units of log2

__global__ void __launch_bounds__(NTH, 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap map_kv, const SharedParams p, const SharedTile* tiles, int parts) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_smem = base;
    unsigned char* p_smem = base + Q_BYTES;
    unsigned char* k_slots = p_smem + 2 * P_BYTES;
    unsigned char* v_slots = k_slots + SLOTS * SLOT_BYTES;
    __shared__ unsigned long long q_full, full_k[SLOTS], empty_k[SLOTS], full_v[SLOTS], empty_v[SLOTS], s_full[2], s_free[2], p_full[2], o_done[2], turn[2];
    __shared__ unsigned tmem_base_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % p.KVH, part = blockIdx.x / p.KVH % parts;
    const SharedTile t = tiles[blockIdx.x / p.KVH / parts];             // (the plan's, from before the batch)
    const int G = p.H / p.KVH;
    const Range keys = part_range(0, shared_keys(p, t), 0, part, parts, BN);
    const int T = keys.hi > keys.lo ? (keys.hi - keys.lo + BN - 1) / BN : 0;
    auto place = [&](int i) { const int rh = t.rh0 + i; return ((size_t)part * p.rows + rh / G) * p.H + kvh * G + rh % G; };
    if (T == 0) {                                           // nothing of this group in this part: the whole CTA leaves together
        pdl_wait();
        pdl_launch_dependents();
        if ((int)threadIdx.x < t.count) p.part_ml[place(threadIdx.x)] = make_float2(-INFINITY, 0.f);
        return;
    }

    if (threadIdx.x == 0) {
        mbar_init(&q_full, 8);
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&full_k[s], 2); mbar_init(&empty_k[s], 1);
            mbar_init(&full_v[s], 2); mbar_init(&empty_v[s], 1);
        }
        mbar_init(&s_full[0], 1); mbar_init(&s_full[1], 1);
        mbar_init(&s_free[0], 4); mbar_init(&s_free[1], 4);
        mbar_init(&p_full[0], 4); mbar_init(&p_full[1], 4);
        mbar_init(&turn[0], 4); mbar_init(&turn[1], 4);
        mbar_init(&o_done[0], 1); mbar_init(&o_done[1], 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_map(&map_kv);
    }
    if (warp == 1) tmem_alloc(&tmem_base_slot, TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem_base = tmem_base_slot;
    volatile int* abort = &abort_flag;
    pdl_wait();                                             // queries, tables and the cache's rows come from the kernels before
    // Only now: the kernel of the requests' own keys starts beside this one, when all CTAs of this one are here, and waits for it at its
    // end; what both read is complete by then.
    pdl_launch_dependents();

    // 512 threads are launched with 128 registers each, 65536 in all: 256 x 40 + 256 x 216
    if (warp < 4 || warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n" ::);
        if (warp == 0 || warp == 2 || warp == 12 || warp == 13) {
            // ---- loads: warps 0 and 12 keys, warps 2 and 13 values --------------------------------------
            const int kv = warp == 0 || warp == 12 ? 0 : 1, half_of = warp >= 12 ? 1 : 0;
            unsigned long long* full = kv ? full_v : full_k;
            unsigned long long* empty = kv ? empty_v : empty_k;
            unsigned char* ring = kv ? v_slots : k_slots;
            const int boxes = BN / p.page * HALVES;                             // of a key tile
            const bool mine = lane < boxes && (lane & 1) == half_of;            // a lane a box, the two warps taking turns
            const int part_bytes = (boxes + 1 - half_of) / 2 * p.page * 128, in_tile = lane / HALVES * p.page;
            // the page of a lane's keys in tile j, on its way PAGES_AHEAD tiles before its copies are ordered.  Behind the part's end (whole
            // pages) a box begins behind the cache's last row, which brings zeros: a masked key's probability of 0 takes no other value away.
            auto behind = [&](int j) { return keys.lo + j * BN + in_tile >= keys.hi; };
            const int behind_all = p.num_pages * 2 * p.KVH * p.page;            // (below 2^31: the launcher)
            auto page_of = [&](int j) -> int {
                if (j >= T || !mine || behind(j)) return 0;
                const int index = (keys.lo + j * BN + in_tile) / p.page;
                return index < p.table_width ? p.table[(size_t)t.slot * p.table_stride + index] : -1;
            };
            int pages[PAGES_AHEAD];
#pragma unroll
            for (int a = 0; a < PAGES_AHEAD; ++a) pages[a] = page_of(a);
            for (int j = 0; j < T; ++j) {
                int page = pages[0];
#pragma unroll
                for (int a = 1; a < PAGES_AHEAD; ++a) pages[a - 1] = pages[a];
                pages[PAGES_AHEAD - 1] = page_of(j + PAGES_AHEAD);
                const int s = j % SLOTS;
                if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((j / SLOTS) & 1) ^ 1, abort, p.fault, 6))) break;
                if (page < 0 || page >= p.num_pages) { atomicExch(p.fault, 3); page = 0; }
                if (lane == 0) mbar_arrive_expect_tx(&full[s], part_bytes);
                __syncwarp();
                if (mine) {
                    const int half = lane % HALVES;
                    tma_load_2d(ring + (size_t)s * SLOT_BYTES + half * HALF_BYTES + in_tile * 128, &map_kv, half * 64,
                                behind(j) ? behind_all : ((page * 2 + kv) * p.KVH + kvh) * p.page, &full[s]);
                }
            }
        } else if (warp == 1) {
            // ---- products, first kind: S_j = Q K_j^T into score buffer j & 1 ----------------------------
            constexpr unsigned IDESC_S = instr_desc(BM, BN, false);
            const unsigned long long q_desc0 = smem_desc(smem_u32(q_smem), 16, 1024);
            const unsigned long long k_desc0 = smem_desc(smem_u32(k_slots), 16, 1024);
            bool ok = mbar_wait(&q_full, 0, abort, p.fault, 6);
            for (int j = 0; j < T; ++j) {
                const int g = j & 1, i = j >> 1, s = j % SLOTS;
                // the group has the scores of its tile before in registers
                ok = ok && (i > 0 ? mbar_wait_both(&s_free[g], (i - 1) & 1, &full_k[s], (j / SLOTS) & 1, abort, p.fault, 6)
                                  : mbar_wait(&full_k[s], (j / SLOTS) & 1, abort, p.fault, 6));
                if (!__all_sync(0xffffffffu, ok)) break;
                fence_after();
                if (elect_one()) {
                    const unsigned long long kd = k_desc0 + (unsigned long long)((s * SLOT_BYTES) >> 4);
                    const unsigned d = tmem_base + COL_S + g * BN;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const unsigned long long off = (unsigned long long)(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4);
                        umma(d, q_desc0 + off, kd + off, IDESC_S, kk != 0);
                    }
                    umma_commit(&empty_k[s]);
                    umma_commit(&s_full[g]);
                }
                __syncwarp();
            }
        } else if (warp == 3) {
            // ---- products, second kind: O_g += P_j V_j ---------------------------------------------------
            constexpr unsigned IDESC_O = instr_desc(BM, HD, true);
            const unsigned long long p_desc0 = smem_desc(smem_u32(p_smem), 16, 1024);
            const unsigned long long v_desc0 = smem_desc(smem_u32(v_slots), HALF_BYTES, 1024);
            for (int j = 0; j < T; ++j) {
                const int g = j & 1, i = j >> 1, s = j % SLOTS;
                if (!__all_sync(0xffffffffu, mbar_wait_both(&p_full[g], i & 1, &full_v[s], (j / SLOTS) & 1, abort, p.fault, 6))) break;
                fence_after();
                if (elect_one()) {
                    const unsigned long long vd = v_desc0 + (unsigned long long)((s * SLOT_BYTES) >> 4);
                    const unsigned long long pd = p_desc0 + (unsigned long long)((g * P_BYTES) >> 4);
                    const unsigned d = tmem_base + COL_O + g * 128;
#pragma unroll
                    for (int kk = 0; kk < BN / 16; ++kk) {    // 16 keys: 32 bytes along a row of P, 16 rows of V
                        umma(d, pd + (unsigned long long)(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4),
                             vd + (unsigned long long)((kk * 2048) >> 4), IDESC_O, (i | kk) != 0);
                    }
                    umma_commit(&empty_v[s]);
                    umma_commit(&o_done[g]);
                }
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n" ::);
        // ---- softmax: one thread per row head in each of the two groups ----------------------
        const int g = warp >= 8 ? 1 : 0;                  // warps 4-7 and 8-11
        const int quarter = warp & 3;                     // the lanes of tensor memory this warp may touch
        const int r = quarter * 32 + lane;
        // the queries, 16-byte pieces, all loads of a thread on their way at once: rows of 128 swizzled bytes, zero beyond the tile
        constexpr int PIECES = BM * HD / 8 / 256;
        uint4 piece[PIECES];
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            const int i = threadIdx.x - 128 + n * 256, row = i / (HD / 8), c = i % (HD / 8);
            piece[n] = make_uint4(0u, 0u, 0u, 0u);
            if (row < t.count) {
                const int rh = t.rh0 + row;
                piece[n] = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (long long)(rh / G) * p.ldq + (kvh * G + rh % G) * HD + c * 8);
            }
        }
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            const int i = threadIdx.x - 128 + n * 256, row = i / (HD / 8), c = i % (HD / 8);
            *reinterpret_cast<uint4*>(q_smem + (c >> 3) * HALF_BYTES + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = piece[n];
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
        // a row before the end of the shared keys is padding: it sees nothing
        const bool row_ok = r < t.count && p.positions[(t.rh0 + min(r, t.count - 1)) / G] >= t.prefix;
        const unsigned lane_bits = (unsigned)(quarter * 32) << 16;
        const unsigned col_s = COL_S + g * BN, col_o = COL_O + g * 128;
        unsigned char* pg_smem = p_smem + g * P_BYTES;
        const bool warp_has_rows = __any_sync(0xffffffffu, row_ok);
        float m_used = -INFINITY, l_sum = 0.f;
        bool ok = true;
        // before the exponentials of the group's tile i: the products of its tile before are done, and the other group's exponentials of
        // the tile before in the row's order
        auto wait_turn = [&](int i) {
            if (g == 0) return i == 0 || mbar_wait_both(&o_done[0], (i - 1) & 1, &turn[0], (i - 1) & 1, abort, p.fault, 6);
            return i == 0 ? mbar_wait(&turn[1], 0, abort, p.fault, 6)
                          : mbar_wait_both(&o_done[1], (i - 1) & 1, &turn[1], i & 1, abort, p.fault, 6);
        };
        int i = 0;                                        // tiles of this group so far
        for (int j = g; j < T; j += 2, ++i) {
            if (!__all_sync(0xffffffffu, mbar_wait(&s_full[g], i & 1, abort, p.fault, 6))) { ok = false; break; }
            fence_after();
            if (!warp_has_rows) {
                // a warp without rows: its rows of P are zero, once and for all.  It follows every phase of o_done and turn all the same: a
                // wait for the last one alone could return a phase early
                if (i == 0) {
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        *reinterpret_cast<uint4*>(pg_smem + r * 128 + (c >> 3) * HALF_BYTES + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                if (!__all_sync(0xffffffffu, wait_turn(i))) { ok = false; break; }
                if (lane == 0) mbar_arrive(&turn[1 - g]);
                fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&s_free[g]); mbar_arrive(&p_full[g]); }
                continue;
            }
            float s[BN];
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) tmem_ld32_issue(tmem_base + lane_bits + col_s + c * 32, s + c * 32);
            tmem_ld_wait();
            tmem_ld_arrived(s);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[g]);
            const int left = keys.hi - keys.lo - j * BN;                // keys of the part from this tile on
            if (left < BN || !row_ok) {
                const int seen = row_ok ? left : 0;
#pragma unroll
                for (int e = 0; e < BN; ++e) s[e] = e < seen ? s[e] : -INFINITY;
            }
            // the row's maximum (the scale is positive), four chains side by side
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < BN; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], s[e]);
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
            // raise the reference maximum only when the row's maximum left it far behind
            const bool raise = mx > m_used + RESCALE_STEP || (m_used == -INFINITY && mx > -INFINITY);
            float alpha = 1.f;
            if (raise) {
                // (a row without a maximum has no sums yet but what is not a number: that stays)
                alpha = m_used == -INFINITY ? 1.f : exp2_fast(m_used - mx);
                m_used = mx;
                l_sum *= alpha;
            }
            // the products of the group's tile before are done: O may be rescaled, P overwritten
            if (!__all_sync(0xffffffffu, wait_turn(i))) { ok = false; break; }
            if (i > 0 && __any_sync(0xffffffffu, raise)) {
                fence_after();
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    float o[32];
                    tmem_ld32(tmem_base + lane_bits + col_o + c * 32, o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] *= alpha;
                    tmem_st32(tmem_base + lane_bits + col_o + c * 32, o);
                }
                fence_before();
            }
            const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
            float ps4[4] = {0.f, 0.f, 0.f, 0.f};
            unsigned char* prow = pg_smem + r * 128;
#pragma unroll
            for (int c = 0; c < BN / 8; ++c) {            // eight keys: one 16-byte chunk of the row of P
                // (probabilities in bfloat16, half a step, 2^-9 of each, at random: the operand's type; their sum stays in 32 bits)
                unsigned pk[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float a = exp2_fast(fmaf(s[c * 8 + e], p.scale_log2, neg_m));       // 2^-inf = 0 for masked keys
                    const float b = exp2_fast(fmaf(s[c * 8 + e + 1], p.scale_log2, neg_m));
                    ps4[e >> 1] += a + b;
                    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                    pk[e >> 1] = *reinterpret_cast<unsigned*>(&h);
                }
                *reinterpret_cast<uint4*>(prow + (c >> 3) * HALF_BYTES + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                if (c == BN / 16 - 1 && lane == 0) mbar_arrive(&turn[1 - g]);
            }
            l_sum += (ps4[0] + ps4[1]) + (ps4[2] + ps4[3]);
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[g]);
        }
        // ---- merge the two groups' halves, each group half of the columns, and leave them through the ring of keys, which has no
        // more copies or products to come once both groups' last products are done --------------------------
        typedef StagedRows<HD> Rows;
        float* stage = reinterpret_cast<float*>(k_slots);
        if (i > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[g], (i - 1) & 1, abort, p.fault, 6));
        // the group's P buffer is free now: it carries the row's maximum and sum to the other group
        reinterpret_cast<float*>(pg_smem)[r] = m_used;
        reinterpret_cast<float*>(pg_smem)[BM + r] = l_sum;
        fence_before();
        asm volatile("bar.sync 1, 256;\n" ::: "memory");        // both groups' products are done, sums are in place
        fence_after();
        if (ok && !*abort) {
            const float* mg0 = reinterpret_cast<const float*>(p_smem);
            const float* mg1 = reinterpret_cast<const float*>(p_smem + P_BYTES);
            const float m0 = mg0[r], m1 = mg1[r], l0 = mg0[BM + r], l1 = mg1[BM + r];
            const float m = fmaxf(m0, m1);
            const float w0 = m0 == -INFINITY ? 1.f : exp2_fast(m0 - m), w1 = m1 == -INFINITY ? 1.f : exp2_fast(m1 - m);
            if (g == 0 && r < t.count) p.part_ml[place(r)] = row_ok ? make_float2(m, l0 * w0 + l1 * w1) : make_float2(-INFINITY, 0.f);
            constexpr int COLS = HD / 2;                  // this group's share of the columns
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
                const int col = g * COLS + c * 32;
                float o0[32], o1[32];
                tmem_ld32_issue(tmem_base + lane_bits + COL_O + col, o0);
                if (T >= 2) tmem_ld32_issue(tmem_base + lane_bits + COL_O + 128 + col, o1);
                tmem_ld_wait();
                tmem_ld_arrived(o0);
                if (T >= 2) tmem_ld_arrived(o1);
#pragma unroll
                for (int e = 0; e < 32; ++e) o0[e] = o0[e] * w0 + (T >= 2 ? o1[e] * w1 : 0.f);
                stage_put<HD>(stage, r, col, o0);
            }
            fence_before();
        }
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        if (!*abort) {
            const int first = Rows::row(warp - 4, lane, 0), col = Rows::col(lane);
#pragma unroll 4
            for (int i = 0; i < Rows::STEPS; ++i) {
                const int row = first + i * Rows::ROWS;
                if (row < t.count) *reinterpret_cast<float4*>(p.part_o + place(row) * HD + col) = Rows::get(stage, row, col);
            }
        }
    }

    if (*abort) {
        // a wait ran out: give copies that may still be in flight time to land before the shared memory is given up
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_free(tmem_base, TMEM_COLS);
    }
}

}  // namespace

bool shared_tc_takes(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

int shared_tc_launch(const SharedParams& p, const SharedTile* tiles, int count, int parts, cudaStream_t stream) {
    CUtensorMap map;
    if (!tensor_map(p.plane, HD, (long long)p.num_pages * 2 * p.KVH * p.page, HD, p.page, false, &map)) return TIS_CUDA_ERROR;
    constexpr int smem = Q_BYTES + 2 * P_BYTES + 2 * SLOTS * SLOT_BYTES + 1024;
    static DeviceOnce configured;
    if (configured([&] { return cudaFuncSetAttribute(shared_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }) != cudaSuccess)
        return tis_check_launch("shared_prefix_attention (shared memory)");
    tis_launch(shared_tc_kernel, dim3((unsigned)(count * parts * p.KVH)), dim3(NTH), (size_t)smem, stream, map, p, tiles, parts);
    return tis_check_launch("shared_prefix_attention");
}

#else

bool shared_tc_takes(int) { return false; }
int shared_tc_launch(const SharedParams&, const SharedTile*, int, int, cudaStream_t) { return TIS_BAD_SIZE; }

#endif
