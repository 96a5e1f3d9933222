// Attention over a shared prefix (shared_attention.cuh): the kernel of the requests' own keys, also of shared keys at head sizes
// and pages that the tcgen05 kernel does not take; the float32 kernel; and the kernel that joins the parts.
//
// The first is bound by the keys' and values' bytes (a request's own keys serve its own few row heads only) or, with few of them, by the
// chain tile -> positions -> pages -> rows.  64 keys a tile come STAGES tiles ahead into shared memory as they are stored, one bulk copy a page
// and operand, ordered by the lanes of a warp, a lane a page (rows are dense in a page; their permuted chunks are free of bank
// conflicts for ldmatrix).  Four warps: with at most 16 row heads each takes a quarter of every tile's keys and they merge at the end; shared
// tiles of up to 64 or 128 row heads give each warp 16 or 32 of them and all keys, so that an operand of keys or values read from shared
// memory serves 32.
// Measured, both kernels and where there is one the join: 2 requests behind 128 keys, 12 heads on 3 of 128, 8.4 us (the chain); 16 behind 4096 with up to
// 512 own keys 16.7 us; in float32 4 behind 1000, heads of 64, 12.6 us.  Own keys of 64 requests, up to 1024 each, 8 kv heads of 128 (201 MB):
// 40 us, 5 TB/s.
#include "tc_common.cuh"
#include "shared_attention.cuh"

#ifndef TIS_HD
#define TIS_HD 128
#endif

namespace {

using namespace shared_attention;

constexpr int HD = TIS_HD;
constexpr unsigned ALL = 0xffffffffu;
constexpr int MAX_PARTS = 128;

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
constexpr int STAGES = HD <= 64 ? 4 : (HD <= 96 ? 3 : 2);
constexpr int MMA_THREADS = 128, LOAD_THREADS = 32;      // four warps compute, one orders copies
constexpr bool QUERIES_STAY = HD <= 128;     // in registers

__device__ __forceinline__ void bulk_copy(void* to, const void* from, int bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(tc::smem_u32(to)), "l"(from), "r"(bytes), "r"(tc::smem_u32(bar)) : "memory");
}

// A tile's rows: position of row head rh0 + i (-1: beyond the tile, or before the end of the shared keys: it sees nothing)
__device__ __forceinline__ int position_of(const SharedParams& p, const SharedTile& t, int i) {
    if (i >= t.count) return -1;
    const int pos = p.positions[(t.rh0 + i) / (p.H / p.KVH)];
    return pos >= t.prefix ? pos : -1;
}

// The end of a request's keys, for the largest position of its rows + 1: no further than its table goes (what lies behind is marked, not walked).
__device__ __forceinline__ int end_of_keys(const SharedParams& p, int last, bool mark) {
    const long long there = min((long long)p.table_width * p.page, 1ll << 30);
    if (last > there && mark) atomicExch(p.fault, 3);
    return (int)min((long long)last, there);
}

// Chunk c of the cache row of a position (common.cuh: cache_chunk), the position's part worked out once.
struct RowChunks {
    int base;
    __device__ __forceinline__ explicit RowChunks(int position) : base(CHUNKS % 8 == 0 ? position & 7 : position % CHUNKS) {}
    __device__ __forceinline__ int operator()(int c) const {
        if (CHUNKS % 8 == 0) return c ^ base;
        return base + c - (base + c >= CHUNKS ? CHUNKS : 0);
    }
};
// the running maximum is raised when a row's scores leave it behind by more than this (in units of log2: sums stay below 2^8 a key)
constexpr float RAISE_STEP = 8.f;

// The result of row head rh of a kv head from its own part (m, l, o in shared memory) and the shared ones: an eighth of its columns.
__device__ __forceinline__ void join_row(const SharedParams& p, float m, float l, const float* o, int rh, int kvh, int eighth) {
    constexpr int COLS = HD / 8, AHEAD = 4;
    const int G = p.H / p.KVH, row = rh / G, head = kvh * G + rh % G;
    const size_t at = (size_t)row * p.H + head, step = (size_t)p.rows * p.H;
    float M = m;
    for (int q0 = 0; q0 < p.shared_parts; q0 += 8) {
        float x8[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) x8[a] = p.part_ml[at + min(q0 + a, p.shared_parts - 1) * step].x;
#pragma unroll
        for (int a = 0; a < 8; ++a) M = fmaxf(M, x8[a]);
    }
    float f = m == -INFINITY ? 1.f : exp2_fast(m - M), sum = l * f, x[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) x[c] = o[eighth * COLS + c] * f;
    for (int q0 = 0; q0 < p.shared_parts; q0 += AHEAD) {
        float2 v[AHEAD][COLS / 2], ml[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            ml[a] = q0 + a < p.shared_parts ? p.part_ml[at + (q0 + a) * step] : make_float2(-INFINITY, 0.f);
            const bool some = !(ml[a].x == -INFINITY && ml[a].y == 0.f);             // (else no keys: nothing was left there)
            const float2* src = reinterpret_cast<const float2*>(p.part_o + (at + (q0 + a) * step) * HD + eighth * COLS);
#pragma unroll
            for (int c = 0; c < COLS / 2; ++c) v[a][c] = some ? src[c] : make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            f = ml[a].x == -INFINITY ? 1.f : exp2_fast(ml[a].x - M);
            sum += ml[a].y * f;
#pragma unroll
            for (int c = 0; c < COLS / 2; ++c) {
                x[2 * c] = fmaf(v[a][c].x, f, x[2 * c]);
                x[2 * c + 1] = fmaf(v[a][c].y, f, x[2 * c + 1]);
            }
        }
    }
    bf16* dst = static_cast<bf16*>(p.out) + (long long)row * p.ldo + head * HD + eighth * COLS;
#pragma unroll
    for (int c = 0; c < COLS; ++c) x[c] = sum == 0.f ? 0.f : x[c] / sum;
    if (p.out_vectors && COLS % 8 == 0) {
#pragma unroll
        for (int c = 0; c < COLS / 8; ++c) tc::store8(dst + c * 8, x + c * 8);
    } else {
#pragma unroll
        for (int c = 0; c < COLS; ++c) dst[c] = __float2bfloat16_rn(x[c]);
    }
}

// The loading warp's wait for a place that the other warps give back.  They may be waiting for the kernel of the shared tiles, which takes as long as it takes: only
// behind it (`waited`) does a wait that runs out mean a fault.  (Apart: the loop over items stays short.)
__device__ __noinline__ bool wait_given_back(unsigned long long* bar, unsigned parity, volatile int* abort, int* fault, bool& waited) {
    if (!waited) {
        for (int spin = 0; spin < tc::MBAR_SPINS; ++spin) {
            if (tc::mbar_done(bar, parity)) return true;
            if ((spin & 1023) == 1023 && *abort) return false;
        }
        pdl_wait();
        waited = true;
    }
    return tc::mbar_wait(bar, parity, abort, fault, 6);
}

// What the loading warp tells the others of an item (a tile, a kv head and a part).
struct Item { int rh0, count, kvh, part, lo, hi, least; bool all; };     // all: every row head sees keys (what rows behind them hold stays there)

// OWN: own tiles (rows end at their positions), else shared ones.  WR warps side by side over the rows, MT sixteens of row heads each; with
// WR 1 the warps share out the keys.  A CTA goes through the items blockIdx.x, + gridDim.x, ..; the loading warp is ahead by the
// ring, and by an item's queries and positions, so that the next item's chain of loads runs under this one's work.
template <bool OWN, int WR, int MT>
__global__ void __launch_bounds__(MMA_THREADS + LOAD_THREADS)
shared_mma_kernel(const SharedParams p, const SharedTile* tiles, int items, int parts, int part0, int beside) {
    constexpr int ROWS = 16 * WR * MT, BLOCKS = WR == 1 ? 1 : KT / 16;      // a warp's sixteens of keys in a tile
    constexpr int SLOTS = WR == 1 ? 2 : 1;                  // items whose queries are here
    extern __shared__ __align__(128) unsigned char smem_raw[];
    bf16* ring = reinterpret_cast<bf16*>(smem_raw);
    bf16* q_smem = ring + STAGES * 2 * TILE_ELEMENTS;       // [slot][row head][HD], dense
    float* merge_o = reinterpret_cast<float*>(q_smem + SLOTS * ROWS * HD);      // WR 1: [two warps][row head][HD]
    __shared__ int row_pos[SLOTS][ROWS];
    __shared__ Item item_of[SLOTS];
    __shared__ float merge_m[4][16], merge_l[4][16];
    __shared__ unsigned long long full[STAGES], empty[STAGES], q_full[SLOTS], q_empty[SLOTS];
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 4); }
        for (int s = 0; s < SLOTS; ++s) { tc::mbar_init(&q_full[s], 1); tc::mbar_init(&q_empty[s], 4); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncthreads();
    volatile int* abort = &abort_flag;
    const int G = p.H / p.KVH;
    // `beside`: the kernel before is that of the shared tiles, which has let this one go when all it reads was complete, and which it waits
    // for at its end instead, so that the join behind this one finds both done.  Every shared kernel waits first and then lets the next go.
    if (!beside) pdl_wait();
    pdl_launch_dependents();

    if (warp == 4) {
        int stage = 0, n = 0;                               // tiles and items so far
        bool ok = true, waited = !beside;                   // for the kernel before
        auto wait_free = [&](unsigned long long* bar, unsigned parity) {
            return tc::mbar_done(bar, parity) || wait_given_back(bar, parity, abort, p.fault, waited);
        };
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x, ++n) {
            const int kvh = item % p.KVH, part = item / p.KVH % parts, slot = n % SLOTS;
            const SharedTile t = tiles[item / p.KVH / parts];
            const int shared = shared_keys(p, t);
            // ---- queries, a copy a row's heads.  (Copies, pages and positions all go out as soon as the tile is known: one round of loads, not three.) ----
            ok = __all_sync(ALL, wait_free(&q_empty[slot], ((n / SLOTS) & 1) ^ 1));
            if (!ok) break;
            for (int row = t.rh0 / G + lane; row * G < t.rh0 + t.count; row += 32) {
                const int a = max(t.rh0, row * G), b = min(t.rh0 + t.count, (row + 1) * G);
                bulk_copy(q_smem + (slot * ROWS + a - t.rh0) * HD, static_cast<const bf16*>(p.q) + (long long)row * p.ldq + (kvh * G + a - row * G) * HD,
                          (b - a) * HD * 2, &q_full[slot]);
            }
            // the first tile's pages, if it is the part that begins with the first key (else, and if they are not there, they are looked up below)
            int early = -1;
            const int first_index = (OWN ? shared / p.page : 0) + lane;
            if (part == 0 && first_index < p.table_width) early = p.table[(size_t)t.slot * p.table_stride + first_index];
            int last = shared, least = 0x7fffffff;          // keys [.., last) are seen by some row; the smallest position of one that sees any
            int pos[ROWS / 32 + 1];
#pragma unroll
            for (int i = 0; i < (ROWS + 31) / 32; ++i) {
                pos[i] = lane + i * 32 < ROWS ? position_of(p, t, lane + i * 32) : -1;
                if (pos[i] >= 0) { least = min(least, pos[i]); if (OWN) last = max(last, min(pos[i], 1 << 30) + 1); }
            }
            least = __reduce_min_sync(ALL, least);
            last = end_of_keys(p, __reduce_max_sync(ALL, last), lane == 0);
            bool all = true;
#pragma unroll
            for (int i = 0; i < (ROWS + 31) / 32; ++i) all = all && (pos[i] >= 0 || lane + i * 32 >= t.count);
            all = __all_sync(ALL, all);
            Range keys = part_range(OWN ? shared : 0, last, OWN ? shared & ~(KT - 1) : 0, part, parts, KT);
            if (least == 0x7fffffff) keys.hi = keys.lo;
            const int kt0 = keys.lo & ~(KT - 1), count = keys.hi > keys.lo ? (keys.hi - kt0 + KT - 1) / KT : 0;
            // pages are looked up a tile ahead, a lane a page
            auto first_page = [&](int j) { return max(kt0 + j * KT, keys.lo) / p.page; };
            auto page_of = [&](int j) {
                const int index = j < count ? first_page(j) + lane : 0;
                return j < count && index * p.page < min(kt0 + (j + 1) * KT, keys.hi) ? page_at(p, t.slot, index) : 0;
            };
            int page = early >= 0 && early < p.num_pages ? early : page_of(0);
            // ---- positions, and what the item is ----
#pragma unroll
            for (int i = 0; i < (ROWS + 31) / 32; ++i)
                if (lane + i * 32 < ROWS) row_pos[slot][lane + i * 32] = pos[i];
            if (lane == 0) item_of[slot] = Item{t.rh0, t.count, kvh, part, keys.lo, keys.hi, least, all};
            __syncwarp();
            if (lane == 0) tc::mbar_arrive_expect_tx(&q_full[slot], t.count * HD * 2);
            // ---- keys and values of tile j: its rows in [lo, hi) ----
            for (int j = 0; j < count; ++j, ++stage) {
                const int next = page_of(j + 1), s = stage % STAGES;
                ok = __all_sync(ALL, wait_free(&empty[s], ((stage / STAGES) & 1) ^ 1));
                if (!ok) break;
                const int from = max(kt0 + j * KT, keys.lo), to = min(kt0 + (j + 1) * KT, keys.hi);
                bf16* k = ring + (size_t)s * 2 * TILE_ELEMENTS;
                if (lane == 0) tc::mbar_arrive_expect_tx(&full[s], (to - from) * HD * 4);
                __syncwarp();
                for (int index = first_page(j) + lane, turn = 0; index * p.page < to; index += 32, ++turn) {
                    if (turn > 0) page = page_at(p, t.slot, index);         // (pages of one row: more than a lane has looked up)
                    const int a = max(from, index * p.page), b = min(to, (index + 1) * p.page);
                    const bf16* src = static_cast<const bf16*>(p.plane) + (((size_t)page * 2 * p.KVH + kvh) * p.page + (a - index * p.page)) * HD;
                    bf16* dst = k + (a - kt0 - j * KT) * HD;
                    bulk_copy(dst, src, (b - a) * HD * 2, &full[s]);
                    bulk_copy(dst + TILE_ELEMENTS, src + (size_t)p.KVH * p.page * HD, (b - a) * HD * 2, &full[s]);
                }
                page = next;
            }
        }
        if (*abort)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);   // copies that may still be on their way get time to land
        if (beside) pdl_wait();
        return;
    }

    // (A wait that ran out ends no loop over the items: the warps meet at barriers in each.)
    bool slept = false;
    for (int item = blockIdx.x, n = 0, stage = 0; item < items; item += gridDim.x, ++n) {
    const int slot = n % SLOTS;
    bool ok = __all_sync(ALL, !*abort && tc::mbar_wait(&q_full[slot], (n / SLOTS) & 1, abort, p.fault, 6));
    const Item keys = item_of[slot];
    const int least = keys.least, kvh = keys.kvh, part = keys.part;
    const int kt0 = keys.lo & ~(KT - 1), count = ok && keys.hi > keys.lo ? (keys.hi - kt0 + KT - 1) / KT : 0;
    const bf16* qs = q_smem + slot * ROWS * HD;
    const int r0 = WR == 1 ? 0 : warp * 16 * MT;            // the warp's first row head
    int pos[MT][2];
    float o[MT][HD / 8][4], m[MT][2], l[MT][2];
    unsigned qf[QUERIES_STAY ? MT : 1][QUERIES_STAY ? HD / 16 : 1][4];
#pragma unroll
    for (int x = 0; x < MT; ++x) {
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[x][n][e] = 0.f;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            pos[x][y] = row_pos[slot][r0 + x * 16 + y * 8 + g];
            m[x][y] = -INFINITY;
            l[x][y] = 0.f;
        }
        if (QUERIES_STAY) {
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                const int qr = r0 + x * 16 + (lane & 15);
                ldmatrix4(qf[QUERIES_STAY ? x : 0][QUERIES_STAY ? k : 0], qs + qr * HD + (2 * k + (lane >> 4)) * 8);
            }
        }
    }
    for (int j = 0; j < count; ++j, ++stage) {
        ok = __all_sync(ALL, tc::mbar_wait(&full[stage % STAGES], (stage / STAGES) & 1, abort, p.fault, 6));
        if (!ok) break;
        const bf16* ks = ring + (size_t)(stage % STAGES) * 2 * TILE_ELEMENTS;
        bf16* vs = const_cast<bf16*>(ks) + TILE_ELEMENTS;
        const int kt = kt0 + j * KT;
        // a warp's keys of the tile (WR 1: a sixteen of its own; else all of them: every warp writes the same zeros and waits for none)
        const int mine0 = WR == 1 ? warp * 16 : 0, mine = WR == 1 ? 16 : KT;
        auto meet = [&]() {
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
        };
        if (kt + mine0 < keys.lo || kt + mine0 + mine > keys.hi) {
            // values of rows that were not copied: nothing that a probability of 0 could not take away
            for (int i = lane; i < mine * CHUNKS; i += 32) {
                const int key = kt + mine0 + i / CHUNKS;
                if (key < keys.lo || key >= keys.hi) *reinterpret_cast<uint4*>(vs + mine0 * HD + i * 8) = make_uint4(0u, 0u, 0u, 0u);
            }
            meet();
        }
        if (OWN && kt + mine0 + mine - 1 > least && least < keys.hi - 1) {
            // Behind the first row's position a key is seen by some rows and not by others, whose probability of 0 does not take away a
            // value that is not finite: such values go apart, and zeros into the products.  (OWN: a warp's keys are its own.)
            static_assert(!OWN || WR == 1, "own tiles share out their keys");
            bool odd = false;
            for (int i = lane; i < mine * CHUNKS; i += 32) {
                const int key = kt + mine0 + i / CHUNKS;
                if (key > least && key < keys.hi) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vs + mine0 * HD + i * 8);
                    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd |= (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
                }
            }
            if (__any_sync(ALL, odd)) {
                // a row that sees such a value has a result that is not finite there, whatever the probability (a positive number, or 0)
                for (int key = max(least + 1, kt + mine0); key < min(keys.hi, kt + mine0 + mine); ++key)
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int d = n * 8 + t4 * 2 + (e & 1);
                            const float v = __bfloat162float(vs[(key - kt) * HD + cache_chunk(d / 8, key, CHUNKS) * 8 + d % 8]);
#pragma unroll
                            for (int x = 0; x < MT; ++x)
                                if (key <= pos[x][e >> 1] && !(fabsf(v) < INFINITY)) o[x][n][e] += v;
                        }
                __syncwarp();
                for (int i = lane; i < mine * CHUNKS; i += 32) {
                    const int key = kt + mine0 + i / CHUNKS;
                    if (key <= least || key >= keys.hi) continue;
                    unsigned short* w = reinterpret_cast<unsigned short*>(vs + mine0 * HD + i * 8);
                    for (int e = 0; e < 8; ++e)
                        if ((w[e] & 0x7f80u) == 0x7f80u) w[e] = 0;
                }
                meet();
            }
        }
#pragma unroll 1
        for (int b = 0; b < BLOCKS; ++b) {
            const int kb = (WR == 1 ? warp : b) * 16;       // 16 keys of the tile
            if (kt + kb >= keys.hi || kt + kb + 15 < keys.lo) continue;
            float s[MT][2][4];
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[x][e >> 2][e & 3] = 0.f;
            const int kr = kb + (lane & 7) + (lane >> 4) * 8, kc = (lane >> 3) & 1;
            const bf16* krow = ks + kr * HD;
            const RowChunks kchunk(kt + kr);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                unsigned bk[4];
                ldmatrix4(bk, krow + kchunk(2 * k + kc) * 8);
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    unsigned a[4];
                    if (QUERIES_STAY) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) a[e] = qf[QUERIES_STAY ? x : 0][QUERIES_STAY ? k : 0][e];
                    } else {
                        const int qr = r0 + x * 16 + (lane & 15);
                        ldmatrix4(a, qs + qr * HD + (2 * k + (lane >> 4)) * 8);
                    }
                    mma(s[x][0], a, bk[0], bk[1]);
                    mma(s[x][1], a, bk[2], bk[3]);
                }
            }
            // every key is there, and every row sees it
            const bool whole = kt + kb >= keys.lo && kt + kb + 15 < keys.hi && (!OWN || kt + kb + 15 <= least) && keys.all;
            unsigned pa[MT][4];
#pragma unroll
            for (int x = 0; x < MT; ++x) {
                if (!whole) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = kt + kb + n * 8 + t4 * 2 + (e & 1), y = e >> 1;
                            const bool in = key >= keys.lo && key < keys.hi && (!OWN || key <= pos[x][y]) && pos[x][y] >= 0;
                            s[x][n][e] = in ? s[x][n][e] : -INFINITY;
                        }
                }
                float top[2];
                bool raise[2];                              // (each row for itself: its bits do not depend on the rows beside it)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    top[y] = fmaxf(fmaxf(s[x][0][2 * y], s[x][0][2 * y + 1]), fmaxf(s[x][1][2 * y], s[x][1][2 * y + 1]));
                    top[y] = fmaxf(top[y], __shfl_xor_sync(ALL, top[y], 1));
                    top[y] = fmaxf(top[y], __shfl_xor_sync(ALL, top[y], 2)) * p.scale_log2;     // (the scale is positive)
                    raise[y] = top[y] > m[x][y] + RAISE_STEP || (m[x][y] == -INFINITY && top[y] > -INFINITY);
                }
                if (__any_sync(ALL, raise[0] || raise[1])) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float up = raise[y] ? top[y] : m[x][y];
                        // (a row without a maximum has no sums yet but what is not finite: that stays)
                        const float f = m[x][y] == -INFINITY || !raise[y] ? 1.f : exp2_fast(m[x][y] - up);
                        l[x][y] *= f;
#pragma unroll
                        for (int n = 0; n < HD / 8; ++n) { o[x][n][2 * y] *= f; o[x][n][2 * y + 1] *= f; }
                        m[x][y] = up;
                    }
                }
                const float neg[2] = {m[x][0] == -INFINITY ? 0.f : -m[x][0], m[x][1] == -INFINITY ? 0.f : -m[x][1]};
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[x][n][e] = exp2_fast(fmaf(s[x][n][e], p.scale_log2, neg[e >> 1]));
                        l[x][e >> 1] += s[x][n][e];
                    }
                // probabilities in bfloat16 (half a step, 2^-9 of each, at random): the tensor cores' operand; their sum stays in 32 bits
                pa[x][0] = pack(s[x][0][0], s[x][0][1]); pa[x][1] = pack(s[x][0][2], s[x][0][3]);
                pa[x][2] = pack(s[x][1][0], s[x][1][1]); pa[x][3] = pack(s[x][1][2], s[x][1][3]);
            }
            const int vr = kb + (lane & 15), vc = lane >> 4;
            const bf16* vrow = vs + vr * HD;
            const RowChunks vchunk(kt + vr);
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                unsigned bv[4];
                ldmatrix4_trans(bv, vrow + vchunk(2 * n + vc) * 8);
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    mma(o[x][2 * n], pa[x], bv[0], bv[1]);
                    mma(o[x][2 * n + 1], pa[x], bv[2], bv[3]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&empty[stage % STAGES]);
    }
    if (!ok && !slept) {                                    // a wait ran out: copies that may still be on their way get time to land
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        slept = true;
    }
    // the item's queries have been read, its place is free
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&q_empty[slot]);
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            l[x][y] += __shfl_xor_sync(ALL, l[x][y], 1);
            l[x][y] += __shfl_xor_sync(ALL, l[x][y], 2);
        }

    auto place = [&](int i) { const int rh = keys.rh0 + i; return ((size_t)(part0 + part) * p.rows + rh / G) * p.H + kvh * G + rh % G; };
    if (WR > 1) {
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int i = r0 + x * 16 + y * 8 + g;
                if (i >= keys.count || !ok) continue;
                const size_t at = place(i);
                if (t4 == 0) p.part_ml[at] = make_float2(m[x][y], l[x][y]);
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
                    *reinterpret_cast<float2*>(p.part_o + at * HD + n * 8 + t4 * 2) = make_float2(o[x][n][2 * y], o[x][n][2 * y + 1]);
            }
    } else {
        // the four warps' shares, sums relative to the largest maximum: warps 2 and 3 to 0 and 1, then 1 to 0
        if (t4 == 0) {
#pragma unroll
            for (int y = 0; y < 2; ++y) { merge_m[warp][g + 8 * y] = m[0][y]; merge_l[warp][g + 8 * y] = l[0][y]; }
        }
        asm volatile("bar.sync 1, 128;\n" ::: "memory");
        float M[2], sum[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int r = g + 8 * y;
            M[y] = fmaxf(fmaxf(merge_m[0][r], merge_m[1][r]), fmaxf(merge_m[2][r], merge_m[3][r]));
            sum[y] = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) sum[y] += merge_m[w][r] == -INFINITY ? merge_l[w][r] : merge_l[w][r] * exp2_fast(merge_m[w][r] - M[y]);
            const float f = m[0][y] == -INFINITY ? 1.f : exp2_fast(m[0][y] - M[y]);
#pragma unroll
            for (int n8 = 0; n8 < HD / 8; ++n8) { o[0][n8][2 * y] *= f; o[0][n8][2 * y + 1] *= f; }
        }
#pragma unroll
        for (int from = 2; from > 0; from >>= 1) {          // warps [from, 2 from) give, warps [0, from) take: each lane's sums, in its own order
            if (warp >= from && warp < 2 * from) {
#pragma unroll
                for (int n8 = 0; n8 < HD / 8; ++n8)
                    *reinterpret_cast<float4*>(merge_o + (((warp - from) * (HD / 8) + n8) * 32 + lane) * 4) = make_float4(o[0][n8][0], o[0][n8][1], o[0][n8][2], o[0][n8][3]);
            }
            asm volatile("bar.sync 1, 128;\n" ::: "memory");
            if (warp < from) {
#pragma unroll
                for (int n8 = 0; n8 < HD / 8; ++n8) {
                    const float4 v = *reinterpret_cast<const float4*>(merge_o + ((warp * (HD / 8) + n8) * 32 + lane) * 4);
                    o[0][n8][0] += v.x; o[0][n8][1] += v.y; o[0][n8][2] += v.z; o[0][n8][3] += v.w;
                }
            }
            if (from > 1) asm volatile("bar.sync 1, 128;\n" ::: "memory");     // (read before it is written again; behind the last round the next
        }                                                                       // item's first barrier is between)
        if (!OWN || p.own_parts > 1) {
            if (warp == 0 && ok) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int i = g + 8 * y;
                    if (i >= keys.count) continue;
                    const size_t at = place(i);
                    if (t4 == 0) p.part_ml[at] = make_float2(M[y], sum[y]);
#pragma unroll
                    for (int n8 = 0; n8 < HD / 8; ++n8)
                        *reinterpret_cast<float2*>(p.part_o + at * HD + n8 * 8 + t4 * 2) = make_float2(o[0][n8][2 * y], o[0][n8][2 * y + 1]);
                }
            }
        } else {
            // ---- the only own part: joined with the shared ones here, eight threads a row head.  The kernel of the shared tiles is waited for
            // only now. ----
            if (warp == 0) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    if (t4 == 0) { merge_m[0][g + 8 * y] = M[y]; merge_l[0][g + 8 * y] = sum[y]; }
#pragma unroll
                    for (int n8 = 0; n8 < HD / 8; ++n8)
                        *reinterpret_cast<float2*>(merge_o + (g + 8 * y) * HD + n8 * 8 + t4 * 2) = make_float2(o[0][n8][2 * y], o[0][n8][2 * y + 1]);
                }
            }
            if (beside) pdl_wait();
            asm volatile("bar.sync 1, 128;\n" ::: "memory");
            const int i = threadIdx.x >> 3;
            if (i < keys.count && ok) join_row(p, merge_m[0][i], merge_l[0][i], merge_o + i * HD, keys.rh0 + i, kvh, threadIdx.x & 7);
            asm volatile("bar.sync 1, 128;\n" ::: "memory");         // (read before the next item writes it)
        }
    }
    }
    if (beside) pdl_wait();
}

// ---- float32: dot products on the CUDA cores, everything in 32 bits ---------------------------------------------------------
// A CTA has R row heads of a tile, four: with eight or sixteen the keys are read fewer times, but a CTA that goes once through code unrolled for
// that many spends its time fetching it (4 requests behind 1000 keys, 12 heads of 64: 20.7 us with 4, 32.4 with 8; 8 requests of 3 rows behind
// 2048, 32 heads of 128: 128 and 167).  A warp takes 32 keys: first a lane a key (its row against the queries in shared memory, which all lanes
// read at once), then, with the probabilities in shared memory, a lane four columns (HD / 4 lanes or the next power of two a key, the
// groups of lanes taking turns).  All loads of 32 keys are independent of one another.  The four warps take turns and merge at the end.
constexpr int F32_LANES = (HD + 31) / 32;
constexpr int F32_QUADS = HD / 4, F32_GROUP = F32_QUADS > 16 ? 32 : F32_QUADS > 8 ? 16 : F32_QUADS > 4 ? 8 : 4;
constexpr int F32_TURNS = 32 / F32_GROUP, F32_EACH = (F32_QUADS + F32_GROUP - 1) / F32_GROUP;        // keys at a time, quads of a lane
constexpr int F32_AHEAD = 8;                // loads of a lane on their way
template <int R> constexpr int f32_floats() { return R * HD + 4 * 32 * R + 4 * R * HD; }     // queries, probabilities, the warps' shares

template <bool OWN, int R>
__global__ void __launch_bounds__(MMA_THREADS)
shared_f32_kernel(const SharedParams p, const SharedTile* tiles, int parts, int part0, int beside) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    float* q_smem = reinterpret_cast<float*>(smem_raw);     // [R][HD]
    float* prob = q_smem + R * HD;                          // [warp][key][R]
    float* merge_o = prob + 4 * 32 * R;                     // [warp][R][HD]
    __shared__ float merge_m[4][R], merge_l[4][R];
    __shared__ size_t row_at[4][32];
    __shared__ int row_pos[16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % p.KVH, part = blockIdx.x / p.KVH % parts, i0 = (int)blockIdx.y * R;
    const SharedTile t = tiles[blockIdx.x / p.KVH / parts];
    if (i0 >= t.count) {                                    // (a tile of fewer row heads than the largest)
        pdl_wait();
        return;
    }
    const int G = p.H / p.KVH;
    constexpr int NCH = HD / 4;
    if (!beside) pdl_wait();                                // (as above)
    pdl_launch_dependents();
    if (threadIdx.x < 16) row_pos[threadIdx.x] = position_of(p, t, threadIdx.x);
    __syncthreads();
    const int shared = shared_keys(p, t);
    int last = shared;
    if (OWN)
        for (int i = 0; i < t.count; ++i) last = max(last, min(row_pos[i], 1 << 30) + 1);
    last = end_of_keys(p, last, threadIdx.x == 0);
    const Range keys = part_range(OWN ? shared : 0, last, OWN ? shared & ~63 : 0, part, parts, 64);
    const size_t v_step = (size_t)p.KVH * p.page * HD;
    const int group = lane / F32_GROUP, quad = lane % F32_GROUP;
    {
        int pos[R], least = 0x7fffffff, most = -1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            pos[r] = i0 + r < t.count ? row_pos[i0 + r] : -1;
            if (pos[r] >= 0) { least = min(least, pos[r]); most = max(most, min(pos[r], 1 << 30)); }
        }
        for (int i = threadIdx.x; i < R * HD; i += MMA_THREADS) {
            const int rh = t.rh0 + min(i0 + i / HD, t.count - 1);
            q_smem[i] = static_cast<const float*>(p.q)[(long long)(rh / G) * p.ldq + (kvh * G + rh % G) * HD + i % HD];
        }
        __syncthreads();
        float m[R], l[R], o[R][F32_EACH][4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int e = 0; e < F32_EACH * 4; ++e) o[r][e / 4][e % 4] = 0.f;
        }
        const int hi = most < 0 ? keys.lo : (OWN ? min(keys.hi, most + 1) : keys.hi);
        for (int k0 = keys.lo + warp * 32; k0 < hi; k0 += 128) {
            // ---- scores: a lane a key (behind the last one: the last once more, seen by no row) ----
            const int key = min(k0 + lane, hi - 1), n = min(32, hi - k0);
            const size_t at = (((size_t)page_at(p, t.slot, key / p.page) * 2 * p.KVH + kvh) * p.page + key % p.page) * HD;
            const float* k = static_cast<const float*>(p.plane) + at;
            row_at[warp][lane] = at + v_step;
            float s[R];
#pragma unroll
            for (int r = 0; r < R; ++r) s[r] = 0.f;
            const int turn = NCH % 8 == 0 ? key & 7 : key % NCH;
            for (int c0 = 0; c0 < NCH; c0 += F32_AHEAD) {
                float4 x[F32_AHEAD];
#pragma unroll
                for (int a = 0; a < F32_AHEAD; ++a) {
                    const int c = min(c0 + a, NCH - 1);
                    x[a] = *reinterpret_cast<const float4*>(k + (NCH % 8 == 0 ? c ^ turn : c + turn - (c + turn >= NCH ? NCH : 0)) * 4);
                }
#pragma unroll
                for (int a = 0; a < F32_AHEAD; ++a) {
                    if (NCH % F32_AHEAD != 0 && c0 + a >= NCH) continue;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float4 y = *reinterpret_cast<const float4*>(q_smem + r * HD + (c0 + a) * 4);
                        s[r] = fmaf(x[a].x, y.x, fmaf(x[a].y, y.y, fmaf(x[a].z, y.z, fmaf(x[a].w, y.w, s[r]))));
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const bool sees = lane < n && pos[r] >= 0 && (!OWN || key <= pos[r]);
                s[r] = sees ? s[r] * p.scale_log2 : -INFINITY;
                float top = s[r];
#pragma unroll
                for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, w));
                if (top > m[r]) {                           // (uniform in the warp)
                    const float f = m[r] == -INFINITY ? 1.f : exp2f(m[r] - top);       // (no sums yet, but what is not finite: that stays)
                    l[r] *= f;
#pragma unroll
                    for (int e = 0; e < F32_EACH * 4; ++e) o[r][e / 4][e % 4] *= f;
                    m[r] = top;
                }
                s[r] = sees ? exp2f(s[r] - (m[r] == -INFINITY ? 0.f : m[r])) : 0.f;
                l[r] += s[r];                               // (a lane's share: added up over the lanes at the end)
                prob[(warp * 32 + lane) * R + r] = s[r];
            }
            __syncwarp();
            // ---- values: a lane four columns of one of the keys whose turn it is ----
            for (int j0 = group; j0 < n; j0 += F32_TURNS * F32_AHEAD) {
#pragma unroll
                for (int e = 0; e < F32_EACH; ++e) {
                    const int c = min(quad + e * F32_GROUP, F32_QUADS - 1);         // (a lane too many reads what its neighbour reads)
                    float4 x[F32_AHEAD];
#pragma unroll
                    for (int a = 0; a < F32_AHEAD; ++a) {
                        const int j = min(j0 + a * F32_TURNS, n - 1), turn_j = NCH % 8 == 0 ? (k0 + j) & 7 : (k0 + j) % NCH;
                        x[a] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.plane) + row_at[warp][j] +
                                                                (NCH % 8 == 0 ? c ^ turn_j : c + turn_j - (c + turn_j >= NCH ? NCH : 0)) * 4);
                    }
#pragma unroll
                    for (int a = 0; a < F32_AHEAD; ++a) {
                        const int j = j0 + a * F32_TURNS;
                        if (j >= n) continue;
                        const bool some = k0 + j > least;   // do not see it: a probability of 0 does not take away what is not finite
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            if (some && (pos[r] < 0 || (OWN && k0 + j > pos[r]))) continue;
                            const float w = prob[(warp * 32 + j) * R + r];
                            o[r][e][0] = fmaf(w, x[a].x, o[r][e][0]);
                            o[r][e][1] = fmaf(w, x[a].y, o[r][e][1]);
                            o[r][e][2] = fmaf(w, x[a].z, o[r][e][2]);
                            o[r][e][3] = fmaf(w, x[a].w, o[r][e][3]);
                        }
                    }
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) l[r] += __shfl_xor_sync(ALL, l[r], w);
#pragma unroll
            for (int e = 0; e < F32_EACH * 4; ++e)
#pragma unroll
                for (int w = F32_GROUP; w < 32; w <<= 1) o[r][e / 4][e % 4] += __shfl_xor_sync(ALL, o[r][e / 4][e % 4], w);
            if (lane == 0) { merge_m[warp][r] = m[r]; merge_l[warp][r] = l[r]; }
#pragma unroll
            for (int e = 0; e < F32_EACH; ++e) {
                const int c = quad + e * F32_GROUP;
                if (group == 0 && c < F32_QUADS)
                    *reinterpret_cast<float4*>(merge_o + (warp * R + r) * HD + c * 4) = make_float4(o[r][e][0], o[r][e][1], o[r][e][2], o[r][e][3]);
            }
        }
        __syncthreads();
        for (int r = warp; r < R && i0 + r < t.count; r += 4) {
            const float M = fmaxf(fmaxf(merge_m[0][r], merge_m[1][r]), fmaxf(merge_m[2][r], merge_m[3][r]));
            float f[4], sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                f[w] = merge_m[w][r] == -INFINITY ? 1.f : exp2f(merge_m[w][r] - M);      // (no keys, or scores that are no numbers: as they are)
                sum += merge_l[w][r] * f[w];
            }
            const int rh = t.rh0 + i0 + r;
            const size_t to = ((size_t)(part0 + part) * p.rows + rh / G) * p.H + kvh * G + rh % G;
            if (lane == 0) p.part_ml[to] = make_float2(M, sum);
            for (int d = lane; d < HD; d += 32) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) x += merge_o[(w * R + r) * HD + d] * f[w];
                p.part_o[to * HD + d] = x;
            }
        }
    }
    if (beside) pdl_wait();
}

// ---- the parts of a row head joined ------------------------------------------------------------------------------------------
// W warps a row head share the parts out and meet in shared memory; each has the loads of several parts on their way.
constexpr int JOIN_THREADS = 128, JOIN_AHEAD = 8;
template <typename T, int W>
__global__ void __launch_bounds__(JOIN_THREADS)
shared_join_kernel(const SharedParams p, T* out, long long ldo, int row_heads, int parts) {
    constexpr int HEADS = JOIN_THREADS / 32 / W;            // row heads of a CTA
    __shared__ float2 ml[HEADS][MAX_PARTS];
    __shared__ float shares[HEADS][W][HD + 1];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp / W, w = warp % W;
    const int i = min((int)blockIdx.x * HEADS + mine, row_heads - 1);      // row, head (the last one again beyond the end)
    pdl_wait();
    for (int q = w * 32 + lane; q < parts; q += W * 32) ml[mine][q] = p.part_ml[(size_t)q * row_heads + i];
    __syncthreads();
    float M = -INFINITY;
    for (int q = lane; q < parts; q += 32) M = fmaxf(M, ml[mine][q].x);
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) M = fmaxf(M, __shfl_xor_sync(ALL, M, e));
    float l = 0.f, o[F32_LANES];
#pragma unroll
    for (int e = 0; e < F32_LANES; ++e) o[e] = 0.f;
    for (int q0 = w; q0 < parts; q0 += W * JOIN_AHEAD) {
        float x[JOIN_AHEAD][F32_LANES], f[JOIN_AHEAD];
#pragma unroll
        for (int a = 0; a < JOIN_AHEAD; ++a) {
            const int q = q0 + a * W;
            const float2 v = q < parts ? ml[mine][q] : make_float2(-INFINITY, 0.f);
            const bool some = !(v.x == -INFINITY && v.y == 0.f);        // (else no keys: nothing was left there)
            f[a] = v.x == -INFINITY ? 1.f : exp2f(v.x - M);
            l += v.y * f[a];
            const float* src = p.part_o + ((size_t)q * row_heads + i) * HD;
#pragma unroll
            for (int e = 0; e < F32_LANES; ++e) x[a][e] = some && lane + e * 32 < HD ? src[lane + e * 32] : 0.f;
        }
#pragma unroll
        for (int a = 0; a < JOIN_AHEAD; ++a)
#pragma unroll
            for (int e = 0; e < F32_LANES; ++e) o[e] = fmaf(x[a][e], f[a], o[e]);
    }
    if (W > 1) {
#pragma unroll
        for (int e = 0; e < F32_LANES; ++e)
            if (lane + e * 32 < HD) shares[mine][w][lane + e * 32] = o[e];
        if (lane == 0) shares[mine][w][HD] = l;
        __syncthreads();
        if (w != 0) return;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < F32_LANES; ++e) o[e] = 0.f;
        for (int a = 0; a < W; ++a) {
            l += shares[mine][a][HD];
#pragma unroll
            for (int e = 0; e < F32_LANES; ++e)
                if (lane + e * 32 < HD) o[e] += shares[mine][a][lane + e * 32];
        }
    }
    if ((int)blockIdx.x * HEADS + mine >= row_heads) return;
    T* dst = out + (long long)(i / p.H) * ldo + i % p.H * HD;
#pragma unroll
    for (int e = 0; e < F32_LANES; ++e)
        if (lane + e * 32 < HD) dst[lane + e * 32] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
}
template <typename T> int launch_join(const SharedParams& p, void* out, long long ldo, int row_heads, int parts, cudaStream_t stream) {
    if (parts > 4) tis_launch(shared_join_kernel<T, 4>, dim3((unsigned)row_heads), dim3(JOIN_THREADS), 0, stream, p, static_cast<T*>(out), ldo, row_heads, parts);
    else tis_launch(shared_join_kernel<T, 1>, dim3((unsigned)((row_heads + 3) / 4)), dim3(JOIN_THREADS), 0, stream, p, static_cast<T*>(out), ldo, row_heads, parts);
    return tis_check_launch("shared_prefix_attention (join)");
}

template <bool OWN> int launch_f32(const SharedParams& p, const SharedTile* tiles, int count, int heads, int parts, int part0, int beside, cudaStream_t stream) {
    constexpr int R = 4, smem = f32_floats<R>() * 4;
    heads = heads < 16 ? heads : 16;                        // (of a tile)
    static DeviceOnce configured;
    if (configured([&] { return cudaFuncSetAttribute(shared_f32_kernel<OWN, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }) != cudaSuccess)
        return tis_check_launch("shared_prefix_attention (shared memory)");
    tis_launch(shared_f32_kernel<OWN, R>, dim3((unsigned)(count * parts * p.KVH), (unsigned)((heads + R - 1) / R)), dim3(MMA_THREADS), (size_t)smem, stream,
               p, tiles, parts, part0, beside);
    return tis_check_launch("shared_prefix_attention");
}

template <bool OWN, int WR, int MT> int launch_mma(const SharedParams& p, const SharedTile* tiles, int count, int parts, int part0, int beside, cudaStream_t stream) {
    constexpr int ROWS = 16 * WR * MT;
    const size_t smem = (size_t)STAGES * 2 * TILE_ELEMENTS * 2 + (size_t)(WR == 1 ? 2 : 1) * ROWS * HD * 2 + (WR == 1 ? 2 * 16 * HD * 4 : 0);
    const int items = count * parts * p.KVH, ctas = WR == 1 ? (HD <= 128 ? 2 : 1) * tc::sm_count() : items;
    static DeviceOnce configured;
    if (configured([&] { return cudaFuncSetAttribute(shared_mma_kernel<OWN, WR, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }) != cudaSuccess)
        return tis_check_launch("shared_prefix_attention (shared memory)");
    tis_launch(shared_mma_kernel<OWN, WR, MT>, dim3((unsigned)(items < ctas ? items : ctas)), dim3(MMA_THREADS + LOAD_THREADS), smem, stream, p, tiles, items, parts, part0, beside);
    return tis_check_launch("shared_prefix_attention");
}

}  // namespace

// shared_attention_tc.cu
bool shared_tc_takes(int page);
int shared_tc_launch(const SharedParams& p, const SharedTile* tiles, int count, int parts, cudaStream_t stream);

TIS_API int tis_shared_attn_head_dim() { return HD; }
// the most row heads of a shared tile: 128, or 64 where a warp's share of 32 does not fit its registers
TIS_API int tis_shared_attn_widest() { return HD <= 128 ? 128 : 64; }

// `own`, `wide`: tiles on the device, own ones of up to 16 row heads, shared ones of up to `wide_rows`: 16, and in bfloat16
// 64 or 128 (tis_shared_attn_widest); `tensor`: shared tiles by the tcgen05 kernel, which takes up to
// 128.  most_heads, own_heads: row heads of the largest group and of the largest request.
// The first `shared_parts` parts of the scratch are the shared tiles', the `own_parts` behind them the own ones'; rows of groups
// without shared keys have empty ones.  `rows`: the rows of the plan, all of which are written.
TIS_API int tis_shared_attn_tensor(int page) { return shared_tc_takes(page); }
struct SharedArgs {
    long long dtype, q, ldq, out, ldo, plane, table, table_stride, table_width, num_pages, positions, own, own_count, wide, wide_count, wide_rows,
        tensor, own_parts, shared_parts, rows, H, KVH, page, part_o, part_ml, fault, stream, most_heads, own_heads;
    double scale;
};
TIS_API int tis_shared_attention(const SharedArgs* a) {
    if (a->rows <= 0) return TIS_OK;
    // (a lane looks for keys up to 32 pages behind the last: their number is held in 32 bits)
    const long long most = 1ll << 30;
    if (a->table_stride > most || a->table_width > most || a->num_pages > most || a->page > (1 << 25) || a->rows * a->H > most ||
        a->own_count * a->own_parts * a->KVH > most || a->wide_count * a->shared_parts * a->KVH > most) {
        tis_set_error("shared_prefix_attention: %lld rows of %lld heads, %lld pages of %lld, tables of %lld", a->rows, a->H, a->num_pages, a->page, a->table_width);
        return TIS_BAD_SIZE;
    }
    const int dtype = (int)a->dtype, rows = (int)a->rows, H = (int)a->H, KVH = (int)a->KVH, page = (int)a->page, num_pages = (int)a->num_pages;
    const int own_count = (int)a->own_count, wide_count = (int)a->wide_count, wide_rows = (int)a->wide_rows, tensor = (int)a->tensor;
    const int own_parts = (int)a->own_parts, shared_parts = (int)a->shared_parts;
    void* out = reinterpret_cast<void*>(a->out);
    const long long ldo = a->ldo;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
    SharedParams p;
    p.q = reinterpret_cast<const void*>(a->q); p.ldq = a->ldq; p.plane = reinterpret_cast<const void*>(a->plane);
    p.table = reinterpret_cast<const int*>(a->table); p.table_stride = (int)a->table_stride; p.table_width = (int)a->table_width; p.num_pages = num_pages;
    p.positions = reinterpret_cast<const int*>(a->positions);
    p.part_o = reinterpret_cast<float*>(a->part_o); p.part_ml = reinterpret_cast<float2*>(a->part_ml);
    p.rows = rows; p.H = H; p.KVH = KVH; p.page = page; p.own_parts = own_parts; p.shared_parts = shared_parts;
    p.out = out; p.ldo = ldo; p.out_vectors = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo % 8 == 0;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.fault = reinterpret_cast<int*>(a->fault);
    if (wide_rows != 16 && (dtype == TIS_F32 || wide_rows > tis_shared_attn_widest() || (wide_rows != 64 && wide_rows != 128))) {
        tis_set_error("shared_prefix_attention: shared tiles of %d row heads", wide_rows);
        return TIS_BAD_SIZE;
    }
    if (own_parts < 1 || shared_parts < 0 || own_parts + shared_parts > MAX_PARTS || (tensor && !(dtype == TIS_BF16 && shared_tc_takes(page) && 2ll * num_pages * KVH * page < 1ll << 31))) {
        tis_set_error("shared_prefix_attention: %d and %d parts, pages of %d", own_parts, shared_parts, page);
        return TIS_BAD_SIZE;
    }
    const SharedTile* o = reinterpret_cast<const SharedTile*>(a->own);
    const SharedTile* w = reinterpret_cast<const SharedTile*>(a->wide);
    const int parts = own_parts + shared_parts, row_heads = rows * H;
    int status = TIS_OK;
    if (dtype == TIS_F32) {
        if (shared_parts > 0) status = launch_f32<false>(p, w, wide_count, (int)a->most_heads, shared_parts, 0, 0, stream);
        if (status == TIS_OK) status = launch_f32<true>(p, o, own_count, (int)a->own_heads, own_parts, shared_parts, shared_parts > 0, stream);
    } else if (dtype == TIS_BF16) {
        if (shared_parts > 0) {
            if (tensor) status = shared_tc_launch(p, w, wide_count, shared_parts, stream);
            else if (wide_rows == 16) status = launch_mma<false, 1, 1>(p, w, wide_count, shared_parts, 0, 0, stream);
            else if (wide_rows == 64) status = launch_mma<false, 4, 1>(p, w, wide_count, shared_parts, 0, 0, stream);
            else status = launch_mma<false, 4, HD <= 128 ? 2 : 1>(p, w, wide_count, shared_parts, 0, 0, stream);
        }
        if (status == TIS_OK) status = launch_mma<true, 1, 1>(p, o, own_count, own_parts, shared_parts, shared_parts > 0, stream);
    } else {
        tis_set_error("shared_prefix_attention: dtype code %d", dtype);
        return TIS_BAD_DTYPE;
    }
    if (status != TIS_OK || (dtype == TIS_BF16 && own_parts == 1)) return status;       // (the own tiles have joined theirs)
    return dtype == TIS_F32 ? launch_join<float>(p, out, ldo, row_heads, parts, stream) : launch_join<bf16>(p, out, ldo, row_heads, parts, stream);
}
