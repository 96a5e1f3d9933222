// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Request b has drafts d_0 .. d_{L-1}, the draft's distributions q_i (none: the drafts are certain, q_i one at d_i), the target's
// p_0 .. p_L and numbers u_0 .. u_k in [0, 1).  Draft i is kept while u_i q_i(d_i) < p_i(d_i) (kept with chance min(1, p / q)).
// Behind the first draft that is not, the next token is drawn from max(p_i - q_i, 0), or from p_i where that has no mass; behind L
// kept ones from p_L.  The draw is by inverse CDF in index order: the lowest token whose running sum exceeds u_k times the whole.
// What is not a positive number (zero, negative, infinite, NaN) has no mass.
//
// Products, differences and sums are in 64 bits: a product of two floats is then exact, a sum of a vocabulary's floats is off by
// some 1e-15 of itself, and a token does not depend on how the row is shared out.  (In 32 bits the sum of 131072 entries is off by
// more than many a token's mass.)
//
// Only one row of p, and behind a rejection one of q, is read: the kernel is bound by those bytes, and for few requests by the
// chain draft -> its probabilities -> row -> sum -> place.  Every warp works out for itself which row it is (a lane a draft: no
// barrier), so the chain has one exchange: a cluster of up to 16 CTAs shares the row, a warp takes a contiguous run of it, and the
// runs' sums go to every CTA of the cluster.  All CTAs then know whose run holds the number; that warp goes through the sums of its
// run's steps and reads one step again.  Measured: 64 requests of 131072 tokens, behind a rejection each (67 MB) 20 us, of it 10 at
// the rate of memory (64-bit sums of every entry: 37 us, the conversions; a search entry by entry of the whole run: 6 us more);
// one request of 32000 tokens 5.3 us.
#include "cluster_reduce.cuh"

namespace {

constexpr int VERIFY_THREADS = 512;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int VERIFY_MAX_CLUSTER = 16;
constexpr int VERIFY_STEPS = 32;            // sums of a run that are kept, to find the place of the number in it
constexpr int VERIFY_MAX_DRAFTS = 31;       // a lane a draft, one more for the token behind them
constexpr unsigned ALL = 0xffffffffu;

struct VerifyParams {
    const float* p; long long p_request, p_row;
    const float* q; long long q_request, q_row;     // null: drafts without a distribution
    const int* drafts; const float* u; const int* lens;
    int* tokens; int* accepted;
    int k, V;
};

__device__ __forceinline__ float positive(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }
__device__ __forceinline__ double mass(float x) { return (double)positive(x); }

// What is left of a row: entries of p less those of q.
struct Row {
    const float* p; const float* q;         // q null: nothing is taken away but the entry `without`
    int without;
    int V;
    bool wide;                              // rows that start on 16 bytes
    // entries i .. i + 3 as they are (beyond the row: zero)
    __device__ __forceinline__ float4 four(const float* x, int i) const {
        if (wide && i + 3 < V) return *reinterpret_cast<const float4*>(x + i);
        const int last = V - 1;             // (read again rather than skipped: loads that nothing decides about go out together)
        float4 r = make_float4(x[min(i, last)], x[min(i + 1, last)], x[min(i + 2, last)], x[min(i + 3, last)]);
        if (i + 3 > last) {
            if (i > last) r.x = 0.f;
            if (i + 1 > last) r.y = 0.f;
            if (i + 2 > last) r.z = 0.f;
            r.w = 0.f;
        }
        return r;
    }
    // what is left of entries i .. i + 3, in 64 bits
    __device__ __forceinline__ void piece(const float4& a, const float4& b, int i, double (&r)[4]) const {
        const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = i + e == without ? 0.0 : fmax(mass(x[e]) - mass(y[e]), 0.0);
    }
    template <int N> __device__ __forceinline__ void load(int i, float4 (&a)[N], float4 (&b)[N]) const {
#pragma unroll
        for (int n = 0; n < N; ++n) a[n] = four(p, i + n * 128);
#pragma unroll
        for (int n = 0; n < N; ++n) b[n] = q != nullptr ? four(q, i + n * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // What is left of N pieces of four entries, 128 apart, added up.  A conversion to 64 bits costs as much as a dozen 32-bit
    // sums, so a difference and a sum are kept as two floats each, the rounded result and what the rounding lost (Dekker 1971,
    // Knuth's two-sum), and converted once: off by some 2^-46 of itself.
    template <int N, bool Q> __device__ __forceinline__ double sum(int i) const {
        float4 a[N], b[N];
#pragma unroll
        for (int n = 0; n < N; ++n) a[n] = four(p, i + n * 128);
        if (Q) {
#pragma unroll
            for (int n = 0; n < N; ++n) b[n] = four(q, i + n * 128);
        }
        float s = 0.f, lost = 0.f, top = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float x[4] = {a[n].x, a[n].y, a[n].z, a[n].w};
            const float y[4] = {Q ? b[n].x : 0.f, Q ? b[n].y : 0.f, Q ? b[n].z : 0.f, Q ? b[n].w : 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float d = fmaxf(x[e], 0.f), d_lost = 0.f;       // (a NaN and what is negative: no mass)
                if (Q) {
                    const float q1 = fmaxf(y[e], 0.f), both = fminf(d, q1), left = d - both;
                    top = fmaxf(top, q1);
                    d_lost = (d - left) - both;
                    d = left;
                } else if (i + n * 128 + e == without) {
                    d = 0.f;
                }
                const float t = s + d, v = t - s;
                lost += (s - (t - v)) + (d - v);
                if (Q) lost += d_lost;
                s = t;
            }
        }
        top = fmaxf(top, s);
        if (top < INFINITY) return (double)s + (double)lost;
        double exact = 0.0;                                     // an infinity has no mass either
#pragma unroll 1
        for (int n = 0; n < N; ++n) {
            double r[4];
            piece(four(p, i + n * 128), q != nullptr ? four(q, i + n * 128) : make_float4(0.f, 0.f, 0.f, 0.f), i + n * 128, r);
            exact += (r[0] + r[1]) + (r[2] + r[3]);
        }
        return exact;
    }
};

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}
__device__ __forceinline__ double warp_running(double v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double w = __shfl_up_sync(ALL, v, o);
        if (lane >= o) v += w;
    }
    return v;
}
__device__ __forceinline__ void store_to_rank(double* local, unsigned rank, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;\n"
                 ::"r"(cluster_reduce::map_to_rank(cluster_reduce::shared_addr(local), rank)), "d"(v) : "memory");
}

// A warp's run is `steps` steps of `strides` times 128 N entries; rank r of the cluster has runs 16 r .. 16 r + 15.
template <int N>
__global__ void __launch_bounds__(VERIFY_THREADS, 2)
verify_kernel(const VerifyParams v, int steps, int strides) {
    __shared__ double step_sum[VERIFY_WARPS][VERIFY_STEPS];
    __shared__ double run_sum[2][VERIFY_WARPS];
    __shared__ double rank_sum[2][VERIFY_MAX_CLUSTER];     // written by every rank; one set for each of the two passes
    pdl_launch_dependents();
    unsigned ranks, rank;
    asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(ranks));
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
    cluster_reduce::cluster_arrive();                       // waited for before the first store to another CTA
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t b = blockIdx.x / ranks;
    pdl_wait();

    // ---- which drafts are kept: a lane a draft, every warp for itself ----
    const int L = v.lens != nullptr ? min(max(v.lens[b], 0), v.k) : v.k;
    const int draft = lane < v.k ? v.drafts[b * v.k + lane] : -1;
    const bool real = draft >= 0 && draft < v.V;
    const double u_last = (double)v.u[b * (v.k + 1) + v.k];
    bool keep = false;
    if (lane < L && real) {
        const double p = mass(v.p[(long long)b * v.p_request + lane * v.p_row + draft]);
        const double q = v.q != nullptr ? mass(v.q[(long long)b * v.q_request + lane * v.q_row + draft]) : 1.0;
        keep = (double)v.u[b * (v.k + 1) + lane] * q < p;
    }
    const int kept = __ffs(~__ballot_sync(ALL, keep)) - 1;  // (at most 31 lanes keep one)
    const int refused = __shfl_sync(ALL, draft, kept);      // the draft at that place, if there is one

    Row row;
    row.p = v.p + (long long)b * v.p_request + kept * v.p_row;
    row.q = kept < L && v.q != nullptr ? v.q + (long long)b * v.q_request + kept * v.q_row : nullptr;
    row.without = kept < L && v.q == nullptr ? refused : -1;
    row.V = v.V;
    const int stride = 128 * N, step = strides * stride;
    const int first = ((int)rank * VERIFY_WARPS + warp) * steps * step;
    int token = -1;
    bool mine = false;
    for (int pass = 0; pass < 2; ++pass) {
        row.wide = ((reinterpret_cast<uintptr_t>(row.p) | reinterpret_cast<uintptr_t>(row.q)) & 15) == 0;
        // ---- sums of the runs, of the CTAs, of the row ----
        double sum = 0.0;
        for (int j = 0; j < steps && first + j * step < v.V; ++j) {
            const int from = first + j * step, to = min(from + step, v.V);
            double s = 0.0;
            if (row.q != nullptr) {
                for (int i = from; i < to; i += stride) s += row.sum<N, true>(i + lane * 4);
            } else {
                for (int i = from; i < to; i += stride) s += row.sum<N, false>(i + lane * 4);
            }
            s = warp_total(s);
            if (lane == 0) step_sum[warp][j] = s;
            sum += s;
        }
        if (lane == 0) run_sum[pass][warp] = sum;
        __syncthreads();
        // (the runs' sums added one after another, the same bits in every lane and warp)
        double cta = 0.0;
#pragma unroll
        for (int w = 0; w < VERIFY_WARPS; ++w) cta += run_sum[pass][w];
        if (pass == 0) cluster_reduce::cluster_wait();      // every CTA of the cluster has started
        if (warp == 0 && lane < (int)ranks) store_to_rank(&rank_sum[pass][rank], (unsigned)lane, cta);
        __syncwarp();
        cluster_reduce::cluster_arrive();
        cluster_reduce::cluster_wait();
        double total = 0.0;
        for (unsigned r = 0; r < ranks; ++r) total += rank_sum[pass][r];
        if (total > 0.0) {
            // ---- whose run holds the number: the first rank, run, lane whose running sum exceeds it (the last with mass where
            // rounding left it beyond all of them) ----
            const double target = u_last * total;
            double before = 0.0, running = 0.0;
            int owner = -1;
            for (unsigned r = 0; r < ranks; ++r) {
                const double s = rank_sum[pass][r];
                if (s > 0.0) { owner = (int)r; before = running; }
                running += s;
                if (s > 0.0 && running > target) break;
            }
            if (owner != (int)rank) break;
            running = before;
            owner = -1;
            for (int w = 0; w < VERIFY_WARPS; ++w) {
                const double s = run_sum[pass][w];
                if (s > 0.0) { owner = w; before = running; }
                running += s;
                if (s > 0.0 && running > target) break;
            }
            if (owner != warp) break;
            __syncwarp();
            running = before;
            int place = -1;
            for (int j = 0; j < steps && first + j * step < v.V; ++j) {
                const double s = step_sum[warp][j];
                if (s > 0.0) { place = j; before = running; }
                running += s;
                if (s > 0.0 && running > target) break;
            }
            running = before;
            const int from = first + place * step, to = min(from + step, v.V);
            bool found = false;
            for (int i = from; i < to && !found; i += stride) {
                float4 a[N], b[N];
                row.load<N>(i + lane * 4, a, b);
                double s[N], upto[N], r[4];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    row.piece(a[n], b[n], i + lane * 4 + n * 128, r);
                    s[n] = (r[0] + r[1]) + (r[2] + r[3]);
                    upto[n] = warp_running(s[n], lane);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    if (found) continue;
                    const unsigned has = __ballot_sync(ALL, s[n] > 0.0);
                    const unsigned over = __ballot_sync(ALL, s[n] > 0.0 && running + upto[n] > target);
                    if (has != 0) {
                        row.piece(a[n], b[n], i + lane * 4 + n * 128, r);
                        double c = running + (upto[n] - s[n]);
                        int entry = -1;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool passed = entry >= 0 && c > target;
                            c += r[e];
                            if (!passed && r[e] > 0.0) entry = i + lane * 4 + n * 128 + e;
                        }
                        // (of the last piece with mass, if none exceeds the number)
                        token = __shfl_sync(ALL, entry, over != 0 ? __ffs(over) - 1 : 31 - __clz(has));
                    }
                    found = over != 0;
                    running += __shfl_sync(ALL, upto[n], 31);
                }
            }
            mine = true;
            break;
        }
        if (pass == 1 || (row.q == nullptr && row.without < 0)) {      // no mass anywhere: no token
            mine = rank == 0 && warp == 0;
            break;
        }
        row.q = nullptr;                                    // nothing is left of p - q: p itself
        row.without = -1;
    }
    if (mine) {
        if (lane <= v.k) v.tokens[b * (v.k + 1) + lane] = lane < kept ? draft : (lane == kept ? token : -1);
        if (lane == 0) v.accepted[b] = kept;
    }
}

template <int N> int verify_launch(const cudaLaunchConfig_t& cfg, const VerifyParams& v, long long run) {
    static DeviceOnce configured;
    if (configured([&] { return cudaFuncSetAttribute(verify_kernel<N>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); }) != cudaSuccess)
        return tis_check_launch("verify_drafts (cluster size)");
    const long long strides = (run + 128 * N * VERIFY_STEPS - 1) / (128 * N * VERIFY_STEPS);
    const long long steps = (run + 128 * N * strides - 1) / (128 * N * strides);
    cudaLaunchKernelEx(&cfg, verify_kernel<N>, v, (int)steps, (int)strides);
    return tis_check_launch("verify_drafts");
}

}  // namespace

// n requests of up to k drafts over V tokens.  p: rows p + b p_request + i p_row (i <= k) of V floats; q likewise (i < k; null: none);
// drafts [n][k], u [n][k + 1], lens [n] (null: k each); tokens [n][k + 1]: the kept drafts, the drawn token (-1: no mass), -1 behind.
struct VerifyArgs { long long p, p_request, p_row, q, q_request, q_row, drafts, u, lens, tokens, accepted, n, k, V, stream; };
TIS_API int tis_verify_drafts(const VerifyArgs* a) {
    const float* p = reinterpret_cast<const float*>(a->p);
    const float* q = reinterpret_cast<const float*>(a->q);
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
    if (a->V > (1 << 30) || a->n > (1 << 30) || a->k > VERIFY_MAX_DRAFTS) {
        tis_set_error("verify_drafts: %lld requests of %lld drafts, vocabulary of %lld", a->n, a->k, a->V);
        return TIS_BAD_SIZE;
    }
    const int n = (int)a->n, k = (int)a->k, V = (int)a->V;
    if (n <= 0) return TIS_OK;
    if (k < 0 || V <= 0) {
        tis_set_error("verify_drafts: %d drafts, vocabulary of %d", k, V);
        return TIS_BAD_SIZE;
    }
    // CTAs a request: as many as are all resident (two to an SM) and have four entries a thread.  us at 1, 2, 4, 8, 16 a request: 64
    // requests of 131072 tokens -, 28.5, 20.1, 27.1, 37.3 (a second round of CTAs goes through the whole chain); one request of 32000 -,
    // 9.3, 8.0, 5.9, 5.3.  A thread's loads ahead (1, 2, 4 pieces): as many as its run has.
    int ranks = VERIFY_MAX_CLUSTER;
    while (ranks > 1 && ((long long)n * ranks > 2 * 148 || V <= (ranks / 2) * VERIFY_THREADS * 4)) ranks >>= 1;
    if ((long long)n * ranks > 0x7fffffffLL) {
        tis_set_error("verify_drafts: %d requests", n);
        return TIS_BAD_SIZE;
    }
    const long long runs = (long long)ranks * VERIFY_WARPS, run = (V + runs - 1) / runs;
    VerifyParams v{p, a->p_request, a->p_row, q, a->q_request, a->q_row, reinterpret_cast<const int*>(a->drafts),
                   reinterpret_cast<const float*>(a->u), reinterpret_cast<const int*>(a->lens), reinterpret_cast<int*>(a->tokens),
                   reinterpret_cast<int*>(a->accepted), k, V};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * ranks));
    cfg.blockDim = dim3(VERIFY_THREADS);
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
    if (run <= 128) return verify_launch<1>(cfg, v, run);
    if (run <= 256) return verify_launch<2>(cfg, v, run);
    return verify_launch<4>(cfg, v, run);
}
