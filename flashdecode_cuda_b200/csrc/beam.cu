// Beam search's selection.  Request r keeps the beams (rows of logits) start[r] .. start[r + 1] - 1, beam b with the score s_b, the
// sum of its tokens' log-probabilities.  A candidate is a beam and a token v,
//     c(b, v) = s_b + x(b, v) - lse_b,      lse_b = log sum_v exp x(b, v),
// and the k best of a request by (c descending, (b - first) V + v ascending) are wanted.
//
// Two kernels.  The first streams the logits once: per row the pieces of the normaliser, and per group of 128 neighbouring
// entries their largest value.  Nothing else of the row has to be looked at again: if T is a number that at least k groups'
// maxima reach, every one of the k best reaches T and lies in a group whose maximum does, and those groups are k or a few more of the
// thousands.  The second kernel, one CTA per request, finds such a T, reads those groups again and ranks what reaches T.
//
// Why the sums are in 64 bits: which of two candidates of different beams comes first hangs on the difference of two
// normalisers.  In 32 bits they are off by some 1e-6, and among the candidates of a large batch two that are nearer than
// that are common (gaps of 1e-2 between neighbours: one pair in ten thousand, and a step of 64 requests has a thousand pairs).  The
// exponentials themselves are taken in 32 bits of differences that are exact or off by half a step; their errors of 1e-7 have no
// common sign and average out over the row.  Groups of 16 are added in 32 bits, then in 64.
#include <math.h>

#include "common.cuh"

namespace fd {

constexpr int BM_GROUP = 128;            // entries per group: four coalesced loads of a warp
constexpr int BM_BATCH = 4;              // groups that a warp has in flight at once
constexpr int BM_SCAN_THREADS = 256, BM_SCAN_WARPS = BM_SCAN_THREADS / 32;
constexpr int BM_PICK_THREADS = 1024, BM_PICK_WARPS = BM_PICK_THREADS / 32;
constexpr int BM_MAX_ROWS = 64;          // beams of one request
constexpr int BM_MAX_K = 128;            // candidates of one request
constexpr int BM_LIST = 512;             // groups that may reach T before the exact cut is taken
constexpr int BM_FOUND = 2048;           // entries that may

__device__ __forceinline__ float warp_max_redux(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// How a row's groups are dealt to CTAs: `per` groups (a multiple of what the CTA's warps have in flight) for each of `splits`.
struct BeamPlan {
    int groups, per, splits;
};
static BeamPlan beam_plan(int n, int V) {
    BeamPlan p;
    constexpr int unit = BM_SCAN_WARPS * BM_BATCH;
    p.groups = (V + BM_GROUP - 1) / BM_GROUP;
    const long long total = (long long)n * p.groups;
    const long long want = (total + 148 * 16 - 1) / (148 * 16);          // two waves of eight CTAs per SM
    const long long per = ((want + unit - 1) / unit) * unit;
    p.per = (int)(per < unit ? unit : per);
    if (p.per > p.groups) p.per = ((p.groups + unit - 1) / unit) * unit;
    p.splits = (p.groups + p.per - 1) / p.per;
    return p;
}

__global__ void __launch_bounds__(BM_SCAN_THREADS)
beam_scan_kernel(const float* __restrict__ logits, int V, int groups, int per, float* __restrict__ gmax, float* __restrict__ part_m,
                 double* __restrict__ part_s) {
    const int row = blockIdx.y, split = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* x = logits + (size_t)row * V;
    float* gm = gmax + (size_t)row * groups;
    const int end = min(groups, (split + 1) * per);
    float m = -INFINITY;                 // the warp's running maximum, the same in all lanes
    double s = 0.0;                      // this lane's sum of exp(x - m)
    float v[BM_BATCH][4], nxt[BM_BATCH][4];
    auto fetch = [&](int g0, float (&d)[BM_BATCH][4]) {
#pragma unroll
        for (int j = 0; j < BM_BATCH; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = (g0 + j) * BM_GROUP + e * 32 + lane;
                d[j][e] = (g0 + j < end && i < V) ? __ldg(x + i) : -INFINITY;
            }
    };
    int g0 = split * per + warp * BM_BATCH;
    fetch(g0, v);
    for (; g0 < end; g0 += BM_SCAN_WARPS * BM_BATCH) {
        fetch(g0 + BM_SCAN_WARPS * BM_BATCH, nxt);
        float best[BM_BATCH], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < BM_BATCH; ++j) {
            best[j] = warp_max_redux(fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
            if (lane == j && g0 + j < end) gm[g0 + j] = best[j];
            top = fmaxf(top, best[j]);
        }
        if (top > m) {                   // warp-uniform, and rare after the first few batches
            s *= (double)expf(m - top);  // m = -inf: times 0
            m = top;
        }
        const float mm = m == -INFINITY ? 0.f : m;          // nothing but -inf so far: every exp below is 0, not NaN
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < BM_BATCH; ++j)
            sum += (expf(v[j][0] - mm) + expf(v[j][1] - mm)) + (expf(v[j][2] - mm) + expf(v[j][3] - mm));
        s += (double)sum;
#pragma unroll
        for (int j = 0; j < BM_BATCH; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = nxt[j][e];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __shared__ float sm[BM_SCAN_WARPS];
    __shared__ double ss[BM_SCAN_WARPS];
    if (lane == 0) { sm[warp] = m; ss[warp] = s; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float M = -INFINITY;
        for (int w = 0; w < BM_SCAN_WARPS; ++w) M = fmaxf(M, sm[w]);
        double S = 0.0;
        for (int w = 0; w < BM_SCAN_WARPS; ++w)
            if (sm[w] != -INFINITY) S += ss[w] * exp((double)sm[w] - (double)M);
            else S += ss[w];             // 0, or NaN
        part_m[(size_t)row * gridDim.x + split] = M;
        part_s[(size_t)row * gridDim.x + split] = S;
    }
}

// A candidate's value as an unsigned number that orders like it; 0 for what is no candidate (-inf, NaN).  row: (max_v x, s_b -
// log sum_v exp(x - max)); the maximum is taken off first, which is exact where x is large.
__device__ __forceinline__ unsigned long long beam_key(double2 row, float x) {
    const double c = ((double)x - row.x) + row.y;
    if (!(c > -INFINITY)) return 0ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(c);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double beam_value(unsigned long long key) {
    return __longlong_as_double((long long)((key >> 63) ? (key & 0x7fffffffffffffffull) : ~key));
}

__device__ __forceinline__ int block_total(int v, int* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const int t = __reduce_add_sync(0xffffffffu, scratch[lane]);
        if (lane == 0) scratch[BM_PICK_WARPS] = t;
    }
    __syncthreads();
    const int t = scratch[BM_PICK_WARPS];
    __syncthreads();
    return t;
}

// The exact cut: of the items 0 .. n - 1 with keys key(i) (0: none) those that are among the k first by (key descending, i
// ascending) are the ones with key > T, or key == T and i <= I.  Found bit by bit, each bit a count over all items.
template <typename Key>
__device__ void exact_cut(int n, int k, Key key, unsigned long long& T, int& I, int* scratch) {
    T = 0ull;
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long t = T | (1ull << bit);
        int c = 0;
        for (int i = threadIdx.x; i < n; i += BM_PICK_THREADS) c += key(i) >= t;
        if (block_total(c, scratch) >= k) T = t;
    }
    I = 0x7fffffff;
    if (T == 0ull) { T = 1ull; return; }                       // fewer than k candidates: all of them
    int c = 0;
    for (int i = threadIdx.x; i < n; i += BM_PICK_THREADS) c += key(i) > T;
    const int need = k - block_total(c, scratch);              // of those equal to T, the first so many
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        c = 0;
        for (int i = threadIdx.x; i <= mid; i += BM_PICK_THREADS) c += key(i) == T;
        if (block_total(c, scratch) >= need) hi = mid; else lo = mid + 1;
    }
    I = lo;
}

// One CTA per request.
__global__ void __launch_bounds__(BM_PICK_THREADS)
beam_pick_kernel(const float* __restrict__ logits, int V, int n, const float* __restrict__ scores, const int* __restrict__ start,
                 int groups, int splits, const float* __restrict__ gmax, const float* __restrict__ part_m,
                 const double* __restrict__ part_s, int k, float* __restrict__ out_s, int* __restrict__ out_row,
                 int* __restrict__ out_tok, int* status) {
    __shared__ double2 off[BM_MAX_ROWS];
    __shared__ int list[BM_LIST];
    __shared__ unsigned long long fkey[BM_FOUND];
    __shared__ int fidx[BM_FOUND];
    __shared__ int scratch[BM_PICK_WARPS + 1];
    __shared__ int n_list, n_found;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int first = start[r], last = start[r + 1];
    const bool good = first >= 0 && last >= first && last <= n && last - first <= BM_MAX_ROWS;
    const int nb = good ? last - first : 0;
    if (!good && t == 0) set_status(status, STATUS_BAD_INDEX);
    for (int j = t; j < k; j += BM_PICK_THREADS) {             // what is not found stays so
        out_s[(size_t)r * k + j] = -INFINITY;
        out_row[(size_t)r * k + j] = -1;
        out_tok[(size_t)r * k + j] = -1;
    }
    if (t == 0) { n_list = 0; n_found = 0; }
    // a row whose score or normaliser is no finite number has no candidates
    for (int b = warp; b < nb; b += BM_PICK_WARPS) {
        const size_t p = (size_t)(first + b) * splits;
        float M = -INFINITY;
        for (int i = lane; i < splits; i += 32) M = fmaxf(M, part_m[p + i]);
        M = warp_max(M);
        double S = 0.0;
        for (int i = lane; i < splits; i += 32) {
            const float mi = part_m[p + i];
            S += mi == -INFINITY ? part_s[p + i] : part_s[p + i] * exp((double)mi - (double)M);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
        if (lane == 0) {
            const double o = (double)scores[first + b] - log(S);
            const bool fine = isfinite(o) && isfinite(M);
            off[b] = make_double2(fine ? (double)M : 0.0, fine ? o : -(double)INFINITY);       // or every key of the row is 0
        }
    }
    __syncthreads();
    if (nb == 0) return;

    const float* gm = gmax + (size_t)first * groups;           // the request's groups, one after another
    const float* x = logits + (size_t)first * V;
    const int N = nb * groups;
    auto group_key = [&](int i) { return beam_key(off[i / groups], gm[i]); };
    unsigned long long mine = 0ull;
    for (int i = t; i < N; i += BM_PICK_THREADS) {
        const unsigned long long q = group_key(i);
        mine = q > mine ? q : mine;
    }
    // T: at least k of the threads' maxima reach it (or all candidates do); a few more than k will do
    unsigned long long T = 0ull;
    if (__syncthreads_count(mine != 0ull) >= k) {
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long q = T | (1ull << bit);
            const int c = __syncthreads_count(mine >= q);
            if (c >= k) {
                T = q;
                if (c <= k + k / 4 + 2) break;
            }
        }
    }
    if (T == 0ull) T = 1ull;
    for (int i = t; i < N; i += BM_PICK_THREADS)
        if (group_key(i) >= T) {
            const int at = atomicAdd(&n_list, 1);
            if (at < BM_LIST) list[at] = i;
        }
    __syncthreads();
    int ng = n_list;
    unsigned long long cut = T;
    bool listed = ng <= BM_LIST;
    if (listed) {
        for (int j = warp; j < ng; j += BM_PICK_WARPS) {
            const int i = list[j], b = i / groups, v0 = (i - b * groups) * BM_GROUP;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = v0 + e * 32 + lane;
                const unsigned long long q = v < V ? beam_key(off[b], x[(size_t)b * V + v]) : 0ull;
                if (q >= T) {
                    const int at = atomicAdd(&n_found, 1);
                    if (at < BM_FOUND) { fkey[at] = q; fidx[at] = b * V + v; }
                }
            }
        }
    }
    __syncthreads();
    if (!listed || n_found > BM_FOUND) {
        // Too many entries reach T: rows that are constant, or nearly.  The k best lie in the k best groups (by maximum, then by
        // place: each of k better groups holds an entry that is better than any of a group behind them), and there are at most
        // k x 128 entries in those; both cuts are exact.
        int I;
        exact_cut(N, k, group_key, T, I, scratch);
        if (t == 0) { n_list = 0; n_found = 0; }
        __syncthreads();
        for (int i = t; i < N; i += BM_PICK_THREADS) {
            const unsigned long long q = group_key(i);
            if (q > T || (q == T && i <= I)) list[atomicAdd(&n_list, 1)] = i;          // k at most
        }
        __syncthreads();
        ng = n_list;
        // in the order of their places, so that an entry's number among them orders like its own place
        int at = 0, own = 0;
        if (t < ng) {
            own = list[t];
            for (int j = 0; j < ng; ++j) at += list[j] < own;
        }
        __syncthreads();
        if (t < ng) list[at] = own;
        __syncthreads();
        auto entry_key = [&](int i) {
            const int g = list[i / BM_GROUP], b = g / groups, v = (g - b * groups) * BM_GROUP + i % BM_GROUP;
            return v < V ? beam_key(off[b], x[(size_t)b * V + v]) : 0ull;
        };
        exact_cut(ng * BM_GROUP, k, entry_key, cut, I, scratch);
        for (int i = t; i < ng * BM_GROUP; i += BM_PICK_THREADS) {
            const unsigned long long q = entry_key(i);
            if (q > cut || (q == cut && i <= I)) {
                const int g = list[i / BM_GROUP], b = g / groups;
                const int p = atomicAdd(&n_found, 1);                                  // k at most
                fkey[p] = q;
                fidx[p] = b * V + (g - b * groups) * BM_GROUP + i % BM_GROUP;
            }
        }
        __syncthreads();
    }
    // an entry's place is the number of entries before it
    const int nf = n_found;
    for (int j = t; j < nf; j += BM_PICK_THREADS) {
        const unsigned long long q = fkey[j];
        const int id = fidx[j];
        int rank = 0;
        for (int i = 0; i < nf; ++i) {
            const unsigned long long o = fkey[i];
            rank += o > q || (o == q && fidx[i] < id);
        }
        if (rank < k) {
            const size_t p = (size_t)r * k + rank;
            out_s[p] = (float)beam_value(q);
            out_row[p] = first + id / V;
            out_tok[p] = id % V;
        }
    }
}

}  // namespace fd

using namespace fd;

// Bytes of scratch that fd_beam_select needs for n rows of V logits (8-byte aligned).
extern "C" long long fd_beam_select_scratch_bytes(int n, int V) {
    if (n <= 0 || V <= 0) return 0;
    const BeamPlan p = beam_plan(n, V);
    return (long long)n * p.splits * 12 + (long long)n * p.groups * 4;
}

// logits [n, V], scores [n] float; start [R + 1] int: request r has the rows start[r] .. start[r + 1] - 1, at most 64.  Out [R, k].
extern "C" int fd_beam_select(const float* logits, int n, int V, const float* scores, const int* start, int R, int k,
                              float* out_s, int* out_row, int* out_tok, void* scratch, int* status, cudaStream_t stream) {
    if (R == 0) return 0;
    FD_REQUIRE(n > 0 && V > 0 && R > 0, -2, "beam_select: %d rows of %d logits for %d requests", n, V, R);
    FD_REQUIRE(n <= 65535, -2, "beam_select: %d rows in one call", n);
    FD_REQUIRE(k >= 1 && k <= BM_MAX_K, -2, "beam_select: %d candidates per request; 1 to %d are taken", k, BM_MAX_K);
    FD_REQUIRE((long long)V * BM_MAX_ROWS < (1ll << 31), -2, "beam_select: a vocabulary of %d", V);
    const BeamPlan p = beam_plan(n, V);
    double* part_s = (double*)scratch;
    float* part_m = (float*)(part_s + (size_t)n * p.splits);
    float* gmax = part_m + (size_t)n * p.splits;
    beam_scan_kernel<<<dim3(p.splits, n), BM_SCAN_THREADS, 0, stream>>>(logits, V, p.groups, p.per, gmax, part_m, part_s);
    int rc = check_launch("beam_select");
    if (rc != 0) return rc;
    beam_pick_kernel<<<R, BM_PICK_THREADS, 0, stream>>>(logits, V, n, scores, start, p.groups, p.splits, gmax, part_m, part_s, k,
                                                        out_s, out_row, out_tok, status);
    return check_launch("beam_select_pick");
}
