// Beam search's selection.  Request r keeps the beams (rows of logits) start[r] .. start[r + 1] - 1, beam b with the score s_b, the
// sum of its tokens' log-probabilities.  A candidate is a beam and a token v,
//     c(b, v) = s_b + x(b, v) - lse_b,      lse_b = log sum_v exp x(b, v),
// and the k best of a request by (c descending, (b - first) V + v ascending) are wanted.
//
// The logits are read once: per row the pieces of the normaliser, and per group of 128 neighbouring entries their largest
// value.  Nothing else of the row has to be looked at again: if T is a number that at least k groups' maxima reach, every one
// of the k best reaches T and lies in a group whose maximum does, and those groups are k or a few more of the thousands.  One CTA per
// request finds such a T, reads those groups again and ranks what reaches T.
//
// Two forms.  Few bytes per request: a thread-block cluster per request reads them, leaves the maxima in its shared memory, and its first
// CTA picks from there - one launch, no memory in between.  More: one kernel streams all rows with the whole GPU, a second one picks
// (the clusters' other CTAs would hold their SMs while the first ones pick).
//
// What bounds it.  Many requests: the scan, by HBM.  64 requests of 8 rows of 152,064 (311 MB, floor 47.6 us) take 62.9 us: the scan 52 (6.0
// TB/s), the pick 11 - a chain of a few dozen block-wide steps on 64 CTAs, which starts early (programmatic launch) but has nothing to do
// before the last row's maxima are there.  Few requests: latency.  One request of 4 rows of 151,936 takes 12 us and seven of 3 to
// 8 rows of 50,257 13, of which the bytes would be 0.4 and 1.1: launch and cluster start 3, streaming 160 KB per CTA 4, the pick 5.
//
// Why the sums are in 64 bits: which of two candidates of different beams comes first hangs on the difference of two
// normalisers.  In 32 bits they are off by some 1e-6, and among the candidates of a large batch two that are nearer than
// that are common (gaps of 1e-2 between neighbours: one pair in ten thousand, and a step of 64 requests has a thousand pairs).  The
// exponentials themselves are taken in 32 bits, of differences d = x - max that are exact or off by half a step (beam_exp); what errors of
// 1e-7 are left have no common sign and average out over the row.  Groups of 16 are added in 32 bits, then in 64.
#include <cooperative_groups.h>
#include <math.h>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace fd {

namespace cg = cooperative_groups;

// Entries per group: 128, four coalesced loads of a warp, or 32, one, for small vocabularies: what reaches T comes from few rows
// where the beams' scores are far apart, and T is only as near the k-th best as those rows' groups are many.
constexpr int BM_GROUP = 128, BM_SMALL_GROUP = 32;
constexpr int BM_SMALL_VOCAB = 16384;
constexpr int BM_UNIT = 128;             // entries that a warp takes at a time
constexpr int BM_BATCH = 4;              // such units that a warp has in flight at once
constexpr int BM_SCAN_THREADS = 256, BM_SCAN_WARPS = BM_SCAN_THREADS / 32;
constexpr int BM_PICK_THREADS = 1024;
constexpr int BM_CLUSTER_THREADS = 512;
constexpr int BM_WIDE = 14;              // clusters of 16 that run at once
constexpr int BM_MAX_ROWS = 64;          // beams of one request
constexpr int BM_MAX_K = 128;            // candidates of one request
constexpr int BM_MAX_VOCAB = 1 << 22;    // so that the numbers of a request's groups and entries stay exact in 32 bits
constexpr int BM_LIST = 512;             // groups that may reach T before the exact cut is taken
constexpr int BM_FOUND = 2048;           // entries that may
constexpr int BM_KEPT = 256;             // entries that are ranked (more than that many get a nearer threshold first)

__device__ __forceinline__ float warp_max_redux(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// How a row's units are dealt to CTAs: `per` units (a multiple of what the CTA's warps have in flight) for each of `splits`.
struct BeamPlan {
    int units, per, splits;
};
static BeamPlan beam_plan(int n, int V) {
    BeamPlan p;
    constexpr int unit = BM_SCAN_WARPS * BM_BATCH;
    p.units = (V + BM_UNIT - 1) / BM_UNIT;
    const long long total = (long long)n * p.units;
    const long long want = (total + 148 * 16 - 1) / (148 * 16);          // two waves of eight CTAs per SM
    const long long per = ((want + unit - 1) / unit) * unit;
    p.per = (int)(per < unit ? unit : per);
    if (p.per > p.units) p.per = ((p.units + unit - 1) / unit) * unit;
    p.splits = (p.units + p.per - 1) / p.per;
    return p;
}

// exp(d) for d <= 0; 0 for -inf, NaN for NaN.  2^p of p = d log2 e, times 1 + rest: what the rounding of p leaves out, which alone would make
// it off by |d| 2^-24.  Over every float: off by 3.3 2^-24 of itself at most down to -33, from there (where it hardly counts in a sum
// that has a 1) by up to 5.5 at -87, since log2 e and ln 2 are rounded too.
__device__ __forceinline__ float beam_exp(float d) {
    float r;
    asm("max.NaN.f32 %0, %0, 0fC3480000;" : "+f"(d));            // -200: 2^p is 0 from there on, and the rest a number
    const float p = __fmul_rn(d, 1.44269502162933349609375f), rest = fmaf(p, -0.693147182464599609375f, d);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p));
    return fmaf(r, rest, r);
}

// A warp's share of one row: units g, g + stride, ... of those before `end`, BM_BATCH neighbours at a time.  The maxima of their groups
// go to gm[group]; (m, s): the largest value (the same in all lanes) and this lane's sum of exp(x - m).
// VEC: a lane has four neighbours (rows that are a multiple of four, 16-byte aligned), else every 32nd.  SMALL: groups of 32.
template <bool VEC, bool SMALL>
__device__ __forceinline__ void beam_scan_row(const float* __restrict__ x, int V, int g, int end, int stride, float* gm, float& m, double& s) {
    const int lane = threadIdx.x & 31;
    float v[BM_BATCH][4], nxt[BM_BATCH][4];
    auto fetch = [&](int g0, float (&d)[BM_BATCH][4]) {
        if (g0 + BM_BATCH <= end && (g0 + BM_BATCH) * BM_UNIT <= V) {           // whole groups: no check per entry
            const float* p = x + (size_t)g0 * BM_UNIT;
#pragma unroll
            for (int j = 0; j < BM_BATCH; ++j) {
                if (VEC) {
                    const float4 q = __ldcs(reinterpret_cast<const float4*>(p + j * BM_UNIT) + lane);
                    d[j][0] = q.x; d[j][1] = q.y; d[j][2] = q.z; d[j][3] = q.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[j][e] = __ldcs(p + j * BM_UNIT + e * 32 + lane);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < BM_BATCH; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = (g0 + j) * BM_UNIT + (VEC ? lane * 4 + e : e * 32 + lane);
                    d[j][e] = g0 + j < end && i < V ? __ldcs(x + i) : -INFINITY;
                }
        }
    };
    if (g < end) fetch(g, v);
    for (; g < end; g += stride) {
        if (g + stride < end) fetch(g + stride, nxt);
        float top = -INFINITY, kept = -INFINITY;                 // lane i keeps the i-th maximum
        if (SMALL) {
#pragma unroll
            for (int j = 0; j < BM_BATCH; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float best = warp_max_redux(v[j][e]);
                    top = fmaxf(top, best);
                    if (lane == j * 4 + e) kept = best;
                }
            if (lane < BM_BATCH * 4 && g + lane / 4 < end && (g * 4 + lane) * BM_SMALL_GROUP < V) gm[g * 4 + lane] = kept;
        } else {
#pragma unroll
            for (int j = 0; j < BM_BATCH; ++j) {
                const float best = warp_max_redux(fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
                top = fmaxf(top, best);
                if (lane == j) kept = best;
            }
            if (lane < BM_BATCH && g + lane < end) gm[g + lane] = kept;
        }
        if (top > m) {                   // warp-uniform, and rare after the first few batches
            s *= (double)beam_exp(m - top);                      // m = -inf: times 0
            m = top;
        }
        const float mm = m == -INFINITY ? 0.f : m;               // nothing but -inf so far: every exp below is 0, not NaN
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < BM_BATCH; ++j)
            sum += (beam_exp(v[j][0] - mm) + beam_exp(v[j][1] - mm)) + (beam_exp(v[j][2] - mm) + beam_exp(v[j][3] - mm));
        s += (double)sum;
#pragma unroll
        for (int j = 0; j < BM_BATCH; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = nxt[j][e];
    }
}

// (m, s) of the CTA's warps as one, in thread 0.
template <int WARPS>
__device__ __forceinline__ void beam_join(float& m, double& s, float* sm, double* ss) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) { sm[warp] = m; ss[warp] = s; }
    __syncthreads();
    if (warp == 0) {
        m = lane < WARPS ? sm[lane] : -INFINITY;
        s = lane < WARPS ? ss[lane] : 0.0;
        const float M = warp_max(m);
        if (m != -INFINITY) s *= exp((double)m - (double)M);     // else 0, or NaN
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        m = M;
    }
}

template <bool VEC, bool SMALL>
__global__ void __launch_bounds__(BM_SCAN_THREADS)
beam_scan_kernel(const float* __restrict__ logits, int V, int units, int groups, int per, float* __restrict__ gmax, float* __restrict__ part_m,
                 double* __restrict__ part_s) {
    pdl_launch_dependents();                                   // the pick is set up while the last rows are read
    const int row = blockIdx.y, split = blockIdx.x, warp = threadIdx.x >> 5;
    float m = -INFINITY;
    double s = 0.0;
    beam_scan_row<VEC, SMALL>(logits + (size_t)row * V, V, split * per + warp * BM_BATCH, min(units, (split + 1) * per), BM_SCAN_WARPS * BM_BATCH,
                       gmax + (size_t)row * groups, m, s);
    __shared__ float sm[BM_SCAN_WARPS];
    __shared__ double ss[BM_SCAN_WARPS];
    beam_join<BM_SCAN_WARPS>(m, s, sm, ss);
    if (threadIdx.x == 0) {
        part_m[(size_t)row * gridDim.x + split] = m;
        part_s[(size_t)row * gridDim.x + split] = s;
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

template <int THREADS>
__device__ __forceinline__ int block_total(int v, int* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const int t = __reduce_add_sync(0xffffffffu, lane < THREADS / 32 ? scratch[lane] : 0);
        if (lane == 0) scratch[32] = t;
    }
    __syncthreads();
    const int t = scratch[32];
    __syncthreads();
    return t;
}

// The exact cut: of the items 0 .. n - 1 with keys key(i) (0: none) those that are among the k first by (key descending, i
// ascending) are the ones with key > T, or key == T and i <= I.  Found bit by bit, each bit a count over all items.
template <int THREADS, typename Key>
__device__ void exact_cut(int n, int k, Key key, unsigned long long& T, int& I, int* scratch) {
    T = 0ull;
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long t = T | (1ull << bit);
        int c = 0;
        for (int i = threadIdx.x; i < n; i += THREADS) c += key(i) >= t;
        if (block_total<THREADS>(c, scratch) >= k) T = t;
    }
    I = 0x7fffffff;
    if (T == 0ull) { T = 1ull; return; }                       // fewer than k candidates: all of them
    int c = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) c += key(i) > T;
    const int need = k - block_total<THREADS>(c, scratch);              // of those equal to T, the first so many
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        c = 0;
        for (int i = threadIdx.x; i <= mid; i += THREADS) c += key(i) == T;
        if (block_total<THREADS>(c, scratch) >= need) hi = mid; else lo = mid + 1;
    }
    I = lo;
}

// What one CTA does for a request once the logits have been read.  off[b]: (max, s_b - log sum exp(x - max)) of its rows; the maxima of
// its groups lie in pieces: piece c, at at(c), has groups c * seg .. of every row, [rows][seg].
struct BeamShared {
    double2 off[BM_MAX_ROWS];
    unsigned long long fkey[BM_FOUND], key[BM_KEPT];
    int fidx[BM_FOUND], idx[BM_KEPT];
    int list[BM_LIST];
    int scratch[33];
    int counts[2][32];
    int n_list, n_found, n_kept;
};
struct BeamOut {
    float* score;
    int* row;
    int* tok;
};

// Division by a number that is not known to the compiler, for numbers below 2^22, divisors up to 2^15 and quotients up to 2^6: i + 1/2
// is exact, the quotient is off by less than 2^6 2^-22, and (i + 1/2) / d is at least 2^-16 from a whole number.
struct BeamDiv {
    float inv;
    int d;
    __device__ __forceinline__ explicit BeamDiv(int v) : inv(1.f / (float)v), d(v) {}
    __device__ __forceinline__ int operator()(int i) const { return (int)(((float)i + 0.5f) * inv); }
};
template <typename At>
struct BeamMaxima {
    BeamDiv row, piece;
    At at;
    __device__ __forceinline__ float operator()(int i, int& b) const {
        b = row(i);
        const int g = i - b * row.d, c = piece(g);
        return at(c)[b * piece.d + g - c * piece.d];
    }
};

__device__ __forceinline__ void beam_none(const BeamOut& out, int r, int k) {     // what is not found stays so
    for (int j = threadIdx.x; j < k; j += blockDim.x) {
        out.score[(size_t)r * k + j] = -INFINITY;
        out.row[(size_t)r * k + j] = -1;
        out.tok[(size_t)r * k + j] = -1;
    }
}

// A row's pieces (m, s) are added up; a row whose score or normaliser is no finite number has no candidates.  Called by a warp.
template <typename Piece>
__device__ __forceinline__ double2 beam_offset(float score, int pieces, Piece piece) {
    const int lane = threadIdx.x & 31;
    float M = -INFINITY;
    for (int i = lane; i < pieces; i += 32) M = fmaxf(M, piece(i).x);
    M = warp_max(M);
    double S = 0.0;
    for (int i = lane; i < pieces; i += 32) {
        const double2 p = piece(i);
        S += p.x == -INFINITY ? p.y : p.y * exp(p.x - (double)M);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
    const double o = (double)score - log(S);
    const bool fine = isfinite(o) && isfinite(M);
    return make_double2(fine ? (double)M : 0.0, fine ? o : -(double)INFINITY);               // -inf: every key of the row is 0
}

// A number that at least k of the threads' `keys` (N of them each, 0: none) reach, and hardly more; 1 where there are fewer than k.
template <int THREADS, int N>
__device__ __forceinline__ unsigned long long beam_threshold(BeamShared& sh, const unsigned long long (&keys)[N], int k) {
    constexpr int WARPS = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int step = 0;
    auto reach = [&](unsigned long long q) {
        if constexpr (N == 1) return __syncthreads_count(keys[0] >= q);
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += keys[i] >= q;
        c = __reduce_add_sync(0xffffffffu, c);
        int* to = sh.counts[step++ & 1];                         // (the one before is still being read)
        if (lane == 0) to[warp] = c;
        __syncthreads();
        return __reduce_add_sync(0xffffffffu, lane < WARPS ? to[lane] : 0);
    };
    if (reach(1ull) < k) return 1ull;
    unsigned long long T = 0ull;
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long q = T | (1ull << bit);
        const int c = reach(q);
        if (c >= k) {
            T = q;
            if (c <= k + k / 4 + 2) break;
        }
    }
    return T;
}

template <int THREADS, int GROUP, typename At>
__device__ void beam_pick(BeamShared& sh, const float* __restrict__ x, int V, int groups, int nb, int first, int seg, At at, int k, int r,
                          const BeamOut& out) {
    constexpr int WARPS = THREADS / 32;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int N = nb * groups;
    const BeamMaxima<At> maxima{BeamDiv(groups), BeamDiv(seg), at};
    auto group_key = [&](int i) {
        int b;
        const float v = maxima(i, b);
        return beam_key(sh.off[b], v);
    };
    if (t == 0) sh.n_list = sh.n_found = sh.n_kept = 0;
    // the thread's largest, and its second: with few groups per thread hardly one has two that reach T
    unsigned long long mine[1] = {0ull}, second = 0ull;
    int where = 0;
#pragma unroll 8
    for (int i = t; i < N; i += THREADS) {
        const unsigned long long q = group_key(i);
        const bool more = q > mine[0];
        second = more ? mine[0] : (q > second ? q : second);
        where = more ? i : where;
        mine[0] = more ? q : mine[0];
    }
    unsigned long long T = beam_threshold<THREADS>(sh, mine, k);
    auto list = [&](int i) {
        const int p = atomicAdd(&sh.n_list, 1);
        if (p < BM_LIST) sh.list[p] = i;
    };
    if (second >= T) {
        for (int i = t; i < N; i += THREADS)
            if (group_key(i) >= T) list(i);
    } else if (mine[0] >= T) {
        list(where);
    }
    __syncthreads();
    int ng = sh.n_list;
    const bool listed = ng <= BM_LIST;
    constexpr int EACH = GROUP / 32;                             // entries of a group per lane
    // `many`: groups that a warp reads at once
    auto read = [&](auto many) {
        constexpr int BATCH = decltype(many)::value;
        for (int j0 = warp; j0 < ng; j0 += WARPS * BATCH) {
            float e[BATCH][EACH];
            int row[BATCH], at0[BATCH];
#pragma unroll
            for (int c = 0; c < BATCH; ++c) {
                const int i = sh.list[min(j0 + c * WARPS, ng - 1)];
                row[c] = maxima.row(i);
                at0[c] = (i - row[c] * groups) * GROUP + lane;
#pragma unroll
                for (int u = 0; u < EACH; ++u)
                    e[c][u] = j0 + c * WARPS < ng && at0[c] + u * 32 < V ? __ldg(x + (size_t)row[c] * V + at0[c] + u * 32) : -INFINITY;
            }
#pragma unroll
            for (int c = 0; c < BATCH; ++c)
#pragma unroll
                for (int u = 0; u < EACH; ++u) {
                    const unsigned long long q = beam_key(sh.off[row[c]], e[c][u]);
                    if (q >= T) {                                // (T is 1 or more: not what is no candidate)
                        const int p = atomicAdd(&sh.n_found, 1);
                        if (p < BM_FOUND) { sh.fkey[p] = q; sh.fidx[p] = row[c] * V + at0[c] + u * 32; }
                    }
                }
        }
    };
    if (listed && ng <= WARPS) read(std::integral_constant<int, 1>());
    else if (listed) read(std::integral_constant<int, EACH == 1 ? 4 : 2>());
    __syncthreads();
    const unsigned long long* key = sh.fkey;
    const int* idx = sh.fidx;
    int nf = sh.n_found;
    bool exact = !listed || nf > BM_FOUND;
    if (!exact && nf > BM_KEPT) {
        // a nearer threshold, from the entries themselves
        unsigned long long own[BM_FOUND / THREADS];
#pragma unroll
        for (int u = 0; u < BM_FOUND / THREADS; ++u) own[u] = t + u * THREADS < nf ? sh.fkey[t + u * THREADS] : 0ull;
        const unsigned long long T2 = beam_threshold<THREADS>(sh, own, k);
#pragma unroll
        for (int u = 0; u < BM_FOUND / THREADS; ++u)
            if (own[u] >= T2 && own[u] != 0ull) {
                const int p = atomicAdd(&sh.n_kept, 1);
                if (p < BM_KEPT) { sh.key[p] = own[u]; sh.idx[p] = sh.fidx[t + u * THREADS]; }
            }
        __syncthreads();
        key = sh.key;
        idx = sh.idx;
        nf = sh.n_kept;
        exact = nf > BM_KEPT;
    }
    if (exact) {
        // Too many entries reach T: rows that are constant, or nearly.  The k best lie in the k best groups (by maximum, then by
        // place: each of k better groups holds an entry that is better than any of a group behind them), and there are at most
        // k x 128 entries in those; both cuts are exact.
        int I;
        exact_cut<THREADS>(N, k, group_key, T, I, sh.scratch);
        if (t == 0) sh.n_list = sh.n_kept = 0;
        __syncthreads();
        for (int i = t; i < N; i += THREADS) {
            const unsigned long long q = group_key(i);
            if (q > T || (q == T && i <= I)) sh.list[atomicAdd(&sh.n_list, 1)] = i;          // k at most
        }
        __syncthreads();
        ng = sh.n_list;
        // in the order of their places, so that an entry's number among them orders like its own place
        int place = 0, own = 0;
        if (t < ng) {
            own = sh.list[t];
            for (int j = 0; j < ng; ++j) place += sh.list[j] < own;
        }
        __syncthreads();
        if (t < ng) sh.list[place] = own;
        __syncthreads();
        auto entry = [&](int i, int& b) {
            const int g = sh.list[i / GROUP];
            b = maxima.row(g);
            return (g - b * groups) * GROUP + i % GROUP;
        };
        auto entry_key = [&](int i) {
            int b;
            const int v = entry(i, b);
            return v < V ? beam_key(sh.off[b], x[(size_t)b * V + v]) : 0ull;
        };
        unsigned long long cut;
        exact_cut<THREADS>(ng * GROUP, k, entry_key, cut, I, sh.scratch);
        for (int i = t; i < ng * GROUP; i += THREADS) {
            const unsigned long long q = entry_key(i);
            if (q > cut || (q == cut && i <= I)) {
                int b;
                const int v = entry(i, b), p = atomicAdd(&sh.n_kept, 1);                     // k at most
                sh.key[p] = q;
                sh.idx[p] = b * V + v;
            }
        }
        __syncthreads();
        key = sh.key;
        idx = sh.idx;
        nf = sh.n_kept;
    }
    // an entry's place is the number of entries before it: a warp counts them for one
    for (int j = warp; j < nf; j += WARPS) {
        const unsigned long long q = key[j];
        const int id = idx[j];
        int before = 0;
#pragma unroll 2
        for (int i = lane; i < nf; i += 32) {
            const unsigned long long o = key[i];
            before += o > q || (o == q && idx[i] < id);
        }
        const int place = __reduce_add_sync(0xffffffffu, before);
        if (lane == 0 && place < k) {
            const size_t p = (size_t)r * k + place;
            out.score[p] = (float)beam_value(q);
            out.row[p] = first + id / V;
            out.tok[p] = id % V;
        }
    }
}

// The rows of request r; none (and a report) where the range is no range.
__device__ __forceinline__ int beam_rows(const int* start, int r, int n, int& first, int* status) {
    first = start[r];
    const int last = start[r + 1];
    if (first >= 0 && last >= first && last <= n && last - first <= BM_MAX_ROWS) return last - first;
    if (threadIdx.x == 0) set_status(status, STATUS_BAD_INDEX);
    return 0;
}

// One CTA per request, behind the scan.
template <int GROUP>
__global__ void __launch_bounds__(BM_PICK_THREADS)
beam_pick_kernel(const float* __restrict__ logits, int V, int n, const float* __restrict__ scores, const int* __restrict__ start,
                 int groups, int splits, const float* __restrict__ gmax, const float* __restrict__ part_m,
                 const double* __restrict__ part_s, int k, const BeamOut out, int* status) {
    __shared__ BeamShared sh;
    const int r = blockIdx.x;
    pdl_wait();
    int first;
    const int nb = beam_rows(start, r, n, first, status);
    beam_none(out, r, k);
    for (int b = threadIdx.x >> 5; b < nb; b += BM_PICK_THREADS / 32) {
        const size_t p = (size_t)(first + b) * splits;
        const double2 o = beam_offset(scores[first + b], splits, [&](int i) { return make_double2(part_m[p + i], part_s[p + i]); });
        if ((threadIdx.x & 31) == 0) sh.off[b] = o;
    }
    __syncthreads();
    if (nb == 0) return;
    const float* gm = gmax + (size_t)first * groups;           // the request's groups, one after another
    beam_pick<BM_PICK_THREADS, GROUP>(sh, logits + (size_t)first * V, V, groups, nb, first, groups, [&](int) { return gm; }, k, r, out);
}

// One cluster per request: each CTA has the same part of every row, each warp the same part of that (so that equal rows have equal
// normalisers, to the bit); the first CTA picks.
template <bool VEC, bool SMALL>
__global__ void __launch_bounds__(BM_CLUSTER_THREADS)
beam_cluster_kernel(const float* __restrict__ logits, int V, int n, const float* __restrict__ scores, const int* __restrict__ start,
                    int units, int groups, int k, const BeamOut out, int* status) {
    constexpr int WARPS = BM_CLUSTER_THREADS / 32;
    extern __shared__ float gm[];                              // [rows][seg]: the maxima of this CTA's groups
    __shared__ BeamShared sh;
    __shared__ double2 parts[BM_MAX_ROWS * WARPS];             // (m, s) of each warp's part of each row
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), r = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int first;
    const int nb = beam_rows(start, r, n, first, status);
    if (rank == 0) beam_none(out, r, k);
    if (nb == 0) return;                                       // the same for the whole cluster
    const int per = (units + C - 1) / C, u0 = rank * per, u1 = min(units, u0 + per);
    constexpr int GROUP = SMALL ? BM_SMALL_GROUP : BM_GROUP;
    const int seg = per * (BM_UNIT / GROUP);                   // groups of a part
    int per_row = 1;                                           // warps that share a row: no more than have work, all rows at once
    while (2 * per_row * nb <= WARPS && per_row * BM_BATCH < per) per_row *= 2;
    for (int b = warp / per_row; b < nb; b += WARPS / per_row) {
        float m = -INFINITY;
        double s = 0.0;
        beam_scan_row<VEC, SMALL>(logits + (size_t)(first + b) * V, V, u0 + (warp % per_row) * BM_BATCH, u1, per_row * BM_BATCH, gm + b * seg - rank * seg, m, s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) parts[b * per_row + warp % per_row] = make_double2(m, s);
    }
    cluster.sync();
    if (rank == 0) {
        for (int b = warp; b < nb; b += WARPS) {
            const double2 o = beam_offset(scores[first + b], C * per_row,
                                          [&](int i) { return *cluster.map_shared_rank(parts + b * per_row + i % per_row, i / per_row); });
            if (lane == 0) sh.off[b] = o;
        }
        __syncthreads();
        beam_pick<BM_CLUSTER_THREADS, GROUP>(sh, logits + (size_t)first * V, V, groups, nb, first, seg,
                                      [&](int c) { return (const float*)cluster.map_shared_rank(gm, c); }, k, r, out);
    }
    cluster.sync();                                            // the maxima have been read
}

}  // namespace fd

using namespace fd;

// Bytes of logits per CTA, and rows per request, up to which the one launch is taken.  Measured, clusters / two kernels, us on the device (a
// call costs the host 10 to 13 and 12 to 17 us, which is what counts when calls follow each other): 4 rows of 151,936 (152 KB per CTA)
// 12.1 / 10.4; 36 ragged rows of 50,257 for 7 requests (65 KB) 13.2 / 10.7; 64 rows of 32,000 for 16 10.1 / 9.5; 106 rows of 2,410 for 53
// 8.2 / 8.4; but 117 of 120,971 for 13 (272 KB) 31 / 22, 512 of 152,064 for 64 93 / 63; 22 rows of 14,151 for one request 21 / 14.5, 240
// of 1,000 for 8 15.8 / 11.6: many rows have many maxima, and of the two picks the one of 1,024 threads that reads them from L2 is the faster.
constexpr long long BM_CLUSTER_BYTES = 160 * 1024;
constexpr int BM_CLUSTER_ROWS = 12;

// Bytes of scratch that fd_beam_select needs for n rows of V logits (8-byte aligned).
extern "C" long long fd_beam_select_scratch_bytes(int n, int V) {
    if (n <= 0 || V <= 0) return 0;
    const BeamPlan p = beam_plan(n, V);
    return (long long)n * p.splits * 12 + (long long)n * p.units * (V <= BM_SMALL_VOCAB ? 16 : 4);
}

extern "C" int fd_sm_count();

static int g_beam_form = 0;
// Which form fd_beam_select takes from now on: 1 = a cluster per request (where its memory suffices), 2 = two kernels, 0 = by the sizes.
// For tests and measurements.
extern "C" int fd_beam_select_set_form(int form) {
    g_beam_form = form;
    return 0;
}

// logits [n, V], scores [n] float; start [R + 1] int: request r has the rows start[r] .. start[r + 1] - 1, at most 64.  Out [R, k].
extern "C" int fd_beam_select(const float* logits, int n, int V, const float* scores, const int* start, int R, int k,
                              float* out_s, int* out_row, int* out_tok, void* scratch, int* status, cudaStream_t stream) {
    if (R == 0) return 0;
    FD_REQUIRE(n >= 0 && V > 0 && R > 0, -2, "beam_select: %d rows of %d logits for %d requests", n, V, R);
    FD_REQUIRE(n <= 65535, -2, "beam_select: %d rows in one call", n);
    FD_REQUIRE(k >= 1 && k <= BM_MAX_K, -2, "beam_select: %d candidates per request; 1 to %d are taken", k, BM_MAX_K);
    FD_REQUIRE(V <= BM_MAX_VOCAB, -2, "beam_select: a vocabulary of %d; up to %d are taken", V, BM_MAX_VOCAB);
    // (places are cleared before the scores are read, and one request's are written while another's rows still are)
    const auto apart = [](const void* p, long long a, const void* q, long long b) {
        const unsigned long long x = (unsigned long long)p, y = (unsigned long long)q;
        return x + a <= y || y + b <= x;
    };
    const long long wide = 4ll * R * k;
    for (const void* o : {(const void*)out_s, (const void*)out_row, (const void*)out_tok})
        FD_REQUIRE(apart(o, wide, logits, 4ll * n * V) && apart(o, wide, scores, 4ll * n) && apart(o, wide, start, 4ll * (R + 1)), -2,
                   "beam_select: an output shares memory with an input");
    FD_REQUIRE(apart(out_s, wide, out_row, wide) && apart(out_s, wide, out_tok, wide) && apart(out_row, wide, out_tok, wide), -2,
               "beam_select: two outputs share memory");
    const BeamOut out{out_s, out_row, out_tok};
    const bool small = V <= BM_SMALL_VOCAB;
    const bool vec = !small && V % 4 == 0 && (reinterpret_cast<unsigned long long>(logits) & 15) == 0;
    const int sms = fd_sm_count(), units = (V + BM_UNIT - 1) / BM_UNIT, size = small ? BM_SMALL_GROUP : BM_GROUP, groups = (V + size - 1) / size;
    // (64 rows of 32,000 for 16 requests took 17.7 us in clusters of 16, of which 14 run at once, and take 10.6 in clusters of 8)
    int C = 16;
    while (C > 1 && (R * C > 2 * sms || units < C || (C == 16 && R > BM_WIDE))) C /= 2;
    // (a request may have all the rows, up to 64)
    const long long smem = 4ll * (n < BM_MAX_ROWS ? n : BM_MAX_ROWS) * ((units + C - 1) / C) * (BM_UNIT / size);
    const bool fits = smem <= 96 * 1024 && R <= 2 * sms;
    if (n > 0 && fits && g_beam_form != 2 && (g_beam_form == 1 || (n <= BM_CLUSTER_ROWS * R && 4ll * n * V <= BM_CLUSTER_BYTES * R * C))) {
        const int which = small ? 2 : (vec ? 1 : 0);
        void (*const kernels[3])(const float*, int, int, const float*, const int*, int, int, int, const BeamOut, int*) = {
            beam_cluster_kernel<false, false>, beam_cluster_kernel<true, false>, beam_cluster_kernel<false, true>};
        static Once once[3];
        if (once[which].first()) {
            cudaError_t err = cudaFuncSetAttribute(kernels[which], cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
            if (err == cudaSuccess) err = cudaFuncSetAttribute(kernels[which], cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (err != cudaSuccess) return fail(-100, "beam_select: %s", cudaGetErrorString(err));
            once[which].done();
        }
        return launch("beam_select", kernels[which], dim3(R * C), dim3(BM_CLUSTER_THREADS), (size_t)smem, stream, dim3(C, 1, 1), logits, V, n,
                      scores, start, units, groups, k, out, status);
    }
    const BeamPlan p = beam_plan(n, V);
    double* part_s = (double*)scratch;
    float* part_m = (float*)(part_s + (size_t)n * p.splits);
    float* gmax = part_m + (size_t)n * p.splits;
    const dim3 grid(p.splits, n);
    if (n > 0) {                         // (else requests without rows: the pick says so)
        if (small) beam_scan_kernel<false, true><<<grid, BM_SCAN_THREADS, 0, stream>>>(logits, V, units, groups, p.per, gmax, part_m, part_s);
        else if (vec) beam_scan_kernel<true, false><<<grid, BM_SCAN_THREADS, 0, stream>>>(logits, V, units, groups, p.per, gmax, part_m, part_s);
        else beam_scan_kernel<false, false><<<grid, BM_SCAN_THREADS, 0, stream>>>(logits, V, units, groups, p.per, gmax, part_m, part_s);
        const int rc = check_launch("beam_select");
        if (rc != 0) return rc;
    }
    return launch_with(true, "beam_select_pick", small ? beam_pick_kernel<BM_SMALL_GROUP> : beam_pick_kernel<BM_GROUP>, dim3(R),
                       dim3(BM_PICK_THREADS), 0, stream, dim3(1, 1, 1), logits, V, n, scores, start, groups, p.splits, (const float*)gmax,
                       (const float*)part_m, (const double*)part_s, k, out, status);
}
