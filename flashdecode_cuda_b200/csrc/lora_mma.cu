// Low-rank adapters in bfloat16 for steps of few tokens per adapter (decode): out[t] = y[t] + scale B (A x[t]).
//
// Such a step reads the adapters' matrices and little else: 2 (S r K + r N) bytes per adapter in use, whatever the number of
// its tokens, so a tile of up to 16 tokens is bound by streaming them.  A cluster of CTAs takes a tile, as in lora.cu: a share of
// K each, the partial sums exchanged through distributed shared memory, then a share of N each, one launch.  What is different:
//   * the products are mma.sync m16n8k16 with the tokens as the 16 rows.  (tcgen05's 128 rows would be padding, and operands that
//     are used once need no trip through shared memory: weights go from global memory to the registers of the lanes that
//     multiply them.  A lane's 16 bytes are 8 neighbouring values of a row; which of the k places they take is free as long as the
//     other operand's values take the same.)
//   * the sums of A x are 32-bit.  B h takes h as two bfloat16 numbers (what rounding takes away from the first is the second),
//     which is 2^-17 of h apart from it and costs one more MMA on operands that are there already.
//
// Measured (device time): 48 tokens of 12 adapters, gate and up of 3584 x 37888, rank 64 (54 MB, floor 8.3 us): 24.0 us - finding the tile 1.3,
// A x 4.5, the exchange 3 to 4, B h 11.7.  The last is what a warp's passes of 32 columns take to come and go (weights, y and the store of
// each: three trips, the next pass's weights asked for before this one multiplies); DRAM is at 32 % of its rate, the tensor pipe at 6 %.
// One token, q/k/v of 1536 x 2048, rank 16: 6.0 us, launch and the chain of trips.  2,179 tokens, 611 of them without an adapter, 3584 x 3584, rank 32: 21.9 us
// (floor 6.6), bound by what the tiles read of A and B out of L2.
#include <cooperative_groups.h>

#include <algorithm>

#include "lora.cuh"
#include "mma_utils.cuh"

namespace fd {

namespace cg = cooperative_groups;

constexpr int LM_THREADS = 256, LM_WARPS = LM_THREADS / 32;
constexpr int LM_ROWS = 16;              // tokens of a tile: the rows of an MMA
constexpr int LM_TILES = 4;              // tiles of 8 rows of A that a warp accumulates at once
constexpr int LM_RED = LM_TILES * 8 + 4; // floats of a token's row of a warp's sums (4: so that neighbouring rows are in other banks)

__device__ __forceinline__ uint4 ldg16(const __nv_bfloat16* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// x is read by every group of rows of A: it may stay in L1
__device__ __forceinline__ uint4 ldx16(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// A row of hi or lo: the slices' places, and 32 more where that puts neighbouring rows into the same banks (a row is then 64 bytes from
// a multiple of 128, and the eight rows that a load of 16 bytes per lane touches cover the banks evenly).
__host__ __device__ __forceinline__ int lora_row_places(int S, int R) {
    const int n = S * ((R + 31) / 32 * 32);
    return n % 64 == 0 ? n + 32 : n;
}

// 32 places of h of 16 tokens (8, without TWO) as the left operand: both numbers of each.  For 8 tokens the second numbers take the
// place of the other 8 tokens, so that one MMA multiplies both; the two halves of its result are added at the end.
template <bool TWO>
struct LoraFrag {
    static constexpr int STEPS = TWO ? 4 : 2;
    uint4 h0, l0, h1, l1;
    __device__ __forceinline__ void load(const __nv_bfloat16* f, int low, int up) {
        h0 = *reinterpret_cast<const uint4*>(f);
        l0 = *reinterpret_cast<const uint4*>(f + low);
        if (TWO) {
            h1 = *reinterpret_cast<const uint4*>(f + up);
            l1 = *reinterpret_cast<const uint4*>(f + up + low);
        }
    }
    // the MMAs of a tile one after another depend on each other: the caller deals them over tiles
    __device__ __forceinline__ void mma(int m, float acc[4], const uint4& w) const {
        if (TWO) {
            if (m == 0) mma_bf16(acc, h0.x, h1.x, h0.y, h1.y, w.x, w.y);
            if (m == 1) mma_bf16(acc, h0.z, h1.z, h0.w, h1.w, w.z, w.w);
            if (m == 2) mma_bf16(acc, l0.x, l1.x, l0.y, l1.y, w.x, w.y);
            if (m == 3) mma_bf16(acc, l0.z, l1.z, l0.w, l1.w, w.z, w.w);
        } else {
            if (m == 0) mma_bf16(acc, h0.x, l0.x, h0.y, l0.y, w.x, w.y);
            if (m == 1) mma_bf16(acc, h0.z, l0.z, h0.w, l0.w, w.z, w.w);
        }
    }
};

__device__ __forceinline__ uint4 lora_sum8(const uint4& y, const float v[8], float scale) {
    uint4 o;
    const __nv_bfloat162* a = reinterpret_cast<const __nv_bfloat162*>(&y);
    uint32_t* d = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = pack_bf16(fmaf(scale, v[2 * i], __low2float(a[i])), fmaf(scale, v[2 * i + 1], __high2float(a[i])));
    return o;
}

// B h for the columns n0 .. n1 - 1, 32 per warp and pass: four groups of 8 columns of one slice.  Which column of an MMA stands for which
// column of the output is free; column c of MMA i is column 2 i + c % 2 of group c / 2, so that a lane ends up with all of a group's 8
// columns of its token: y and out move 16 bytes at a time, and a pass of 32 columns is two loads and two stores per lane beside the
// weights.  The groups are neighbours, or every other one where two slices take turns (gate and up).
// What bounds it is the load and store pipe (a warp's 16 bytes per lane are eight rows' 64 bytes) beside the memory, so h stays in
// registers from pass to pass (for ranks up to 64), and nothing is selected where what is read does no harm: rows of no token read token 0's y and are not
// stored, groups behind n1 read the last one's weights, chunks behind the rank the first one's against zeros in h.
// NC: chunks of 32 places of h at once; HELD: those are all there are (the rank is at most 32 NC), and stay.
template <int NC, bool TWO, bool HELD = true>
__device__ __forceinline__ void lora_expand(const LoraArgs& p, const __nv_bfloat16* b, const __nv_bfloat16* y, __nv_bfloat16* out,
                                            const __nv_bfloat16* hi, const __nv_bfloat16* lo, int WB, int t0, int t1, int n0, int n1,
                                            int r8, float scale) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int Rc = (p.R + 31) / 32 * 32;                         // places of a slice in hi and lo
    const __nv_bfloat16* h = hi + g * WB + q * 8;
    const int low = (int)(lo - hi), up = 8 * WB;                 // from hi to lo; from a token's row to that of the one eight behind it
    const __nv_bfloat16 *yp0 = y + (size_t)max(t0, 0) * p.N, *yp1 = y + (size_t)max(t1, 0) * p.N;
    __nv_bfloat16 *op0 = out + (size_t)max(t0, 0) * p.N, *op1 = out + (size_t)max(t1, 0) * p.N;
    const __nv_bfloat16* bp = b + (size_t)(g & 1) * p.R + q * 8;
    // Passes come in pairs that share 64 columns.  Lane i knows the slice of group i of those (-1: behind the last): asked for before
    // the pass's weights, which are asked for before the pass before multiplies (where there are registers for both), or each
    // pass would be two or three trips to memory, one after the other.
    struct Pass {
        int at, border, og, slice;
        bool there, one, in;
        uint4 w[NC][4], y0, y1;
    };
    constexpr bool EARLY = HELD && (NC == 1 || !TWO);
    auto slice_of = [&](int at) {
        const int n = n0 + (at >> 1) * 64 + lane * 8;
        return p.col_slice != nullptr && lane < 8 && n < n1 ? (int)__ldg(p.col_slice + n / 8) : -1;
    };
    auto weights = [&](Pass& s, int wg, int j0) {
        const __nv_bfloat16* wp = bp + (size_t)wg * p.R;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (NC > 1 && j0 + c * 32 >= r8) break;
            const int j = j0 + c * 32 + q * 8 < r8 ? j0 + c * 32 : -q * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) s.w[c][i] = ldg16(wp + 2 * i * p.R + j);
        }
    };
    auto open = [&](Pass& s, int at, int border, int groups) -> int {
        const int base = n0 + (at >> 1) * 64, half = at & 1;
        s.at = at;
        s.border = border;
        s.there = base < n1;
        if (!s.there) return 0;
        int step = 8, first = base + half * 32;
        s.slice = 0;
        s.one = true;                                            // all four groups are of one slice
        if (p.col_slice != nullptr) {
            const int c = min(groups, p.S - 1);
            const int c0 = __shfl_sync(0xffffffffu, c, 0), c1 = __shfl_sync(0xffffffffu, c, 1), c4 = __shfl_sync(0xffffffffu, c, 4);
            const bool turns = __all_sync(0xffffffffu, c < 0 || c == (lane & 1 ? c1 : c0)) && c1 >= 0 && c0 != c1;
            if (turns) {
                step = 16;
                first = base + half * 8;
                s.slice = half ? c1 : c0;
            } else {
                s.slice = half ? c4 : c0;
                s.one = __all_sync(0xffffffffu, c < 0 || (lane >> 2) != half || c == s.slice);
            }
        }
        s.og = first + q * step;                                 // the lane's group of outputs
        s.in = s.og < n1;
        if (!s.one) {                                            // a border between slices inside the four groups: a pass for each slice,
            s.slice = border;                                    // which stores the groups that are its own
            s.in = s.in && min((int)__ldg(p.col_slice + s.og / 8), p.S - 1) == border;
        }
        s.slice = max(s.slice, 0);                               // (a pass behind n1 multiplies something, and stores nothing)
        const int wg = min(first + (g >> 1) * step, n1 - 8);     // and of weights
        weights(s, wg, 0);
        if (s.in) {
            s.y0 = *reinterpret_cast<const uint4*>(yp0 + s.og);
            if (TWO) s.y1 = *reinterpret_cast<const uint4*>(yp1 + s.og);
        }
        return wg;
    };
    int held = -1;                                               // the slice that f is of
    LoraFrag<TWO> f[NC];
    Pass now, next;
    int known = slice_of(warp), ahead = slice_of(warp + LM_WARPS);
    int wg = open(now, warp, 0, known);
    while (now.there) {
        const bool again = !now.one && now.border + 1 < p.S;
        const int at = again ? now.at : now.at + LM_WARPS, groups = again ? known : ahead;
        int next_wg = 0;
        if (EARLY) next_wg = open(next, at, again ? now.border + 1 : 0, groups);
        float acc[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        for (int j0 = 0; j0 < (HELD ? 1 : r8); j0 += 32 * NC) {
            if (j0 > 0) weights(now, wg, j0);
            if (!HELD || now.slice != held) {
#pragma unroll
                for (int c = 0; c < NC; ++c) f[c].load(h + now.slice * Rc + min(j0 + c * 32, Rc - 32), low, up);
                held = now.slice;
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (NC > 1 && j0 + c * 32 >= r8) break;
#pragma unroll
                for (int m = 0; m < LoraFrag<TWO>::STEPS; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[c].mma(m, acc[i], now.w[c][i]);
            }
        }
        if (now.in) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) v[2 * i + e] = TWO ? acc[i][e] : acc[i][e] + acc[i][2 + e];
            if (t0 >= 0) *reinterpret_cast<uint4*>(op0 + now.og) = lora_sum8(now.y0, v, scale);
            if (TWO) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) v[2 * i + e] = acc[i][2 + e];
                if (t1 >= 0) *reinterpret_cast<uint4*>(op1 + now.og) = lora_sum8(now.y1, v, scale);
            }
        }
        if (EARLY) {
            now = next;
            wg = next_wg;
        } else {
            wg = open(now, at, again ? now.border + 1 : 0, groups);
        }
        if (!again) {
            known = ahead;
            ahead = slice_of(at + LM_WARPS);
        }
    }
}

__global__ void __launch_bounds__(LM_THREADS, 2)
lora_rows_kernel(const LoraArgs p, int copies) {
    extern __shared__ __align__(16) unsigned char lm_smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, q = lane & 3;                       // an MMA's row or column, and the lane's place along k
    const int W = p.S * p.R;                                     // a token's A x
    const int Rc = (p.R + 31) / 32 * 32, WB = lora_row_places(p.S, p.R);      // ... as bfloat16: slices in whole chunks, and a row
    float* red = reinterpret_cast<float*>(lm_smem);              // [LM_WARPS][LM_ROWS][LM_RED]
    float* part = red + LM_WARPS * LM_ROWS * LM_RED;             // [LM_ROWS][W] this CTA's sums
    __nv_bfloat16* hi = reinterpret_cast<__nv_bfloat16*>(part + LM_ROWS * W);          // [LM_ROWS][WB] the cluster's sums, zeros behind an adapter's rank
    __nv_bfloat16* lo = hi + LM_ROWS * WB;                       // ... and what hi leaves of them
    __shared__ int tok[LM_ROWS];
    __shared__ LoraTile tile_s;
    if (warp == 0) {
        const LoraTile f = lora_tile(p, blockIdx.x / (C * copies), LM_ROWS);
        if (lane < LM_ROWS) {
            int t = lane < f.count ? p.order[f.begin + lane] : -1;
            if (lane < f.count && (t < 0 || t >= p.T)) { set_status(p.status, STATUS_BAD_INDEX); t = -1; }
            tok[lane] = t;
        }
        if (lane == 0) tile_s = f;
    }
    __syncthreads();
    const LoraTile tile = tile_s;
    if (tile.adapter == -2) return;                              // the same for the whole cluster
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x);
    const __nv_bfloat16* y = static_cast<const __nv_bfloat16*>(p.y);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    const int share = blockIdx.x % (C * copies), per = ((p.N + 63) / 64 + C * copies - 1) / (C * copies) * 64;
    const int n0 = min(p.N, share * per), n1 = min(p.N, n0 + per);               // this CTA's columns
    const bool in_place = static_cast<const void*>(out) == p.y;
    const int e = max(tile.adapter, 0), r = tile.adapter < 0 ? 0 : min(max(p.ranks[e], 0), p.R);
    if (r == 0) {                                                // nothing to add
        if (in_place) return;
        lora_copy<uint4>(tok, tile.count, p.y, p.out, p.N / 8, n0 / 8, n1 / 8, tid, LM_THREADS);
        return;
    }
    const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + (size_t)e * W * p.K;
    const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.b) + (size_t)e * p.N * p.R;
    const int r8 = (r + 7) / 8 * 8, tiles = r8 / 8;              // rows of A in tiles of 8, per slice
    // --- A x: this CTA's share of K, cut over its warps in chunks of 32
    const int kper = ((p.K + 31) / 32 + C - 1) / C * 32, k0 = rank * kper, k1 = min(p.K, k0 + kper);
    const int t0 = tok[g], t1 = tok[g + 8];
    const __nv_bfloat16* x0 = x + (size_t)max(t0, 0) * p.K;
    const __nv_bfloat16* x1 = x + (size_t)max(t1, 0) * p.K;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < LM_ROWS * WB; i += LM_THREADS)         // places behind the rank, rows of no token: operands that must be numbers
        reinterpret_cast<uint32_t*>(hi)[i] = 0u;
    // Groups of 32 rows of A; a pass takes up to eight groups, and deals the warps that are left over to parts of the K range.
    const int all = p.S * tiles, groups = (all + LM_TILES - 1) / LM_TILES;
    for (int first = 0; first < groups; first += LM_WARPS) {
        const int G = min(LM_WARPS, groups - first), parts = LM_WARPS / G, mine_g = warp / parts, mine_p = warp - mine_g * parts;
        if (mine_g < G) {
            float acc[LM_TILES][4];
            const __nv_bfloat16* rows[LM_TILES];
            const int u0 = (first + mine_g) * LM_TILES, nu = min(LM_TILES, all - u0);
#pragma unroll
            for (int i = 0; i < LM_TILES; ++i) {
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
                const int u = u0 + min(i, nu - 1), s = u / tiles;
                rows[i] = a + (size_t)(s * p.R + (u - s * tiles) * 8 + g) * p.K;
            }
            // whole chunks, nothing selected: rows of no token read token 0's x, and what comes of them goes nowhere
            const int kw = k1 - (k1 - k0) % 32;
            int k = k0 + mine_p * 32 + q * 8;
#pragma unroll 2
            for (; k < kw; k += parts * 32) {
                uint4 w[LM_TILES];
#pragma unroll
                for (int i = 0; i < LM_TILES; ++i) w[i] = ldg16(rows[i] + k);
                const uint4 xa = ldx16(x0 + k), xb = ldx16(x1 + k);
#pragma unroll
                for (int i = 0; i < LM_TILES; ++i) mma_bf16(acc[i], xa.x, xb.x, xa.y, xb.y, w[i].x, w[i].y);
#pragma unroll
                for (int i = 0; i < LM_TILES; ++i) mma_bf16(acc[i], xa.z, xb.z, xa.w, xb.w, w[i].z, w[i].w);
            }
            if (k - q * 8 < k1) {                                // the end of K: a multiple of 8, so a lane's values are all there or none
                const bool in = k < k1;
                const uint4 xa = in ? ldx16(x0 + k) : none, xb = in ? ldx16(x1 + k) : none;
#pragma unroll
                for (int i = 0; i < LM_TILES; ++i) {
                    const uint4 w = in ? ldg16(rows[i] + k) : none;
                    mma_bf16(acc[i], xa.x, xb.x, xa.y, xb.y, w.x, w.y);
                    mma_bf16(acc[i], xa.z, xb.z, xa.w, xb.w, w.z, w.w);
                }
            }
            float* mine = red + warp * LM_ROWS * LM_RED;
#pragma unroll
            for (int i = 0; i < LM_TILES; ++i) {
                *reinterpret_cast<float2*>(mine + g * LM_RED + i * 8 + q * 2) = make_float2(acc[i][0], acc[i][1]);
                *reinterpret_cast<float2*>(mine + (g + 8) * LM_RED + i * 8 + q * 2) = make_float2(acc[i][2], acc[i][3]);
            }
        }
        __syncthreads();
        // a warp takes whole tiles of 8 rows of A: the sums of all tokens over the group's parts
        for (int u = warp; u < min(all - first * LM_TILES, G * LM_TILES); u += LM_WARPS) {
            const int gi = u / LM_TILES, uu = first * LM_TILES + u, s = uu / tiles, j = (uu - s * tiles) * 8 + (lane & 7);
            const float* f = red + gi * parts * LM_ROWS * LM_RED + (u - gi * LM_TILES) * 8 + (lane & 7);
#pragma unroll
            for (int row = lane >> 3; row < LM_ROWS; row += 4) {
                float v = 0.f;
                for (int w = 0; w < parts; ++w) v += f[(w * LM_ROWS + row) * LM_RED];
                part[row * W + s * p.R + j] = j < r ? v : 0.f;
            }
        }
        __syncthreads();
    }
    // --- the cluster's sums, in the order of the ranks; every CTA reads all of them
    cluster.sync();
    const int width = p.S * r8, used = width * tile.count;       // (token, place) pairs that matter
    for (int i = tid; i < used; i += LM_THREADS) {
        const int row = i / width, c = i - row * width, s = c / r8, j = c - s * r8;
        const float* f = part + row * W + s * p.R + j;
        float v = 0.f;
        if (C == 16) {                                           // all in flight at once
#pragma unroll
            for (int k = 0; k < 16; ++k) v += *cluster.map_shared_rank(f, k);
        } else {
#pragma unroll 4
            for (int k = 0; k < C; ++k) v += *cluster.map_shared_rank(f, k);
        }
        hi[row * WB + s * Rc + j] = __float2bfloat16_rn(v);
        lo[row * WB + s * Rc + j] = __float2bfloat16_rn(lora_rest(v));
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");        // the others' sums have been read
    __syncthreads();

    // --- B h
    const float scale = p.scale[e];
    if (tile.count > 8) {
        if (r8 <= 32) lora_expand<1, true>(p, b, y, out, hi, lo, WB, t0, t1, n0, n1, r8, scale);
        else if (r8 <= 64) lora_expand<2, true>(p, b, y, out, hi, lo, WB, t0, t1, n0, n1, r8, scale);
        else lora_expand<2, true, false>(p, b, y, out, hi, lo, WB, t0, t1, n0, n1, r8, scale);
    } else {
        if (r8 <= 32) lora_expand<1, false>(p, b, y, out, hi, lo, WB, t0, t1, n0, n1, r8, scale);
        else if (r8 <= 64) lora_expand<2, false>(p, b, y, out, hi, lo, WB, t0, t1, n0, n1, r8, scale);
        else lora_expand<2, false, false>(p, b, y, out, hi, lo, WB, t0, t1, n0, n1, r8, scale);
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");          // this CTA's sums have been read by all
}

// Whether the tensor-core kernels take the sizes: 16-byte pieces of every row, and a rank whose h fits the registers.
bool lora_mma_takes(const LoraArgs& p) {
    const unsigned long long all = (unsigned long long)p.x | (unsigned long long)p.a | (unsigned long long)p.b |
                                   (unsigned long long)p.y | (unsigned long long)p.out;
    return (all & 15) == 0 && p.K % 8 == 0 && p.N % 8 == 0 && p.R % 8 == 0 && p.R <= 128;
}

int lora_rows(const LoraArgs& p, int sms, cudaStream_t stream) {
    const long long tiles = lora_max_tiles(p, LM_ROWS);
    const int most = p.K > p.N ? p.K : p.N;
    // The largest cluster of which all run at once, by the tiles that there should be, and
    // where half of them would still run at once, several clusters share a tile's columns (and each computes A x: the second reads A from
    // L2).  One cluster too many takes a second wave: 3584 x 37888 in two slices, rank 64, 8 tokens of 8 adapters in 16 clusters of 16 29
    // us, in 8 22; 17 adapters in 34 clusters of 8 45, in 17 35.
    const long long likely = lora_likely_tiles(p);
    int C = 16;
    while (C > 1 && (likely > lora_room(C, sms) || most < 64 * C)) C /= 2;
    int copies = std::max(1, (int)(lora_room(C, sms) / likely));
    while (copies > 1 && p.N < 256 * C * copies) --copies;
    FD_REQUIRE(tiles * C * copies < (1ll << 31), -2, "lora_add: %d tokens", p.T);
    const int W = p.S * p.R;
    const size_t smem = sizeof(float) * (LM_WARPS * LM_ROWS * LM_RED + (size_t)LM_ROWS * W) + 2 * sizeof(__nv_bfloat16) * (size_t)LM_ROWS * lora_row_places(p.S, p.R);
    static Once once;
    if (once.first()) {
        cudaError_t err = cudaFuncSetAttribute(lora_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
        if (err == cudaSuccess) err = cudaFuncSetAttribute(lora_rows_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (err != cudaSuccess) return fail(-100, "lora_add: %s", cudaGetErrorString(err));
        once.done();
    }
    return launch("lora_add", lora_rows_kernel, dim3((unsigned)(tiles * C * copies)), dim3(LM_THREADS), smem, stream, dim3(C, 1, 1), p, copies);
}

}  // namespace fd
