// Low-rank adapters in bfloat16 for steps of few tokens per adapter (decode): out[t] = y[t] + scale B (A x[t]).
//
// Such a step reads the adapters' matrices and little else: 2 (S r K + r N) bytes per adapter in use, whatever the number of
// its tokens, so a tile of up to 16 tokens is bound by streaming them.  A cluster of CTAs takes a tile, as in lora.cu: a share of
// K each, the partial sums exchanged through distributed shared memory, then a share of N each, one launch.  What is different:
//   * the products are mma.sync m16n8k16 with the tokens as the 16 rows.  (tcgen05's 128 rows would be padding, and operands that
//     are used once need no trip through shared memory: weights go from global memory to the registers of the lanes that
//     multiply them.  A lane's 16 bytes are 8 neighbouring values of a row; which of the k places they take is free as long as the
//     other operand's values take the same.)
//   * the CTA's share of B is one piece of memory, of which L2 is asked for at the start, so that it arrives while A x is computed.
//   * the sums of A x are 32-bit.  B h takes h as two bfloat16 numbers (what rounding takes away from the first is the second),
//     which is 2^-17 of h apart from it and costs one more MMA on operands that are there already.
#include <cooperative_groups.h>

#include "lora.cuh"
#include "mma_utils.cuh"

namespace fd {

namespace cg = cooperative_groups;

constexpr int LM_THREADS = 256, LM_WARPS = LM_THREADS / 32;
constexpr int LM_ROWS = 16;              // tokens of a tile: the rows of an MMA
constexpr int LM_TILES = 8;              // tiles of 8 rows of A that a warp accumulates at once
constexpr int LM_RED = LM_TILES * 8 + 4; // floats of a token's row of a warp's sums (4: so that neighbouring rows are in other banks)

__device__ __forceinline__ uint4 ldg16(const __nv_bfloat16* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// x is read by every group of rows of A: it may stay in L1
__device__ __forceinline__ uint4 ldx16(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

__global__ void __launch_bounds__(LM_THREADS, 2)
lora_rows_kernel(const LoraArgs p) {
    extern __shared__ __align__(16) unsigned char lm_smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, q = lane & 3;                       // an MMA's row or column, and the lane's place along k
    const int W = p.S * p.R, WB = W + 8;                         // a token's A x; its row as bfloat16, 16 bytes apart from a multiple of 128
    float* red = reinterpret_cast<float*>(lm_smem);              // [LM_WARPS][LM_ROWS][LM_RED]
    float* part = red + LM_WARPS * LM_ROWS * LM_RED;             // [LM_ROWS][W] this CTA's sums
    __nv_bfloat16* hi = reinterpret_cast<__nv_bfloat16*>(part + LM_ROWS * W);          // [LM_ROWS][WB] the cluster's sums
    __nv_bfloat16* lo = hi + LM_ROWS * WB;                       // ... and what hi leaves of them
    __shared__ int tok[LM_ROWS];
    __shared__ LoraTile tile_s;
    if (warp == 0) {
        const LoraTile f = lora_tile(p, blockIdx.x / C, LM_ROWS);
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
    const int per = ((p.N + 31) / 32 + C - 1) / C * 32, n0 = rank * per, n1 = min(p.N, n0 + per);
    const bool in_place = static_cast<const void*>(out) == p.y;
    const int e = max(tile.adapter, 0), r = tile.adapter < 0 ? 0 : min(max(p.ranks[e], 0), p.R);
    if (r == 0) {                                                // nothing to add
        if (in_place) return;
        for (int i = 0; i < tile.count; ++i)
            if (tok[i] >= 0)
                for (int n = n0 + tid * 8; n < n1; n += LM_THREADS * 8)
                    *reinterpret_cast<uint4*>(out + (size_t)tok[i] * p.N + n) = *reinterpret_cast<const uint4*>(y + (size_t)tok[i] * p.N + n);
        return;
    }
    const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + (size_t)e * W * p.K;
    const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.b) + (size_t)e * p.N * p.R;
    const int r8 = (r + 7) / 8 * 8, tiles = r8 / 8;              // rows of A in tiles of 8, per slice
    // (an adapter of less than half the room's rank would have L2 fetch more that is not used than what is)
    if (tid == 0 && n0 < n1 && 2 * r8 >= p.R) {
        const __nv_bfloat16* f = b + (size_t)n0 * p.R;
        const unsigned bytes = (unsigned)(n1 - n0) * p.R * 2;
        for (unsigned o = 0; o < bytes; o += 65536) {
            const unsigned n = min(65536u, bytes - o);
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(reinterpret_cast<const unsigned char*>(f) + o), "r"(n) : "memory");
        }
    }

    // --- A x: this CTA's share of K, cut over its warps in chunks of 32
    const int kper = ((p.K + 31) / 32 + C - 1) / C * 32, k0 = rank * kper, k1 = min(p.K, k0 + kper);
    const int t0 = tok[g], t1 = tok[g + 8];
    const __nv_bfloat16* x0 = x + (size_t)max(t0, 0) * p.K;
    const __nv_bfloat16* x1 = x + (size_t)max(t1, 0) * p.K;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < LM_ROWS * W; i += LM_THREADS) part[i] = 0.f;
    for (int u0 = 0; u0 < p.S * tiles; u0 += LM_TILES) {
        float acc[LM_TILES][4];
        const __nv_bfloat16* rows[LM_TILES];
        const int nu = min(LM_TILES, p.S * tiles - u0);
#pragma unroll
        for (int i = 0; i < LM_TILES; ++i) {
            acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            const int u = u0 + min(i, nu - 1), s = u / tiles;
            rows[i] = a + (size_t)(s * p.R + (u - s * tiles) * 8 + g) * p.K;
        }
        for (int k = k0 + warp * 32 + q * 8; k - q * 8 < k1; k += LM_WARPS * 32) {
            const bool in = k < k1;                              // K is a multiple of 8: a lane's 8 values are all there or none
            uint4 w[LM_TILES];
#pragma unroll
            for (int i = 0; i < LM_TILES; ++i) w[i] = in && i < nu ? ldg16(rows[i] + k) : none;
            const uint4 xa = in && t0 >= 0 ? ldx16(x0 + k) : none, xb = in && t1 >= 0 ? ldx16(x1 + k) : none;
#pragma unroll
            for (int i = 0; i < LM_TILES; ++i)
                if (i < nu) {
                    mma_bf16(acc[i], xa.x, xb.x, xa.y, xb.y, w[i].x, w[i].y);
                    mma_bf16(acc[i], xa.z, xb.z, xa.w, xb.w, w[i].z, w[i].w);
                }
        }
        float* mine = red + warp * LM_ROWS * LM_RED;
#pragma unroll
        for (int i = 0; i < LM_TILES; ++i) {
            *reinterpret_cast<float2*>(mine + g * LM_RED + i * 8 + q * 2) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(mine + (g + 8) * LM_RED + i * 8 + q * 2) = make_float2(acc[i][2], acc[i][3]);
        }
        __syncthreads();
        for (int i = tid; i < LM_ROWS * nu * 8; i += LM_THREADS) {
            const int row = i / (nu * 8), c = i - row * nu * 8, u = u0 + c / 8, s = u / tiles, j = (u - s * tiles) * 8 + (c & 7);
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < LM_WARPS; ++w) v += red[(w * LM_ROWS + row) * LM_RED + c];
            part[row * W + s * p.R + j] = j < r ? v : 0.f;
        }
        __syncthreads();
    }
    // --- the cluster's sums: each CTA adds up a share of them, in the order of the ranks, and hands it to all
    cluster.sync();
    const int used = p.S * r8 * tile.count;                      // (place, token) pairs that matter
    for (int i = rank * LM_THREADS + tid; i < used; i += C * LM_THREADS) {
        const int row = i / (p.S * r8), c = i - row * p.S * r8, s = c / r8, at = s * p.R + (c - s * r8);
        float v = 0.f;
        for (int k = 0; k < C; ++k) v += *cluster.map_shared_rank(part + row * W + at, k);
        const __nv_bfloat16 h = __float2bfloat16_rn(v), l = __float2bfloat16_rn(v - __bfloat162float(h));
        for (int k = 0; k < C; ++k) {
            *cluster.map_shared_rank(hi + row * WB + at, k) = h;
            *cluster.map_shared_rank(lo + row * WB + at, k) = l;
        }
    }
    // rows of no token: their results go nowhere, but they are operands
    for (int i = tile.count * WB + tid; i < LM_ROWS * WB; i += LM_THREADS) hi[i] = lo[i] = __float2bfloat16_rn(0.f);
    cluster.sync();

    // --- B h: 32 columns per warp and pass, in tiles of 8
    const float scale = p.scale[e];
    const bool two = tile.count > 8;
    for (int base = n0 + warp * 32; base < n1; base += LM_WARPS * 32) {
        float acc[4][4];
        uint32_t y0[4], y1[4];
        int at[4];                                               // the tile's slice in h
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            const int n = base + i * 8;
            const bool in = n < n1;
            at[i] = in && p.col_slice != nullptr ? min((int)p.col_slice[n >> 3], p.S - 1) * p.R : 0;
            y0[i] = in && t0 >= 0 ? *reinterpret_cast<const uint32_t*>(y + (size_t)t0 * p.N + n + q * 2) : 0u;
            y1[i] = in && t1 >= 0 ? *reinterpret_cast<const uint32_t*>(y + (size_t)t1 * p.N + n + q * 2) : 0u;
        }
        for (int j = q * 8; j - q * 8 < r8; j += 64) {           // two chunks of 32 places at once
            uint4 w[2][4];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = base + i * 8 + g;
                    w[c][i] = j + c * 32 < r8 && n < n1 ? ldg16(b + (size_t)n * p.R + j + c * 32) : none;
                }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (j - q * 8 + c * 32 >= r8) break;
                const bool in = j + c * 32 < r8;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int o = at[i] + j + c * 32;
                    const uint4 h0 = in ? *reinterpret_cast<const uint4*>(hi + g * WB + o) : none;
                    const uint4 l0 = in ? *reinterpret_cast<const uint4*>(lo + g * WB + o) : none;
                    const uint4 h1 = in && two ? *reinterpret_cast<const uint4*>(hi + (g + 8) * WB + o) : none;
                    const uint4 l1 = in && two ? *reinterpret_cast<const uint4*>(lo + (g + 8) * WB + o) : none;
                    mma_bf16(acc[i], h0.x, h1.x, h0.y, h1.y, w[c][i].x, w[c][i].y);
                    mma_bf16(acc[i], h0.z, h1.z, h0.w, h1.w, w[c][i].z, w[c][i].w);
                    mma_bf16(acc[i], l0.x, l1.x, l0.y, l1.y, w[c][i].x, w[c][i].y);
                    mma_bf16(acc[i], l0.z, l1.z, l0.w, l1.w, w[c][i].z, w[c][i].w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = base + i * 8 + q * 2;
            if (base + i * 8 >= n1) continue;
            const __nv_bfloat162 a0 = *reinterpret_cast<const __nv_bfloat162*>(&y0[i]), a1 = *reinterpret_cast<const __nv_bfloat162*>(&y1[i]);
            if (t0 >= 0)
                *reinterpret_cast<uint32_t*>(out + (size_t)t0 * p.N + n) =
                    pack_bf16(__low2float(a0) + scale * acc[i][0], __high2float(a0) + scale * acc[i][1]);
            if (t1 >= 0)
                *reinterpret_cast<uint32_t*>(out + (size_t)t1 * p.N + n) =
                    pack_bf16(__low2float(a1) + scale * acc[i][2], __high2float(a1) + scale * acc[i][3]);
        }
    }
}

// Whether the tensor-core kernels take the sizes: 16-byte pieces of every row.
bool lora_mma_takes(const LoraArgs& p) {
    const unsigned long long all = (unsigned long long)p.x | (unsigned long long)p.a | (unsigned long long)p.b |
                                   (unsigned long long)p.y | (unsigned long long)p.out;
    return (all & 15) == 0 && p.K % 8 == 0 && p.N % 8 == 0 && p.R % 8 == 0;
}

int lora_rows(const LoraArgs& p, int sms, cudaStream_t stream) {
    const long long tiles = lora_max_tiles(p, LM_ROWS);
    const int most = p.K > p.N ? p.K : p.N;
    int C = 16;
    while (C > 1 && (tiles * C > 2 * sms || most < 64 * C)) C /= 2;
    FD_REQUIRE(tiles * C < (1ll << 31), -2, "lora_add: %d tokens", p.T);
    const int W = p.S * p.R;
    const size_t smem = sizeof(float) * (LM_WARPS * LM_ROWS * LM_RED + (size_t)LM_ROWS * W) + 2 * sizeof(__nv_bfloat16) * (size_t)LM_ROWS * (W + 8);
    cudaError_t err = cudaFuncSetAttribute(lora_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(lora_rows_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err != cudaSuccess) return fail(-100, "lora_add: %s", cudaGetErrorString(err));
    return launch("lora_add", lora_rows_kernel, dim3((unsigned)(tiles * C)), dim3(LM_THREADS), smem, stream, dim3(C, 1, 1), p);
}

}  // namespace fd
