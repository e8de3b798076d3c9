// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + scale B (A x[t]), each token with its adapter's
// matrices.  This is the form for every type and size; lora_mma.cu has the ones for bfloat16 on the tensor cores.
//
// One launch.  A cluster of CTAs takes a tile of up to 16 tokens of one adapter: each CTA multiplies its share of K (A x is a long
// sum for few values), the partial sums are added over the cluster out of shared memory in the order of the ranks, and each
// CTA expands its share of the N columns.  A x never leaves the chip and no second launch waits for the first.
// All sums are 32-bit; one rounding at the end.  The cuts of K depend on the sizes alone, so that no bit of a token's result
// depends on the other tokens of the step.
// What bounds it.  A few tokens: latency (24 tokens of 5 adapters, float32, 8960 x 1536, rank 16: 10.5 us; the bytes would take 0.5): launch
// and cluster start, one trip for the segments and one for the tokens, one pass over a CTA's share of A, the exchange, one pass over B.
// Many tokens: the FMAs and what they read from shared memory, since every tile of 16 reads its matrices anew (800 tokens, float32, three
// slices of rank 33, 464 x 5224: 64 us; the bytes would take 7).  bfloat16 comes here only with sizes that are no multiples of 8.
#include <cooperative_groups.h>

#include "lora.cuh"

extern "C" int fd_sm_count();

namespace fd {

namespace cg = cooperative_groups;

constexpr int LR_THREADS = 256, LR_WARPS = LR_THREADS / 32;
constexpr int LR_ROWS = 16;              // tokens of a tile
constexpr int LR_CHUNK = 1024;           // columns of x in shared memory at once
constexpr int LR_J = 4;                  // rows of A that a warp multiplies at once: each x out of shared memory is used four times

template <typename T> __device__ __forceinline__ void load4(const T* p, float v[4], bool whole, int n) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            const float4 q = *reinterpret_cast<const float4*>(p);
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
            const uint2 q = *reinterpret_cast<const uint2*>(p);
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
            v[0] = __low2float(h[0]); v[1] = __high2float(h[0]); v[2] = __low2float(h[1]); v[3] = __high2float(h[1]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? to_float(p[e]) : 0.f;
}

// Floats per token for a CTA's sums: every row of A, or the few of a small rank once for each of the warps that share them.
__host__ __device__ __forceinline__ int lora_sums(int S, int R) {
    const int all = (S * R + LR_J - 1) / LR_J * LR_J;
    return all < LR_J * LR_WARPS ? LR_J * LR_WARPS : all;
}

template <typename T>
__global__ void __launch_bounds__(LR_THREADS, 2)
lora_general_kernel(const LoraArgs p, int copies, int chunk) {
    extern __shared__ __align__(16) float lr_smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int Rp = (p.R + 3) & ~3, W = p.S * Rp;                 // a token's A x: S slices of Rp places
    float* xs = lr_smem;                                         // [LR_ROWS][chunk]
    float* part = xs + LR_ROWS * chunk;                       // [parts][LR_ROWS][U] this CTA's sums, of the rows of A that the adapter has
    float* h = part + LR_ROWS * lora_sums(p.S, p.R);             // [LR_ROWS][W] the cluster's
    __shared__ int tok[LR_ROWS];
    __shared__ LoraTile tile_s;
    if (warp == 0) {
        const LoraTile f = lora_tile(p, blockIdx.x / (C * copies), LR_ROWS);
        if (lane < LR_ROWS) {
            int t = lane < f.count ? p.order[f.begin + lane] : -1;
            if (lane < f.count && (t < 0 || t >= p.T)) { set_status(p.status, STATUS_BAD_INDEX); t = -1; }
            tok[lane] = t;
        }
        if (lane == 0) tile_s = f;
    }
    __syncthreads();
    const LoraTile tile = tile_s;
    if (tile.adapter == -2) return;                              // the same for the whole cluster
    // this CTA's columns of the output
    const int shares = C * copies, per = (((p.N + 7) / 8 + shares - 1) / shares) * 8, n0 = min(p.N, (int)(blockIdx.x % shares) * per), n1 = min(p.N, n0 + per);
    const T* y = static_cast<const T*>(p.y);
    T* out = static_cast<T*>(p.out);
    const int e = max(tile.adapter, 0), r = tile.adapter < 0 ? 0 : min(max(p.ranks[e], 0), p.R);
    if (r == 0) {                                                // nothing to add
        if (static_cast<const void*>(out) == p.y) return;
        constexpr int per16 = 16 / (int)sizeof(T);               // n0 and n1 are multiples of 8, or N
        if (p.N % per16 == 0 && ((reinterpret_cast<unsigned long long>(p.y) | reinterpret_cast<unsigned long long>(p.out)) & 15) == 0)
            lora_copy<uint4>(tok, tile.count, p.y, p.out, p.N / per16, n0 / per16, n1 / per16, tid, LR_THREADS);
        else
            lora_copy<T>(tok, tile.count, p.y, p.out, p.N, n0, n1, tid, LR_THREADS);
        return;
    }
    const T* x = static_cast<const T*>(p.x);
    const T* a = static_cast<const T*>(p.a) + (size_t)e * p.S * p.R * p.K;
    // Groups of LR_J rows of A for the warps; those that are left over share a group's columns.  (By the adapter's rank and the sizes.)
    const int kper = (((p.K + 3) / 4 + C - 1) / C) * 4, k0 = rank * kper, k1 = min(p.K, k0 + kper);
    const int U = (p.S * r + LR_J - 1) / LR_J * LR_J, groups = U / LR_J;
    const int parts = max(1, min(LR_WARPS / max(groups, 1), (kper + 127) / 128));
    for (int i = tid; i < parts * LR_ROWS * U; i += LR_THREADS) part[i] = 0.f;

    // --- A x over this CTA's share of K
    constexpr unsigned long long unit = 4 * sizeof(T) - 1;       // rows that begin where four values can be loaded at once
    const bool whole4 = (p.K & 3) == 0 && ((reinterpret_cast<unsigned long long>(p.x) | reinterpret_cast<unsigned long long>(p.a)) & unit) == 0;
    for (int c0 = k0; c0 < k1; c0 += chunk) {
        const int w = min(chunk, k1 - c0), w4 = (w + 3) / 4;
        __syncthreads();
        for (int i = tid; i < LR_ROWS * w4; i += LR_THREADS) {
            const int row = i / w4, c = (i - row * w4) * 4;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (tok[row] >= 0) load4(x + (size_t)tok[row] * p.K + c0 + c, v, whole4, w - c);
            *reinterpret_cast<float4*>(xs + row * chunk + c) = make_float4(v[0], v[1], v[2], v[3]);
        }
        __syncthreads();
        for (int gi = warp; gi < groups * parts; gi += LR_WARPS) {
            const int u0 = gi / parts * LR_J, mine = gi % parts;
            float acc[LR_J * LR_ROWS];
#pragma unroll
            for (int i = 0; i < LR_J * LR_ROWS; ++i) acc[i] = 0.f;
            const T* rows[LR_J];
#pragma unroll
            for (int j = 0; j < LR_J; ++j) {
                const int u = min(u0 + j, p.S * r - 1), s = u / r;
                rows[j] = a + (size_t)(s * p.R + (u - s * r)) * p.K + c0;
            }
            for (int c = mine * 128 + lane * 4; c < w; c += parts * 128) {
                float av[LR_J][4];
#pragma unroll
                for (int j = 0; j < LR_J; ++j) load4(rows[j] + c, av[j], whole4, w - c);
#pragma unroll
                for (int i = 0; i < LR_ROWS; ++i) {
                    const float4 xv = *reinterpret_cast<const float4*>(xs + i * chunk + c);
#pragma unroll
                    for (int j = 0; j < LR_J; ++j)
                        acc[j * LR_ROWS + i] += av[j][0] * xv.x + av[j][1] * xv.y + av[j][2] * xv.z + av[j][3] * xv.w;
                }
            }
            // 64 sums over the lanes: halves are exchanged, so that after five steps each lane has two of them
            int first = 0;
#pragma unroll
            for (int o = 16, n = LR_J * LR_ROWS / 2; o >= 1; o >>= 1, n >>= 1) {
                const bool up = (lane & o) != 0;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const float give = up ? acc[i] : acc[i + n], keep = up ? acc[i + n] : acc[i];
                    acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
                first += up ? n : 0;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = (first + i) / LR_ROWS, row = (first + i) % LR_ROWS;
                part[(mine * LR_ROWS + row) * U + u0 + j] += acc[i];               // (rows behind the rank: the last one's once more)
            }
        }
    }
    if (parts > 1) {
        __syncthreads();
        for (int i = tid; i < LR_ROWS * U; i += LR_THREADS) {
            float v = part[i];
            for (int q = 1; q < parts; ++q) v += part[q * LR_ROWS * U + i];
            part[i] = v;
        }
    }
    cluster.sync();
    for (int i = tid; i < LR_ROWS * W; i += LR_THREADS) {
        const int row = i / W, pl = i - row * W, s = pl / Rp, j = pl - s * Rp;
        float v = 0.f;
        if (j < r && row < tile.count) {
            const float* f = part + row * U + s * r + j;
            if (C == 16) {                                       // all in flight at once
#pragma unroll
                for (int c = 0; c < 16; ++c) v += *cluster.map_shared_rank(f, c);
            } else {
#pragma unroll 4
                for (int c = 0; c < C; ++c) v += *cluster.map_shared_rank(f, c);
            }
        }
        h[i] = v;
    }
    cluster.sync();                                              // the others' sums have been read, and h is whole

    // --- B h over this CTA's columns
    const T* b = static_cast<const T*>(p.b) + (size_t)e * p.N * p.R;
    const float scale = p.scale[e];
    const bool vec = (p.R & 3) == 0 && (reinterpret_cast<unsigned long long>(p.b) & unit) == 0;
    for (int n = n0 + tid; n < n1; n += LR_THREADS) {
        const int s = p.col_slice != nullptr ? min((int)p.col_slice[n >> 3], p.S - 1) : 0;
        const T* bn = b + (size_t)n * p.R;
        const float* hs = h + s * Rp;
        // (all of y before the first store: out may be y, and each load would wait for the store before it)
        float acc[LR_ROWS], yv[LR_ROWS];
#pragma unroll
        for (int i = 0; i < LR_ROWS; ++i) {
            acc[i] = 0.f;
            yv[i] = tok[i] >= 0 ? to_float(y[(size_t)tok[i] * p.N + n]) : 0.f;
        }
        for (int j = 0; j < r; j += 4) {
            float bv[4];
            load4(bn + j, bv, vec, r - j);
#pragma unroll
            for (int i = 0; i < LR_ROWS; ++i) {
                const float4 hv = *reinterpret_cast<const float4*>(hs + i * W + j);
                acc[i] += bv[0] * hv.x + bv[1] * hv.y + bv[2] * hv.z + bv[3] * hv.w;
            }
        }
#pragma unroll
        for (int i = 0; i < LR_ROWS; ++i)
            if (tok[i] >= 0) out[(size_t)tok[i] * p.N + n] = from_float<T>(yv[i] + scale * acc[i]);
    }
}

// CTAs of a cluster: enough to spread one tile's matrices, by the sizes alone (so a float32 token's bits are the same in any step).  Measured,
// float32, clusters of 16 / 8 / 4, us: q/k/v of 1536 x 2048, rank 16: 1 token 9.2 / 10.8 / 12.1, 16 of 16 adapters 19.5 / 13.1 / 12.6, 2,500
// of 4 180 / 90 / 66; 8960 x 1536 (here 16): 1 token 10.2, 32 of 32 34; 3584 x 3584, rank 32: 1 token 10.4 / 15.0 / 16.8, 500 of 4
// 46 / 24 / 30, 2,500 203 / 133 / 120.
static int lora_cluster(const LoraArgs& p) {
    const int most = p.K > p.N ? p.K : p.N;
    return p.K >= 4096 ? 16 : (most >= 1024 ? 8 : (most >= 512 ? 4 : (most >= 256 ? 2 : 1)));
}

template <typename T>
static int launch_general(const LoraArgs& p, cudaStream_t stream) {
    const int C = lora_cluster(p), W = p.S * ((p.R + 3) & ~3);
    const int kper = (((p.K + 3) / 4 + C - 1) / C) * 4, chunk = kper < LR_CHUNK ? kper : LR_CHUNK;
    const size_t smem = sizeof(float) * LR_ROWS * (chunk + (size_t)W + lora_sums(p.S, p.R));
    const long long tiles = lora_max_tiles(p, LR_ROWS);
    // where the tiles leave SMs idle, several clusters share a tile's columns (each computes the same A x)
    int copies = (int)(lora_room(C, fd_sm_count()) / lora_likely_tiles(p));
    while (copies > 1 && p.N < LR_THREADS * C * copies) --copies;
    if (copies < 1) copies = 1;
    FD_REQUIRE(tiles * C * copies < (1ll << 31), -2, "lora_add: %d tokens", p.T);
    static Once once;
    if (once.first()) {
        cudaError_t err = cudaFuncSetAttribute(lora_general_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (err == cudaSuccess) err = cudaFuncSetAttribute(lora_general_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (err != cudaSuccess) return fail(-100, "lora_add: %s", cudaGetErrorString(err));
        once.done();
    }
    return launch("lora_add", lora_general_kernel<T>, dim3((unsigned)(tiles * C * copies)), dim3(LR_THREADS), smem, stream, dim3(C, 1, 1), p, copies, chunk);
}

}  // namespace fd

using namespace fd;

// Tiles of 128 are taken for segments of so many tokens on average (the adapters' tokens are known on the device only)
//   * from LORA_TILE_TOKENS tokens on, where tiles of 16 would read LORA_TILE_BYTES of A and B (out of L2, most of them),
//   * from LORA_TILE_FEW on, where they would read LORA_TILE_FEW_BYTES, if a tile gets a cluster of 8 or the slices' ranks add up to
//     LORA_TILE_WIDE: between 16 and 20 tiles clusters of 4 leave half of the GPU idle, and tiles of 16 lose only if they multiply much.
// Measured, tiles of 16 / of 128, us:
//   3584 x 3584, rank 32: 1,024 tokens 13 / 19, 1,900 22 / 24, 2,048 22 / 29, 2,800 35 / 30, 4,096 36 / 31, 16,384 132 / 81
//   2048 x 2560 in three slices, rank 16: 1,500 18 / 19, 2,048 20 / 23, 2,800 32 / 26, 16,384 121 / 62
//   592 x 768 in two slices, rank 8: 2,800 12 / 15, 4,096 (8 MB) 12 / 16, 5,500 (11 MB) 19 / 18, 16,384 46 / 29
//   4096 x 6144 in three slices, rank 16: 1,024 22 / 26, 1,500 (75 MB) 36 / 28, 2,048 37 / 39, 2,800 60 / 40
//   3584 x 37888 in two slices, rank 16: 1,024 60 / 76, 1,500 106 / 77, 2,048 111 / 136; rank 64: 1,024 87 / 94, 1,500 155 / 96, 2,048 160 / 160
//   13824 x 5120, rank 64: 512 23 / 32, 1,024 39 / 34, 2,048 66 / 52, 16,384 469 / 166
constexpr int LORA_TILE_SEGMENT = 64, LORA_TILE_TOKENS = 2600, LORA_TILE_FEW = 1200, LORA_TILE_WIDE = 64;
constexpr long long LORA_TILE_BYTES = 10000000, LORA_TILE_FEW_BYTES = 64000000;
static bool lora_many(const LoraArgs& p) {
    const long long bytes = (long long)(p.T / 16) * 2 * p.R * ((long long)p.S * p.K + p.N);
    if (p.T / p.n_seg < LORA_TILE_SEGMENT) return false;
    if (p.T >= LORA_TILE_TOKENS) return bytes >= LORA_TILE_BYTES;
    return p.T >= LORA_TILE_FEW && bytes >= LORA_TILE_FEW_BYTES && (p.S * p.R >= LORA_TILE_WIDE || lora_tile_cluster(p, fd_sm_count()) == 8);
}

static int g_lora_form = 0;
// Which form the bfloat16 steps on the tensor cores take from now on: 1 = tiles of 16 tokens, 2 = tiles of 128 where they take the
// sizes, 0 = by the sizes.  For tests and measurements.
extern "C" int fd_lora_set_form(int form) {
    g_lora_form = form;
    return 0;
}

extern "C" int fd_lora_add(const void* x, const void* a, const void* b, const float* scale, const int* ranks, const int* order,
                           const int* start, const int* ids, const void* y, void* out, const unsigned char* col_slice, int dtype,
                           int T, int K, int N, int E, int R, int S, int n_seg, int* status, cudaStream_t stream) {
    if (T == 0 || N == 0 || n_seg == 0) return 0;
    FD_REQUIRE(T > 0 && K > 0 && N > 0 && E > 0 && R > 0 && n_seg > 0, -2,
               "lora_add: %d tokens, %d x %d, %d adapters of rank %d, %d segments", T, K, N, E, R, n_seg);
    FD_REQUIRE(K < (1 << 27) && N < (1 << 27), -2, "lora_add: %d x %d; up to 2^27 columns are taken", K, N);
    FD_REQUIRE(S >= 1 && S <= 4, -2, "lora_add: %d packed projections; 1 to 4 are taken", S);
    FD_REQUIRE(R <= 256 && S * R <= 512, -2, "lora_add: rank %d of %d packed projections; up to 256, and 512 in all, are taken", R, S);
    FD_REQUIRE(S == 1 || (col_slice != nullptr && N % 8 == 0), -2, "lora_add: %d packed projections need col_slice and N a multiple of 8", S);
    const LoraArgs p{x, a, b, scale, ranks, order, start, ids, y, out, col_slice, status, T, K, N, E, R, S, n_seg};
    if (dtype == 0) return launch_general<float>(p, stream);
    if (!lora_mma_takes(p)) return launch_general<__nv_bfloat16>(p, stream);
    const bool many = g_lora_form == 0 ? lora_many(p) : g_lora_form == 2;
    return many && lora_tiles_take(p) ? lora_tiles(p, fd_sm_count(), stream) : lora_rows(p, fd_sm_count(), stream);
}
