// Low-rank adapters in bfloat16 for steps of many tokens per adapter (prompts): out[t] = y[t] + scale B (A x[t]).
//
// Such a step reads x and y and writes out, and does 2 r operations with every element of them, so it is bound by memory as long
// as the products keep up: at rank 64 they would take all that mma.sync has, which is why they are tcgen05.mma here.  A cluster of CTAs
// takes 128 tokens of one adapter:
//   1. D1 [128 x S r] = x A^T over the CTA's share of K.  Blocks of 64 columns of x (rows by the tokens' list, so they may lie
//      anywhere) and of A go to a ring of swizzled tiles by cp.async; one thread issues the MMAs; D1 is in tensor memory.
//   2. The cluster's partial sums are added in the order of the ranks: each CTA adds 128 / C tokens' and hands them to all,
//      as two bfloat16 numbers each (what rounding takes away from the first is the second: 2^-17 of A x is lost, not 2^-9).
//   3. D2 [128 x 128] = h B^T for the CTA's share of the columns.  y and B of the next tile are on their way while this one is
//      multiplied and stored.  A tile whose columns belong to several slices (gate and up) multiplies each slice's h with the rows
//      of B that are its own, the others zero.
// y comes to and out leaves from shared memory in rows, so that both move whole lines although a thread's D2 is one row.
#include <cooperative_groups.h>

#include <algorithm>

#include "lora.cuh"
#include "mma_utils.cuh"
#include "tcgen05.cuh"

namespace fd {

namespace cg = cooperative_groups;

constexpr int LT_ROWS = 128, LT_COLS = 128, LT_THREADS = 256;
constexpr int LT_X_BYTES = LT_ROWS * 128;        // a block of 64 columns of x: rows of 128 bytes
constexpr int LT_TILE = 128 * 128;               // a tile of 64 columns of 128 rows
constexpr int LT_Y_ROW = LT_COLS * 2 + 16;       // a row of y in shared memory; 16: neighbouring rows in other banks
constexpr int LT_Y_BYTES = LT_ROWS * LT_Y_ROW;
constexpr int LT_STAGES = 8;
constexpr int LT_SMEM = 222 * 1024;
constexpr int LT_MAX_W = 192;                    // columns of D1

struct LoraTilePlan {
    int chunks;              // 64-column tiles of a slice of h
    int stages;              // of the ring of step 1
    size_t smem;
};

static LoraTilePlan lora_tile_plan(const LoraArgs& p) {
    LoraTilePlan f;
    const int r16 = (p.R + 15) / 16 * 16, W = p.S * r16;
    f.chunks = (p.R + 63) / 64;
    const size_t stage = LT_X_BYTES + (size_t)W * 128;
    const size_t later = (size_t)p.S * f.chunks * LT_TILE * 3 + 2 * LT_Y_BYTES;          // hi, lo, B; y twice
    f.stages = (int)std::min<size_t>(LT_STAGES, (LT_SMEM - 1024) / stage);
    f.smem = 1024 + std::max(later, f.stages * stage);
    // the partial sums lie behind hi and lo
    const size_t sums = (size_t)p.S * f.chunks * LT_TILE * 2 + (size_t)LT_ROWS * (W + 4) * 4;
    f.smem = std::max(f.smem, 1024 + sums);
    if (W > LT_MAX_W || f.stages < 4 || f.smem > LT_SMEM) f.stages = 0;
    return f;
}

bool lora_tiles_take(const LoraArgs& p) { return lora_tile_plan(p).stages > 0; }

__device__ __forceinline__ uint32_t lt_swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

__global__ void __launch_bounds__(LT_THREADS, 1)
lora_tile_kernel(const LoraArgs p, const int chunks, const int stages, const unsigned long long wait_ns) {
    extern __shared__ unsigned char lt_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)lt_smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long bars[LT_STAGES + 1];      // the MMAs that read a stage are done; D2 (and, at first, D1) is
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ int tok[LT_ROWS];
    __shared__ LoraTile tile_s;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i <= LT_STAGES; ++i) mbar_init(s_addr(&bars[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        const LoraTile f = lora_tile(p, blockIdx.x / C, LT_ROWS);
        for (int i = lane; i < LT_ROWS; i += 32) {
            int t = i < f.count ? p.order[f.begin + i] : -1;
            if (i < f.count && (t < 0 || t >= p.T)) { set_status(p.status, STATUS_BAD_INDEX); t = -1; }
            tok[i] = t;
        }
        if (lane == 0) tile_s = f;
    }
    __syncthreads();
    const LoraTile tile = tile_s;
    if (tile.adapter == -2) return;                              // the same for the whole cluster
    const __nv_bfloat16* y = static_cast<const __nv_bfloat16*>(p.y);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    const int e = max(tile.adapter, 0), r = tile.adapter < 0 ? 0 : min(max(p.ranks[e], 0), p.R);
    if (r == 0) {                                                // nothing to add
        if (static_cast<const void*>(out) == p.y) return;
        for (int i = warp; i < tile.count; i += LT_THREADS / 32)
            if (tok[i] >= 0)
                for (int n = (rank * 32 + lane) * 8; n < p.N; n += C * 32 * 8)
                    *reinterpret_cast<uint4*>(out + (size_t)tok[i] * p.N + n) = *reinterpret_cast<const uint4*>(y + (size_t)tok[i] * p.N + n);
        return;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t d1 = tmem_slot, d2 = d1 + 256;
    const uint32_t base = s_addr(smem);
    const int r16 = (r + 15) / 16 * 16, W = p.S * r16;           // D1's columns: each slice's in whole MMAs
    const uint32_t done = s_addr(&bars[LT_STAGES]);

    // ---- 1. D1 = x A^T over this CTA's share of K ----
    const int blocks = (p.K + 63) / 64, bper = (blocks + C - 1) / C, b0 = rank * bper, nb = max(0, min(blocks, b0 + bper) - b0);
    const int stage_bytes = LT_X_BYTES + W * 128;
    {
        const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x);
        const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + (size_t)e * p.S * p.R * p.K;
        const int chunk = tid & 7, row0 = tid >> 3;              // a thread's 16 bytes of rows row0, row0 + 32, ...
        const __nv_bfloat16* xr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xr[i] = tok[row0 + 32 * i] >= 0 ? x + (size_t)tok[row0 + 32 * i] * p.K : nullptr;
        auto fetch = [&](int it) {
            const int k = (b0 + it) * 64 + chunk * 8;
            const bool in = k < p.K;                             // K is a multiple of 8
            const uint32_t s = base + (it % stages) * stage_bytes;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool there = in && xr[i] != nullptr;
                cp_async16(s + lt_swizzled(row0 + 32 * i, chunk), there ? xr[i] + k : x, there ? 16 : 0);
            }
            for (int u = row0; u < W; u += 32) {
                const int sl = u / r16, j = u - sl * r16;
                const bool there = in && j < p.R;
                cp_async16(s + LT_X_BYTES + lt_swizzled(u, chunk), there ? a + (size_t)(sl * p.R + j) * p.K + k : a, there ? 16 : 0);
            }
        };
        // two stages of slack: the one that is filled again was multiplied two blocks ago
        const int ahead = stages - 2;
        for (int it = 0; it < ahead; ++it) {
            if (it < nb) fetch(it);
            cp_async_commit();
        }
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(W >> 3) << 17) | ((uint32_t)(LT_ROWS >> 4) << 24);
        for (int it = 0; it < nb; ++it) {
            // blocks up to `it` have landed: the newest ahead - 1 groups may be under way
            switch (ahead) {
                case 2: cp_async_wait<1>(); break;
                case 3: cp_async_wait<2>(); break;
                case 4: cp_async_wait<3>(); break;
                case 5: cp_async_wait<4>(); break;
                default: cp_async_wait<5>(); break;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncthreads();
            if (tid == 0 && !abort_flag) {
                tc_fence_after();
                const uint32_t s = base + (it % stages) * stage_bytes;
                const uint64_t adesc = smem_desc_sw128(s), bdesc = smem_desc_sw128(s + LT_X_BYTES);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) tc_mma(d1, adesc + 2 * kk, bdesc + 2 * kk, idesc, (it | kk) != 0);
                tc_commit(s_addr(&bars[it % stages]));
                if (it == nb - 1) tc_commit(done);
            }
            const int next = it + ahead;
            if (next < nb) {
                if (it >= 2) mbar_wait(s_addr(&bars[(it - 2) % stages]), ((it - 2) / stages) & 1, &abort_flag, p.status, wait_ns);
                fetch(next);
            }
            cp_async_commit();
        }
        cp_async_wait<0>();
        if (nb > 0) mbar_wait(done, 0, &abort_flag, p.status, wait_ns);
    }
    uint32_t phase = nb > 0 ? 1 : 0;                             // of `done`
    tc_fence_after();
    __syncthreads();

    // ---- 2. the cluster's sums ----
    const int hbytes = p.S * chunks * LT_TILE;                   // hi, then lo, as tiles [slice][64 columns] of 128 rows
    const int quarter = warp & 3, half = warp >> 2;              // a warp reads lanes 32 quarter .. of tensor memory
    float* part = reinterpret_cast<float*>(smem + 2 * hbytes);   // [128][W + 4]
    {
        const int row = quarter * 32 + lane;
        for (int c0 = half * 16; c0 < W; c0 += 32) {
            uint32_t v[16];
            if (nb > 0) {
                tc_ld16(d1 + ((uint32_t)(quarter * 32) << 16) + c0, v);
                tc_wait_ld();
            }
            const int j0 = c0 % r16;                             // r16 is a multiple of 16: one slice
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = nb > 0 && j0 + i < r ? __uint_as_float(v[i]) : 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(part + row * (W + 4) + c0 + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        }
    }
    tc_fence_before();
    cluster.sync();
    {
        const int rows = LT_ROWS / C, per_row = W / 8;
        for (int i = tid; i < rows * per_row; i += LT_THREADS) {
            const int row = rank * rows + i / per_row, c = (i % per_row) * 8, sl = c / r16, j = c - sl * r16;
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = 0.f;
            for (int k = 0; k < C; ++k) {
                const float4* f = reinterpret_cast<const float4*>(cluster.map_shared_rank(part, k) + row * (W + 4) + c);
                const float4 f0 = f[0], f1 = f[1];
                v[0] += f0.x; v[1] += f0.y; v[2] += f0.z; v[3] += f0.w;
                v[4] += f1.x; v[5] += f1.y; v[6] += f1.z; v[7] += f1.w;
            }
            const uint4 hi = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            const uint4 lo = make_uint4(pack_bf16_rest(v[0], v[1]), pack_bf16_rest(v[2], v[3]), pack_bf16_rest(v[4], v[5]), pack_bf16_rest(v[6], v[7]));
            unsigned char* at = smem + (sl * chunks + j / 64) * LT_TILE + lt_swizzled(row, (j % 64) / 8);
            for (int k = 0; k < C; ++k) {
                unsigned char* to = cluster.map_shared_rank(at, k);
                *reinterpret_cast<uint4*>(to) = hi;
                *reinterpret_cast<uint4*>(to + hbytes) = lo;
            }
        }
    }
    asm volatile("fence.proxy.async;" ::: "memory");             // written by threads, read by the MMAs of any CTA
    cluster.sync();
    asm volatile("fence.proxy.async;" ::: "memory");

    // ---- 3. out = y + scale h B^T for this CTA's tiles of 128 columns ----
    const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.b) + (size_t)e * p.N * p.R;
    const float scale = p.scale[e];
    const int tiles = (p.N + LT_COLS - 1) / LT_COLS;
    const uint32_t bbuf = base + 2 * hbytes, ybuf = bbuf + hbytes;
    unsigned char* ymem = smem + 3 * hbytes;
    auto fetch_y = [&](int n0, int buf) {
        const int chunk = tid & 15, n = n0 + chunk * 8;
        if (n < p.N)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = (tid >> 4) + 16 * i;
                if (tok[row] >= 0) cp_async16(ybuf + buf * LT_Y_BYTES + row * LT_Y_ROW + chunk * 16, y + (size_t)tok[row] * p.N + n, 16);
            }
    };
    // the slices among the columns of a tile, as bits
    auto slices_of = [&](int n0) -> unsigned {
        if (p.col_slice == nullptr) return 1u;
        const int n = n0 + (lane & 15) * 8;
        return __reduce_or_sync(0xffffffffu, n < p.N ? 1u << min((int)__ldg(p.col_slice + n / 8), p.S - 1) : 0u);
    };
    auto fetch_b = [&](int n0, unsigned present) {
        const int per_row = r16 / 8, row = tid >> 1, n = n0 + row;                     // two threads share a row
        const int own = p.col_slice != nullptr && n < p.N ? min((int)__ldg(p.col_slice + n / 8), p.S - 1) : 0;
        for (int sl = 0; sl < p.S; ++sl) {
            if (!(present >> sl & 1)) continue;
            const uint32_t at = bbuf + sl * chunks * LT_TILE;
            for (int c = tid & 1; c < per_row; c += 2) {
                const bool there = n < p.N && own == sl && c * 8 < p.R;
                cp_async16(at + (c >> 3) * LT_TILE + lt_swizzled(row, c & 7), there ? b + (size_t)n * p.R + c * 8 : b, there ? 16 : 0);
            }
        }
    };
    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(LT_COLS >> 3) << 17) | ((uint32_t)(LT_ROWS >> 4) << 24);
    int buf = 0;
    unsigned present = 0;
    if (rank < tiles) {
        present = slices_of(rank * LT_COLS);
        fetch_y(rank * LT_COLS, 0);
        fetch_b(rank * LT_COLS, present);
    }
    cp_async_commit();
    for (int t = rank; t < tiles; t += C) {
        const int n0 = t * LT_COLS, n1 = (t + C) * LT_COLS;
        cp_async_wait<0>();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (tid == 0 && !abort_flag) {
            tc_fence_after();
            uint32_t more = 0;
            for (int sl = 0; sl < p.S; ++sl) {
                if (!(present >> sl & 1)) continue;
                for (int kk = 0; kk < r16 / 16; ++kk) {
                    const uint32_t at = (sl * chunks + (kk >> 2)) * LT_TILE;
                    const uint64_t bdesc = smem_desc_sw128(bbuf + at) + 2 * (kk & 3);
                    tc_mma(d2, smem_desc_sw128(base + at) + 2 * (kk & 3), bdesc, idesc, more);
                    more = 1;
                    tc_mma(d2, smem_desc_sw128(base + hbytes + at) + 2 * (kk & 3), bdesc, idesc, 1);
                }
            }
            tc_commit(done);
        }
        if (n1 < p.N) fetch_y(n1, buf ^ 1);
        const unsigned next = n1 < p.N ? slices_of(n1) : 0u;
        mbar_wait(done, phase & 1, &abort_flag, p.status, wait_ns);
        ++phase;
        tc_fence_after();
        if (n1 < p.N) fetch_b(n1, next);
        cp_async_commit();
        {
            unsigned char* yrow = ymem + buf * LT_Y_BYTES + (quarter * 32 + lane) * LT_Y_ROW + half * 128;
#pragma unroll
            for (int c0 = 0; c0 < 64; c0 += 32) {
                uint32_t v[32];
                __syncwarp();
                tc_ld32(d2 + ((uint32_t)(quarter * 32) << 16) + half * 64 + c0, v);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint4* q = reinterpret_cast<uint4*>(yrow + (c0 + i) * 2);
                    const uint4 a = *q;
                    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
                    uint4 o;
                    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[j] = pack_bf16(fmaf(scale, __uint_as_float(v[i + 2 * j]), __low2float(h[j])),
                                         fmaf(scale, __uint_as_float(v[i + 2 * j + 1]), __high2float(h[j])));
                    *q = o;
                }
            }
        }
        tc_fence_before();
        __syncthreads();
        {
            const int chunk = tid & 15, n = n0 + chunk * 8;
            if (n < p.N)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int row = (tid >> 4) + 16 * i;
                    if (tok[row] >= 0)
                        *reinterpret_cast<uint4*>(out + (size_t)tok[row] * p.N + n) =
                            *reinterpret_cast<const uint4*>(ymem + buf * LT_Y_BYTES + row * LT_Y_ROW + chunk * 16);
                }
        }
        present = next;
        buf ^= 1;
    }
    cp_async_wait<0>();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(d1), "r"(512) : "memory");
    }
}

int lora_tiles(const LoraArgs& p, int sms, cudaStream_t stream) {
    const LoraTilePlan f = lora_tile_plan(p);
    const long long tiles = lora_max_tiles(p, LT_ROWS);
    int C = 8;
    while (C > 1 && (tiles * C > sms || (p.K + 63) / 64 < C)) C /= 2;
    FD_REQUIRE(tiles * C < (1ll << 31), -2, "lora_add: %d tokens", p.T);
    static Once once;
    if (once.first()) {
        const cudaError_t err = cudaFuncSetAttribute(lora_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_SMEM);
        if (err != cudaSuccess) return fail(-100, "lora_add: %s", cudaGetErrorString(err));
        once.done();
    }
    return launch("lora_add", lora_tile_kernel, dim3((unsigned)(tiles * C)), dim3(LT_THREADS), f.smem, stream, dim3(C, 1, 1), p, f.chunks, f.stages,
                  g_tc_wait_ns);
}

}  // namespace fd
