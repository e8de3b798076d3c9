// Low-rank adapters in bfloat16 for steps of many tokens per adapter (prompts): out[t] = y[t] + scale B (A x[t]).
//
// Such a step reads x and y and writes out, and does 2 r operations with every element of them, so it is bound by memory as long
// as the products keep up: at rank 64 they would take all that mma.sync has, which is why they are tcgen05.mma here.  A cluster of CTAs
// takes 128 tokens of one adapter:
//   1. D1 [128 x S r] = x A^T over the CTA's share of K, in tensor memory: one 32-bit sum over all of it (one output in 240 is a bfloat16
//      step from that of shorter sums, one in 390 with tiles of 16).  Blocks of 64 columns of x and A go through a ring of swizzled tiles.
//   2. The cluster's partial sums are added in the order of the ranks: each CTA adds 128 / C tokens' and hands them to all,
//      as two bfloat16 numbers each (what rounding takes away from the first is the second: 2^-17 of A x is lost, not 2^-9).
//   3. D2 [128 x 128] = h B^T for the CTA's share of the columns, a product for every slice that has columns in the tile (gate and up
//      both); the epilogue takes each column from its own.  The tiles' y and B are a stage or two ahead.
// One warp asks for copies, one thread issues MMAs, eight warps do the rest.  out takes y's place in shared memory, so that it leaves in
// whole lines although a thread's share of D2 is a row.
//
// A wait that runs out before step 2 stops the whole cluster: its sums lack a part, and nothing is stored.  One in step 3 stops its own
// CTA, whose tiles from there on stay as they were.  Copies and MMAs in flight end before their memory is used again or given up.
//
// Measured: four prompts of 1,900 to 2,048 tokens, 13824 x 5120, rank 64 (390 MB, floor 59.7 us): 92 us, 4.2 TB/s - finding the tile 3, step 1 47
// (an SM takes 57 GB/s, a third of it A, which every tile reads anew out of L2), step 2 5, step 3 32 (5.1 TB/s of y and out).  The two
// streams follow one another, the exchange stands between them, and 65 tiles in clusters of 2 leave 18 SMs idle.  Tensor pipe 11 %.
#include <cooperative_groups.h>

#include <algorithm>

#include "lora.cuh"
#include "mma_utils.cuh"
#include "tcgen05.cuh"

namespace fd {

namespace cg = cooperative_groups;

constexpr int LT_ROWS = 128, LT_COLS = 128;
constexpr int LT_EPI = 8, LT_THREADS = (2 + LT_EPI) * 32;
constexpr int LT_TILE = 128 * 128;               // bytes of a tile of 64 columns of 128 rows
constexpr int LT_Y_BYTES = 2 * LT_TILE;          // y's tile of 128 columns: two of those
constexpr int LT_RING = 8, LT_OUT_RING = 3;      // most stages of step 1 and of step 3
constexpr int LT_SMEM = 225 * 1024;
// Clusters with an SM for each CTA that run at once; they have to lie within one of the GPU's groups of 16 to 18 SMs.  One more takes a second
// wave: 13824 x 5120, rank 64, 15 tiles 36 us and 16 65 (in clusters of 4: 52), 33 tiles 56 us and 34 99 (in clusters of 2: 88).
constexpr int LT_ROOM8 = 15, LT_ROOM4 = 33;
constexpr int LT_MAX_W = 192;                    // columns of D1

struct LoraTilePlan {
    int chunks;              // 64-column tiles of a slice of h
    int stages, out_stages;  // of the rings of steps 1 and 3
    size_t smem;
};

static LoraTilePlan lora_tile_plan(const LoraArgs& p) {
    LoraTilePlan f;
    const int W = p.S * ((p.R + 15) / 16 * 16);
    f.chunks = (p.R + 63) / 64;
    const size_t room = LT_SMEM - 1024, h = 2 * (size_t)p.S * f.chunks * LT_TILE;         // h: both numbers
    const size_t stage = LT_TILE + (size_t)W * 128, out_stage = LT_Y_BYTES + (size_t)f.chunks * LT_TILE;
    const size_t sums = h + (size_t)LT_ROWS * (W + 4) * 4;                                  // step 2's sums lie behind h
    f.stages = (int)std::min<size_t>(LT_RING, room / stage);
    f.out_stages = h < room ? (int)std::min<size_t>(LT_OUT_RING, (room - h) / out_stage) : 0;
    f.smem = 1024 + std::max(std::max(f.stages * stage, h + f.out_stages * out_stage), sums);
    if (W > LT_MAX_W || f.stages < 3 || f.out_stages < 2 || f.smem > LT_SMEM) f.stages = 0;
    return f;
}

// (a copy's row of a or b is a 32-bit number)
bool lora_tiles_take(const LoraArgs& p) {
    return (long long)p.E * p.N < (1ll << 31) && (long long)p.E * p.S * p.R < (1ll << 31) && lora_tile_plan(p).stages > 0;
}

// CTAs of a tile, by the tiles that there should be: T / 128, and a part of one for each segment's last.  One tile too many for a wave costs
// some 15 to 20 % over clusters of half the size (34 tiles of 3584 x 3584, rank 32: 54 us, 45 in clusters of 2), clusters of half the size
// where there was room cost 45 to 75 % (32 tiles: 45 us, 31 in clusters of 4), so a quarter of a tile is counted, not the half that
// segments of any length leave empty.
int lora_tile_cluster(const LoraArgs& p, int sms) {
    const long long likely = std::min(lora_max_tiles(p, LT_ROWS), std::max<long long>((p.T + LT_ROWS - 1) / LT_ROWS, p.T / LT_ROWS + p.n_seg / 4));
    int C = 8;
    while (C > 1 && (likely > (C == 8 ? LT_ROOM8 : (C == 4 ? LT_ROOM4 : sms / C)) || (p.K + 63) / 64 < C)) C /= 2;
    return C;
}

__device__ __forceinline__ uint32_t lt_swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// four rows of a map with boxes of one row
__device__ __forceinline__ void lt_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int r0, int r1, int r2, int r3) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(col), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
__device__ __forceinline__ void lt_ld8(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}

// A barrier of the epilogue's warps: whether all of them are well.
__device__ __forceinline__ bool lt_all_epi(bool ok) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((uint32_t)ok), "n"(LT_EPI * 32) : "memory");
    return all != 0;
}

// x and y in boxes of 128 rows, of 16, and of one (for gathers).
struct LoraMaps {
    CUtensorMap x[3], y[3], a, b;
};

// The rows of a tile's tokens: neighbours all of them (a prompt's tokens are), or 16 by 16, or gathered four by four: 32 copies of 512 bytes
// for a tile's 64 columns instead of one of 16 KB, at some 85 cycles of the asking warp each.
struct LoraRows {
    bool all;
    int first;               // of the tile
    int group;               // lanes 0 .. 7: the first of 16 neighbours, or -1
    int rows[4];             // this lane's four of the tile
    // rows of no token read others', and what comes of them is not stored
    __device__ __forceinline__ explicit LoraRows(const int* tok, int count) {
        const int lane = threadIdx.x & 31;
        first = max(tok[0], 0);
        bool row = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = tok[lane * 4 + i];
            rows[i] = max(t, 0);
            row = row && (lane * 4 + i >= count || t == tok[0] + lane * 4 + i);
        }
        all = __all_sync(0xffffffffu, row && tok[0] >= 0);
        const int g = (lane & 7) * 16;
        group = max(tok[g], 0);
        for (int i = 1; i < 16; ++i)
            if (g + i < count && tok[g + i] != group + i) group = -1;
        if (tok[g] < 0 && g < count) group = -1;
    }
    // the 64 columns from col on of all rows, to the tile at dst; called by a whole warp
    __device__ __forceinline__ void ask(uint32_t dst, const CUtensorMap* maps, uint32_t bar, int col) const {
        const int lane = threadIdx.x & 31;
        if (all) {
            if (lane == 0) tma_load_2d(dst, maps, bar, col, first);
            return;
        }
        if (lane < 8 && group >= 0) tma_load_2d(dst + lane * 2048, maps + 1, bar, col, group);
        if (__shfl_sync(0xffffffffu, group, lane >> 2) < 0) lt_gather4(dst + lane * 512, maps + 2, bar, col, rows[0], rows[1], rows[2], rows[3]);
    }
};

__global__ void __launch_bounds__(LT_THREADS, 1)
lora_tile_kernel(const __grid_constant__ LoraMaps maps, const LoraArgs p, const int chunks, const int stages, const int out_stages,
                 const unsigned long long wait_ns, const int skip_last) {
    extern __shared__ unsigned char lt_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)lt_smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[LT_RING], empty[LT_RING], out_full[LT_OUT_RING], out_empty[LT_OUT_RING], acc_full[2],
        acc_empty[2], d1_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ int tok[LT_ROWS];
    __shared__ LoraTile tile_s;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < LT_RING; ++i) {
            mbar_init(s_addr(&full[i]), 1);
            mbar_init(s_addr(&empty[i]), 1);
        }
        for (int i = 0; i < LT_OUT_RING; ++i) {
            mbar_init(s_addr(&out_full[i]), 1);
            mbar_init(s_addr(&out_empty[i]), LT_EPI);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_addr(&acc_full[i]), 1);
            mbar_init(s_addr(&acc_empty[i]), LT_EPI);
        }
        mbar_init(s_addr(&d1_full), 1);
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
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    const int e = max(tile.adapter, 0), r = tile.adapter < 0 ? 0 : min(max(p.ranks[e], 0), p.R);
    if (r == 0) {                                                // nothing to add
        if (static_cast<const void*>(out) == p.y) return;
        const int per = (p.N / 8 + C - 1) / C, u0 = min(p.N / 8, rank * per);
        lora_copy<uint4>(tok, tile.count, p.y, p.out, p.N / 8, u0, min(p.N / 8, u0 + per), tid, LT_THREADS);
        return;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, base = s_addr(smem);
    // D1's columns: R of each slice, in whole MMAs.  (Those behind an adapter's rank are dropped: a slice's rows of A come in one copy,
    // whose size is the same for every adapter, and it is copies that cost, some 85 cycles of the asking warp each.)
    const int r16 = (p.R + 15) / 16 * 16, W = p.S * r16;
    const int hbytes = p.S * chunks * LT_TILE;                   // hi, then lo, as tiles [slice][64 columns] of 128 rows
    const int blocks = (p.K + 63) / 64, bper = (blocks + C - 1) / C, b0 = rank * bper, nb = max(0, min(blocks, b0 + bper) - b0);
    const int stage_bytes = LT_TILE + W * 128, out_stage_bytes = LT_Y_BYTES + chunks * LT_TILE;
    const int tiles = (p.N + LT_COLS - 1) / LT_COLS;
    const int accs = p.S <= 2 ? 2 : 1;                           // accumulators of step 3: S x 128 of the 512 columns each

    // ---- 1. D1 = x A^T over this CTA's share of K ----
    const LoraRows rows(tok, tile.count);
    int asked = 0;                                               // blocks, then tiles, that warp 0 has asked for
    if (warp == 0) {
        for (int it = 0; it < nb; ++it) {
            const int s = it % stages, k = (b0 + it) * 64;
            if (it >= stages && !__all_sync(0xffffffffu, mbar_wait(s_addr(&empty[s]), (it / stages - 1) & 1, &abort_flag, p.status, wait_ns))) break;
            const uint32_t bar = s_addr(&full[s]), at = base + s * stage_bytes;
            if (lane == 0) mbar_expect_tx(bar, stage_bytes);
            __syncwarp();
            if (rows.all && lane == 0) tma_load_2d(at, maps.x, bar, k, rows.first);
            // (tests: a cluster's first CTA leaves out one copy of its last block)
            if (lane < p.S && !(skip_last == 1 && rank == 0 && it == nb - 1 && lane == 0))
                tma_load_2d(at + LT_TILE + lane * r16 * 128, &maps.a, bar, k, (e * p.S + lane) * p.R);
            ++asked;
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(W >> 3) << 17) | ((uint32_t)(LT_ROWS >> 4) << 24);
        for (int it = 0; it < nb; ++it) {
            const int s = it % stages;
            if (!mbar_wait(s_addr(&full[s]), (it / stages) & 1, &abort_flag, p.status, wait_ns)) break;
            tc_fence_after();
            const uint64_t adesc = smem_desc_sw128(base + s * stage_bytes), bdesc = smem_desc_sw128(base + s * stage_bytes + LT_TILE);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) tc_mma(tmem, adesc + 2 * kk, bdesc + 2 * kk, idesc, (it | kk) != 0);
            tc_commit(s_addr(&empty[s]));
        }
        tc_commit(s_addr(&d1_full));
    }
    else if (warp >= 2 && !rows.all) {
        // rows that lie here and there take many copies: eight warps ask for 16 rows each
        const int g = warp - 2, first = __shfl_sync(0xffffffffu, rows.group, g);
        for (int it = 0; it < nb; ++it) {
            const int s = it % stages, k = (b0 + it) * 64;
            if (it >= stages && !__all_sync(0xffffffffu, mbar_wait(s_addr(&empty[s]), (it / stages - 1) & 1, &abort_flag, p.status, wait_ns))) break;
            const uint32_t bar = s_addr(&full[s]), at = base + s * stage_bytes;
            if (first >= 0) {
                if (lane == 0) tma_load_2d(at + g * 2048, maps.x + 1, bar, k, first);
            } else if (lane >> 2 == g) {
                lt_gather4(at + lane * 512, maps.x + 2, bar, k, rows.rows[0], rows.rows[1], rows.rows[2], rows.rows[3]);
            }
            __syncwarp();
        }
    }
    __syncwarp();

    // ---- 2. the cluster's sums ----
    const int quarter = warp & 3, half = (warp - 2) >> 2, et = tid - 64;         // of the epilogue warps: the lanes of tensor memory, the columns
    float* part = reinterpret_cast<float*>(smem + 2 * hbytes);   // [128][W + 4]
    volatile int* const gave_up = &abort_flag;
    if (warp >= 2) mbar_wait(s_addr(&d1_full), 0, &abort_flag, p.status, wait_ns);
    __syncthreads();
    // Every MMA of step 1 has ended then, and if no wait ran out every copy: the ring's memory is free.  Else the copies are waited for:
    // those that warp 0 has asked for, and, where others ask too, what they may have asked for beyond (which nobody completes).
    if (*gave_up) {
        if (warp == 0) {
            int here = 0;
            for (int it = max(0, asked - stages); it < min(nb, asked + (rows.all ? 0 : 1)); ++it)
                mbar_wait(s_addr(&full[it % stages]), (it / stages) & 1, &here, nullptr, wait_ns);
        }
        __syncthreads();
    }
    if (warp >= 2) {
        const bool ok = !*gave_up && nb > 0;
        tc_fence_after();
        const int row = quarter * 32 + lane;
        for (int c0 = half * 16; c0 < W; c0 += 32) {
            uint32_t v[16];
            if (ok) {
                tc_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c0, v);
                tc_wait_ld();
            }
            const int j0 = c0 % r16;                             // r16 is a multiple of 16: one slice
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = ok && j0 + i < r ? __uint_as_float(v[i]) : 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(part + row * (W + 4) + c0 + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        }
        tc_fence_before();
    }
    __syncwarp();
    cluster.sync();
    const int lacks = lane < C ? *cluster.map_shared_rank(&abort_flag, lane) : 0;          // (nobody waits with it until the next barrier)
    {
        const int share = LT_ROWS / C, per_row = W / 8;
        for (int i = tid; i < share * per_row; i += LT_THREADS) {
            const int row = rank * share + i / per_row, c = (i % per_row) * 8, sl = c / r16, j = c - sl * r16;
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
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = lora_rest(v[q]);
            const uint4 lo = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            unsigned char* at = smem + (sl * chunks + j / 64) * LT_TILE + lt_swizzled(row, (j % 64) / 8);
            for (int k = 0; k < C; ++k) {
                unsigned char* to = cluster.map_shared_rank(at, k);
                *reinterpret_cast<uint4*>(to) = hi;
                *reinterpret_cast<uint4*>(to + hbytes) = lo;
            }
        }
    }
    asm volatile("fence.proxy.async;" ::: "memory");             // written by threads, read by the MMAs of any CTA; and part's memory takes copies
    const int end = __any_sync(0xffffffffu, lacks) ? 0 : tiles;  // a sum that lacks a part: no tile is computed
    cluster.sync();
    asm volatile("fence.proxy.async;" ::: "memory");

    // ---- 3. out = y + scale h B^T for this CTA's tiles of 128 columns ----
    const uint32_t ring = base + 2 * hbytes;                     // stages: y, then B
    asked = 0;
    int issued = 0;                                              // tiles whose MMAs warp 1 has issued
    if (warp == 0) {
        int i = 0;
        for (int t = rank; t < end; t += C, ++i) {
            const int s = i % out_stages, n0 = t * LT_COLS;
            if (i >= out_stages && !__all_sync(0xffffffffu, mbar_wait(s_addr(&out_empty[s]), (i / out_stages - 1) & 1, &abort_flag, p.status, wait_ns))) break;
            const uint32_t bar = s_addr(&out_full[s]), at = ring + s * out_stage_bytes;
            const bool both = n0 + 64 < p.N;
            if (lane == 0) mbar_expect_tx(bar, both ? out_stage_bytes : out_stage_bytes - LT_TILE);
            __syncwarp();
            rows.ask(at, maps.y, bar, n0);
            if (both) rows.ask(at + LT_TILE, maps.y, bar, n0 + 64);
            // (tests: each CTA leaves out one copy of its last tile)
            if (lane < chunks && !(skip_last == 2 && t + C >= end && lane == 0))
                tma_load_2d(at + LT_Y_BYTES + lane * LT_TILE, &maps.b, bar, lane * 64, e * p.N + n0);
            ++asked;
        }
    } else if (warp == 1) {
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(LT_COLS >> 3) << 17) | ((uint32_t)(LT_ROWS >> 4) << 24);
        const int steps = (r + 15) / 16;                         // as far as the adapter's rank reaches
        int i = 0;
        for (int t = rank; t < end; t += C, ++i) {
            const int s = i % out_stages, acc = i % accs, n = t * LT_COLS + (lane & 15) * 8;
            // the slices that have columns in this tile
            const unsigned present = p.col_slice == nullptr ? 1u
                : __reduce_or_sync(0xffffffffu, n < p.N ? 1u << min((int)__ldg(p.col_slice + n / 8), p.S - 1) : 0u);
            if (!__all_sync(0xffffffffu, mbar_wait(s_addr(&out_full[s]), (i / out_stages) & 1, &abort_flag, p.status, wait_ns))) break;
            if (i >= accs && !__all_sync(0xffffffffu, mbar_wait(s_addr(&acc_empty[acc]), (i / accs - 1) & 1, &abort_flag, p.status, wait_ns))) break;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t at = ring + s * out_stage_bytes + LT_Y_BYTES;
                for (int sl = 0; sl < p.S; ++sl) {
                    if (!(present >> sl & 1)) continue;
                    const uint32_t d = tmem + (acc * p.S + sl) * LT_COLS, h = base + sl * chunks * LT_TILE;
                    for (int kk = 0; kk < steps; ++kk) {
                        const uint64_t bdesc = smem_desc_sw128(at + (kk >> 2) * LT_TILE) + 2 * (kk & 3);
                        tc_mma(d, smem_desc_sw128(h + (kk >> 2) * LT_TILE) + 2 * (kk & 3), bdesc, idesc, kk != 0);
                        tc_mma(d, smem_desc_sw128(h + hbytes + (kk >> 2) * LT_TILE) + 2 * (kk & 3), bdesc, idesc, 1);
                    }
                }
                tc_commit(s_addr(&acc_full[acc]));
            }
            ++issued;
            __syncwarp();
        }
    } else {
        const float scale = p.scale[e];
        int i = 0;
        for (int t = rank; t < end; t += C, ++i) {
            const int s = i % out_stages, acc = i % accs, n0 = t * LT_COLS;
            // lane j < 8: the slice of this warp's group j of 8 columns
            const int n = n0 + half * 64 + (lane & 7) * 8;
            const int own = p.col_slice != nullptr && n < p.N ? min((int)__ldg(p.col_slice + n / 8), p.S - 1) : 0;
            bool ok = mbar_wait(s_addr(&out_full[s]), (i / out_stages) & 1, &abort_flag, p.status, wait_ns);
            ok = ok && mbar_wait(s_addr(&acc_full[acc]), (i / accs) & 1, &abort_flag, p.status, wait_ns);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            unsigned char* stage = smem + 2 * hbytes + s * out_stage_bytes;
            if (ok) {
                unsigned char* mine = stage + half * LT_TILE;
                const int row = quarter * 32 + lane;
                const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + acc * p.S * LT_COLS + half * 64;
#pragma unroll
                for (int g0 = 0; g0 < 8; g0 += 4) {
                    uint32_t v[32];
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        lt_ld8(from + __shfl_sync(0xffffffffu, own, g0 + g) * LT_COLS + (g0 + g) * 8, v + g * 8);
                    tc_wait_ld();
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint4* q = reinterpret_cast<uint4*>(mine + lt_swizzled(row, g0 + g));
                        const uint4 a = *q;
                        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
                        uint4 o;
                        uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            w[j] = pack_bf16(fmaf(scale, __uint_as_float(v[g * 8 + 2 * j]), __low2float(h[j])),
                                             fmaf(scale, __uint_as_float(v[g * 8 + 2 * j + 1]), __high2float(h[j])));
                        *q = o;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_addr(&acc_empty[acc]));
            if (!lt_all_epi(ok)) break;                          // a warp stores what all of them have left: all of the tile, or nothing from here on
            // rows in whole lines: 16 lanes a row
            const int chunk = et & 15, col = n0 + chunk * 8;
            if (col < p.N) {
                const unsigned char* from = stage + (chunk >> 3) * LT_TILE;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int row = (et >> 4) + 16 * j;
                    if (tok[row] >= 0)
                        *reinterpret_cast<uint4*>(out + (size_t)tok[row] * p.N + col) = *reinterpret_cast<const uint4*>(from + lt_swizzled(row, chunk & 7));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(s_addr(&out_empty[s]));
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*gave_up) {                                              // copies and MMAs that nobody waited for
        int here = 0;
        if (warp == 0)
            for (int i = max(0, asked - out_stages); i < asked; ++i)
                mbar_wait(s_addr(&out_full[i % out_stages]), (i / out_stages) & 1, &here, nullptr, wait_ns);
        if (warp == 1) {
            mbar_wait(s_addr(&d1_full), 0, &here, nullptr, wait_ns);
            for (int i = max(0, issued - accs); i < issued; ++i) mbar_wait(s_addr(&acc_full[i % accs]), (i / accs) & 1, &here, nullptr, wait_ns);
        }
        __syncwarp();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// A map of a row-major matrix [rows, cols] in boxes of box_rows x 64 columns with the 128-byte swizzle; made anew for every call.
static int lora_map(CUtensorMap* map, const void* ptr, long long rows, int cols, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return fail(-4, "lora_add: the driver does not export cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * 2};
    const cuuint32_t box[2] = {64u, (cuuint32_t)box_rows}, step[2] = {1u, 1u};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(-4, "lora_add: cuTensorMapEncodeTiled failed with code %d for a %lld x %d matrix", (int)r, rows, cols);
    return 0;
}

int lora_tiles(const LoraArgs& p, int sms, cudaStream_t stream) {
    const LoraTilePlan f = lora_tile_plan(p);
    const long long tiles = lora_max_tiles(p, LT_ROWS);
    const int C = lora_tile_cluster(p, sms);
    FD_REQUIRE(tiles * C < (1ll << 31), -2, "lora_add: %d tokens", p.T);
    LoraMaps maps;
    int rc = lora_map(&maps.a, p.a, (long long)p.E * p.S * p.R, p.K, (p.R + 15) / 16 * 16);
    if (rc == 0) rc = lora_map(&maps.b, p.b, (long long)p.E * p.N, p.R, LT_COLS);
    const int boxes[3] = {LT_ROWS, 16, 1};
    for (int i = 0; i < 3 && rc == 0; ++i) {
        rc = lora_map(&maps.x[i], p.x, p.T, p.K, boxes[i]);
        if (rc == 0) rc = lora_map(&maps.y[i], p.y, p.T, p.N, boxes[i]);
    }
    if (rc != 0) return rc;
    static Once once;
    if (once.first()) {
        const cudaError_t err = cudaFuncSetAttribute(lora_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_SMEM);
        if (err != cudaSuccess) return fail(-100, "lora_add: %s", cudaGetErrorString(err));
        once.done();
    }
    return launch("lora_add", lora_tile_kernel, dim3((unsigned)(tiles * C)), dim3(LT_THREADS), f.smem, stream, dim3(C, 1, 1), maps, p, f.chunks,
                  f.stages, f.out_stages, g_tc_wait_ns, g_tc_skip_last);
}

}  // namespace fd
