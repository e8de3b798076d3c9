// What the kernels of the low-rank adapters share: their arguments, and the way from a tile's number to its tokens.
#pragma once

#include "common.cuh"

namespace fd {

// out[t] = y[t] + scale[e] B_e (A_e x[t]), e the adapter of token t.  Tokens come in the order `order`, cut by `start` into segments
// of one adapter each (`ids`; -1: no adapter, out[t] = y[t]).  a [E][S R][K], b [E][N][R]: a packed product of S projections has an
// A of its own for each; tile of 8 columns c / 8 belongs to projection col_slice[c / 8] (null: S = 1).  Adapter e uses the first
// ranks[e] of the R rows and columns.
struct LoraArgs {
    const void* x;
    const void* a;
    const void* b;
    const float* scale;
    const int* ranks;
    const int* order;
    const int* start;
    const int* ids;
    const void* y;
    void* out;
    const unsigned char* col_slice;
    int* status;
    int T, K, N, E, R, S, n_seg;
};

struct LoraTile {
    int adapter;             // -1: the tokens have none;  -2: there is no such tile
    int begin, count;        // its tokens are order[begin] .. order[begin + count - 1]
};

// Tile number `tile` of the segments cut into tiles of `rows` tokens.  Called by one whole warp; every lane gets the answer.
__device__ __forceinline__ LoraTile lora_tile(const LoraArgs& p, int tile, int rows) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    LoraTile f{-2, 0, 0};
    for (int base = 0; base < p.n_seg; base += 32) {
        int lo = 0, n = 0, id = -1;
        if (base + lane < p.n_seg) {
            lo = p.start[base + lane];
            const int hi = p.start[base + lane + 1];
            id = p.ids[base + lane];
            n = hi - lo;
            if (lo < 0 || n < 0 || hi > p.T) { set_status(p.status, STATUS_BAD_INDEX); n = 0; }
        }
        const int tiles = (n + rows - 1) / rows;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + sum > tile);
        if (hit != 0u) {
            const int src = __ffs(hit) - 1;
            const int skipped = tile - before - __shfl_sync(0xffffffffu, sum - tiles, src);
            f.begin = __shfl_sync(0xffffffffu, lo, src) + skipped * rows;
            f.count = min(rows, __shfl_sync(0xffffffffu, n, src) - skipped * rows);
            f.adapter = __shfl_sync(0xffffffffu, id, src);
            if (f.adapter < -1 || f.adapter >= p.E) {
                set_status(p.status, STATUS_BAD_INDEX);
                f.adapter = -2;
            }
            return f;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return f;
}

// Rows of tokens without an adapter (or of one that leaves the projection alone) as they are, for an output of its own: units u0 ..
// u1 - 1 of `count` rows of `units`, by `threads` threads.  Eight loads of a thread before its first store: one after another, a
// tile of 128 rows of 4,872 took 150 us, longer than any tile with products.
template <typename U>
__device__ __forceinline__ void lora_copy(const int* tok, int count, const void* from, void* to, int units, int u0, int u1, int t, int threads) {
    const U* f = static_cast<const U*>(from);
    U* o = static_cast<U*>(to);
    // (rows of up to 2^27 units, 16 of them, or of 2^24, 128: numbers of up to 2^31)
    const unsigned width = u1 > u0 ? u1 - u0 : 0, total = width * count;
    for (unsigned i0 = t; i0 < total; i0 += threads * 8) {
        U v[8];
        size_t at[8];
        bool here[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned i = i0 + j * threads, row = i / width;
            const int token = i < total ? tok[row] : -1;
            here[j] = token >= 0;
            at[j] = here[j] ? (size_t)token * units + u0 + (i - row * width) : 0;
            if (here[j]) v[j] = f[at[j]];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (here[j]) o[at[j]] = v[j];
    }
}

// What rounding to bfloat16 takes away from a sum of A x; nothing from an infinite one (inf - inf would make NaN of every output of its
// token that the sum reaches, also of those that are infinite).
__device__ __forceinline__ float lora_rest(float v) {
    const float h = __bfloat162float(__float2bfloat16_rn(v));
    return isinf(h) ? 0.f : v - h;
}

// The most tiles there can be: every segment ends with one that may not be full.
inline long long lora_max_tiles(const LoraArgs& p, int rows) { return (p.T + (long long)(rows - 1) * p.n_seg) / rows; }

// Tiles of 16 tokens that there should be: T / 16, and a part of one for each segment's last; of single tokens one each.
inline long long lora_likely_tiles(const LoraArgs& p) {
    const long long most = lora_max_tiles(p, 16), some = (long long)p.T / 16 + p.n_seg / 4;
    return most < p.n_seg || most < some ? most : (some > p.n_seg ? some : p.n_seg);
}

// Clusters of C CTAs, two CTAs to an SM, that run at once: a cluster lies within one of the GPU's groups of some 18 SMs.
inline int lora_room(int C, int sms) { return C == 16 ? 14 : (C == 8 ? 33 : 2 * sms / C); }

// The kernels on the tensor cores (lora_mma.cu): whether they take the sizes, and the launch.
bool lora_mma_takes(const LoraArgs& p);
int lora_rows(const LoraArgs& p, int sms, cudaStream_t stream);
// ... and with tiles of 128 tokens (lora_tcgen05.cu): whether they take the sizes too, and the launch.
bool lora_tiles_take(const LoraArgs& p);
int lora_tile_cluster(const LoraArgs& p, int sms);
int lora_tiles(const LoraArgs& p, int sms, cudaStream_t stream);

}  // namespace fd
