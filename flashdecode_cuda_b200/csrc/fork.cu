// Sequences that go on as several beams: what a slot of the cache holds is copied to other slots, for all layers in one
// launch.  Full cache blocks need no copy, their users share them; what is copied is
//   * the filled part of the last block of every layer's keys and values (fd_copy_blocks),
//   * the state of fixed size that recurrent layers keep per slot (fd_copy_states).
// No destination is a source or appears twice (a child takes the place of a sequence that ends), so a copy needs no second buffer
// and no order.
//
// Both move bytes and do nothing else: bound by HBM, half of the traffic reads and half writes.  A thread moves 16 bytes at a
// time with several loads in flight before the first store; tensors whose rows are no multiple of that are moved in the largest
// unit that divides them.  A CTA per copy and plane of blocks (per copy and 32 KB of states): a full server's copies are thousands of CTAs,
// and one request's are a CTA per SM or two, whose time is the launch and two trips to memory.
// Measured: 90 copies of up to 64 tokens in 96 planes of 8 heads of 128 (1.11 GB) 172.9 us, 6.44 TB/s, a plain copy's rate; 3 copies in 56
// planes of 2 heads (6 MB) 2.8 us; 60 slots of 48 states (3.16 GB) 490 us, 6.45 TB/s; 3 slots of 12 states (10 MB) 3.4 us.
#include "common.cuh"

namespace fd {

constexpr int CP_THREADS = 256;
constexpr int CP_UNROLL = 4;

template <typename V> __device__ __forceinline__ V cp_load(const V* p) { return __ldcs(p); }
template <typename V> __device__ __forceinline__ void cp_store(V* p, V v) { *p = v; }

// pool [planes][num_blocks][heads][block_size][row] in units of V, `row` units per token and head.  grid: (copies, planes).
template <typename V>
__global__ void __launch_bounds__(CP_THREADS)
copy_blocks_kernel(V* __restrict__ pool, long long num_blocks, int heads, int block_size, int row, const int* __restrict__ src,
                   const int* __restrict__ dst, const int* __restrict__ count, int* status) {
    const int i = blockIdx.x;
    const int s = src[i], d = dst[i], c = count[i];
    if (s < 0 || s >= num_blocks || d < 0 || d >= num_blocks || c < 0 || c > block_size) {
        if (threadIdx.x == 0 && blockIdx.y == 0) set_status(status, STATUS_BAD_INDEX);
        return;
    }
    const long long head = (long long)block_size * row, block = head * heads;
    V* plane = pool + (long long)blockIdx.y * num_blocks * block;
    const V* from = plane + s * block;
    V* to = plane + d * block;
    const unsigned seg = (unsigned)(c * row), total = seg * heads;       // the filled places of the block, head after head
    for (unsigned u0 = threadIdx.x; u0 < total; u0 += CP_THREADS * CP_UNROLL) {
        V v[CP_UNROLL];
        long long o[CP_UNROLL];
#pragma unroll
        for (int j = 0; j < CP_UNROLL; ++j) {
            const unsigned u = u0 + j * CP_THREADS;
            if (u < total) {
                const unsigned h = u / seg;
                o[j] = (long long)h * head + (u - h * seg);
                v[j] = cp_load(from + o[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < CP_UNROLL; ++j)
            if (u0 + j * CP_THREADS < total) cp_store(to + o[j], v[j]);
    }
}

constexpr int CP_STATES = 64;            // states of one launch: their addresses travel as the kernel's arguments
constexpr int CP_CHUNK = 32768;          // bytes of a state that a CTA moves
struct StateList {
    unsigned char* base[CP_STATES];
    long long bytes[CP_STATES];          // of one slot
    int first[CP_STATES + 1];            // the state's first chunk
    int n;
};

template <typename V>
__device__ __forceinline__ void copy_span(const unsigned char* from, unsigned char* to, int bytes) {
    const V* f = reinterpret_cast<const V*>(from);
    V* t = reinterpret_cast<V*>(to);
    const int n = bytes / (int)sizeof(V);
    for (int u0 = threadIdx.x; u0 < n; u0 += CP_THREADS * CP_UNROLL) {
        V v[CP_UNROLL];
#pragma unroll
        for (int j = 0; j < CP_UNROLL; ++j)
            if (u0 + j * CP_THREADS < n) v[j] = cp_load(f + u0 + j * CP_THREADS);
#pragma unroll
        for (int j = 0; j < CP_UNROLL; ++j)
            if (u0 + j * CP_THREADS < n) cp_store(t + u0 + j * CP_THREADS, v[j]);
    }
}

// grid: (chunks of all states, copies)
__global__ void __launch_bounds__(CP_THREADS)
copy_states_kernel(const __grid_constant__ StateList L, int slots, const int* __restrict__ src, const int* __restrict__ dst, int* status) {
    const int s = src[blockIdx.y], d = dst[blockIdx.y], c = blockIdx.x;
    if (s < 0 || s >= slots || d < 0 || d >= slots) {
        if (threadIdx.x == 0 && c == 0) set_status(status, STATUS_BAD_INDEX);
        return;
    }
    int lo = 0, hi = L.n - 1;            // the last state that begins at or before this chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (L.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const long long bytes = L.bytes[lo], at = (long long)(c - L.first[lo]) * CP_CHUNK;
    const unsigned char* from = L.base[lo] + (long long)s * bytes + at;
    unsigned char* to = L.base[lo] + (long long)d * bytes + at;
    const int n = (int)(bytes - at < CP_CHUNK ? bytes - at : CP_CHUNK);
    const unsigned long long all = (unsigned long long)L.base[lo] | (unsigned long long)bytes;
    if ((all & 15) == 0) copy_span<uint4>(from, to, n);
    else if ((all & 3) == 0) copy_span<unsigned int>(from, to, n);
    else copy_span<unsigned char>(from, to, n);
}

}  // namespace fd

using namespace fd;

// pool: [planes, num_blocks, heads, block_size, row_bytes]; src, dst, count [n] int: count[i] tokens of block src[i] to dst[i].
extern "C" int fd_copy_blocks(void* pool, int planes, long long num_blocks, int heads, int block_size, long long row_bytes,
                              const int* src, const int* dst, const int* count, int n, int* status, cudaStream_t stream) {
    if (n == 0 || planes == 0 || heads == 0 || block_size == 0 || row_bytes == 0) return 0;
    FD_REQUIRE(n > 0 && planes > 0 && num_blocks > 0 && heads > 0 && block_size > 0 && row_bytes > 0, -2,
               "copy_blocks: %d copies in a pool of %d planes, %lld blocks, %d heads, %d tokens, %lld bytes", n, planes, num_blocks, heads,
               block_size, row_bytes);
    FD_REQUIRE(planes <= 65535, -2, "copy_blocks: %d planes in one call", planes);
    FD_REQUIRE((long long)heads * block_size * row_bytes < (1ll << 31), -2, "copy_blocks: a block of %lld bytes",
               (long long)heads * block_size * row_bytes);
    const unsigned long long all = (unsigned long long)pool | (unsigned long long)row_bytes;
    const dim3 grid(n, planes);
    if ((all & 15) == 0)
        copy_blocks_kernel<uint4><<<grid, CP_THREADS, 0, stream>>>((uint4*)pool, num_blocks, heads, block_size, (int)(row_bytes / 16), src, dst, count, status);
    else if ((all & 3) == 0)
        copy_blocks_kernel<unsigned int><<<grid, CP_THREADS, 0, stream>>>((unsigned int*)pool, num_blocks, heads, block_size, (int)(row_bytes / 4), src, dst, count, status);
    else
        copy_blocks_kernel<unsigned char><<<grid, CP_THREADS, 0, stream>>>((unsigned char*)pool, num_blocks, heads, block_size, (int)row_bytes, src, dst, count, status);
    return check_launch("copy_blocks");
}

// states: n_states addresses; bytes: of all slots of each; src, dst [n] int (device).
extern "C" int fd_copy_states(void* const* states, const long long* bytes, int n_states, int slots, const int* src, const int* dst,
                              int n, int* status, cudaStream_t stream) {
    if (n == 0 || n_states == 0) return 0;
    if (slots == 0) return 0;
    FD_REQUIRE(n > 0 && n <= 65535 && n_states > 0 && slots > 0, -2, "copy_states: %d copies of %d states of %d slots", n, n_states, slots);
    for (int at = 0; at < n_states; at += CP_STATES) {
        StateList L;
        L.n = 0;
        long long chunks = 0;
        for (int j = at; j < n_states && j < at + CP_STATES; ++j) {
            const long long one = bytes[j] / slots;
            if (one <= 0) continue;
            L.base[L.n] = (unsigned char*)states[j];
            L.bytes[L.n] = one;
            L.first[L.n++] = (int)chunks;
            chunks += (one + CP_CHUNK - 1) / CP_CHUNK;
            FD_REQUIRE(chunks < (1ll << 31), -2, "copy_states: states of too many bytes");
        }
        if (L.n == 0) continue;
        L.first[L.n] = (int)chunks;
        copy_states_kernel<<<dim3((unsigned)chunks, n), CP_THREADS, 0, stream>>>(L, slots, src, dst, status);
        const int rc = check_launch("copy_states");
        if (rc != 0) return rc;
    }
    return 0;
}
