// What the two kernels of the attention for trees of drafted tokens share: the work list, which every block derives from
// the requests' lengths by itself, and the merge of what different blocks have found for one row.
//
// A unit is one request, one key/value head and one tile of rows (up to ROWS pairs of a node and a query head of the group that
// shares the key/value head); its work is the blocks of KEYS keys that one of its rows may see. All units' blocks stand in one
// line, request by request, and each block of the grid takes an equal, unbroken part of that line: a long request is spread over as many
// blocks as it takes, short ones share a block, and no list has to be made on the host (a captured launch follows the
// lengths that its buffers hold when it is replayed). A unit that lies inside one part is finished there; of a unit that is cut, every block
// leaves its rows' unnormalised outputs, maxima and sums in the scratch, and a second, small launch merges them in the
// order of the line.
#pragma once
#include "common.cuh"

constexpr int TREE_MAX_NODES = 64;     // a node's view of its request's nodes is one 64-bit mask
constexpr int TREE_MIN_BLOCKS = 2;     // no block takes fewer key blocks than this (of a line that has them)

struct TreeLine {
    const int* cu_q; const int* ctx_len; int R, KV, window, npt;          // npt: nodes of a row tile
};
// One request: n nodes behind c committed tokens; key blocks b0 .. b0 + nb - 1 hold what its nodes may see.
struct TreeRequest { int begin, n, c, lo, tiles, b0, nb; };

template <int KEYS>
__device__ __forceinline__ TreeRequest tree_request(const TreeLine& a, int r) {
    TreeRequest q;
    q.begin = a.cu_q[r];
    const int n = a.cu_q[r + 1] - q.begin;
    q.c = a.ctx_len[r] - n;
    q.n = min(n, TREE_MAX_NODES);
    const bool none = n <= 0 || q.c < 0;                                 // a request without nodes has no part of the line
    q.tiles = none ? 0 : (q.n + a.npt - 1) / a.npt;
    q.lo = a.window > 0 ? max(0, q.c - a.window + 1) : 0;                // the first node's position is c
    q.b0 = q.lo / KEYS;
    q.nb = none ? 0 : (q.c + q.n - 1) / KEYS + 1 - q.b0;
    return q;
}

// A place of the line: key block b of unit (request r, key/value head kvh, tile).
struct TreePlace { int r, kvh, tile, b; TreeRequest q; };

template <int KEYS>
__device__ __forceinline__ long long tree_blocks(const TreeLine& a, int r) {
    if (r >= a.R) return 0;
    const TreeRequest q = tree_request<KEYS>(a, r);
    return (long long)q.tiles * a.KV * q.nb;
}
// All lanes of a warp: the length of the line.
template <int KEYS>
__device__ __forceinline__ long long tree_total(const TreeLine& a) {
    long long sum = 0;
    for (int r = threadIdx.x & 31; r < a.R; r += 32) sum += tree_blocks<KEYS>(a, r);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
// All lanes of a warp: where position `at` of the line lies (0 <= at < total).
template <int KEYS>
__device__ __forceinline__ TreePlace tree_find(const TreeLine& a, long long at) {
    const int lane = threadIdx.x & 31;
    TreePlace p{};
    for (int r0 = 0; r0 < a.R; r0 += 32) {
        const long long mine = tree_blocks<KEYS>(a, r0 + lane);
        long long upto = mine;                                           // inclusive sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, upto > at);
        if (here) {
            const int src = __ffs(here) - 1;
            at -= __shfl_sync(0xffffffffu, upto - mine, src);
            p.r = r0 + src;
            break;
        }
        at -= __shfl_sync(0xffffffffu, upto, 31);
    }
    p.q = tree_request<KEYS>(a, p.r);
    const int unit = (int)(at / p.q.nb);
    p.b = p.q.b0 + (int)(at - (long long)unit * p.q.nb);
    p.kvh = unit / p.q.tiles;
    p.tile = unit - p.kvh * p.q.tiles;
    return p;
}
// The first block of the unit behind p's (there is one).
template <int KEYS>
__device__ __forceinline__ void tree_next_unit(const TreeLine& a, TreePlace& p) {
    if (++p.tile == p.q.tiles) {
        p.tile = 0;
        if (++p.kvh == a.KV) {
            p.kvh = 0;
            do p.q = tree_request<KEYS>(a, ++p.r); while (p.q.tiles == 0 && p.r + 1 < a.R);
        }
    }
    p.b = p.q.b0;
}
// How many blocks of the grid have a part of the line, and where the part of block i begins.
__device__ __forceinline__ int tree_parts(long long total, int grid) {
    return (int)max(1LL, min((long long)grid, total / TREE_MIN_BLOCKS));
}
__device__ __forceinline__ long long tree_part(long long total, int parts, int i) { return total * i / parts; }

// Which of the nodes a node sees: its mask without the bits of nodes that the request does not have and, with a window, without those
// nodes further up than the window (on the way to a node the higher bit is the nearer node).
__device__ __forceinline__ unsigned long long tree_mask(unsigned long long m, int n, int window) {
    if (n < 64) m &= (1ULL << n) - 1;
    if (window > 0)
        for (int over = __popcll(m) - window; over > 0; --over) m &= m - 1;
    return m;
}
// Visible keys of a row, 32 from kc on, as bits: committed keys from `lo` (at most c) to c - 1, then the nodes of `mask` at c + bit.
__device__ __forceinline__ unsigned tree_bits(unsigned long long mask, int c, int lo, int kc) {
    const int d = c - kc;                                                // committed keys from kc on
    unsigned w = d >= 32 ? 0xffffffffu : d > 0 ? ((1u << d) - 1u) | (unsigned)(mask << d) : -d < 64 ? (unsigned)(mask >> -d) : 0u;
    const int s = lo - kc;
    if (s > 0) w = s >= 32 ? 0u : w & (0xffffffffu << s);
    return w;
}

// The scratch: 2 * blocks slots of [rows][dh] outputs, then [2 * blocks][rows][2] maxima and sums. A block's first segment has slot
// 2 * block, one that it begins (and the next block goes on with) slot 2 * block + 1.
__host__ __device__ __forceinline__ size_t tree_scratch_floats(int blocks, int rows, int dh) { return (size_t)2 * blocks * rows * (dh + 2); }

template <typename TT>
struct TreeMerge { TreeLine line; const float* scratch; TT* out; int blocks, dh, H, G; };

// Block (i, y): the unit that the beginning of part i cuts, if no part before it does; a warp per row, rows y * warps .. of the tile.
template <int ROWS, int KEYS, typename TT>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeMerge<TT> p) {
    const int lane = threadIdx.x & 31;
    bl_pdl_wait();
    bl_pdl_trigger();
    const long long total = tree_total<KEYS>(p.line);
    if (total == 0) return;
    const int parts = tree_parts(total, p.blocks), i = blockIdx.x + 1;
    if (i >= parts) return;
    const long long at = tree_part(total, parts, i);
    const TreePlace u = tree_find<KEYS>(p.line, at);
    const long long begin = at - (u.b - u.q.b0), end = begin + u.q.nb;
    if (at == begin || tree_part(total, parts, i - 1) > begin) return;   // not cut here, or cut before
    const int row = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int nodes = min(p.line.npt, u.q.n - u.tile * p.line.npt);
    if (row >= nodes * p.G) return;
    const int first = tree_part(total, parts, i - 1) == begin ? 2 * (i - 1) : 2 * (i - 1) + 1;
    const float* stats = p.scratch + (size_t)2 * p.blocks * ROWS * p.dh;
    int last = i;                                                        // parts i - 1 .. last hold the unit
    while (last + 1 < parts && tree_part(total, parts, last + 1) < end) ++last;
    float m = -INFINITY;
    for (int k = i - 1 + lane; k <= last; k += 32) m = fmaxf(m, stats[2 * ((size_t)(k < i ? first : 2 * k) * ROWS + row)]);
    m = bl_warp_max(m);
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.f;
#pragma unroll 4
    for (int k = i - 1; k <= last; ++k) {
        const size_t slot = (size_t)(k < i ? first : 2 * k) * ROWS + row;
        const float2 ml = *reinterpret_cast<const float2*>(stats + 2 * slot);
        const float w = exp2f(ml.x - m_use);
        l = fmaf(w, ml.y, l);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < p.dh) o[j] = fmaf(w, p.scratch[slot * p.dh + lane + 32 * j], o[j]);
    }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const int node = row / p.G, head = u.kvh * p.G + row - node * p.G;
    TT* dst = p.out + ((size_t)(u.q.begin + u.tile * p.line.npt + node) * p.H + head) * p.dh;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < p.dh) bl_store(dst + lane + 32 * j, o[j] * inv);
}
