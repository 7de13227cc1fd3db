// What the two kernels of the attention for trees of drafted tokens share: the work list, which every block derives from
// the requests' lengths by itself, and the merge of what different blocks have found for one row.
//
// A unit is one request, one key/value head and one tile of rows (up to ROWS pairs of a node and a query head of the group that
// shares the key/value head); its work is the blocks of KEYS keys that one of its rows may see. All units' blocks stand in one
// line, request by request, and each block of the grid takes an equal, unbroken part of that line: a long request is spread over as many
// blocks as it takes, short ones share a block, and no list has to be made on the host (a captured launch follows the
// lengths that its buffers hold when it is replayed). A part that would begin or end up to SNAP key blocks from the edge of
// a unit begins or ends there (a piece of a unit has its costs beside its key blocks: its queries, the pipeline's start, its outputs). A unit that lies inside one part is finished there; of a unit that is cut, every block
// leaves its rows' unnormalised outputs, maxima and sums in the scratch, and a second, small launch merges them in the
// order of the line.
#pragma once
#include "common.cuh"
#include <atomic>

constexpr int TREE_MAX_NODES = 64;     // a node's view of its request's nodes is one 64-bit mask

struct TreeLine {
    const int* cu_q; const int* ctx_len; int R, KV, window, npt;          // npt: nodes of a row tile
    int inv_npt;                                                         // 65,536 / npt, rounded up: x / npt = x inv_npt >> 16 for x < 1,024
};
inline TreeLine tree_line(const int* cu_q, const int* ctx_len, int R, int KV, int window, int npt) {
    return TreeLine{cu_q, ctx_len, R, KV, window, npt, (65536 + npt - 1) / npt};
}
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
    q.tiles = none ? 0 : (q.n + a.npt - 1) * a.inv_npt >> 16;           // x < 128, npt <= 64: x (inv npt - 65,536) < 65,536
    q.lo = a.window > 0 ? max(0, q.c - a.window + 1) : 0;                // the first node's position is c
    q.b0 = q.lo / KEYS;
    q.nb = none ? 0 : (q.c + q.n - 1) / KEYS + 1 - q.b0;
    return q;
}

// A place of the line: key block b of unit (request r, key/value head kvh, tile).
struct TreePlace { int r, kvh, tile, b; TreeRequest q; };

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

// A unit that the beginning of a part cuts, and no part before it: what the merge needs to know. parts = 0: there is none.
struct TreeCut { int parts, first, slot, tok, nodes, kvh, items, pad; };           // slots: first, then slot, slot + 2, .. (parts - 1 of them)
// A block's part of the line: `left` key blocks from `place` on (0: none), and what there is to merge at its beginning.
struct TreeShare { TreePlace place; int left; TreeCut cut; };

// The share of block i of `grid`, by all lanes of a warp (the same answer in each). No part has fewer than MIN blocks before parts
// snap (of a line that has them). The line is shorter than 2^31 (the host sees to it). `ends`: 32 words of shared memory.
template <int KEYS, int MIN, int SNAP>
__device__ __forceinline__ TreeShare tree_share(const TreeLine& a, int grid, int i, int* ends) {
    constexpr unsigned ALL = 0xffffffffu;
    const int lane = threadIdx.x & 31, each = (a.R + 31) / 32;           // lane l adds up requests l * each ..
    auto blocks = [&](const TreeRequest& q) { return q.tiles * a.KV * q.nb; };
    int upto = 0;
#pragma unroll 2
    for (int r = lane * each; r < min(a.R, (lane + 1) * each); ++r) upto += blocks(tree_request<KEYS>(a, r));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(ALL, upto, o);
        if (lane >= o) upto += up;
    }
    ends[lane] = upto;
    __syncwarp();
    const int total = __shfl_sync(ALL, upto, 31);
    TreeShare s{};
    if (total == 0) return s;
    const int parts = max(1, min(grid, total / MIN)), per = total / parts, more = total - per * parts;
    if (i >= parts) return s;
    auto edge = [&](int k) { return per * k + min(k, more); };
    // Lanes 0, 1 and 2 look up where parts i - 1, i and i + 1 begin, each by itself.
    const int k = i - 1 + lane;
    int at = k <= 0 ? 0 : total, begin = 0, length = 0;
    TreePlace p{};
    if (lane < 3 && k >= 0 && k < parts) {
        at = edge(k);
        int l = 0;
#pragma unroll
        for (int half = 16; half > 0; half >>= 1)
            if (ends[l + half - 1] <= at) l += half;
        int from = l > 0 ? ends[l - 1] : 0;
        p.r = l * each;
        p.q = tree_request<KEYS>(a, p.r);
        while (from + blocks(p.q) <= at) {
            from += blocks(p.q);
            p.q = tree_request<KEYS>(a, ++p.r);
        }
        const int unit = (at - from) / p.q.nb;
        length = p.q.nb;
        begin = from + unit * length;
        p.kvh = unit / p.q.tiles;
        p.tile = unit - p.kvh * p.q.tiles;
        if (SNAP > 0 && at - begin <= SNAP) at = begin;
        if (SNAP > 0 && at > begin && begin + length - at <= SNAP) {
            begin = at = begin + length;
            if (at < total) tree_next_unit<KEYS>(a, p);
            length = p.q.nb;
        }
        p.b = p.q.b0 + at - begin;
    }
    const int before = __shfl_sync(ALL, at, 0), start = __shfl_sync(ALL, at, 1), end = __shfl_sync(ALL, at, 2);
    begin = __shfl_sync(ALL, begin, 1);
    length = __shfl_sync(ALL, length, 1);
    s.left = end - start;
    if (s.left == 0) return s;
    int* words = reinterpret_cast<int*>(&p);
#pragma unroll
    for (int x = 0; x < (int)(sizeof(TreePlace) / sizeof(int)); ++x) words[x] = __shfl_sync(ALL, words[x], 1);
    s.place = p;
    if (start > begin && before <= begin) {                              // parts i - 1, i, .. hold pieces of the unit
        int inside = 0;
        for (int x = i + lane; x < parts && edge(x) < begin + length - SNAP; x += 32) ++inside;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) inside += __shfl_xor_sync(ALL, inside, o);
        s.cut.parts = 1 + inside;
        s.cut.first = before == begin ? 2 * (i - 1) : 2 * (i - 1) + 1;
        s.cut.slot = 2 * i;
        s.cut.tok = p.q.begin + p.tile * a.npt;
        s.cut.nodes = min(a.npt, p.q.n - p.tile * a.npt);
        s.cut.kvh = p.kvh;
    }
    return s;
}
// Whether the line is short enough for 32-bit places, whatever the lengths: every request with the most blocks that its table has room for.
inline bool tree_line_fits(int R, int KV, int npt, int max_pages, int page_size, int keys) {
    const long long tiles = (TREE_MAX_NODES + npt - 1) / npt, blocks = ((long long)max_pages * page_size + keys - 1) / keys + 1;
    return (long long)R * KV * tiles <= 0x7fffffffLL / blocks;
}

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

// The scratch: a TreeCut per block, then 2 * blocks slots of [dh / 4][rows][4] outputs (a thread has a row: neighbouring threads write
// neighbouring 16 bytes; dh rounded up to fours), then [2 * blocks][rows][2] maxima and sums. A block's first segment has slot 2 * block, one that it begins (and the next
// block goes on with) slot 2 * block + 1.
__host__ __device__ __forceinline__ size_t tree_slot(int rows, int dh) { return (size_t)rows * ((dh + 3) & ~3); }
__host__ __device__ __forceinline__ size_t tree_scratch_floats(int blocks, int rows, int dh) { return (size_t)8 * blocks + 2 * blocks * (tree_slot(rows, dh) + 2 * rows); }
__device__ __forceinline__ float* tree_outputs(float* scratch, int blocks) { return scratch + (size_t)8 * blocks; }
__device__ __forceinline__ float* tree_stats(float* scratch, int blocks, int rows, int dh) { return scratch + (size_t)8 * blocks + 2 * blocks * tree_slot(rows, dh); }
// Columns 4 c4 .. of a row
__device__ __forceinline__ float4* tree_cols(float* outputs, size_t slot, int rows, int dh, int row, int c4) {
    return reinterpret_cast<float4*>(outputs + slot * tree_slot(rows, dh)) + (size_t)c4 * rows + row;
}

// Lets a kernel have `bytes` of shared memory on the current device (the limit is the device's, once on each: `done` has their bits).
inline cudaError_t tree_allow_smem(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ULL << (dev & 63);
    if (done.load() & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

template <typename TT>
struct TreeMerge { float* scratch; TT* out; int blocks, dh, H, G; };

constexpr int TREE_MERGE_WARPS = 8, TREE_MERGE_MAX = 320;                // blocks of the attention's grid, at most
constexpr int TREE_MERGE_MANY = 8;                                       // more parts than this: several blocks share 32 rows
// Columns of a merging warp, of NC at few parts, and the blocks that share 32 rows then.
__host__ __device__ constexpr int tree_merge_cols(int nc) { return nc > 8 ? nc / 4 : 4; }
__device__ __forceinline__ int tree_merge_items(const TreeCut& cut, int G, int nc) {
    return cut.parts == 0 ? 0 : (cut.nodes * G + 31) / 32 * (cut.parts > TREE_MERGE_MANY ? nc / tree_merge_cols(nc) : 1);
}

// o = sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k over the parts k of each unit that is cut, in their order. The blocks share the rows of all
// cut units out, 32 at a time: lane = row, a warp has NC columns (of a unit with many parts, as when one long request is on all SMs, a
// quarter of them, four at least), and the finished rows leave through shared memory.
template <int ROWS, int NC, typename TT>
struct TreeMergeTile {
    template <int COLS>
    static __device__ __forceinline__ void run(const TreeMerge<TT>& p, const TreeCut& cut, int row0, int col_first, float* tile) {
        constexpr int LD = TREE_MERGE_WARPS * COLS + 1;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = cut.nodes * p.G, row = row0 + lane, col0 = col_first + warp * COLS;
        float* outs = tree_outputs(p.scratch, p.blocks);
        const float* stats = tree_stats(p.scratch, p.blocks, ROWS, p.dh);
        const bool live = row < rows;
        float m = -INFINITY, l = 0.f, o[COLS] = {};
        constexpr int AHEAD = COLS <= 4 ? 8 : COLS <= 8 ? 4 : 2;                         // parts whose numbers are asked for together
        for (int k0 = 0; k0 < cut.parts; k0 += AHEAD) {
            float2 ml[AHEAD];
            float4 v[AHEAD][COLS / 4];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int k = k0 + u;
                const bool there = live && k < cut.parts;
                const size_t slot = k == 0 ? cut.first : cut.slot + 2 * (k - 1);
                ml[u] = there ? *reinterpret_cast<const float2*>(stats + 2 * (slot * ROWS + row)) : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int j = 0; j < COLS; j += 4)
                    v[u][j / 4] = there && col0 + j < p.dh ? *tree_cols(outs, slot, ROWS, p.dh, row, (col0 + j) / 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {                            // one part more, against the larger of the two maxima
                const float top = fmaxf(m, ml[u].x), use = top == -INFINITY ? 0.f : top;
                const float a = exp2f(m - use), b = exp2f(ml[u].x - use);
                m = top;
                l = l * a + ml[u].y * b;
#pragma unroll
                for (int j = 0; j < COLS; j += 4) {
                    o[j] = o[j] * a + v[u][j / 4].x * b; o[j + 1] = o[j + 1] * a + v[u][j / 4].y * b;
                    o[j + 2] = o[j + 2] * a + v[u][j / 4].z * b; o[j + 3] = o[j + 3] * a + v[u][j / 4].w * b;
                }
            }
        }
        const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
        for (int j = 0; j < COLS; ++j) tile[lane * LD + warp * COLS + j] = o[j] * inv;
        __syncthreads();
        for (int x = tid; x < 32 * TREE_MERGE_WARPS * COLS; x += 32 * TREE_MERGE_WARPS) {
            const int r = x / (TREE_MERGE_WARPS * COLS), c = x - r * (TREE_MERGE_WARPS * COLS), node = (row0 + r) / p.G;
            if (row0 + r < rows && col_first + c < p.dh)
                bl_store(p.out + ((size_t)(cut.tok + node) * p.H + cut.kvh * p.G + row0 + r - node * p.G) * p.dh + col_first + c, tile[r * LD + c]);
        }
        __syncthreads();
    }
};

template <int ROWS, int NC, typename TT>
__global__ void __launch_bounds__(32 * TREE_MERGE_WARPS) tree_merge_kernel(const TreeMerge<TT> p) {
    constexpr int MANY = tree_merge_cols(NC), SHARE = NC / MANY, EACH = TREE_MERGE_MAX / 32;
    __shared__ float tile[32 * (TREE_MERGE_WARPS * NC + 1)];
    const int lane = threadIdx.x & 31;
    bl_pdl_wait();
    bl_pdl_trigger();
    // Each warp looks through the cuts for itself (lane l at cuts l * per ..): one load, no barrier.
    const TreeCut* cuts = reinterpret_cast<const TreeCut*>(p.scratch);
    const int per = (p.blocks + 31) / 32;
    int items[EACH], mine = 0;
#pragma unroll
    for (int x = 0; x < EACH; ++x) items[x] = x < per && lane * per + x < p.blocks ? cuts[lane * per + x].items : 0;
#pragma unroll
    for (int x = 0; x < EACH; ++x) mine += items[x];
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        const int src = __ffs(__ballot_sync(0xffffffffu, upto > item)) - 1;
        int nth = item - (upto - mine), at = 0;                          // the lane that holds it finds its cut
#pragma unroll
        for (int x = 0; x < EACH; ++x)
            if (at == x && nth >= items[x]) { nth -= items[x]; ++at; }
        nth = __shfl_sync(0xffffffffu, nth, src);
        const TreeCut cut = cuts[__shfl_sync(0xffffffffu, lane * per + at, src)];
        if (cut.parts > TREE_MERGE_MANY) TreeMergeTile<ROWS, NC, TT>::template run<MANY>(p, cut, nth / SHARE * 32, nth % SHARE * (TREE_MERGE_WARPS * MANY), tile);
        else TreeMergeTile<ROWS, NC, TT>::template run<NC>(p, cut, nth * 32, 0, tile);
    }
}
