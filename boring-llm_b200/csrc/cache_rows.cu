// What happens to cached rows between the steps: the rows of accepted drafted tokens move together (bl_accept_tree), and blocks (pages,
// state slots) are copied for requests that part ways (bl_copy_blocks). Both walk the tensors of all layers in one launch.
#include "common.cuh"
#include "api.h"
#include <new>
#include <string.h>

namespace {

// ---- accepted drafts ---------------------------------------------------------------------------------------------
// Node i of a request (at most 64) holds a token; mask[i] has the bits of its ancestors and its own; sampled[i] is the token that the
// model gives behind node i. Node 0 (a token that is certain) is accepted; any other node i is when its token is the one sampled
// behind its parent, the highest ancestor bit, and all nodes on its way are. No walk is needed: the nodes that agree
// with their parents are one 64-bit word A (a ballot), and node i is accepted when it is one of them and mask[i] & ~A = 0. The deepest accepted node
// (the lowest of several) ends the path. Node j of the path moves from cache row c + path[j] to c + j, in every layer: since path[j] >= j a
// thread that takes its 16 bytes of a few rows before it writes them, in ascending order, overwrites nothing that it still needs, and no
// two threads share a byte.
// Every block works the path out again (64 ids from L2, two ballots): one launch. Bound by latency at a few requests and by the bytes moved
// at many.
constexpr int NODES = 64, THREADS = 256, BATCH = 8;

struct Accept {
    const int* sampled; const int* tokens; const unsigned long long* mask; const int* cu_q; const int* ctx_len;
    const int* table; int max_pages;
    char* k; char* v; long long k_layer, v_layer;                        // bytes from one layer to the next
    int layers, KV, page_size, row_bytes;
    int* counts; int* path; int* answer;
};

template <typename P>
__global__ void __launch_bounds__(THREADS) accept_tree_kernel(const Accept p) {
    __shared__ unsigned long long s_mask[NODES];
    __shared__ int s_sampled[NODES], s_path[NODES];
    __shared__ long long s_src[NODES], s_dst[NODES];                     // rows (page * KV * page_size + place) that move, in order
    __shared__ int s_count, s_moves;
    const int r = blockIdx.y, tid = threadIdx.x;
    bl_pdl_wait();
    bl_pdl_trigger();
    const int begin = p.cu_q[r], q_len = p.cu_q[r + 1] - begin, c = p.ctx_len[r] - q_len, n = c < 0 ? 0 : min(q_len, NODES);
    if (tid < 32) {
        unsigned long long m[2];
        int tok[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = tid + 32 * h;
            m[h] = i < n ? p.mask[begin + i] : 0;
            tok[h] = i < n ? p.tokens[begin + i] : 0;
            s_mask[i] = m[h];
            s_sampled[i] = i < n ? p.sampled[begin + i] : 0;
        }
        __syncwarp();
        unsigned agree[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = tid + 32 * h;
            const unsigned long long above = m[h] & ((1ULL << i) - 1);
            bool yes = i == 0 && n > 0 && m[h] == 1;
            if (i > 0 && i < n && above != 0) {
                const int parent = 63 - __clzll((long long)above);
                yes = tok[h] == s_sampled[parent] && m[h] == (s_mask[parent] | (1ULL << i));
            }
            agree[h] = __ballot_sync(0xffffffffu, yes);
        }
        const unsigned long long A = ((unsigned long long)agree[1] << 32) | agree[0];
        int key = 0;                                                     // depth, then the lower node
#pragma unroll
        for (int h = 0; h < 2; ++h)                                      // (a mask without its node's own bit has no node that agrees)
            if ((agree[h] >> tid & 1) && (m[h] & ~A) == 0) key = max(key, __popcll(m[h]) * NODES + NODES - 1 - (tid + 32 * h));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        const unsigned long long way = key ? s_mask[NODES - 1 - (key & (NODES - 1))] : 0;
        const int count = __popcll(way);
        const int stay = __popcll(way & ~(way + 1));                     // the first nodes of the path that are nodes 0, 1, ..: in place
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = tid + 32 * h;
            if (way >> i & 1) {
                const int j = __popcll(way & ((1ULL << i) - 1));
                s_path[j] = i;
                if (j >= stay) {
                    const int* table = p.table + (size_t)r * p.max_pages;
                    const int a = c + i, b = c + j, pa = table[a / p.page_size], pb = table[b / p.page_size];
                    const long long page_rows = (long long)p.KV * p.page_size;
                    s_src[j - stay] = pa < 0 || pb < 0 ? -1 : pa * page_rows + a % p.page_size;
                    s_dst[j - stay] = pb * page_rows + b % p.page_size;
                }
            }
        }
        if (tid == 0) { s_count = count; s_moves = count - stay; }
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid < NODES) {
        const int node = tid < s_count ? s_path[tid] : -1;
        p.path[(size_t)r * NODES + tid] = node;
        p.answer[(size_t)r * NODES + tid] = node >= 0 ? s_sampled[node] : -1;
        if (tid == 0) p.counts[r] = s_count;
    }
    const int moves = s_moves;
    if (moves == 0) return;
    const int pieces = p.row_bytes / (int)sizeof(P);
    const long long strands = (long long)p.layers * 2 * p.KV * pieces;   // (layer, keys or values, head, piece of the row)
    for (long long s = (long long)blockIdx.x * THREADS + tid; s < strands; s += (long long)gridDim.x * THREADS) {
        const int piece = (int)(s % pieces), rest = (int)(s / pieces), kvh = rest % p.KV, lt = rest / p.KV;
        char* base = (lt & 1 ? p.v + (lt >> 1) * p.v_layer : p.k + (lt >> 1) * p.k_layer) + (long long)kvh * p.page_size * p.row_bytes + (long long)piece * sizeof(P);
        for (int j0 = 0; j0 < moves; j0 += BATCH) {
            P x[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (j0 + u < moves && s_src[j0 + u] >= 0) x[u] = *reinterpret_cast<const P*>(base + s_src[j0 + u] * p.row_bytes);
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (j0 + u < moves && s_src[j0 + u] >= 0) *reinterpret_cast<P*>(base + s_dst[j0 + u] * p.row_bytes) = x[u];
        }
    }
}

// ---- copied blocks -----------------------------------------------------------------------------------------------
// A thread block copies up to 16 KB of one block of one layer of one tensor, 16 bytes a thread and step, all loads in front of the
// stores. The pairs stand in the launch's parameters: no list has to reach the device first.
constexpr int MAX_TENSORS = 8, CHUNK = 16 * 1024, COPY_THREADS = 256;

struct CopyTensor { char* base; long long layer, block, bytes; int first, layers; };   // first: of its (layer, pair) items in the grid
template <int N> struct CopyList { CopyTensor t[MAX_TENSORS]; int tensors, pairs; int pair[2 * N]; };

template <typename P, int N>
__global__ void __launch_bounds__(COPY_THREADS) copy_blocks_kernel(const __grid_constant__ CopyList<N> p) {
    constexpr int STEPS = CHUNK / (COPY_THREADS * (int)sizeof(uint4));
    bl_pdl_wait();
    bl_pdl_trigger();
    int t = 0;
    while (t + 1 < p.tensors && (int)blockIdx.x >= p.t[t + 1].first) ++t;
    const CopyTensor& x = p.t[t];
    const int item = (int)blockIdx.x - x.first, layer = item / p.pairs, pair = item - layer * p.pairs;
    const char* src = x.base + layer * x.layer + p.pair[2 * pair] * x.block;
    char* dst = x.base + layer * x.layer + p.pair[2 * pair + 1] * x.block;
    for (long long at = (long long)blockIdx.y * CHUNK; at < x.bytes; at += (long long)gridDim.y * CHUNK) {
        const long long end = min(x.bytes, at + CHUNK);
        for (long long o0 = at + threadIdx.x * sizeof(P); o0 < end; o0 += (long long)STEPS * COPY_THREADS * sizeof(P)) {
            P v[STEPS];
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                const long long o = o0 + (long long)u * COPY_THREADS * sizeof(P);
                if (o < end) v[u] = *reinterpret_cast<const P*>(src + o);
            }
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                const long long o = o0 + (long long)u * COPY_THREADS * sizeof(P);
                if (o < end) *reinterpret_cast<P*>(dst + o) = v[u];
            }
        }
    }
}

template <int N>
int launch_copies(const CopyTensor* tensors, int n_tensors, const int* pairs, int n_pairs, int unit, cudaStream_t s) {
    CopyList<N> list;
    list.tensors = n_tensors;
    memcpy(list.t, tensors, sizeof(CopyTensor) * n_tensors);
    for (int p0 = 0; p0 < n_pairs; p0 += N) {
        list.pairs = n_pairs - p0 < N ? n_pairs - p0 : N;
        memcpy(list.pair, pairs + 2 * p0, sizeof(int) * 2 * list.pairs);
        long long items = 0, most = 1;
        for (int t = 0; t < list.tensors; ++t) {
            if (items + (long long)list.t[t].layers * list.pairs > 2147483647LL) BL_FAIL("bl_copy_blocks: more copies than a launch takes");
            list.t[t].first = (int)items;
            items += (long long)list.t[t].layers * list.pairs;
            if (list.t[t].bytes > most) most = list.t[t].bytes;
        }
        if (items == 0) return 0;
        const long long chunks = (most + CHUNK - 1) / CHUNK;
        const dim3 grid((unsigned)items, (unsigned)(chunks < 65535 ? chunks : 65535));
        if (unit == 16) BL_CUDA(bl_launch_dependent(copy_blocks_kernel<uint4, N>, grid, dim3(COPY_THREADS), 0, s, list));
        else if (unit == 4) BL_CUDA(bl_launch_dependent(copy_blocks_kernel<unsigned, N>, grid, dim3(COPY_THREADS), 0, s, list));
        else BL_CUDA(bl_launch_dependent(copy_blocks_kernel<unsigned char, N>, grid, dim3(COPY_THREADS), 0, s, list));
        BL_CHECK_LAUNCH("bl_copy_blocks");
    }
    return 0;
}

// What a list of pairs must be: inside the tensors, no target twice, and no target that is also a source (copies run in any order).
int check_pairs(const int* pairs, int n, long long blocks) {
    const size_t words = (size_t)((blocks + 63) / 64);
    unsigned long long* seen = new (std::nothrow) unsigned long long[words]();
    if (seen == nullptr) BL_FAIL("bl_copy_blocks: no host memory for %lld blocks", blocks);
    int bad = -1, why = 0;
    for (int i = 0; i < n && bad < 0; ++i) {
        const int s = pairs[2 * i], d = pairs[2 * i + 1];
        if (s < 0 || d < 0 || s >= blocks || d >= blocks) { bad = i; why = 1; }
        else if (seen[d >> 6] >> (d & 63) & 1) { bad = i; why = 2; }
        else seen[d >> 6] |= 1ULL << (d & 63);
    }
    for (int i = 0; i < n && bad < 0; ++i)
        if (seen[pairs[2 * i] >> 6] >> (pairs[2 * i] & 63) & 1) { bad = i; why = 3; }
    delete[] seen;
    if (bad < 0) return 0;
    const int s = pairs[2 * bad], d = pairs[2 * bad + 1];
    if (why == 1) BL_FAIL("bl_copy_blocks: pair %d copies block %d to %d, outside 0..%lld", bad, s, d, blocks - 1);
    if (why == 2) BL_FAIL("bl_copy_blocks: block %d is the target of two copies", d);
    BL_FAIL("bl_copy_blocks: block %d is both source and target of a copy", s);
}

}  // namespace

extern "C" int bl_accept_tree(const int* sampled, const int* tokens, const long long* mask, const int* cu_q, const int* ctx_len,
                              const int* block_table, int max_pages, void* k_pages, void* v_pages, int elem_bytes, long long k_layer_stride,
                              long long v_layer_stride, int layers, int KV, int page_size, int dh, int* counts, int* path, int* answer, int R,
                              void* stream) {
    if (R == 0) return 0;
    if (R < 0 || R > 65535) BL_FAIL("bl_accept_tree: %d requests are not built (at most 65,535)", R);
    if (layers < 0 || KV <= 0 || page_size <= 0 || dh <= 0 || max_pages <= 0 || (elem_bytes != 2 && elem_bytes != 4))
        BL_FAIL("bl_accept_tree: bad sizes layers=%d KV=%d page=%d head=%d pages=%d element=%d", layers, KV, page_size, dh, max_pages, elem_bytes);
    Accept a{sampled, tokens, reinterpret_cast<const unsigned long long*>(mask), cu_q, ctx_len, block_table, max_pages, (char*)k_pages,
             (char*)v_pages, k_layer_stride * elem_bytes, v_layer_stride * elem_bytes, layers, KV, page_size, dh * elem_bytes, counts, path, answer};
    const long long all = (long long)(uintptr_t)k_pages | (long long)(uintptr_t)v_pages | a.k_layer | a.v_layer | a.row_bytes;
    const int unit = all % 16 == 0 ? 16 : elem_bytes;
    const long long strands = (long long)layers * 2 * KV * (a.row_bytes / unit);
    long long gx = (strands + THREADS - 1) / THREADS;
    gx = gx < 1 ? 1 : gx > 65535 ? 65535 : gx;
    const dim3 grid((unsigned)gx, (unsigned)R);
    if (unit == 16) BL_CUDA(bl_launch_dependent(accept_tree_kernel<uint4>, grid, dim3(THREADS), 0, (cudaStream_t)stream, a));
    else if (unit == 4) BL_CUDA(bl_launch_dependent(accept_tree_kernel<unsigned>, grid, dim3(THREADS), 0, (cudaStream_t)stream, a));
    else BL_CUDA(bl_launch_dependent(accept_tree_kernel<unsigned short>, grid, dim3(THREADS), 0, (cudaStream_t)stream, a));
    BL_CHECK_LAUNCH("bl_accept_tree");
    return 0;
}

extern "C" int bl_copy_blocks(int n_tensors, const long long* tensors, const int* pairs, int n_pairs, void* stream) {
    if (n_tensors < 0 || n_pairs < 0) BL_FAIL("bl_copy_blocks: bad sizes");
    if (n_tensors == 0 || n_pairs == 0) return 0;
    if (n_tensors > MAX_TENSORS) BL_FAIL("bl_copy_blocks: %d tensors are more than the %d of a launch", n_tensors, MAX_TENSORS);
    long long fewest = tensors[4], all = 0;
    CopyTensor t[MAX_TENSORS];
    for (int i = 0; i < n_tensors; ++i) {
        const long long* x = tensors + 5 * i;
        if (x[2] < 0 || x[3] < 0 || x[3] > 0x7fffffffLL || x[4] < 0 || x[4] > 0x7fffffffLL) BL_FAIL("bl_copy_blocks: bad sizes of tensor %d", i);
        if (x[4] < fewest) fewest = x[4];
        all |= x[0] | x[1] | x[2];
        t[i] = CopyTensor{(char*)x[0], x[1], x[2], x[2], 0, (int)x[3]};
    }
    if (check_pairs(pairs, n_pairs, fewest)) return 1;
    const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    if (n_pairs <= 32) return launch_copies<32>(t, n_tensors, pairs, n_pairs, unit, (cudaStream_t)stream);
    return launch_copies<1024>(t, n_tensors, pairs, n_pairs, unit, (cudaStream_t)stream);
}
