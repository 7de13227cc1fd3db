// Attention of the nodes of a tree of drafted tokens over the paged cache, on the CUDA cores: 32-bit numbers, and
// bfloat16 with head and page sizes that the tensor-core kernel (attention_tree_tc.cu) is not built for.
//
// Request r brings n nodes, whose keys and values lie in its cache rows c .. c + n - 1 behind its c committed tokens. Node i sees the
// committed keys j (with a window those with j + window > its position) and the nodes of its mask (its ancestors and itself); its
// position is c + popcount(mask) - 1. out = sum_j softmax_j(scale q . k_j) v_j, in the online form, statistics in 32 bits:
// m' = max(m, max s), l' = l 2^(m - m') + sum 2^(s - m'), o' = o 2^(m - m') + sum 2^(s - m') v, s in the base-2 domain.
//
// A block holds 64 rows (pairs of a node and a query head of a group) and walks blocks of 64 keys: S as a 64 x 64 product with 4 x 4
// outputs a thread, P through shared memory with the keys outermost, O += P V with 4 rows x dh / 16 columns a thread. Keys of the next
// block arrive (cp.async) under the softmax and P V, values under S. The line of work and the merge are those of attention_tree.cuh.
// Rows of the cache that no node of the request may see are not read: zeros stand in their place.
#include "attention_tree.cuh"
#include "api.h"
#include <atomic>

namespace {

constexpr int ROWS = 64, KEYS = 64, THREADS = 256, LDP = ROWS + 4;

template <typename TT>
struct Params {
    TreeLine line;
    const TT* q; const TT* kc; const TT* vc; TT* out;
    const unsigned long long* mask; const int* table; int max_pages;
    int H, G, dh, page_size; float scale_log2; float* scratch;
};

__device__ __forceinline__ void cp16(float* dst, const float* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// 64 rows of dh values (row i at src + offs[i], offs < 0: zeros; rows of q, keys or values) into shared rows of `ld` floats, of which the last dp - dh are zeros.
template <typename TT, bool VEC>
__device__ __forceinline__ void copy_rows(float* dst, int ld, const TT* src, const long long* offs, int dh, int dp) {
    const int pieces = dp >> 2;
    for (int i = threadIdx.x; i < KEYS * pieces; i += THREADS) {
        const int row = i / pieces, d = (i - row * pieces) << 2;
        const long long off = offs[row];
        float* to = dst + row * ld + d;
        if constexpr (VEC && sizeof(TT) == 4) {
            cp16(to, reinterpret_cast<const float*>(src) + (off < 0 ? 0 : off + d), off >= 0);
        } else if constexpr (VEC) {
            uint2 v = make_uint2(0u, 0u);
            if (off >= 0) v = *reinterpret_cast<const uint2*>(src + off + d);
            const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&v.x), b = *reinterpret_cast<const __nv_bfloat162*>(&v.y);
            *reinterpret_cast<float4*>(to) = make_float4(__low2float(a), __high2float(a), __low2float(b), __high2float(b));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] = off >= 0 && d + j < dh ? bl_load(src + off + d + j) : 0.f;
        }
    }
    cp_commit();
}

// NV: columns of the output a thread owns are tx * 4 + 64 * v, v < NV.
template <typename TT, bool VEC, int NV>
__global__ void __launch_bounds__(THREADS, NV == 1 ? 2 : 1) attention_tree_kernel(const Params<TT> p) {
    extern __shared__ __align__(16) float sm[];
    __shared__ long long offs[2][KEYS], q_offs[ROWS];                    // where the keys of this block and the next lie, and the rows of q
    __shared__ TreeShare s_share;
    __shared__ int s_ends[32];
    const int dp = (p.dh + 3) & ~3, ld = dp + 4;
    float* qs = sm;                                                      // [ROWS][ld]
    float* ks = qs + ROWS * ld;                                          // [KEYS][ld]
    float* vs = ks + KEYS * ld;                                          // [KEYS][ld]
    float* ps = vs + KEYS * ld;                                          // [KEYS][LDP]
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    bl_pdl_wait();
    bl_pdl_trigger();
    if (tid < 32) {
        TreeShare s = tree_share<KEYS, 1, 0>(p.line, gridDim.x, blockIdx.x, s_ends);
        if (tid == 0) {
            s_share = s;
            s.cut.items = tree_merge_items(s.cut, p.G, 8 * NV);
            reinterpret_cast<TreeCut*>(p.scratch)[blockIdx.x] = s.cut;
        }
    }
    __syncthreads();
    TreePlace w = s_share.place;
    int left = s_share.left;
    const long long page_stride = (long long)p.line.KV * p.page_size * p.dh;

    for (bool first = true; left > 0; first = false) {
        const TreeRequest& rq = w.q;
        const int n_blocks = min(left, rq.b0 + rq.nb - w.b);
        const int node0 = w.tile * p.line.npt, nodes = min(p.line.npt, rq.n - node0);
        const int* table = p.table + (size_t)w.r * p.max_pages;
        const int hi = rq.c + rq.n - 1;
        auto place = [&](int b, int buf) {                               // where the keys of block b lie; -1: no node may see the key
            if (tid < KEYS) {
                const int j = b * KEYS + tid;
                long long off = -1;
                if (j >= rq.lo && j <= hi) off = table[j / p.page_size] * page_stride + ((long long)w.kvh * p.page_size + j % p.page_size) * p.dh;
                offs[buf][tid] = off;
            }
        };
        // the tile's rows of q, and what each of this thread's four rows may see
        __syncthreads();                                                 // the segment before has been read
        place(w.b, 0);
        if (tid >= KEYS && tid < KEYS + ROWS) {
            const int row = tid - KEYS, node = row / p.G;
            q_offs[row] = node < nodes ? ((long long)(rq.begin + node0 + node) * p.H + w.kvh * p.G + row - node * p.G) * p.dh : -1;
        }
        __syncthreads();
        copy_rows<TT, VEC>(qs, ld, p.q, q_offs, p.dh, dp);               // q and the first keys arrive together
        copy_rows<TT, VEC>(ks, ld, p.kc, offs[0], p.dh, dp);
        const bool rows_here = (tid >> 5) * 8 < nodes * p.G;             // a warp has eight rows: without one it only copies
        unsigned long long seen[4];
        int lo[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int node = (ty * 4 + a) / p.G;
            seen[a] = 0; lo[a] = 0x7fffffff;                             // rows that the tile does not have see nothing
            if (node < nodes) {
                const unsigned long long m = p.mask[rq.begin + node0 + node];
                const int pos = rq.c + max(__popcll(rq.n < 64 ? m & ((1ULL << rq.n) - 1) : m) - 1, 0);
                seen[a] = tree_mask(m, rq.n, p.line.window);
                lo[a] = p.line.window > 0 ? min(max(0, pos - p.line.window + 1), rq.c) : 0;
            }
        }
        float m[4], l[4], o[4][4 * NV];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            m[a] = -INFINITY; l[a] = 0.f;
#pragma unroll
            for (int j = 0; j < 4 * NV; ++j) o[a][j] = 0.f;
        }
        for (int i = 0; i < n_blocks; ++i) {
            const int k0 = (w.b + i) * KEYS, buf = i & 1;
            copy_rows<TT, VEC>(vs, ld, p.vc, offs[buf], p.dh, dp);       // (behind the barrier that ends the block before)
            if (i + 1 < n_blocks) place(w.b + i + 1, buf ^ 1);
            cp_wait<1>();
            __syncthreads();                                             // keys are there
            float s[4][4];
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[a][j] = 0.f;
#pragma unroll 2
            for (int d = 0; rows_here && d < dp; d += 4) {
                float4 qa[4], kb[4];
#pragma unroll
                for (int a = 0; a < 4; ++a) qa[a] = *reinterpret_cast<const float4*>(qs + (ty * 4 + a) * ld + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) kb[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * ld + d);
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[a][j] = fmaf(qa[a].x, kb[j].x, s[a][j]); s[a][j] = fmaf(qa[a].y, kb[j].y, s[a][j]);
                        s[a][j] = fmaf(qa[a].z, kb[j].z, s[a][j]); s[a][j] = fmaf(qa[a].w, kb[j].w, s[a][j]);
                    }
            }
            __syncthreads();                                             // keys have been read
            if (i + 1 < n_blocks) copy_rows<TT, VEC>(ks, ld, p.kc, offs[buf ^ 1], p.dh, dp);
            else cp_commit();
            if (rows_here) {
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool sees = tree_bits(seen[a], rq.c, lo[a], k0 + tx + 16 * j) & 1u;
                    s[a][j] = sees ? s[a][j] * p.scale_log2 : -INFINITY;
                    top = fmaxf(top, s[a][j]);
                }
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                const float m_new = fmaxf(m[a], top), m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = exp2f(m[a] - m_use);
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) { s[a][j] = exp2f(s[a][j] - m_use); sum += s[a][j]; }
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                l[a] = l[a] * alpha + sum;
                m[a] = m_new;
#pragma unroll
                for (int j = 0; j < 4 * NV; ++j) o[a][j] *= alpha;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4*>(ps + (tx + 16 * j) * LDP + ty * 4) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
            }
            cp_wait<1>();
            __syncthreads();                                             // values and P are there
#pragma unroll 4
            for (int j = 0; rows_here && j < KEYS; ++j) {
                const float4 pr = *reinterpret_cast<const float4*>(ps + j * LDP + ty * 4);
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int col = tx * 4 + 64 * v;
                    if (col < dp) {
                        const float4 x = *reinterpret_cast<const float4*>(vs + j * ld + col);
                        const float pa[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            o[a][4 * v] = fmaf(pa[a], x.x, o[a][4 * v]); o[a][4 * v + 1] = fmaf(pa[a], x.y, o[a][4 * v + 1]);
                            o[a][4 * v + 2] = fmaf(pa[a], x.z, o[a][4 * v + 2]); o[a][4 * v + 3] = fmaf(pa[a], x.w, o[a][4 * v + 3]);
                        }
                    }
                }
            }
            __syncthreads();                                             // values and P have been read
        }
        cp_wait<0>();
        const bool whole = n_blocks == rq.nb;
        const size_t slot = 2 * (size_t)blockIdx.x + (first ? 0 : 1);
        float* stats = tree_stats(p.scratch, gridDim.x, ROWS, p.dh) + slot * ROWS * 2;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int row = ty * 4 + a, node = row / p.G;
            if (node >= nodes) continue;
            if (whole) {
                const float inv = l[a] > 0.f ? 1.0f / l[a] : 0.f;
                TT* dst = p.out + ((size_t)(rq.begin + node0 + node) * p.H + w.kvh * p.G + row - node * p.G) * p.dh;
#pragma unroll
                for (int j = 0; j < 4 * NV; ++j) {
                    const int col = tx * 4 + 64 * (j >> 2) + (j & 3);
                    if (col < p.dh) bl_store(dst + col, o[a][j] * inv);
                }
            } else if (tx == 0) {
                stats[2 * row] = m[a]; stats[2 * row + 1] = l[a];
            }
        }
        if (!whole) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (tx * 4 + 64 * v >= dp) continue;
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *tree_cols(tree_outputs(p.scratch, gridDim.x), slot, ROWS, p.dh, ty * 4 + a, tx + 16 * v) =
                        make_float4(o[a][4 * v], o[a][4 * v + 1], o[a][4 * v + 2], o[a][4 * v + 3]);
            }
        }
        left -= n_blocks;
        if (left > 0) tree_next_unit<KEYS>(p.line, w);
    }
}

size_t smem_bytes(int dh) { return ((size_t)(ROWS + 2 * KEYS) * (((dh + 3) & ~3) + 4) + (size_t)KEYS * LDP) * sizeof(float); }

// Blocks that the device holds at once (also the number of parts that the line is cut into at most).
int resident_blocks(int dh) {
    const int per_sm = dh <= 64 ? 2 : 1;                                 // by registers (and 118 KB of shared memory at a head size of 128)
    return bl_device_sms() * per_sm;
}

template <typename TT, bool VEC, int NV>
int launch(const Params<TT>& p, int blocks, cudaStream_t s) {
    static std::atomic<bool> configured{false};
    const size_t smem = smem_bytes(p.dh);
    if (!configured) {
        BL_CUDA(cudaFuncSetAttribute(attention_tree_kernel<TT, VEC, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(64 * NV)));
        configured = true;
    }
    BL_CUDA(bl_launch_dependent(attention_tree_kernel<TT, VEC, NV>, dim3(blocks), dim3(THREADS), smem, s, p));
    BL_CHECK_LAUNCH("bl_attention_tree");
    TreeMerge<TT> mg{p.scratch, p.out, blocks, p.dh, p.H, p.G};
    BL_CUDA(bl_launch_dependent(tree_merge_kernel<ROWS, 8 * NV, TT>, dim3(4 * bl_device_sms()), dim3(32 * TREE_MERGE_WARPS), 0, s, mg));
    BL_CHECK_LAUNCH("bl_attention_tree (merge)");
    return 0;
}

template <typename TT>
int run(Params<TT> p, int blocks, cudaStream_t s) {
    const bool vec = p.dh % 4 == 0 && (((uintptr_t)p.q | (uintptr_t)p.kc | (uintptr_t)p.vc) & (sizeof(TT) * 4 - 1)) == 0;
    if (p.dh <= 64) return vec ? launch<TT, true, 1>(p, blocks, s) : launch<TT, false, 1>(p, blocks, s);
    if (p.dh <= 128) return vec ? launch<TT, true, 2>(p, blocks, s) : launch<TT, false, 2>(p, blocks, s);
    return vec ? launch<TT, true, 4>(p, blocks, s) : launch<TT, false, 4>(p, blocks, s);
}

}  // namespace

extern "C" long long bl_attention_tree_scratch(int dh) { return (long long)tree_scratch_floats(resident_blocks(dh), ROWS, dh); }

extern "C" int bl_attention_tree(const void* q, const void* k_cache, const void* v_cache, int dtype, const int* cu_q, const int* ctx_len,
                                 const long long* mask, const int* block_table, int max_pages, void* out, float* scratch, int T, int R, int H,
                                 int KV, int dh, int page_size, int window, float scale, void* stream) {
    if (T == 0 || R == 0) return 0;
    if (H <= 0 || KV <= 0 || H % KV != 0) BL_FAIL("bl_attention_tree: %d heads cannot share %d key/value heads", H, KV);
    if (H / KV > ROWS) BL_FAIL("bl_attention_tree: %d query heads on one key/value head are not built (at most %d)", H / KV, ROWS);
    if (dh <= 0 || dh > 256) BL_FAIL("bl_attention_tree: head size %d is not built (1 to 256)", dh);
    if (T < 0 || R < 0 || max_pages <= 0 || page_size <= 0 || window < 0) BL_FAIL("bl_attention_tree: bad sizes T=%d R=%d pages=%d page=%d window=%d", T, R, max_pages, page_size, window);
    if (!(scale > 0.f)) BL_FAIL("bl_attention_tree: the scale of the scores must be positive (got %g)", (double)scale);
    if (scratch == nullptr) BL_FAIL("bl_attention_tree: no scratch");
    const int G = H / KV, blocks = resident_blocks(dh), npt = ROWS / G < TREE_MAX_NODES ? ROWS / G : TREE_MAX_NODES;
    if (!tree_line_fits(R, KV, npt, max_pages, page_size, KEYS) || blocks > TREE_MERGE_MAX)
        BL_FAIL("bl_attention_tree: %d requests with tables of %d pages of %d tokens are more work than a launch counts", R, max_pages, page_size);
    const TreeLine line = tree_line(cu_q, ctx_len, R, KV, window, npt);
    const auto* mk = reinterpret_cast<const unsigned long long*>(mask);
    const float scale_log2 = scale * 1.4426950408889634f;
    if (dtype == BL_F32)
        return run(Params<float>{line, (const float*)q, (const float*)k_cache, (const float*)v_cache, (float*)out, mk, block_table, max_pages, H, G,
                                 dh, page_size, scale_log2, scratch}, blocks, (cudaStream_t)stream);
    if (dtype == BL_BF16)
        return run(Params<__nv_bfloat16>{line, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k_cache, (const __nv_bfloat16*)v_cache,
                                         (__nv_bfloat16*)out, mk, block_table, max_pages, H, G, dh, page_size, scale_log2, scratch}, blocks,
                   (cudaStream_t)stream);
    BL_FAIL("bl_attention_tree: unknown dtype %d", dtype);
}
