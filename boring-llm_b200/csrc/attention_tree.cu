// Attention of the nodes of a tree of drafted tokens over the paged cache, on the CUDA cores: 32-bit numbers, and
// bfloat16 with head and page sizes that the tensor-core kernel (attention_tree_tc.cu) is not built for.
//
// Request r brings n nodes, whose keys and values lie in its cache rows c .. c + n - 1 behind its c committed tokens. Node i sees the
// committed keys j (with a window those with j + window > its position) and the nodes of its mask (its ancestors and itself); its
// position is c + popcount(mask) - 1. out = sum_j softmax_j(scale q . k_j) v_j, in the online form, statistics in 32 bits:
// m' = max(m, max s), l' = l 2^(m - m') + sum 2^(s - m'), o' = o 2^(m - m') + sum 2^(s - m') v, s in the base-2 domain.
//
// A block holds 64 rows (pairs of a node and a query head of a group) and walks blocks of 64 keys: S as a 64 x 64 product with 8 x 4
// outputs a thread, P through shared memory with the keys outermost, O += P V with 8 rows x dh / 16 columns a thread. Values arrive
// (cp.async) under S; the next keys under the softmax and P V where they have room beside P (head sizes up to 64), else P lies where the
// keys were. Two blocks share an SM and hide each other's waits. Bound by the loads from shared memory together with the multiply-adds at large
// sizes (12 loads, two wavefronts each, for 128; 16 requests of 64 nodes at 900 to 2,000 tokens, 28 / 4 heads of 128: 659 us, 27 TFLOP/s;
// with 4 x 4 outputs a thread 1,063, with a branch for the columns past the head size in P V 780). At small sizes a chain: lengths and
// pages 3 us, first loads 2, S 3.5, softmax 1.5, P V 3.3, outputs 1, merge 8 (four requests of 13 nodes, 14 / 2 heads of 64: 30.5 us). Tried
// without gain: two multiply-adds to an instruction (f32x2); parts counted in halves of key blocks. The line of work and the merge are those of
// attention_tree.cuh.
// Rows of the cache that no node of the request may see are not read: zeros stand in their place.
#include "attention_tree.cuh"
#include "api.h"

namespace {

constexpr int ROWS = 64, KEYS = 64, THREADS = 128, LDP = ROWS + 4;

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
__global__ void __launch_bounds__(THREADS, NV <= 2 ? 2 : 1) attention_tree_kernel(const Params<TT> p) {
    constexpr bool BESIDE = NV == 1;                                     // P has room beside the keys
    extern __shared__ __align__(16) float sm[];
    __shared__ long long offs[2][KEYS], q_offs[ROWS];                    // where the keys of this block and the next lie, and the rows of q
    __shared__ unsigned long long s_seen[ROWS];                          // what each row may see
    __shared__ int s_lo[ROWS], s_ends[32];
    __shared__ TreeShare s_share;
    const int dp = (p.dh + 3) & ~3, ld = dp + 4;
    float* qs = sm;                                                      // [ROWS][ld]
    float* ks = qs + ROWS * ld;                                          // [KEYS][ld], and P [KEYS][LDP] where it has no room of its own
    float* vs = ks + (BESIDE ? KEYS * ld : max(KEYS * ld, KEYS * LDP));  // [KEYS][ld]
    float* ps = BESIDE ? vs + KEYS * ld : ks;
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
    int cols[NV];                                                        // columns past the head size take the last ones again: no branch, not stored
#pragma unroll
    for (int v = 0; v < NV; ++v) cols[v] = min(tx * 4 + 64 * v, dp - 4);

    for (bool first = true; left > 0; first = false) {
        const TreeRequest& rq = w.q;
        const int n_blocks = min(left, rq.b0 + rq.nb - w.b);
        const int node0 = w.tile * p.line.npt, nodes = min(p.line.npt, rq.n - node0);
        const int* table = p.table + (size_t)w.r * p.max_pages;
        const int hi = rq.c + rq.n - 1;
        const int lo_most = p.line.window > 0 ? max(0, rq.c + rq.n - p.line.window) : 0;     // no row's first committed key lies behind this (or behind c)
        auto place = [&](int b, int buf) {                               // where the keys of block b lie; -1: no node may see the key
            if (tid < KEYS) {
                const int j = b * KEYS + tid;
                long long off = -1;
                if (j >= rq.lo && j <= hi) off = table[j / p.page_size] * page_stride + ((long long)w.kvh * p.page_size + j % p.page_size) * p.dh;
                offs[buf][tid] = off;
            }
        };
        __syncthreads();                                                 // the segment before has been read
        place(w.b, 0);
        if (tid >= KEYS) {
            const int row = tid - KEYS, node = row / p.G;
            q_offs[row] = node < nodes ? ((long long)(rq.begin + node0 + node) * p.H + w.kvh * p.G + row - node * p.G) * p.dh : -1;
            unsigned long long seen = 0;
            int lo = 0x7fffffff;                                         // rows that the tile does not have see nothing
            if (node < nodes) {
                const unsigned long long m = p.mask[rq.begin + node0 + node];
                const int pos = rq.c + max(__popcll(rq.n < 64 ? m & ((1ULL << rq.n) - 1) : m) - 1, 0);
                seen = tree_mask(m, rq.n, p.line.window);
                lo = p.line.window > 0 ? min(max(0, pos - p.line.window + 1), rq.c) : 0;
            }
            s_seen[row] = seen;
            s_lo[row] = lo;
        }
        __syncthreads();
        copy_rows<TT, VEC>(qs, ld, p.q, q_offs, p.dh, dp);               // q and the first keys arrive together
        copy_rows<TT, VEC>(ks, ld, p.kc, offs[0], p.dh, dp);
        const bool rows_here = (tid >> 5) * 16 < nodes * p.G;            // a warp has sixteen rows: without one it only copies
        float m[8], l[8], o[8][4 * NV];
#pragma unroll
        for (int a = 0; a < 8; ++a) {
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
            float s[8][4];
#pragma unroll
            for (int a = 0; a < 8; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[a][j] = 0.f;
            if (rows_here) {
#pragma unroll 2
                for (int d = 0; d < dp; d += 4) {
                    float4 kb[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) kb[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * ld + d);
#pragma unroll
                    for (int a = 0; a < 8; ++a) {
                        const float4 qa = *reinterpret_cast<const float4*>(qs + (ty * 8 + a) * ld + d);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            s[a][j] = fmaf(qa.x, kb[j].x, s[a][j]); s[a][j] = fmaf(qa.y, kb[j].y, s[a][j]);
                            s[a][j] = fmaf(qa.z, kb[j].z, s[a][j]); s[a][j] = fmaf(qa.w, kb[j].w, s[a][j]);
                        }
                    }
                }
            }
            __syncthreads();                                             // keys have been read
            if (BESIDE && i + 1 < n_blocks) copy_rows<TT, VEC>(ks, ld, p.kc, offs[buf ^ 1], p.dh, dp);
            else cp_commit();
            if (rows_here) {
                if (k0 + KEYS <= rq.c && k0 >= lo_most) {                // every row sees all of these keys
#pragma unroll
                    for (int a = 0; a < 8; ++a)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[a][j] *= p.scale_log2;
                } else {
#pragma unroll
                    for (int a = 0; a < 8; ++a) {
                        const unsigned long long seen = s_seen[ty * 8 + a];
                        const int lo = s_lo[ty * 8 + a];
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[a][j] = tree_bits(seen, rq.c, lo, k0 + tx + 16 * j) & 1u ? s[a][j] * p.scale_log2 : -INFINITY;
                    }
                }
#pragma unroll
                for (int a = 0; a < 8; ++a) {
                    float top = fmaxf(fmaxf(s[a][0], s[a][1]), fmaxf(s[a][2], s[a][3]));
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
                for (int j = 0; j < 4; ++j) {
                    float* dst = ps + (tx + 16 * j) * LDP + ty * 8;
                    *reinterpret_cast<float4*>(dst) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
                    *reinterpret_cast<float4*>(dst + 4) = make_float4(s[4][j], s[5][j], s[6][j], s[7][j]);
                }
            }
            cp_wait<1>();
            __syncthreads();                                             // values and P are there
            if (rows_here) {
#pragma unroll 4
                for (int j = 0; j < KEYS; ++j) {
                    const float4 pa = *reinterpret_cast<const float4*>(ps + j * LDP + ty * 8), pb = *reinterpret_cast<const float4*>(ps + j * LDP + ty * 8 + 4);
                    const float pr[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        const float4 x = *reinterpret_cast<const float4*>(vs + j * ld + cols[v]);
#pragma unroll
                        for (int a = 0; a < 8; ++a) {
                            o[a][4 * v] = fmaf(pr[a], x.x, o[a][4 * v]); o[a][4 * v + 1] = fmaf(pr[a], x.y, o[a][4 * v + 1]);
                            o[a][4 * v + 2] = fmaf(pr[a], x.z, o[a][4 * v + 2]); o[a][4 * v + 3] = fmaf(pr[a], x.w, o[a][4 * v + 3]);
                        }
                    }
                }
            }
            __syncthreads();                                             // values and P have been read
            if (!BESIDE && i + 1 < n_blocks) copy_rows<TT, VEC>(ks, ld, p.kc, offs[buf ^ 1], p.dh, dp);
        }
        cp_wait<0>();
        const bool whole = n_blocks == rq.nb;
        const size_t slot = 2 * (size_t)blockIdx.x + (first ? 0 : 1);
        float* stats = tree_stats(p.scratch, gridDim.x, ROWS, p.dh) + slot * ROWS * 2;
#pragma unroll
        for (int a = 0; a < 8; ++a) {
            const int row = ty * 8 + a, node = row / p.G;
            if (node >= nodes) continue;
            if (whole) {
                const float inv = l[a] > 0.f ? 1.0f / l[a] : 0.f;
                TT* dst = p.out + q_offs[row];
#pragma unroll
                for (int j = 0; j < 4 * NV; ++j) {
                    const int col = tx * 4 + 64 * (j >> 2) + (j & 3);
                    if (col < p.dh) bl_store(dst + col, o[a][j] * inv);
                }
                continue;
            }
            if (tx == 0) { stats[2 * row] = m[a]; stats[2 * row + 1] = l[a]; }
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (tx * 4 + 64 * v < dp)
                    *tree_cols(tree_outputs(p.scratch, gridDim.x), slot, ROWS, p.dh, row, tx + 16 * v) =
                        make_float4(o[a][4 * v], o[a][4 * v + 1], o[a][4 * v + 2], o[a][4 * v + 3]);
        }
        left -= n_blocks;
        if (left > 0) tree_next_unit<KEYS>(p.line, w);
    }
}

size_t smem_bytes(int dh) {
    const size_t row = ((dh + 3) & ~3) + 4, keys = KEYS * row, probs = (size_t)KEYS * LDP;
    return (ROWS * row + KEYS * row + (dh <= 64 ? keys + probs : keys > probs ? keys : probs)) * sizeof(float);
}

// Blocks that the device holds at once (also the number of parts that the line is cut into at most): by registers up to a head size of 128, by
// shared memory above.
int resident_blocks(int dh) { return bl_device_sms() * (dh <= 128 ? 2 : 1); }

template <typename TT, bool VEC, int NV>
int launch(const Params<TT>& p, int blocks, cudaStream_t s) {
    static std::atomic<unsigned long long> allowed{0};
    const size_t smem = smem_bytes(p.dh);
    BL_CUDA(tree_allow_smem((const void*)attention_tree_kernel<TT, VEC, NV>, (int)smem_bytes(64 * NV), allowed));
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
