// Attention of the nodes of a tree of drafted tokens over the paged cache on the fifth-generation tensor cores: bfloat16, head sizes 64
// and 128, pages of 16. Formula, masks and positions are those of attention_tree.cu, the line of work that the blocks share out and the merge
// of units that are cut those of attention_tree.cuh (units of 256 rows, blocks of 64 keys).
//
// One block per SM walks its part of the line, segment by segment (a segment: some key blocks of one unit, which is one or two tiles of 128
// rows), through one pipeline that does not drain between segments:
//   copies    q rows of a tile as one box per 64 dimensions (pairs of node and query head are rows of q as they lie); of a key block one
//             box per page and tensor: 16 keys as two groups of 8 rows x (dh / 64) atoms of 128 bytes, so that a key block lies in shared
//             memory as [8 groups][atoms][8 rows][128 bytes], which the operand descriptors walk with a group stride of atoms x 1,024. One
//             warp copies keys, one values (a box costs its thread about 0.1 us). A page that no node may see is asked for behind the
//             end of the cache: zeros arrive.
//   S = Q K^T tcgen05.mma, M 128 x N 64 x K dh, into one of four buffers of tensor memory;
//   softmax   two groups of four warps, a thread per row, take every second task (a tile and a key block): maximum, then P = 2^(s - m)
//             as bfloat16 over the upper half of its scores; m moves only when a block's maximum passes it by 2^8 (then O is rescaled in
//             tensor memory). With two tiles a group keeps one; with one, the groups take the key blocks in turn, each with an output
//             of its own, and add the two up at the end. Warps without rows pass their turn;
//   O += P V  tcgen05.mma, M 128 x N dh x K 64, A from tensor memory, V as it lies.
// The next two blocks' scores are computed meanwhile. Only blocks with nodes, or at the edge of a window, look at masks.
// Values behind the request's last row, in a page that was copied, are set to zero (0 x whatever an old request left must stay 0).
// P is rounded to bfloat16 (half a step, 2^-8 of each weight, as the operand of a bfloat16 product must be); the sum is of the 32-bit values.
//
// What bounds it: with two full tiles the products and the hand-overs between the warps together. 64 requests of 64 nodes, 28 / 4 heads of
// 128, contexts of 2,003 to 4,001: 220 us in a row of captured calls, 724 TFLOP/s (827 with the rows that tiles lack); 260 us and 612 in long runs, where the power
// cap takes the clock down. The launch by itself 208 us and the merge 20, of which most lies under its end. 16 such requests (profiler, 75 us): the tensor pipes are
// active in 46 % of the cycles, DRAM at 28 % of its rate. An MMA of N 64 reads 6 KB of shared memory in 32 cycles, more than the 4 KB that there are; a key block of
// 128 would need the tensor memory that the second pair of score buffers has. With one request or few, the chains at the ends: lengths, pages, first
// copies and scores (3 us), outputs (1) and the merge (7 to 14 us by itself). Tried: key blocks of 128 in two passes over the scores 1.3 times as long; one group of row warps
// 1.6 times; 2^x by polynomials on the FMA pipes, scalar arithmetic, other orders of the exponentials: nothing.
//
// Every wait on an mbarrier is bounded; a block whose bound runs out records a code in a status word
// (bl_attention_tree_tc_status), its warps leave their loops, its copies are waited for, its tensor memory is freed.
#include "tcgen05.cuh"
#include "attention_tree.cuh"
#include <atomic>

namespace {

constexpr const char* WHO = "bl_attention_tree_tc";
constexpr int ROWS = 128, UNIT_ROWS = 2 * ROWS, KEYS = 64, PAGE = 16, PAGES = KEYS / PAGE;
constexpr int TMEM_COLS = 512, COL_P = KEYS / 2;
constexpr int ROW_WARPS = 8, COPY_WARPS = 2;                             // two groups of row warps; then: S (and q), PV, copies (12 warps: 168 registers)
constexpr int WARP_S = ROW_WARPS, WARP_PV = WARP_S + 1, WARP_COPY = WARP_PV + 1;
constexpr int THREADS = 32 * (WARP_COPY + COPY_WARPS);
constexpr uint32_t WAIT_LIMIT = 1u << 22;
// Of the line's parts (attention_tree.cuh): a unit of up to 7 key blocks is never cut, small units go one to a block. 64 requests of 8 nodes at
// 30 to 100 tokens (16 / 2 heads of 128) 8.1 us, with parts of four blocks at least 15.8; 20 of 30 nodes at 100 to 400 (28 / 4) 18.5, snapped over
// two blocks 22.4.
constexpr int MIN = 1, SNAP = 3;

template <int DH_>
struct Shape {
    static constexpr int DH = DH_, ATOMS = DH / 64;
    static constexpr int K_STAGES = DH == 64 ? 12 : 5, V_STAGES = DH == 64 ? 12 : 5;
    static constexpr int SBUFS = 4, COL_O = SBUFS * KEYS;         // tensor memory: scores, then two outputs of DH columns
    static constexpr int GROUP = ATOMS * 1024;                           // eight keys
    static constexpr int Q_BYTES = ATOMS * ROWS * 128, KV_BYTES = KEYS / 8 * GROUP;
    static constexpr int OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + K_STAGES * KV_BYTES, OFF_XCH = OFF_V + V_STAGES * KV_BYTES;
    static constexpr int OFF_BARS = OFF_XCH + 2 * ROWS * 8;              // the groups' maxima and sums: [2][128] pairs of floats
    static constexpr int SMEM_BYTES = OFF_BARS + 768;
    static_assert(SMEM_BYTES <= 227 * 1024 && COL_O + 2 * DH <= TMEM_COLS, "shape does not fit an SM");
};

__device__ int g_status = 0;           // 0 = fine; else the code of the first wait that ran out

struct Params {
    TreeLine line;
    __nv_bfloat16* out; const unsigned long long* mask; const int* table; int max_pages;
    int H, G, npt, no_group; float scale_log2; float* scratch;                // no_group: the first group of 8 rows behind the cache
};

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait of a whole warp, with the same answer in all lanes: false when the bound ran out or another warp of the block has given
// up. Most waits find their phase complete: the test that cannot block answers in half the time of the one that may. (A wait for
// the phase before the first, parity 1 of a new barrier, finds it complete.)
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* give_up, int code) {
    if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, WAIT_LIMIT, give_up, &g_status, code));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %3, %4}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(0), "r"(c3) : "memory");
}
// D (+)= A . B with the A operand in tensor memory (lane = row, a 32-bit column = two bfloat16 along K)
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 :: "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                    "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// tcgen05.wait::ld tied to the registers of the load it completes: nothing that reads them may be moved above it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
// 16 columns, and the wait for all loads, tied to what they bring
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld16_arrived(uint32_t (&a)[16], uint32_t (&b)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                   "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]) :: "memory");
    asm volatile("" : "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]),
                      "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15]) :: "memory");
}
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float ex2(float x) {                          // 2^x on the special-function unit (about 2 ulp; 2^-inf = 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}
// An operand in shared memory, 128-byte swizzle, its groups of 8 rows `group` bytes apart (tcgen05.cuh's form has 1,024).
__device__ __forceinline__ uint64_t desc_groups(uint32_t addr, int group, int atom = 16) {
    return (smem_desc(addr) & ~(((uint64_t)0x3FFF << 32) | ((uint64_t)0x3FFF << 16))) | ((uint64_t)(group >> 4) << 32) | ((uint64_t)(atom >> 4) << 16);
}

// kind::f16 instruction descriptors: D 32-bit, A and B bfloat16, N >> 3 at bit 17, M >> 4 at bit 24; bit 16: B lies keys x head size.
constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(KEYS >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
template <int DH> constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(DH >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);

// A counter of blocks as (index mod N, parity of the index div N).
template <int N> struct Ring {
    int at = 0; uint32_t par = 0;
    __device__ __forceinline__ void next() { if (++at == N) { at = 0; par ^= 1; } }
};

template <class S>
__global__ void __launch_bounds__(THREADS, 1)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const Params p) {
    constexpr int DH = S::DH, ATOMS = S::ATOMS, K_STAGES = S::K_STAGES, V_STAGES = S::V_STAGES, SBUFS = S::SBUFS, COL_O = S::COL_O;
    constexpr int GROUP = S::GROUP, KV_BYTES = S::KV_BYTES, Q_BYTES = S::Q_BYTES;
    extern __shared__ __align__(1024) unsigned char smem[];
    if (threadIdx.x == 0) { tma_prefetch_map(&map_q); tma_prefetch_map(&map_k); tma_prefetch_map(&map_v); }
    const uint32_t base = smem_u32(smem), bars = base + S::OFF_BARS;
    const uint32_t full_q = bars, q_free = bars + 8;
    const uint32_t s_done0 = bars + 16, p_ready0 = s_done0 + 8 * SBUFS, buf_free0 = p_ready0 + 8 * SBUFS;
    const uint32_t full_k0 = buf_free0 + 8 * SBUFS, k_free0 = full_k0 + 8 * K_STAGES, full_v0 = k_free0 + 8 * K_STAGES, v_free0 = full_v0 + 8 * V_STAGES;
    volatile int* give_up = reinterpret_cast<volatile int*>(smem + S::OFF_BARS + 576);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::OFF_BARS + 584);
    TreeShare* s_share = reinterpret_cast<TreeShare*>(smem + S::OFF_BARS + 592);
    int* s_ends = reinterpret_cast<int*>(smem + S::OFF_XCH);             // (the exchange of the row warps is later)
    static_assert(16 + 8 * (3 * SBUFS + 2 * K_STAGES + 2 * V_STAGES) <= 576 && 592 + sizeof(TreeShare) <= 768, "barriers overlap");
    const int warp = uniform_warp(), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        *give_up = (base & 1023u) ? 1 : 0;                               // the swizzled tiles need 1024-byte alignment
        if (base & 1023u) atomicCAS(&g_status, 0, 9);
        mbar_init(full_q, 1); mbar_init(q_free, 1);
        for (int i = 0; i < SBUFS; ++i) { mbar_init(s_done0 + 8 * i, 1); mbar_init(p_ready0 + 8 * i, ROWS / 32); mbar_init(buf_free0 + 8 * i, 1); }
        for (int i = 0; i < K_STAGES; ++i) { mbar_init(full_k0 + 8 * i, 1); mbar_init(k_free0 + 8 * i, 1); }
        for (int i = 0; i < V_STAGES; ++i) { mbar_init(full_v0 + 8 * i, 1); mbar_init(v_free0 + 8 * i, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Tensor memory before the wait for the kernel before (which has taken its own before it let this one start).
    if (warp == WARP_S) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32((const void*)tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    bl_pdl_wait();
    if (warp == 0) {
        TreeShare s = tree_share<KEYS, MIN, SNAP>(p.line, gridDim.x, blockIdx.x, s_ends);
        if (lane == 0) {
            *s_share = s;
            s.cut.items = tree_merge_items(s.cut, p.G, DH / 8);
            reinterpret_cast<TreeCut*>(p.scratch)[blockIdx.x] = s.cut;
        }
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    bl_pdl_trigger();                                                    // the next kernel may start: this block has its tensor memory
    const uint32_t tmem = *tmem_slot;
    TreePlace w = s_share->place;
    int left = s_share->left;
    bool ok = !*give_up;
    // The segments of this block's part, one after the other: f(segment, its key blocks, whether the unit has two tiles of rows). The
    // work of a segment is a row of tasks: with two tiles, both tiles on key block 0, both on key block 1, ..; with one, the key
    // blocks. Tasks alternate between the groups of row warps throughout the kernel: the task's number decides the group (mod 2) and the
    // buffer of scores (mod SBUFS).
    auto segments = [&](auto f) {
        for (int seg = 0; ok && left > 0; ++seg) {
            const int n = min(left, w.q.b0 + w.q.nb - w.b);
            f(seg, n, w.q.n - w.tile * p.line.npt > p.npt && p.line.npt > p.npt);
            left -= n;
            if (left > 0) tree_next_unit<KEYS>(p.line, w);
        }
    };

    if (warp >= WARP_COPY) {
        // ================= copies of keys and of values: lanes 0..7 look up a page each, one thread issues
        const bool keys = warp == WARP_COPY;
        const int stages = keys ? K_STAGES : V_STAGES;
        const CUtensorMap* map = keys ? &map_k : &map_v;
        const uint32_t full0 = keys ? full_k0 : full_v0, free0 = keys ? k_free0 : v_free0;
        const uint32_t dst0 = base + (keys ? S::OFF_K : S::OFF_V);
        auto group_of = [&]() -> int {                                   // lane's page of the block w.b, as a group of 8 rows of the cache
            const int first = w.b * KEYS + (lane & (PAGES - 1)) * PAGE;
            if (first > w.q.c + w.q.n - 1 || first + PAGE - 1 < w.q.lo) return p.no_group;
            return (p.table[(size_t)w.r * p.max_pages + first / PAGE] * p.line.KV + w.kvh) * 2;
        };
        int at = 0, used = 0;
        uint32_t par = 0;
        ok = __all_sync(0xffffffffu, ok);
        int group = left > 0 ? group_of() : 0;
        while (ok && left > 0) {
            int group_next = 0;                                          // on its way during this block's copies
            const uint32_t bar = full0 + 8 * at, dst = dst0 + at * KV_BYTES;
            if (--left > 0) {
                if (++w.b == w.q.b0 + w.q.nb) tree_next_unit<KEYS>(p.line, w);
                group_next = group_of();
            }
            ok = wait_warp(free0 + 8 * at, par ^ 1, give_up, keys ? 3 : 7);
            if (!ok) break;
            int g[PAGES];
#pragma unroll
            for (int pg = 0; pg < PAGES; ++pg) g[pg] = __shfl_sync(0xffffffffu, group, pg);
            if (elect_one()) {
                mbar_expect_tx(bar, KV_BYTES);
#pragma unroll
                for (int pg = 0; pg < PAGES; ++pg) tma_load_4d(dst + pg * 2 * GROUP, map, bar, g[pg]);
            }
            __syncwarp();
            used = min(used + 1, stages);
            if (++at == stages) { at = 0; par ^= 1; }
            group = group_next;
        }
        // a block that gave up lets its own copies land before its shared memory goes to the next block
        if (lane == 0 && *give_up && !(base & 1023u)) {
            for (; used > 0; --used) {
                if (at == 0) { at = stages; par ^= 1; }
                --at;
                mbar_wait_landed(full0 + 8 * at, par, 1u << 16);
            }
        }
    } else if (warp == WARP_S) {
        // ================= q of a unit, then S of each task. The whole warp goes through the loops, one thread issues
        Ring<K_STAGES> st;
        int task = 0, q_loads = 0;
        ok = __all_sync(0xffffffffu, ok);
        segments([&](int seg, int n_any, bool two_any) {
            const int n = __shfl_sync(0xffffffffu, n_any, 0), tiles = __shfl_sync(0xffffffffu, two_any ? 2 : 1, 0);
            ok = wait_warp(q_free, (uint32_t)(seg - 1) & 1, give_up, 1);
            if (!ok) return;
            if (elect_one()) {
                mbar_expect_tx(full_q, (uint32_t)(ATOMS * p.G * p.npt * 128) * tiles);
                for (int tile = 0; tile < tiles; ++tile) {
#pragma unroll
                    for (int a = 0; a < ATOMS; ++a)
                        tma_load_3d(base + tile * Q_BYTES + a * ROWS * 128, &map_q, full_q, a * 64, w.kvh * p.G, w.q.begin + w.tile * p.line.npt + tile * p.npt);
                }
            }
            __syncwarp();
            ++q_loads;
            ok = wait_warp(full_q, (uint32_t)seg & 1, give_up, 2);
            for (int j = 0; ok && j < n; ++j) {
                ok = wait_warp(full_k0 + 8 * st.at, st.par, give_up, 6);
                for (int tile = 0; ok && tile < tiles; ++tile, ++task) {
                    const int buf = task & (SBUFS - 1);
                    ok = wait_warp(buf_free0 + 8 * buf, (uint32_t)(task / SBUFS + 1) & 1, give_up, 4);
                    if (!ok) break;
                    fence_after_sync();
                    if (elect_one()) {
#pragma unroll
                        for (int at = 0; at < ATOMS; ++at) {
                            const uint64_t a = smem_desc(base + tile * Q_BYTES + at * ROWS * 128);
                            const uint64_t b = desc_groups(base + S::OFF_K + st.at * KV_BYTES + at * 1024, GROUP);
#pragma unroll
                            for (int k = 0; k < 4; ++k) umma_bf16(tmem + buf * KEYS, a + 2 * k, b + 2 * k, IDESC_S, (at | k) != 0);
                        }
                        umma_commit(s_done0 + 8 * buf);
                        if (tile + 1 == tiles) umma_commit(k_free0 + 8 * st.at);
                        if (tile + 1 == tiles && j + 1 == n) umma_commit(q_free);
                    }
                    __syncwarp();
                }
                st.next();
            }
        });
        if (lane == 0 && *give_up && q_loads > 0) mbar_wait_landed(full_q, (uint32_t)(q_loads - 1) & 1, 1u << 16);
    } else if (warp == WARP_PV) {
        Ring<V_STAGES> st;
        int task = 0;
        ok = __all_sync(0xffffffffu, ok);
        segments([&](int, int n_any, bool two_any) {
            const int n = __shfl_sync(0xffffffffu, n_any, 0), tiles = __shfl_sync(0xffffffffu, two_any ? 2 : 1, 0);
            for (int j = 0; ok && j < n; ++j) {
                ok = wait_warp(full_v0 + 8 * st.at, st.par, give_up, 5);
                for (int tile = 0; ok && tile < tiles; ++tile, ++task) {
                    const int buf = task & (SBUFS - 1);
                    ok = wait_warp(p_ready0 + 8 * buf, (uint32_t)(task / SBUFS) & 1, give_up, 12);
                    if (!ok) break;
                    fence_after_sync();
                    const bool begins = j < (tiles == 2 ? 1 : 2);        // the group's first product of the segment
                    if (elect_one()) {
                        const uint64_t bv = desc_groups(base + S::OFF_V + st.at * KV_BYTES, GROUP, 1024);
#pragma unroll
                        for (int kk = 0; kk < KEYS / 16; ++kk)           // 16 keys a step: 8 columns of P, two groups of V
                            umma_bf16_ts(tmem + COL_O + (task & 1) * DH, tmem + buf * KEYS + COL_P + kk * 8, bv + (uint64_t)(kk * (2 * GROUP >> 4)),
                                         IDESC_PV<DH>, (kk == 0 && begins) ? 0u : 1u);
                        umma_commit(buf_free0 + 8 * buf);
                        if (tile + 1 == tiles) umma_commit(v_free0 + 8 * st.at);
                    }
                    __syncwarp();
                }
                st.next();
            }
        });
    } else {
        // ================= the row warps: two groups of four, a thread a row of a tile = lane of tensor memory
        constexpr float RESCALE = 8.f;
        const int grp = warp >> 2, row = (warp & 3) * 32 + lane, node = row / p.G;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16, t_o = tmem + COL_O + grp * DH + lane_off, t_other = tmem + COL_O + (grp ^ 1) * DH + lane_off;
        float2* xch = reinterpret_cast<float2*>(smem + S::OFF_XCH);
        int own = 0, done = 0, behind = 0;                               // this group's tasks, all tasks and key blocks so far
        // Task 2 own + grp is this group's next: its buffer of scores, and the parity of its phase on the buffer's barriers.
        static_assert(SBUFS == 4, "two buffers of scores for each group");
        auto buf_of = [&](int nth) { return ((nth & 1) << 1) | grp; };
        auto par_of = [&](int nth) { return (uint32_t)(nth >> 1) & 1u; };
        // Waits for the product P V of this group's last task. A wait for a phase is valid while the barrier is at most one phase behind it
        // (phases are told apart by parity alone): the phase before on the buffer's barrier is the product of SBUFS tasks ago, without
        // which the scores of that last task, which this group has read, would not have been issued. Nor is the barrier ahead: products are
        // issued in the order of the tasks, and the second task behind it waits for this group.
        auto product_done = [&](int code) -> bool {
            const bool fine = wait_warp(buf_free0 + 8 * buf_of(own - 1), par_of(own - 1), give_up, code);
            if (fine) fence_after_sync();
            return fine;
        };
        ok = __all_sync(0xffffffffu, ok);
        // What a row may see, asked for ahead: the mask of the node that this thread's row has in the unit at `u` (0: the tile has no such row).
        auto is_two = [&](const TreePlace& u) { return u.q.n - u.tile * p.line.npt > p.npt && p.line.npt > p.npt; };
        auto ask_mask = [&](const TreePlace& u, int tasks_before) -> unsigned long long {
            const int tile = is_two(u) ? (tasks_before & 1) ^ grp : 0, at = u.tile * p.line.npt + tile * p.npt;
            return left > 0 && node < min(p.npt, u.q.n - at) ? p.mask[(size_t)u.q.begin + at + node] : 0;
        };
        unsigned long long node_mask = ask_mask(w, 0);
        for (int seg = 0; left > 0; ++seg) {                             // (a warp that has given up still comes to the groups' barriers)
            const TreeRequest q = w.q;
            const int n = min(left, q.b0 + q.nb - w.b);
            const bool two = is_two(w);
            const int first = (done & 1) ^ grp;                          // this group's first task of the segment
            const int tile = two ? first : 0, node0 = w.tile * p.line.npt + tile * p.npt, nodes = min(p.npt, q.n - node0), hi = q.c + q.n - 1;
            const bool valid = node < nodes, warp_rows = (warp & 3) * 32 < nodes * p.G;
            unsigned long long seen = 0;
            int lo = q.c;                                                // a row that the tile does not have sees nothing that matters
            if (valid) {
                const int pos = q.c + max(__popcll(q.n < 64 ? node_mask & ((1ULL << q.n) - 1) : node_mask) - 1, 0);
                seen = tree_mask(node_mask, q.n, p.line.window);
                lo = p.line.window > 0 ? min(max(0, pos - p.line.window + 1), q.c) : 0;
            }
            float m = -INFINITY, l = 0.f;
            const int tasks = two ? 2 * n : n;
            for (int k = first; k < tasks; k += 2) {
                    const int buf = buf_of(own), k0 = (w.b + (two ? k >> 1 : k)) * KEYS;
                    const uint32_t t_s = tmem + buf * KEYS + lane_off, t_p = t_s + COL_P;
                    ok = ok && wait_warp(s_done0 + 8 * buf, par_of(own), give_up, 8);
                    if (!ok) break;
                    fence_after_sync();
                    if (warp_rows) {
                        const bool all_seen = k0 + KEYS <= q.c && k0 >= lo;
                        auto mask = [&](uint32_t (&s)[32], int c) {      // a key that the row does not see becomes -inf
                            const unsigned bits = tree_bits(seen, q.c, lo, k0 + 32 * c);
#pragma unroll
                            for (int x = 0; x < 32; ++x) s[x] = (bits >> x) & 1u ? s[x] : 0xff800000u;
                        };
                        uint32_t s[2][32];
                        tmem_ld32(t_s, s[0]);
                        tmem_ld32(t_s + 32, s[1]);
                        tmem_ld_wait(s[0]);
                        tmem_ld_wait(s[1]);
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (!all_seen) mask(s[c], c);
#pragma unroll
                            for (int x = 0; x < 32; x += 2) mx[(x >> 1) & 3] = max3(mx[(x >> 1) & 3], __uint_as_float(s[c][x]), __uint_as_float(s[c][x + 1]));
                        }
                        const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2);
                        if (__any_sync(0xffffffffu, m_new > m + RESCALE)) {
                            const float alpha = ex2(m - (m_new == -INFINITY ? 0.f : m_new));
                            m = m_new;
                            l *= alpha;
                            if (k > first) {                             // what has been added so far moves to the new reference
                                ok = product_done(11);
                                if (!ok) break;
#pragma unroll 1
                                for (int h = 0; h < DH / 16; ++h) {
                                    uint32_t v[16];
                                    tmem_ld16_wait(t_o + h * 16, v);
#pragma unroll
                                    for (int x = 0; x < 16; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * alpha);
                                    tmem_st16(t_o + h * 16, v);
                                }
                            }
                        }
                        const float m_use = m == -INFINITY ? 0.f : m;
                        uint64_t sum2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
                        const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2), minus_m2 = f2_pack(-m_use, -m_use);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t pk[16];
#pragma unroll
                            for (int g = 0; g < 32; g += 16) {           // sixteen at a time, in place
                                float x[16];
#pragma unroll
                                for (int y = 0; y < 16; y += 2)
                                    f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c][g + y]), __uint_as_float(s[c][g + y + 1])), scale2, minus_m2), x[y], x[y + 1]);
#pragma unroll
                                for (int y = 0; y < 16; ++y) asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x[y]));
#pragma unroll
                                for (int y = 0; y < 8; ++y) {
                                    sum2[y & 1] = f2_add(sum2[y & 1], f2_pack(x[2 * y], x[2 * y + 1]));
                                    pk[g / 2 + y] = pack_bf16(x[2 * y], x[2 * y + 1]);
                                }
                            }
                            tmem_st16(t_p + 16 * c, pk);
                        }
                        float s_a, s_b, s_c, s_d;
                        f2_unpack(sum2[0], s_a, s_c);
                        f2_unpack(sum2[1], s_b, s_d);
                        l += (s_a + s_b) + (s_c + s_d);
                    }
                    // the last page of the request: values behind its last row become zeros (once: the first tile's product is the first)
                    if (hi >= k0 && hi < k0 + KEYS && (hi + 1) % PAGE != 0 && tile == 0) {
                        const int block = behind + (two ? k >> 1 : k), stage = block % V_STAGES;
                        ok = wait_warp(full_v0 + 8 * stage, (uint32_t)(block / V_STAGES) & 1, give_up, 10);
                        if (ok) {
                            const int r0 = hi + 1 - k0, rows = PAGE - r0 % PAGE;         // rows r0 .. r0 + rows - 1 of the stage
                            for (int x = row; x < rows * ATOMS * 8; x += ROWS) {
                                const int key = r0 + x / (ATOMS * 8), piece = x % (ATOMS * 8);
                                *reinterpret_cast<uint4*>(smem + S::OFF_V + stage * KV_BYTES + (key >> 3) * GROUP + (piece >> 3) * 1024 + (key & 7) * 128 + (piece & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    tmem_st_wait();
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready0 + 8 * buf);
                    ++own;
            }
            done += tasks;
            behind += n;
            left -= n;
            TreePlace next = w;                                          // the next unit and its mask arrive during the outputs
            if (left > 0) {
                tree_next_unit<KEYS>(p.line, next);
                node_mask = ask_mask(next, done);
            }
            // the segment's outputs (against m, not divided by l yet), once the group's last product has been added
            const bool whole = n == q.nb, had = tasks > first;
            ok = ok && (!had || product_done(13));
            float w_own = 1.f, w_other = 0.f;
            int h0 = 0, h1 = DH / 16;
            if (!two) {
                // both groups have a part of these rows: each takes half of the columns of both outputs
                xch[grp * ROWS + row] = make_float2(m, l);
                fence_before_sync();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                fence_after_sync();
                const float2 o = xch[(grp ^ 1) * ROWS + row];
                const float mm = fmaxf(m, o.x), m_use = mm == -INFINITY ? 0.f : mm;
                w_own = ex2(m - m_use); w_other = ex2(o.x - m_use);
                m = mm;
                l = l * w_own + o.y * w_other;
                h0 = grp * (DH / 32); h1 = h0 + DH / 32;
            }
            const bool other = !two && tasks > (first ^ 1);
            const float inv = whole ? (l > 0.f ? 1.0f / l : 0.f) : 1.0f;
            w_own *= inv; w_other *= inv;
            const size_t slot = 2 * (size_t)blockIdx.x + (seg == 0 ? 0 : 1);
            const int unit_row = tile * p.npt * p.G + row;
            float4* part = tree_cols(tree_outputs(p.scratch, gridDim.x), slot, UNIT_ROWS, DH, unit_row, 0);
            auto out_row = [&](int r) { return p.out + (((size_t)q.begin + node0 + r / p.G) * p.H + w.kvh * p.G + r % p.G) * DH; };
            __nv_bfloat16 *dst_even = out_row(row & ~1), *dst_odd = out_row(row | 1);
            const bool valid_even = (row & ~1) < nodes * p.G, valid_odd = (row | 1) < nodes * p.G;
            if (ok && warp_rows) {
                // sixteen columns at a time, the next ones on their way meanwhile
                uint32_t own_a[16], other_a[16], own_b[16], other_b[16];
                auto ask = [&](uint32_t (&own16)[16], uint32_t (&other16)[16], int h) {
                    if (had) tmem_ld16(t_o + h * 16, own16);
                    if (other) tmem_ld16(t_other + h * 16, other16);
                };
                auto emit = [&](uint32_t (&own16)[16], uint32_t (&other16)[16], int h) {
                    float f[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        f[x] = had ? __uint_as_float(own16[x]) * w_own : 0.f;
                        if (other) f[x] = fmaf(__uint_as_float(other16[x]), w_other, f[x]);
                    }
                    if (whole) {
                        // 32 bytes of a row leave together: neighbouring lanes exchange halves, so that both write the even lane's row, then the odd one's
                        uint32_t b[8], mine[4], theirs[4];
#pragma unroll
                        for (int x = 0; x < 8; ++x) b[x] = pack_bf16(f[2 * x], f[2 * x + 1]);
                        const bool odd = lane & 1;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? b[x] : b[4 + x], 1);
                            mine[x] = odd ? b[4 + x] : b[x];
                            theirs[x] = got;
                        }
                        const uint4 own_half = make_uint4(mine[0], mine[1], mine[2], mine[3]), other_half = make_uint4(theirs[0], theirs[1], theirs[2], theirs[3]);
                        if (odd ? valid_even : valid) *reinterpret_cast<uint4*>(dst_even + h * 16 + (odd ? 8 : 0)) = odd ? other_half : own_half;
                        if (odd ? valid : valid_odd) *reinterpret_cast<uint4*>(dst_odd + h * 16 + (odd ? 8 : 0)) = odd ? own_half : other_half;
                    } else if (valid) {
#pragma unroll
                        for (int x = 0; x < 16; x += 4) part[(size_t)(h * 4 + x / 4) * UNIT_ROWS] = make_float4(f[x], f[x + 1], f[x + 2], f[x + 3]);
                    }
                };
                ask(own_a, other_a, h0);
#pragma unroll 1
                for (int h = h0; h < h1; h += 2) {                       // (a group has an even number of sixteens)
                    tmem_ld16_arrived(own_a, other_a);
                    ask(own_b, other_b, h + 1);
                    emit(own_a, other_a, h);
                    __syncwarp();
                    tmem_ld16_arrived(own_b, other_b);
                    if (h + 2 < h1) ask(own_a, other_a, h + 2);
                    emit(own_b, other_b, h + 1);
                    __syncwarp();
                }
            }
            if (valid && !whole && h0 == 0)
                *reinterpret_cast<float2*>(tree_stats(p.scratch, gridDim.x, UNIT_ROWS, DH) + (slot * UNIT_ROWS + unit_row) * 2) = make_float2(m, l);
            fence_before_sync();                                         // the outputs have been read: the next unit's first products may write them
            if (!two) asm volatile("bar.sync 1, 256;" ::: "memory");
            w = next;
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == WARP_S) {
        __syncwarp();
        fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

int make_map(CUtensorMap* map, const void* ptr, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    BlEncodeTiled enc = bl_tensor_map_encoder();
    if (enc == nullptr) BL_FAIL("%s: cuTensorMapEncodeTiled is not available from the driver", WHO);
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(ptr), dims, strides, box, ones,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) BL_FAIL("%s: cuTensorMapEncodeTiled failed with code %d", WHO, (int)r);
    return 0;
}

template <class S>
int launch(const void* q, const void* k_cache, const void* v_cache, const Params& p, int T, int blocks, cudaStream_t stream) {
    constexpr cuuint64_t DH = S::DH;
    CUtensorMap mq, mk, mv;
    const cuuint64_t q_dims[3] = {DH, (cuuint64_t)p.H, (cuuint64_t)T}, q_strides[2] = {DH * 2, (cuuint64_t)p.H * DH * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.npt};
    const cuuint64_t dims[4] = {64, 8, (cuuint64_t)S::ATOMS, (cuuint64_t)p.no_group}, strides[3] = {DH * 2, 128, 8 * DH * 2};
    const cuuint32_t box[4] = {64, 8, (cuuint32_t)S::ATOMS, 2};
    if (make_map(&mq, q, 3, q_dims, q_strides, q_box) || make_map(&mk, k_cache, 4, dims, strides, box) || make_map(&mv, v_cache, 4, dims, strides, box)) return 1;
    static std::atomic<unsigned long long> allowed{0};
    BL_CUDA(tree_allow_smem((const void*)attention_tree_tc_kernel<S>, S::SMEM_BYTES, allowed));
    BL_CUDA(bl_launch_dependent(attention_tree_tc_kernel<S>, dim3(blocks), dim3(THREADS), (size_t)S::SMEM_BYTES, stream, mq, mk, mv, p));
    BL_CHECK_LAUNCH("bl_attention_tree_tc");
    // the most key blocks that a unit can have: where none can be cut there is nothing to merge (one request of 8 nodes at 300: 3 us of launch)
    const long long room = ((long long)p.max_pages * PAGE + KEYS - 1) / KEYS, seen = p.line.window > 0 ? ((long long)p.line.window + TREE_MAX_NODES + KEYS) / KEYS + 1 : room;
    if ((room < seen ? room : seen) <= 2 * SNAP + 1) return 0;
    TreeMerge<__nv_bfloat16> mg{p.scratch, p.out, blocks, S::DH, p.H, p.G};
    BL_CUDA(bl_launch_dependent(tree_merge_kernel<UNIT_ROWS, S::DH / 8, __nv_bfloat16>, dim3(4 * blocks), dim3(32 * TREE_MERGE_WARPS), 0, stream, mg));
    BL_CHECK_LAUNCH("bl_attention_tree_tc (merge)");
    return 0;
}

}  // namespace

extern "C" int bl_attention_tree_tc_supported(int H, int KV, int dh, int page_size) {
    return (dh == 64 || dh == 128) && page_size == PAGE && KV > 0 && H > 0 && H % KV == 0 && H / KV <= ROWS;
}
extern "C" long long bl_attention_tree_tc_scratch(int dh) { return (long long)tree_scratch_floats(bl_device_sms(), UNIT_ROWS, dh); }

extern "C" int bl_attention_tree_tc(const void* q, const void* k_cache, const void* v_cache, const int* cu_q, const int* ctx_len,
                                    const long long* mask, const int* block_table, int max_pages, void* out, float* scratch, int T, int R,
                                    int n_pages, int H, int KV, int dh, int page_size, int window, float scale, void* stream) {
    if (T == 0 || R == 0) return 0;
    if (!bl_attention_tree_tc_supported(H, KV, dh, page_size))
        BL_FAIL("%s: %d heads of %d on %d key/value heads with pages of %d are not built (64 or 128, pages of 16)", WHO, H, dh, KV, page_size);
    if (T < 0 || R < 0 || max_pages <= 0 || n_pages <= 0 || window < 0 || (long long)n_pages * KV * 2 > 0x7ffffff0LL)
        BL_FAIL("%s: bad sizes T=%d R=%d pages=%d table=%d window=%d", WHO, T, R, n_pages, max_pages, window);
    if (!(scale > 0.f)) BL_FAIL("%s: the scale of the scores must be positive (got %g)", WHO, (double)scale);
    if (scratch == nullptr) BL_FAIL("%s: no scratch", WHO);
    if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)scratch) & 15)
        BL_FAIL("%s: q, the caches, out and scratch must be 16-byte aligned", WHO);
    const int G = H / KV, npt = ROWS / G < TREE_MAX_NODES ? ROWS / G : TREE_MAX_NODES;
    const int unit = 2 * npt < TREE_MAX_NODES ? 2 * npt : TREE_MAX_NODES;
    if (!tree_line_fits(R, KV, unit, max_pages, PAGE, KEYS) || bl_device_sms() > TREE_MERGE_MAX)
        BL_FAIL("%s: %d requests with tables of %d pages are more work than a launch counts", WHO, R, max_pages);
    Params p{tree_line(cu_q, ctx_len, R, KV, window, unit), (__nv_bfloat16*)out, reinterpret_cast<const unsigned long long*>(mask), block_table, max_pages,
             H, G, npt, n_pages * KV * 2, scale * 1.4426950408889634f, scratch};
    if (dh == 64) return launch<Shape<64>>(q, k_cache, v_cache, p, T, bl_device_sms(), (cudaStream_t)stream);
    return launch<Shape<128>>(q, k_cache, v_cache, p, T, bl_device_sms(), (cudaStream_t)stream);
}

// Reads and clears the status word: 0 when no block has given up on a wait since the last call. Codes: 1 q to be read, 2 q, 3 / 7 a stage of keys /
// values to become free, 4 a buffer of scores to become free, 5 values, 6 keys, 8 scores, 10 values (row warps), 11 / 13 the output, 12 P, 9 shared
// memory not 1024-byte aligned. Synchronises the device.
extern "C" int bl_attention_tree_tc_status(int* status) {
    int v = 0, zero = 0;
    BL_CUDA(cudaMemcpyFromSymbol(&v, g_status, sizeof(int)));
    if (v != 0) BL_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    *status = v;
    return 0;
}
