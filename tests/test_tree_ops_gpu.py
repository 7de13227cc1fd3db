"""The operators of steps with drafted trees and of forked requests, each against its formula in 64 bits or node by node, at the sizes,
masks and layouts where they can go wrong."""
import numpy as np
import pytest
import torch

from tree_cases import TreeStep, accept_by_walk, grown, masks_of, signed

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def ops():
    from boring_llm_b200.kernels import ops as o
    return o


# (query heads, key/value heads, head size, page size)
SHAPES = [(14, 2, 64, 16), (4, 2, 16, 16), (3, 1, 32, 8), (5, 5, 48, 16), (16, 2, 128, 16), (2, 1, 256, 4), (7, 1, 33, 5), (64, 1, 64, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,KV,dh,page", SHAPES)
def test_attention_tree(H, KV, dh, page, dtype):
    """Trees of 1 to 64 nodes behind no token, one, and some that end inside and at the end of a page, with a request of no nodes."""
    counts, committed = [1, 8, 0, 64, 17, 3, 1, 33], [0, 1, 5, 15, 16, 64, 128, 250]
    s = TreeStep(counts, committed, H, KV, dh, page, dtype, 1, device=DEV)
    s.check(s.run(), probabilities_bf16=dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 2, 5, 20, 64, 150])
@pytest.mark.parametrize("dh,page", [(64, 16), (48, 16), (128, 16)])
def test_attention_tree_window(dh, page, window, dtype):
    """Windows that end inside the tree, inside the committed rows, and before them; pages that a window has passed may be gone."""
    s = TreeStep([9, 64, 2, 30], [3, 200, 131, 40], 4, 2, dh, page, dtype, 2, device=DEV)
    for r, c in enumerate(s.committed):
        for i in range(max(0, c - window + 1) // page):
            s.k[s.table[r, i].long()] = float("nan")
            s.v[s.table[r, i].long()] = float("nan")
    got = s.run(window)
    for t in (s.k, s.v):                                          # (the formula works on zeros where the pages are gone)
        t[~torch.isfinite(t)] = 0.0
    s.check(got, window, probabilities_bf16=dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("requests,committed", [(1, 3000), (3, 1111), (1, 20000), (70, 30)])
def test_attention_tree_cut_keys(requests, committed, dtype):
    """Few requests with many keys (units cut over many blocks and merged) and many with few (several units a block)."""
    lengths = [committed - 7 * r for r in range(requests)] if committed > 600 else [committed + r for r in range(requests)]
    for dh, KV in ((64, 2), (128, 1)):
        s = TreeStep([13 + r % 5 for r in range(requests)], lengths, 4, KV, dh, 16, dtype, 3, device=DEV)
        s.check(s.run(), probabilities_bf16=dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_many_requests(dtype):
    """More requests than lanes, several a lane, some of them without nodes; rows behind the last request stay as they were."""
    counts = [(r * 7) % 5 for r in range(333)]
    s = TreeStep(counts, [(r * 13) % 90 for r in range(333)], 4, 2, 64, 16, dtype, 13, device=DEV)
    T = sum(counts)
    s.q = torch.cat([s.q, torch.full((9, 256), float("nan"), dtype=dtype, device=DEV)])
    s.mask = torch.cat([s.mask, torch.ones(9, dtype=torch.int64, device=DEV)])
    out = torch.full_like(s.q, 7.0)
    s.run(out=out)
    assert (out[T:] == 7.0).all()
    s.q, s.mask = s.q[:T], s.mask[:T]
    s.check(out[:T], probabilities_bf16=dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh", [64, 40])
def test_attention_tree_any_mask(dh, dtype):
    """Masks that are no trees: rows that see nothing (with and without committed rows), later nodes, nodes that are not there."""
    masks = [0, 0b110, 0, 1 << 63 | 1, 0b111] + [0, (1 << 64) - 1, 0b1000]
    s = TreeStep([5, 3], [0, 19], 4, 2, dh, 16, dtype, 4, masks=masks, device=DEV)
    got = s.run()
    assert not got[0].any() and not got[2].any()                  # nothing to see
    s.check(got, probabilities_bf16=dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_sharp_scores(dtype):
    """Scores of some hundred units: the running maximum moves often and most weights are zero."""
    s = TreeStep([20, 64], [700, 90], 4, 2, 64, 16, dtype, 5, device=DEV, spread=30.0)
    got = s.run()
    s.check(got, probabilities_bf16=dtype == torch.bfloat16)


def test_attention_tree_requests_do_not_touch():
    """A cache row that is not finite stays in its request; a request's rows do not depend on the others in the batch."""
    for dtype in (torch.float32, torch.bfloat16):
        s = TreeStep([9, 30, 12], [100, 40, 300], 4, 2, 64, 16, dtype, 6, device=DEV)
        before = s.run()
        s.v[s.table[1, 0].long()] = float("inf")
        s.k[s.table[1, 2].long()] = float("nan")
        after = s.run()
        assert torch.equal(before[:9], after[:9]) and torch.equal(before[39:], after[39:])
        assert not torch.isfinite(after[9:39]).all()


def test_attention_tree_unaligned_operands():
    """Caches and rows that begin off a 16-byte boundary."""
    for dtype, dh in ((torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)):
        s = TreeStep([9, 2], [100, 40], 4, 2, dh, 16, dtype, 7, device=DEV)
        want = s.run()
        for name in ("q", "k", "v"):
            t = getattr(s, name)
            room = torch.empty(t.numel() + 1, dtype=dtype, device=DEV)
            room[1:].copy_(t.reshape(-1))
            setattr(s, name, room[1:].view(t.shape))
        out = torch.empty(s.q.numel() + 1, dtype=dtype, device=DEV)[1:].view(s.q.shape)
        s.run(out=out)
        s.check(out, probabilities_bf16=dtype == torch.bfloat16)
        s.check(want, probabilities_bf16=dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_streams_and_graphs(dtype):
    """A second stream; a captured call whose buffers get another step; two captured calls beside each other; the same answer each time."""
    a = TreeStep([9, 30, 12, 5], [100, 400, 300, 7], 4, 2, 64, 16, dtype, 8, device=DEV)
    b = TreeStep([9, 30, 12, 5], [900, 3, 50, 260], 4, 2, 64, 16, dtype, 9, device=DEV)
    want_a, want_b = a.run(), b.run()
    assert torch.equal(want_a, a.run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = a.run()
    side.synchronize()
    assert torch.equal(on_side, want_a)
    graphs = []
    for s in (a, b):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(s.q)
        with torch.cuda.graph(g):
            s.run(out=out)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want_a) and torch.equal(graphs[1][1], want_b)
    # b's step through a's captured call (the pools differ in size: b's caches go in whole)
    big = TreeStep([9, 30, 12, 5], [900, 400, 300, 260], 4, 2, 64, 16, dtype, 10, device=DEV)
    g, out = torch.cuda.CUDAGraph(), torch.empty_like(big.q)
    with torch.cuda.graph(g):
        big.run(out=out)
    for s, want in ((a, want_a), (b, want_b)):
        big.q.copy_(s.q); big.k[:s.k.shape[0]].copy_(s.k); big.v[:s.v.shape[0]].copy_(s.v)
        big.cu_q.copy_(s.cu_q); big.ctx_len.copy_(s.ctx_len); big.mask.copy_(s.mask)
        big.table.fill_(-1); big.table[:, :s.table.shape[1]].copy_(s.table)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_attention_tree_as_single_tokens():
    """A tree that is one node is a decode step; a chain is a portion of a prompt."""
    o = ops()
    for dtype in (torch.float32, torch.bfloat16):
        s = TreeStep([1, 1], [70, 5], 4, 2, 64, 16, dtype, 11, device=DEV)
        c = TreeStep([12, 1], [70, 5], 4, 2, 64, 16, dtype, 12, device=DEV, masks=masks_of([-1] + list(range(11))) + [1])
        for x in (s, c):
            plain = torch.empty_like(x.q)
            tok_req = torch.repeat_interleave(torch.arange(2), torch.tensor(x.counts)).to(torch.int32).to(DEV)
            o.attention_plain(x.q, x.k, x.v, tok_req, x.cu_q, x.ctx_len, x.table, plain, 4, 0, x.scale)
            x.check(plain)
            x.check(x.run(), probabilities_bf16=dtype == torch.bfloat16)


# ---- accepted drafts ---------------------------------------------------------------------------------------------------


def accept_case(counts, committed, KV, dh, page, layers, dtype, seed, vocab=3, apart=False):
    rng = np.random.default_rng(seed)
    s = TreeStep(counts, committed, KV, KV, dh, page, torch.float32, seed)
    T = sum(counts)
    tokens, sampled = rng.integers(0, vocab, T).astype(np.int32), rng.integers(0, vocab, T).astype(np.int32)
    pages = s.k.shape[0]
    kv = torch.randn(layers, 2, pages, KV, page, dh, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    k, v = (kv[:, 0], kv[:, 1]) if not apart else (kv[:, 0].contiguous(), kv[:, 1].contiguous())
    return s, tokens, sampled, k, v


def accept_want(s, tokens, sampled, k, v):
    k, v = k.clone(), v.clone()
    paths, trees, t0 = [], iter(s.trees), 0
    for r, n in enumerate(s.counts):
        parents = next(trees) if n else []
        path = accept_by_walk(parents, tokens[t0:t0 + n], sampled[t0:t0 + n])
        at = lambda row: (int(s.table[r, row // s.page]), row % s.page)
        rows = [(k[:, p, :, i].clone(), v[:, p, :, i].clone()) for p, i in (at(s.committed[r] + node) for node in path)]
        for j, (kr, vr) in enumerate(rows):
            p, i = at(s.committed[r] + j)
            k[:, p, :, i], v[:, p, :, i] = kr, vr
        paths.append((path, [int(sampled[t0 + node]) for node in path]))
        t0 += n
    return paths, k, v


def accept_run(s, tokens, sampled, k, v):
    dev = lambda a: torch.from_numpy(a).to(DEV)
    return ops().accept_tree(dev(sampled), dev(tokens), s.mask.to(DEV), s.cu_q.to(DEV), s.ctx_len.to(DEV), k, v, s.table.to(DEV))


def check_accept(s, tokens, sampled, k, v):
    paths, k_want, v_want = accept_want(s, tokens, sampled, k, v)
    counts, path, answer = (t.tolist() for t in accept_run(s, tokens, sampled, k, v))
    for r, (way, toks) in enumerate(paths):
        assert counts[r] == len(way) and path[r] == way + [-1] * (64 - len(way)) and answer[r] == toks + [-1] * (64 - len(way))
    assert torch.equal(k, k_want) and torch.equal(v, v_want)
    return counts


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("KV,dh,page,layers", [(2, 64, 16, 3), (1, 33, 5, 2), (3, 6, 4, 1), (4, 128, 16, 2)])
def test_accept_tree(KV, dh, page, layers, dtype):
    """Random trees and a vocabulary of three: paths of all lengths, siblings with one token, rows that cross pages."""
    lengths = set()
    for seed in range(6):
        case = accept_case([1, 64, 0, 17, 40, 2, 33], [0, 3, 9, 16, 31, 100, 47], KV, dh, page, layers, dtype, seed, vocab=2 + seed % 3, apart=seed % 2 == 1)
        lengths |= set(check_accept(*case))
    assert len(lengths) > 4


def test_accept_tree_long_paths():
    """Chains of 64 that are taken whole (nothing moves), and paths whose every node moves, over other rows of the path."""
    for parents in ([-1] + list(range(63)), [-1, 0] + list(range(0, 62))):
        s, tokens, sampled, k, v = accept_case([64], [21], 2, 64, 16, 2, torch.bfloat16, 3)
        s.trees, s.masks = [parents], masks_of(parents)
        s.mask = torch.tensor(signed(s.masks), dtype=torch.int64)
        tokens[:], sampled[:] = 7, 7
        counts = check_accept(s, tokens, sampled, k, v)
        assert counts == [bin(s.masks[63]).count("1")]


def test_accept_tree_masks_that_are_no_trees():
    """Nodes whose mask is not their parent's with their own bit, further roots, and a request whose node 0 is none: never accepted."""
    s, tokens, sampled, k, v = accept_case([6, 3], [10, 20], 2, 64, 16, 1, torch.float32, 4)
    tokens[:], sampled[:] = 5, 5
    s.mask = torch.tensor([0b1, 0b10, 0b101, 0b1010, 0b11101, 0b111111, 0b11, 0b10, 0b101], dtype=torch.int64)
    before = k.clone(), v.clone()
    counts, path, answer = accept_run(s, tokens, sampled, k, v)
    assert counts.tolist() == [2, 0] and path[0, :3].tolist() == [0, 2, -1] and path[1, 0].item() == -1 and answer[1, 0].item() == -1
    row = lambda t, i: t[:, int(s.table[0, (10 + i) // 16]), :, (10 + i) % 16]
    assert torch.equal(row(k, 1), row(before[0], 2)) and torch.equal(row(v, 1), row(before[1], 2))


def test_accept_tree_streams_and_graphs():
    s, tokens, sampled, k, v = accept_case([64, 30, 12], [21, 40, 7], 2, 64, 16, 4, torch.bfloat16, 5, vocab=2)
    start = k.clone(), v.clone()
    paths, k_want, v_want = accept_want(s, tokens, sampled, k, v)
    dev = [torch.from_numpy(sampled).to(DEV), torch.from_numpy(tokens).to(DEV), s.mask.to(DEV), s.cu_q.to(DEV), s.ctx_len.to(DEV)]
    table = s.table.to(DEV)
    ops().accept_tree(*dev, k, v, table)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops().accept_tree(*dev, k, v, table)
    side = torch.cuda.Stream()
    for _ in range(3):
        k.copy_(start[0]); v.copy_(start[1])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        side.synchronize()
        assert got[0].tolist() == [len(p) for p, _ in paths] and torch.equal(k, k_want) and torch.equal(v, v_want)


# ---- copied blocks -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (24, 2, 70, 2, 16, 64)), (torch.float32, (3, 2, 50, 1, 5, 33)), (torch.bfloat16, (2, 2, 90, 1, 3, 7)),
                                         (torch.int32, (2, 2, 60, 11)), (torch.int8, (1, 2, 60, 13)), (torch.float32, (2, 2, 12, 100, 101))])
@pytest.mark.parametrize("n", [1, 5, 25])
def test_copy_blocks(dtype, shape, n):
    """Pages and state slots of all layers, of sizes that are whole 16-byte pieces, 4-byte pieces and neither, over 16 KB and under."""
    rng = np.random.default_rng(n)
    N = shape[2]
    n = min(n, N // 3)
    t = (torch.randn(shape, generator=torch.Generator().manual_seed(1)) * 50).to(dtype).to(DEV)
    order = rng.permutation(N).tolist()
    pairs = [(order[int(rng.integers(0, n))], d) for d in order[n:2 * n]]
    want = t.clone()
    for s, d in pairs:
        want[:, :, d] = want[:, :, s]
    ops().copy_blocks([t[:, 0], t[:, 1]], pairs)
    assert torch.equal(t, want)


def test_copy_blocks_many_pairs_and_tensors():
    """More pairs than a launch holds, and tensors with different blocks in one call."""
    a = torch.randn(2, 5000, 3, 4, device=DEV)
    b = torch.randn(3, 6000, 40, device=DEV, dtype=torch.bfloat16)
    pairs = [(i, 2600 + i) for i in range(2300)]
    want_a, want_b = a.clone(), b.clone()
    want_a[:, 2600:4900], want_b[:, 2600:4900] = a[:, :2300], b[:, :2300]
    ops().copy_blocks([a, b], pairs)
    assert torch.equal(a, want_a) and torch.equal(b, want_b)
    ops().copy_blocks([a], [])
    ops().copy_blocks([], [(0, 1)])
    assert torch.equal(a, want_a)


def test_copy_blocks_streams_and_graphs():
    t = torch.randn(4, 30, 1000, device=DEV)
    g = torch.cuda.CUDAGraph()
    ops().copy_blocks([t], [(0, 29)])
    with torch.cuda.graph(g):
        ops().copy_blocks([t], [(1, 2), (1, 3)])
    side = torch.cuda.Stream()
    for _ in range(3):
        t.normal_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        side.synchronize()
        assert torch.equal(t[:, 2], t[:, 1]) and torch.equal(t[:, 3], t[:, 1]) and not torch.equal(t[:, 4], t[:, 1])


def test_draft_step_from_scores_to_pages():
    """The operators as a step runs them: attention over the trees, the accepted rows moved, then attention of the next tokens over the
    moved rows, which gives what a cache filled token by token gives. And a fork of the request goes on alone."""
    o = ops()
    for dtype in (torch.float32, torch.bfloat16):
        s = TreeStep([24, 13], [60, 35], 4, 2, 64, 16, dtype, 20, device=DEV)
        s.check(s.run(), probabilities_bf16=dtype == torch.bfloat16)
        rng = np.random.default_rng(1)
        tokens, sampled = rng.integers(0, 2, 37).astype(np.int32), rng.integers(0, 2, 37).astype(np.int32)
        rows_k, rows_v = [s.rows_of(r, s.k) for r in range(2)], [s.rows_of(r, s.v) for r in range(2)]
        kl, vl = s.k.unsqueeze(0), s.v.unsqueeze(0)
        counts, path, _ = o.accept_tree(torch.from_numpy(sampled).to(DEV), torch.from_numpy(tokens).to(DEV), s.mask, s.cu_q, s.ctx_len, kl, vl, s.table)
        m = counts.tolist()
        # what a cache of the accepted tokens alone holds
        after = TreeStep([1, 1], [s.committed[r] + m[r] for r in range(2)], 4, 2, 64, 16, dtype, 21, device=DEV)
        after.k, after.v, after.table = s.k.clone(), s.v.clone(), s.table
        for r in range(2):
            way = list(range(s.committed[r])) + [s.committed[r] + i for i in path[r, :m[r]].tolist()]
            assert torch.equal(after.rows_of(r, s.k)[:, :len(way)], rows_k[r][:, way])
            assert torch.equal(after.rows_of(r, s.v)[:, :len(way)], rows_v[r][:, way])
        after.check(after.run(), probabilities_bf16=dtype == torch.bfloat16)
        # request 0 forks: its last page is copied to a free one, the fork writes its next row there
        free = [p for p in range(s.k.shape[0]) if p not in s.table.flatten().tolist()]
        last = int(after.table[0, (after.committed[0]) // 16])
        o.copy_blocks([after.k.unsqueeze(0), after.v.unsqueeze(0)], [(last, free[0])])
        fork = after.table.clone()
        fork[0, after.committed[0] // 16] = free[0]
        before = after.run()
        after.table = fork
        assert torch.equal(after.run(), before)


@pytest.fixture(autouse=True)
def waits_ended():
    """No block has given up on a bounded wait."""
    yield
    ops().check_status()
