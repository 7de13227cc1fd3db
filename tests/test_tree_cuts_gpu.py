"""The tree attention where its forms meet: units of two row tiles that are cut, windows that are cut, blocks that pass from units of one tile to units
of two; accepted paths of masks that are no trees; keys and values written by the product on pairs of SMs beside their positions; steps of many
nodes and of many shapes."""

import numpy as np
import pytest
import torch

import helpers
import test_generate_gpu as generation
from tree_cases import TreeStep, signed
from test_tree_ops_gpu import accept_case, accept_run

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def ops():
    from boring_llm_b200.kernels import ops as o
    return o


@pytest.fixture(autouse=True)
def waits_ended():
    """No block has given up on a bounded wait."""
    yield
    ops().check_status()


def check(s, window=0):
    got = s.run(window)
    assert torch.equal(got, s.run(window))
    if window:                                                    # (the formula works on zeros where pages are gone)
        for t in (s.k, s.v):
            t[~torch.isfinite(t)] = 0.0
    s.check(got, window, probabilities_bf16=got.dtype == torch.bfloat16)


@pytest.mark.parametrize("masks,count,path", [
    ([0b1, 0b11, 0b101, 0b0111], 2, [0, 1]),                      # node 3 sees two children of node 0 and not itself
    ([0b1, 0b11, 0b111, 0b0111], 3, [0, 1, 2]),                   # ... and one that sees all of a path, but not itself
    ([0b1, 0b111, 0b101, 0b1101], 3, [0, 2, 3]),                  # node 1 sees itself and a later node
    ([0b1, 0b10, 0b110, 0b111], 1, [0]),                          # further roots
    ([0b1, 0b01, 0b01, 0b01], 1, [0])])
def test_a_node_that_does_not_see_itself_is_not_accepted(masks, count, path):
    """Every node holds the token that is sampled everywhere: only the masks decide."""
    s, tokens, sampled, k, v = accept_case([4], [13], 2, 64, 16, 2, torch.float32, 4)
    tokens[:], sampled[:] = 5, 5
    s.mask = torch.tensor(signed(masks), dtype=torch.int64)
    before = k.clone(), v.clone()
    counts, way, answer = accept_run(s, tokens, sampled, k, v)
    assert counts.tolist() == [count] and way[0].tolist() == path + [-1] * (64 - count) and answer[0].tolist() == [5] * count + [-1] * (64 - count)
    row = lambda t, i: t[:, int(s.table[0, (13 + i) // 16]), :, (13 + i) % 16]
    for j in range(4):
        node = path[j] if j < count else j
        assert torch.equal(row(k, j), row(before[0], node)) and torch.equal(row(v, j), row(before[1], node))


def test_drafted_steps_of_many_requests_share_their_captured_shapes(model_folders):
    """Eight requests that draft as much as their text gives: a captured step for each padded number of nodes, and the right tokens."""
    from boring_llm_b200 import Engine
    d = model_folders("D", "bfloat16", 0.02)
    rng = np.random.default_rng(2)
    phrases = [helpers.random_tokens(300, 5, 70 + i) for i in range(4)]
    prompts = [sum((phrases[int(rng.integers(0, 4))] for _ in range(6 + i)), []) for i in range(8)]
    eng = Engine(d, dtype="bfloat16", ctx_size=256, max_num_seqs=8, max_tokens=2048, draft_tokens=31, debug_poison=True)
    got = eng.generate(prompts, n_predict=60, ignore_eos=True)
    for p, o in zip(prompts, got):
        assert len(o) == 60
        generation.check_greedy(d, p, o, "bfloat16")
    assert 0 < len(eng.runner._tree_graphs) <= 7 and eng.stats()["accepted_tokens"] > 0
    eng.runner.cache.check()


def tree_of(out, at, vocab, n):
    """n nodes: the certain token, a long wrong chain, and behind it the three right tokens."""
    wrong = (out[at + 1] + 1) % vocab
    tokens, parents = [out[at]] + [wrong] * (n - 4), [-1] + list(range(n - 4))
    return tokens + out[at + 1:at + 4], parents + [0, n - 3, n - 2]


@pytest.mark.parametrize("cuda_graphs", [True, False])
def test_steps_of_many_nodes(model_folders, cuda_graphs):
    """256 nodes and more: the product on pairs of SMs writes keys and values, the tree attention reads them, the right branch (the last one) is kept and its
    rows have moved: what is said afterwards is what the plain implementation says."""
    from boring_llm_b200 import Engine, StepEntry, TreeEntry
    from boring_llm_b200.sampling.params import SamplingParams, XorShift64
    d = model_folders("D", "bfloat16", 0.02)
    vocab = helpers.TINY["D"]["vocab_size"]
    run = Engine(d, dtype="bfloat16", ctx_size=512, max_num_seqs=8, max_tokens=4096, cuda_graphs=cuda_graphs).runner
    prompts = [helpers.random_tokens(vocab, 20 + 33 * i, 60 + i) for i in range(8)]
    truth = []
    for i, p in enumerate(prompts):
        out = [int(run.step([StepEntry(("t", i), p, [len(p) - 1])])[0].argmax())]
        while len(out) < 14:
            out.append(int(run.step([StepEntry(("t", i), [out[-1]], [0])])[0].argmax()))
        truth.append(out)
        run.free_request(("t", i))
        run.step([StepEntry(i, p, [])])
    said = [[t[0]] for t in truth]
    whole = 0
    for _ in range(3):
        entries = []
        for i in range(8):
            at = len(said[i]) - 1
            # (a request that has left the truth at a near tie goes on alone)
            tokens, parents = tree_of(truth[i], at, vocab, 40) if said[i] == truth[i][:at + 1] else ([said[i][-1]] * 40, [-1] + list(range(39)))
            entries.append(TreeEntry(i, tokens, parents))
        got = run.step_tree(entries, [(SamplingParams(), XorShift64(0), None)] * 8)
        for i in range(8):
            whole += len(got[i]) == 4
            said[i] += got[i][:4]
            run.truncate(i, len(prompts[i]) + len(said[i]) - 1)
    assert whole > 12                                             # most trees hold
    for i in range(8):
        said[i].append(int(run.step([StepEntry(i, [said[i][-1]], [0])])[0].argmax()))
        generation.check_greedy(d, prompts[i], said[i], "bfloat16")
    run.check_kernels()
    assert (run.graph_steps > 0) == cuda_graphs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,KV,dh", [(28, 4, 128), (14, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("counts,committed", [([64], [6000]), ([64, 33, 40], [3000, 1500, 2501]), ([64, 50, 20, 64, 37, 36, 5, 64], [700 + 61 * r for r in range(8)])])
def test_units_of_two_tiles_that_are_cut(counts, committed, H, KV, dh, dtype):
    """64 nodes of 7 or 8 query heads are a unit of two row tiles (of 126 or 128 rows) and what is left of the nodes: over few requests every unit lies in
    several blocks, whose parts of both tiles are merged; few parts and many."""
    check(TreeStep(counts, committed, H, KV, dh, 16, dtype, 31, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [460, 1000, 2049])
@pytest.mark.parametrize("H,KV,dh,counts,committed", [(4, 2, 64, [13, 30, 1], [3000, 1500, 2501]), (28, 4, 128, [64, 40], [2500, 2300]), (16, 2, 128, [24, 17, 64], [4003, 999, 30])])
def test_windows_that_are_cut(H, KV, dh, counts, committed, window, dtype):
    """Windows of more key blocks than a unit has that is never cut; the pages that they have passed hold NaN."""
    s = TreeStep(counts, committed, H, KV, dh, 16, dtype, 32, device=DEV)
    for r, c in enumerate(committed):
        for i in range(max(0, c - window + 1) // 16):
            s.k[s.table[r, i].long()] = float("nan")
            s.v[s.table[r, i].long()] = float("nan")
    check(s, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,KV,dh", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("window", [0, 130])
def test_units_of_one_and_two_tiles_in_turn(H, KV, dh, window, dtype):
    """More units than blocks, of one and of two tiles, of one key block and of several: a block goes through all of them in one pipeline."""
    rng = np.random.default_rng(5)
    counts = [int(n) for n in rng.choice([1, 5, 17, 18, 19, 35, 36, 37, 40, 54, 55, 64], 120)]
    committed = [int(c) for c in rng.choice([0, 1, 15, 50, 63, 64, 130, 200, 330, 420], 120)]
    check(TreeStep(counts, committed, H, KV, dh, 16, dtype, 33, device=DEV), window)


@pytest.mark.parametrize("rows", [256, 333, 700])
@pytest.mark.parametrize("H,KV,dh,d", [(14, 2, 64, 896), (16, 2, 128, 264), (4, 2, 64, 128)])
def test_the_product_on_pairs_writes_rows_beside_positions(rows, H, KV, dh, d):
    """Keys and values lie in the cache rows that it is given, rotated by the step's table, whose positions are others; nothing else is written.
    Against the formula in 64 bits: a sum of d products and a bias in 32 bits, (d + 1) 2^-24 of the sum of magnitudes, two products and a sum of
    the rotation (3 x 2^-24 more), then one rounding to bfloat16."""
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(rows)
    width, page, requests = (H + 2 * KV) * dh, 16, 5
    tok_req = torch.sort(torch.randint(0, requests, (rows,), generator=g, device=DEV)).values.to(torch.int32)
    per = -(-rows // page) + 2
    table = torch.randperm(requests * per, generator=g, device=DEV).to(torch.int32).view(requests, per)
    positions = torch.randint(0, 900, (rows,), generator=g, device=DEV, dtype=torch.int32)
    cache_rows = torch.cat([torch.randperm(n, generator=g, device=DEV) + 7 for n in torch.bincount(tok_req, minlength=requests).tolist()]).to(torch.int32)
    inv = 10000.0 ** (-torch.arange(dh // 2, device=DEV).float() / (dh // 2))
    x = (torch.randn(rows, d, generator=g, device=DEV) * 0.5).bfloat16()
    w = (torch.randn(width, d, generator=g, device=DEV) / d ** 0.5).bfloat16()
    b = torch.randn(width, generator=g, device=DEV).bfloat16()
    assert o.qkv_rope_tc_supported(x, w, H, KV, dh, page)
    cs, sn = o.rope_table(positions, inv, dh // 2, 1.0)
    q = torch.empty(rows, H * dh, dtype=torch.bfloat16, device=DEV)
    k = torch.full((requests * per, KV, page, dh), float("nan"), dtype=torch.bfloat16, device=DEV)
    v = k.clone()
    o.qkv_rope_tc(x, w, b, cache_rows, tok_req, table, cs, sn, q, k, v, H, KV, dh)
    full = x.double() @ w.double().T + b.double()
    mags = (x.double().abs() @ w.double().abs().T + b.double().abs()) * (d + 4) * 2.0 ** -24
    full, mags = full.view(rows, H + 2 * KV, dh), mags.view(rows, H + 2 * KV, dh)
    c, s = cs.double()[:, None], sn.double()[:, None]
    lo, hi = full[..., :dh // 2], full[..., dh // 2:]
    turned = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    slack = torch.cat([mags[..., :dh // 2] * c.abs() + mags[..., dh // 2:] * s.abs(), mags[..., dh // 2:] * c.abs() + mags[..., :dh // 2] * s.abs()], -1)
    at = table[tok_req.long(), (cache_rows // page).long()].long(), (cache_rows % page).long()
    for got, want, room in ((q.view(rows, H, dh), turned[:, :H], slack[:, :H]), (k[at[0], :, at[1]], turned[:, H:H + KV], slack[:, H:H + KV]),
                            (v[at[0], :, at[1]], full[:, H + KV:], mags[:, H + KV:])):
        assert ((got.double() - want).abs() <= room * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all()
    written = torch.zeros(requests * per, page, dtype=torch.bool, device=DEV)
    written[at] = True
    for t in (k, v):
        assert torch.isnan(t.transpose(1, 2)[~written]).all()
