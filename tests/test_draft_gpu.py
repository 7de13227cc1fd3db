"""Steps with drafted trees and forked requests through the runner and the engine: the tokens are those of one step after the other."""
import numpy as np
import pytest
import torch

import helpers
import test_generate_gpu as generation

pytestmark = pytest.mark.gpu


def engine(d, dtype, **kw):
    from boring_llm_b200 import Engine
    opts = dict(dtype=dtype, ctx_size=256, max_num_seqs=8, max_tokens=2048, prefill_chunk=16)
    opts.update(kw)
    return Engine(d, **opts)


def repeating(name, n, seed):
    """A prompt in which runs of tokens come back."""
    rng = np.random.default_rng(seed)
    phrases = [helpers.random_tokens(helpers.TINY[name]["vocab_size"], 6, seed + i) for i in range(3)]
    out = []
    while len(out) < n:
        out += phrases[int(rng.integers(0, 3))]
    return out[:n]


@pytest.mark.parametrize("std", [0.02, 0.25])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_drafts_do_not_change_the_tokens(model_folders, name, dtype, std):
    """Head sizes 16, 32, 48 and 64, windows of 20 and 150 positions; greedy and drawn; poisoned free pages."""
    d = model_folders(name, dtype, std)
    prompts = [repeating(name, n, 40 + n) for n in (7, 30, 65)]
    plain, drafted = engine(d, dtype), engine(d, dtype, draft_tokens=12, debug_poison=True)
    greedy = plain.generate(prompts, n_predict=40, ignore_eos=True)
    got = drafted.generate(prompts, n_predict=40, ignore_eos=True)
    assert [len(o) for o in got] == [40, 40, 40]
    s = drafted.stats()
    assert s["drafted_tokens"] > 0 and s["live_requests"] == 0 and s["pages_in_use"] == [0] * len(s["pages_in_use"])
    drafted.runner.cache.check()
    if dtype == "float32":
        assert got == greedy
        drawn = dict(n_predict=30, temperature=0.9, top_k=20, seed=11, ignore_eos=True)
        assert drafted.generate(prompts, **drawn) == plain.generate(prompts, **drawn)
    elif std == 0.02:
        for p, o in zip(prompts, got):
            generation.check_greedy(d, p, o, dtype)


def test_drafts_are_accepted_and_steps_captured(model_folders):
    """Text that repeats itself: fewer steps than tokens, most of them replays of captured ones."""
    d = model_folders("D", "bfloat16", 0.02)
    prompt = [5, 9, 14, 23] * 12
    plain, drafted = engine(d, "bfloat16"), engine(d, "bfloat16", draft_tokens=15)
    a, b = plain.generate([prompt], n_predict=120, ignore_eos=True), drafted.generate([prompt], n_predict=120, ignore_eos=True)
    generation.check_greedy(d, prompt, b[0], "bfloat16")
    s = drafted.stats()
    assert len(b[0]) == 120 and s["accepted_tokens"] > 30 and s["steps"] < plain.stats()["steps"] - 30
    assert drafted.runner.graph_steps > 0 and len(a[0]) == 120


def follow(runner, rid, tokens):
    """The greedy tokens behind `tokens`, one step after the other."""
    from boring_llm_b200 import StepEntry
    out = []
    for _ in range(tokens):
        logits = runner.step([StepEntry(rid, [out[-1]] if out else [follow.first], [0])])
        out.append(int(logits[0].argmax()))
    return out


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "C", "D"])
def test_step_tree_keeps_the_right_branch(model_folders, name, dtype):
    """Trees whose right branch is the last of several: it is taken whole, its rows have moved, and the request goes on as if it had been fed token
    by token. In steps of several requests, with wrong trees beside right ones."""
    from boring_llm_b200 import StepEntry, TreeEntry
    from boring_llm_b200.sampling.params import SamplingParams, XorShift64
    d = model_folders(name, dtype, 0.02 if dtype == "bfloat16" else 0.25)
    vocab = helpers.TINY[name]["vocab_size"]
    eng = engine(d, dtype)
    run = eng.runner
    prompts = [helpers.random_tokens(vocab, n, n) for n in (21, 50, 15)]
    # the truth, token by token
    truth = []
    for i, p in enumerate(prompts):
        logits = run.step([StepEntry(("t", i), p, [len(p) - 1])])
        out = [int(logits[0].argmax())]
        for _ in range(12):
            out.append(int(run.step([StepEntry(("t", i), [out[-1]], [0])])[0].argmax()))
        truth.append(out)
        run.free_request(("t", i))
    for i, p in enumerate(prompts):
        run.step([StepEntry(i, p, [])])
    for round_ in range(3):                                      # the third is a replay of the captured step
        wrong = lambda t: (t + 1) % vocab
        entries, rows, want = [], [], []
        at = 3 * round_
        for i, out in enumerate(truth):
            # node 0, a wrong chain of three, a wrong branch, the right chain of three (all wrong for the last request)
            right = [out[at + 1], out[at + 2], out[at + 3]] if i < 2 else [wrong(out[at + 1])] * 3
            tokens = [out[at], wrong(out[at + 1]), wrong(out[at + 1]), 0, wrong(wrong(out[at + 1])), right[0], right[1], right[2]]
            parents = [-1, 0, 1, 2, 0, 0, 5, 6]
            if i == 2:
                tokens, parents = tokens[:5], parents[:5]
            entries.append(TreeEntry(i, tokens, parents))
            rows.append((SamplingParams(), XorShift64(0), None))
            want.append(out[at + 1:at + 5] if i < 2 else out[at + 1:at + 2])
        got = run.step_tree(entries, rows)
        assert got == want
        # the last request is brought to where the others are
        for k in (1, 2):
            assert int(run.step([StepEntry(2, [truth[2][at + k]], [0])])[0].argmax()) == truth[2][at + k + 1]
        for i in (0, 1):                                          # of the four sampled tokens three are behind node 0; the fourth node's row goes back
            run.truncate(i, len(prompts[i]) + at + 3)
    run.check_kernels()


def test_step_tree_refuses(model_folders):
    from boring_llm_b200 import StepEntry, TreeEntry
    from boring_llm_b200.engine import OutOfPages, StepError
    from boring_llm_b200.sampling.params import SamplingParams, XorShift64
    eng = engine(model_folders("A", "float32"), "float32", ctx_size=64, max_tokens=64)
    run = eng.runner
    run.step([StepEntry("a", list(range(40)), [])])
    row = (SamplingParams(), XorShift64(0), None)
    for entries, rows in (([], []), ([TreeEntry("a", [1], [-1])], []), ([TreeEntry("b", [1], [-1])], [row]), ([TreeEntry("a", [1, 2], [-1])], [row]),
                          ([TreeEntry("a", [], [])], [row]), ([TreeEntry("a", [1, 2], [-1, 1])], [row]), ([TreeEntry("a", [1, 256], [-1, 0])], [row]),
                          ([TreeEntry("a", [1] * 25, [-1] + list(range(24)))], [row]), ([TreeEntry("a", [1], [-1])] * 2, [row] * 2),
                          ([TreeEntry("a", [1], [-1])], [(SamplingParams(repeat_penalty=1.2), XorShift64(0), None)])):
        with pytest.raises(StepError):
            run.step_tree(entries, rows)
    run.step([StepEntry("b", [1] * 16, [])])
    with pytest.raises(OutOfPages):
        run.step_tree([TreeEntry("a", [1] * 20, [-1] + list(range(19)))], [row])
    assert run.cache.get("a").num_tokens == 40
    run.cache.check()


FAMILIES = ["fezopel", "kavotar", "miforax", "dapuzen", "gipinex", "zuvevik"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("family", FAMILIES)
def test_every_family_forks_and_says_whether_it_drafts(family, dtype):
    """Recurrent state, matrix memories, latent rows, windows, chunks, one number beside a key, a request's last token: a fork goes on as
    its source does. Drafts are refused where a mixer keeps state or attends in a way of its own."""
    import importlib
    import boring_llm_b200 as b
    from boring_llm_b200.sampling.params import SamplingParams
    shapes = importlib.import_module(f"test_{family}_gpu").SHAPES
    for raw in shapes.values():
        cfg = getattr(b, f"{family.capitalize()}Config").from_dict(raw)
        opts = dict(dtype=dtype, ctx_size=128, max_num_seqs=4, max_tokens=1024, device="cuda:0")
        with pytest.raises(ValueError, match="draft_tokens"):
            b.Engine.from_random(cfg, 0, b.EngineOptions(draft_tokens=4, **opts), std=0.2)
        eng = b.Engine.from_random(cfg, 0, b.EngineOptions(debug_poison=True, **opts), std=0.2)
        req = eng.add_request([3, 9, 4, 7, 1, 2, 8] * 5, SamplingParams(n_predict=60, ignore_eos=True))
        while len(req.output) < 9:
            eng.step()
        new = eng.fork(req)
        assert new.output == req.output
        eng.run_until_done()
        if dtype == "float32":
            assert new.output == req.output and len(new.output) == 60
        eng.runner.cache.check()
        assert eng.stats()["live_requests"] == 0


@pytest.mark.parametrize("name", ["A", "C"])
def test_forks_share_their_past(model_folders, name):
    """Greedy forks say what their source says; pages are shared; the copy is made when one of them writes; drawn ones go their own ways."""
    from boring_llm_b200.sampling.params import SamplingParams
    d = model_folders(name, "float32")
    eng = engine(d, "float32", debug_poison=True)
    prompt = helpers.random_tokens(helpers.TINY[name]["vocab_size"], 37, 5)
    alone = eng.generate([prompt], n_predict=30, ignore_eos=True)[0]
    req = eng.add_request(prompt, SamplingParams(n_predict=30, ignore_eos=True))
    with pytest.raises(ValueError):
        eng.fork(req)                                             # its prompt is not computed
    while len(req.output) < 6:
        eng.step()
    eng.drain()
    used = eng.stats()["pages_in_use"]
    twin = eng.fork(req)
    other = eng.fork(req, SamplingParams(n_predict=30, temperature=1.5, seed=9, ignore_eos=True))
    assert eng.stats()["pages_in_use"] == used
    eng.run_until_done()
    assert req.output == twin.output == alone and other.output[:len(alone) // 5] == alone[:len(alone) // 5] and other.output != alone
    with pytest.raises(ValueError):
        eng.fork(req)                                             # it has ended
    eng.runner.cache.check()
    assert eng.stats()["pages_in_use"] == [0] * len(used)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "C"])
def test_several_answers_to_a_prompt(model_folders, name, dtype):
    """`generate(n=)`: the answers are those of separate requests with their seeds; more answers than slots; a prompt of one token."""
    eng = engine(model_folders(name, dtype), dtype, max_num_seqs=3)
    vocab = helpers.TINY[name]["vocab_size"]
    prompts = [helpers.random_tokens(vocab, n, n) for n in (33, 1, 50)]
    drawn = dict(n_predict=12, temperature=0.8, top_p=0.9, ignore_eos=True)
    got = eng.generate(prompts, n=4, seed=20, **drawn)
    assert len(got) == 12 and all(len(o) == 12 for o in got)
    if dtype == "float32":
        for i, p in enumerate(prompts):
            for k in range(4):
                assert got[4 * i + k] == eng.generate([p], seed=20 + 4 * i + k, **drawn)[0]
    eng.runner.cache.check()
    s = eng.stats()
    assert s["live_requests"] == 0 and s["pages_in_use"] == [0] * len(s["pages_in_use"])
    with pytest.raises(ValueError):
        eng.generate([[1]], n=0)


def test_drafts_and_forks_together(model_folders):
    d = model_folders("A", "float32")
    prompt = repeating("A", 30, 3)
    want = engine(d, "float32").generate([prompt], n=3, n_predict=25, temperature=0.7, seed=2, ignore_eos=True)
    eng = engine(d, "float32", draft_tokens=10, debug_poison=True)
    assert eng.generate([prompt], n=3, n_predict=25, temperature=0.7, seed=2, ignore_eos=True) == want
    eng.runner.cache.check()


def test_a_source_that_ends_before_the_copy_is_made(model_folders):
    """A page that a fork goes on in a copy of is given back by its source, and poisoned, before the step that copies it."""
    from boring_llm_b200 import StepEntry
    eng = engine(model_folders("A", "float32"), "float32", debug_poison=True)
    run = eng.runner
    prompt = helpers.random_tokens(256, 21, 4)
    run.step([StepEntry("a", prompt, [])])
    want = run.step([StepEntry("a", [7], [0])]).clone()
    run.truncate("a", 21)
    run.fork_request("a", "b")
    assert run.cache.reserve("b", 1) and run.cache.has_copies         # as a scheduler reserves ahead of the step
    run.free_request("a")
    got = run.step([StepEntry("c", prompt[:5], []), StepEntry("b", [7], [0])])
    assert not run.cache.has_copies and torch.equal(got, want)
    run.cache.check()


def test_fork_hands_on_what_ends_meanwhile(model_folders):
    """A request that ends in the step that was launched ahead is among those that the next step returns."""
    from boring_llm_b200.sampling.params import SamplingParams
    eng = engine(model_folders("A", "bfloat16"), "bfloat16")
    long, short = (eng.add_request([5, 6, 7], SamplingParams(n_predict=n, ignore_eos=True)) for n in (40, 12))
    done = []
    while len(short.output) < 11:
        done += eng.step()
    assert eng._inflight is not None and not done
    new = eng.fork(long)
    while not done:
        done += eng.step()
    assert short in done and short.finish_reason == "length"
    eng.run_until_done()
    assert len(new.output) == len(long.output) == 40


@pytest.mark.parametrize("rows", [3, 40, 70, 300])
@pytest.mark.parametrize("H,KV,dh,d,layout", [(4, 2, 64, 256, 0), (14, 2, 64, 896, 0), (4, 2, 32, 128, 1)])
def test_cache_rows_beside_positions(rows, H, KV, dh, d, layout):
    """The kernels that rotate and write keys and values put them where `cache_rows` says, rotated by `positions`."""
    from boring_llm_b200.kernels import ops as o
    g = torch.Generator(device="cuda").manual_seed(rows)
    width, page, pages = (H + 2 * KV) * dh, 16, rows // 16 + 9
    positions = torch.randint(0, 900, (rows,), generator=g, device="cuda", dtype=torch.int32)
    cache_rows = torch.randperm(rows, generator=g, device="cuda").to(torch.int32) + 5
    tok_req = torch.zeros(rows, dtype=torch.int32, device="cuda")
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(1, -1)
    inv = (10000.0 ** (-torch.arange(dh // 2, device="cuda").float() / (dh // 2)))
    place = lambda c, r: c[table[0, (r // page).long()].long(), :, (r % page).long()]       # [rows, KV, dh]
    for dtype in (torch.float32, torch.bfloat16):
        qkv = torch.randn(rows, width, generator=g, device="cuda")
        outs = []
        for kw in ({}, {"cache_rows": cache_rows}):
            q = torch.empty(rows, H * dh, dtype=dtype, device="cuda")
            k = torch.zeros(max(pages, 60), KV, page, dh, dtype=dtype, device="cuda")
            v = torch.zeros_like(k)
            wide = torch.arange(60, dtype=torch.int32, device="cuda").view(1, -1)
            if kw:
                o.rope_kv_write(qkv, positions, tok_req, table, inv, dh // 2, 1.0, q, k, v, H, KV, dh, layout, **kw)
                outs.append((q, place(k, cache_rows), place(v, cache_rows)))
            else:                                                 # each row as a request of its own: positions may come twice
                own = torch.arange(rows, dtype=torch.int32, device="cuda")
                each = torch.empty(rows, KV, dh, dtype=dtype, device="cuda"), torch.empty(rows, KV, dh, dtype=dtype, device="cuda")
                for t in range(rows):
                    o.rope_kv_write(qkv[t:t + 1].contiguous(), positions[t:t + 1].contiguous(), tok_req[:1], wide, inv, dh // 2, 1.0, q[t:t + 1], k, v,
                                    H, KV, dh, layout)
                    p = int(positions[t])
                    each[0][t], each[1][t] = k[p // page, :, p % page], v[p // page, :, p % page]
                outs.append((q, *each))
        for a, b in zip(*outs):
            assert torch.equal(a, b)
    # the fused kernel of few rows gives with `cache_rows` what it gives without, elsewhere
    if rows <= 64:
        x, nw = torch.randn(rows, d, generator=g, device="cuda"), torch.rand(d, generator=g, device="cuda") + 0.5
        w = (torch.randn(width, d, generator=g, device="cuda") / d ** 0.5).bfloat16()
        own = torch.arange(rows, dtype=torch.int32, device="cuda")
        got = []
        for cr, pos in ((None, cache_rows), (cache_rows, cache_rows), (cache_rows, positions)):
            q = torch.empty(rows, H * dh, dtype=torch.bfloat16, device="cuda")
            k = torch.zeros(max(pages, 60), KV, page, dh, dtype=torch.bfloat16, device="cuda")
            v = torch.zeros_like(k)
            o.norm_qkv_rope(x, nw, 1e-6, w, None, pos.contiguous(), tok_req, table, inv, 1.0, q, k, v, H, KV, dh, layout, cache_rows=cr)
            got.append((q, k, v))
        assert all(torch.equal(a, b) for a, b in zip(got[0], got[1]))
        assert torch.equal(got[1][2], got[2][2]) and not torch.equal(got[1][1], got[2][1])      # values alike, keys turned otherwise
