"""What the host does around a step of drafted trees: what it keeps, gives back, pads, and what a failure leaves behind."""
import pytest
import torch

import drafted_steps as steps
from boring_llm_b200 import EngineOptions, StepEntry, TreeEntry
from boring_llm_b200.cache import CacheManager, PagedKVSpec
from boring_llm_b200.engine import OutOfPages, StepError
from boring_llm_b200.engine.scheduler import FINISHED, RUNNING, AdmissionError, Scheduler
from boring_llm_b200.kernels import KernelError, ops
from boring_llm_b200.sampling.params import SamplingParams, XorShift64

FULL, WIN = PagedKVSpec(1, 4, 0), PagedKVSpec(1, 4, 20)


def chain(rid, n, first=1):
    return TreeEntry(rid, [first] * n, [-1] + list(range(n - 1)))


def row(**kw):
    params = SamplingParams(**kw)
    return params, XorShift64(params.seed), None


def gave_up():
    raise KernelError("a block gave up on a bounded wait (made up by the test)")


# ---- a step that fails ---------------------------------------------------------------------------------------------------


def test_a_failed_tree_step_changes_nothing(monkeypatch):
    """A wait that ran out is seen before tokens are committed and generators advance: cache, pages and random numbers are as they were."""
    steps.host(monkeypatch, steps.whole_chains)
    run = steps.runner()
    rows = []
    for i, n in enumerate((20, 16)):
        steps.put(run, i, n)
        rows.append(row(temperature=1.0, seed=i))
    states, free = [r[1].state for r in rows], run.cache.free_pages()
    run.check_kernels = gave_up
    for _ in range(2):
        with pytest.raises(KernelError):
            run.step_tree([chain(0, 30), chain(1, 5)], rows)
        assert [run.cache.get(i).num_tokens for i in (0, 1)] == [20, 16] and run.cache.free_pages() == free
        assert [r[1].state for r in rows] == states and run.accepted == run.drafted == run.steps == 0
        run.cache.check()
    run.check_kernels = lambda: None
    assert run.step_tree([chain(0, 30), chain(1, 5)], rows) == [[7] * 30, [7] * 5]
    assert [run.cache.get(i).num_tokens for i in (0, 1)] == [50, 21]


def test_a_tree_step_that_accepts_nothing_changes_nothing(monkeypatch):
    """No request's tokens are committed when the answer of another one is impossible."""
    def says(batch, R):
        counts, tokens = steps.only_node_0(batch, R)
        counts[1] = 0
        return counts, tokens
    steps.host(monkeypatch, says)
    run = steps.runner()
    rows = [row(temperature=1.0, seed=i) for i in range(3)]
    for i in range(3):
        steps.put(run, i, 16)
    states, free = [r[1].state for r in rows], run.cache.free_pages()
    with pytest.raises(StepError):
        run.step_tree([chain(i, 4) for i in range(3)], rows)
    assert [run.cache.get(i).num_tokens for i in range(3)] == [16] * 3 and run.cache.free_pages() == free
    assert [r[1].state for r in rows] == states and run.accepted == run.drafted == 0
    run.cache.check()


def test_the_engine_goes_on_after_a_failed_drafted_step(monkeypatch):
    """The requests' records and the cache agree after the error, and the next step feeds the same token at the same place."""
    steps.host(monkeypatch, steps.whole_chains)
    eng = steps.engine(monkeypatch)
    req = steps.hold(eng, [1, 2, 3, 1, 2, 3], SamplingParams(n_predict=40, ignore_eos=True))
    eng.runner.check_kernels = gave_up
    with pytest.raises(KernelError):
        eng.step()
    eng.runner.cache.check()
    assert req.state == RUNNING and req.output == [1]
    assert eng.runner.cache.get(req.request_id).num_tokens == req.num_computed == 6
    eng.runner.check_kernels = lambda: None
    assert eng.step() == []
    assert eng.runner.cache.get(req.request_id).num_tokens == req.num_computed == 6 + len(req.output) - 1 > 6


@pytest.mark.parametrize("draft_tokens", [0, 8])
def test_a_failed_step_that_has_committed_ends_its_requests(monkeypatch, draft_tokens):
    """A step without drafts has committed its tokens by the time that its kernels are checked: its requests end with an error, the others stay."""
    steps.host(monkeypatch)
    eng = steps.engine(monkeypatch, draft_tokens=draft_tokens, lookahead=False)

    def step_and_sample(entries, rows, sampler):
        for e in entries:
            eng.runner.cache.commit(e.request_id, len(e.tokens))
        return [5] * len(rows)
    eng.runner.step_and_sample = step_and_sample
    req = steps.hold(eng, [1, 2, 3, 4], SamplingParams(n_predict=40, ignore_eos=True, repeat_penalty=1.1))
    eng.runner.check_kernels = gave_up
    with pytest.raises(KernelError):
        eng.step()
    eng.runner.cache.check()
    assert req.state == FINISHED and req.finish_reason == "error" and not eng.scheduler.has_work()
    assert eng.runner.cache.live_requests() == []
    # one that fails before anything is committed leaves its requests as they were
    eng.runner.check_kernels = lambda: None
    req = steps.hold(eng, [1, 2, 3, 4], SamplingParams(n_predict=40, ignore_eos=True, repeat_penalty=1.1))
    eng.runner.step_and_sample = lambda *a: gave_up()
    with pytest.raises(KernelError):
        eng.step()
    assert req.state == RUNNING and req.num_computed == eng.runner.cache.get(req.request_id).num_tokens == 4
    eng.runner.step_and_sample = step_and_sample
    assert eng.step() == [] and req.output[-1] == 5


def test_a_failed_drain_ends_the_requests_of_the_step_ahead(monkeypatch):
    """`drain` reads a step whose tokens are committed: when that fails its requests end, as they do inside `step`."""
    steps.host(monkeypatch)
    eng = steps.engine(monkeypatch, draft_tokens=0)
    req = steps.hold(eng, [1, 2, 3, 4], SamplingParams(n_predict=40, ignore_eos=True))
    sched = eng.scheduler.schedule()
    eng.runner.cache.commit(req.request_id, 1)                    # as launching the step does
    eng._inflight = (sched, None)
    eng.runner.collect_decode = lambda pending: [5]
    eng.runner.check_kernels = gave_up
    with pytest.raises(KernelError):
        eng.fork(req)
    eng.runner.cache.check()
    assert req.finish_reason == "error" and eng.runner.cache.live_requests() == [] and eng._inflight is None


# ---- pages ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("specs", [[FULL], [FULL, WIN]])
def test_pages_of_rejected_nodes_go_back(monkeypatch, specs):
    """A rejected tree leaves as many pages free as a step of one token."""
    steps.host(monkeypatch)
    run, plain = steps.runner(specs, max_tokens=640), CacheManager(specs, 16, 640, 16)
    for i, n in enumerate((16, 31, 32, 5)):
        steps.put(run, i, n)
        plain.add_request(i)
        assert plain.reserve(i, n)
        plain.commit(i, n)
    for _ in range(20):
        run.step_tree([chain(i, 40 + i) for i in range(4)], [row() for _ in range(4)])
        for i in range(4):
            assert plain.reserve(i, 1)
            plain.commit(i, 1)
        assert run.cache.free_pages() == plain.free_pages()
        run.cache.check()


def test_pages_of_accepted_nodes_stay(monkeypatch):
    steps.host(monkeypatch, steps.whole_chains)
    run = steps.runner()
    steps.put(run, 0, 20)
    run.step_tree([chain(0, 30)], [row()])
    assert run.cache.get(0).num_tokens == 50 and len(run.cache.get(0).tables[0]) == 4
    run.cache.check()


def test_forks_that_write_in_one_step_need_a_copy_less(monkeypatch):
    """Of all owners of a page the last that writes keeps it: a step of all of them needs one copy less than it has owners."""
    steps.host(monkeypatch)
    for step in ("tokens", "trees"):
        run = steps.runner(max_tokens=64)                         # four pages
        run.storage.copy_pages = lambda: run.cache.take_copies()
        steps.put(run, "a", 20)
        for new in ("b", "c"):
            run.cache.fork("a", new)
        assert run.cache.free_pages() == [2]                      # copies for two of the three
        if step == "trees":
            run.step_tree([chain(r, 2) for r in "abc"], [row() for _ in "abc"])
        else:
            run._prepare([StepEntry(r, [1], [0]) for r in "abc"])
        run.cache.check()
        assert run.cache.free_pages() == [0] and len({run.cache.get(r).tables[0][1] for r in "abc"}) == 3
        # an owner that does not write keeps the page: every writer needs a copy
        run = steps.runner(max_tokens=48)
        run.storage.copy_pages = lambda: run.cache.take_copies()
        steps.put(run, "a", 20)
        for new in ("b", "c"):
            run.cache.fork("a", new)
        with pytest.raises(OutOfPages):
            if step == "trees":
                run.step_tree([chain(r, 2) for r in "bc"], [row() for _ in "bc"])
            else:
                run._prepare([StepEntry(r, [1], [0]) for r in "bc"])
        assert run.cache.free_pages() == [1] and not run.cache.has_copies
        run.cache.check()


# ---- padded steps ----------------------------------------------------------------------------------------------------------


def test_padded_tree_steps_share_their_shapes(monkeypatch):
    """Eight requests with up to 31 drafted tokens each, step by step: a shape for each padded number of nodes, captured once each."""
    import random
    rng = random.Random(0)
    steps.host(monkeypatch)
    run = steps.runner(max_num_seqs=64, max_tokens=64 * 256)
    for i in range(32):
        steps.put(run, i, 20)
    for _ in range(300):
        run.step_tree([chain(i, rng.randint(1, 32)) for i in range(8)], [row()] * 8)
        for i in range(8):
            run.truncate(i, 20)
    assert len(set(steps.Batch.made)) == len(steps.Batch.made) <= 7
    assert len(set(steps.Batch.captured)) == len(steps.Batch.captured) <= 7
    steps.Batch.made.clear()
    for requests in list(range(1, 33)) * 4:
        run.step_tree([chain(i, rng.randint(1, 512 // requests if requests > 8 else 32)) for i in range(requests)], [row()] * requests)
        for i in range(requests):
            run.truncate(i, 20)
    assert len(steps.Batch.made) == len(set(steps.Batch.made)) <= 40                  # none was thrown out and made again


@pytest.mark.parametrize("ctx_size,page,counts", [(ctx_size, page, counts) for ctx_size, page in ((256, 16), (24, 1), (40, 5), (64, 64))
                                                  for counts in ([1], [8], [3, 5, 1], [16], [13] * 5, [1] * 16, [20, 20, 20, 7]) if max(counts) < ctx_size - 3])
def test_the_padding_of_a_tree_step_is_a_step_of_its_own(monkeypatch, counts, ctx_size, page):
    """Padding nodes stand in requests of at most 64 on the spare page: each sees itself, in a row that it writes, that its table holds and that
    lies inside its request's length; no request of the step is touched by them."""
    checked = []

    def says(batch, R):
        h, T, live = batch.h, batch.T, sum(counts)
        begin, ends = h["cu_q"][:-1], h["cu_q"][1:]
        n = ends - begin
        assert h["cu_q"][0] == 0 and ends[-1] == T and (n >= 0).all() and (n <= 64).all()
        assert list(n[:R]) == counts and ends[R - 1] == live
        for t in range(live, T):
            r = int(h["tok_req"][t])
            assert r >= R and begin[r] <= t < ends[r]
            node, c = t - begin[r], h["ctx_len"][r] - n[r]
            assert int(h["mask"][t]) == 1 << int(node) and c == 0
            at = int(h["cache_rows"][t])
            assert at == c + node and h["positions"][t] == 0 and h["slots"][r] == run.storage.trash_slot
            assert at // page < h["tables"].shape[2] and (h["tables"][:, r, at // page] == run.storage.trash_page).all()
        for r in range(R, len(n)):
            assert h["ctx_len"][r] >= n[r]
        checked.append(T)
        return steps.only_node_0(batch, R)
    steps.host(monkeypatch, says)
    run = steps.runner(ctx_size=ctx_size, page_size=page)
    for i in range(len(counts)):
        steps.put(run, i, 3)
    for _ in range(3):
        run.step_tree([chain(i, n) for i, n in enumerate(counts)], [row()] * len(counts))
        for i in range(len(counts)):
            run.truncate(i, 3)
    assert len(checked) == 3 and checked[0] % 16 == 0 and checked[0] - sum(counts) < 64


# ---- requests and options ------------------------------------------------------------------------------------------------


def test_what_ended_in_front_of_a_refused_fork_is_still_handed_out(monkeypatch):
    """A request that ends in the step that a fork reads first is work until a step has returned it, also when the fork is refused."""
    steps.host(monkeypatch)
    eng = steps.engine(monkeypatch, draft_tokens=0)
    req = steps.hold(eng, [1, 2, 3, 4], SamplingParams(n_predict=2, ignore_eos=True))
    sched = eng.scheduler.schedule()
    eng.runner.cache.commit(req.request_id, 1)
    eng._inflight = (sched, None)
    eng.runner.collect_decode = lambda pending: [5]
    with pytest.raises(ValueError):
        eng.fork(req)
    assert req.state == FINISHED and eng.scheduler.has_work()
    assert eng.step() == [req] and not eng.scheduler.has_work() and eng.step() == []
    # `run_until_done` takes it as well
    req = steps.hold(eng, [1, 2, 3, 4], SamplingParams(n_predict=2, ignore_eos=True))
    sched = eng.scheduler.schedule()
    eng.runner.cache.commit(req.request_id, 1)
    eng._inflight = (sched, None)
    with pytest.raises(ValueError):
        eng.fork(req)
    eng.run_until_done()
    assert not eng.scheduler.has_work()


def test_positional_options_stand_where_they_stood():
    o = EngineOptions("bfloat16", 16, 0, 4096, 64, 2048, 512, True, 2, True, True, "cuda:1")
    assert o.debug_poison is True and o.device == "cuda:1" and o.draft_tokens == 0


def test_a_finished_request_keeps_no_drafting_index(monkeypatch):
    steps.host(monkeypatch, steps.whole_chains)
    eng = steps.engine(monkeypatch)
    req = steps.hold(eng, [1, 2, 3, 1, 2, 3], SamplingParams(n_predict=3, ignore_eos=True))
    assert eng.step() == [req] and req.output == [1, 7, 7] and req.history is None
    req = steps.hold(eng, [1, 2, 3, 1, 2, 3], SamplingParams(n_predict=30, ignore_eos=True))
    assert eng.step() == [] and req.history is not None
    eng.scheduler.abort(req.request_id)
    assert req.history is None and eng.scheduler.finished[req.request_id] is req


@pytest.mark.parametrize("pairs", [[(1, 2, 3), (4,)], [(0, 1), (2, 3, 4), (5,)], [(), (0, 1, 2, 3)]])
def test_copies_that_are_no_pairs_are_refused(pairs):
    """As many numbers as pairs have, but not two by two."""
    with pytest.raises(KernelError, match="pairs"):
        ops.copy_blocks([torch.zeros(2, 9, 4)], pairs)


@pytest.mark.parametrize("requests,budget,each", [(1, 2048, 64), (8, 2048, 64), (9, 2048, 56), (64, 2048, 8), (64, 256, 4), (600, 2048, None)])
def test_drafts_of_a_step_stay_within_a_captured_one(requests, budget, each):
    """Every node has a row of logits: however many requests draft, a step has no more nodes than a captured one takes."""
    o = EngineOptions(ctx_size=256, max_num_seqs=requests, max_tokens=requests * 32, max_num_batched_tokens=max(budget, 6 * requests), prefill_chunk=6, draft_tokens=63)
    s = Scheduler(CacheManager([FULL], 16, o.capacity_tokens, requests), o)
    for i in range(requests):
        s.add(i, [1, 2, 3, 1, 2, 3], SamplingParams(n_predict=100))
    while s.waiting:
        step = s.schedule()
        for e in step.entries:
            s.cache.commit(e.request_id, len(e.tokens))
        s.apply(step, [1 if len(e.tokens) > 1 else 2 for e, said in zip(step.entries, step.samples) if said])
    s.options.max_num_batched_tokens = max(budget, requests)
    trees = s.draft(s.schedule())
    if each is None:
        assert trees is None
    else:
        assert [len(t) for t, _ in trees] == [each] * requests and requests * each <= 512
