"""Drafted trees and forks on the host: drafting, masks, the scheduler's records, shared pages and their copies."""
import random

import pytest

from boring_llm_b200 import EngineOptions
from boring_llm_b200.cache import CacheError, CacheManager, PagedKVSpec, StateSpec
from boring_llm_b200.engine.draft import History, tree_masks
from boring_llm_b200.engine.scheduler import RUNNING, AdmissionError, Scheduler
from boring_llm_b200.sampling.params import SamplingParams

FULL = PagedKVSpec(2, 16, 0)
WIN = PagedKVSpec(2, 16, 20)


def history(tokens, **kw):
    h = History(**kw)
    h.extend(tokens)
    return h


def test_masks_are_ancestors():
    assert tree_masks([-1, 0, 1, 0, 3, 2]) == [0b1, 0b11, 0b111, 0b1001, 0b11001, 0b100111]
    assert tree_masks([]) == []


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, -1], [-1, 0, 3], [-1] + list(range(64))])
def test_what_is_no_tree_is_refused(parents):
    with pytest.raises(ValueError):
        tree_masks(parents)


def test_draft_follows_the_longest_run_that_came_before():
    assert history([1, 2, 3, 4, 9, 2, 3]).draft(8) == ([3, 4, 9, 2, 3, 4, 9, 2], [-1, 0, 1, 2, 3, 4, 5, 6])      # goes on from itself
    assert history([1, 2, 3, 4, 9, 2, 3]).draft(3) == ([3, 4, 9], [-1, 0, 1])
    assert history([1, 2, 3, 4, 9, 2, 3]).draft(8, depth=1) == ([3, 4], [-1, 0])
    # the latest place is the chain, an earlier one branches off where it differs
    assert history([5, 1, 7, 8, 5, 1, 7, 9, 5, 1]).draft(16, depth=3) == ([1, 7, 9, 5, 8, 5], [-1, 0, 1, 2, 1, 4])
    assert history([5, 1, 7, 8, 5, 1, 7, 9, 5, 1]).draft(16, branches=1, depth=3) == ([1, 7, 9, 5], [-1, 0, 1, 2])
    assert history([1, 2, 3]).draft(8) == ([3], [-1])
    assert history([4, 4, 4, 4]).draft(4) == ([4, 4, 4, 4], [-1, 0, 1, 2])
    with pytest.raises(ValueError):
        history([]).draft(4)


def test_history_grows_token_by_token():
    rng = random.Random(0)
    tokens = [rng.randrange(4) for _ in range(200)]
    whole, grown = history(tokens), History()
    for t in tokens:
        grown.extend([t])
    assert whole.draft(64) == grown.draft(64)
    got, parents = grown.draft(64)
    tree_masks(parents)
    assert got[0] == tokens[-1] and len(got) == len(parents) > 4
    children = {}
    for i, (t, p) in enumerate(zip(got, parents)):
        assert children.setdefault((p, t), i) == i              # no node has two children with one token


def scheduler(**kw):
    options = EngineOptions(ctx_size=kw.pop("ctx_size", 64), max_num_seqs=4, max_tokens=256, draft_tokens=kw.pop("draft_tokens", 8), **kw)
    return Scheduler(CacheManager([FULL], 16, 256, 4), options)


def decoding(s, prompt, n_predict=30, first=None, **kw):
    req = s.add(len(s.running), prompt, SamplingParams(n_predict=n_predict, **kw))
    step = s.schedule()
    for e in step.entries:
        s.cache.commit(e.request_id, len(e.tokens))
    s.apply(step, [prompt[0] if first is None else first] * sum(step.samples))
    return req


def test_drafts_of_a_step():
    s = scheduler()
    req = decoding(s, [1, 2, 3, 1, 2, 3])
    step = s.schedule()
    assert s.draft(step) == [([1, 2, 3, 1, 2, 3, 1, 2, 3], [-1, 0, 1, 2, 3, 4, 5, 6, 7])]
    said = [[2, 3, 9]]
    s.cache.commit(req.request_id, 3)
    assert s.apply_drafted(step, said) == []
    assert req.output == [1, 2, 3, 9] and req.num_computed == 9 and req.remaining == 1
    assert s.schedule().entries[0].tokens == [9]


def test_drafts_end_with_the_request():
    s = scheduler()
    req = decoding(s, [1, 2, 3, 1, 2, 3], n_predict=3)
    step = s.schedule()
    assert s.draft(step) == [([1, 2], [-1, 0])]                   # one more token may follow the next one
    assert s.apply_drafted(step, [[2, 3, 3]]) == [req]
    assert req.output == [1, 2, 3] and req.finish_reason == "length" and req.request_id not in s.cache
    s = scheduler()
    req = decoding(s, [1, 2, 3, 1, 2, 3], eos_token_ids=(2,))
    step = s.schedule()
    assert s.apply_drafted(step, [[2, 3]]) == [req] and req.output == [1, 2] and req.finish_reason == "stop"
    s = scheduler(ctx_size=9)
    req = decoding(s, [1, 2, 3, 1, 2, 3])
    tokens, _ = s.draft(s.schedule())[0]
    assert len(tokens) <= 3                                       # rows 6, 7 and 8


def test_steps_that_are_not_drafted():
    s = scheduler()
    decoding(s, [1, 2, 3, 4], first=9)
    assert s.draft(s.schedule()) is None                          # nothing has come before
    s = scheduler()
    decoding(s, [1, 2, 3, 1, 2, 3], repeat_penalty=1.1)
    assert s.draft(s.schedule()) is None
    s = scheduler()
    s.add("p", [1, 2, 1, 2], SamplingParams())
    assert s.draft(s.schedule()) is None                          # a prompt
    with pytest.raises(ValueError):
        EngineOptions(draft_tokens=64)


# ---- shared pages ------------------------------------------------------------------------------------------------------


def test_fork_shares_and_the_writer_copies():
    m = CacheManager([FULL], 16, 160, 4)
    m.add_request("a")
    assert m.reserve("a", 40)
    m.commit("a", 40)
    m.fork("a", "b")
    m.check()
    assert m.get("b").tables == m.get("a").tables == [[0, 1, 2]] and m.free_pages() == [7]
    assert m.pages_needed("b", 1) == [1] and m.pages_needed("b", 9) == [2]
    assert m.reserve("b", 1)
    m.check()
    assert m.get("b").tables == [[0, 1, 3]] and m.take_copies() == [[(2, 3)]] and not m.has_copies
    assert m.reserve("a", 1) and m.get("a").tables == [[0, 1, 2]] and not m.has_copies      # the page is a's alone by now
    m.free("a")
    m.check()
    assert m.free_pages() == [7]                                  # page 2 is back; 0 and 1 are b's
    m.free("b")
    m.check()
    assert m.free_pages() == [10]


def test_fork_at_a_page_boundary_and_of_a_prefix():
    m = CacheManager([FULL], 16, 160, 4)
    m.add_request("a")
    m.reserve("a", 32)
    m.commit("a", 32)
    m.fork("a", "b")
    assert m.reserve("b", 1) and m.get("b").tables == [[0, 1, 2]] and not m.has_copies
    m.fork("a", "c", 20)
    assert m.get("c").num_tokens == 20 and m.get("c").tables == [[0, 1]]
    m.truncate("b", 10)                                           # back into a shared page: b goes on in a copy
    m.check()
    assert m.reserve("b", 1) and m.take_copies() == [[(0, 2)]]
    for bad in (33, -1):
        with pytest.raises(CacheError):
            m.fork("a", "d", bad)
    with pytest.raises(CacheError):
        m.fork("a", "b")
    m.check()


def test_fork_needs_room_for_the_copy_when_it_writes():
    m = CacheManager([FULL], 16, 32, 4)
    m.add_request("a")
    m.reserve("a", 20)
    m.commit("a", 20)
    m.fork("a", "b")
    assert not m.can_reserve("b", 1) and not m.reserve("b", 1) and m.pages_short("b", 1) == 1 and not m.has_copies
    m.free("a")
    assert m.reserve("b", 1) and not m.has_copies
    m.check()


def test_fork_with_windows_and_state():
    m = CacheManager([FULL, WIN, StateSpec((3,))], 16, 160, 4)
    m.add_request("a")
    for _ in range(50):
        m.reserve("a", 1)
        m.commit("a", 1)
    assert m.get("a").tables[1][:1] == [-1]
    with pytest.raises(CacheError):
        m.fork("a", "b", 49)                                      # state holds all tokens
    m.fork("a", "b")
    m.check()
    assert m.reserve("b", 1) and [len(c) for c in m.take_copies()] == [1, 1]
    m = CacheManager([WIN], 16, 160, 4)
    m.add_request("a")
    for _ in range(50):
        m.reserve("a", 1)
        m.commit("a", 1)
    with pytest.raises(CacheError):
        m.fork("a", "b", 20)                                      # the window has passed


def test_random_forks_lose_no_page():
    rng = random.Random(3)
    m = CacheManager([FULL, WIN], 16, 400, 8)
    m.add_request(0)
    m.reserve(0, 5)
    m.commit(0, 5)
    names = 1
    for _ in range(4000):
        live = m.live_requests()
        kind = rng.random()
        if kind < 0.15 and m.has_free_slot():
            src = rng.choice(live) if live else None
            if src is None:
                m.add_request(names)
            else:
                m.fork(src, names)
            names += 1
        elif kind < 0.25 and len(live) > 1:
            m.free(rng.choice(live))
        elif kind < 0.3 and live:
            r = rng.choice(live)
            try:
                m.truncate(r, rng.randint(0, m.get(r).num_tokens))
            except CacheError:
                pass
        elif live:
            r, n = rng.choice(live), rng.randint(1, 20)
            before = [list(t) for t in m.get(r).tables]
            if m.reserve(r, n):
                for gi, pairs in enumerate(m.take_copies()):
                    assert len(pairs) <= 1
                    for s, d in pairs:
                        at = m.get(r).num_tokens // 16
                        assert before[gi][at] == s and m.get(r).tables[gi][at] == d
                for g, t in zip(m.paged_groups, m.get(r).tables):
                    for i in range(m.get(r).num_tokens // 16, len(t)):
                        assert t[i] < 0 or not g.pool.is_shared(t[i])        # what is written next is the request's own
                m.commit(r, rng.randint(0, n))
            else:
                m.free(r)
        m.check()


def test_scheduler_forks_running_requests():
    s = scheduler()
    req = decoding(s, [1, 2, 3, 4])
    new = s.fork(req, "f", SamplingParams(n_predict=20, seed=7), 3, 0)
    assert new.state == RUNNING and new.output == [] and new.remaining == 1 and s.running == [req, new]
    step = s.schedule()
    assert [(e.request_id, e.tokens) for e in step.entries] == [(0, [1]), ("f", [4])] and step.samples == [True, True]
    for n_keep, n_output, n_predict in ((5, 1, 20), (4, 0, 20), (4, 1, 1)):
        with pytest.raises(AdmissionError):
            s.fork(req, "g", SamplingParams(n_predict=n_predict), n_keep, n_output)
    s.abort(0)
    with pytest.raises(AdmissionError):
        s.fork(req, "g", SamplingParams(n_predict=20), 3, 0)
    s.cache.check()
