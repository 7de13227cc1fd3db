"""Steps of drafted trees without a GPU: a runner and an engine around a model that is only shapes, whose steps say what a test tells
them to say. The host's part of a step (checks, pages, buffers, what is kept of it) is the real one."""
import numpy as np
import torch

from boring_llm_b200 import EngineOptions
from boring_llm_b200.cache import PagedKVSpec
from boring_llm_b200.engine import engine as engine_module
from boring_llm_b200.engine import runner as runner_module


class Shapes:
    """What a runner asks a model for."""
    vocab_size, graph_safe, takes_trees = 256, True, True

    def __init__(self, specs=None):
        self.specs = [PagedKVSpec(1, 4, 0)] if specs is None else specs

    def cache_specs(self):
        return self.specs


class Batch(runner_module._TreeBatch):
    """A step whose kernels do nothing. `says(batch, R)` gives (counts, tokens [R, 64]); `made` are the shapes of all batches."""
    made, captured, says = [], [], None

    def __init__(self, runner, T, R):
        super().__init__(runner, T, R)
        Batch.made.append((T, R))

    def run(self, runner):
        pass

    def capture(self, runner):
        Batch.captured.append((self.T, self.R))
        self.graph = type("Graph", (), {"replay": lambda self: None})()

    def read(self, R):
        return Batch.says(self, R)


def only_node_0(batch, R):
    """Every request's first node alone is accepted; the model says 7 behind it."""
    tokens = np.full((R, 64), -1, dtype=np.int32)
    tokens[:, 0] = 7
    return np.ones(R, dtype=np.int32), tokens


def whole_chains(batch, R):
    """Every node is accepted (trees that are chains); the model says 7 behind each."""
    n = np.diff(batch.h["cu_q"][:R + 1]).astype(np.int32)
    tokens = np.full((R, 64), -1, dtype=np.int32)
    for r in range(R):
        tokens[r, :n[r]] = 7
    return n, tokens


def host(monkeypatch, says=only_node_0):
    """From here on batches of drafted trees are `Batch`es in ordinary memory."""
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    monkeypatch.setattr(runner_module, "_TreeBatch", Batch)
    Batch.made, Batch.captured, Batch.says = [], [], staticmethod(says)


def options(**kw):
    o = dict(ctx_size=256, max_num_seqs=16, max_tokens=4096, device="cpu")
    o.update(kw)
    return EngineOptions(**o)


def runner(specs=None, **kw):
    run = runner_module.ModelRunner(Shapes(specs), options(**kw))
    run.check_kernels = lambda: None
    return run


def engine(monkeypatch, **kw):
    """An engine whose prompts are computed by nobody: `hold` puts requests where their prompts are done."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    kw.setdefault("draft_tokens", 8)
    eng = engine_module.Engine((type("Config", (), {})(), Shapes()), options(**kw))
    eng.runner.check_kernels = lambda: None
    return eng


def hold(eng, prompt, params):
    """A request that runs, its prompt computed and its first token (the prompt's first one again) sampled."""
    req = eng.add_request(prompt, params)
    step = eng.scheduler.schedule()
    for e in step.entries:
        eng.runner.cache.commit(e.request_id, len(e.tokens))
    eng.scheduler.apply(step, [r.prompt[0] if r is req else 7 for r in step.requests])
    return req


def put(run, rid, n):
    """A live request with n committed tokens."""
    run.cache.add_request(rid)
    assert run.cache.reserve(rid, n)
    run.cache.commit(rid, n)
