"""What the operators of drafted trees and forked requests refuse, before a device is touched; the line of work that the attention's
blocks share out."""
import array
import ctypes

import numpy as np
import pytest
import torch

from boring_llm_b200.kernels import KernelError, library, ops
from tree_cases import TreeStep


def step(**changes):
    s = TreeStep([3, 2], [5, 9], 4, 2, 16, 16, torch.float32, 0)
    args = dict(q=s.q, k_cache=s.k, v_cache=s.v, cu_q=s.cu_q, ctx_len=s.ctx_len, mask=s.mask, block_table=s.table, out=torch.empty_like(s.q), H=4,
                window=0, scale=0.25)
    args.update({k: v(args[k]) if callable(v) else v for k, v in changes.items()})
    return args


@pytest.mark.parametrize("change,what", [
    (dict(mask=lambda t: t.int()), "mask"), (dict(mask=lambda t: t[:-1]), "q"), (dict(cu_q=lambda t: t[:-1]), "cu_q"), (dict(cu_q=lambda t: t.long()), "cu_q"),
    (dict(ctx_len=lambda t: t.float()), "ctx_len"), (dict(block_table=lambda t: t[:1]), "block_table"), (dict(block_table=lambda t: t.long()), "block_table"),
    (dict(block_table=lambda t: t.t().contiguous().t()), "block_table"), (dict(H=3), "heads"), (dict(H=0), "heads"), (dict(k_cache=lambda t: t[:, :0], v_cache=lambda t: t[:, :0]), "heads"), (dict(H=8), "q"),
    (dict(q=lambda t: t.half()), "float32 or bfloat16"), (dict(q=lambda t: t.bfloat16()), "k_cache"), (dict(k_cache=lambda t: t[0]), "k_cache"),
    (dict(v_cache=lambda t: t[:, :, :, :8]), "v_cache"), (dict(out=lambda t: t.bfloat16()), "out"), (dict(q=lambda t: t.t().contiguous().t()), "contiguous"),
    (dict(), "CUDA")])
def test_attention_tree_refuses(change, what):
    with pytest.raises(KernelError, match=what):
        ops.attention_tree(**step(**change))


def test_more_nodes_than_a_mask_has_bits():
    with pytest.raises(KernelError, match="more than 64"):
        ops.attention_tree(torch.zeros(130, 64), torch.zeros(9, 2, 16, 16), torch.zeros(9, 2, 16, 16), torch.tensor([0, 65, 130], dtype=torch.int32),
                           torch.tensor([70, 70], dtype=torch.int32), torch.ones(130, dtype=torch.int64), torch.zeros(2, 9, dtype=torch.int32),
                           torch.zeros(130, 64), 4, 0, 1.0)


def c_attention(H=4, KV=2, dh=16, page=16, window=0, scale=0.25, dtype=0, max_pages=2, scratch=1):
    fn = library.load().bl_attention_tree
    null = ctypes.c_void_p(0)
    return fn(null, null, null, dtype, null, null, null, null, max_pages, null, ctypes.c_void_p(scratch), 5, 2, H, KV, dh, page, window, ctypes.c_float(scale), null)


@pytest.mark.parametrize("change,what", [(dict(H=5), "cannot share"), (dict(H=130, KV=2), "at most 64"), (dict(dh=257), "head size 257"), (dict(dh=0), "head size 0"),
                                         (dict(page=0), "bad sizes"), (dict(window=-1), "bad sizes"), (dict(max_pages=0), "bad sizes"), (dict(scale=0.0), "positive"),
                                         (dict(scale=float("nan")), "positive"), (dict(dtype=7), "dtype 7"), (dict(scratch=0), "no scratch")])
def test_attention_tree_c_entry_refuses(change, what):
    assert c_attention(**change) == 1 and what in library.load().bl_last_error().decode()


def accept_args(**changes):
    s = TreeStep([3, 2], [5, 9], 2, 2, 16, 16, torch.float32, 0)
    kv = torch.zeros(3, 2, s.k.shape[0], 2, 16, 16)
    ids = torch.zeros(5, dtype=torch.int32)
    args = dict(sampled=ids, token_ids=ids, mask=s.mask, cu_q=s.cu_q, ctx_len=s.ctx_len, k_pages=kv[:, 0], v_pages=kv[:, 1], block_table=s.table)
    args.update({k: v(args[k]) if callable(v) else v for k, v in changes.items()})
    return args


@pytest.mark.parametrize("change,what", [
    (dict(sampled=lambda t: t.long()), "sampled"), (dict(token_ids=lambda t: t[:4]), "token_ids"), (dict(mask=lambda t: t.int()), "mask"),
    (dict(k_pages=lambda t: t[0]), "k_pages"), (dict(v_pages=lambda t: t[:2]), "k_pages, v_pages"), (dict(v_pages=lambda t: t.bfloat16()), "v_pages"),
    (dict(k_pages=lambda t: t.half()), "float32 or bfloat16"), (dict(k_pages=lambda t: t.transpose(2, 4).contiguous().transpose(2, 4)), "k_pages"),
    (dict(k_pages=lambda t: t[:1].expand(3, -1, -1, -1, -1)), "overlap"), (dict(block_table=lambda t: t[:1]), "block_table"), (dict(), "CUDA")])
def test_accept_tree_refuses(change, what):
    with pytest.raises(KernelError, match=what):
        ops.accept_tree(**accept_args(**change))


def test_accept_tree_refuses_keys_that_are_the_values():
    args = accept_args()
    with pytest.raises(KernelError, match="two tensors"):
        ops.accept_tree(**dict(args, v_pages=args["k_pages"]))


@pytest.mark.parametrize("tensors,pairs,what", [
    ([torch.zeros(5)], [(0, 1)], "layers, blocks"), ([torch.zeros(2, 5, 4).transpose(1, 2)], [(0, 1)], "contiguous"),
    ([torch.zeros(1, 5, 4).expand(3, -1, -1)], [(0, 1)], "overlap"), ([torch.zeros(2, 5, 4)], [(0, 1, 2)], "pairs"), ([torch.zeros(2, 5, 4)], [(0, 1 << 40)], "pairs"),
    ([torch.zeros(2, 5, 4)], [(0, 1.5)], "pairs"), ([torch.zeros(2, 5, 4)], [(0, 1)], "CUDA")])
def test_copy_blocks_refuses(tensors, pairs, what):
    with pytest.raises(KernelError, match=what):
        ops.copy_blocks(tensors, pairs)


@pytest.mark.parametrize("pairs,what", [([(0, 5)], "outside"), ([(-1, 2)], "outside"), ([(5, 2)], "outside"), ([(0, 2), (1, 2)], "target of two"),
                                        ([(0, 2), (2, 3)], "both source and target"), ([(1, 1)], "both source and target")])
def test_copy_blocks_c_entry_refuses(pairs, what):
    flat = array.array("i", [x for p in pairs for x in p])
    lib = library.load()
    tensors = array.array("q", [4096, 64, 64, 1, 5] * 9)
    at = lambda a: ctypes.c_void_p(a.buffer_info()[0])
    assert lib.bl_copy_blocks(1, at(tensors), at(flat), len(pairs), ctypes.c_void_p(0)) == 1
    assert what in lib.bl_last_error().decode()
    assert lib.bl_copy_blocks(9, at(tensors), at(flat), 1, ctypes.c_void_p(0)) == 1
    assert "more than the 8" in lib.bl_last_error().decode()


@pytest.mark.parametrize("least,snap", [(1, 0), (1, 3), (4, 2)])
@pytest.mark.parametrize("grid", [1, 3, 148, 296])
def test_the_line_of_work_is_shared_out_whole(grid, least, snap):
    """attention_tree.cuh restated: for units of any lengths, the parts cover the line once, no piece of a cut unit is shorter than a
    part and as short as the distance at which parts snap to its edges, every piece has a slot of its own, and each cut unit is merged once, from all of its pieces in their order."""
    rng = np.random.default_rng(grid)
    for trial in range(120):
        units = rng.integers(1, [8, 60, 400][trial % 3], int(rng.integers(1, 40))).tolist()
        begins = np.concatenate([[0], np.cumsum(units)])
        total = int(begins[-1])
        parts = max(1, min(grid, total // least))
        per, more = total // parts, total % parts
        edge = lambda k: per * k + min(k, more)

        def unit_of(x):
            u = int(np.searchsorted(begins, x, side="right")) - 1
            return u, int(begins[u]), units[u]

        def snapped(k):
            if k <= 0:
                return 0
            if k >= parts or edge(k) >= total:
                return total
            x = edge(k)
            _, begin, length = unit_of(x)
            return begin if x - begin <= snap else begin + length if begin + length - x <= snap else x

        slots, merged = {}, []
        for i in range(parts):
            at, end, first = snapped(i), snapped(i + 1), True
            assert at <= end
            while at < end:
                u, begin, length = unit_of(at)
                n = min(end, begin + length) - at
                if n != length:
                    assert n > snap or n >= per
                    slot = 2 * i + (0 if first else 1)
                    assert slot not in slots
                    slots[slot] = u
                at, first = at + n, False
        assert snapped(0) == 0 and snapped(parts) == total
        for i in range(1, parts):
            start, before = snapped(i), snapped(i - 1)
            if snapped(i + 1) == start:
                continue
            u, begin, length = unit_of(start)
            if start == begin or before > begin:
                continue
            inside = sum(1 for k in range(i, parts) if edge(k) < begin + length - snap)
            first = 2 * (i - 1) if before == begin else 2 * (i - 1) + 1
            assert [first] + [2 * k for k in range(i, i + inside)] == sorted(s for s, unit in slots.items() if unit == u)
            merged.append(u)
        assert sorted(merged) == sorted(set(slots.values()))
