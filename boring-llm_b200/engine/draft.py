"""Drafted tokens for a request from its own text: what followed the last tokens when they came before.

The reference has no such step; its loop feeds one token after the other (src/model.br:2293-2304). The drafts of a request are a
tree: node 0 is the token that is certain (the last one sampled), the first guess hangs from it as a chain, further
guesses branch off where they differ. The model runs all nodes at once; which of them it agrees with is found on the device.
"""
from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

MAX_NODES = 64                # nodes of one request in a step: what a node sees of them is a 64-bit mask


def tree_masks(parents: Sequence[int]) -> List[int]:
    """Each node's ancestors and itself as the bits of a number. `parents[0]` is -1, every other node's parent comes before it."""
    if len(parents) > MAX_NODES:
        raise ValueError(f"a tree of {len(parents)} nodes (at most {MAX_NODES})")
    masks: List[int] = []
    for i, p in enumerate(parents):
        if not (p == -1 if i == 0 else 0 <= p < i):
            raise ValueError(f"node {i}: parent {p} is not one of the nodes before it")
        masks.append((masks[p] if i else 0) | 1 << i)
    return masks


class History:
    """A request's tokens with the places where each run of up to `longest` tokens has ended so far."""

    def __init__(self, longest: int = 3, keep: int = 8):
        self.longest, self.keep = longest, keep       # places kept of each run: the last ones
        self.tokens: List[int] = []
        self._places: Dict[Tuple[int, ...], List[int]] = {}

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            # the runs that end in front of this token are worth looking up once there is a token behind them
            n = len(self.tokens)
            for k in range(1, min(self.longest, n) + 1):
                places = self._places.setdefault(tuple(self.tokens[n - k:]), [])
                places.append(n)
                if len(places) > self.keep:
                    del places[0]
            self.tokens.append(t)

    def draft(self, nodes: int, branches: int = 4, depth: int = 16) -> Tuple[List[int], List[int]]:
        """(tokens, parents) of a tree of up to `nodes` nodes whose node 0 is the last token: what followed the longest run of last
        tokens that has come before, latest place first, up to `branches` places and `depth` tokens each."""
        if not self.tokens:
            raise ValueError("no tokens to draft from")
        tokens, parents = [self.tokens[-1]], [-1]
        child: Dict[Tuple[int, int], int] = {}
        nodes = min(nodes, MAX_NODES)
        for k in range(min(self.longest, len(self.tokens)), 0, -1):
            places = self._places.get(tuple(self.tokens[-k:]))
            if not places:
                continue
            for at in places[:-branches - 1:-1]:
                node, guess = 0, self.tokens[at:at + depth]
                for j in range(depth - len(guess)):      # behind the last token the guess goes on from itself: text that repeats
                    guess.append(guess[j])
                for t in guess:
                    nxt = child.get((node, t))
                    if nxt is None:
                        if len(tokens) >= nodes:
                            return tokens, parents
                        nxt = child[(node, t)] = len(tokens)
                        tokens.append(t)
                        parents.append(node)
                    node = nxt
            break
        return tokens, parents
