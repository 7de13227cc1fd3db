"""Steps with trees of drafted tokens for the tests: random trees and pages, and the operators in 64 bits, request by request."""
import math

import numpy as np
import torch


def masks_of(parents):
    """The bits of each node's ancestors and its own."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else 0) | 1 << i)
    return out


def signed(masks):
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def grown(rng, n, chain=0.5):
    """Parents of n nodes: the node before with probability `chain`, else any node before."""
    return [-1] + [i - 1 if rng.random() < chain else int(rng.integers(0, i)) for i in range(1, n)]


class TreeStep:
    """`counts[r]` nodes behind `committed[r]` tokens of each request; pages in random order, with NaN in every row that no request holds."""

    def __init__(self, counts, committed, H, KV, dh, page, dtype, seed, masks=None, device="cpu", spread=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.counts, self.committed, self.H, self.KV, self.dh, self.page = counts, committed, H, KV, dh, page
        held = [c + n for c, n in zip(committed, counts)]
        need = [-(-n // page) for n in held]
        pages = sum(need) + 3
        order = rng.permutation(pages)
        table = np.full((len(counts), max(need + [1]) + 1), -1, dtype=np.int32)
        k = torch.full((pages, KV, page, dh), float("nan"), dtype=dtype)
        v = k.clone()
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
            for i in range(n):
                rows = min(page, held[r] - i * page)
                k[table[r, i], :, :rows] = (torch.randn(KV, rows, dh, generator=g) * spread).to(dtype)
                v[table[r, i], :, :rows] = torch.randn(KV, rows, dh, generator=g).to(dtype)
        self.trees = [grown(rng, n) for n in counts if n > 0]
        if masks is None:
            masks = [m for t in self.trees for m in masks_of(t)]
        T = sum(counts)
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        dev = lambda t: t.to(device)
        self.q = dev((torch.randn(T, H * dh, generator=g) * 1.5).to(dtype))
        self.k, self.v, self.table = dev(k), dev(v), dev(torch.from_numpy(table))
        self.cu_q, self.ctx_len = dev(torch.from_numpy(cu)), dev(torch.tensor(held, dtype=torch.int32))
        self.masks = masks
        self.mask = dev(torch.tensor(signed(masks), dtype=torch.int64))
        self.scale = 1.0 / math.sqrt(dh)

    def run(self, window=0, out=None):
        from boring_llm_b200.kernels import ops
        out = torch.empty_like(self.q) if out is None else out
        ops.attention_tree(self.q, self.k, self.v, self.cu_q, self.ctx_len, self.mask, self.table, out, self.H, window, self.scale)
        return out

    def rows_of(self, r, t):
        """Rows 0 .. held - 1 of request r in cache tensor t, [KV, held, dh] in 64 bits."""
        n = self.committed[r] + self.counts[r]
        pages = self.table[r, :-(-n // self.page)].long()
        return t[pages].permute(1, 0, 2, 3).reshape(self.KV, -1, self.dh)[:, :n].double()

    def want(self, window=0):
        """(out, bound): the formula in 64 bits, and by how much a kernel with 32-bit sums may be off it, the rounding of the stored
        result not counted. With u = 2^-24 (half a step in 32 bits): a score is a chain of dh products, off by at most (dh + 2) u
        sum |q k| scale, its difference from the maximum and 2^x add some units more; a weight's relative error is that of its exponent
        (twice: numerator and denominator), and the sums over N keys (cut and merged) add at most (N + 16) u each."""
        u = 2.0 ** -24
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=self.q.device)
        bound = torch.zeros_like(out)
        G, t0 = self.H // self.KV, 0
        for r, n in enumerate(self.counts):
            c = self.committed[r]
            if n == 0:
                continue
            ms = [m & ((1 << n) - 1) for m in self.masks[t0:t0 + n]]
            pos = torch.tensor([c + max(bin(m).count("1") - 1, 0) for m in ms])
            sees = torch.zeros(n, c + n, dtype=torch.bool)
            sees[:, :c] = True if window == 0 else torch.arange(c)[None, :] + window > pos[:, None]
            for i, m in enumerate(ms):
                nodes = [k for k in range(n) if m >> k & 1]
                sees[i, [c + k for k in (nodes if window == 0 else nodes[-window:])]] = True
            sees = sees.to(self.q.device)
            keys, values = self.rows_of(r, self.k), self.rows_of(r, self.v)
            for h in range(self.H):
                cols = slice(h * self.dh, (h + 1) * self.dh)
                q, k, v = self.q[t0:t0 + n, cols].double(), keys[h // G], values[h // G]
                s = (q @ k.T * self.scale).masked_fill(~sees, -math.inf)
                mags = (q.abs() @ k.abs().T * self.scale).masked_fill(~sees, 0.0).amax(1, keepdim=True)
                top = s.amax(1, keepdim=True)
                w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                total = w.sum(1, keepdim=True)
                w = w / torch.where(total == 0, 1.0, total)
                out[t0:t0 + n, cols] = w @ v
                most = (w @ v.abs())
                bound[t0:t0 + n, cols] = most * u * (2 * ((self.dh + 2) * mags + 4 * mags + 8) + 2 * (c + n + 16))
            t0 += n
        return out, bound

    def check(self, got, window=0, probabilities_bf16=False):
        """`probabilities_bf16`: the kernel rounds the weights to bfloat16 before the product with the values, half a step (2^-8) of each."""
        want, bound = self.want(window)
        if probabilities_bf16:
            bound = bound + 2.0 ** -8 * self.weighted(window)
        half = torch.finfo(got.dtype).eps / 2
        allowed = bound * (1 + half) + half * want.abs() + 1e-30
        off = (got.double() - want).abs()
        assert torch.isfinite(got).all()
        worst = (off / allowed).max().item() if off.numel() else 0.0
        assert worst <= 1.0, f"off by {worst:.3f} of what rounding allows"

    def weighted(self, window=0):
        """sum_j w_j |v_j| of every output."""
        keep, self.v = self.v, self.v.abs()
        try:
            return self.want(window)[0]
        finally:
            self.v = keep


def accept_by_walk(parents, tokens, sampled):
    """The path of one request, node by node."""
    def deepest(node):
        best = [node]
        for child in range(len(parents)):
            if parents[child] == node and child != node and tokens[child] == sampled[node]:
                way = [node] + deepest(child)
                if len(way) > len(best) or (len(way) == len(best) and way[-1] < best[-1]):
                    best = way
        return best
    return deepest(0) if parents else []
