"""Plain forms of the work on trees of drafted tokens, in 64 bits on the CPU, with the inputs that the tests hand to both sides."""
import math
import random

import torch


def random_tree(nodes, rng, deep=0.3):
    """Parents of a tree of `nodes` nodes: each is a child of the node before it with probability `deep`, else of any before it."""
    return [-1] + [i - 1 if rng.random() < deep else rng.randrange(i) for i in range(1, nodes)]


def signed_words(bits, words):
    out = []
    for w in range(words):
        v = bits >> 64 * w & (1 << 64) - 1
        out.append(v - (1 << 64) if v >> 63 else v)
    return out


class TreeCase:
    """Requests of (kept, nodes) with their pages; slots of no token hold NaN.  `seen_of` [request][node] -> set of nodes."""

    def __init__(self, requests, heads, kv_heads, dim, page, dtype, seed, v_dim=None, key_chunk=8, words=None, spare_rows=0, spare_pages=3):
        rng = random.Random(seed)
        gen = torch.Generator().manual_seed(seed)
        self.requests, self.heads, self.kv_heads, self.dim, self.page, self.dtype = requests, heads, kv_heads, dim, page, dtype
        self.v_dim = v_dim or dim
        self.key_chunk = key_chunk
        per = [-(-(kept + nodes) // page) for kept, nodes in requests]
        total = sum(per) + spare_pages
        order = torch.randperm(total, generator=gen).tolist()
        self.k_pages = torch.full((total, kv_heads, dim // key_chunk, page, key_chunk), float("nan"), dtype=dtype)
        self.v_pages = torch.full((total, kv_heads, self.v_dim, page), float("nan"), dtype=dtype)
        self.tables = torch.full((len(requests), max(per + [1])), -1, dtype=torch.int32)
        self.keys, self.values, self.parents, self.seen_of, positions = [], [], [], [], []
        starts = [0]
        for s, (kept, nodes) in enumerate(requests):
            mine, order = order[: per[s]], order[per[s]:]
            self.tables[s, : per[s]] = torch.tensor(mine, dtype=torch.int32)
            n = kept + nodes
            k = torch.randn((n, kv_heads, dim), generator=gen).to(dtype)
            v = torch.randn((n, kv_heads, self.v_dim), generator=gen).to(dtype)
            self.keys.append(k)
            self.values.append(v)
            for t in range(n):
                self.put(s, t)
            parents = random_tree(nodes, rng) if nodes else []
            depth, seen = [], []
            for i, p in enumerate(parents):
                depth.append(depth[p] + 1 if i else 0)
                seen.append((set(seen[p]) if i else set()) | {i})
            self.parents.append(parents)
            self.seen_of.append(seen)
            positions += [kept + d for d in depth]
            starts.append(starts[-1] + nodes)
        rows = starts[-1] + spare_rows
        self.rows, self.live_rows = rows, starts[-1]
        self.words = words or max(1, -(-max([n for _, n in requests] + [1]) // 64))
        self.seg_start = torch.tensor(starts, dtype=torch.int32)
        self.kept = torch.tensor([kept for kept, _ in requests], dtype=torch.int32)
        self.row_pos = torch.tensor(positions + [0] * spare_rows, dtype=torch.int32)
        self.joint = torch.randn((rows, heads * dim + 40), generator=gen).to(dtype)      # the queries are columns of a wider matrix
        self.sinks = torch.randn(heads, generator=gen)

    def put(self, s, t):
        """The key and value of request s's slot t into its page."""
        page = int(self.tables[s, t // self.page])
        self.k_pages[page, :, :, t % self.page] = self.keys[s][t].view(self.kv_heads, -1, self.key_chunk)
        self.v_pages[page, :, :, t % self.page] = self.values[s][t]

    @property
    def seen(self):
        rows = [signed_words(sum(1 << j for j in seen), self.words) for per in self.seen_of for seen in per]
        rows += [[-1] * self.words] * (self.rows - self.live_rows)
        return torch.tensor(rows, dtype=torch.int64).reshape(self.rows, self.words)

    def visible(self, s, i, window):
        """The slots that node i of request s sees."""
        kept, nodes = self.requests[s]
        row0 = int(self.seg_start[s])
        pos = int(self.row_pos[row0 + i])
        low = pos - window + 1 if window else -(1 << 40)
        slots = [t for t in range(max(low, 0), kept)]
        slots += [kept + j for j in sorted(self.seen_of[s][i]) if j < nodes and int(self.row_pos[row0 + j]) >= low]
        pages = self.k_pages.shape[0]
        return [t for t in slots if t // self.page < self.tables.shape[1] and 0 <= int(self.tables[s, t // self.page]) < pages]

    def expected(self, scale, window=0, sinks=False):
        """(outputs, how far a kernel's may be off) as float64 [rows, heads * v_dim]; rows of no request stay NaN.

        The bound: scores are sums of dim products in 32 bits, each product and sum rounded (2^-24 relative): delta = (dim + 8) 2^-24 sum |q k| |scale|
        covers them, the scale, the base-2 exponent's factor and a maximum of the same size.  A weight is then off by 2 delta relative
        (its own score's error and the reference point's cancel in the quotient, the sum's does not), the sums of n terms by (n + 16) 2^-23;
        in bfloat16 a weight is rounded once more before it meets the value (2^-8) and the result once (2^-8)."""
        out = torch.full((self.rows, self.heads, self.v_dim), float("nan"), dtype=torch.float64)
        bound = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        q = self.joint[:, : self.heads * self.dim].double().reshape(self.rows, self.heads, self.dim)
        step = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -24
        for s, (kept, nodes) in enumerate(self.requests):
            row0 = int(self.seg_start[s])
            keys, values = self.keys[s].double(), self.values[s].double()
            for i in range(nodes):
                slots = self.visible(s, i, window)
                if not slots:
                    out[row0 + i] = 0.0
                    continue
                k = keys[slots].repeat_interleave(group, dim=1)            # [n, heads, dim]
                v = values[slots].repeat_interleave(group, dim=1)
                z = (k * q[row0 + i][None]).sum(-1) * scale                # [n, heads]
                delta = (self.dim + 8) * 2.0 ** -24 * ((k * q[row0 + i][None]).abs().sum(-1) * abs(scale)).amax(0)
                top = z.amax(0)
                if sinks:
                    top = torch.maximum(top, self.sinks.double())
                w = torch.exp(z - top)
                below = w.sum(0)
                if sinks:
                    below = below + torch.exp(self.sinks.double() - top)
                out[row0 + i] = (w[:, :, None] * v).sum(0) / below[:, None]
                spread = (w[:, :, None] * v.abs()).sum(0) / below[:, None]
                relative = 2 * delta + (len(slots) + 16) * 2.0 ** -23 + (step if self.dtype == torch.bfloat16 else 0.0)
                bound[row0 + i] = relative[:, None] * spread * 1.05 + step * out[row0 + i].abs() * 1.05 + 1e-30
        return out.reshape(self.rows, -1), bound.reshape(self.rows, -1)


def follow(parents, drafted, chosen, most):
    """(path, newest) of one tree."""
    if not parents:
        return [], -1
    path = [0]
    while len(path) < most:
        at = path[-1]
        fits = [c for c in range(at + 1, len(parents)) if parents[c] == at and drafted[c] == chosen[at]]
        if not fits:
            break
        path.append(fits[0])
    return path, chosen[path[-1]]


def compare(got, want, bound):
    """The largest share of the bound that an element takes; rows that are NaN in `want` are left out by the caller."""
    got = got.double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    share = torch.where(same, torch.zeros_like(want), (got - want).abs() / bound)
    return float(torch.where(torch.isnan(share), torch.full_like(share, math.inf), share).max()) if share.numel() else 0.0
