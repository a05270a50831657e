"""The plain kernels of `reference_ops.py` with the drafts' operators beside them, on the CPU, for tests of the engine's own logic."""
import torch

import draft_reference as plain
from reference_ops import ReferenceOps


class PlainTreeOps(ReferenceOps):
    def rope_kv_store(self, qkv, row_pos, row_seg, tables, cos, sin, k_pages, v_pages, heads, kv_heads, head_dim, rope_dims, pairing, page_size,
                      v_dim=None, key_chunk=8, row_slot=None):
        args = (heads, kv_heads, head_dim, rope_dims, pairing, page_size, v_dim, key_chunk)
        if row_slot is None or k_pages is None:
            super().rope_kv_store(qkv, row_pos, row_seg, tables, cos, sin, k_pages, v_pages, *args)
            return
        super().rope_kv_store(qkv, row_pos, row_seg, tables, cos, sin, None, None, *args)          # rotated where it lies
        v_dim = v_dim or head_dim
        for r, slot in enumerate(row_slot.tolist()):
            page, off = int(tables[int(row_seg[r]), slot // page_size]), slot % page_size
            keys, values = qkv[r, heads * head_dim: (heads + kv_heads) * head_dim], qkv[r, (heads + kv_heads) * head_dim:]
            k_pages[page, :, :, off, :] = keys.view(kv_heads, head_dim // key_chunk, key_chunk)
            v_pages[page, :, :, off] = values.view(kv_heads, v_dim)

    def tree_attention(self, q, k_pages, v_pages, tables, row_pos, seg_start, kept, seen, out, heads, kv_heads, head_dim, page_size, scale,
                       max_context, window=None, sinks=None, v_dim=None, key_chunk=8, max_nodes=None):
        v_dim, group, starts = v_dim or head_dim, heads // kv_heads, seg_start.tolist()
        for s, (row0, end) in enumerate(zip(starts, starts[1:])):
            n = int(kept[s])
            for r in range(row0, end):
                low = int(row_pos[r]) - window + 1 if window else -1
                slots = [t for t in range(n) if t >= low]
                slots += [n + j for j in range(end - row0) if int(seen[r, j // 64]) >> j % 64 & 1 and int(row_pos[row0 + j]) >= low]
                slots = [t for t in slots if t // page_size < tables.shape[1] and 0 <= int(tables[s, t // page_size]) < k_pages.shape[0]]
                at = torch.tensor(slots, dtype=torch.long)
                page, off = tables[s, at // page_size].long(), at % page_size
                k = k_pages[page, :, :, off, :].double().reshape(len(slots), kv_heads, head_dim).repeat_interleave(group, 1)
                v = v_pages[page, :, :, off].double().repeat_interleave(group, 1)
                z = (k * q[r].double().view(heads, head_dim)).sum(-1) * scale
                if sinks is not None:
                    z = torch.cat([z, sinks.double()[None]])
                w = torch.softmax(z, 0)[: len(slots)]
                out[r] = (w[:, :, None] * v).sum(0).reshape(-1).to(out.dtype)
        return out

    def follow_tree(self, drafted, parents, seg_start, chosen, path, length, newest):
        starts = seg_start.tolist()
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            walked, token = plain.follow(parents[a:b].tolist(), drafted[a:b].tolist(), chosen[a:b].tolist(), path.shape[1])
            path[s] = torch.tensor(walked + [-1] * (path.shape[1] - len(walked)))
            length[s], newest[s] = len(walked), token

    def move_tokens(self, k_store, v_store, tables, kept, path, length):
        page_size = k_store.shape[-2]
        for s in range(tables.shape[0]):
            for i, node in enumerate(path[s, : int(length[s])].tolist()):
                (a, b), (c, d) = divmod(int(kept[s]) + node, page_size), divmod(int(kept[s]) + i, page_size)
                source, target = int(tables[s, a]), int(tables[s, c])
                if source >= 0 and target >= 0:
                    k_store[:, target, :, :, d] = k_store[:, source, :, :, b]
                    v_store[:, target, :, :, d] = v_store[:, source, :, :, b]

    def copy_pages(self, stores, source, target):
        for store in stores:
            store[:, target] = store[:, source]
