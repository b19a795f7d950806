"""The operators for drafted tokens in plain PyTorch / numpy, 64 bits: the reference of their kernels, and (`PlainDraftOps`) a plain
kernel table that the engine's host-side logic runs on without a GPU."""
from __future__ import annotations
import numpy as np
import torch

from plain_ops import PlainOps


def ancestors_of(parents, words=None) -> np.ndarray:
    """int32 (n, words): bit j of row i: node j is node i or one of its ancestors."""
    n = len(parents)
    bits = np.zeros((n, words or -(-n // 32)), np.uint32)
    for i, p in enumerate(parents):
        if p >= 0:
            bits[i] = bits[p]
        bits[i, i // 32] |= np.uint32(1 << (i % 32))
    return bits.view(np.int32)


def depths_of(parents) -> list[int]:
    out = []
    for p in parents:
        out.append(out[p] + 1 if p >= 0 else 0)
    return out


def attend(q, keys, values, table, seg, pos, seq_row, ancestors, heads, kv_heads, hd, scale, window):
    """(result, sum of weights x |values|) in float64, rows without keys and rows of padding zero. Only the places that a row sees
    are read."""
    n, page, group = q.shape[0], keys.shape[2], heads // kv_heads
    out = torch.zeros(n, heads, hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    bits = ancestors.cpu().numpy().view(np.uint32)
    for i in range(n):
        s = int(seq_row[i])
        if s < 0:
            continue
        rows, start, p = int(seg[s, 1]), int(seg[s, 2]), int(pos[i])
        places = list(range(max(0, p - window + 1) if window else 0, start))
        places += [start + j for j in range(rows) if j // 32 < bits.shape[1] and bits[i, j // 32] >> np.uint32(j % 32) & np.uint32(1)]
        if not places:
            continue
        at = torch.tensor(places)
        pages = table[s].long()[at // page]
        k, v = keys[pages, :, at % page].double(), values[pages, :, at % page].double()      # (places, kv heads, hd)
        for h in range(heads):
            w = torch.softmax((k[:, h // group] @ q[i, h * hd:(h + 1) * hd].double()) * scale, 0)
            out[i, h] = w @ v[:, h // group]
            size[i, h] = w @ v[:, h // group].abs()
    return out.view(n, heads * hd), size.view(n, heads * hd)


def softmax64(x, t) -> np.ndarray:
    z = x.astype(np.float64) / t
    e = np.exp(z - z.max())
    return e / e.sum()


def draw(p, u) -> int:
    total = np.cumsum(p)
    return min(int(np.searchsorted(total, u * total[-1], side="right")), len(p) - 1)


def verify(logits, draft, temperature, uniform, tokens, parents, seg):
    """(path with -1 at every row that no kept node fills, count, next ids)."""
    path = np.full(len(tokens), -1, np.int32)
    count, last = np.zeros(len(seg), np.int32), np.full(len(seg), -1, np.int32)
    vocab = logits.shape[1]
    for s, (row0, n, *_) in enumerate(np.asarray(seg)):
        if n <= 0:
            continue
        t, node, kept = float(temperature[s]), 0, [0]
        while True:
            row = np.asarray(logits[row0 + node], np.float32)
            children = [j for j in range(node + 1, n) if parents[row0 + j] == node]
            taken = None
            if not t > 0:
                best = int(np.argmax(row))
                taken = next((j for j in children if tokens[row0 + j] == best), None)
                answer = best
            elif not np.isfinite(row.max()):      # a NaN, +inf, or nothing above -inf
                answer = vocab - 1
            else:
                p = softmax64(row, t)
                q = softmax64(np.asarray(draft[row0 + node], np.float32), t) if draft is not None and children else None
                for j in children:
                    x = tokens[row0 + j]
                    if uniform[row0 + j] * (1.0 if q is None else q[x]) < p[x]:
                        taken = j
                        break
                    rest = p.copy()
                    if q is None:
                        rest[x] = 0.0
                    else:
                        rest = np.maximum(p - q, 0.0)
                        q = q.copy()
                        q[x] = 0.0
                        q /= q.sum() or 1.0
                    if rest.sum() > 0:
                        p = rest / rest.sum()
                answer = draw(p, uniform[row0]) if taken is None else -1
            if taken is None:
                break
            node = taken
            kept.append(node)
        path[row0:row0 + len(kept)] = kept
        count[s], last[s] = len(kept), answer
    return path, count, last


def keep(pool, table, seg, path, count) -> None:
    page, was = pool.shape[-2], pool.clone()
    for s, (row0, n, start, _) in enumerate(seg.tolist()):
        for k in range(int(count[s])):
            a, b = start + int(path[row0 + k]), start + k
            pool[:, int(table[s, b // page])][..., b % page, :] = was[:, int(table[s, a // page])][..., a % page, :]


def copy(pool, src, dst) -> None:
    pool[:, dst.long()] = pool[:, src.long()].clone()


class PlainDraftOps(PlainOps):
    """`PlainOps` with the operators for drafted tokens."""

    def rope_kv_write(self, qkv, cos, sin, meta, cache, q_out, num_heads, num_kv_heads, head_dim) -> None:
        place = getattr(meta, "place", None)
        if place is None:
            return super().rope_kv_write(qkv, cos, sin, meta, cache, q_out, num_heads, num_kv_heads, head_dim)
        n, hq, hkv, hd = qkv.shape[0], num_heads, num_kv_heads, head_dim
        x = qkv.view(n, hq + 2 * hkv, hd)
        c, s = cos[meta.pos.long()][:, None], sin[meta.pos.long()][:, None]
        a, b = x[:, :hq + hkv, :hd // 2], x[:, :hq + hkv, hd // 2:]
        rot = torch.cat([a * c - b * s, b * c + a * s], -1)
        q_out.copy_(torch.where((meta.seq_row >= 0)[:, None, None], rot[:, :hq], 0.0).reshape(n, hq * hd).to(q_out.dtype))
        table = meta.table(cache.group)
        for i in range(n):
            if cache.write and meta.seq_row[i] >= 0:
                at = int(place[i])
                page = int(table[int(meta.seq_row[i]), at // cache.page_size])
                assert page >= 0
                cache.keys[page, :, at % cache.page_size] = rot[i, hq:].to(cache.keys.dtype)
                cache.values[page, :, at % cache.page_size] = x[i, hq + hkv:].to(cache.values.dtype)

    def tree_attention(self, q, cache, meta, out, num_heads, num_kv_heads, head_dim, scale, window) -> None:
        o, _ = attend(q, cache.keys, cache.values, meta.table(cache.group), meta.seg, meta.pos, meta.seq_row, meta.ancestors, num_heads,
                      num_kv_heads, head_dim, scale, window)
        out.copy_(o.to(out.dtype))

    def verify_tree(self, logits, draft, temperature, uniform, tokens, parents, seg, path, count, next_ids) -> None:
        p, c, i = verify(logits.numpy(), None if draft is None else draft.numpy(), temperature.numpy(), uniform.numpy(), tokens.numpy(),
                         parents.numpy(), seg.numpy())
        for row0, n, *_ in seg.tolist():
            path[row0:row0 + n] = torch.from_numpy(p[row0:row0 + n])
        count.copy_(torch.from_numpy(c))
        next_ids.copy_(torch.from_numpy(i))

    def keep_rows(self, pool, table, seg, path, count) -> None:
        keep(pool, table, seg, path, count)

    def copy_pages(self, pool, src, dst) -> None:
        copy(pool, src, dst)
