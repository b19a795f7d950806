"""What the speed of the operators for drafted tokens is measured on: attention of a drafted tree over the paged cache, the
verdict on the drafts, the cache's kept rows moved together, and copies of cache pages.

A case is a dict; its `op`:
  attend   one layer's attention of `requests` requests that bring a tree of up to `nodes` drafted tokens each, behind up to
           `context` cached tokens (spread evenly down to half of it), over pages of `page` tokens
  verify   `requests` requests with trees of up to `nodes` nodes: which drafted tokens stand, and the token behind them, from
           the target's logits and either the drafter's logits (`drafter`) or the bare tokens of a drafter without any
  keep     the kept nodes' cache rows of `requests` requests moved together, over all `layers`
  copy     `pages` cache pages copied to other pages, over all `layers`
Head layouts and vocabularies are those of this package's presets and tests.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
# (query heads, kv heads, head size, layers, vocabulary) of the dense decoders that this package is run with
SIZES = {"llama-3.1-8b": (32, 8, 128, 32, 128256), "qwen2.5-0.5b": (14, 2, 64, 24, 151936), "qwen2.5-32b": (40, 8, 128, 64, 152064),
         "tiny-llama": (4, 2, 16, 2, 256)}


def _attend(model, requests, nodes, context, dtype="bfloat16", page=16, window=0, chain=False):
    return {"op": "attend", "model": model, "dtype": dtype, "requests": requests, "nodes": nodes, "context": context, "page": page,
            "window": window, "chain": chain}


def _verify(model, requests, nodes, drafter, chain=False):
    return {"op": "verify", "model": model, "requests": requests, "nodes": nodes, "drafter": drafter, "chain": chain}


def _keep(model, requests, nodes, dtype="bfloat16", page=16):
    return {"op": "keep", "model": model, "dtype": dtype, "requests": requests, "nodes": nodes, "page": page}


def _copy(model, pages, dtype="bfloat16", page=16):
    return {"op": "copy", "model": model, "dtype": dtype, "pages": pages, "page": page}


def listed():
    return [
        # one user, a short text: a chain of a few drafted tokens, all latency
        {"name": "attend 0.5b 1 x 5 at 300", **_attend("qwen2.5-0.5b", 1, 5, 300, chain=True)},
        # one user's long text, a tree of guesses
        {"name": "attend 8b 1 x 27 at 30000", **_attend("llama-3.1-8b", 1, 27, 30000)},
        # a busy server, short chains
        {"name": "attend 8b 64 x 6 at 4096", **_attend("llama-3.1-8b", 64, 6, 4096, chain=True)},
        # wide trees of a large model over long texts: several tiles of rows per kv head
        {"name": "attend 32b 4 x 64 at 12000", **_attend("qwen2.5-32b", 4, 64, 12000)},
        # the true 32-bit path
        {"name": "attend 0.5b f32 4 x 13 at 500", **_attend("qwen2.5-0.5b", 4, 13, 500, dtype="float32")},
        # one user, a drafter that only looks tokens up
        {"name": "verify 8b 1 x 5", **_verify("llama-3.1-8b", 1, 5, False, chain=True)},
        # trees from a draft model
        {"name": "verify 8b 8 x 16 drafter", **_verify("llama-3.1-8b", 8, 16, True)},
        # a busy server, chains from a draft model
        {"name": "verify 0.5b 64 x 6 drafter", **_verify("qwen2.5-0.5b", 64, 6, True, chain=True)},
        # after a verdict: one user, and a busy server
        {"name": "keep 0.5b 1 x 8", **_keep("qwen2.5-0.5b", 1, 8)},
        {"name": "keep 8b 64 x 16", **_keep("llama-3.1-8b", 64, 16)},
        # a request continued in three ways, its last page copied; and every request of a server
        {"name": "copy 0.5b 3 pages", **_copy("qwen2.5-0.5b", 3)},
        {"name": "copy 8b 192 pages", **_copy("llama-3.1-8b", 192)},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "verify", "verify", "keep", "copy"))
    if op == "attend":
        if rng.random() < 0.3:
            model = rng.choice(("qwen2.5-0.5b", "tiny-llama"))
            return _attend(model, _log(rng, 1, 8), _log(rng, 1, 24), _log(rng, 1, 1500), dtype="float32", page=rng.choice((4, 16)),
                           chain=rng.random() < 0.3)
        model = rng.choice(("llama-3.1-8b", "llama-3.1-8b", "qwen2.5-0.5b", "qwen2.5-32b"))
        requests = _log(rng, 1, 64)
        return _attend(model, requests, _log(rng, 1, 64 if requests <= 8 else 16), _log(rng, 1, min(40000, 200000 // requests)),
                       page=rng.choice((8, 16, 16, 32)), window=rng.choice((0, 0, 0, _log(rng, 64, 4096))), chain=rng.random() < 0.3)
    if op == "verify":
        model, drafter = rng.choice(("llama-3.1-8b", "qwen2.5-0.5b", "tiny-llama")), rng.random() < 0.6
        requests = _log(rng, 1, 64)
        return _verify(model, requests, _log(rng, 1, max(1, min(40, 300 // requests))), drafter, chain=rng.random() < 0.4)
    model, dtype = rng.choice((("llama-3.1-8b", "bfloat16"), ("qwen2.5-0.5b", "bfloat16"), ("qwen2.5-0.5b", "float32"), ("tiny-llama", "float32")))
    page = rng.choice((4, 16, 16, 32))
    if op == "keep":
        return _keep(model, _log(rng, 1, 48), _log(rng, 2, 40), dtype=dtype, page=page)
    return _copy(model, _log(rng, 1, 2048 // page), dtype=dtype, page=page)


def spread(longest, n):
    """n lengths from `longest` down to half of it."""
    return [longest - (longest // 2) * i // max(1, n - 1) for i in range(n)]


def node_counts(case):
    """Nodes of each request's tree: the most, then ragged ones below it."""
    return [max(1, case["nodes"] - (i % 3) * (case["nodes"] // 4)) for i in range(case["requests"])]


# ---- inputs, from the seed alone

class Step:
    """A step's metadata: what the step function keeps of it on the device."""

    def __init__(self, pos, seq_row, seg, tables, ancestors, max_context, max_portion):
        self.pos, self.seq_row, self.seg, self.tables, self.ancestors = pos, seq_row, seg, tables, ancestors
        self.max_context, self.max_portion = max_context, max_portion

    def table(self, group):
        return self.tables


class Cache:
    """A layer's keys and values, (pages, kv heads, page, head size)."""

    def __init__(self, keys, values, page_size):
        self.keys, self.values, self.page_size, self.group, self.write = keys, values, page_size, 0, True


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _trees(rng, counts, chain):
    """parents (N,), depths (N,): node 0 of a request is its root, a node's parent stands before it. Not chains: new nodes go to
    nodes near the root more often than to deep ones, two to four children each."""
    parents, depths = [], []
    for n in counts:
        par = [-1] + [i - 1 if chain else max(0, (i - 1) // 2 - int(rng.integers(0, 2))) for i in range(1, n)]
        dep = [0] * n
        for i in range(1, n):
            dep[i] = dep[par[i]] + 1
        parents += par
        depths += dep
    return np.array(parents, np.int32), np.array(depths, np.int32)


def _segments(counts, starts):
    seg = np.zeros((len(counts), 4), np.int32)
    seg[:, 0] = np.concatenate([[0], np.cumsum(counts)[:-1]])
    seg[:, 1], seg[:, 2], seg[:, 3] = counts, starts, -1
    return seg


def _tables(rng, lengths, page):
    """Block tables of requests with these many tokens, pages in random order, and the number of pages."""
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need)).astype(np.int32)
    table = np.full((len(lengths), max(need)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    rng, gen = np.random.default_rng(seed), _generator(seed)
    heads, kv, hd, layers, vocab = SIZES[case["model"]]
    dtype = DTYPES[case.get("dtype", "float32")]
    if case["op"] == "copy":
        total = 2 * case["pages"] + 1
        pool = torch.randn((layers, total, 2, kv, case["page"], hd), generator=gen, device="cuda", dtype=dtype)
        order = rng.permutation(total).astype(np.int32)
        # (some pages go to several places: a request continued in several ways)
        src = order[rng.integers(0, case["pages"], case["pages"])]
        return {**case, "pool": pool, "src": _cuda(src), "dst": _cuda(order[case["pages"]:2 * case["pages"]])}
    counts = node_counts(case)
    if case["op"] == "keep":
        starts = [7 * i % (3 * case["page"]) for i in range(case["requests"])]
        table, pages = _tables(rng, [s + n for s, n in zip(starts, counts)], case["page"])
        pool = torch.randn((layers, pages, 2, kv, case["page"], hd), generator=gen, device="cuda", dtype=dtype)
        path, count = np.full(sum(counts), -1, np.int32), np.zeros(len(counts), np.int32)
        seg = _segments(counts, starts)
        for i, n in enumerate(counts):
            count[i] = kept = _kept(i, n)
            path[seg[i, 0]] = 0
            path[seg[i, 0] + 1: seg[i, 0] + kept] = np.sort(rng.permutation(n - 2)[:kept - 1]) + 2
        return {**case, "pool": pool, "table": _cuda(table), "seg": _cuda(seg), "path": _cuda(path), "count": _cuda(count)}
    parents, depths = _trees(rng, counts, case["chain"])
    if case["op"] == "attend":
        starts = spread(case["context"], case["requests"])
        table, pages = _tables(rng, [s + n for s, n in zip(starts, counts)], case["page"])
        seg = _segments(counts, starts)
        words = -(-max(counts) // 32)
        ancestors = np.zeros((sum(counts), words), np.uint32)
        for r, (row0, n, _, _) in enumerate(seg):
            for i in range(n):
                if parents[row0 + i] >= 0:
                    ancestors[row0 + i] = ancestors[row0 + parents[row0 + i]]
                ancestors[row0 + i, i // 32] |= np.uint32(1 << (i % 32))
        row = np.repeat(np.arange(len(counts), dtype=np.int32), counts)
        pool = torch.randn((pages, 2, kv, case["page"], hd), generator=gen, device="cuda", dtype=dtype)
        q = torch.randn((sum(counts), heads * hd), generator=gen, device="cuda", dtype=torch.float32).mul_(1.5).to(dtype)
        meta = Step(_cuda(np.array(starts, np.int32)[row] + depths), _cuda(row), _cuda(seg), _cuda(table), _cuda(ancestors.view(np.int32)),
                    max(s + n for s, n in zip(starts, counts)), max(counts))
        return {**case, "q": q, "cache": Cache(pool[:, 0], pool[:, 1], case["page"]), "meta": meta, "out": torch.empty_like(q), "heads": heads,
                "kv": kv, "hd": hd, "scale": hd ** -0.5}
    # verify: logits like a model's, a few tokens far above the rest; the drafter's are the target's with an error of its own. Every
    # request has its own temperature, each fifth is greedy. A node's children are draws from the drafter without replacement (or, of a
    # drafter without probabilities, likely tokens).
    seg = _segments(counts, [0] * len(counts))
    n = sum(counts)
    logits = torch.randn((n, vocab), generator=gen, device="cuda") * 2.5
    logits += 13.0 * (torch.rand((n, vocab), generator=gen, device="cuda") < 12.0 / vocab)
    draft = logits + torch.randn((n, vocab), generator=gen, device="cuda") * 0.4
    temperature = np.array([0.0 if i % 5 == 4 else 0.6 + 0.1 * (i % 4) for i in range(len(counts))], np.float32)
    row = np.repeat(np.arange(len(counts)), counts)
    t = _cuda(np.where(temperature > 0, temperature, 0.1)[row].astype(np.float32))[:, None]
    noise = -torch.log(-torch.log(torch.rand((n, vocab), generator=gen, device="cuda").clamp_(1e-9, 1 - 1e-7)))
    best = (draft / t + noise).topk(min(8, vocab), dim=1).indices.cpu().numpy()
    rank, seen = np.zeros(n, np.int64), {}
    parent_row = np.where(parents >= 0, parents + seg[row, 0], np.arange(n))
    for i in range(n):
        if parents[i] >= 0:
            rank[i] = seen.get(parent_row[i], 0)
            seen[parent_row[i]] = rank[i] + 1
    tokens = np.where(parents >= 0, best[parent_row, np.minimum(rank, best.shape[1] - 1)], rng.integers(0, vocab, n)).astype(np.int32)
    return {**case, "logits": logits, "draft": draft if case["drafter"] else None, "temperature": _cuda(temperature),
            "uniform": _cuda(rng.random(n)), "tokens": _cuda(tokens), "parents": _cuda(parents), "seg": _cuda(seg),
            "path": torch.empty(n, dtype=torch.int32, device="cuda"), "count": torch.empty(len(counts), dtype=torch.int32, device="cuda"),
            "next": torch.empty(len(counts), dtype=torch.int32, device="cuda")}


def _kept(i, n):
    """How many nodes of request i's tree of n are kept: one to about a third of them, the root among them."""
    return 1 + (1 + i % max(1, n // 3) if n >= 3 else 0)


# ---- one pass

_tables_of_kernels = {}


def _kernels(dtype):
    if dtype not in _tables_of_kernels:
        from fusezap_core_b200.kernels import cuda_ops
        _tables_of_kernels[dtype] = cuda_ops(dtype)
    return _tables_of_kernels[dtype]


def run(s):
    op = s["op"]
    if op == "attend":
        if own:
            _kernels(s["dtype"]).tree_attention(s["q"], s["cache"], s["meta"], s["out"], s["heads"], s["kv"], s["hd"], s["scale"], s["window"])
            return s["out"]
        return attend(s["q"], s["cache"].keys, s["cache"].values, s["meta"], s["heads"], s["kv"], s["hd"], s["scale"], s["window"])
    if op == "verify":
        if own:
            _kernels("float32").verify_tree(s["logits"], s["draft"], s["temperature"], s["uniform"], s["tokens"], s["parents"], s["seg"],
                                            s["path"], s["count"], s["next"])
            return s["path"], s["count"], s["next"]
        return verify(s["logits"], s["draft"], s["temperature"], s["uniform"], s["tokens"], s["parents"], s["seg"], s["nodes"])
    if op == "keep":
        if own:
            _kernels(s["dtype"]).keep_rows(s["pool"], s["table"], s["seg"], s["path"], s["count"])
        else:
            keep(s["pool"], s["table"], s["seg"], s["path"], s["count"])
        return s["pool"]
    if own:
        _kernels(s["dtype"]).copy_pages(s["pool"], s["src"], s["dst"])
    else:
        src, dst = s["src"].long(), s["dst"].long()
        s["pool"][:, dst] = s["pool"][:, src]
    return s["pool"]


def attend(q, keys, values, meta, heads, kv, hd, scale, window):
    """softmax(scale q k^T) v over the places before the request's tree (from position - window + 1 on, with a window) and the tree's
    places whose bit is set, in 32 bits."""
    seg, page = meta.seg.long(), keys.shape[2]
    n, group, most, longest = q.shape[0], heads // kv, meta.max_portion, meta.max_context
    place = torch.arange(longest, device=q.device)
    table = meta.tables.long()[:, :(longest + page - 1) // page]
    at = table.repeat_interleave(page, 1)[:, :longest].clamp_min(0), (place % page).expand(seg.shape[0], longest)
    there = (place < (seg[:, 2] + seg[:, 1])[:, None])[:, :, None, None]
    k = torch.where(there, keys[at[0], :, at[1]].float(), 0.0).permute(0, 2, 3, 1)              # (S, kv, hd, L)
    v = torch.where(there, values[at[0], :, at[1]].float(), 0.0).permute(0, 2, 1, 3)            # (S, kv, L, hd)
    row = seg[:, :1] + torch.arange(most, device=q.device)
    live = torch.arange(most, device=q.device) < seg[:, 1:2]
    row = torch.where(live, row, 0)
    pos, bits = meta.pos.long()[row], meta.ancestors[row]
    queries = q.float()[row].view(seg.shape[0], most, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(seg.shape[0], kv, most * group, hd)
    node = place - seg[:, 2:3]
    word = (node // 32).clamp(0, bits.shape[2] - 1)[:, None, :].expand(-1, most, -1)
    set_ = (torch.gather(bits, 2, word).long() >> (node % 32)[:, None, :]) & 1 > 0
    first = (pos - window + 1).clamp_min(0) if window else torch.zeros_like(pos)
    seen = torch.where((node >= 0)[:, None, :], set_ & (node < seg[:, 1:2])[:, None, :], place >= first[:, :, None])
    seen = seen[:, None, :, None, :]
    score = (queries @ k).mul_(scale).view(seg.shape[0], kv, most, group, longest).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    mixed = (weight.view(seg.shape[0], kv, most * group, longest) @ v).view(seg.shape[0], kv, most, group, hd)
    mixed = mixed / torch.where(total > 0, total, 1.0)
    out = torch.empty((n, heads, hd), dtype=q.dtype, device=q.device)
    out[row[live]] = mixed.permute(0, 2, 1, 3, 4).reshape(seg.shape[0], most, heads, hd)[live].to(q.dtype)
    return out.view(n, heads * hd)


def verify(logits, draft, temperature, uniform, tokens, parents, seg, nodes):
    """The walk from each request's root, all requests side by side, one drafted token each at a time (a token's acceptance depends on
    the siblings before it), in 64 bits."""
    seg, par, tok = seg.long(), parents.long(), tokens.long()
    requests, vocab, dev = seg.shape[0], logits.shape[1], logits.device
    each, at = torch.arange(requests, device=dev), seg[:, 0].clone()
    greedy = (temperature <= 0)[:, None]
    t = torch.where(greedy, 1.0, temperature.double()[:, None])
    index = torch.arange(vocab, device=dev)

    def softmax(x):
        e = (x.double() / t - (x.double() / t).amax(1, keepdim=True)).exp()
        return e / e.sum(1, keepdim=True)

    def target(rows):
        return torch.where(greedy, (index == logits[rows].argmax(1)[:, None]).double(), softmax(logits[rows]))

    r = target(at)
    q = softmax(draft[at]) if draft is not None else None
    path = torch.full((tokens.shape[0],), -1, dtype=torch.int32, device=dev)
    path[at] = 0
    count = torch.ones(requests, dtype=torch.int64, device=dev)
    for place in range(1, nodes):      # nodes stand behind their parents and siblings in order: one pass over the places is the walk
        row = (seg[:, 0] + place).clamp_max(tokens.shape[0] - 1)
        child = (place < seg[:, 1]) & (par[row] == at - seg[:, 0])
        x = tok[row]
        px = r[each, x]
        qx = q[each, x] if q is not None else torch.ones_like(px)
        accept = child & torch.where(greedy[:, 0], px > 0, uniform[row] * qx < px)
        reject = (child & ~accept & ~greedy[:, 0])[:, None]
        path[torch.where(accept, seg[:, 0] + count, seg[:, 0])] = torch.where(accept, place, 0).int()
        count += accept
        at = torch.where(accept, row, at)
        one = (index == x[:, None]).double()
        rest = (r - q).clamp_min_(0) if q is not None else r * (1 - one)
        mass = rest.sum(1, keepdim=True)
        r = torch.where(reject & (mass > 0), rest / mass, r)
        if q is not None:
            left = q * (1 - one)
            mass = left.sum(1, keepdim=True)
            q = torch.where(reject, left / torch.where(mass > 0, mass, 1.0), q)
            q = torch.where(accept[:, None], softmax(draft[at]), q)
        r = torch.where(accept[:, None], target(at), r)
    run_ = r.cumsum(1)
    sampled = (run_ <= (uniform[seg[:, 0]] * run_[:, -1])[:, None]).sum(1).clamp_max(vocab - 1)
    return path, count.int(), torch.where(greedy[:, 0], r.argmax(1), sampled).int()


def keep(pool, table, seg, path, count):
    """Place start + path[k] -> start + k for k < count, all sources read before a destination is written."""
    seg, page = seg.long(), pool.shape[4]
    row = torch.arange(path.shape[0], device=pool.device)
    request = (row[:, None] >= seg[:, 0]).sum(1) - 1
    k = row - seg[request, 0]
    stays = k < count.long()[request]
    request, k, path = request[stays], k[stays], path.long()[stays]
    src, dst = seg[request, 2] + path, seg[request, 2] + k
    table = table.long()
    moved = pool[:, table[request, src // page], :, :, src % page]
    pool[:, table[request, dst // page], :, :, dst % page] = moved


# ---- the work that no form of a pass can do without

def work(case):
    heads, kv, hd, layers, vocab = SIZES[case["model"]]
    size = 2 if case.get("dtype") == "bfloat16" else 4
    if case["op"] == "copy":
        return {"bytes": 2 * case["pages"] * layers * 2 * kv * case["page"] * hd * size, "flops": 0}
    counts = node_counts(case)
    if case["op"] == "keep":
        rows = sum(_kept(i, n) - 1 for i, n in enumerate(counts))      # (the root stays where it is)
        return {"bytes": 2 * rows * layers * 2 * kv * hd * size + 8 * len(counts), "flops": 0}
    if case["op"] == "attend":
        keys = [min(s, case["window"]) if case["window"] else s for s in spread(case["context"], case["requests"])]
        depth = 1 + (case["nodes"] / 2 if case["chain"] else math.log2(case["nodes"] + 1) / 1.5)      # nodes that a node sees, about
        return {"bytes": sum(k + n for k, n in zip(keys, counts)) * 2 * kv * hd * size + 2 * sum(counts) * heads * hd * size,
                "flops": sum(4 * n * (k + depth) for k, n in zip(keys, counts)) * heads * hd}
    # the rows of the root and of what is accepted: about two nodes of a longer tree on these logits, about one without a drafter (a
    # greedy request needs no drafter's rows)
    visited = 3 if case["drafter"] else 2
    rows = sum(min(n, visited) * (1 + (1 if case["drafter"] and i % 5 != 4 else 0)) for i, n in enumerate(counts))
    return {"bytes": rows * vocab * 4 + sum(counts) * 20 + 8 * len(counts), "flops": rows * vocab * 4}


# ---- what a pass gives, from the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        pool, src, dst = s["pool"], s["src"].cpu().tolist(), s["dst"].cpu().tolist()
        was = pool.clone()
        for a, b in zip(src, dst):
            pool[:, b].copy_(was[:, a])
        return pool.double() if pool.numel() < 1 << 28 else None
    seg = s["seg"].cpu().numpy() if "seg" in s else s["meta"].seg.cpu().numpy()
    if case["op"] == "keep":
        pool, table, path, count = s["pool"], s["table"].cpu().numpy(), s["path"].cpu().numpy(), s["count"].cpu().numpy()
        was, page = pool.clone(), case["page"]
        for i, (row0, n, start, _) in enumerate(seg):
            for k in range(count[i]):
                a, b = start + path[row0 + k], start + k
                pool[:, int(table[i, b // page]), :, :, int(b % page)] = was[:, int(table[i, a // page]), :, :, int(a % page)]
        return pool.double() if pool.numel() < 1 << 28 else None
    if case["op"] == "verify":
        return _exact_verify(s, seg)
    heads, kv, hd, _, _ = SIZES[case["model"]]
    m, page, window = s["meta"], case["page"], case["window"]
    out = torch.zeros((s["q"].shape[0], heads, hd), dtype=torch.float64, device="cuda")
    pos, bits = m.pos.cpu().numpy(), m.ancestors.cpu().numpy().view(np.uint32)
    for i, (row0, n, start, _) in enumerate(seg):
        pages = m.tables[i, :-(-(start + n) // page)].long()
        k = s["cache"].keys[pages].double().transpose(1, 2).reshape(-1, kv, hd)[:start + n]
        v = s["cache"].values[pages].double().transpose(1, 2).reshape(-1, kv, hd)[:start + n]
        allowed = np.zeros((n, start + n), bool)
        for j in range(n):
            lo = max(0, pos[row0 + j] - window + 1) if window else 0
            allowed[j, lo:start] = True
            for a in range(n):
                allowed[j, start + a] = bool(bits[row0 + j, a // 32] >> np.uint32(a % 32) & np.uint32(1))
        allowed = torch.from_numpy(allowed).cuda()
        for h in range(heads):
            g = h // (heads // kv)
            w = s["q"][row0:row0 + n, h * hd:(h + 1) * hd].double() @ k[:, g].T * s["scale"]
            w = torch.softmax(w.masked_fill(~allowed, -math.inf), -1)
            out[row0:row0 + n, h] = w @ v[:, g]
    return out.view(-1, heads * hd)


def _exact_verify(s, seg):
    """Request by request and child by child, in numpy."""
    temperature, uniform = s["temperature"].cpu().numpy(), s["uniform"].cpu().numpy()
    tokens, parents = s["tokens"].cpu().numpy(), s["parents"].cpu().numpy()
    path, count, last = np.full(len(tokens), -1, np.int32), np.zeros(len(seg), np.int32), np.zeros(len(seg), np.int32)

    def softmax(x, t):
        e = np.exp(x.cpu().numpy().astype(np.float64) / t - float(x.max()) / t)
        return e / e.sum()

    for i, (row0, n, _, _) in enumerate(seg):
        t, node, kept = float(temperature[i]), 0, [0]
        while True:
            children = [j for j in range(1, n) if parents[row0 + j] == node]
            taken = None
            if t <= 0:
                r, best = None, int(s["logits"][row0 + node].cpu().numpy().argmax())
                taken = next((j for j in children if tokens[row0 + j] == best), None)
            else:
                r = softmax(s["logits"][row0 + node], t)
                q = softmax(s["draft"][row0 + node], t) if s["draft"] is not None and children else None
                for j in children:
                    x = tokens[row0 + j]
                    if uniform[row0 + j] * (1.0 if q is None else q[x]) < r[x]:
                        taken = j
                        break
                    if q is None:
                        rest = r.copy()
                        rest[x] = 0.0
                    else:
                        rest = np.maximum(r - q, 0.0)
                        q = q.copy()
                        q[x] = 0.0
                        q /= q.sum() or 1.0
                    r = rest / rest.sum() if rest.sum() > 0 else r
            if taken is None:
                break
            node = taken
            kept.append(node)
        path[row0:row0 + len(kept)] = kept
        count[i] = len(kept)
        if t <= 0:
            last[i] = best
        else:
            total = np.cumsum(r)
            last[i] = min(int(np.searchsorted(total, uniform[row0] * total[-1], side="right")), len(total) - 1)
    return path, count, last
