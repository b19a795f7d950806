"""The kernels for drafted tokens against their definitions in 64 bits (`plain_drafts`), where they can go wrong: trees and chains of
one node and more, empty contexts, contexts that end inside a page and inside a key tile, windows, rows that see nothing, places
that hold no numbers, odd groups and head sizes, vocabularies that no vector divides."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import plain_drafts as plain

pytestmark = pytest.mark.gpu
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
NAN = float("nan")


def ops_of(dtype):
    from fusezap_core_b200.kernels import cuda_ops
    return cuda_ops(dtype)


def chain(n):
    return [i - 1 for i in range(n)]


def bushy(n, seed=0):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]


# ---------------------------------------------------------------------------------------------- attention

def tree_case(dtype, heads, kv, hd, page, requests, window=0, pad=0, seed=0, words=None, spare=3, poison=True):
    """requests: (places before the tree, parents) each, or (places, None) for one that has no rows in the step. Every place of the
    pool that belongs to no request's context or tree holds NaN."""
    gen = torch.Generator().manual_seed(seed)
    counts = [len(p) if p is not None else 0 for _, p in requests]
    need = [-(-(b + n) // page) for (b, _), n in zip(requests, counts)]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen).tolist()
    table = torch.full((len(requests), max(need + [1]) + 1), -1, dtype=torch.int32)
    pool = torch.full((total, 2, kv, page, hd), NAN if poison else 7.0)
    seg = torch.zeros(len(requests), 4, dtype=torch.int32)
    n_rows = sum(counts) + pad
    words = words or max(1, -(-max(counts) // 32))
    pos, row, bits = torch.zeros(n_rows, dtype=torch.int32), torch.full((n_rows,), -1, dtype=torch.int32), np.zeros((n_rows, words), np.int32)
    at = taken = 0
    for s, ((b, parents), n) in enumerate(zip(requests, counts)):
        pages = order[taken:taken + need[s]]
        taken += need[s]
        table[s, :need[s]] = torch.tensor(pages, dtype=torch.int32)
        for place in range(b + n):
            pool[pages[place // page], :, :, place % page] = torch.randn(2, kv, hd, generator=gen)
        if parents is None:
            continue
        seg[s] = torch.tensor([at, n, b, -1])
        pos[at:at + n] = torch.tensor([b + d for d in plain.depths_of(parents)])
        row[at:at + n] = s
        bits[at:at + n] = plain.ancestors_of(parents, words)
        if window:      # pages that lie wholly before every row's window are given back
            for pi in range(max(0, b - window + 1) // page):
                table[s, pi] = -1
        at += n
    q = torch.randn(n_rows, heads * hd, generator=gen) * 2
    meta = SimpleNamespace(pos=pos, seq_row=row, seg=seg, ancestors=torch.from_numpy(bits), tables=table,
                           max_context=max([b + n for (b, _), n in zip(requests, counts)]))
    return SimpleNamespace(q=q.to(DT[dtype]), pool=pool.to(DT[dtype]), meta=meta, heads=heads, kv=kv, hd=hd, page=page, window=window,
                           scale=hd ** -0.5, dtype=dtype)


def on_gpu(c):
    m = c.meta
    meta = SimpleNamespace(pos=m.pos.cuda(), seq_row=m.seq_row.cuda(), seg=m.seg.cuda(), ancestors=m.ancestors.cuda(), max_context=m.max_context)
    tables = m.tables.cuda()
    meta.table = lambda group: tables
    pool = c.pool.cuda()
    cache = SimpleNamespace(keys=pool[:, 0], values=pool[:, 1], page_size=c.page, group=0, write=True)
    return c.q.cuda(), cache, meta


def run_tree(c, ops=None):
    q, cache, meta = on_gpu(c)
    out = torch.full_like(q, NAN)
    ops = ops or ops_of(c.dtype)
    ops.tree_attention(q, cache, meta, out, c.heads, c.kv, c.hd, c.scale, c.window)
    ops.check_errors()
    return out


def reference(c):
    m = c.meta
    return plain.attend(c.q, c.pool[:, 0], c.pool[:, 1], m.tables, m.seg, m.pos, m.seq_row, m.ancestors, c.heads, c.kv, c.hd, c.scale, c.window)


def tree_tolerance(c, ref, size):
    """Per value. A score is off by at most ds = (hd + 4) half steps of float32 times |q| |k| scale (and the exponent's own rounding),
    which makes weights relatively 2 ds wrong together with their sum; the sums over L places are off by (L + 64) half steps relative to
    sum w |v| (64: pieces, the division). bfloat16: the output's one rounding, and the weights' rounding to bfloat16 in the tensor-core
    kernel, each half a step of 2^-8."""
    unit = 2.0 ** -24
    q = c.q.float().view(-1, c.hd).norm(dim=1).max()
    finite = torch.nan_to_num(c.pool[:, 0].float(), nan=0.0, posinf=0.0, neginf=0.0)
    k = finite.reshape(-1, c.hd).norm(dim=1).max()
    ds = (c.hd + 4) * unit * float(q * k) * c.scale
    tol = (2 * ds + (c.meta.max_context + 64) * unit) * size + 1e-30
    return tol + (2.0 ** -8 * (ref.abs() + size) if c.dtype == "bfloat16" else unit * ref.abs())


def assert_tree(c, out, rows=slice(None)):
    ref, size = reference(c)
    got, ref, size = out.double().cpu()[rows], ref[rows], size[rows]
    assert torch.isfinite(got).all(), "not finite"
    over = (got - ref).abs() - tree_tolerance(c, ref, size)
    assert over.max() <= 0, f"off by {float((got - ref).abs().max()):.3e}, {float(over.max()):.3e} more than allowed, at {int(over.argmax())}"


SIZES = [(4, 4, 64), (14, 2, 64), (32, 8, 128), (10, 2, 128), (3, 1, 32), (6, 2, 48), (40, 1, 128), (8, 2, 256), (2, 1, 512), (4, 2, 16)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,hd", SIZES)
def test_tree_attention_sizes(dtype, heads, kv, hd):
    c = tree_case(dtype, heads, kv, hd, 16, [(37, bushy(9)), (0, bushy(5, 1)), (130, chain(3)), (300, [-1])], pad=3)
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [1, 3, 4, 8, 16, 24, 48, 64])
def test_tree_attention_pages(dtype, page):
    c = tree_case(dtype, 8, 2, 64, page, [(127, bushy(6)), (128, bushy(7, 1)), (129, bushy(8, 2)), (16, bushy(17, 3)), (257, chain(4))])
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("start", [0, 1, 15, 16, 17, 63, 64, 100, 127, 128, 256, 383, 1000])
def test_tree_attention_context_lengths(dtype, start):
    c = tree_case(dtype, 8, 2, 128, 16, [(start, bushy(11)), (start + 5, [-1])])
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 64, 100, 257])
@pytest.mark.parametrize("shape", [chain, bushy])
def test_tree_attention_nodes(dtype, nodes, shape):
    c = tree_case(dtype, 6, 2, 64, 16, [(90, shape(nodes)), (200, shape(max(1, nodes // 3)))], pad=2)
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 129, 500])
def test_tree_attention_windows(dtype, window):
    c = tree_case(dtype, 8, 2, 64, 16, [(333, bushy(9)), (40, chain(12)), (64, bushy(5)), (0, chain(3)), (1000, chain(7))], window=window)
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_long_contexts(dtype):
    c = tree_case(dtype, 8, 2, 128, 16, [(5000, bushy(20)), (3001, bushy(33)), (20, chain(2))])
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("heads,kv,hd,page", [(32, 8, 128, 16), (10, 2, 128, 8), (14, 2, 64, 16), (8, 1, 64, 32)])
def test_tree_attention_more_rows_than_a_tile(heads, kv, hd, page):
    """Steps whose requests have more than 128 rows per kv head on average, beside some that have few, none or one tile too many."""
    G = heads // kv
    full, many = 128 // G, 1 + 300 // G
    c = tree_case("bfloat16", heads, kv, hd, page, [(300, bushy(many)), (700, bushy(2 * full, 1)), (129, bushy(2 * full + 1, 2)), (50, [-1]), (0, bushy(many, 3)),
                                                    (1500, bushy(3 * full, 4)), (128, bushy(4 * full + 3, 5)), (77, None)], pad=2)
    assert c.q.shape[0] * G > 128 * 8
    assert_tree(c, run_tree(c))
    c = tree_case("bfloat16", heads, kv, hd, page, [(333, bushy(many)), (40, chain(full + 5))], window=90 + full)
    assert_tree(c, run_tree(c))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_many_requests_and_empty_ones(dtype):
    rng = np.random.default_rng(5)
    reqs = [(int(rng.integers(0, 200)), None if i % 7 == 3 else bushy(int(rng.integers(1, 8)), i)) for i in range(70)]
    c = tree_case(dtype, 4, 2, 64, 16, reqs, pad=5)
    out = run_tree(c)
    assert_tree(c, out)
    assert (out[-5:] == 0).all()


def test_tree_attention_requests_that_share_rows_are_reported():
    """Two requests that name the same rows: the scratch has room for every row once."""
    from fusezap_core_b200.kernels.table import KernelError
    c = tree_case("bfloat16", 8, 2, 64, 16, [(300, bushy(30)), (300, bushy(30, 1))])
    c.meta.seg[0] = c.meta.seg[1]
    c.meta.seg[:, 0], c.meta.seg[:, 1] = 0, 60
    q, cache, meta = on_gpu(c)
    ops = ops_of("bfloat16")
    ops.tree_attention(q, cache, meta, torch.empty_like(q), c.heads, c.kv, c.hd, c.scale, 0)
    with pytest.raises(KernelError, match="outside the step"):
        ops.check_errors()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_rows_that_see_nothing(dtype):
    c = tree_case(dtype, 8, 2, 64, 16, [(0, bushy(6)), (50, bushy(6))])
    c.meta.ancestors[2] = 0
    c.meta.ancestors[8] = 0           # still sees its context
    c.meta.ancestors[9] = -1          # bits beyond the tree's rows count as unset
    out = run_tree(c)
    assert (out[2] == 0).all()
    assert_tree(c, out)


# what no request's (first row, rows, first place) is, by field
BAD_SEGMENTS = [(0, -4), (0, 2 ** 31 - 3), (1, 2 ** 31 - 1), (1, 60), (2, -100), (2, 2 ** 31 - 1)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("field,value", BAD_SEGMENTS)
def test_tree_attention_reports_requests_outside_the_step(dtype, field, value):
    from fusezap_core_b200.kernels.table import KernelError
    c = tree_case(dtype, 8, 2, 64, 16, [(45, bushy(6)), (150, bushy(9)), (20, bushy(5))], pad=2)
    good = [*range(6), *range(15, 22)]
    c.meta.seg[1, field] = value
    q, cache, meta = on_gpu(c)
    out = torch.full_like(q, NAN)
    ops = ops_of(dtype)
    ops.tree_attention(q, cache, meta, out, c.heads, c.kv, c.hd, c.scale, 0)
    with pytest.raises(KernelError, match="outside the step"):
        ops.check_errors()
    assert (out[6:15] == 0).all()
    c.meta.seg[1] = torch.tensor([6, 9, 150, -1])
    assert_tree(c, out, good)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_tree_attention_unseen_places_take_no_part(dtype, bad):
    parents = [-1, 0, 0, 1, 2]
    c = tree_case(dtype, 8, 2, 64, 16, [(45, parents), (20, parents)])
    place = 45 + 2
    c.pool[c.meta.tables[0, place // 16].long(), :, :, place % 16] = bad
    sees = [2, 4]
    out = run_tree(c)
    assert not torch.isfinite(out[sees].float()).any()
    c.pool[c.meta.tables[0, place // 16].long(), :, :, place % 16] = 1.0
    assert_tree(c, out, [i for i in range(10) if i not in sees])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_places_before_the_window_take_no_part(dtype):
    c = tree_case(dtype, 8, 2, 64, 16, [(333, chain(9))], window=70)
    # place 264 is seen by the first two rows (positions 333 and ..: 333 - 70 + 1 = 264), 263 by none
    for place in (263, 256):
        c.pool[c.meta.tables[0, place // 16].long(), :, :, place % 16] = NAN
    out = run_tree(c)
    assert_tree(c, out)
    place = 264
    c.pool[c.meta.tables[0, place // 16].long(), :, :, place % 16] = NAN
    out = run_tree(c)
    assert not torch.isfinite(out[0].float()).any()
    c.pool[c.meta.tables[0, place // 16].long(), :, :, place % 16] = 1.0
    assert_tree(c, out, list(range(1, 9)))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_large_scores(dtype):
    c = tree_case(dtype, 8, 2, 64, 16, [(150, bushy(9)), (700, chain(3))], poison=False)
    c.q *= 16
    c.pool[:, 0] *= 4
    assert_tree(c, run_tree(c))


def test_tree_attention_float32_rows_do_not_depend_on_the_step():
    reqs = [(300, bushy(9)), (2000, chain(4)), (77, bushy(30, 2)), (0, [-1])]
    c = tree_case("float32", 14, 2, 64, 16, reqs, seed=3)
    whole = run_tree(c)
    at = 0
    for s, (b, parents) in enumerate(reqs):
        n = len(parents)
        m = c.meta
        seg = m.seg[s:s + 1].clone()
        seg[0, 0] = 0
        alone = SimpleNamespace(**{**vars(c), "q": c.q[at:at + n], "meta": SimpleNamespace(
            pos=m.pos[at:at + n], seq_row=torch.zeros(n, dtype=torch.int32), seg=seg, ancestors=m.ancestors[at:at + n], tables=m.tables[s:s + 1],
            max_context=m.max_context)})
        assert torch.equal(run_tree(alone), whole[at:at + n])
        at += n


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [0, 2000])
def test_tree_attention_float32_rows_are_the_same_in_either_tile(hd, window):
    """A step of 44 rows by 7 heads and 32 pieces, whose tiles have 64 rows (more than 16 a request, and 512 blocks), against its requests one
    by one, whose tiles have 16 (256 blocks at most)."""
    reqs = [(300, bushy(9)), (2900, chain(4)), (1700, bushy(30, 2)), (0, [-1])]
    c = tree_case("float32", 14, 2, hd, 16, reqs, window=window, seed=4)
    whole, at, m = run_tree(c), 0, c.meta
    assert_tree(c, whole)
    for s, (b, parents) in enumerate(reqs):
        n, seg = len(parents), m.seg[s:s + 1].clone()
        seg[0, 0] = 0
        alone = SimpleNamespace(**{**vars(c), "q": c.q[at:at + n], "meta": SimpleNamespace(
            pos=m.pos[at:at + n], seq_row=torch.zeros(n, dtype=torch.int32), seg=seg, ancestors=m.ancestors[at:at + n], tables=m.tables[s:s + 1],
            max_context=m.max_context)})
        assert torch.equal(run_tree(alone), whole[at:at + n])
        at += n


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_replayed_with_other_lengths(dtype):
    """One recorded call, replayed after the metadata, the queries and the cache have changed under it."""
    a = tree_case(dtype, 8, 2, 128, 16, [(900, bushy(9)), (40, chain(7))], seed=1)
    b = tree_case(dtype, 8, 2, 128, 16, [(33, bushy(9, 4)), (880, chain(7))], seed=2, spare=3 + 0)
    pages = max(a.pool.shape[0], b.pool.shape[0])
    grow = lambda p: torch.cat([p, torch.full((pages - p.shape[0], *p.shape[1:]), NAN, dtype=p.dtype)])
    a.pool, b.pool = grow(a.pool), grow(b.pool)
    width = max(a.meta.tables.shape[1], b.meta.tables.shape[1])
    for c in (a, b):
        c.meta.tables = torch.cat([c.meta.tables, torch.full((2, width - c.meta.tables.shape[1]), -1, dtype=torch.int32)], 1)
        c.meta.max_context = 1000
    ops = ops_of(dtype)
    q, cache, meta = on_gpu(a)
    out = torch.empty_like(q)
    ops.tree_attention(q, cache, meta, out, 8, 2, 128, a.scale, 0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.tree_attention(q, cache, meta, out, 8, 2, 128, a.scale, 0)
    q2, cache2, meta2 = on_gpu(b)
    q.copy_(q2)
    cache.keys.copy_(cache2.keys)
    cache.values.copy_(cache2.values)
    for name in ("pos", "seq_row", "seg", "ancestors"):
        getattr(meta, name).copy_(getattr(meta2, name))
    meta.table(0).copy_(meta2.table(0))
    out.fill_(NAN)
    g.replay()
    ops.check_errors()
    assert_tree(b, out)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_attention_on_two_streams_at_once(dtype):
    cases = [tree_case(dtype, 8, 2, 128, 16, [(900 + 50 * i, bushy(9, i)), (40, chain(7))], seed=i) for i in range(2)]
    ops, streams, outs, keep = ops_of(dtype), [torch.cuda.Stream() for _ in cases], [], []
    for c, s in zip(cases, streams):
        keep.append(on_gpu(c))
        outs.append(torch.empty_like(keep[-1][0]))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, (q, cache, meta), out in zip(cases, streams, keep, outs):
            with torch.cuda.stream(s):
                ops.tree_attention(q, cache, meta, out, 8, 2, 128, c.scale, 0)
    torch.cuda.synchronize()
    ops.check_errors()
    for c, out in zip(cases, outs):
        assert_tree(c, out)


# ---------------------------------------------------------------------------------------------- verdict

def verify_case(vocab, trees, drafter, seed=0, spread=2.0, error=0.5, greedy=lambda s: s % 4 == 3, pad=0):
    """trees: parents of each request (an empty list: no rows). Children are drawn from the drafter without replacement, as far as the
    vocabulary goes."""
    rng = np.random.default_rng(seed)
    n = sum(len(t) for t in trees) + pad
    logits = (rng.standard_normal((n, vocab)) * spread).astype(np.float32)
    draft = (logits + rng.standard_normal((n, vocab)) * error).astype(np.float32)
    seg, parents, tokens, temperature = np.zeros((len(trees), 4), np.int32), np.full(n, -1, np.int32), np.zeros(n, np.int32), np.zeros(len(trees), np.float32)
    at = 0
    for s, t in enumerate(trees):
        seg[s] = (at, len(t), 1000 * s, -1)
        temperature[s] = 0.0 if greedy(s) else 0.5 + 0.25 * (s % 3)
        drawn = {}
        for j, p in enumerate(t):
            parents[at + j] = p
            if p < 0:
                tokens[at + j] = rng.integers(vocab)
                continue
            z = draft[at + p] / (temperature[s] or 0.3) + rng.gumbel(size=vocab)
            z[drawn.setdefault(p, [])] = -np.inf
            tokens[at + j] = int(z.argmax())
            if len(drawn[p]) + 1 < vocab:
                drawn[p].append(tokens[at + j])
        at += len(t)
    return dict(logits=logits, draft=draft if drafter else None, temperature=temperature, uniform=rng.random(n), tokens=tokens, parents=parents, seg=seg)


def run_verify(c):
    n, S = len(c["tokens"]), len(c["seg"])
    dev = {k: None if v is None else torch.from_numpy(v).cuda() for k, v in c.items()}
    out = [torch.full((k,), -7, dtype=torch.int32, device="cuda") for k in (n, S, S)]
    ops = ops_of("float32")
    ops.verify_tree(dev["logits"], dev["draft"], dev["temperature"], dev["uniform"], dev["tokens"], dev["parents"], dev["seg"], *out)
    ops.check_errors()
    return [t.cpu().numpy() for t in out]


def assert_verify(c):
    path, count, ids = run_verify(c)
    rpath, rcount, rids = plain.verify(c["logits"], c["draft"], c["temperature"], c["uniform"], c["tokens"], c["parents"], c["seg"])
    rows = np.zeros(len(path), bool)
    for row0, n, *_ in c["seg"]:
        rows[row0:row0 + n] = True
    np.testing.assert_array_equal(count, rcount)
    np.testing.assert_array_equal(ids, rids)
    np.testing.assert_array_equal(path[rows], rpath[rows])
    assert (path[~rows] == -7).all(), "a row beside the requests' was written"
    return count


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 257, 1024, 4099, 32000, 50021, 128256])
def test_verify_vocabularies(vocab, drafter):
    assert_verify(verify_case(vocab, [bushy(9), chain(5), [-1], bushy(14, 3), chain(4), [-1, 0, 0, 0, 0]], drafter, seed=vocab, pad=2))


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("requests", [1, 14, 15, 33, 75, 300])
def test_verify_requests(requests, drafter):
    c = verify_case(4500 * 8 if requests < 40 else 8200, [[] if s % 9 == 5 else bushy(1 + s % 7, s) for s in range(requests)], drafter, seed=requests)
    count = assert_verify(c)
    assert not drafter or requests < 14 or count.max() > 2      # (the walk went somewhere)


@pytest.mark.parametrize("drafter", [True, False])
def test_verify_many_siblings(drafter):
    """A drafter that is far off: most children fall, and p and q shrink child by child."""
    trees = [[-1] + [0] * 12 + [1, 1, 5, 5, 12, 12, 13, 15]] * 6
    assert_verify(verify_case(600, trees, drafter, seed=3, spread=1.0, error=2.5, greedy=lambda s: False))
    assert_verify(verify_case(7, [[-1] + [0] * 9] * 40, drafter, seed=4, spread=1.0, error=2.0, greedy=lambda s: False))


def test_verify_drafter_equal_to_the_target_keeps_its_first_children():
    c = verify_case(3000, [chain(8), bushy(20)] * 3, True, error=0.0, greedy=lambda s: False)
    c["draft"] = c["logits"].copy()
    assert (assert_verify(c)[::2] == 8).all()


def test_verify_tokens_left_out():
    """Logits of -inf (tokens filtered away) at the start of every lane's run, the rows' ends, and all but one."""
    c = verify_case(5000, [bushy(9), chain(5), bushy(7, 2)], True, seed=9, greedy=lambda s: s == 1)
    c["logits"][:, :3000] = -np.inf
    c["draft"][:, 4000:] = -np.inf
    c["logits"][3, :] = -np.inf
    c["logits"][3, 17] = 0.5
    c["draft"][5, :] = -np.inf
    c["draft"][5, 4999] = -3.0
    assert_verify(c)


def test_verify_rows_without_a_distribution():
    for bad in (NAN, np.inf, None):
        c = verify_case(5000, [chain(3), bushy(5)], False, seed=10, greedy=lambda s: False)
        for row in (0, 3):
            if bad is None:
                c["logits"][row] = -np.inf
            else:
                c["logits"][row, 4321] = bad
        count = assert_verify(c)
        assert (count == 1).all()
    c = verify_case(5000, [chain(3)], False, seed=11, greedy=lambda s: True)      # greedy: a NaN is the maximum, as in argmax
    c["logits"][0, 77] = NAN
    c["tokens"][1] = 77
    assert assert_verify(c)[0] >= 2


def test_verify_numbers_at_their_ends():
    c = verify_case(4096 * 9, [chain(4)] * 20, True, seed=12, greedy=lambda s: False)
    c["uniform"][:40] = 0.0
    c["uniform"][40:] = 1.0 - 2.0 ** -53
    assert_verify(c)


def test_verify_small_and_large_temperatures():
    c = verify_case(20000, [bushy(6, s) for s in range(8)], True, seed=13, greedy=lambda s: False)
    c["temperature"][:] = [1e-3, 0.01, 0.1, 1.0, 3.0, 30.0, 1e3, 1e-2]
    assert_verify(c)


def test_verify_temperatures_at_the_ends_of_float32():
    c = verify_case(20000, [bushy(6, s) for s in range(8)], False, seed=15, greedy=lambda s: False)
    c["logits"][:, 100:9000] = -np.inf
    c["temperature"][:] = [1e-45, 1e-38, 1e-30, 1e-10, 1e10, 1e30, 1e-3, 1e4]
    assert_verify(c)
    few = run_verify(c | dict(temperature=np.full(8, 1e30, np.float32)))
    for t in (1e35, np.inf):      # (above 1e30: as 1e30)
        for a, b in zip(run_verify(c | dict(temperature=np.full(8, t, np.float32))), few):
            np.testing.assert_array_equal(a, b)


def test_verify_masks_of_the_lowest_value():
    """-inf beside the lowest finite value, alone and under ordinary logits; and rows of large logits."""
    low = np.finfo(np.float32).min
    c = verify_case(9000, [bushy(7, s) for s in range(6)], True, seed=16, greedy=lambda s: False)
    c["logits"][:, 2000:5000], c["logits"][:, 6000:] = low, -np.inf
    for row in (0, 7, 14):      # (roots: nothing else in the row)
        c["logits"][row] = np.where(np.arange(9000) % 3 == 0, np.float32(low), np.float32(-np.inf))
    c["draft"][7] = np.where(np.arange(9000) % 2 == 0, np.float32(low), np.float32(-np.inf))
    c["logits"][21, :2000] *= 1e30
    c["logits"][28] += 3e7
    assert_verify(c)


def test_verify_refuses_vocabularies_above_eight_million():
    from fusezap_core_b200.kernels.table import KernelError
    vocab = (8 << 20) + 4
    logits = torch.zeros((1, vocab), device="cuda")
    out = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(5)]
    seg = torch.tensor([[0, 1, 0, 0]], dtype=torch.int32, device="cuda")
    with pytest.raises(KernelError):
        ops_of("float32").verify_tree(logits, None, torch.ones(1, device="cuda"), torch.zeros(1, dtype=torch.float64, device="cuda"), out[0], out[1] - 1, seg, *out[2:])


@pytest.mark.parametrize("drafter", [True, False])
def test_verify_keeps_the_targets_distribution(drafter):
    """Over many requests the first token behind the root (a child that stands, or the draw) is distributed as softmax(logits / T):
    each token's share within five standard deviations."""
    vocab, requests, t = 6, 20000, 0.7
    rng = np.random.default_rng(14)
    logits, draft = rng.standard_normal(vocab).astype(np.float32), rng.standard_normal(vocab).astype(np.float32)
    q = plain.softmax64(draft, t)
    first = rng.choice(vocab, requests, p=q)
    left = np.where(np.arange(vocab) == first[:, None], 0.0, q)
    second = (rng.random((requests, 1)) > np.cumsum(left / left.sum(1, keepdims=True), 1)).sum(1)
    n = 3 * requests
    tokens = np.stack([np.zeros(requests), first, second], 1).astype(np.int32).reshape(-1)
    c = dict(logits=np.tile(logits, (n, 1)), draft=np.tile(draft, (n, 1)) if drafter else None, temperature=np.full(requests, t, np.float32),
             uniform=rng.random(n), tokens=tokens, parents=np.tile(np.array([-1, 0, 0], np.int32), requests),
             seg=np.stack([3 * np.arange(requests), np.full(requests, 3), np.zeros(requests), np.zeros(requests)], 1).astype(np.int32))
    path, count, ids = run_verify(c)
    got = np.where(count > 1, tokens[3 * np.arange(requests) + np.maximum(path[1::3], 0)], ids)
    p = plain.softmax64(logits, t)
    share = np.bincount(got, minlength=vocab) / requests
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / requests)).all(), (share, p)


def test_verify_reports_bad_trees():
    from fusezap_core_b200.kernels.table import KernelError
    c = verify_case(100, [chain(3), chain(3)], False, greedy=lambda s: False)
    c["tokens"][1] = 100
    with pytest.raises(KernelError, match="embedding table"):
        run_verify(c)
    c = verify_case(100, [chain(1025), chain(2)], False, greedy=lambda s: True)
    with pytest.raises(KernelError, match="outside the step"):
        run_verify(c)
    c = verify_case(100, [chain(3)], False)
    c["seg"][0, 1] = 4
    with pytest.raises(KernelError, match="outside the step"):
        run_verify(c)


# ---- verdicts: requests that are none beside sound ones, and sums near their borders

@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("bad", [(0, 2 ** 31 - 1), (0, 17), (-4, 20), (-(2 ** 31), 2 ** 31 - 1), (-(2 ** 31), 2 ** 31 - 8), (2 ** 31 - 1, 3), (3, 0), (2, -7)])
def test_verify_beside_requests_that_are_none(bad, drafter):
    """A first request whose rows do not lie in the step but would cover the others': it alone has no verdict. Steps whose rows' statistics
    are taken ahead of the walks (2 to 6 rows a request), the scratch holding what it likes."""
    from fusezap_core_b200.kernels.table import KernelError
    c = verify_case(3000, [chain(4), bushy(4, 1), chain(4), bushy(4, 2)], drafter, seed=21, greedy=lambda s: s == 2)
    c["seg"][0, :2] = bad
    dev = {k: None if v is None else torch.from_numpy(v).cuda() for k, v in c.items()}
    out = [torch.full((k,), -7, dtype=torch.int32, device="cuda") for k in (16, 4, 4)]
    ops = ops_of("float32")
    garbage = [torch.full((16 * 24 * k,), 255, dtype=torch.uint8, device="cuda") for k in (1, 2, 4)]
    del garbage
    ops.verify_tree(dev["logits"], dev["draft"], dev["temperature"], dev["uniform"], dev["tokens"], dev["parents"], dev["seg"], *out)
    if bad[1] > 0:
        with pytest.raises(KernelError, match="outside the step"):
            ops.check_errors()
    ops.check_errors()
    path, count, ids = (t.cpu().numpy() for t in out)
    c["seg"][0, :2] = 0
    rpath, rcount, rids = plain.verify(c["logits"], c["draft"], c["temperature"], c["uniform"], c["tokens"], c["parents"], c["seg"])
    np.testing.assert_array_equal(count, rcount)
    np.testing.assert_array_equal(ids, rids)
    np.testing.assert_array_equal(path[4:], rpath[4:])
    assert (path[:4] == -7).all()


def test_verify_draws_at_a_rounding_from_the_border():
    """Rows of two tokens and numbers just below and above the first one's share, taken to 40 digits. The share is off by at most
    1.7e-15 of itself: a weight exp(-t), t <= 4, by 4 * 2^-52 for its exponent's rounded scale and 6e-16 for the table, the polynomial and
    their products, then a sum and a product. The numbers are 2^-48 = 3.6e-15 away."""
    from decimal import Decimal, localcontext
    rng = np.random.default_rng(22)
    S = 3000
    temperature = rng.uniform(0.5, 2.0, S).astype(np.float32)
    logits = (rng.uniform(-1, 1, (S, 2)) * temperature[:, None]).astype(np.float32)
    above = rng.integers(0, 2, S)
    uniform = np.empty(S)
    with localcontext() as ctx:
        ctx.prec = 40
        for s in range(S):
            share = 1 / (1 + ((Decimal(float(logits[s, 1])) - Decimal(float(logits[s, 0]))) / Decimal(float(temperature[s]))).exp())
            uniform[s] = float(share * (1 + (1 if above[s] else -1) * Decimal(2) ** -48))
    seg = np.stack([np.arange(S), np.ones(S), np.zeros(S), np.zeros(S)], 1).astype(np.int32)
    _, count, ids = run_verify(dict(logits=logits, draft=None, temperature=temperature, uniform=uniform, tokens=np.zeros(S, np.int32),
                                    parents=np.full(S, -1, np.int32), seg=seg))
    assert (count == 1).all()
    np.testing.assert_array_equal(ids, above)


def border_case(rows, seed, sibling, pad=0):
    """rows: (logits, the drafter's logits, token) each: that token is a child and falls; then (`sibling`) a second child or else the draw has
    its number close beside its border, alternately above and below, at the distance that 64 bits resolve: p and q are known to 2^-48 of
    themselves at best (exponents up to 12, a sum), so max(p - q, 0) over its sum `left` to 2^-47 / left in either computation, its running
    sums to vocab 2^-53 more; 2^-42 / left + vocab 2^-51 leaves room for both."""
    rng = np.random.default_rng(seed)
    vocab, n = len(rows[0][0]), 3 if sibling else 2
    S = len(rows)
    N = S * n + pad
    logits, draft = np.zeros((N, vocab), np.float32), np.zeros((N, vocab), np.float32)
    tokens, parents, uniform = np.zeros(N, np.int32), np.full(N, -1, np.int32), rng.random(N)
    for s, (a, b, x) in enumerate(rows):
        at = s * n
        logits[at:at + n], draft[at:at + n], parents[at + 1:at + n] = a, b, 0
        tokens[at + 1], uniform[at + 1] = x, 1.0 - 2.0 ** -53
        p, q = plain.softmax64(a, 1.0), plain.softmax64(b, 1.0)
        assert q[x] > 1.004 * p[x]
        rest = np.maximum(p - q, 0.0)
        left = rest.sum()
        off = (2.0 ** -42 / left + vocab * 2.0 ** -51) * (1 if s % 2 else -1)
        if sibling:
            q[x] = 0.0
            odds = np.where(q > 0, rest / left / np.maximum(q / q.sum(), 1e-300), 0.0)
            could = np.flatnonzero((odds > 1e-3) & (odds < 0.999))
            y = int(could[rng.integers(len(could))])
            # (what one token's odds are known to: its own difference counts, not the whole)
            own = 2.0 ** -42 * p[y] / rest[y]
            tokens[at + 2], uniform[at + 2] = y, odds[y] * (1 + off + np.sign(off) * own)
        else:
            upto = np.cumsum(rest / left)
            could = np.flatnonzero((rest / left > 8 * abs(off)) & (upto < 1 - 8 * abs(off)))
            u = upto[could[rng.integers(len(could))]] + off if len(could) else 0.5
            if np.abs(upto - u).min() >= 0.5 * abs(off):      # (no other border there)
                uniform[at] = u
    seg = np.stack([n * np.arange(S), np.full(S, n), np.zeros(S), np.zeros(S)], 1).astype(np.int32)
    return dict(logits=logits, draft=draft, temperature=np.ones(S, np.float32), uniform=uniform, tokens=tokens, parents=parents, seg=seg)


@pytest.mark.parametrize("ahead", [True, False])
@pytest.mark.parametrize("small,sibling", [(0.3, False), (3.0, True), (3e-3, False), (3e-5, False), (6e-6, False)])
def test_verify_a_token_as_likely_for_the_drafter(small, sibling, ahead):
    """Rows with one token that has much of p and of q, or nearly all, within 1e-7 of the same: whether p exceeds q there is not for float32 sums
    to say. The others, `small` times as likely in all, go round, so that p's and q's sums are the same but for a change of one of them."""
    rng = np.random.default_rng(int(small * 1e7) + sibling)
    rows = []
    for _ in range(2000):
        a = np.concatenate([[0.0], np.log(small * rng.dirichlet(np.ones(5)) + 1e-3 * small)]).astype(np.float32)
        b = a.copy()
        b[1:] = np.roll(a[1:], 1)
        b[3] += np.float32(rng.uniform(-1e-7, 1e-7) / np.exp(float(b[3])))
        p, q = plain.softmax64(a, 1.0), plain.softmax64(b, 1.0)
        falls = [x for x in range(1, 6) if q[x] > 1.01 * p[x]]
        if not falls:
            continue
        if sibling:      # (some token has less of what is left than the drafter has of it)
            rest, q[falls[0]] = np.maximum(p - q, 0.0), 0.0
            odds = rest / rest.sum() / np.maximum(q / q.sum(), 1e-300)
            if not ((odds > 1e-3) & (odds < 0.999)).any():
                continue
        order = rng.permutation(6)
        rows.append((a[order], b[order], int(np.flatnonzero(order == falls[0])[0])))
    assert len(rows) > 400
    assert_verify(border_case(rows, 23, sibling, pad=0 if ahead else 8 * len(rows)))


@pytest.mark.parametrize("requests", [1, 8, 14, 30, 70, 80])
@pytest.mark.parametrize("error", [0.3, 1e-2, 1e-3, 1e-4, 1e-5, 4e-6])
def test_verify_drafters_near_the_target(error, requests):
    """The drafter's logits are the target's but for `error`, and one unlikely token's that falls; numbers close beside the borders of what
    is left, with as many blocks a request as a step of that many takes."""
    rng = np.random.default_rng(requests)
    vocab = 33001
    for sibling in (True, False):
        rows = []
        for _ in range(requests):
            a = (rng.standard_normal(vocab) * 2).astype(np.float32)
            b = (a.astype(np.float64) + rng.standard_normal(vocab) * error).astype(np.float32)
            x = int(a.argmin())
            b[x] = a[x] + np.float32(0.1 + 2 * error)
            rows.append((a, b, x))
        assert_verify(border_case(rows, 24, sibling))


# ---------------------------------------------------------------------------------------------- rows and pages moved

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 2, 4, 16, 64), (2, 2, 1, 4, 5), (5, 3, 16, 24), (1, 16, 96), (2, 2, 2, 1, 8), (1, 2, 8, 8, 128), (1, 7, 3)])
def test_keep_rows(dtype, shape):
    slots, page = shape[0], shape[-2]
    rng = np.random.default_rng(sum(shape))
    spec = [(0, 9, [0, 2, 3, 8]), (5, 1, [0]), (16, 20, list(range(1, 20, 2))), (31, 6, [0, 1, 2]), (2, 0, []), (47, 40, sorted(rng.permutation(40)[:25].tolist())),
            (11, 5, []), (9, 12, [11])]
    need = [-(-(b + n) // page) for b, n, _ in spec]
    order = rng.permutation(sum(need) + 2).tolist()
    table = torch.full((len(spec), max(need)), -1, dtype=torch.int32)
    seg, path, count, at, taken = torch.zeros(len(spec), 4, dtype=torch.int32), [], [], 0, 0
    for s, (b, n, kept) in enumerate(spec):
        table[s, :need[s]] = torch.tensor(order[taken:taken + need[s]], dtype=torch.int32)
        seg[s] = torch.tensor([at, n, b, -1])
        path += kept + [-1] * (n - len(kept))
        count.append(len(kept))
        at += n
        taken += need[s]
    path, count = torch.tensor(path + [-1], dtype=torch.int32), torch.tensor(count, dtype=torch.int32)
    pool = torch.randn(slots, len(order), *shape[1:]).to(dtype)
    want, got = pool.clone(), pool.cuda()
    plain.keep(want, table, seg, path, count)
    ops = ops_of("float32")
    ops.keep_rows(got, table.cuda(), seg.cuda(), path.cuda(), count.cuda())
    ops.check_errors()
    assert torch.equal(got.cpu(), want)


def test_keep_rows_leaves_a_request_whose_path_is_none():
    from fusezap_core_b200.kernels.table import KernelError
    ops = ops_of("float32")
    table = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device="cuda")
    seg = torch.tensor([[0, 6, 1, -1], [6, 5, 3, -1]], dtype=torch.int32, device="cuda")
    pool = torch.randn(2, 4, 2, 3, 4, 8, device="cuda")
    good = [0, 2, 4, -1, -1, -1]
    for path, count, why in (([0, 3, 2, -1, -1, -1], 3, "outside the step"), ([0, 2, 2, -1, -1, -1], 3, "outside the step"), ([0, 6, -1, -1, -1, -1], 2, "outside the step"),
                             ([-1] * 6, 1, "outside the step"), (good, 7, "outside the step"), (good, 3, "no page")):
        other = [0, 4, -1, -1, -1] if why == "no page" else [0, -1, -1, -1, -1]      # (its place 3 + 4 has no page)
        was, now = pool.clone(), pool.clone()
        ops.keep_rows(now, table, seg, torch.tensor(path + other, dtype=torch.int32, device="cuda"),
                      torch.tensor([count, 2 if why == "no page" else 1], dtype=torch.int32, device="cuda"))
        with pytest.raises(KernelError, match=why):
            ops.check_errors()
        bad = [0, 1] if why != "no page" else [2]
        assert torch.equal(now[:, bad], was[:, bad])


@pytest.mark.parametrize("field,value", BAD_SEGMENTS)
def test_moved_rows_and_verdicts_of_requests_outside_the_step(field, value):
    from fusezap_core_b200.kernels.table import KernelError
    ops = ops_of("float32")
    table = torch.tensor([[0, 1, 4], [2, 3, 5]], dtype=torch.int32, device="cuda")
    seg = torch.tensor([[0, 6, 1, -1], [6, 5, 3, -1]], dtype=torch.int32)
    seg[1, field] = value
    pool = torch.randn(2, 6, 2, 3, 4, 8, device="cuda")
    path = torch.tensor([0, 2, 4, -1, -1, -1, 0, 4, -1, -1, -1], dtype=torch.int32, device="cuda")
    was, now = pool.clone(), pool.clone()
    ops.keep_rows(now, table, seg.cuda(), path, torch.tensor([3, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(KernelError, match="outside the step"):
        ops.check_errors()
    assert torch.equal(now[:, [2, 3, 5]], was[:, [2, 3, 5]]) and not torch.equal(now[:, [0, 1, 4]], was[:, [0, 1, 4]])
    if field == 2:
        return      # (verdicts do not read it)
    c = verify_case(3000, [chain(6), chain(5)], True, greedy=lambda s: False)
    c["seg"][1, field] = value
    with pytest.raises(KernelError, match="outside the step"):
        run_verify(c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 2, 4, 16, 64), (2, 2, 1, 4, 5), (1, 1, 3), (2, 16, 24), (32, 2, 8, 16, 128), (1, 2, 8, 64, 128)])
def test_copy_pages(dtype, shape):
    gen = torch.Generator().manual_seed(1)
    order = torch.randperm(23, generator=gen)
    src, dst = order[:5][torch.randint(0, 5, (11,), generator=gen)].int(), order[5:16].int()
    pool = torch.randn(shape[0], 23, *shape[1:], generator=gen).to(dtype)
    want, got = pool.clone(), pool.cuda()
    plain.copy(want, src, dst)
    ops = ops_of("float32")
    ops.copy_pages(got, src.cuda(), dst.cuda())
    ops.check_errors()
    assert torch.equal(got.cpu(), want)


def test_copy_pages_leaves_out_pages_outside_the_pool():
    from fusezap_core_b200.kernels.table import KernelError
    ops = ops_of("float32")
    pool = torch.randn(2, 5, 2, 3, 4, 8, device="cuda")
    want = pool.clone()
    want[:, 3] = want[:, 1]
    ops.copy_pages(pool, torch.tensor([1, 5, 0, -1], dtype=torch.int32, device="cuda"), torch.tensor([3, 2, 5, 4], dtype=torch.int32, device="cuda"))
    with pytest.raises(KernelError, match="no page"):
        ops.check_errors()
    assert torch.equal(pool, want)


# ---------------------------------------------------------------------------------------------- refusals

def test_refusals():
    from fusezap_core_b200.kernels.table import KernelError
    ops = ops_of("bfloat16")
    c = tree_case("bfloat16", 8, 2, 64, 16, [(20, bushy(5))])
    q, cache, meta = on_gpu(c)
    out = torch.empty_like(q)

    def refused(match, q=q, cache=cache, out=out, heads=8, kv=2, hd=64, scale=0.1, **other):
        m = SimpleNamespace(**{**vars(meta), **other})
        with pytest.raises(KernelError, match=match):
            ops.tree_attention(q, cache, m, out, heads, kv, hd, scale, 0)

    refused("dtype", q=q.float())
    refused("scale", scale=0.0)
    refused("scale", scale=NAN)
    refused("is on cpu", q=q.cpu())
    refused("shape", out=out[:-1])
    refused("shape", pos=meta.pos[:-1])
    refused("dtype", ancestors=meta.ancestors.long())
    refused("shape", seg=meta.seg[:, :3].contiguous())
    refused("contiguous", q=torch.empty_like(q).t().contiguous().t())
    refused("key pool", cache=SimpleNamespace(**{**vars(cache), "page_size": 8}))
    refused("head_dim", q=torch.empty(5, 8 * 24, dtype=torch.bfloat16, device="cuda"), out=torch.empty(5, 8 * 24, dtype=torch.bfloat16, device="cuda"), hd=24,
            cache=SimpleNamespace(**{**vars(cache), "keys": torch.empty(4, 2, 2, 16, 24, dtype=torch.bfloat16, device="cuda")[:, 0],
                                     "values": torch.empty(4, 2, 2, 16, 24, dtype=torch.bfloat16, device="cuda")[:, 1]}))
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    f = lambda *s: torch.zeros(s, device="cuda")
    good = dict(logits=f(3, 10), draft=f(3, 10), temperature=f(1), uniform=f(3).double(), tokens=i32(3), parents=i32(3), seg=i32(1, 4), path=i32(3), count=i32(1), next_ids=i32(1))
    for name, bad in (("logits", f(3, 10).bfloat16()), ("draft", f(3, 9)), ("temperature", f(2)), ("uniform", f(3)), ("tokens", i32(4)), ("parents", i32(3).long()),
                      ("seg", i32(1, 3)), ("path", i32(2)), ("count", i32(2)), ("next_ids", i32(1).cpu())):
        with pytest.raises(KernelError):
            ops.verify_tree(**{**good, name: bad})
    pool = torch.zeros(2, 4, 2, 1, 4, 8, device="cuda")
    for bad in (dict(pool=pool.transpose(0, 1)), dict(pool=pool.cpu()), dict(table=i32(2, 2)), dict(path=i32(3).long()), dict(count=i32(2))):
        with pytest.raises(KernelError):
            ops.keep_rows(**{**dict(pool=pool, table=i32(1, 2), seg=i32(1, 4), path=i32(3), count=i32(1)), **bad})
    for bad in (dict(src=i32(2)), dict(dst=i32(3).float()), dict(pool=pool[:, ::2])):
        with pytest.raises(KernelError):
            ops.copy_pages(**{**dict(pool=pool, src=i32(3), dst=i32(3)), **bad})
    ops.check_errors()


# ---------------------------------------------------------------------------------------------- the step function

def small_model(name, dtype, tmp_path, max_len=1024):
    from fusezap_core_b200 import load_model
    from util import make_model_dir
    d, cfg, opts = make_model_dir(name, tmp_path, dtype)
    return load_model(d, dtype, "cuda:0", max_len=max_len), cfg, opts


def runner_for(model, page, pages=700, nodes=64, rows=640):
    from fusezap_core_b200.cache import CacheManager
    from fusezap_core_b200.engine import StepRunner
    cache = CacheManager(model.cache_needs(), model.state_needs(), page, pages, 8, model.max_len, model.ops.dtype, "cuda:0")
    return StepRunner(model, cache, max_rows=rows, max_segments=8, max_tree_nodes=nodes), cache


@pytest.mark.parametrize("name,dtype,page", [("tiny_llama", "float32", 4), ("tiny_window", "float32", 8), ("tiny_hd64", "float32", 16),
                                              ("tiny_hd64", "bfloat16", 16), ("tiny_hd128", "bfloat16", 16), ("tiny_hd128", "bfloat16", 8), ("tiny_hd128", "bfloat16", 4)])
def test_drafted_steps_equal_steps_of_single_tokens(name, dtype, page, tmp_path):
    """Trees around the tokens that plain decoding gives, verified greedily, kept and continued. float32: the tokens are the same and so are
    the logits, up to the tolerance of one model in two cuttings; bfloat16: the logits are, the tokens are taken as they come."""
    from fusezap_core_b200.engine import Portion
    from util import assert_close, prompts
    model, cfg, opts = small_model(name, dtype, tmp_path, max_len=512 if name != "tiny_llama" else 128)
    run, cache = runner_for(model, page)
    plain_run, plain_cache = runner_for(model, page)
    P = prompts(cfg, (5, 41, 90), seed=3) if name == "tiny_llama" else prompts(cfg, (33, 200, 310), seed=3)
    for r, c in ((run, cache), (plain_run, plain_cache)):
        r.run([Portion(i, p[:-1], []) for i, p in enumerate(P)])
    rng = np.random.default_rng(0)
    have = [list(p) for p in P]
    V = cfg["vocab_size"]
    for step in range(6):
        # what plain decoding gives next, on a copy of the books: two tokens of each request, forgotten afterwards
        portions = []
        for i in range(len(P)):
            tokens, parents, under = [have[i][-1], int(rng.integers(V))], [-1, 0], 0
            for _ in range(int(rng.integers(0, 4))):
                tokens += [int(rng.integers(V)), int(rng.integers(V))]
                parents += [under, under]
                under = len(tokens) - 2
            portions.append(Portion(i, tokens, range(len(tokens)), parents=parents))
        # the right token among the root's children in every other step
        first = plain_run.run([Portion(i, [have[i][-1]], [0]) for i in range(len(P))]).argmax(1).tolist()
        if step % 2:
            for p, t in zip(portions, first):
                p.tokens[1] = t
        starts = run.prepare(portions)
        logits = run.forward()
        n, s = logits.shape[0], len(P)
        path, count, ids = run.verify(logits, torch.zeros(s, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda"))
        run.keep(path, count)
        model.ops.check_errors()
        got, kept = logits.clone(), count.tolist()
        run.commit_kept(portions, starts, kept)
        cache.check()
        at = 0
        for i, (p, k) in enumerate(zip(portions, kept)):
            nodes = path[at:at + k].tolist()
            assert dtype == "bfloat16" or not step % 2 or k > 1, "the right token was among the root's children"
            new = [p.tokens[j] for j in nodes[1:]] + [int(ids[i])]
            # the same tokens one by one (the first has run above)
            ref = []
            for j, t in enumerate(new[:-1]):
                ref.append(plain_run.run([Portion(i, [t], [0])])[0].clone())
            if ref:
                assert_close(got[[at + j for j in nodes[1:]]].cpu().numpy(), torch.stack(ref).cpu().numpy(), dtype, f"step {step}, request {i}")
            if dtype == "float32":
                assert int(ids[i]) == (int(ref[-1].argmax()) if ref else first[i])
            have[i] += new
            at += len(p.tokens)
            assert cache.computed[i] == plain_cache.computed[i] == len(have[i]) - 1
    # the caches hold the same: the next token's logits agree
    last = [run_.run([Portion(i, [h[-1]], [0]) for i, h in enumerate(have)]).clone() for run_ in (run, plain_run)]
    assert_close(last[0].cpu().numpy(), last[1].cpu().numpy(), dtype, "after the drafts")


@pytest.mark.parametrize("name,dtype", [("tiny_hd64", "float32"), ("tiny_hd128", "bfloat16")])
def test_a_recorded_step_of_trees_replayed_over_others(name, dtype, tmp_path):
    """One recorded tree step with its verdict and the move of the kept rows, replayed with other trees, contexts and requests."""
    from fusezap_core_b200.engine import Portion
    from util import prompts
    model, cfg, opts = small_model(name, dtype, tmp_path)
    run, cache = runner_for(model, 16)
    other, other_cache = runner_for(model, 16)
    P = prompts(cfg, (60, 130, 311), seed=5)
    for r in (run, other):
        r.run([Portion(i, p[:-1], []) for i, p in enumerate(P)])
    V = cfg["vocab_size"]
    rng = np.random.default_rng(7)
    temperature, uniform = torch.tensor([0.0, 0.8, 1.1], device="cuda"), torch.empty(24, dtype=torch.float64, device="cuda")
    graph = out = None
    for step in range(5):
        portions = []
        for i, n in enumerate((9, 5, 10)):
            parents = [-1] + [int(rng.integers(0, j)) for j in range(1, n)]
            portions.append(Portion(i, [int(t) for t in rng.integers(0, V, n)], range(n), parents=parents))
        uniform.copy_(torch.from_numpy(rng.random(24)))
        results = []
        for r, c in ((run, cache), (other, other_cache)):
            starts = r.prepare(portions)
            r.meta.max_context = 512

            def step_of(r=r):
                logits = r.forward()
                path, count, ids = r.verify(logits, temperature, uniform)
                r.keep(path, count)
                return logits, path, count, ids

            if r is run and step == 1:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = step_of()
            if r is run and graph is not None:
                graph.replay()
                got = out
            else:
                got = step_of()
            model.ops.check_errors()
            results.append([t.clone() for t in got])
            r.commit_kept(portions, starts, got[2].tolist())
            c.check()
        assert all(torch.equal(a, b) for a, b in zip(*results)), f"step {step}"


def test_forked_requests_on_the_device(tmp_path):
    from fusezap_core_b200.engine import Portion
    from util import assert_close, prompts
    model, cfg, opts = small_model("tiny_hd128", "bfloat16", tmp_path)
    run, cache = runner_for(model, 16)
    p = prompts(cfg, (75,), seed=6)[0]
    run.run([Portion("a", p, [])])
    run.fork("a", "b")
    cache.check()
    more = {r: prompts(cfg, (9,), seed=s)[0] for r, s in (("a", 7), ("b", 8))}
    for j in range(9):
        lg = run.run([Portion(r, [more[r][j]], [0]) for r in ("a", "b")]).clone()
    for k, r in enumerate(("a", "b")):
        cache.reset()
        ref = run.run([Portion("x", p, [])])
        for t in more[r]:
            ref = run.run([Portion("x", [t], [0])]).clone()
        assert_close(lg[k:k + 1].cpu().numpy(), ref.cpu().numpy(), "bfloat16", r)
    model.ops.check_errors()


@pytest.mark.parametrize("heads,kv,hd,page", [(4, 4, 64, 16), (32, 8, 128, 16), (10, 2, 128, 8)])
def test_the_general_kernel_takes_what_the_tensor_core_kernel_takes(heads, kv, hd, page):
    ops = ops_of("bfloat16")
    c = tree_case("bfloat16", heads, kv, hd, page, [(37, bushy(9)), (0, bushy(5, 1)), (700, chain(3)), (300, [-1])], pad=3)
    assert_tree(c, run_tree(c))
    ops.tree_tensor_cores = False
    try:
        assert_tree(c, run_tree(c))
    finally:
        ops.tree_tensor_cores = True


def test_bad_tables_are_reported():
    """A page that is missing, one outside the pool, a row outside its request: an error, and nothing outside is read or written."""
    from fusezap_core_b200.kernels.table import KernelError
    for dtype in ("float32", "bfloat16"):
        for change, why in ((lambda m: m.tables.__setitem__((0, 2), -1), "no page"), (lambda m: m.tables.__setitem__((0, 2), 10 ** 6), "no page"),
                            (lambda m: m.seq_row.__setitem__(0, 7), "outside the step"), (lambda m: m.seg.__setitem__((0, 1), 3), "outside the step")):
            c = tree_case(dtype, 8, 2, 64, 16, [(60, bushy(9)), (20, bushy(4))])
            change(c.meta)
            with pytest.raises(KernelError, match=why):
                run_tree(c)
