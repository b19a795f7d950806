"""Drafted trees through the step function on the CPU (plain kernel table): logits of every way down a tree equal those of the same tokens
run one after the other; after a verdict the cache is as if only the kept tokens had been run; requests continued several ways;
what is refused."""
import numpy as np
import pytest
import torch

import plain_drafts
import plain_model
from fusezap_core_b200 import load_model
from fusezap_core_b200.cache import CacheManager, KVNeed, LatentNeed, OutOfPages, PageAllocator
from fusezap_core_b200.engine import Portion, StepRunner
from plain_drafts import PlainDraftOps
from util import make_model_dir, prompts, read_weights


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    out = {}
    for name in ("tiny_llama", "tiny_qwen2", "tiny_window"):
        d, cfg, opts = make_model_dir(name, tmp_path_factory.mktemp(name))
        out[name] = (load_model(d, "float32", "cpu", max_len=160, ops=PlainDraftOps()), cfg, opts, read_weights(d))
    return out


def runner_for(model, opts, pages=64, nodes=40):
    cache = CacheManager(model.cache_needs(), model.state_needs(), opts["page_size"], pages, 8, 160, torch.float32, "cpu")
    return StepRunner(model, cache, max_rows=160, max_tree_nodes=nodes), cache


def way(parents, j):
    out = []
    while j >= 0:
        out.append(j)
        j = parents[j]
    return out[::-1]


TREES = [[-1, 0, 0, 1, 1, 2, 3], [-1], [-1, 0, 1, 2], [-1, 0, 0, 0, 3]]


@pytest.mark.parametrize("name", ["tiny_llama", "tiny_qwen2", "tiny_window"])
def test_every_way_down_a_tree_has_the_logits_of_its_tokens(models, name):
    model, cfg, opts, w = models[name]
    run, cache = runner_for(model, opts)
    P = prompts(cfg, (13, 1, 30, 17), seed=4)
    rng = np.random.default_rng(1)
    run.run([Portion(i, p[:-1], []) for i, p in enumerate(P) if len(p) > 1])
    nodes = [[p[-1]] + rng.integers(0, cfg["vocab_size"], len(t) - 1).tolist() for p, t in zip(P, TREES)]
    portions = [Portion(i, n, range(len(n)), parents=t) for i, (n, t) in enumerate(zip(nodes, TREES))]
    portions[1] = Portion(1, nodes[1], [0])      # (a plain token beside the trees)
    run.prepare(portions)
    logits, at = run.forward().numpy().copy(), 0
    for i, t in enumerate(TREES):
        for j in range(len(t)):
            ids = P[i][:-1] + [nodes[i][k] for k in way(t, j)]
            np.testing.assert_allclose(logits[at + j], plain_model.forward(cfg, w, ids).numpy()[-1], rtol=1e-4, atol=2e-5)
        at += len(t)
    assert [cache.computed[i] for i in range(4)] == [12, 0, 29, 16], "nothing is computed before it is kept"


def greedy(cfg, w, prompt, n):
    ids = list(prompt)
    for _ in range(n):
        ids.append(int(plain_model.forward(cfg, w, ids).numpy()[-1].argmax()))
    return ids[len(prompt):]


@pytest.mark.parametrize("name", ["tiny_llama", "tiny_window"])
def test_greedy_tokens_with_drafts_are_the_tokens_without(models, name):
    """Trees that hold the right tokens, some of them or none: the tokens are those of plain greedy decoding, and the cache holds them."""
    model, cfg, opts, w = models[name]
    run, cache = runner_for(model, opts)
    P = prompts(cfg, (9, 21), seed=5)
    want = [greedy(cfg, w, p, 14) for p in P]
    have = [[] for _ in P]
    rng = np.random.default_rng(2)
    run.run([Portion(i, p[:-1], []) for i, p in enumerate(P)])
    steps = kept_in_all = 0
    while min(len(h) for h in have) < 10:
        portions = []
        for i, p in enumerate(P):
            last, known = (p + have[i])[-1], want[i][len(have[i]):]
            good = known[:int(rng.integers(0, 4))]
            # node 0, a wrong child, then the right tokens one below the other (each beside a wrong sibling), one of them wrong at the end
            tokens, parents, under = [last, (known[0] + 1) % cfg["vocab_size"]], [-1, 0], 0
            for t in good:
                tokens += [t, (t + 3) % cfg["vocab_size"]]
                parents += [under, under]
                under = len(tokens) - 2
            portions.append(Portion(i, tokens, range(len(tokens)), parents=parents))
        starts = run.prepare(portions)
        logits = run.forward()
        path, count, ids = run.verify(logits, torch.zeros(2), torch.zeros(logits.shape[0], dtype=torch.float64))
        run.keep(path, count)
        run.commit_kept(portions, starts, count.tolist())
        cache.check()
        for i, (p, seg) in enumerate(zip(portions, run.meta.segments)):
            kept = path[seg.row0: seg.row0 + int(count[i])].tolist()
            have[i] += [p.tokens[k] for k in kept[1:]] + [int(ids[i])]
            assert cache.computed[i] == len(P[i]) + len(have[i]) - 1
            assert len([x for x in cache.table(0, i) if x >= 0]) <= -(-cache.computed[i] // cache.page_size)
        steps += 1
        kept_in_all += int(count.sum())
    assert kept_in_all > 2 * steps, "drafted tokens stood"
    for i in range(2):
        assert have[i][:10] == want[i][:10]
    # the cache is what the tokens one by one would have left: the next logits say so
    for i, p in enumerate(P):
        ids = p + have[i]
        lg = run.run([Portion(i, ids[cache.computed[i]:], [len(ids) - cache.computed[i] - 1])]).numpy()[0]
        np.testing.assert_allclose(lg, plain_model.forward(cfg, w, ids).numpy()[-1], rtol=1e-4, atol=2e-5)


def test_forked_requests_go_their_own_ways(models):
    model, cfg, opts, w = models["tiny_qwen2"]
    run, cache = runner_for(model, opts)
    p = prompts(cfg, (21,), seed=6)[0]
    run.run([Portion("a", p, [])])
    before = cache.num_free_pages
    run.fork("a", "b")
    run.fork("a", "c")
    page = cache.page_size
    assert before - cache.num_free_pages == (2 if len(p) % page else 0), "only the page that is not full is copied"
    assert cache.table(0, "a")[:len(p) // page] == cache.table(0, "b")[:len(p) // page]
    cache.check()
    more = {r: prompts(cfg, (7,), seed=s)[0] for r, s in (("a", 7), ("b", 8), ("c", 9))}
    for j in range(7):
        lg = run.run([Portion(r, [more[r][j]], [0]) for r in ("a", "b", "c")]).numpy().copy()
    for k, r in enumerate(("a", "b", "c")):
        np.testing.assert_allclose(lg[k], plain_model.forward(cfg, w, p + more[r]).numpy()[-1], rtol=1e-4, atol=2e-5)
    cache.free("a")
    cache.check()
    lg = run.run([Portion("b", [5], [0])]).numpy()
    np.testing.assert_allclose(lg[0], plain_model.forward(cfg, w, p + more["b"] + [5]).numpy()[-1], rtol=1e-4, atol=2e-5)
    cache.free("b")
    cache.free("c")
    cache.check()
    assert cache.num_free_pages == cache.num_pages


def test_refusals(models):
    model, cfg, opts, _ = models["tiny_llama"]
    run, cache = runner_for(model, opts, nodes=6)
    ok = Portion("a", [1, 2, 3], range(3), parents=[-1, 0, 1])
    for bad, why in ((Portion("a", [1, 2], [], parents=[-1]), "no tree"), (Portion("a", [1, 2], [], parents=[0, 0]), "no tree"),
                     (Portion("a", [1, 2], [], parents=[-1, -1]), "no tree"), (Portion("a", [1, 2, 3], [], parents=[-1, 2, 0]), "no tree"),
                     (Portion("a", list(range(7)), [], parents=[-1] + list(range(6))), "max_tree_nodes"),
                     (Portion("a", [1], [], parents=[-1], src=0), "given")):
        with pytest.raises(ValueError, match=why):
            run.prepare([bad])
    with pytest.raises(ValueError, match="verify, keep"):
        run.run([ok])
    with pytest.raises(ValueError, match="max_tree_nodes"):
        StepRunner(model, cache, max_rows=20).prepare([ok])
    with pytest.raises(ValueError, match="1 to"):
        StepRunner(model, cache, max_rows=20, max_tree_nodes=1025)
    starts = run.prepare([ok, Portion("b", [4], [])])
    logits = run.forward()
    u, t = torch.zeros(4, dtype=torch.float64), torch.zeros(2)
    with pytest.raises(ValueError, match="every row"):
        run.verify(logits, t, u)
    with pytest.raises(ValueError, match="commit_kept"):
        run.commit([ok], starts)
    with pytest.raises(ValueError, match="kept"):
        run.commit_kept([ok], starts, [0])
    run.run([Portion("c", [1], [0])])
    with pytest.raises(ValueError, match="no drafted trees"):
        run.verify(logits, t, u)
    with pytest.raises(ValueError, match="no drafted trees"):
        run.keep(None, None)


def test_kept_counts_that_do_not_fit_the_step_change_no_books(models):
    model, _, opts, _ = models["tiny_llama"]
    run, cache = runner_for(model, opts, nodes=6)
    portions = [Portion("a", [1, 2, 3], range(3), parents=[-1, 0, 0]), Portion("b", [4, 5], range(2), parents=[-1, 0])]
    starts = run.prepare(portions)
    run.forward()
    for counts in ([2], [2, 1, 1], [], [2, 0], [2, 3]):
        with pytest.raises(ValueError, match="kept"):
            run.commit_kept(portions, starts, counts)
        assert cache.computed == {"a": 0, "b": 0}
    with pytest.raises(ValueError, match="kept"):
        run.commit_kept(portions, starts[:1], [2, 1])
    run.commit_kept(portions, starts, [2, 1])
    assert cache.computed == {"a": 2, "b": 1}
    cache.check()


def test_windows_and_other_mixers_refuse(models, tmp_path):
    model, cfg, opts, _ = models["tiny_window"]
    run, cache = runner_for(model, opts)
    with pytest.raises(ValueError, match="window of 12"):
        run.prepare([Portion("a", list(range(13)), [], parents=list(range(-1, 12)))])
    run.prepare([Portion("a", list(range(12)), [], parents=list(range(-1, 11)))])
    from fusezap_core_b200.engine.model import random_model
    from fusezap_core_b200.cli import load_preset
    for preset in ("tiny-gimupel", "tiny-muretar", "tiny-nepudra"):
        other = random_model(load_preset(preset), "float32", "cpu", ops=_Anything())
        cache = CacheManager(other.cache_needs(), other.state_needs(), 4, 8, 2, 32, torch.float32, "cpu")
        with pytest.raises(ValueError, match="not taken"):
            StepRunner(other, cache, max_rows=8, max_tree_nodes=4)


def test_parts_with_methods_of_their_own_refuse(models, monkeypatch):
    """What a mixer or a position encoding says of trees holds for the methods it has, not for those that a derived class brings."""
    from fusezap_core_b200.parts.attention import GQAttention
    from fusezap_core_b200.parts.rope import RotaryEncoding
    model, _, opts, _ = models["tiny_llama"]

    class Derived(GQAttention):
        def cache_need(self):
            return super().cache_need()

    class Own(GQAttention):
        def forward(self, ctx, h, cache):
            raise NotImplementedError

    class Below(Own):
        pass

    class OwnForTrees(Own):
        takes_trees = True

    class Rope(RotaryEncoding):
        pass

    class Store(RotaryEncoding):
        def rotate_and_store(self, ctx, qkv, q_out, cache, num_heads, num_kv_heads, head_dim):
            raise NotImplementedError

    class Product(RotaryEncoding):
        def project_rotate_store(self, *a):
            return False

    class StoreForTrees(Store):
        takes_trees = True

    mixer = model.layers[-1].mixer
    for part, kinds in ((mixer, ((Derived, True), (Own, False), (Below, False), (OwnForTrees, True))),
                        (model.positions[mixer.position_name()], ((Rope, True), (Store, False), (Product, False), (StoreForTrees, True)))):
        for kind, takes in kinds:
            with monkeypatch.context() as m:
                m.setattr(part, "__class__", kind)
                if takes:
                    runner_for(model, opts)
                else:
                    with pytest.raises(ValueError, match=f"not taken by {kind.__name__}"):
                        runner_for(model, opts)


class _Anything:
    """A kernel table that takes every size and runs nothing."""
    dtype = torch.float32

    def __getattr__(self, name):
        if name.startswith("__"):
            raise AttributeError(name)
        if name == "recurrent_state_shape":
            return lambda h, k, v: (h, k, v)
        return lambda *a, **k: None


# ---------------------------------------------------------------------------------------------- pages

def manager(needs=None, pages=16, page_size=4, states=None, requests=4):
    return CacheManager(needs or {0: KVNeed(2, 16, 0)}, states or {}, page_size, pages, requests, 64, torch.float32, "cpu", allocate=bool(states))


def test_shared_pages_are_free_when_the_last_holder_gives_them_back():
    a = PageAllocator(3)
    p = a.allocate(2)
    a.share([p[0]])
    a.free(p)
    assert a.num_free == 2 and a.holders(p[0]) == 1
    a.check()
    a.free([p[0]])
    with pytest.raises(AssertionError, match="not held"):
        a.free([p[0]])
    with pytest.raises(AssertionError, match="not held"):
        a.share([p[0]])
    a.check()


def test_trim_gives_back_what_lies_behind_the_computed_places():
    m = manager()
    m.ensure("a", 6)
    m.commit("a", 6)
    m.ensure("a", 6 + 9)
    assert len(m.table(0, "a")) == 4
    m.commit("a", 8)
    m.trim("a")
    assert len(m.table(0, "a")) == 2 and m.num_free_pages == 14
    m.trim("a")
    m.check()
    m.ensure("a", 9)
    assert len(m.table(0, "a")) == 3
    with pytest.raises(KeyError):
        m.trim("b")


@pytest.mark.parametrize("computed", [0, 1, 4, 7, 8, 30])
def test_fork_over_windows_latents_and_random_orders(computed):
    import random
    m = manager({0: KVNeed(2, 16, 0), 1: KVNeed(2, 16, 9), 2: LatentNeed(24)}, pages=40)
    m.ensure("a", max(1, computed))
    m.commit("a", computed)
    copies, slots = m.fork("a", "b")
    assert slots is None and [len(c) for c in copies] == [1 if computed % 4 else 0] * 3
    for g, c in enumerate(copies):
        if c:
            assert c[0] == (m.table(g, "a")[computed // 4], m.table(g, "b")[computed // 4]) and c[0][0] != c[0][1]
    m.check()
    rng = random.Random(computed)
    live, n = {"a": computed, "b": computed}, 0
    for _ in range(200):
        r = rng.choice(sorted(live)) if live else None
        what = rng.random()
        if r is None or (what < 0.2 and len(live) < 6 and m.can_fork(r)):
            n += 1
            new = f"r{n}"
            if r is None:
                m.ensure(new, 1)
                m.commit(new, 1)
                live[new] = 1
            else:
                m.fork(r, new)
                live[new] = live[r]
        elif what < 0.35:
            m.free(r)
            del live[r]
        elif m.can_ensure(r, min(64, live[r] + 5)):
            m.ensure(r, min(64, live[r] + 5))
            live[r] = min(64, live[r] + rng.randint(1, 5))
            m.commit(r, live[r])
            m.trim(r)
        m.check()
    for r in list(live):
        m.free(r)
    m.check()
    assert all(g.allocator.num_free == 40 for g in m.groups)


def test_a_request_is_not_set_back_into_pages_that_it_shares():
    """What it would write anew there is what the other has computed."""
    m = manager({0: KVNeed(2, 16, 0), 1: LatentNeed(24)})
    m.ensure("a", 14)
    m.commit("a", 14)
    m.commit("a", 13)
    m.commit("a", 14)
    m.fork("a", "b")
    for req in ("a", "b"):
        m.commit(req, 13)      # (the page that is not full is each one's own)
        m.commit(req, 12)
        for n in (11, 8, 1, 0):
            with pytest.raises(ValueError, match="shares"):
                m.commit(req, n)
            assert m.computed[req] == 12
    m.check()
    m.free("b")
    m.commit("a", 5)
    m.ensure("a", 9)
    m.commit("a", 9)
    m.check()


def test_fork_refusals_and_state():
    m = manager(pages=3)
    m.ensure("a", 10)
    m.commit("a", 10)
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    assert not m.holds("b")
    m.check()
    with pytest.raises(KeyError):
        m.fork("x", "y")
    m = manager(states={(0, "s"): (3,)}, requests=2)
    m.ensure("a", 3)
    m.commit("a", 3)
    copies, slots = m.fork("a", "b")
    assert slots == (m.state_slot("a"), m.state_slot("b")) and slots[0] != slots[1]
    with pytest.raises(OutOfPages):
        m.fork("a", "c")
    with pytest.raises(ValueError, match="already"):
        m.fork("a", "b")
    m.check()
