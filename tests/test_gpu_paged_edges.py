"""GPU tests of the paged cache where something has gone wrong or is over: packed vectors that are no numbers behind a window's edge, recorded steps after their end, failures halfway, pools that are nearly full or have been
gathered.
Tolerances are those of test_gpu_paged."""
import random
from importlib import import_module

import pytest
import torch

from test_gpu_many import HALF
from test_gpu_paged import BF, F16, F32, check, contents, feed, make, rand, states
from test_gpu_parity import DEV

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a HIP device; there is no CPU fallback to test")


@pytest.mark.parametrize("side", [1, 3], ids=["keys", "values"])
@pytest.mark.parametrize("D,G,dtype,kb,vb,new,P", [
    (128, 4, BF, 4, 2, 1, 64), (128, 4, BF, 4, 2, 4, 64), (128, 8, F16, 6, 4, 1, 64), (64, 4, F16, 6, 4, 1, 128), (64, 2, BF, 8, 8, 3, 64), (96, 2, BF, 4, 2, 1, 64), (256, 4, BF, 4, 2, 1, 64), (256, 2, F16, 8, 4, 2, 64),
    (128, 4, BF, 4, 2, 40, 64), (128, 4, F16, 6, 4, 40, 64), (64, 4, BF, 8, 8, 33, 64), (80, 2, BF, 4, 4, 20, 64), (96, 4, F16, 4, 4, 30, 64), (256, 2, BF, 4, 2, 20, 64), (128, 1, BF, 4, 2, 40, 32),
    (128, 2, F32, 4, 2, 1, 64), (128, 2, F32, 4, 4, 40, 64), (256, 1, F32, 2, 8, 9, 32)])
def test_packed_vectors_that_are_no_numbers_stay_with_those_who_see_them(pkg, D, G, dtype, kb, vb, new, P, side):
    W, n = 150, 700
    cache = make(pkg, D, 2, dtype, kb, vb, 16, P=P)
    seqs = cache.add(2)
    feed(cache, seqs, (n, 390), seed=1)
    step = feed(cache, seqs, (new, new), seed=2, commit=False)
    q = rand((2 * new, 2 * G, D), 3, dtype)
    norms = cache.packed_pages(0)[side]
    for kw in ({"sliding_window": W}, {"sliding_window": W, "softcap": 20.0, "slopes": torch.linspace(0.01, 0.1, 2 * G, device=DEV)}):
        want = step.attend(q, 0, **kw)
        check(want, q, step, **kw)
        # a norm of its first kv head that the first `seen` of the new tokens see: none, the token just outside the window or further out; some
        for seen in sorted({-45, -20, 0, new // 2}):
            t = n - W + seen
            at = cache.tables(seqs[0])[0][t // P], 0, t % P
            for value in (float("inf"), float("nan")):
                kept = norms[at].clone()
                norms[at] = value
                got = step.attend(q, 0, **kw)
                norms[at] = kept
                if seen > 0:
                    if side == 3 or value != value:          # (an infinite key may be one that nobody likes)
                        assert not bool(torch.isfinite(got[:seen, :G]).any())
                    got[:seen, :G] = want[:seen, :G]
                check(got, q, step, **kw)


def recorded(pkg):
    """A cache with an open step that a graph has recorded: (cache, its sequences, step, graph, result)."""
    cache = make(pkg, H=2, window=20, pages=40, plain=40)
    seqs = cache.add(2)
    feed(cache, seqs, (300, 63), seed=1)
    step = cache.step(seqs, (9, 1))
    k, v, q = states(10, 2, 128, 1, BF), states(10, 2, 128, 2, BF), rand((10, 8, 128), 3, BF)
    step.append(k, v, 0)
    step.attend(q, 0)
    step.attend(q[:, :2], 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.append(k, v, 0)
        outs = [step.attend(q, 0), step.attend(q[:, :2], 0)]
    graph.replay()
    torch.cuda.synchronize()
    check(outs[0], q, step)
    k.fill_(7.0), v.fill_(7.0)
    return cache, seqs, step, graph, outs


@pytest.mark.parametrize("change", ["step", "free", "fork", "reorder", "place", "cancel", "resize"])
def test_replays_of_a_step_that_is_over_do_nothing(pkg, change):
    cache, seqs, step, graph, outs = recorded(pkg)
    if change == "cancel":
        step.cancel()
    else:
        step.commit()
    others = cache.add(2)
    if change == "free":
        cache.free(seqs)
    elif change == "fork":
        others += cache.fork(seqs)
    elif change == "reorder":
        cache.reorder(seqs, [0, 0])
    elif change == "place":
        cache.place(others, [0, 64], [70, 1])
    elif change == "resize":
        cache.resize(pages=41, plain_pages=42)
    if change != "place":
        feed(cache, others, [100] * len(others), seed=5)
    for out in outs:
        out.fill_(5.0)
    torch.cuda.synchronize()
    before = cache._plain.view(torch.int16).clone(), cache._pool.clone()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache._plain.view(torch.int16), before[0]) and torch.equal(cache._pool, before[1])
        assert all(bool((out == 5.0).all()) for out in outs)
    step = feed(cache, others, [3] * len(others), seed=6, commit=False)
    q = rand((3 * len(others), 8, 128), 4, BF)
    if change != "place":
        check(step.attend(q, 0), q, step)


def tables(cache):
    """All that says which pages are whose."""
    return (cache.free_pages(), sorted(cache._packed_pages.free), sorted(cache._plain_pages.free), list(cache._packed_pages.held), list(cache._plain_pages.held),
            {s: (cache.lengths([s]), cache.tables(s)) for s in cache._seqs}, dict(cache._packed_of))


@pytest.mark.parametrize("what", ["step", "fork", "reorder", "reorder in a full pool"])
def test_a_failure_halfway_leaves_the_tables_as_they_were(pkg, monkeypatch, what):
    module = import_module("turboquant-pytorch_amd.paged_cache")
    cache = make(pkg, H=2, window=64, plain=40)
    a, b, c = cache.add(3)
    feed(cache, [a, b, c], (200, 130, 70), seed=1)
    shared = cache.fork([a, b, b])
    feed(cache, [a], (64,), seed=2)          # (packs a page that the fork still holds uncompressed)
    assert cache._packed_of
    seqs = [a, b, c] + shared
    if "full" in what:
        (d,) = cache.add(1)
        cache.place([d], [0], [64 * cache.free_pages()[1]])
    before = tables(cache)

    def fail(*args, **kw):
        raise MemoryError("no room for this")
    with monkeypatch.context() as m:
        m.setattr(module.PagedStep, "_upload", fail)
        m.setattr(module._native, "copy_pages", fail)
        with pytest.raises(MemoryError):
            if what == "step":
                cache.step(seqs, 70)
            elif what == "fork":
                cache.fork([a, b, b])
            else:
                cache.reorder(seqs, [2, 2, 2, 5, 5, 4] if "full" in what else [0, 0, 1, 2, 2, 2])
    assert tables(cache) == before and cache._open is None
    if "full" in what:
        cache.free([d])
    cache.reorder(seqs, [0, 0, 1, 2, 2, 2])
    step = feed(cache, seqs, 3, seed=3, commit=False)
    q = rand((18, 8, 128), 3, BF)
    check(step.attend(q, 0), q, step)
    step.commit()
    cache.free(seqs)
    assert cache.free_pages() == (64, 40) and not cache._packed_of


def test_pages_that_only_ending_sequences_share_have_room_for_others(pkg):
    cache = make(pkg, H=1, window=128, pages=4, plain=3)
    (a,) = cache.add(1)
    feed(cache, [a], 64, seed=1)
    (b,) = cache.fork([a])                   # (a whole page, shared)
    (c,) = cache.add(1)
    feed(cache, [c], 10, seed=2)
    assert cache.free_pages()[1] == 1
    cache.reorder([a, b, c], [2, 2, 2])      # two copies of a page: into the free one and the one that a and b end with
    assert cache.free_pages()[1] == 0 and cache.lengths([a, b, c]) == [10, 10, 10] and len({cache.tables(s)[1][0] for s in (a, b, c)}) == 3
    step = feed(cache, [a, b, c], 1, seed=3, commit=False)
    q = rand((3, 2, 128), 3, BF)
    check(step.attend(q, 0), q, step)
    # one of them goes on: its page stays, and there is room for one copy less than it takes
    cache = make(pkg, H=1, window=128, pages=4, plain=3)
    (a,) = cache.add(1)
    feed(cache, [a], 64, seed=1)
    b, d = cache.fork([a, a])
    (c,) = cache.add(1)
    feed(cache, [c], 10, seed=2)
    before = tables(cache)
    with pytest.raises(pkg._native.TqError, match="uncompressed pages"):
        cache.reorder([a, b, c, d], [2, 2, 2, 0])
    assert tables(cache) == before

@pytest.mark.parametrize("seed", range(6))
def test_gathers_between_all_other_calls(pkg, seed):
    rng = random.Random(seed)
    cache, kept, seqs, at = make(pkg, H=1, window=rng.choice((0, 50, 128)), layers=2, pages=30, plain=60), {}, [], 0
    for turn in range(60):
        what = rng.choice(("add", "step", "step", "step", "fork", "reorder", "free", "resize", "resize"))
        if what == "add" and len(seqs) < 6:
            seqs += cache.add(1)
            for layer in range(2):
                kept[seqs[-1], layer] = []
        elif what == "step" and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            counts = [rng.choice((0, 1, 1, 2, 60, 130)) for _ in some]
            if sum(-(-c // 64) + 1 for c in counts) > cache.free_pages()[1]:
                cache.resize(plain_pages=400, pages=100)
            step = feed(cache, some, counts, seed=100 + turn, kept=kept, commit=False)
            if sum(counts):
                q = rand((sum(counts), 2, 128), turn, BF)
                check(step.attend(q, turn % 2), q, step, turn % 2)
        elif what == "fork" and 0 < len(seqs) < 5:
            if cache.free_pages()[1] < 1:
                cache.resize(plain_pages=400, pages=100)
            s = rng.choice(seqs)
            seqs += cache.fork([s])
            for layer in range(2):
                kept[seqs[-1], layer] = list(kept[s, layer])
        elif what == "reorder" and seqs:
            if cache.free_pages()[1] < len(seqs):
                cache.resize(plain_pages=400, pages=100)
            parents = [rng.randrange(len(seqs)) for _ in seqs]
            cache.reorder(seqs, parents)
            kept = {(s, layer): list(kept[seqs[p], layer]) for s, p in zip(seqs, parents) for layer in range(2)}
        elif what == "free" and len(seqs) > 1:
            s = seqs.pop(rng.randrange(len(seqs)))
            cache.free([s])
            kept = {k: v for k, v in kept.items() if k[0] != s}
        elif what == "resize":
            cache.resize(*((None, None) if rng.random() < 0.5 else (100, 200)))
        for s in seqs if turn % 5 == 4 else ():
            pages, plain = cache.tables(s)
            assert max(pages + [0]) < cache.packed_pages(0)[0].shape[0] and max(plain + [0]) < cache.plain_pages().shape[0]
            for layer in range(2):
                if not kept[s, layer]:
                    continue
                k, v = (torch.cat([t[i] for t in kept[s, layer]]).transpose(0, 1) for i in (0, 1))
                n = 64 * len(pages)
                assert cache.lengths([s]) == [k.shape[1]]
                for side, comp in enumerate((cache.codec(layer).key_compressor, cache.codec(layer).val_compressor)):
                    if n:
                        want, views = comp.compress((k, v)[side][:, :n].unsqueeze(0)), cache.packed_pages(layer)
                        assert torch.equal(views[2 * side][torch.tensor(pages, device=DEV)].transpose(0, 1).flatten(1, 2), want["idx_bytes"][0])
                    held = cache.plain_pages()[plain, layer, side].transpose(0, 1).flatten(1, 2)[:, :k.shape[1] - n]
                    assert torch.equal(held, (k, v)[side][:, n:])
    cache.free(seqs)
    cache.resize()
    assert cache.free_pages() == (1, 1) and not cache._packed_of


def test_a_layer_that_was_not_appended_to_is_not_attended_to(pkg):
    cache = make(pkg, H=2, layers=3)
    seqs = cache.add(2)
    feed(cache, seqs, (100, 7), seed=1)
    step = cache.step(seqs, (1, 3))
    k, v, q = states(4, 2, 128, 1, BF), states(4, 2, 128, 2, BF), rand((4, 8, 128), 3, BF)
    # tokens that go into the pages without append
    at = [(cache.tables(s)[1][p // 64], p % 64) for s, places in zip(seqs, ((100 - 64 * len(cache.tables(seqs[0])[0]),), (7, 8, 9))) for p in places]
    for i, (page, place) in enumerate(at):
        cache.plain_pages()[page, 0, 0, :, place], cache.plain_pages()[page, 0, 1, :, place] = k[i], v[i]
    want = step.attend(q, 0)
    check(want, q, step)
    step.append(k, v, 0)
    assert torch.equal(step.attend(q, 0), want)
    for layer in (1, 2):
        with pytest.raises(RuntimeError, match="appended"):
            step.attend(q, layer)
        step.append(k, v, layer)
        check(step.attend(q, layer), q, step, layer)
    step.commit()


@pytest.mark.parametrize("dtype,size", [(BF, 1e2), (BF, 1e4), (BF, 1e18), (F16, 1e2), (F16, 2e3), (F32, 1e3), (F32, 1e6), (F32, 1e18)])
@pytest.mark.parametrize("D,new", [(128, 1), (128, 5), (64, 40), (256, 1), (80, 7)])
def test_a_query_far_along_one_key_has_its_value(pkg, dtype, size, D, new):
    """Logits so large that one token has all of the weight: what the others are behind by is more than both are off by (the delta of test_gpu_paged, twice), and 40 more, so that their weights are below
    2^-57 together with how many there are."""
    kb, vb = (4, 4) if D == 80 else (4, 2)
    cache = make(pkg, D, 1, dtype, kb, vb, 20)
    (seq,) = cache.add(1)
    feed(cache, [seq], (500,), seed=1)
    step = feed(cache, [seq], (new,), seed=3, commit=False)
    k, v = (t[0] for t in contents(cache, seq))
    u, u_v = (2.0 ** -11 if dtype == BF else 2.0 ** -20) + D * 2.0 ** -24, 2.0 ** -10 if dtype != F32 else 2.0 ** -18
    unit = k / k.norm(dim=-1, keepdim=True)
    gap = (unit @ k.T).clone()
    gap = gap.diagonal() - gap.masked_fill(torch.eye(len(k), dtype=torch.bool, device=DEV), float("-inf")).amax(-1)
    # the packed token and the uncompressed one that stand out most
    old = 64 * len(cache.tables(seq)[0])
    for t in (int(gap[:old].argmax()), old + int(gap[old:500].argmax())):
        q = (size * unit[t]).to(dtype)
        z = (k @ q.double()) * D ** -0.5
        delta = u * D ** -0.5 * q.double().norm() * k.norm(dim=-1).amax()
        others = torch.cat((z[:t], z[t + 1:])).amax()
        assert float(z[t] - others - 2 * delta) >= 40.0
        out = step.attend(q.expand(new, 2, D).contiguous(), 0).double()
        assert float(((out - v[t]).norm(dim=-1) / v[t].norm()).max()) <= HALF[dtype] + u_v


@pytest.mark.parametrize("D,G,dtype,P", [(128, 4, BF, 64), (64, 2, F16, 64), (256, 4, BF, 64), (80, 2, BF, 64), (128, 2, F32, 64), (128, 4, F16, 32)])
def test_logits_that_are_all_minus_infinity_make_no_number(pkg, D, G, dtype, P):
    cache = make(pkg, D, 1, dtype, 4, 4, 64, P=P)
    seqs = cache.add(3)
    feed(cache, seqs, (300, 0, 0), seed=1)
    for counts in ((1, 1, 1), (1, 20, 1)):
        step = cache.step(seqs, counts)
        k, v, q = states(sum(counts), 1, D, 2, dtype), states(sum(counts), 1, D, 3, dtype), rand((sum(counts), G, D), 4, dtype)
        q[..., 3] = q[..., 3].abs() + 1
        k[1], k[2] = 0.0, 0.0
        k[1, 0, 3] = k[2, 0, 3] = float("-inf")          # (its queries' logits: -infinity; of the second sequence the first token alone or the first two, of the first one none)
        step.append(k, v, 0)
        for kw in ({}, {"sliding_window": 1}):
            out = step.attend(q, 0, **kw)
            nothing = torch.zeros(sum(counts), dtype=torch.bool, device=DEV)
            nothing[1:3 if sum(counts) > 3 else 2] = True
            if sum(counts) == 3:
                nothing[2] = True                        # (the third sequence's only token is the other one)
            assert bool(torch.isnan(out[nothing]).all()) and bool(torch.isfinite(out[~nothing]).all())
        step.cancel()


def test_queries_that_are_no_numbers_stay_by_themselves(pkg):
    for dtype, D, G, new in ((BF, 128, 4, 1), (F16, 64, 4, 2), (BF, 128, 4, 33), (F16, 128, 4, 33), (BF, 80, 2, 17), (F32, 128, 2, 9), (BF, 256, 4, 1), (F16, 256, 2, 20)):
        cache = make(pkg, D, 2, dtype, 4, 2 if D != 80 else 4, 30)
        seqs = cache.add(2)
        feed(cache, seqs, (500, 90), seed=1)
        step = feed(cache, seqs, (new, new), seed=2, commit=False)
        q = rand((2 * new, 2 * G, D), 3, dtype)
        want = step.attend(q, 0)
        for value in (float("inf"), float("nan")):
            wild = q.clone()
            wild[0, 0, 3] = value
            wild[new, G, 5] = -value
            got = step.attend(wild, 0)
            assert bool(torch.isnan(got[0, 0]).all()) and bool(torch.isnan(got[new, G]).all())
            got[0, 0], got[new, G] = want[0, 0], want[new, G]
            check(got, q, step)
