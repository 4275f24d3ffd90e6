"""GPU tests of beam search's choice and of caches whose sequences follow the beams.

Sums are chosen in 64 bits from sums of exponentials in float32: a sum of n terms of one sign is off by at most some 2^-24 (log2 n + a few) relative, and so its logarithm in the
absolute; returned values add the rounding to float32.  Choices have to be the oracle's, but where sums of different beams are nearer to each other than that."""
import copy

import pytest
import torch

from test_gpu_parity import DEV, outlier_kv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a HIP device; there is no CPU fallback to test")


def sums(logits, scores):
    s = scores.double().unsqueeze(-1) + torch.log_softmax(logits.double(), -1)
    bad = torch.isnan(s).any(-1, keepdim=True) | ~torch.isfinite(scores).unsqueeze(-1)
    return torch.where(bad, torch.full_like(s, float("-inf")), s)


def check(got, logits, scores, best):
    logits, scores = logits.cpu(), scores.cpu()
    B, K, V = logits.shape
    s = sums(logits, scores).flatten(1)
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices[:, :best]
    values, tokens, parents = (t.cpu() for t in got)
    assert values.dtype == torch.float32 and tokens.dtype == parents.dtype == torch.int64 and tuple(values.shape) == (B, best)
    at = parents * V + tokens
    near = torch.where(torch.isfinite(s.gather(1, order)), s.gather(1, order), torch.zeros(())).abs().amax() if order.numel() else 0.0
    slack = 2.0 ** -18 + 2.0 ** -23 * float(near)
    want = s.gather(1, order)
    same = at == order
    # where they are not the oracle's, sums meet within the slack
    mine = s.gather(1, at)
    close = (mine - want).abs() <= 2 * slack
    assert bool((same | close).all())
    assert bool((same | torch.isfinite(mine)).all())
    finite = torch.isfinite(mine)
    assert bool(((values.double() - mine).abs()[finite] <= slack).all()) and bool((values[~finite] == float("-inf")).all())
    for row in at.tolist():
        assert len(set(row)) == len(row)
    return same


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,best", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 32000, 8), (3, 5, 50257, 10), (2, 8, 128256, 16), (1, 16, 4097, 64), (5, 2, 511, 64), (1, 1, 262144, 64),
                                        (40, 4, 1000, 4), (2, 300, 33, 40), (64, 8, 16385, 8), (1, 1024, 100, 64)])
def test_choice_is_the_formula(pkg, dtype, B, K, V, best):
    g = torch.Generator(device=DEV)
    g.manual_seed(B * K + V)
    logits = (3.0 * torch.randn((B, K, V), generator=g, device=DEV)).to(dtype)
    scores = -10.0 + 2.0 * torch.randn((B, K), generator=g, device=DEV)
    got = pkg.beam_select(logits, scores, best)
    same = check(got, logits, scores, best)
    assert bool(same.all())           # (of these inputs no sums are that near)
    again = pkg.beam_select(logits, scores, best)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_ties_go_to_the_lowest(pkg):
    for B, K, V, best in ((1, 1, 40000, 64), (2, 4, 100, 64), (1, 8, 20000, 16), (3, 3, 3, 9)):
        for fill in (0.0, -50000.0):
            logits, scores = torch.full((B, K, V), fill, device=DEV), torch.zeros((B, K), device=DEV)
            values, tokens, parents = pkg.beam_select(logits, scores, best)
            at = torch.arange(best, device=DEV).expand(B, best)
            assert torch.equal(tokens, at % V) and torch.equal(parents, at // V)
            assert torch.allclose(values, torch.full_like(values, -torch.tensor(float(V)).log().item()), atol=1e-5)
    logits = torch.zeros((1, 3, 70000), device=DEV, dtype=torch.bfloat16)
    logits[0, 1, 60000:60020] = 2.0
    logits[0, 2] = logits[0, 1]
    values, tokens, parents = pkg.beam_select(logits, torch.zeros((1, 3), device=DEV), 50)
    check((values, tokens, parents), logits, torch.zeros((1, 3)), 50)
    assert tokens[0, :20].tolist() == list(range(60000, 60020)) and parents[0, :20].tolist() == [1] * 20 and parents[0, 20:40].tolist() == [2] * 20


def test_beams_that_are_no_numbers(pkg):
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    base = torch.randn((2, 4, 20000), generator=g, device=DEV)
    scores = torch.zeros((2, 4), device=DEV)
    for value, where in ((nan, (0, 1, 7)), (inf, (0, 1, 19999)), (nan, (1, 3, slice(None))), (-inf, (0, 2, slice(None))), (-inf, (1, slice(None), slice(3, None))),
                         (-inf, (0, slice(None), slice(None))), (nan, (0, slice(None), 5)), (nan, (1, 0, slice(100, 700)))):
        logits = base.clone()
        logits[where] = value
        for best in (4, 33, 64):
            check(pkg.beam_select(logits, scores, best), logits, scores, best)
    # beams that have not begun: the first one alone is continued
    begun = torch.tensor([[0.0, -inf, -inf, -inf]] * 2, device=DEV)
    values, tokens, parents = pkg.beam_select(base, begun, 4)
    assert bool((parents == 0).all()) and torch.equal(tokens, torch.topk(base[:, 0], 4).indices)
    for bad in (nan, inf, -inf):
        one = scores.clone()
        one[0, 0] = bad
        check(pkg.beam_select(base, one, 8), base, one, 8)
    none = torch.full_like(scores, -inf)
    values, tokens, parents = pkg.beam_select(base, none, 4)
    assert bool((values == -inf).all()) and tokens.tolist() == [[0, 1, 2, 3]] * 2 and bool((parents == 0).all())


def test_layouts_of_logits(pkg):
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn((3, 2, 4, 5003), generator=g, device=DEV).to(dtype)
        scores = torch.randn((3, 4), generator=g, device=DEV)
        for logits in (wide[:, 1], wide[:, 0, :, 1:5000], wide[:, 0, :, ::2], wide[:, 0, :1].expand(3, 4, 5003), wide[:, 0].transpose(0, 1).contiguous().transpose(0, 1)):
            check(pkg.beam_select(logits, scores, 8), logits, scores, 8)
        check(pkg.beam_select(wide[:, 0], scores.t().contiguous().t(), 8), wide[:, 0], scores, 8)
        check(pkg.beam_select(wide[:, 0], scores.double(), 8), wide[:, 0], scores, 8)
    assert pkg.beam_select(wide[:, 0], scores)[0].shape == (3, 4) and pkg.beam_select(wide[:, 0], scores, 0)[0].shape == (3, 0)
    assert pkg.beam_select(wide[:0, 0], scores[:0], 3)[1].shape == (0, 3)


def test_choice_replays(pkg):
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    logits, scores = torch.randn((2, 4, 30000), generator=g, device=DEV), torch.randn((2, 4), generator=g, device=DEV)
    pkg.beam_select(logits, scores, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.beam_select(logits, scores, 8)
    for _ in range(3):
        logits.copy_(torch.randn((2, 4, 30000), generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        check(got, logits, scores, 8)
        assert all(torch.equal(x, y) for x, y in zip(got, pkg.beam_select(logits, scores, 8)))


# ---- caches that follow ------------------------------------------------------------------------------------------------------------
def filled(pkg, B, H, n, w, D, dtype, layers=2, kb=4, vb=2, **kw):
    cache = pkg.V3Cache(key_bits=kb, value_bits=vb, residual_window=w, n_layers=layers, **kw)
    for layer in range(layers):
        if n + w:
            k, v = (outlier_kv((B, H, n + w, D), seed=10 * layer + i, dtype=dtype).to(DEV) for i in (0, 1))
            cache.append(k, v, layer)
    return cache


def held(cache):
    out = []
    for st in cache._stores.values():
        n = st.n_compressed
        out += [t[:, :, :n].clone() for t in (st.k_idx, st.k_nrm, st.v_idx, st.v_nrm) if t is not None]
        out += [t.clone() for t in st.window()]
        if st.weights is not None:
            out.append(st.weights[:, :, :n + st.n_recent].clone())          # (what lies behind is nobody's)
    return out


@pytest.mark.parametrize("B,H,n,w,D,dtype,kw", [
    (4, 2, 1000, 128, 128, torch.bfloat16, {}),
    (1, 2, 100, 16, 128, torch.bfloat16, {}),
    (8, 8, 333, 17, 64, torch.float16, {"kb": 6, "vb": 4}),
    (9, 1, 65, 0, 80, torch.float32, {"kb": 8, "vb": 8}),
    (12, 3, 31, 5, 45, torch.bfloat16, {"track_weights": True}),      # odd sizes: runs of two bytes
    (5, 2, 1, 1, 33, torch.float32, {"kb": 3}),
    (64, 1, 70, 8, 128, torch.bfloat16, {}),
    (65, 2, 40, 8, 128, torch.bfloat16, {"track_weights": True}),
    (300, 1, 64, 4, 96, torch.float16, {}),
    (1024, 1, 33, 3, 128, torch.bfloat16, {}),
    (6, 2, 0, 20, 128, torch.bfloat16, {}),                              # nothing packed yet
])
def test_rows_follow_their_parents(pkg, B, H, n, w, D, dtype, kw):
    g = torch.Generator()
    g.manual_seed(B)
    cycle = torch.roll(torch.arange(B), 1)
    for parents in (torch.arange(B), cycle, torch.zeros(B, dtype=torch.int64), torch.randint(0, B, (B,), generator=g), torch.randperm(B, generator=g).to(torch.int32)):
        cache = filled(pkg, B, H, n, w, D, dtype, **kw)
        for st in cache._stores.values():
            if st.weights is not None:
                st.weights.copy_(torch.rand(st.weights.shape, generator=g))
        if n > 3 and D in (128, 64, 96) and dtype != torch.float32:      # (a window that does not begin its buffer)
            t = outlier_kv((B, H, 1, D), seed=9, dtype=dtype).to(DEV)
            for layer in range(2):
                cache.append(t, t, layer)
        before = held(cache)
        cache.reorder(parents.to(DEV))
        for x, y in zip(held(cache), before):
            assert torch.equal(x, y[parents.long().to(DEV)])


def test_rows_without_a_parent_in_the_batch_stay(pkg):
    cache = filled(pkg, 4, 2, 100, 8, 128, torch.bfloat16)
    before = held(cache)
    cache.reorder(torch.tensor([4, -1, 0, 2 ** 40], device=DEV))
    for x, y in zip(held(cache), before):
        assert torch.equal(x, y[torch.tensor([0, 1, 0, 3], device=DEV)])


def test_reordering_replays(pkg):
    cache = filled(pkg, 4, 2, 100, 8, 128, torch.bfloat16)
    parents = torch.tensor([1, 2, 3, 0], device=DEV)
    before = held(cache)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.reorder(parents)
    order = torch.arange(4, device=DEV)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        order = order[parents]
        for x, y in zip(held(cache), before):
            assert torch.equal(x, y[order])
        parents.copy_(torch.tensor([[3, 3, 0, 1], [0, 1, 2, 3], [2, 2, 2, 2], [1, 0, 1, 0]][i]))


def test_beam_search_over_a_dense_and_a_paged_cache(pkg):
    """The same search over both: the same beams are chosen as if every beam had a cache to itself."""
    G, K, H, D, V, n = 2, 3, 2, 128, 500, 140
    dense = pkg.V3Cache(residual_window=64, n_layers=1)
    paged = pkg.PagedV3Cache(D, H, residual_window=64, n_layers=1, pages=40, plain_pages=60, device=DEV)
    k, v = (outlier_kv((G, H, n, D), seed=i, dtype=torch.bfloat16).to(DEV) for i in (0, 1))
    dense.append(k.repeat_interleave(K, 0), v.repeat_interleave(K, 0), 0)
    first = paged.add(G)
    step = paged.step(first, n)
    step.append(k.transpose(1, 2).flatten(0, 1), v.transpose(1, 2).flatten(0, 1), 0)
    step.commit()
    copies = paged.fork([s for s in first for _ in range(K - 1)])
    seqs = [s for g in range(G) for s in [first[g]] + copies[g * (K - 1):(g + 1) * (K - 1)]]
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    head, embed = torch.randn((H * 2 * D, V), generator=g, device=DEV), torch.randn((V, 3, H * 2, D), generator=g, device=DEV)
    scores = torch.tensor([[0.0] + [float("-inf")] * (K - 1)] * G, device=DEV)
    tokens, paths = torch.zeros((G, K), dtype=torch.int64, device=DEV), torch.zeros((G, K, 0), dtype=torch.int64, device=DEV)
    for i in range(100):
        x = embed[tokens.flatten()].to(torch.bfloat16)                    # [G K, 3, 2 H, D]
        q, kn, vn = x[:, 0], x[:, 1, :H], x[:, 2, :H]
        dense.append(kn.unsqueeze(2), vn.unsqueeze(2), 0)
        a = dense.attend(q.unsqueeze(2), 0)[:, :, 0]
        step = paged.step(seqs, 1)
        step.append(kn, vn, 0)
        b = step.attend(q, 0)
        step.commit()
        # both within their roundings of one another (what is packed is not the same: a page at a time here)
        if i < 10:
            assert ((a.float() - b.float()).norm() / a.float().norm()).item() < 0.35
        logits = (b.float().flatten(1) @ head).view(G, K, V)
        values, tokens, parents = paged.beam_step(seqs, logits, scores)
        again = dense.beam_step(logits, scores)
        assert torch.equal(values, again[0]) and torch.equal(tokens, again[1]) and torch.equal(parents, again[2])
        paths = torch.cat((torch.take_along_dim(paths, parents.unsqueeze(-1), 1), tokens.unsqueeze(-1)), -1)
        scores = values
    # what the caches hold is what each path's tokens were
    paths = torch.cat((torch.zeros((G, K, 1), dtype=torch.int64, device=DEV), paths[:, :, :-1]), -1).flatten(0, 1)
    st = dense._stores[0]
    recent = embed[paths[:, -64:]][:, :, 1, :H].transpose(1, 2).to(torch.bfloat16)
    assert torch.equal(st.window()[0], recent)
    for row, s in enumerate(seqs):
        pages, plain = paged.tables(s)
        count = paged.lengths([s])[0] - 64 * len(pages)
        held_keys = paged.plain_pages()[plain, 0, 0].transpose(0, 1).flatten(1, 2)[:, :count]
        assert torch.equal(held_keys[:, -64:], recent[row])
        old = torch.cat((k[row // K], embed[paths[row]][:, 1, :H].transpose(0, 1).to(torch.bfloat16)), 1)[:, :64 * len(pages)]
        want = paged.codec(0).key_compressor.compress(old.unsqueeze(0))
        assert torch.equal(paged.packed_pages(0)[0][pages].transpose(0, 1).flatten(1, 2), want["idx_bytes"][0])


def test_hugging_face_caches_follow_their_beams(pkg):
    pytest.importorskip("transformers")
    cache = pkg.hf_cache_class()(residual_window=8, n_layers=1)
    k, v = (outlier_kv((4, 2, 50, 128), seed=i, dtype=torch.bfloat16).to(DEV) for i in (0, 1))
    full_k, full_v = cache.update(k, v, 0)
    cache.reorder_cache(torch.tensor([2, 0, 0, 3], device=DEV))
    t = outlier_kv((4, 2, 1, 128), seed=5, dtype=torch.bfloat16).to(DEV)
    got_k, got_v = cache.update(t, t, 0)
    order = torch.tensor([2, 0, 0, 3], device=DEV)
    assert torch.equal(got_k[:, :, :42], full_k[order][:, :, :42]) and torch.equal(got_v[:, :, :42], full_v[order][:, :, :42])
    assert torch.equal(got_k[:, :, 43:50], k[order][:, :, 43:50]) and torch.equal(got_k[:, :, 50:], t)


def test_refusals(pkg):
    cache = filled(pkg, 4, 2, 100, 8, 128, torch.bfloat16)
    native = pkg._native
    for bad in (torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros((4, 1), dtype=torch.int64, device=DEV), torch.zeros(4, device=DEV), torch.zeros(4, dtype=torch.bool, device=DEV), [0, 1, 2, 3]):
        with pytest.raises(ValueError):
            cache.reorder(bad)
    with pytest.raises(native.TqError):
        cache.reorder(torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        filled(pkg, 1025, 1, 4, 1, 8, torch.bfloat16).reorder(torch.zeros(1025, dtype=torch.int64, device=DEV))
    pkg.V3Cache().reorder(torch.zeros(3, dtype=torch.int64, device=DEV))          # nothing is cached
    logits, scores = torch.zeros((2, 2, 10), device=DEV), torch.zeros((2, 2), device=DEV)
    for args in ((logits[0], scores), (logits, scores[:1]), (logits, scores, 21), (logits, scores, -1), (logits, scores, 1.5), (logits, scores, True), (logits, scores.long())):
        with pytest.raises(ValueError):
            pkg.beam_select(*args)
    with pytest.raises(ValueError):
        pkg.beam_select(torch.zeros((1, 1, 100), device=DEV), torch.zeros((1, 1), device=DEV), 65)
    with pytest.raises(ValueError):
        pkg.beam_select(torch.zeros((1, 1025, 2), device=DEV), torch.zeros((1, 1025), device=DEV), 1)
    for args in ((logits.cpu(), scores), (logits, scores.cpu()), (logits.double(), scores)):
        with pytest.raises(native.TqError):
            pkg.beam_select(*args)
    with pytest.raises(ValueError):
        cache.beam_step(torch.zeros((1, 3, 10), device=DEV), torch.zeros((1, 3), device=DEV))
    assert copy.deepcopy(cache) is not cache
