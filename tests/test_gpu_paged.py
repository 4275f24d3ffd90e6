"""GPU tests of the paged cache: attention of new tokens over packed and plain pages against the formula in float64, what lies in the pages, sequences that share, fork and move.

Tolerances.  With u = 2^-11 (bfloat16: queries and levels enter the products as one fp16 value each, half a step 2^-12 relative) or u = 2^-20 (two fp16 terms each, 22 bits, and what is
left out) and D 2^-24 for a float32 sum of D products, a logit is off by at most delta = (u + D 2^-24) * scale * |q| |k|.  The cap's slope is at most one, so it adds only its own
evaluation (half a dozen roundings of values up to the cap, 2^-21 cap); the bias by distance adds the rounding of the sum, 2^-23 of the largest |logit|.  The weights of a row are off by
2 delta together, and a result by expm1(2 delta) + u_v of the longest value vector that the row sees (u_v = 2^-10: weight, level and norm, an fp16 rounding of 2^-12 each and
as much for the sums of a few thousand tokens; 2^-18 in two terms), plus half a step of its type."""
import pytest
import torch

from test_gpu_many import HALF, dequantised
from test_gpu_parity import DEV, outlier_kv

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a HIP device; there is no CPU fallback to test")


def rand(shape, seed, dtype):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def make(pkg, D=128, H=2, dtype=BF, kb=4, vb=2, window=40, layers=1, pages=64, plain=64, P=64, **kw):
    cache = pkg.PagedV3Cache(D, H, kb, vb, window, n_layers=layers, pages=pages, plain_pages=plain, page_tokens=P, dtype=dtype, device=DEV, **kw)
    # memory as it may come: NaN in every float
    cache._pool.fill_(255)
    cache._plain.fill_(float("nan"))
    return cache


def states(n, H, D, seed, dtype):
    """[n, H, D] with outlier channels."""
    return outlier_kv((1, H, max(n, 1), D), seed=seed, dtype=dtype)[0].transpose(0, 1)[:n].contiguous().to(DEV)


def feed(cache, seqs, counts, seed=0, kept=None, commit=True):
    """A step of random tokens in every layer; kept: (sequence, layer) -> list of (keys, values)."""
    step = cache.step(seqs, counts)
    for layer in range(cache.n_layers):
        k, v = (states(sum(step.counts), cache.kv_heads, cache.head_dim, 1000 * seed + 10 * layer + i, cache.dtype) for i in (1, 2))
        step.append(k, v, layer)
        at = 0
        for s, c in zip(seqs, step.counts):
            if kept is not None:
                kept.setdefault((s, layer), []).append((k[at:at + c], v[at:at + c]))
            at += c
    if commit:
        step.commit()
    return step


def contents(cache, seq, layer=0):
    """Keys and values a sequence holds, float64 [H, tokens, D], from its pages."""
    pages, plain = cache.tables(seq)
    codec, total = cache.codec(layer), cache.lengths([seq])[0]
    views, out = cache.packed_pages(layer), []
    for side, comp in enumerate((codec.key_compressor, codec.val_compressor)):
        idx, nrm = (t[torch.tensor(pages, dtype=torch.int64, device=DEV)].transpose(0, 1).flatten(1, 2) for t in views[2 * side:2 * side + 2])
        old = dequantised(comp, (idx, nrm))
        new = cache.plain_pages()[torch.tensor(plain, dtype=torch.int64, device=DEV), layer, side].transpose(0, 1).flatten(1, 2)
        out.append(torch.cat((old, new[:, :total - old.shape[1]].double()), 1))
    return out


def check(out, q, step, layer=0, scale=None, softcap=None, slopes=None, sliding_window=None):
    """Every result vector within the bound of the module's docstring."""
    cache, at = step.cache, 0
    D, H, dtype = cache.head_dim, cache.kv_heads, cache.dtype
    scale = D ** -0.5 if scale is None else scale
    u, u_v = (2.0 ** -11, 2.0 ** -10) if dtype == BF else (2.0 ** -20, 2.0 ** -18)
    assert out.shape == q.shape and out.dtype == q.dtype and bool(torch.isfinite(out).all())
    errors = []
    for s, new in zip(step.seqs, step.counts):
        if not new:
            continue
        k, v = contents(cache, s, layer)
        total, Hq = k.shape[1], q.shape[1]
        G = Hq // H
        mine = q[at:at + new].double().transpose(0, 1).reshape(H, G * new, D)
        z = (mine @ k.transpose(1, 2)).reshape(Hq, new, total) * scale
        if softcap:
            z = softcap * torch.tanh(z / softcap)
        distance = torch.arange(total - new, total, device=DEV).unsqueeze(1) - torch.arange(total, device=DEV)
        if slopes is not None:
            z = z - slopes.double().view(Hq, 1, 1) * distance
        seen = (distance >= 0) & (distance < (sliding_window or total + 1))
        z = torch.where(seen, z, torch.full_like(z, float("-inf")))
        p = torch.softmax(z, -1)
        ref = (p.reshape(H, G * new, total) @ v).reshape(Hq, new, D).transpose(0, 1)
        reach = (mine.norm(dim=-1).view(H, G * new, 1) * k.norm(dim=-1).view(H, 1, total)).reshape(Hq, new, total)
        delta = (u + D * 2.0 ** -24) * abs(scale) * torch.where(seen, reach, torch.zeros_like(reach)).amax(-1)
        delta = delta + (2.0 ** -21 * softcap if softcap else 0.0) + (2.0 ** -23 * torch.where(seen, z, torch.zeros_like(z)).abs().amax(-1) if slopes is not None else 0.0)
        lengths = v.norm(dim=-1).repeat_interleave(G, 0).unsqueeze(1)
        longest = torch.where(seen, lengths, torch.zeros_like(lengths)).amax(-1)
        got = out[at:at + new].double()
        bound = HALF[dtype] * ref.norm(dim=-1) + ((torch.expm1(2 * delta) + u_v) * longest).transpose(0, 1) + 1e-30
        worst = ((got - ref).norm(dim=-1) / bound).max().item()
        assert worst <= 1.0, f"sequence {s}: error {worst:.3f} of the bound"
        errors.append(((got - ref).norm().item(), ref.norm().item()))
        at += new
    if errors:       # and not only within the worst case: the whole tensor as near as its type has it
        rel = sum(e ** 2 for e, _ in errors) ** 0.5 / sum(r ** 2 for _, r in errors) ** 0.5
        assert rel <= {BF: 5e-3, F16: 1e-3, F32: 1e-5}[dtype], rel


SHAPES = [
    # D, H, group, dtype, kb, vb, page, window, lengths before, new tokens
    (128, 2, 4, BF, 4, 2, 64, 40, (0, 1, 63, 64, 65, 300), (1, 1, 1, 1, 1, 1)),
    (128, 8, 4, BF, 4, 2, 64, 128, (700, 0, 1000), (1, 1, 1)),
    (128, 1, 1, BF, 4, 2, 32, 0, (0, 31, 32, 33, 500), (1, 1, 1, 1, 33)),
    (128, 2, 7, BF, 3, 2, 64, 17, (1000, 0, 129), (70, 5, 0)),
    (128, 2, 4, F16, 6, 4, 64, 40, (300, 5, 64), (1, 40, 64)),
    (128, 2, 2, F32, 4, 2, 64, 40, (300, 5, 64), (1, 40, 3)),
    (64, 3, 4, BF, 4, 2, 64, 20, (500, 10), (33, 1)),
    (64, 2, 16, F16, 6, 4, 128, 64, (600, 250, 3), (1, 9, 1)),
    (64, 2, 2, BF, 8, 8, 256, 64, (600, 250, 3), (20, 1, 1)),
    (80, 2, 4, BF, 4, 2, 64, 20, (300, 90), (17, 1)),
    (80, 8, 1, F32, 4, 4, 64, 128, (400, 77), (77, 77)),
    (88, 2, 3, F16, 4, 4, 64, 20, (200,), (40,)),
    (96, 2, 8, BF, 8, 2, 64, 20, (333, 64), (1, 70)),
    (256, 1, 4, BF, 4, 2, 64, 20, (300, 64), (1, 40)),
    (256, 2, 2, F16, 8, 4, 64, 33, (200, 1), (3, 1)),
    (256, 1, 2, F32, 2, 8, 32, 8, (100, 40), (9, 1)),
    (128, 1, 8, BF, 8, 4, 1024, 100, (2500,), (5,)),
    (128, 2, 4, BF, 5, 7, 64, 0, (640, 64), (256, 1)),
]


@pytest.mark.parametrize("shaped", [{}, {"softcap": 5.0}, {"slopes": True}, {"sliding_window": 70}, {"softcap": 30.0, "slopes": True, "sliding_window": 33}], ids=["plain", "cap", "slopes", "window", "all"])
@pytest.mark.parametrize("D,H,G,dtype,kb,vb,P,window,before,new", SHAPES)
def test_attention_is_the_formula(pkg, D, H, G, dtype, kb, vb, P, window, before, new, shaped):
    cache = make(pkg, D, H, dtype, kb, vb, window, P=P, pages=64, plain=max(16, 4096 // P))
    seqs = cache.add(len(before))
    feed(cache, seqs, before, seed=1)
    step = feed(cache, seqs, new, seed=2, commit=False)
    q = rand((sum(new), H * G, D), 3, dtype)
    shaped = dict(shaped)
    if "slopes" in shaped:
        shaped["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / (H * G)) for i in range(H * G)], device=DEV)
    out = step.attend(q, 0, **shaped)
    check(out, q, step, **shaped)
    assert torch.equal(out, step.attend(q, 0, **shaped)), "a call repeated has the same bits"


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 63, 64, 65, 500, 2 ** 31])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_sliding_windows_of_any_length(pkg, window, dtype):
    cache = make(pkg, dtype=dtype, window=16, plain=64)
    seqs = cache.add(3)
    feed(cache, seqs, (200, 64, 1))
    step = feed(cache, seqs, (1, 100, 2), seed=1, commit=False)
    q = rand((103, 8, 128), 5, dtype)
    check(step.attend(q, 0, sliding_window=window), q, step, sliding_window=window)


def test_splits_of_long_rows_meet(pkg):
    for dtype, kb, vb, G, new in ((BF, 4, 2, 4, 1), (F16, 6, 4, 4, 1), (BF, 4, 2, 4, 100), (F32, 4, 4, 2, 3)):
        cache = make(pkg, H=2, dtype=dtype, kb=kb, vb=vb, window=100, pages=400, plain=200)
        seqs = cache.add(2)
        feed(cache, seqs, (9000, 333))
        feed(cache, seqs, (9000, 0), seed=7)
        step = feed(cache, seqs, (new, 1), seed=1, commit=False)
        q = rand((new + 1, 2 * G, 128), 5, dtype)
        for kw in ({}, {"softcap": 20.0}, {"sliding_window": 5000}):
            check(step.attend(q, 0, **kw), q, step, **kw)


@pytest.mark.parametrize("D,H,G,dtype,kb,vb,n,new", [
    (128, 8, 4, BF, 4, 2, 170, 1), (128, 8, 1, BF, 4, 2, 170, 1), (128, 4, 4, BF, 4, 2, 170, 2), (128, 8, 4, F16, 6, 4, 100, 4), (64, 8, 4, F16, 6, 4, 170, 1), (64, 8, 8, BF, 8, 8, 100, 1),
    (96, 8, 2, BF, 4, 2, 170, 1), (96, 8, 16, F16, 3, 2, 70, 1), (256, 8, 4, BF, 4, 2, 100, 1), (256, 8, 8, BF, 4, 2, 100, 1), (256, 8, 16, F16, 8, 8, 70, 1), (80, 8, 4, BF, 4, 2, 100, 1)])
def test_more_rows_than_the_device_takes_at_a_time(pkg, D, H, G, dtype, kb, vb, n, new):
    lengths = [(0, 700, 64, 129, 1, 320, 63)[i % 7] + 3 * (i // 7) for i in range(n)]
    cache = make(pkg, D, H, dtype, kb, vb, 20, pages=16 * n, plain=16 * n)
    seqs = cache.add(n)
    feed(cache, seqs, lengths, seed=1)
    step = feed(cache, seqs, [new] * n, seed=2, commit=False)
    q = rand((n * new, H * G, D), 3, dtype)
    check(step.attend(q, 0), q, step)
    check(step.attend(q, 0, sliding_window=90), q, step, sliding_window=90)


@pytest.mark.parametrize("D,H,G,dtype,kb,vb,P", [(128, 2, 4, BF, 4, 2, 64), (128, 1, 7, F16, 4, 2, 32), (64, 2, 1, F16, 6, 4, 64), (64, 1, 4, BF, 4, 2, 128), (80, 2, 4, BF, 4, 2, 64), (96, 1, 2, F16, 4, 2, 64),
                                                 (256, 1, 2, BF, 4, 2, 64), (256, 1, 1, F16, 8, 8, 256), (128, 1, 2, F32, 4, 2, 64), (72, 1, 1, F32, 4, 4, 64)])
def test_prompts_that_nothing_is_packed_of_yet(pkg, D, H, G, dtype, kb, vb, P):
    new = (600, 1, 257, 0, 32, 255)
    cache = make(pkg, D, H, dtype, kb, vb, 64, P=P, pages=64, plain=128)
    seqs = cache.add(len(new))
    feed(cache, seqs, (0, 300, 31, 5, 0, 1), seed=1)
    step = feed(cache, seqs, new, seed=2, commit=False)
    q = rand((sum(new), H * G, D), 3, dtype)
    check(step.attend(q, 0), q, step)
    check(step.attend(q, 0, sliding_window=45, softcap=20.0), q, step, sliding_window=45, softcap=20.0)


def test_values_that_are_no_numbers_in_a_long_prompt(pkg):
    for dtype, D in ((BF, 128), (F16, 64), (BF, 80), (F32, 128)):
        cache = make(pkg, D, 1, dtype, 4, 4, 64, plain=32)
        (seq,) = cache.add(1)
        step = cache.step([seq], 600)
        k, v = states(600, 1, D, 1, dtype), states(600, 1, D, 2, dtype)
        q = rand((600, 2, D), 3, dtype)
        step.append(k, v, 0)
        whole = step.attend(q, 0)
        v[333, 0, 5], v[500, 0, 6], v[501, 0, 6], v[599, 0, 7] = float("inf"), float("inf"), float("-inf"), float("nan")
        step.append(k, v, 0)
        out = step.attend(q, 0)
        rows = torch.arange(600, device=DEV)
        want = whole.clone()
        want[rows >= 333, :, 5] = float("inf")
        want[rows == 500, :, 6] = float("inf")
        want[rows >= 501, :, 6] = float("nan")
        want[rows == 599, :, 7] = float("nan")
        assert torch.equal(torch.isfinite(out), torch.isfinite(want)) and torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(out[torch.isfinite(out)], whole[torch.isfinite(want)])
        out = step.attend(q, 0, sliding_window=100)
        assert bool(torch.isfinite(out[433:500]).all()) and bool(torch.isinf(out[333:433, :, 5]).all()) and bool(torch.isfinite(out[501:599, :, 5]).all())


@pytest.mark.parametrize("D,G,dtype,kb,vb,new", [(64, 71, BF, 4, 2, (1, 3, 1)), (128, 40, F16, 4, 2, (1, 1, 2)), (256, 33, BF, 4, 2, (1, 2, 1)), (80, 64, F32, 4, 4, (2, 1, 1)), (128, 128, BF, 8, 8, (1, 1, 1)),
                                                 (96, 17, F16, 4, 4, (1, 1, 1))])
def test_many_query_heads_of_one_kv_head(pkg, D, G, dtype, kb, vb, new):
    cache = make(pkg, D, 1, dtype, kb, vb, 30, pages=64, plain=40)
    seqs = cache.add(3)
    feed(cache, seqs, (2000, 0, 95), seed=1)
    step = feed(cache, seqs, new, seed=2, commit=False)
    q = rand((sum(new), G, D), 3, dtype)
    check(step.attend(q, 0), q, step)
    check(step.attend(q, 0, sliding_window=1000), q, step, sliding_window=1000)


def test_threads_and_steps_at_once(pkg):
    import threading
    caches, steps, qs, wants = [], [], [], []
    for k in range(4):
        cache = make(pkg, 128, 4, BF if k % 2 else F16, pages=80, plain=80)
        seqs = cache.add(5)
        feed(cache, seqs, (900, 3, 64, 2500, 0), seed=k)
        step = feed(cache, seqs, (1, 1, 20, 1, 70), seed=10 + k, commit=False)
        q = rand((93, 16, 128), k, cache.dtype)
        caches.append(cache); steps.append(step); qs.append(q); wants.append(step.attend(q, 0))
    got = [[] for _ in range(4)]

    def work(k):
        stream = torch.cuda.Stream(DEV) if k % 2 else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[k].append(steps[k].attend(qs[k], 0))
            stream.synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(len(g) == 20 and all(torch.equal(x, w) for x in g) for g, w in zip(got, wants))


def test_layers_of_their_own_widths_and_codecs(pkg):
    cache = make(pkg, 128, 2, BF, 4, 2, 20, layers=4, protected_layers=1, pages=40, plain=40)
    assert len({(cache.codec(i).key_bits, cache.codec(i).value_bits) for i in range(4)}) > 1
    seqs = cache.add(3)
    feed(cache, seqs, (300, 0, 70), seed=1)
    q = rand((5, 8, 128), 3, BF)

    def every_layer(step):
        for _ in range(2):
            for layer in range(4):
                check(step.attend(q, layer), q, step, layer)
                check(step.attend(q, layer, sliding_window=33), q, step, layer, sliding_window=33)
    every_layer(feed(cache, seqs, (1, 3, 1), seed=2, commit=False))
    every_layer(feed(cache, seqs, (1, 3, 1), seed=3, commit=False))
    cache.resize(pages=50, plain_pages=50)
    step = feed(cache, seqs, (1, 3, 1), seed=4, commit=False)
    every_layer(step)
    other = pkg.PagedV3Cache(128, 2, 4, 2, 20, n_layers=4, pages=1, plain_pages=1, dtype=BF, device=DEV)
    before = step.attend(q, 1)
    cache.codec(1).key_compressor = pkg.MSECompressor(128, cache.codec(1).key_bits, seed=77, device="cpu")       # (what is packed means something else now)
    assert other.codec(1).key_bits == cache.codec(1).key_bits and not torch.equal(before, step.attend(q, 1))
    check(step.attend(q, 1), q, step, 1)


@pytest.mark.parametrize("D,H,G,dtype,kb,vb,most", [(128, 8, 1, BF, 4, 2, 4), (64, 4, 2, F16, 6, 4, 2), (128, 4, 1, F16, 8, 8, 8), (96, 4, 4, BF, 4, 2, 4), (256, 4, 1, BF, 4, 2, 8), (256, 2, 2, F16, 4, 2, 8)])
def test_rows_of_different_numbers_of_query_vectors(pkg, D, H, G, dtype, kb, vb, most):
    n = 150
    cache = make(pkg, D, H, dtype, kb, vb, 30, pages=12 * n, plain=12 * n)
    seqs = cache.add(n)
    feed(cache, seqs, [(0, 200, 64, 450, 31, 130)[i % 6] for i in range(n)], seed=1)
    new = [(i * 7) % (most + 1) for i in range(n)]
    step = feed(cache, seqs, new, seed=2, commit=False)
    q = rand((sum(new), H * G, D), 3, dtype)
    check(step.attend(q, 0), q, step)
    check(step.attend(q, 0, sliding_window=40, softcap=30.0), q, step, sliding_window=40, softcap=30.0)


def test_scale_and_layouts_of_queries(pkg):
    cache = make(pkg, H=2, layers=2, protected_layers=1)            # (8 bits in both)
    seqs = cache.add(2)
    feed(cache, seqs, (150, 10))
    step = feed(cache, seqs, (3, 30), seed=1, commit=False)
    q = rand((33, 4, 128), 5, BF)
    want = step.attend(q, 1, scale=0.3)
    check(want, q, step, layer=1, scale=0.3)
    assert torch.equal(step.attend(q.transpose(0, 1).contiguous().transpose(0, 1), 1, scale=0.3), want)      # head by head
    odd = torch.empty(33 * 4 * 128 + 1, dtype=BF, device=DEV)[1:].view(33, 4, 128).copy_(q)
    assert torch.equal(step.attend(odd, 1, scale=0.3), want)                                                   # no 16-byte loads
    wide = torch.zeros((33, 4, 256), dtype=BF, device=DEV)
    wide[:, :, ::2] = q
    assert torch.equal(step.attend(wide[:, :, ::2], 1, scale=0.3), want)                                       # elements apart
    assert torch.equal(step.attend(q[:, :1].expand(33, 4, 128), 1), step.attend(q[:, :1].repeat(1, 4, 1), 1))  # one query for all heads


@pytest.mark.parametrize("dtype,D,kb,vb", [(BF, 128, 4, 2), (F16, 64, 6, 4), (F32, 128, 8, 8), (BF, 80, 4, 4), (BF, 256, 3, 2)])
def test_pages_hold_what_the_codec_makes(pkg, dtype, D, kb, vb):
    cache, kept = make(pkg, D, 2, dtype, kb, vb, window=50, layers=3, plain=40), {}
    seqs = cache.add(3)
    for i, counts in enumerate(((70, 3, 0), (1, 200, 64), (130, 1, 50), (0, 0, 1))):
        feed(cache, seqs, counts, seed=i, kept=kept)
    for s in seqs:
        for layer in range(3):
            pages, plain = cache.tables(s)
            k, v = (torch.cat([t[i] for t in kept[s, layer]]).transpose(0, 1) for i in (0, 1))
            total = k.shape[1]
            assert cache.lengths([s]) == [total] and len(pages) == max(0, total - 50) // 64 and len(plain) == -(-(total - 64 * len(pages)) // 64)
            views = cache.packed_pages(layer)
            for n, p in enumerate(pages):
                for side, comp in enumerate((cache.codec(layer).key_compressor, cache.codec(layer).val_compressor)):
                    want = comp.compress((k, v)[side][:, 64 * n:64 * n + 64].unsqueeze(0))
                    assert torch.equal(views[2 * side][p], want["idx_bytes"][0]) and torch.equal(views[2 * side + 1][p], want["vec_norms"][0])
            for side in (0, 1):
                held = cache.plain_pages()[plain, layer, side].transpose(0, 1).flatten(1, 2)[:, :total - 64 * len(pages)]
                assert torch.equal(held, (k, v)[side][:, 64 * len(pages):])


def test_same_bytes_as_a_dense_cache(pkg):
    paged, dense = make(pkg, H=2, window=64, layers=2), pkg.V3Cache(residual_window=64, n_layers=2)
    seqs = paged.add(2)
    step = paged.step(seqs, 192)
    for layer in range(2):
        k, v = (states(384, 2, 128, layer + i, BF) for i in (10, 20))
        step.append(k, v, layer)
        dense.append(*(t.view(2, 192, 2, 128).transpose(1, 2) for t in (k, v)), layer)
    step.commit()
    for layer in range(2):
        st, views = dense._stores[layer], paged.packed_pages(layer)
        for view, t in zip(views, (st.k_idx, st.k_nrm, st.v_idx, st.v_nrm)):
            for b, s in enumerate(seqs):
                held = view[torch.tensor(paged.tables(s)[0], device=DEV)].transpose(0, 1).flatten(1, 2)
                assert torch.equal(held, t[b, :, :128])


def test_values_that_are_no_numbers_stay_with_those_who_see_them(pkg):
    for dtype in (BF, F16, F32):
        cache = make(pkg, H=1, dtype=dtype, window=30)
        seqs = cache.add(2)
        feed(cache, seqs, (100, 50))
        step = cache.step(seqs, (40, 40))
        k, v = states(80, 1, 128, 4, dtype), states(80, 1, 128, 5, dtype)
        step.append(k, v, 0)
        q = rand((80, 2, 128), 6, dtype)
        want = [step.attend(q, 0), step.attend(q, 0, sliding_window=5)]
        v2, k2 = v.clone(), k.clone()
        v2[20, 0, 7], v2[21, 0, 8] = float("inf"), float("nan")
        k2[30] = float("nan")
        step.append(k2, v2, 0)
        for got, ref, window in zip((step.attend(q, 0), step.attend(q, 0, sliding_window=5)), want, (1000, 5)):
            assert torch.equal(got[:20], ref[:20]) and torch.equal(got[40:], ref[40:])
            own = got[20:30].float()
            reach = torch.arange(10) < window
            assert bool((own[reach][:, :, 7] == float("inf")).all()) and bool(torch.isnan(own[1:][reach[:9]][:, :, 8]).all())
            rest = torch.ones(128, dtype=torch.bool)
            rest[7] = rest[8] = False
            assert torch.equal(got[20:30][:, :, rest], ref[20:30][:, :, rest])
            assert bool(torch.isnan(got[30:min(40, 30 + window)]).all())
        assert torch.equal(step.attend(q, 0, sliding_window=5)[36:40], want[1][36:40])


def test_large_logits(pkg):
    for dtype, size in ((BF, 300.0), (F16, 100.0), (F32, 1e4)):
        cache = make(pkg, H=1, dtype=dtype, window=20)
        seqs = cache.add(1)
        feed(cache, seqs, (500,))
        step = feed(cache, seqs, (2,), seed=3, commit=False)
        q = rand((2, 2, 128), 6, dtype) * size
        out = step.attend(q, 0)
        k, v = contents(cache, seqs[0])
        # (one key has all of the weight, or what rounding makes of the first few)
        assert bool(torch.isfinite(out).all()) and bool((out.double().norm(dim=-1) <= 1.01 * v.norm(dim=-1).amax()).all())
        check(step.attend(q, 0, softcap=10.0), q, step, softcap=10.0) if dtype != BF else None


def test_a_cap_far_above_the_logits(pkg):
    # cap tanh(z / cap) is z (1 - (z / cap)^2 / 3): with |z| below 100 and a cap of 10^5 or more no different from z by 2^-21 of it, so weights by 2^-15 at most; what is left is which
    # way a result is rounded (few, by 2^-7 or 2^-10 of themselves)
    for dtype, most in ((BF, 0.0), (F16, 0.0), (F32, 2e-5)):
        for new in (1, 20):
            cache = make(pkg, 128, 2, dtype)
            seqs = cache.add(2)
            feed(cache, seqs, (500, 70), seed=1)
            step = feed(cache, seqs, (new, new), seed=2, commit=False)
            q = rand((2 * new, 8, 128), 3, dtype)
            plain = step.attend(q, 0).double()
            for cap in (1e5, 1e12, 2.0 ** 100):
                if dtype != F32:
                    with pytest.raises(ValueError):
                        step.attend(q, 0, softcap=cap)
                    continue
                assert (step.attend(q, 0, softcap=cap).double() - plain).norm() <= most * plain.norm()
            for cap in (1024.0, 700.0):
                check(step.attend(q, 0, softcap=cap), q, step, softcap=cap)
            small = step.attend(q, 0, softcap=2.0 ** -100).double()      # all logits are zero
            assert bool(torch.isfinite(small).all())


def test_a_step_that_is_taken_back(pkg):
    cache, other = make(pkg), make(pkg)
    kept = []
    for c in (cache, other):
        seqs = c.add(3)
        feed(c, seqs, (100, 0, 63), seed=1)
        if c is cache:
            before = c.free_pages(), c.lengths(seqs), [c.tables(s) for s in seqs]
            step = c.step(seqs, (200, 1, 65))
            with pytest.raises(RuntimeError):
                c.free(seqs)                     # (its commit lacks every layer)
            step.cancel()
            assert (c.free_pages(), c.lengths(seqs), [c.tables(s) for s in seqs]) == before
            step.cancel()
            with pytest.raises(RuntimeError):
                step.append(states(266, 2, 128, 1, BF), states(266, 2, 128, 2, BF), 0)
        step = feed(c, seqs, (1, 2, 130), seed=2, commit=False)
        q = rand((133, 8, 128), 3, BF)
        kept.append(step.attend(q, 0))
        step.commit()
        step.cancel()                            # (nothing: it is over)
        assert c.lengths(seqs) == [101, 2, 193]
    assert torch.equal(*kept)


def test_a_recorded_step_outlives_its_name(pkg):
    cache = make(pkg)
    seqs = cache.add(2)
    feed(cache, seqs, (300, 70), seed=1)
    step = feed(cache, seqs, (1, 1), seed=2, commit=False)
    q = rand((2, 8, 128), 3, BF)
    want = step.attend(q, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.attend(q, 0)
    step.commit()
    del step
    noise = [torch.full((1 << k,), 0x7fffffff, dtype=torch.int32, device=DEV) for k in range(4, 14) for _ in range(8)]       # (what has been given back is taken and overwritten)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and len(noise)


def test_beams_fork_share_and_move(pkg):
    cache, kept = make(pkg, H=2, window=70, layers=2, plain=60), {}
    (a,) = cache.add(1)
    feed(cache, [a], 300, kept=kept)
    free = cache.free_pages()
    beams = [a] + cache.fork([a, a, a])
    for s in beams[1:]:
        for layer in range(2):
            kept[s, layer] = list(kept[a, layer])
    assert [cache.tables(s)[0] for s in beams] == [cache.tables(a)[0]] * 4
    assert cache.free_pages() == (free[0], free[1] - 3)           # (300 tokens: 44 in the page being filled)
    g = torch.Generator()
    g.manual_seed(1)
    for i in range(90):
        step = feed(cache, beams, 1, seed=100 + i, kept=kept, commit=False)
        if i % 30 == 0:
            q = rand((4, 8, 128), i, BF)
            for layer in range(2):
                check(step.attend(q, layer), q, step, layer)
        step.commit()
        parents = torch.randint(0, 4, (4,), generator=g).tolist()
        cache.reorder(beams, parents if i % 2 else torch.tensor(parents, device=DEV))
        kept = {(s, layer): list(kept[beams[p], layer]) for s, p in zip(beams, parents) for layer in range(2)}
        if i == 45:
            cache.resize(pages=20, plain_pages=50)
    for s in beams:
        for layer in range(2):
            k, v = (torch.cat([t[i] for t in kept[s, layer]]).transpose(0, 1) for i in (0, 1))
            pages, plain = cache.tables(s)
            n = 64 * len(pages)
            assert n == (390 - 70) // 64 * 64 and cache.lengths([s]) == [390]
            for side, comp in enumerate((cache.codec(layer).key_compressor, cache.codec(layer).val_compressor)):
                want = comp.compress((k, v)[side][:, :n].unsqueeze(0))
                views = cache.packed_pages(layer)
                assert torch.equal(views[2 * side][torch.tensor(pages, device=DEV)].transpose(0, 1).flatten(1, 2), want["idx_bytes"][0])
                held = cache.plain_pages()[plain, layer, side].transpose(0, 1).flatten(1, 2)[:, :390 - n]
                assert torch.equal(held, (k, v)[side][:, n:])
    cache.free(beams)
    assert cache.free_pages() == (20, 50) and not cache._packed_of


def test_a_page_packed_by_one_serves_the_others_that_share_it(pkg):
    cache = make(pkg, H=1, window=64, pages=8, plain=20)
    (a,) = cache.add(1)
    feed(cache, [a], 128)
    (b,) = cache.fork([a])
    assert cache.free_pages()[0] == 7
    feed(cache, [a], 64, seed=1)
    assert cache.free_pages()[0] == 6
    feed(cache, [b], 64, seed=2)
    assert cache.tables(a)[0] == cache.tables(b)[0] and cache.free_pages()[0] == 6
    cache.free([a])
    feed(cache, [b], 64, seed=3)
    cache.free([b])
    assert cache.free_pages() == (8, 20) and not cache._packed_of


def test_pages_stay_plain_while_packed_ones_are_short(pkg):
    cache = make(pkg, H=1, window=0, pages=1, plain=20)
    a, b = cache.add(2)
    feed(cache, [a], 200)
    assert len(cache.tables(a)[0]) == 1 and len(cache.tables(a)[1]) == 3
    step = feed(cache, [a, b], (3, 5), seed=1, commit=False)
    q = rand((8, 2, 128), 1, BF)
    check(step.attend(q, 0), q, step)
    step.commit()
    cache.resize(pages=10, plain_pages=30)
    feed(cache, [a], 1, seed=4)
    assert len(cache.tables(a)[0]) == 3
    with pytest.raises(pkg._native.TqError, match="uncompressed pages"):
        cache.step([b], 64 * 40)
    assert cache.lengths([a, b]) == [204, 5]


def test_pools_past_four_gigabytes(pkg):
    cache = pkg.PagedV3Cache(128, 8, 4, 2, 64, n_layers=1, pages=100000, plain_pages=20000, device=DEV)
    low = cache.add(1)
    cache.place(low, [99950 * 64], [19950 * 64])
    assert cache._pool.numel() > 2 ** 32 and cache._plain.numel() * 2 > 2 ** 32
    seqs = cache.add(2)
    feed(cache, seqs, (500, 70))
    step = feed(cache, seqs, (20, 1), seed=1, commit=False)
    assert min(cache.tables(seqs[0])[0]) >= 99950 and min(cache.tables(seqs[0])[1]) >= 19950
    q = rand((21, 16, 128), 1, BF)
    check(step.attend(q, 0), q, step)
    (f,) = cache.fork([seqs[1]])
    assert all(torch.equal(x, y) for x, y in zip(contents(cache, f), contents(cache, seqs[1])))


def test_recorded_steps_replay(pkg):
    cache = make(pkg, H=2, window=20, plain=80)
    seqs = cache.add(3)
    feed(cache, seqs, (300, 20, 0))
    step = cache.step(seqs, (1, 7, 2))
    k, v, q = states(10, 2, 128, 1, BF), states(10, 2, 128, 2, BF), rand((10, 8, 128), 3, BF)
    step.append(k, v, 0)
    step.attend(q, 0, softcap=9.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.append(k, v, 0)
        out = step.attend(q, 0, softcap=9.0)
        with pytest.raises(RuntimeError, match="recorded"):
            step.attend(q, 0, sliding_window=9)
        with pytest.raises(RuntimeError, match="recorded"):
            step.commit()
    for i in range(4):
        for t, seed in ((k, 10 + i), (v, 20 + i)):
            t.copy_(states(10, 2, 128, seed, BF))
        q.copy_(rand((10, 8, 128), 30 + i, BF))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        check(got, q, step, softcap=9.0)
        assert torch.equal(step.attend(q, 0, softcap=9.0), got)


def test_other_streams(pkg):
    cache = make(pkg, H=2, window=20, plain=80)
    seqs = cache.add(2)
    feed(cache, seqs, (300, 20))
    torch.cuda.synchronize()
    side, third = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        step = feed(cache, seqs, (5, 40), seed=1, commit=False)
        q = rand((45, 8, 128), 1, BF)
        a = step.attend(q, 0)
    third.wait_stream(side)
    with torch.cuda.stream(third):
        b = step.attend(q, 0)
        q.record_stream(third)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    check(a, q, step)


def test_nothing_to_do(pkg):
    cache = make(pkg, H=2)
    seqs = cache.add(2)
    step = cache.step(seqs, 0)
    empty = torch.empty((0, 2, 128), dtype=BF, device=DEV)
    step.append(empty, empty, 0)
    assert step.attend(torch.empty((0, 8, 128), dtype=BF, device=DEV), 0).shape == (0, 8, 128)
    step.commit()
    step.commit()
    assert cache.fork([]) == [] and cache.add(0) == [] and cache.lengths(seqs) == [0, 0]
    cache.reorder([], [])
    cache.free([])
    cache.step([], []).commit()
    cache.resize()
    assert cache.free_pages() == (1, 1)


def test_refusals(pkg):
    cache = make(pkg, H=2, layers=2, plain=10)
    a, b = cache.add(2)
    native = pkg._native
    for bad in ((1.5,), (-1,), (True,), (1, 1)):
        with pytest.raises(ValueError):
            cache.step([a], bad)
    with pytest.raises(ValueError):
        cache.step([a, a], 1)
    with pytest.raises(ValueError):
        cache.step([99], 1)
    with pytest.raises(native.TqError):
        cache.step([a], 64 * 10 + 1)
    assert cache.lengths([a]) == [0] and cache.free_pages()[1] == 10
    step = cache.step([a], 5)
    k = states(5, 2, 128, 1, BF)
    q = rand((5, 4, 128), 1, BF)
    for bad in (k[:4], k.float(), k[:, :1], k.transpose(0, 1)):
        with pytest.raises(ValueError):
            step.append(bad, k, 0)
        with pytest.raises(ValueError):
            step.append(k, bad, 0)
    with pytest.raises(native.TqError):
        step.append(k.cpu(), k, 0)
    for layer in (2, -1, 0.5, True):
        with pytest.raises(ValueError):
            step.append(k, k, layer)
    step.append(k, k, 0)
    with pytest.raises(RuntimeError, match="layers"):
        step.commit()
    step.append(k, k, 1)
    for bad in (q[:4], q.half(), q[:, :3], q[0], q[:, :0]):
        with pytest.raises(ValueError):
            step.attend(bad, 0)
    with pytest.raises(native.TqError):
        step.attend(q.cpu(), 0)
    for kw in ({"softcap": 0.0}, {"softcap": -1.0}, {"softcap": float("inf")}, {"softcap": float("nan")}, {"sliding_window": 0}, {"sliding_window": 1.5}, {"sliding_window": True},
               {"slopes": torch.zeros(3, device=DEV)}, {"slopes": torch.zeros(4, dtype=torch.int32, device=DEV)}):
        with pytest.raises(ValueError):
            step.attend(q, 0, **kw)
    with pytest.raises(native.TqError):
        step.attend(q, 0, slopes=torch.zeros(4))
    step.commit()
    for call in (lambda: step.attend(q, 0), lambda: step.append(k, k, 0)):
        with pytest.raises(RuntimeError, match="committed"):
            call()
    for bad in ([0], [0, 2], [0, -1], [0.5, 0], [True, False]):
        with pytest.raises(ValueError):
            cache.reorder([a, b], bad)
    with pytest.raises(ValueError):
        cache.reorder([a, b], torch.tensor([0.0, 1.0]))
    with pytest.raises(ValueError):
        cache.free([a, a])
    with pytest.raises(ValueError):
        cache.place([a], [64], [0])
    with pytest.raises(ValueError):
        cache.place([b], [63], [0])
    with pytest.raises(ValueError):
        cache.resize(plain_pages=0)
    with pytest.raises(native.TqError):
        cache.fork([a] * 20)
    assert cache.free_pages() == (64, 9) and cache.lengths([a, b]) == [5, 0]
