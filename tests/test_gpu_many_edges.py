"""GPU tests of attention of several queries and of eviction at their edges: nothing to attend to, numbers that are none, queries of very different size, several
threads, and forms that only large calls take.

Tolerances, per result vector.  Half a step of fp16 is 2^-11.  A logit is off by at most u * scale * |q| |k| with
  bfloat16          u = 2^-10 + D 2^-22: query and level are one fp16 value each
  float16, float32  u = 2^-19 + D 2^-22: two fp16 terms each (2^-22 is left of either, the product of the rests is left out)
where D 2^-22 stands for float32 sums of at most 4 D products, those of the rotation among them.  Weights of a row are off by 2 delta together, and a result by
expm1(2 delta) + u_v of the longest value vector that the query sees, with
  bfloat16, float16 u_v = 2^-9: weight, weight times norm and level are one fp16 value each, and the sum of weights may be made of the rounded ones: 4 x 2^-11
  float32           u_v = 2^-18: two fp16 terms each
and (S / 8 + 100) 2^-24 more for float32 sums over S keys, of which a wave adds up an eighth at most and the others' sums are joined to its own
(the way back out of the codec's space is in two terms throughout), plus half a step of the result's type."""
import threading

import pytest
import torch

from test_gpu_many import BF, F16, F32, HALF, contents, dequantised, make_cache, rand, random_tree, reference
from test_gpu_parity import DEV, outlier_kv

pytestmark = pytest.mark.gpu
LOGIT = {BF: 2.0 ** -10, F16: 2.0 ** -19, F32: 2.0 ** -19}
VALUE = {BF: 2.0 ** -9, F16: 2.0 ** -9, F32: 2.0 ** -18}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a HIP device; there is no CPU fallback to test")


def near(out, q, k, v, seen, scale=None):
    """Every result vector within the bound of the module's docstring; the weights [B,H,G,T,S]."""
    ref, p, seen, scale = reference(q, k, v, seen, scale)
    B, Hq, T, D = q.shape
    H, S = k.shape[1], k.shape[2]
    nothing = torch.zeros((), dtype=torch.float64, device=DEV)
    reach = q.double().norm(dim=-1).reshape(B, H, -1, T, 1) * k.norm(dim=-1).view(B, H, 1, 1, S)
    delta = ((LOGIT[q.dtype] + D * 2.0 ** -22) * abs(scale) * torch.where(seen, reach, nothing).amax(-1)).reshape(B, Hq, T)
    longest = torch.where(seen, v.norm(dim=-1).view(B, H, 1, 1, S), nothing).amax(-1).reshape(B, Hq, T)
    error = (out.double() - ref).norm(dim=-1)
    bound = HALF[q.dtype] * ref.norm(dim=-1) + (torch.expm1(2 * delta) + VALUE[q.dtype] + (S / 8 + 100) * 2.0 ** -24) * longest + 1e-30
    worst = (error / bound).max().item()
    assert bool(torch.isfinite(out).all()) and worst <= 1.0, f"error {worst:.3f} of the bound"
    return p


def states(pkg, B, H, S, w, D, dtype, kb=4, vb=2, seed=0):
    """A codec, dictionaries of S tokens of which the last w are uncompressed, and what they hold in float64."""
    codec = pkg.TurboQuantV3(D, key_bits=kb, value_bits=vb, residual_window=w, layer_idx=8, device=DEV)
    ck, cv = codec.compress_kv(outlier_kv((B, H, S, D), seed=seed, dtype=dtype).to(DEV), outlier_kv((B, H, S, D), seed=seed + 1, dtype=dtype).to(DEV))
    held = [torch.cat((dequantised(comp, (c["compressed"]["idx_bytes"], c["compressed"]["vec_norms"])), c["fp16"].double()), 2)
            for c, comp in ((ck, codec.key_compressor), (cv, codec.val_compressor))]
    return codec, ck, cv, held[0], held[1]


@pytest.fixture
def new_memory_is_nan():
    """Floating-point memory that nobody has written holds NaN."""
    torch.use_deterministic_algorithms(True)
    yield
    torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("D,dtype", [(128, BF), (64, F16), (33, F32), (256, F32)])
def test_nothing_to_attend_to(pkg, new_memory_is_nan, D, dtype):
    """Zeros, wherever the last token has left: a cache without a window after evict(0), dictionaries of nothing, a draft of no token over nothing."""
    cache = make_cache(pkg, 2, 2, 40, 0, D, dtype, track_weights=True)
    q, one = rand((2, 4, 7, D), 1, dtype), rand((2, 4, 1, D), 2, dtype)
    cache.attend(one, 1)
    cache.evict(0, 1)
    out = cache.attend(one, 1)
    assert out.shape == one.shape and torch.equal(out, torch.zeros_like(one)) and cache.attention_weights(1).shape == (2, 2, 0)
    k, v = rand((2, 2, 7, D), 3, dtype), rand((2, 2, 7, D), 4, dtype)
    alone = make_cache(pkg, 2, 2, 0, 0, D, dtype)
    assert torch.equal(cache.attend_tree(q, k, v, 1), alone.attend_tree(q, k, v, 1))
    for c in (cache, alone):
        assert torch.equal(c.attend_tree(q, k[:, :, :0], v[:, :, :0], 1, torch.zeros(7, 0, dtype=torch.bool, device=DEV)), torch.zeros_like(q))
    codec, ck, cv, _, _ = states(pkg, 2, 2, 50, 0, D, dtype)
    nk, nv, left, kept = codec.evict_kv(ck, cv, torch.ones(2, 2, 50, device=DEV), 0)
    assert left.shape == kept.shape == (2, 2, 0)
    for kw in ({}, {"lengths": torch.tensor([3, 0], device=DEV)}, {"mask": torch.zeros(2, 0, dtype=torch.bool, device=DEV)}, {"weights": left}):
        assert torch.equal(codec.attend_kv(q, nk, nv, **kw), torch.zeros_like(q))
    cache.append(k[:, :, :1], v[:, :, :1], 1)            # and on from there
    K, V = contents(cache)
    near(cache.attend(one, 1), one, K, V, torch.ones(1, dtype=torch.bool, device=DEV))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,n", [(128, 60), (128, 3000), (64, 100), (80, 100), (96, 2000), (256, 60), (33, 60)])
def test_infinite_values_at_any_coordinate(pkg, D, n, dtype):
    """One infinite element of a drafted value is found wherever it lies; the query that sees it has it there, and only there."""
    B, H, T = 1, 1, 4
    cache = make_cache(pkg, B, H, n, 5, D, dtype)
    q, k, v = rand((B, H, T, D), 1, dtype), rand((B, H, T, D), 2, dtype), rand((B, H, T, D), 3, dtype)
    tree = torch.eye(T, dtype=torch.bool, device=DEV)
    want = cache.attend_tree(q, k, v, 1, tree)
    for d in range(0, D, 5):
        bad = v.clone()
        bad[0, 0, d % T, d] = float("inf") if d % 2 else float("nan")
        out = cache.attend_tree(q, k, bad, 1, tree)
        assert not bool(torch.isfinite(out[0, 0, d % T, d]))
        out[0, 0, d % T, d] = want[0, 0, d % T, d]
        assert torch.equal(out, want), d


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,n", [(128, 40), (128, 1000), (64, 40), (80, 300), (256, 50), (33, 40)])
def test_logits_far_below_zero(pkg, D, n, dtype):
    """A query that points away from every key has the key with the largest logit all the same, below -1e30 as everywhere."""
    codec = pkg.TurboQuantV3(D, key_bits=4, value_bits=4, residual_window=0, layer_idx=8, device=DEV)
    along = rand((1, 1, 1, D), 1, F32)
    ks, vs = (along * torch.arange(2, n + 2, device=DEV).view(1, 1, n, 1)).to(dtype), rand((1, 1, n, D), 2, dtype)
    ck, cv = codec.compress_kv(ks.flip(2).contiguous(), vs)            # the shortest key is the last; the next is half as long again
    V = dequantised(codec.val_compressor, (cv["compressed"]["idx_bytes"], cv["compressed"]["vec_norms"]))[:, :, -1:]
    for size in (1.0, 1e25, 1e31, 1e33):
        q = (-size * along).to(dtype)
        got = codec.attend_kv(q, ck, cv)
        # (its weight is one but for exp(-|along|^2 / sqrt(D)) at the least, logits being as far apart as that)
        slack = HALF[dtype] + VALUE[dtype] + (n / 8 + 100) * 2.0 ** -24 + (0.0 if size > 1 else 4 * n * torch.exp(-0.9 * along.double().norm() ** 2 / D ** 0.5).item())
        assert (got.double() - V).norm() <= slack * vs.double().norm(dim=-1).amax(), size


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("D,n,w", [(128, 60, 5), (128, 3000, 40), (64, 900, 0), (96, 500, 7), (256, 300, 3), (33, 200, 20)])
def test_sums_of_large_logits(pkg, D, n, w, T, dtype):
    """Logits of which the last bit is more than an exponent can be: no query gives a key more than its weight can be, and none gives less than nothing."""
    codec, ck, cv, K, V = states(pkg, 2, 2, n + w, w, D, dtype)
    for size in (1e3, 3e4) if dtype is F16 else (1e3, 1e6, 1e12, 1e20):
        q, sums = (size * rand((2, 4, T, D), 1, F32)).clamp(-6e4, 6e4).to(dtype) if dtype is F16 else (size * rand((2, 4, T, D), 1, F32)).to(dtype), torch.zeros(2, 2, n + w, device=DEV)
        out = codec.attend_kv(q, ck, cv, weights=sums, scale=1e3 if dtype is F16 else None)
        assert bool(torch.isfinite(out).all()) and bool((sums >= 0).all()) and bool((sums <= 1.01 * 2 * T).all()), size


# (head dimension, tokens packed, window): one split of a row, several with the launch that joins them, and the kernel for all dimensions
FORMS = [(128, 60, 5), (128, 3000, 0), (64, 1500, 40), (80, 700, 0), (96, 60, 20), (256, 900, 3), (33, 50, 0), (33, 700, 9)]

@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,n,w", FORMS)
def test_queries_that_are_no_numbers(pkg, D, n, w, dtype, bad):
    """NaN for the query vector concerned, however its tokens are split; the others as ever. What keys receive is NaN in its rows and nowhere else."""
    B, H, G, T = 2, 2, 2, 5
    codec, ck, cv, K, V = states(pkg, B, H, n + w, w, D, dtype)
    q = rand((B, H * G, T, D), 1, dtype)
    q[1, 3, 2, 7] = bad
    seen = torch.ones(n + w, dtype=torch.bool, device=DEV)
    for track in (False, True):
        sums = torch.zeros(B, H, n + w, device=DEV)
        out = codec.attend_kv(q, ck, cv, **({"weights": sums} if track else {}))
        assert bool(torch.isnan(out[1, 3, 2]).all())
        fine, clean = out.clone(), q.clone()
        fine[1, 3, 2], clean[1, 3, 2] = 0.0, 0.0
        fine[1, 3, 2] = codec.attend_kv(clean, ck, cv)[1, 3, 2]
        near(fine, clean, K, V, seen)
        if track:
            assert bool(torch.isnan(sums[1, 1]).all()) and bool(torch.isfinite(sums[0]).all()) and bool(torch.isfinite(sums[1, 0]).all())
    hidden = torch.zeros(B, n + w, dtype=torch.bool, device=DEV)
    assert not bool(codec.attend_kv(q, ck, cv, mask=hidden)[1, 3, 2].any())          # (it sees nothing)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,n,w", FORMS)
def test_keys_that_are_no_numbers(pkg, D, n, w, dtype):
    """A NaN key among those that a query sees is a NaN result, wherever it lies and whatever else there is; an infinite value is no finite result, however small its weight."""
    B, H, G, T = 1, 2, 2, 4
    cache = make_cache(pkg, B, H, n, w, D, dtype)
    q, k, v = rand((B, H * G, T, D), 1, dtype), rand((B, H, T, D), 2, dtype), rand((B, H, T, D), 3, dtype)
    tree = torch.eye(T, dtype=torch.bool, device=DEV)
    want, lone = cache.attend_tree(q, k, v, 1, tree), make_cache(pkg, B, H, 0, w, D, dtype)
    lone_want = lone.attend_tree(q, k, v, 1, tree)
    bad_k = k.clone()
    bad_k[0, 1, 2, 3] = float("nan")                  # kv head 1: query heads 2 and 3, token 2
    for c, clean in ((cache, want), (lone, lone_want)):
        out = c.attend_tree(q, bad_k, v, 1, tree)
        assert bool(torch.isnan(out[0, 2:, 2]).all())
        keep = torch.ones(H * G, T, dtype=torch.bool, device=DEV)
        keep[2:, 2] = False
        assert torch.equal(out[0, keep], clean[0, keep])
    far_k, far_v = k.clone(), v.clone()
    far_k[0, 0, 1], far_v[0, 0, 1, 5] = -300.0 * q[0, 0, 1], float("inf")           # a weight that underflows to zero, for query head 0
    out = cache.attend_tree(q, far_k, far_v, 1, tree)
    assert not bool(torch.isfinite(out[0, 0, 1, 5])) and not bool(torch.isfinite(out[0, 1, 1, 5]))
    assert bool(torch.isfinite(out[0, 0, 1, :5]).all()) and torch.equal(out[0, 0, [0, 2, 3]], want[0, 0, [0, 2, 3]])
    codec, ck, cv, _, _ = states(pkg, B, H, n + w, w, D, dtype)
    ck["compressed"]["vec_norms"][0, 1, n // 2] = float("nan")
    sums = torch.zeros(B, H, n + w, device=DEV)
    out = codec.attend_kv(q, ck, cv, weights=sums)
    assert bool(torch.isnan(out[0, 2:]).all()) and bool(torch.isfinite(out[0, :2]).all()) and bool(torch.isnan(sums[0, 1]).all()) and bool(torch.isfinite(sums[0, 0]).all())
    assert bool(torch.isnan(codec.attend_kv(q, ck, cv)[0, 2:]).all())


@pytest.mark.parametrize("D,n,w,T,factor,dtype", [
    (128, 60, 5, 9, 1e12, BF), (128, 3000, 16, 9, 1e25, BF), (128, 3000, 16, 40, 1e25, BF), (64, 700, 0, 3, 1e9, BF), (80, 700, 8, 9, 1e25, BF), (256, 900, 0, 9, 1e15, BF),
    (33, 500, 4, 20, 1e25, BF), (128, 1000, 7, 9, 2e4, F16), (128, 60, 0, 70, 1e12, F32), (96, 900, 9, 9, 1e25, F32), (72, 300, 0, 1, 1e12, F32), (40, 90, 3, 33, 1e12, F32),
])
def test_a_query_far_larger_than_its_neighbours(pkg, D, n, w, T, factor, dtype):
    """Queries that are worked on together do not have to be of one size: what a row of padding holds has no effect on the others."""
    B, H, G = 2, 2, 3
    codec, ck, cv, K, V = states(pkg, B, H, n + w, w, D, dtype)
    q = rand((B, H * G, T, D), 1, dtype)
    if dtype is F16:
        q = q / 64
    # along the longest key of its row, which then has all of its weight
    longest = K.norm(dim=-1).argmax(-1)
    for b in range(B):
        for h in range(H):
            along = K[b, h, longest[b, h]]
            q[b, h * G + 1, T // 2] = (along / along.abs().max() * factor).to(dtype)
    seen = torch.ones(n + w, dtype=torch.bool, device=DEV)
    near(codec.attend_kv(q, ck, cv), q, K, V, seen)
    sums = torch.zeros(B, H, n + w, device=DEV)
    p = near(codec.attend_kv(q, ck, cv, weights=sums), q, K, V, seen)
    p[:, :, 1, T // 2] = 0                               # (what the large one gives a key is some number from zero to one: its logits have no last bit that counts)
    got = p.sum((2, 3))
    delta = (2.0 ** -19 + D * 2.0 ** -22) * D ** -0.5 * q.double().norm(dim=-1).reshape(B, H, G, T, 1) * K.norm(dim=-1).amax(-1).view(B, H, 1, 1, 1)
    delta[:, :, 1, T // 2] = 0
    slack = (p * torch.expm1(2 * delta)).sum((2, 3)) + got * (T * G + 8 + (n + w) / 8 + 100) * 2.0 ** -23 + 1e-30
    assert bool((sums.double() >= got - slack).all()) and bool((sums.double() <= got + slack + 1.01).all())
    touched = (sums.double() > got + slack).sum(-1)
    assert bool((touched <= (n + w) // 4).all())         # (it is one key's, or a few that lie as far in its direction)


def run_threads(work):
    """Every function of `work` in a thread of its own; the first exception is raised here."""
    errors = []

    def guarded(f):
        try:
            f()
        except BaseException as e:          # noqa: B036
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(f,)) for f in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


def test_nothing_is_handed_on_through_memory_that_others_use(pkg):
    """The launches of a call hand their sums on through memory of the call's own: the scratch that decode steps of a stream share stays as it is."""
    D, native = 128, pkg._native
    plain, tracked = make_cache(pkg, 2, 2, 3000, 16, D, BF), make_cache(pkg, 2, 2, 3000, 16, D, BF, track_weights=True)
    odd = make_cache(pkg, 1, 2, 300, 16, 33, BF)
    codec, ck, cv, _, _ = states(pkg, 2, 2, 2000, 16, D, BF)
    q, k, v, one = rand((2, 4, 6, D), 1, BF), rand((2, 2, 6, D), 2, BF), rand((2, 2, 6, D), 3, BF), rand((2, 4, 1, D), 4, BF)
    plain.attend(one, 1)
    assert native._step_scratch
    for buf in native._step_scratch.values():
        buf.fill_(12345.0)
    for _ in range(2):
        plain.attend_tree(q, k, v, 1)
        tracked.attend(one, 1)
        odd.attend_tree(q[:1, :, :, :33], k[:1, :, :, :33], v[:1, :, :, :33], 1)
        codec.attend_kv(q, ck, cv, weights=torch.zeros(2, 2, 2000, device=DEV))
    torch.cuda.synchronize()
    assert all(bool((buf == 12345.0).all()) for buf in native._step_scratch.values())


def test_decode_steps_of_several_launches_share_no_memory(pkg):
    """The same for the decode step of float32 caches, which takes three launches."""
    native = pkg._native
    one_launch, three = make_cache(pkg, 1, 2, 900, 16, 128, BF), make_cache(pkg, 1, 2, 900, 16, 128, F32)
    assert one_launch._stores[1].one_launch and not three._stores[1].one_launch
    q = rand((1, 4, 1, 128), 1, F32)
    one_launch.attend(q.to(BF), 1)
    want = three.attend(q, 1)
    assert native._step_scratch
    for buf in native._step_scratch.values():
        buf.fill_(12345.0)
    got = three.attend(q, 1)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(bool((buf == 12345.0).all()) for buf in native._step_scratch.values())
    other, other_q = make_cache(pkg, 2, 2, 700, 16, 128, F32, seed=3), rand((2, 4, 1, 128), 2, F32)
    pairs = [(three, q, want), (other, other_q, other.attend(other_q, 1)), (one_launch, q.to(BF), one_launch.attend(q.to(BF), 1))]
    got = [[] for _ in pairs]

    def steps(i):
        for _ in range(50):
            got[i].append(pairs[i][0].attend(pairs[i][1], 1))
    run_threads([lambda i=i: steps(i) for i in range(len(pairs))])
    torch.cuda.synchronize()
    for outs, (_, _, w) in zip(got, pairs):
        assert len(outs) == 50 and all(torch.equal(o, w) for o in outs)


def test_threads_on_one_stream(pkg):
    """Calls of several threads whose launches meet on one stream answer as each does alone."""
    caches = [make_cache(pkg, 1, 4, 3000 + 40 * i, 32, 128, BF, seed=i) for i in range(2)]
    odd = make_cache(pkg, 1, 4, 400, 8, 33, BF)
    sets = [(rand((1, 16, 9, 128), i, BF), rand((1, 4, 9, 128), 10 + i, BF), rand((1, 4, 9, 128), 20 + i, BF)) for i in range(2)]
    small = tuple(t[..., :33].contiguous() for t in sets[0])
    want = [c.attend_tree(*s, 1) for c, s in zip(caches, sets)]
    want_odd, one = odd.attend_tree(*small, 1), rand((1, 16, 1, 128), 30, BF)
    want_step = caches[0].attend(one, 1)
    torch.cuda.synchronize()
    got = [[] for _ in range(4)]

    def tree(i):
        for _ in range(50):
            got[i].append(caches[i].attend_tree(*sets[i], 1))

    def rest():
        for _ in range(50):
            got[2].append(odd.attend_tree(*small, 1))

    def steps():
        for _ in range(50):
            got[3].append(caches[0].attend(one, 1))
    run_threads([lambda: tree(0), lambda: tree(1), rest, steps])
    torch.cuda.synchronize()
    for outs, w in zip(got, (*want, want_odd, want_step)):
        assert len(outs) == 50 and all(torch.equal(o, w) for o in outs)


@pytest.mark.parametrize("S,w", [(200, 16), (200, 0)])
def test_flat_dictionaries(pkg, S, w):
    """Codes of all vectors one after the other, as decompress_kv takes them."""
    codec, ck, cv, _, _ = states(pkg, 2, 2, S, w, 128, BF)
    flat = [dict(c, compressed=dict(c["compressed"], idx_bytes=c["compressed"]["idx_bytes"].reshape(-1, c["compressed"]["idx_bytes"].shape[-1]),
                                    vec_norms=c["compressed"]["vec_norms"].reshape(-1))) for c in (ck, cv)]
    q = rand((2, 4, 3, 128), 1, BF)
    for a, b in zip(codec.decompress_kv(*flat), codec.decompress_kv(ck, cv)):
        assert torch.equal(a, b)
    assert torch.equal(codec.attend_kv(q, *flat), codec.attend_kv(q, ck, cv))
    sums = torch.rand(2, 2, S, device=DEV)
    assert torch.equal(codec.evict_kv(*flat, sums, 50)[3], codec.evict_kv(ck, cv, sums, 50)[3])


def test_drafts_whose_values_are_more_than_their_keys(pkg):
    """Refused, the first time and every other."""
    cache = make_cache(pkg, 2, 2, 300, 16, 128, BF)
    q, k, v = rand((2, 4, 6, 128), 1, BF), rand((2, 2, 6, 128), 2, BF), rand((2, 2, 9, 128), 3, BF)
    for _ in range(3):
        with pytest.raises(ValueError, match="do not go with"):
            cache.attend_tree(q, k, v, 1)
        cache.attend_tree(q, k, v[:, :, :6], 1)


@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_lengths_of_any_whole_type(pkg, kind):
    """More keys than the type can count, and lengths below zero where it has them."""
    codec, ck, cv, K, V = states(pkg, 3, 2, 40000, 0, 64, BF, 2, 2)
    q = rand((3, 2, 1, 64), 1, BF)
    lengths = torch.tensor([100, 0, 7], dtype=kind, device=DEV)
    if kind is not torch.uint8:
        lengths[1] = -5
    out = codec.attend_kv(q, ck, cv, lengths=lengths)
    near(out, q, K, V, (torch.arange(40000, device=DEV) < lengths.view(-1, 1)).view(3, 1, 1, 1, -1))
    assert not bool(out[1].any())


def test_a_draft_over_nothing_settles_nothing(pkg):
    """A cache that has seen a draft, and nothing else, takes states of any other head dimension."""
    cache, fresh = pkg.V3Cache(n_layers=4), pkg.V3Cache(n_layers=4)
    q, k = rand((1, 4, 3, 64), 1, BF), rand((1, 2, 3, 64), 2, BF)
    cache.attend_tree(q, k, k, 1)
    states_, one = outlier_kv((1, 2, 200, 128), seed=3, dtype=BF).to(DEV), rand((1, 4, 1, 128), 4, BF)
    for c in (cache, fresh):
        c.append(states_, states_, 1)
    assert torch.equal(cache.attend(one, 1), fresh.attend(one, 1)) and cache._stores[1].comp.head_dim == 128
    with pytest.raises(ValueError):                     # (what is cached has settled it)
        cache.append(k, k, 1)
    assert torch.equal(cache.attend(one, 1), fresh.attend(one, 1))


@pytest.mark.parametrize("B,H,G,S,w,T,D,dtype", [
    (8, 8, 4, 600, 40, 40, 128, BF), (8, 8, 4, 420, 0, 40, 64, BF), (8, 8, 4, 500, 300, 40, 96, BF),      # two tiles of queries a block, a row in one split
    (16, 8, 4, 3000, 16, 8, 64, BF), (16, 8, 4, 3000, 0, 8, 128, F16), (16, 9, 2, 3100, 9, 16, 80, F32),  # 128 tiles and more, rows in several splits
    (1, 2, 4, 70001, 16, 2, 64, BF), (1, 2, 4, 70001, 0, 2, 128, BF), (1, 1, 3, 50000, 5, 3, 96, F16), (1, 2, 2, 40000, 0, 5, 33, BF),      # 30 to 64 splits
])
def test_forms_of_large_calls(pkg, B, H, G, S, w, T, D, dtype):
    codec, ck, cv, K, V = states(pkg, B, H, S, w, D, dtype)
    q = rand((B, H * G, T, D), 1, dtype)
    lengths = torch.full((B,), S, dtype=torch.int32, device=DEV)
    lengths[::3] = S // 3
    seen = (torch.arange(S, device=DEV) < lengths.view(-1, 1)).view(B, 1, 1, 1, S)
    near(codec.attend_kv(q, ck, cv, lengths=lengths), q, K, V, seen)


@pytest.mark.parametrize("G,T", [(4, 1), (4, 12)])
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, F16), (96, F32)])
def test_sums_over_long_rows(pkg, D, dtype, G, T):
    B, H, S, w = 2, 2, 20011, 30
    codec, ck, cv, K, V = states(pkg, B, H, S, w, D, dtype)
    q, sums = rand((B, H * G, T, D), 1, dtype), torch.zeros(B, H, S, device=DEV)
    lengths = torch.tensor([S, 9000], dtype=torch.int32, device=DEV)
    seen = (torch.arange(S, device=DEV) < lengths.view(-1, 1)).view(B, 1, 1, 1, S)
    p = near(codec.attend_kv(q, ck, cv, lengths=lengths, weights=sums), q, K, V, seen)
    delta = (2.0 ** -19 + D * 2.0 ** -22) * D ** -0.5 * q.double().norm(dim=-1).reshape(B, H, G, T, 1) * K.norm(dim=-1).amax(-1).view(B, H, 1, 1, 1)
    got = p.sum((2, 3))
    assert bool(((sums.double() - got).abs() <= (p * torch.expm1(2 * delta)).sum((2, 3)) + got * (T * G + 8 + S / 8 + 100) * 2.0 ** -23 + 1e-30).all())
    assert not bool(sums[1, :, 9000:].any())
