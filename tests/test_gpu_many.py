"""GPU tests of attention for several query tokens from the packed form (V3Cache.attend_tree, TurboQuantV3.attend_kv), of the attention sums
a cache keeps, and of eviction by them, against the formulas in float64.

Tolerances.  With u = 2^-11 (16-bit caches in bfloat16: queries and levels enter the products as one fp16 value each, half a step 2^-12 relative) or
u = 2^-20 (two fp16 terms each, 22 bits, and what is left out) and D 2^-24 for a float32 sum of D products, a logit is off by at most
delta = (u + D 2^-24) * scale * sum_j |q'_j k'_j|, the weights of a row together by 2 delta, and a result by 2 delta + u_v of the longest value vector
that the row sees (rotations keep lengths; u_v = 2^-10: weight, level and norm, an fp16 rounding of 2^-12 each and as much for the sums of a few thousand tokens; 2^-18 in
two terms), plus half a step of its type."""
import copy
import pickle

import pytest
import torch

from test_gpu_parity import DEV, outlier_kv

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a HIP device; there is no CPU fallback to test")


def levels_of(comp, packed):
    """Rotated vectors norm * level[code], float64 [B,H,n,D], from the bytes."""
    idx, nrm = packed
    ipb, bits, D = 8 // comp.bits, comp.bits, comp.head_dim
    codes = torch.stack([(idx.long() >> (bits * (ipb - 1 - i))) & ((1 << bits) - 1) for i in range(ipb)], -1).flatten(-2)[..., :D]
    return comp.centroids.to(DEV).double()[codes] * nrm.double().unsqueeze(-1)


def dequantised(comp, packed):
    return levels_of(comp, packed) @ comp.Pi.to(DEV).double()


def reference(q, k, v, seen, scale=None):
    """float64 attention [B,Hq,T,D], what each key receives [B,H,S], and the bound on a result's error in units of (delta's u, u_v, half)."""
    B, Hq, T, D = q.shape
    H, S = k.shape[1], k.shape[2]
    G = Hq // H
    scale = D ** -0.5 if scale is None else scale
    q64 = q.double().reshape(B, H, G * T, D)
    logits = (q64 @ k.transpose(-2, -1)).reshape(B, H, G, T, S) * scale
    seen = torch.broadcast_to(seen, logits.shape)
    logits = torch.where(seen, logits, torch.full_like(logits, float("-inf")))
    top = logits.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(logits - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(logits))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    out = (p.reshape(B, H, G * T, S) @ torch.nan_to_num(v)).reshape(B, Hq, T, D)
    return out, p, seen, scale


def check(out, q, k, v, seen, kc=None, exact_terms=None, scale=None, k_rot=None):
    """Every result vector within the bound of the module's docstring."""
    ref, p, seen, scale = reference(q, k, v, seen, scale)
    B, Hq, T, D = q.shape
    H, S = k.shape[1], k.shape[2]
    narrow = q.dtype == torch.bfloat16 if exact_terms is None else not exact_terms
    u, u_v = (2.0 ** -11, 2.0 ** -10) if narrow else (2.0 ** -20, 2.0 ** -18)
    # sum_j |q'_j k'_j| <= |q| |k|
    reach = q.double().norm(dim=-1).reshape(B, H, -1, T, 1) * torch.nan_to_num(k).norm(dim=-1).view(B, H, 1, 1, S)
    delta = ((u + D * 2.0 ** -24) * abs(scale) * torch.where(seen, reach, torch.zeros_like(reach)).amax(-1)).reshape(B, Hq, T)
    longest = torch.where(seen, torch.nan_to_num(v).norm(dim=-1).view(B, H, 1, 1, S), torch.zeros_like(reach)).amax(-1).reshape(B, Hq, T)
    err = (out.double() - ref).norm(dim=-1)
    bound = HALF[q.dtype] * ref.norm(dim=-1) + (torch.expm1(2 * delta) + u_v) * longest + 1e-30
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert bool(torch.isfinite(out).all()) and worst <= 1.0, f"error {worst:.3f} of the bound"
    # and not only within the worst case: the whole tensor as near as its type has it
    if err.numel() and ref.norm() > 0:
        rel = ((out.double() - ref).norm() / ref.norm()).item()
        assert rel <= {torch.bfloat16: 5e-3, torch.float16: 1e-3, torch.float32: 1e-5}[q.dtype], rel
    return ref, p


def make_cache(pkg, B, H, n, w, D, dtype, kb=4, vb=2, seed=0, **kw):
    cache = pkg.V3Cache(key_bits=kb, value_bits=vb, residual_window=w, n_layers=4, **kw)
    k, v = outlier_kv((B, H, n + w, D), seed=seed, dtype=dtype).to(DEV), outlier_kv((B, H, n + w, D), seed=seed + 1, dtype=dtype).to(DEV)
    if n + w:
        cache.append(k, v, 1)
    return cache


def contents(cache, layer=1):
    """Everything a layer holds, float64."""
    st = cache._stores[layer]
    n = st.n_compressed
    parts = []
    for comp, idx, nrm, win in ((st.comp.key_compressor, st.k_idx, st.k_nrm, st.window()[0]), (st.comp.val_compressor, st.v_idx, st.v_nrm, st.window()[1])):
        old = dequantised(comp, (idx[:, :, :n], nrm[:, :, :n])) if n else win.double()[:, :, :0]
        parts.append(torch.cat((old, win.double()), 2))
    return parts


def rand(shape, seed, dtype):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def random_tree(T, seed, batch=None):
    g = torch.Generator()
    g.manual_seed(seed)
    out = torch.zeros((batch or 1, T, T), dtype=torch.bool)
    for b in range(batch or 1):
        for i in range(T):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if parent >= 0:
                out[b, i] = out[b, parent]
            out[b, i, i] = True
    return (out if batch else out[0]).to(DEV)


BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("B,H,G,n,w,T,D,dtype,kb,vb", [
    (1, 1, 1, 1, 0, 1, 128, BF, 4, 2),            # one packed token, one draft
    (1, 2, 4, 300, 128, 8, 128, BF, 4, 2),
    (2, 2, 4, 1000, 17, 13, 128, F16, 6, 4),
    (1, 8, 4, 4097, 128, 16, 128, BF, 4, 2),
    (1, 1, 7, 2049, 5, 64, 128, BF, 3, 2),        # 448 query vectors
    (3, 2, 1, 33, 16, 33, 64, F16, 4, 4),
    (2, 3, 2, 130, 64, 5, 80, F32, 4, 4),
    (1, 2, 8, 777, 128, 9, 96, BF, 4, 2),
    (2, 1, 3, 515, 31, 7, 256, BF, 8, 8),
    (1, 2, 2, 100, 8, 40, 256, F32, 2, 8),
    (1, 2, 2, 95, 8, 3, 33, F16, 4, 2),           # a dimension that fills no byte evenly
    (1, 1, 2, 64, 32, 6, 8, F32, 1, 1),
    (1, 2, 16, 640, 0, 2, 64, BF, 8, 4),
    (2, 2, 2, 333, 128, 11, 128, F32, 4, 2),
    (1, 2, 4, 700, 128, 21, 128, BF, 8, 1),
    (1, 2, 4, 700, 128, 21, 64, BF, 2, 6),
    (1, 1, 4, 0, 20, 4, 128, BF, 4, 2),           # nothing packed yet
    (1, 2, 2, 300, 20, 9, 72, F16, 4, 4),
    (2, 1, 4, 200, 8, 40, 96, F32, 8, 2),
    (1, 2, 3, 150, 16, 33, 88, BF, 4, 4),
    (1, 1, 4, 1000, 64, 64, 96, BF, 4, 2),
    (1, 2, 5, 600, 40, 17, 64, F32, 2, 2),
    (1, 2, 4, 32, 0, 70, 80, BF, 2, 2),
    (1, 1, 2, 517, 200, 11, 128, F32, 8, 8),
    (1, 1, 2, 517, 200, 11, 72, BF, 2, 2),        # 18 bytes a vector
])
def test_tree_against_float64(pkg, B, H, G, n, w, T, D, dtype, kb, vb):
    cache = make_cache(pkg, B, H, n, w, D, dtype, kb, vb, seed=n + T)
    q = rand((B, H * G, T, D), 5, dtype)
    k, v = outlier_kv((B, H, T, D), seed=21, dtype=dtype).to(DEV), outlier_kv((B, H, T, D), seed=22, dtype=dtype).to(DEV)
    K, V = contents(cache)
    before = [t.clone() for t in cache._stores[1].window()]
    for batch in (None, B):
        tree = random_tree(T, T, batch)
        out = cache.attend_tree(q, k, v, 1, tree)
        assert out.dtype == dtype and out.shape == q.shape and out.is_contiguous()
        seen = torch.cat((torch.ones(T, K.shape[2], dtype=torch.bool, device=DEV).expand(tree.shape[:-2] + (T, K.shape[2])), tree), -1)
        seen = seen if batch is None else seen.view(B, 1, 1, T, -1)
        check(out, q, torch.cat((K, k.double()), 2), torch.cat((V, v.double()), 2), seen)
        assert torch.equal(out, cache.attend_tree(q, k, v, 1, tree))
    chain = torch.ones(T, T, dtype=torch.bool, device=DEV).tril()
    assert torch.equal(cache.attend_tree(q, k, v, 1), cache.attend_tree(q, k, v, 1, chain))
    assert cache.get_seq_length(1) == n + w and all(torch.equal(a, b) for a, b in zip(before, cache._stores[1].window()))


@pytest.mark.parametrize("B,H,G,S,w,T,D,dtype,kb,vb", [
    (1, 1, 1, 1, 0, 1, 128, BF, 4, 2),
    (4, 4, 1, 1500, 0, 1, 64, F16, 6, 4),
    (3, 2, 4, 513, 128, 77, 128, BF, 4, 4),
    (2, 2, 4, 2000, 0, 100, 128, F16, 4, 4),
    (2, 8, 1, 203, 0, 77, 80, F32, 4, 4),
    (2, 2, 2, 128, 128, 3, 128, BF, 4, 2),         # all of it window
    (5, 1, 3, 97, 32, 31, 96, F16, 3, 2),
    (2, 1, 2, 300, 10, 65, 256, BF, 4, 8),
    (2, 2, 9, 260, 0, 15, 64, BF, 2, 2),
])
@pytest.mark.parametrize("how", ["lengths", "mask", "both", "none"])
def test_cross_against_float64(pkg, B, H, G, S, w, T, D, dtype, kb, vb, how):
    codec = pkg.TurboQuantV3(D, key_bits=kb, value_bits=vb, residual_window=w, layer_idx=8, device=DEV)
    ks, vs = outlier_kv((B, H, S, D), seed=S, dtype=dtype).to(DEV), outlier_kv((B, H, S, D), seed=S + 1, dtype=dtype).to(DEV)
    ck, cv = codec.compress_kv(ks, vs)
    q = rand((B, H * G, T, D), 6, dtype)
    parts = []
    for c, comp in ((ck, codec.key_compressor), (cv, codec.val_compressor)):
        old = [] if c["compressed"] is None else [dequantised(comp, (c["compressed"]["idx_bytes"], c["compressed"]["vec_norms"]))]
        parts.append(torch.cat(old + [c["fp16"].double()], 2))
    K, V = parts
    g = torch.Generator()
    g.manual_seed(S)
    lengths = torch.randint(0, S + 1, (B,), generator=g).to(torch.int32)
    lengths[-1] = S + 3                     # more than there are
    if B > 1:
        lengths[0] = 0                      # a sequence without a key
    mask = torch.rand(B, S, generator=g) > 0.3
    if B > 2:
        mask[1] = False
    lengths, mask = lengths.to(DEV), mask.to(DEV)
    seen = torch.ones(B, S, dtype=torch.bool, device=DEV)
    kw = {}
    if how in ("lengths", "both"):
        kw["lengths"] = lengths
        seen &= torch.arange(S, device=DEV) < lengths.view(-1, 1)
    if how in ("mask", "both"):
        kw["mask"] = mask
        seen &= mask
    prior = torch.rand(B, H, S, generator=g).to(DEV)
    sums = prior.clone()
    out = codec.attend_kv(q, ck, cv, **kw)
    ref, p = check(out, q, K, V, seen.view(B, 1, 1, 1, S))
    if how != "none":
        empty = ~seen.any(-1)
        assert not bool(out[empty].any())
    again = codec.attend_kv(q, ck, cv, weights=sums, **kw)
    check(again, q, K, V, seen.view(B, 1, 1, 1, S))
    # what keys receive comes from the two-term products whatever the type
    reach = (2.0 ** -20 + D * 2.0 ** -24) * D ** -0.5 * (q.double().norm(dim=-1).reshape(B, H, -1).amax(-1) * K.norm(dim=-1).amax(-1)).unsqueeze(-1)
    got = p.sum((2, 3))
    assert bool(((sums.double() - prior.double() - got).abs() <= got * torch.expm1(2 * reach) + got * (T * G + 8) * 2.0 ** -24 + (prior + got) * 2.0 ** -23).all())
    assert torch.equal(sums[~seen.unsqueeze(1).expand(B, H, S)], prior[~seen.unsqueeze(1).expand(B, H, S)])


def test_queries_of_any_layout_and_type(pkg):
    """Strided queries and drafts, heads and tokens swapped, vectors off the 16-byte grid, drafts of another type."""
    cache = make_cache(pkg, 2, 2, 200, 32, 128, BF)
    q = rand((2, 6, 8, 128), 1, BF)
    k, v = rand((2, 6, 2, 128), 2, BF), rand((2, 6, 2, 128), 3, BF)
    want = cache.attend_tree(q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), 1)
    assert torch.equal(cache.attend_tree(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 1), want)
    wide = torch.zeros(2, 8, 6, 131, dtype=BF, device=DEV)
    wide[..., 3:] = q.transpose(1, 2)
    assert torch.equal(cache.attend_tree(wide[..., 3:], k.transpose(1, 2), v.transpose(1, 2), 1), want)
    turned = q.transpose(1, 2).transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(cache.attend_tree(turned, k.transpose(1, 2), v.transpose(1, 2), 1), want)
    one = rand((2, 2, 1, 128), 4, BF)
    assert torch.equal(cache.attend_tree(q.transpose(1, 2)[:, :, :1].expand(2, 8, 3, 128), one.expand(2, 2, 3, 128), one.expand(2, 2, 3, 128), 1)[:, :, 0],
                       cache.attend_tree(q.transpose(1, 2)[:, :, :1], one, one, 1)[:, :, 0])
    half = cache.attend_tree(q.transpose(1, 2), k.transpose(1, 2).float(), v.transpose(1, 2).half(), 1)
    assert half.dtype == BF and (half.float() - want.float()).norm() <= 2.0 ** -7 * want.float().norm()


@pytest.mark.parametrize("D,dtype", [(128, BF), (128, F16), (64, BF), (80, F32), (256, BF)])
def test_infinities_and_nan_that_nobody_sees(pkg, D, dtype):
    """Keys and values a query does not see have no effect on it, whatever they hold."""
    B, H, G, T, n, w = 2, 2, 2, 6, 70, 16
    cache = make_cache(pkg, B, H, n, w, D, dtype)
    q, k, v = rand((B, H * G, T, D), 1, dtype), rand((B, H, T, D), 2, dtype), rand((B, H, T, D), 3, dtype)
    tree = torch.eye(T, dtype=torch.bool, device=DEV)
    want = cache.attend_tree(q, k, v, 1, tree)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, :, 2], bad_v[:, :, 2, ::3], bad_v[:, :, 4, 1] = float("nan"), float("inf"), float("nan")
    got = cache.attend_tree(q, bad_k, bad_v, 1, tree)
    others = [0, 1, 3, 5]
    assert torch.equal(got[:, :, others], want[:, :, others])
    assert bool(torch.isnan(got[:, :, 2]).all()) and bool(torch.isnan(got[:, :, 4, 1]).all())
    assert torch.equal(got[:, :, 4, 2:], want[:, :, 4, 2:])
    codec = pkg.TurboQuantV3(D, residual_window=w, layer_idx=8, device=DEV)
    ks, vs = rand((B, H, 90, D), 4, dtype), rand((B, H, 90, D), 5, dtype)
    hidden = torch.zeros(B, 90, dtype=torch.bool, device=DEV)
    hidden[:, [0, 33, 89]] = True
    clean = codec.compress_kv(ks, vs)
    # (in the packed form, where such a vector has such a norm: compress works on 64-wide vectors in pairs, and an infinite one takes its neighbour along)
    dirty = copy.deepcopy(clean)
    dirty[0]["compressed"]["vec_norms"][:, :, 0], dirty[1]["compressed"]["vec_norms"][:, :, 33] = float("inf"), float("nan")
    dirty[0]["fp16"][:, :, -1], dirty[1]["fp16"][:, :, -1] = float("nan"), float("inf")
    assert torch.equal(codec.attend_kv(q, *dirty, mask=~hidden), codec.attend_kv(q, *clean, mask=~hidden))
    lengths = torch.tensor([33, 20], device=DEV)
    keep = torch.ones(B, 90, dtype=torch.bool, device=DEV)
    keep[:, 0] = False                 # (the rest lies behind the lengths)
    assert torch.equal(codec.attend_kv(q, *dirty, mask=keep, lengths=lengths), codec.attend_kv(q, *clean, mask=keep, lengths=lengths))


@pytest.mark.parametrize("factor", [1e-30, 1e-6, 3e4, 1e20])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_queries_of_any_size(pkg, factor, dtype):
    """Rotated queries leave the range of fp16 in both directions; a scale takes the logits back where they belong."""
    cache = make_cache(pkg, 1, 2, 300, 16, 128, dtype)
    q, k, v = rand((1, 4, 3, 128), 1, F32), rand((1, 2, 3, 128), 2, dtype), rand((1, 2, 3, 128), 3, dtype)
    big = (q * factor).to(dtype)
    K, V = contents(cache)
    seen = torch.cat((torch.ones(3, K.shape[2], dtype=torch.bool, device=DEV), torch.ones(3, 3, dtype=torch.bool, device=DEV).tril()), 1)
    check(cache.attend_tree(big, k, v, 1, scale=128 ** -0.5 / factor), big, torch.cat((K, k.double()), 2), torch.cat((V, v.double()), 2), seen, scale=128 ** -0.5 / factor)


def test_values_of_any_size(pkg):
    """Value norms over the whole range of fp16, small ones first: the sums' units go with the largest so far."""
    codec = pkg.TurboQuantV3(128, key_bits=4, value_bits=4, residual_window=0, layer_idx=8, device=DEV)
    ks, vs = rand((1, 2, 700, 128), 1, F32), rand((1, 2, 700, 128), 2, F32)
    vs = vs * torch.logspace(-5, 3, 700, device=DEV).view(1, 1, -1, 1)
    for flip in (False, True):
        x = vs.flip(2).contiguous() if flip else vs
        ck, cv = codec.compress_kv(ks, x)
        q = rand((1, 4, 5, 128), 3, F32)
        K = dequantised(codec.key_compressor, (ck["compressed"]["idx_bytes"], ck["compressed"]["vec_norms"]))
        V = dequantised(codec.val_compressor, (cv["compressed"]["idx_bytes"], cv["compressed"]["vec_norms"]))
        for lengths in (None, torch.tensor([40], device=DEV)):
            seen = torch.ones(700, dtype=torch.bool, device=DEV) if lengths is None else torch.arange(700, device=DEV) < 40
            check(codec.attend_kv(q, ck, cv, lengths=lengths), q, K, V, seen)


@pytest.mark.parametrize("D,kb,dtype", [(64, 2, BF), (64, 4, F16), (64, 8, BF), (128, 2, F16), (128, 4, BF), (128, 6, BF), (256, 2, BF), (256, 4, F16), (256, 8, BF), (128, 4, F32), (96, 4, BF)])
@pytest.mark.parametrize("G,T", [(1, 1), (3, 1), (4, 4), (5, 3), (17, 1), (4, 9)])
def test_sums_of_few_and_many_queries(pkg, G, T, D, kb, dtype):
    """Up to 16 query vectors a row have a launch of their own; tokens that are not whole runs, a masked sequence, a window.  The bound of test_cross_against_float64."""
    B, H, S, w = 2, 3, 611, 37
    codec = pkg.TurboQuantV3(D, key_bits=kb, value_bits=2, residual_window=w, layer_idx=8, device=DEV)
    ck, cv = codec.compress_kv(outlier_kv((B, H, S, D), seed=G, dtype=dtype).to(DEV), outlier_kv((B, H, S, D), seed=T, dtype=dtype).to(DEV))
    K, V = (torch.cat((dequantised(comp, (c["compressed"]["idx_bytes"], c["compressed"]["vec_norms"])), c["fp16"].double()), 2)
            for c, comp in ((ck, codec.key_compressor), (cv, codec.val_compressor)))
    q = rand((B, H * G, T, D), D, dtype)
    seen = torch.ones(B, S, dtype=torch.bool, device=DEV)
    seen[1, ::3], seen[1, 590:] = False, False
    prior = torch.rand(B, H, S, device=DEV)
    sums = prior.clone()
    _, p = check(codec.attend_kv(q, ck, cv, mask=seen, weights=sums), q, K, V, seen.view(B, 1, 1, 1, S))
    reach = (2.0 ** -20 + D * 2.0 ** -24) * D ** -0.5 * (q.double().norm(dim=-1).reshape(B, H, -1).amax(-1) * K.norm(dim=-1).amax(-1)).unsqueeze(-1)
    got = p.sum((2, 3))
    assert bool(((sums.double() - prior.double() - got).abs() <= got * torch.expm1(2 * reach) + got * (T * G + 8) * 2.0 ** -24 + (prior + got) * 2.0 ** -23).all())
    assert torch.equal(sums[1, :, ::3], prior[1, :, ::3]) and torch.equal(sums[1, :, 590:], prior[1, :, 590:])


def test_tracked_attention_sums(pkg):
    """Sums of several steps, tokens going from the window into the packed store in between."""
    B, H, G, D = 2, 2, 4, 128
    cache, plain = make_cache(pkg, B, H, 150, 16, D, BF, track_weights=True), make_cache(pkg, B, H, 150, 16, D, BF)
    sums = torch.zeros(B, H, 166, dtype=torch.float64, device=DEV)
    for step in range(40):
        if step:
            k, v = rand((B, H, 1, D), 100 + step, BF), rand((B, H, 1, D), 200 + step, BF)
            cache.append(k, v, 1)
            plain.append(k, v, 1)
            sums = torch.cat((sums, sums.new_zeros(B, H, 1)), 2)
        q = rand((B, H * G, 1, D), 300 + step, BF)
        out = cache.attend(q, 1)
        K, V = contents(cache)
        ref, p = check(out, q, K, V, torch.ones(K.shape[2], dtype=torch.bool, device=DEV))
        sums += p.sum((2, 3))
        assert (out.float() - plain.attend(q, 1).float()).norm() <= 2.0 ** -6 * out.float().norm()
    got = cache.attention_weights(1)
    assert got.shape == sums.shape and ((got.double() - sums).abs() <= 2e-5 * sums + 1e-7).all()
    assert abs(got.double().sum().item() - 40 * B * H * G) < 1e-2
    other = copy.deepcopy(cache)
    other.attend(q, 1)
    assert torch.equal(cache.attention_weights(1), got) and not torch.equal(other.attention_weights(1), got)
    assert torch.equal(pickle.loads(pickle.dumps(cache)).attention_weights(1), got)


@pytest.mark.parametrize("B,H,n,w,keep,D,dtype,kb,vb", [
    (1, 2, 300, 16, 100, 128, BF, 4, 2),
    (2, 3, 1025, 0, 1, 128, BF, 4, 2),
    (1, 1, 5000, 7, 4999, 64, F16, 6, 4),
    (2, 2, 64, 128, 0, 96, BF, 3, 2),
    (1, 4, 333, 10, 33, 80, F32, 4, 4),
    (1, 2, 100, 3, 50, 33, F16, 2, 8),
    (3, 1, 40000, 5, 20001, 128, BF, 4, 2),
    (1, 2, 1024, 0, 1023, 64, BF, 2, 2), (1, 1, 1, 0, 1, 64, BF, 2, 2), (2, 1, 4096, 1, 5, 64, BF, 2, 2), (1, 1, 16385, 0, 16000, 64, BF, 2, 2),
    (1, 2, 65536, 3, 1030, 64, BF, 2, 2), (1, 2, 65537, 3, 40000, 64, BF, 2, 2), (1, 1, 200001, 0, 777, 64, BF, 2, 2),
])
def test_evict_keeps_the_largest(pkg, B, H, n, w, keep, D, dtype, kb, vb):
    codec = pkg.TurboQuantV3(D, key_bits=kb, value_bits=vb, residual_window=w, layer_idx=8, device=DEV)
    ks, vs = outlier_kv((B, H, n + w, D), seed=1, dtype=dtype).to(DEV), outlier_kv((B, H, n + w, D), seed=2, dtype=dtype).to(DEV)
    ck, cv = codec.compress_kv(ks, vs)
    g = torch.Generator()
    g.manual_seed(n)
    cases = {"spread": torch.exp(3 * torch.randn(B, H, n + w, generator=g)), "ties": torch.randint(0, 3, (B, H, n + w), generator=g).float(), "equal": torch.zeros(B, H, n + w),
             "signs": torch.randn(B, H, n + w, generator=g)}
    odd = torch.randn(B, H, n + w, generator=g)
    odd[..., ::7], odd[..., 1::11], odd[..., 2::13], odd[..., 3::17], odd[..., 4::19] = float("nan"), float("inf"), -0.0, 0.0, float("-inf")
    cases["odd"] = odd
    for name, weights in cases.items():
        weights = weights.to(DEV)
        nk, nv, left, kept = codec.evict_kv(ck, cv, weights, keep)
        order = torch.sort(torch.where(weights[:, :, :n] == 0, torch.zeros_like(weights[:, :, :n]), weights[:, :, :n]), dim=-1, descending=True, stable=True).indices
        want = torch.sort(order[:, :, :keep], dim=-1).values
        assert torch.equal(kept, want), name
        for new, old in ((nk, ck), (nv, cv)):
            assert new["shape"] == (B, H, keep + w, D) and new["split_at"] == keep and new["compressed"]["shape"] == (B, H, keep, D)
            assert torch.equal(new["compressed"]["idx_bytes"], torch.take_along_dim(old["compressed"]["idx_bytes"], want.unsqueeze(-1), 2))
            assert torch.equal(new["compressed"]["vec_norms"].view(torch.int16), torch.take_along_dim(old["compressed"]["vec_norms"].view(torch.int16), want, 2))
            assert torch.equal(new["fp16"], old["fp16"])
        rest = torch.cat((torch.take_along_dim(weights[:, :, :n], want, 2), weights[:, :, n:]), 2)
        assert torch.equal(left.view(torch.int32), rest.view(torch.int32))
    if keep:
        full = codec.decompress_kv(ck, cv)
        thin = codec.decompress_kv(nk, nv)
        for f, t in zip(full, thin):
            assert torch.equal(t[:, :, :keep], torch.take_along_dim(f[:, :, :n], want.unsqueeze(-1), 2)) and torch.equal(t[:, :, keep:], f[:, :, n:])
    everything = codec.evict_kv(ck, cv, weights, n + 5)
    assert torch.equal(everything[3], torch.arange(n, device=DEV).expand(B, H, n)) and torch.equal(everything[0]["compressed"]["idx_bytes"], ck["compressed"]["idx_bytes"])


@pytest.mark.parametrize("n,keep", [(2000, 100), (3000, 1700), (40000, 300), (1100003, 400000)])
def test_evict_of_weights_that_lie_close(pkg, n, keep):
    """More NaN than stay above numbers anywhere (the range of what is searched ends at the largest whole number), neighbours among float32, a few values many times."""
    codec = pkg.TurboQuantV3(64, key_bits=2, value_bits=2, residual_window=0, layer_idx=8, device=DEV)
    ck, cv = codec.compress_kv(rand((1, 2, n, 64), 1, BF), rand((1, 2, n, 64), 2, BF))
    g = torch.Generator()
    g.manual_seed(n)
    places = torch.stack([torch.randperm(n, generator=g) for _ in range(2)]).unsqueeze(0)
    neighbours = (places.int() + 0x3f8abcde).view(torch.float32)
    many_nan = torch.where(places < 2 * keep, torch.full((), float("nan")), neighbours)
    few_values = (places.int() % 3 + 0x3f8abcde).view(torch.float32)
    steps = (places.int() // 700 * 5 + 0x3f8abcde).view(torch.float32)
    far = torch.where(places < 300, torch.full((), float("inf")), neighbours * torch.tensor([1e-38, -1e30]).view(1, 2, 1))
    for name, weights in {"neighbours": neighbours, "many NaN": many_nan, "few values": few_values, "steps": steps, "far": far}.items():
        weights = weights.to(DEV)
        kept = codec.evict_kv(ck, cv, weights, keep)[3]
        want = torch.sort(torch.sort(weights, dim=-1, descending=True, stable=True).indices[:, :, :keep], dim=-1).values
        assert torch.equal(kept, want), name


@pytest.mark.parametrize("D,dtype", [(128, BF), (96, F16), (80, F32)])
def test_generation_with_drafts_and_a_budget(pkg, D, dtype, tmp_path):
    """The operators as they are used together: verify a draft, append what is accepted, attend, thin out when over the budget, go on."""
    B, H, G, w, T, keep = 2, 2, 2, 16, 6, 60
    cache = make_cache(pkg, B, H, 90, w, D, dtype, track_weights=True)
    seen = 90 + w
    for step in range(8):
        tree = random_tree(T, step)
        q, k, v = rand((B, H * G, T, D), 10 + step, dtype), rand((B, H, T, D), 20 + step, dtype), rand((B, H, T, D), 30 + step, dtype)
        K, V = contents(cache)
        out = cache.attend_tree(q, k, v, 1, tree)
        check(out, q, torch.cat((K, k.double()), 2), torch.cat((V, v.double()), 2), torch.cat((torch.ones(T, K.shape[2], dtype=torch.bool, device=DEV), tree), 1))
        path = torch.nonzero(tree[T - 1 - step % 3]).flatten()
        cache.append(k[:, :, path], v[:, :, path], 1)
        seen += path.numel()
        q1 = rand((B, H * G, 1, D), 40 + step, dtype)
        K, V = contents(cache)
        check(cache.attend(q1, 1), q1, K, V, torch.ones(K.shape[2], dtype=torch.bool, device=DEV))
        if cache._stores[1].n_compressed > keep + 8:
            before, sums = contents(cache), cache.attention_weights(1).clone()
            n = cache._stores[1].n_compressed
            kept = cache.evict(keep, 1)
            after = contents(cache)
            for a, b in zip(after, before):
                assert torch.equal(a, torch.cat((torch.take_along_dim(b[:, :, :n], kept.unsqueeze(-1), 2), b[:, :, n:]), 2))
            assert torch.equal(cache.attention_weights(1), torch.cat((torch.take_along_dim(sums[:, :, :n], kept, 2), sums[:, :, n:]), 2))
        assert cache.get_seq_length(1) == seen
    path = str(tmp_path / "cache.safetensors")
    cache.save(path)
    again = pkg.V3Cache.load(path, device=DEV)
    assert torch.equal(again.attention_weights(1), cache.attention_weights(1)) and again.get_seq_length(1) == seen
    assert torch.equal(again.attend(q1, 1), cache.attend(q1, 1))
    k1, v1 = rand((B, H, 1, D), 50, dtype), rand((B, H, 1, D), 51, dtype)
    fk, fv = cache.update(k1, v1, 1)
    K, V = contents(cache)
    assert fk.shape == K.shape and torch.equal(fk[:, :, -1:], k1)
    assert (fk.double() - K).norm() <= 4e-3 * K.norm()


def test_nothing_cached_yet(pkg):
    cache = pkg.V3Cache(n_layers=4)
    q, k, v = rand((2, 4, 5, 128), 1, BF), rand((2, 2, 5, 128), 2, BF), rand((2, 2, 5, 128), 3, BF)
    tree = random_tree(5, 3)
    tree[2] = False                       # sees nothing at all
    out = cache.attend_tree(q, k, v, 0, tree)
    check(out, q, k.double(), v.double(), tree)
    assert not bool(out[:, :, 2].any()) and cache.get_seq_length(0) == 0
    some = cache.attend_tree(q, k[:, :, :3], v[:, :, :3], 0, tree[:, :3])
    check(some, q, k.double()[:, :, :3], v.double()[:, :, :3], tree[:, :3])


def test_captured_and_replayed(pkg):
    """Two graphs and eager calls between them, with their own scratch."""
    cache = make_cache(pkg, 1, 2, 500, 32, 128, BF, track_weights=True)
    q, k, v = rand((1, 8, 6, 128), 1, BF), rand((1, 2, 6, 128), 2, BF), rand((1, 2, 6, 128), 3, BF)
    tree, q1 = random_tree(6, 1), rand((1, 8, 1, 128), 4, BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend_tree(q, k, v, 1, tree)
        cache.attend(q1, 1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        out_a = cache.attend_tree(q, k, v, 1, tree)
    with torch.cuda.graph(b):
        out_b = cache.attend(q1, 1)
    torch.cuda.synchronize()
    for step in range(4):
        q.copy_(rand(q.shape, 50 + step, BF))
        q1.copy_(rand(q1.shape, 60 + step, BF))
        cache.attention_weights(1).zero_()
        a.replay()
        b.replay()
        torch.cuda.synchronize()
        sums = cache.attention_weights(1).clone()
        got_a, got_b = out_a.clone(), out_b.clone()
        assert torch.equal(got_a, cache.attend_tree(q, k, v, 1, tree))
        cache.attention_weights(1).zero_()
        assert torch.equal(got_b, cache.attend(q1, 1)) and torch.equal(sums, cache.attention_weights(1))
        torch.cuda.synchronize()


def test_two_streams_at_once(pkg):
    cache = make_cache(pkg, 1, 4, 3000, 32, 128, BF)
    sets = [(rand((1, 16, 9, 128), i, BF), rand((1, 4, 9, 128), 10 + i, BF), rand((1, 4, 9, 128), 20 + i, BF)) for i in range(2)]
    want = [cache.attend_tree(*s, 1) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(cache.attend_tree(*s, 1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


def test_many_queries_go_in_parts(pkg, monkeypatch):
    """A call whose scratch would be too large takes its queries in parts; results and sums are those of the parts."""
    codec = pkg.TurboQuantV3(64, key_bits=4, value_bits=4, residual_window=8, layer_idx=8, device=DEV)
    ck, cv = codec.compress_kv(rand((2, 2, 150, 64), 1, BF), rand((2, 2, 150, 64), 2, BF))
    q = rand((2, 4, 70, 64), 3, BF)
    w0, w1 = torch.zeros(2, 2, 150, device=DEV), torch.zeros(2, 2, 150, device=DEV)
    lengths = torch.tensor([150, 60], device=DEV)
    whole = codec.attend_kv(q, ck, cv, lengths=lengths, weights=w0)
    cache = make_cache(pkg, 2, 2, 100, 8, 64, BF)
    k, v = rand((2, 2, 70, 64), 4, BF), rand((2, 2, 70, 64), 5, BF)
    tree = random_tree(70, 1, 2)
    chained, treed = cache.attend_tree(q, k, v, 1), cache.attend_tree(q, k, v, 1, tree)
    monkeypatch.setattr(pkg._native, "MANY_SCRATCH", 1 << 17)
    parts = codec.attend_kv(q, ck, cv, lengths=lengths, weights=w1)
    assert (parts.float() - whole.float()).norm() <= 2.0 ** -8 * whole.float().norm() and (w0 - w1).abs().max() <= 1e-4
    for a, b in ((chained, cache.attend_tree(q, k, v, 1)), (treed, cache.attend_tree(q, k, v, 1, tree))):
        assert (a.float() - b.float()).norm() <= 2.0 ** -8 * a.float().norm()


def test_offsets_past_32_bits(pkg):
    """The last row of a store of more than 2^32 bytes of codes."""
    B, H, n, cap, D = 1, 9, 70, 1 << 23, 128
    codec = pkg.TurboQuantV3(D, key_bits=4, value_bits=2, residual_window=0, layer_idx=8, device=DEV)
    k_store, v_store = (torch.empty((B, H, cap, g), dtype=torch.uint8, device=DEV) for g in (64, 32))
    kn_store, vn_store = (torch.empty((B, H, cap), dtype=torch.float16, device=DEV) for _ in range(2))
    assert (H - 1) * cap * 64 >= 1 << 32
    ks, vs = rand((B, H, n, D), 1, BF), rand((B, H, n, D), 2, BF)
    codec.key_compressor.compress_into(ks, k_store[:, :, -n:], kn_store[:, :, -n:])
    codec.val_compressor.compress_into(vs, v_store[:, :, -n:], vn_store[:, :, -n:])
    packed = ((k_store[:, :, -n:], kn_store[:, :, -n:]), (v_store[:, :, -n:], vn_store[:, :, -n:]))
    dense = tuple((i.contiguous(), m.contiguous()) for i, m in packed)
    q = rand((B, H * 2, 3, D), 3, BF)
    kc, vc = codec.key_compressor, codec.val_compressor
    tables = (kc.table(q.device), vc.table(q.device))
    call = lambda p: pkg._native.attend_many(q, p, n, tables, (kc.bits, vc.bits))  # noqa: E731
    assert torch.equal(call(packed), call(dense))
    weights = torch.rand(B, H, n, device=DEV)
    far, near = pkg._native.evict(packed, n, (4, 2), D, weights, 33), pkg._native.evict(dense, n, (4, 2), D, weights, 33)
    assert all(torch.equal(a, b) for x, y in zip(far[0], near[0]) for a, b in zip(x, y)) and torch.equal(far[2], near[2])


def test_one_step_calls_answer_as_the_general_ones(pkg, monkeypatch):
    """Eager calls go by one extension call where everything lies as the library takes it: the same bits as without it, window turned or not."""
    cache = make_cache(pkg, 2, 2, 300, 16, 128, BF, track_weights=True)
    k1, v1 = rand((2, 2, 5, 128), 7, BF), rand((2, 2, 5, 128), 8, BF)
    for i in range(5):                                    # (the window is a ring of buffer slots: its first token moves)
        cache.append(k1[:, :, i:i + 1], v1[:, :, i:i + 1], 1)
    q, k, v, tree = rand((2, 8, 9, 128), 1, BF), rand((2, 2, 9, 128), 2, BF), rand((2, 2, 9, 128), 3, BF), random_tree(9, 1, 2)
    codec = pkg.TurboQuantV3(128, key_bits=4, value_bits=2, residual_window=16, layer_idx=8, device=DEV)
    ck, cv = codec.compress_kv(rand((2, 2, 200, 128), 4, BF), rand((2, 2, 200, 128), 5, BF))
    lengths, mask = torch.tensor([150, 0], dtype=torch.int32, device=DEV), torch.rand(2, 200, device=DEV) < 0.5

    def answers():
        w = torch.zeros(2, 2, 200, device=DEV)
        cache.attention_weights(1).zero_()
        out = [cache.attend_tree(q, k, v, 1, tree), cache.attend_tree(q, k, v, 1), cache.attend(q[:, :, :1], 1), cache.attention_weights(1).clone(),
               codec.attend_kv(q, ck, cv, lengths=lengths, mask=mask, weights=w, scale=0.1), w]
        nk, nv, left, kept = codec.evict_kv(ck, cv, w, 33)
        return out + [nk["compressed"]["idx_bytes"], nk["compressed"]["vec_norms"], nv["compressed"]["idx_bytes"], nv["compressed"]["vec_norms"], left, kept]
    answers()                                             # (the scratch of the stream is there afterwards)
    one_step = answers()
    monkeypatch.setattr(pkg._native, "attend_many_store", lambda *a: None)

    class Without:
        evict = staticmethod(lambda *a: None)

        def __getattr__(self, name):
            return getattr(real, name)
    real = pkg._native.fast()
    monkeypatch.setattr(pkg._native, "fast", lambda: Without())
    for i, (a, b) in enumerate(zip(one_step, answers())):
        assert torch.equal(a, b), i


def test_eviction_from_the_cache_that_models_use(pkg):
    """Positions go on after an eviction, masks are made for the keys that are left, and update answers with those and the new ones."""
    cache = pkg.hf_cache_class()(key_bits=4, value_bits=2, residual_window=8, n_layers=4, track_weights=True)
    k, v = rand((1, 2, 90, 128), 1, BF), rand((1, 2, 90, 128), 2, BF)
    cache.update(k, v, 1)
    for i in range(3):
        cache.attend(rand((1, 4, 1, 128), 10 + i, BF), 1)
    assert cache.get_mask_sizes(1, 1) == (91, 0)
    kept = cache.evict(30, 1)
    assert kept.shape == (1, 2, 30) and cache.get_seq_length(1) == 90 and cache.get_mask_sizes(5, 1) == (38 + 5, 52)
    k1, v1 = rand((1, 2, 4, 128), 3, BF), rand((1, 2, 4, 128), 4, BF)
    fk, fv = cache.update(k1, v1, 1)                      # (the window's oldest four tokens are packed by that)
    K, V = contents(cache)
    assert fk.shape == (1, 2, 42, 128) and torch.equal(fk[:, :, -4:], k1) and torch.equal(fv[:, :, -4:], v1)
    assert (fk.double() - K).norm() <= 4e-3 * K.norm() and (fv.double() - V).norm() <= 4e-3 * V.norm() and cache.get_seq_length(1) == 94
    q = rand((1, 4, 1, 128), 5, BF)
    check(cache.attend(q, 1), q, K, V, torch.ones(42, dtype=torch.bool, device=DEV))
    assert cache.evict(100, 1).shape == (1, 2, 34) and not cache.evict(0)[1].numel() and cache.get_mask_sizes(1, 1) == (9, 86)
