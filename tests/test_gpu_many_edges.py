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
