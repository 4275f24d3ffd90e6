"""GPU tests of beam search: equal sums however the logits lie in memory, and caches whose answer is still due."""
import pytest
import torch

from test_gpu_beams import check
from test_gpu_parity import DEV, outlier_kv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a HIP device; there is no CPU fallback to test")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,best", [(1, 4, 50257, 8), (3, 8, 5003, 16), (16, 8, 32003, 16), (2, 5, 513, 20), (40, 4, 4099, 8), (1, 3, 2047, 9), (1, 64, 8191, 64)])
def test_equal_beams_go_by_their_order(pkg, dtype, B, K, V, best):
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    for trial in range(4):
        # (rows of an odd length begin at every alignment there is)
        logits = (3.0 * torch.randn((B, 1, V), generator=g, device=DEV)).to(dtype).expand(B, K, V).contiguous()
        scores = torch.randn((B, 1), generator=g, device=DEV).expand(B, K).contiguous()
        same = check(pkg.beam_select(logits, scores, best), logits, scores, best)
        assert bool(same.all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V", [(2, 4, 8000), (1, 4, 50257), (16, 8, 20001), (3, 1, 1), (2, 2, 9), (1, 2, 511), (1, 2, 512), (1, 2, 2048)])
def test_a_choice_does_not_depend_on_where_logits_lie(pkg, dtype, B, K, V):
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    logits, scores, best = (3.0 * torch.randn((B, K, V), generator=g, device=DEV)).to(dtype), torch.randn((B, K), generator=g, device=DEV), min(2 * K, K * V)
    want = pkg.beam_select(logits, scores, best)
    check(want, logits, scores, best)
    for ahead in range(1, 9):
        for row in (V + ahead, V + 16):
            # NaN around the rows: nothing of it is read for a logit
            wide = torch.full((B * K * row + ahead,), float("nan"), dtype=dtype, device=DEV)
            view = wide[ahead:].view(B, K, row)[:, :, :V]
            view.copy_(logits)
            assert all(torch.equal(x, y) for x, y in zip(pkg.beam_select(view, scores, best), want))


def test_a_pending_step_is_answered_before_beams_move(pkg):
    pytest.importorskip("transformers")
    for call in (lambda c: c.reorder(torch.tensor([1, 0], device=DEV)), lambda c: c.reorder_cache(torch.tensor([1, 0], device=DEV)),
                 lambda c: c.beam_step(torch.randn((1, 2, 50), device=DEV), torch.zeros((1, 2), device=DEV))):
        cache = pkg.hf_cache_class()(residual_window=8, n_layers=1, packed_attention=True)
        k, v = (outlier_kv((2, 2, 50, 128), seed=i, dtype=torch.bfloat16).to(DEV) for i in (0, 1))
        t = outlier_kv((2, 2, 1, 128), seed=5, dtype=torch.bfloat16).to(DEV)
        cache.update(k, v, 0)
        call(cache)                          # (nothing is due)
        before = [x.clone() for x in cache._stores[0].window()]
        cache.update(t, t, 0)
        held = [x.clone() for x in cache._stores[0].window()]
        with pytest.raises(RuntimeError, match="never answered"):
            call(cache)
        assert all(torch.equal(x, y) for x, y in zip(cache._stores[0].window(), held)) and len(before) == 2
