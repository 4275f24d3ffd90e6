"""What attention over several queries, kept sums and eviction refuse: found on the host, before anything is launched."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_entry_points_check_their_arguments(pkg):
    native = pkg._native
    L = native.lib()
    r = native.TqAttendRequest(batch=1, heads=2, group=2, n_queries=3, tokens=100, packed_row_stride=0, head_dim=128, dtype=2, bits_k=4, bits_v=2, scale=1.0)
    assert L.tq_attend_many_scratch(ctypes.byref(r)) > 0
    assert L.tq_attend_many_scratch(None) == -1 and L.tq_attend_many(None, None, 0, None) == -1
    assert L.tq_attend_many(ctypes.byref(r), None, 0, None) == -1                   # no queries
    for field, value, status in (("dtype", 3, -4), ("bits_k", 0, -2), ("bits_v", 9, -2), ("head_dim", 7, -3), ("head_dim", 257, -3), ("batch", -1, -5), ("heads", -1, -5),
                                 ("group", -1, -5), ("n_queries", -1, -5), ("tokens", -1, -5), ("tokens", 1 << 31, -5), ("packed_row_stride", 99, -5), ("group", 1 << 31, -5),
                                 ("batch", 1 << 30, -5), ("packed_row_stride", -1, -5)):
        bad = native.TqAttendRequest.from_buffer_copy(r)
        setattr(bad, field, value)
        assert L.tq_attend_many_scratch(ctypes.byref(bad)) == status, field
        assert L.tq_attend_many(ctypes.byref(bad), 16, 1 << 40, None) == status, field
    bad = native.TqAttendRequest.from_buffer_copy(r)
    bad.window.tokens = 65537
    assert L.tq_attend_many_scratch(ctypes.byref(bad)) == -5
    ready = native.TqAttendRequest.from_buffer_copy(r)
    for name in ("queries", "out", "k_idx", "k_norms", "v_idx", "v_norms", "table_k", "table_v"):
        setattr(ready, name, 4096)
    ready.packed_row_stride = 128
    need = L.tq_attend_many_scratch(ctypes.byref(ready))
    assert L.tq_attend_many(ctypes.byref(ready), 4096, need - 1, None) == -10
    assert L.tq_attend_many(ctypes.byref(ready), 4100, need, None) == -8
    for name in ("queries", "out", "table_k", "table_v", "k_norms", "v_norms", "lengths", "weights"):
        bad = native.TqAttendRequest.from_buffer_copy(ready)
        bad.weights_stride = 1000
        setattr(bad, name, 4097)
        assert L.tq_attend_many(ctypes.byref(bad), 4096, need, None) == -8, name
    for name in ("queries", "out", "k_idx", "k_norms", "v_idx", "v_norms", "table_k", "table_v"):
        bad = native.TqAttendRequest.from_buffer_copy(ready)
        setattr(bad, name, None)
        assert L.tq_attend_many(ctypes.byref(bad), 4096, need, None) == -1, name
    bad = native.TqAttendRequest.from_buffer_copy(ready)
    bad.weights, bad.weights_stride = 4096, 99
    assert L.tq_attend_many(ctypes.byref(bad), 4096, need, None) == -5
    bad = native.TqAttendRequest.from_buffer_copy(ready)
    bad.drafts.k = bad.drafts.v = 4096
    bad.drafts.tokens = 2                                                           # not one for each query, and no tree
    assert L.tq_attend_many(ctypes.byref(bad), 4096, 1 << 40, None) == -5
    bad.drafts.k = None
    assert L.tq_attend_many(ctypes.byref(bad), 4096, 1 << 40, None) == -1
    bad = native.TqAttendRequest.from_buffer_copy(ready)
    bad.batch, bad.mask, bad.mask_stride = 2, 4096, 99
    assert L.tq_attend_many(ctypes.byref(bad), 4096, 1 << 40, None) == -5
    empty = native.TqAttendRequest.from_buffer_copy(r)
    empty.n_queries = 0
    assert L.tq_attend_many(ctypes.byref(empty), None, 0, None) == 0                # nothing to do


def test_evict_entry_point_checks_its_arguments(pkg):
    native = pkg._native
    L = native.lib()
    full = native.TqPackedStore(4096, 4096, 4096, 4096, 0)
    call = lambda frm=full, to=full, w=4096, ws=300, wo=4096, wos=300, rest=5, rows=2, tokens=100, keep=50, D=128, bk=4, bv=2, kept=4096, scratch=None, words=0: L.tq_evict(  # noqa: E731
        ctypes.byref(frm) if frm is not None else None, ctypes.byref(to) if to is not None else None, w, ws, wo, wos, rest, rows, tokens, keep, D, bk, bv, kept, scratch, words, None)
    assert call(frm=None) == -1 and call(to=None) == -1 and call(w=None) == -1 and call(wo=None) == -1 and call(kept=None) == -1
    assert call(bk=0) == -2 and call(bv=9) == -2 and call(D=7) == -3 and call(D=300) == -3
    for bad in ({"rows": -1}, {"tokens": -1}, {"keep": -1}, {"keep": 101}, {"rest": -1}, {"rest": 65537}, {"ws": 104}, {"wos": 54}, {"rows": 1 << 31},
                {"frm": native.TqPackedStore(4096, 4096, 4096, 4096, 99)}, {"to": native.TqPackedStore(4096, 4096, 4096, 4096, 49)},
                {"to": native.TqPackedStore(4096, 4096, 4096, 4096, -1)}):
        assert call(**bad) == -5, bad
    assert call(w=4098) == -8 and call(wo=4098) == -8 and call(kept=4100) == -8 and call(frm=native.TqPackedStore(4096, 4097, 4096, 4096, 0)) == -8
    assert call(frm=native.TqPackedStore(4096, 4096, None, 4096, 0)) == -1 and call(to=native.TqPackedStore(None, 4096, 4096, 4096, 0)) == -1
    assert call(rows=0) == 0 and call(keep=0, rest=0) == 0
    need = L.tq_evict_scratch(2, 40000)
    assert need > 0 and L.tq_evict_scratch(2, 32768) == 0 and L.tq_evict_scratch(-1, 40000) == -5 and L.tq_evict_scratch(1, 1 << 31) == -5
    long_rows = {"tokens": 40000, "ws": 50000}
    assert call(**long_rows) == -1 and call(**long_rows, scratch=4096, words=need - 1) == -10 and call(**long_rows, scratch=4098, words=need) == -8


def test_cpu_tensors_are_refused(pkg):
    cache = pkg.V3Cache(n_layers=2, track_weights=True)
    q, k = torch.zeros(1, 4, 2, 128), torch.zeros(1, 2, 2, 128)
    with pytest.raises(pkg._native.TqError):
        cache.attend_tree(q, k, k, 0)
    codec = pkg.TurboQuantV3(128, residual_window=128)
    ck, cv = codec.compress_kv(k, k)
    with pytest.raises(pkg._native.TqError):
        codec.attend_kv(q, ck, cv)


def test_state_that_the_calls_need(pkg):
    cache = pkg.V3Cache(n_layers=2)
    with pytest.raises(ValueError, match="nothing is cached"):
        cache.attention_weights(0)
    assert cache.evict(5) == {}
    for keep in (-1, 1.5, True):
        with pytest.raises(ValueError, match="whole number"):
            cache.evict(keep)
    store = cache._store(torch.zeros(1, 2, 3, 128), 0)
    assert store.weights is None
    with pytest.raises(ValueError, match="does not track"):
        cache.evict(5, 0)
    tracked = pkg.V3Cache(n_layers=2, residual_window=16, track_weights=True)
    store = tracked._store(torch.zeros(1, 2, 3, 128), 0)
    store.reserve(300)
    assert store.weights.shape == (1, 2, store.capacity + 16) and not bool(store.weights.any())
    assert tracked.attention_weights(0).shape == (1, 2, 0)


def test_dictionaries_that_do_not_go_together(pkg):
    codec = pkg.TurboQuantV3(128, residual_window=16)
    k = torch.zeros(1, 2, 8, 128)
    ck, cv = codec.compress_kv(k, k)
    longer, _ = codec.compress_kv(torch.zeros(1, 2, 9, 128), torch.zeros(1, 2, 9, 128))
    with pytest.raises(ValueError, match="same tokens"):
        codec.attend_kv(k, longer, cv)
    with pytest.raises(ValueError, match="head dimension"):
        pkg.TurboQuantV3(64)._packed_pairs(ck, cv)
    nk, nv, left, kept = codec.evict_kv(ck, cv, torch.zeros(1, 2, 8), 3)           # all of it window: nothing leaves
    assert nk["split_at"] == 8 and kept.shape == (1, 2, 0) and left.shape == (1, 2, 8)
    with pytest.raises(ValueError, match="weights must be"):
        codec.evict_kv(ck, cv, torch.zeros(1, 2, 7), 3)


def test_structures_match_the_header(pkg, tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler to read the header with")
    pairs = ((pkg._native.TqPlainTokens, "tq_plain_tokens"), (pkg._native.TqAttendRequest, "tq_attend_request"), (pkg._native.TqPackedStore, "tq_packed_store"))
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tqamd.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", sizeof({c}));\n' + "".join(f'  printf("%zu ", offsetof({c}, {f[0]}));\n' for f in py._fields_) for py, c in pairs) + "  return 0;\n}\n")
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [x for py, _ in pairs for x in (ctypes.sizeof(py), *(getattr(py, f[0]).offset for f in py._fields_))]
