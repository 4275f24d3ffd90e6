"""What attention over pages, moved pages and beam search's choice refuse, and how a step's work is shared: found and decided on the host, before anything is launched."""
import ctypes
import itertools

import numpy as np
import pytest
import torch


def plan(pkg, sequences, heads=2, group=4, window=0, D=128, dtype=2, room=100000, page=64):
    native = pkg._native
    records = np.zeros((len(sequences), native.PAGED_SEQ), np.int32)
    for r, (fresh, total, packed) in zip(records, sequences):
        r[1:4] = fresh, total, packed
    counts = native.TqPagedCounts()
    items, merges = np.empty((room, native.PAGED_ITEM), np.int32), np.empty((room, native.PAGED_MERGE), np.int32)
    rc = native.lib().tq_paged_plan(records.ctypes.data, len(records), heads, group, window, D, dtype, page, items.ctypes.data, room, merges.ctypes.data, room, ctypes.byref(counts))
    blocks = items.ravel()[counts.items * native.PAGED_ITEM:][:counts.blocks + 1 if counts.few else 0].tolist()
    assert rc or (counts.few == 0) == (not blocks) and (not blocks or (blocks[0] == 0 and blocks[-1] == counts.few and blocks == sorted(blocks)))
    return rc, counts, items[:counts.items], merges[:counts.merges]


SEQUENCES = [
    [(1, 1, 0)], [(1, 64, 0)], [(1, 65, 64)], [(1, 2048, 1856)], [(1, 40000, 39872)], [(512, 33000, 32000)], [(77, 77, 0), (1, 1003, 832), (0, 500, 320), (33, 4000, 3904)],
    [(1, 100 + 97 * i, (97 * i) // 64 * 64) for i in range(64)], [(1, 1 << 20, (1 << 20) - 256)] * 3, [(2000, 2000, 0)], [(5, 300, 192), (0, 0, 0)],
]


@pytest.mark.parametrize("window", [0, 1, 33, 4096])
@pytest.mark.parametrize("sequences", SEQUENCES)
def test_a_plan_covers_what_is_seen_once(pkg, sequences, window):
    for heads, group, D, dtype, page in ((8, 4, 128, 2, 64), (8, 4, 128, 2, 32), (1, 1, 64, 1, 128), (2, 7, 256, 2, 64), (8, 1, 80, 0, 64)):
        rc, counts, items, merges = plan(pkg, sequences, heads, group, window, D, dtype, page=page)
        few = page >= 64 and dtype and D in (64, 96, 128, 256)
        small = [bool(few and f * group <= 16) for f, _, _ in sequences]
        assert all(small[b] == (i < counts.few) for i, b in enumerate(items[:, 0].tolist()))
        assert counts.vectors == max([f * group for (f, _, _), s in zip(sequences, small) if s and f] or [0])
        assert rc == 0 and counts.tiles in ((1, 2) if dtype and D in (64, 128) else (1,)) and 1 <= counts.columns <= 32
        by_group = {}
        for it in items.tolist():
            for h in range(heads) if it[7] < 0 else (it[7],):
                by_group.setdefault((it[0], it[1], h), []).append(it[2:6] + [it[6] if it[6] < 0 or it[7] >= 0 else it[6] + h])
        records, joined = [], {(m[0], m[1], m[2]): m[3:6] for m in merges.tolist()}
        assert len(joined) == len(merges)
        for b, (fresh, total, packed) in enumerate(sequences):
            tiles = -(-fresh * group // 32)
            step, unit = (1, 64) if small[b] else (counts.tiles, 32)
            for t0 in range(0, tiles, step):
              for head in range(heads):
                parts = by_group.pop((b, t0, head))
                first, last = total - fresh + t0 * 32 // group, total - fresh + min(fresh - 1, ((t0 + step) * 32 - 1) // group)
                lo = max(0, first - window + 1) if window else 0
                covered = set()
                for a, z, u, w, _ in parts:
                    assert a % unit == 0 and u % 32 == 0 and 0 <= a <= z <= packed and 0 <= u <= w <= total - packed and (z > a or w > u)
                    assert (z % unit == 0 or z == packed)
                    for x in itertools.chain(range(a // 32, -(-z // 32)), range(1 << 26 | u // 32, 1 << 26 | -(-w // 32))):
                        assert x not in covered
                        covered.add(x)
                want = set(range(lo // unit * unit // 32, -(-packed // 32))) if lo < packed else set()
                want |= set(range(1 << 26 | max(0, lo - packed) // 32, 1 << 26 | -(-(last + 1 - packed) // 32)))
                assert covered == want
                if len(parts) > 1:
                    start, n, gap = joined.pop((b, t0, head))
                    assert sorted(p[4] for p in parts) == list(range(start, start + n * gap, gap)) and n == len(parts) <= 64
                    assert counts.columns >= min(32, fresh * group - 32 * t0)
                    records += [p[4] for p in parts]
                else:
                    assert parts[0][4] == -1
        assert not by_group and not joined and sorted(records) == list(range(counts.records))


def test_plans_are_refused_or_ask_for_room(pkg):
    assert plan(pkg, [])[0] == 0 and plan(pkg, [(0, 5, 0)])[1].items == 0
    for bad in ((5, 4, 0), (-1, 4, 0), (1, 4, 4), (1, 4, -64), (1 << 30, 1 << 30, 0)):
        assert plan(pkg, [bad])[0] == -5
    for kw in ({"heads": 0}, {"group": 0}, {"window": -1}):
        assert plan(pkg, [(1, 5, 0)], **kw)[0] == -5
    rc, counts, _, _ = plan(pkg, SEQUENCES[7], room=3)
    assert rc == -10 and counts.items > 3
    assert pkg._native.lib().tq_paged_plan(None, 1, 1, 1, 0, 128, 2, 64, None, 0, None, 0, ctypes.byref(counts)) == -1
    assert pkg._native.lib().tq_paged_plan(None, 0, 1, 1, 0, 128, 2, 64, None, 0, None, 0, None) == -1


def test_which_combinations_there_are(pkg):
    supported = pkg._native.lib().tq_paged_supported
    for D in range(1, 300):
        for kb, vb in itertools.product(range(0, 10), (1, 2, 4, 8)):
            fine = 2 <= kb <= 8 and vb >= 2 and (D in (64, 128, 256) or (64 < D <= 96 and D % 8 == 0 and (D // (8 // kb)) % 4 == 0 and (D // (8 // vb)) % 4 == 0))
            assert supported(D, 2, kb, vb) == int(fine)
    assert not supported(128, 3, 4, 2)
    for kw in ({"head_dim": 100}, {"head_dim": 128, "key_bits": 1}, {"head_dim": 72, "value_bits": 2}, {"head_dim": 128, "page_tokens": 48}, {"head_dim": 128, "page_tokens": 16},
               {"head_dim": 128, "pages": 0}, {"head_dim": 128, "plain_pages": 1.5}, {"head_dim": 128, "kv_heads": 0}, {"head_dim": 128, "residual_window": -1}):
        kw = {"kv_heads": 2, "n_layers": 1, "pages": 4, "plain_pages": 4, **kw}
        with pytest.raises(ValueError):
            pkg.PagedV3Cache(**kw)
    with pytest.raises(pkg._native.TqError):
        pkg.PagedV3Cache(128, 2, n_layers=1, pages=4, plain_pages=4, device="cpu")
    with pytest.raises(pkg._native.TqError):
        pkg.PagedV3Cache(128, 2, n_layers=1, pages=4, plain_pages=4, dtype=torch.float64)


def test_attention_checks_its_request(pkg):
    native = pkg._native
    L = native.lib()
    rc, counts, _, _ = plan(pkg, [(1, 40000, 39872)], heads=8)
    r = native.TqPagedRequest(counts=counts, scale=1.0, heads=8, group=4, page_tokens=64, head_dim=128, dtype=2, bits_k=4, bits_v=2)
    for name in ("queries", "out", "packed_pool", "plain_pool", "table_k", "table_v", "sequences", "tables", "items", "merges"):
        setattr(r, name, 4096)
    need = L.tq_paged_scratch(ctypes.byref(counts), 8, 128)
    assert rc == 0 and counts.merges == 8 and need == counts.records * counts.columns * 130
    assert L.tq_paged_attend(ctypes.byref(r), 4096, need - 1, None) == -10 and L.tq_paged_attend(None, None, 0, None) == -1
    assert L.tq_paged_scratch(None, 8, 128) == -1 and L.tq_paged_scratch(ctypes.byref(counts), 0, 128) == -5 and L.tq_paged_scratch(ctypes.byref(counts), 8, 7) == -3
    copy = lambda: native.TqPagedRequest.from_buffer_copy(r)  # noqa: E731
    for field, value, status in (("dtype", 3, -4), ("bits_k", 0, -2), ("bits_v", 9, -2), ("bits_k", 1, -3), ("head_dim", 100, -3), ("heads", 0, -5), ("group", 0, -5), ("page_tokens", 48, -5),
                                 ("page_tokens", 16, -5), ("sliding_window", -1, -5), ("softcap", -1.0, -5), ("softcap", float("nan"), -5), ("softcap", float("inf"), -5), ("softcap", 1e-38, -5), ("softcap", 1025.0, -5)):
        bad = copy()
        setattr(bad, field, value)
        assert L.tq_paged_attend(ctypes.byref(bad), 4096, 1 << 40, None) == status, field
    for name in ("queries", "out", "packed_pool", "plain_pool", "table_k", "table_v", "sequences", "tables", "items", "merges"):
        bad = copy()
        setattr(bad, name, None)
        assert L.tq_paged_attend(ctypes.byref(bad), 4096, need, None) == -1, name
        setattr(bad, name, 4097)
        assert L.tq_paged_attend(ctypes.byref(bad), 4096, need, None) == -8, name
    assert L.tq_paged_attend(ctypes.byref(r), None, need, None) == -1 and L.tq_paged_attend(ctypes.byref(r), 4100, need, None) == -8
    for name in ("packed_page_stride", "k_norms", "v_idx", "v_norms", "plain_page_stride", "plain_values"):
        bad = copy()
        setattr(bad, name, 8)
        assert L.tq_paged_attend(ctypes.byref(bad), 4096, need, None) == -8, name
    bad = copy()
    bad.counts.tiles = 2
    bad.dtype = 0
    assert L.tq_paged_attend(ctypes.byref(bad), 4096, 1 << 40, None) == -5
    for field, value in (("few", -1), ("few", counts.items + 1), ("vectors", 0), ("vectors", 17)):
        bad = copy()
        setattr(bad.counts, field, value)
        assert L.tq_paged_attend(ctypes.byref(bad), 4096, 1 << 40, None) == -5, field
    bad = copy()
    bad.counts.items = 0
    assert L.tq_paged_attend(ctypes.byref(bad), None, 0, None) == 0


def test_moves_check_their_arguments(pkg):
    native = pkg._native
    L = native.lib()
    run = lambda *v: (native.TqMoveSegment * 1)(v)  # noqa: E731
    assert L.tq_reorder(None, 0, 4, 2, None, None) == 0 and L.tq_reorder(None, 1, 4, 2, 4096, None) == -1
    assert L.tq_reorder(run(4096, 4096, 1024, 100), 1, 4, 2, None, None) == -1 and L.tq_reorder(run(4096, 4096, 1024, 100), 1, 4, 2, 4097, None) == -8
    assert L.tq_reorder(run(4096, 4096, 1024, 100), 1, 1025, 2, 4096, None) == -10
    for bad, status in (((None, 4096, 1024, 100), -1), ((4096, 4096, 1024, -1), -5), ((4096, 4096, 99, 100), -5), ((4096, 1000, 1024, 100), -5), ((4096, -4096, 1024, 100), -5),
                        ((4096, 1 << 40, 1 << 32, 1 << 31), -5)):
        assert L.tq_reorder(run(*bad), 1, 4, 2, 4096, None) == status, bad
    assert L.tq_reorder(run(4096, 4096, 1024, 100), 1, -1, 2, 4096, None) == -5 and L.tq_reorder(run(4096, 4096, 1024, 100), -1, 1, 2, 4096, None) == -5
    pairs = np.array([[1, 2, 64], [3, 4, 128]], np.int32)
    copy = lambda p=pairs, a=4096, sa=4096, b=8192, sb=4096, rows=4, row=256, n=2: L.tq_copy_pages(a, sa, b, sb, rows, row, None if p is None else p.ctypes.data, n, None)  # noqa: E731
    assert copy(n=0) == 0 and copy(rows=0) == 0
    assert copy(a=None) == -1 and copy(b=None) == -1 and copy(p=None) == -1
    assert copy(a=4100) == -8 and copy(sb=4100) == -8 and copy(row=250) == -8 and copy(p=np.array([[1, 2, 60]] * 2, np.int32)) == -8
    assert copy(n=-1) == -5 and copy(rows=-1) == -5 and copy(sa=512) == -5
    for bad in ([-1, 2, 64], [1, -2, 64], [1, 2, -16], [1, 2, 272]):
        assert copy(p=np.array([[1, 2, 64], bad], np.int32)) == -5
    put = lambda k=4096, v=4096, pool=4096, slots=4096, n=3, h=2, b=256, p=64, s=4096: L.tq_put_tokens(k, v, 512, 256, 512, 256, pool, s, 2048, slots, n, h, b, p, None)  # noqa: E731
    assert put(n=0) == 0 and put(k=None) == -1 and put(v=None) == -1 and put(pool=None) == -1 and put(slots=None) == -1
    assert put(k=4097) == -8 and put(slots=4098) == -8 and put(n=-1) == -5 and put(p=48) == -5 and put(p=0) == -5 and put(b=1 << 20) == -5 and put(s=-1) == -5


def test_choice_checks_its_arguments(pkg):
    native = pkg._native
    L = native.lib()
    need = L.tq_beam_scratch(2, 4, 1000, 8)
    assert need > 0
    for bad in ((-1, 4, 1000, 8), (2, -1, 1000, 8), (2, 4, -1, 8), (2, 4, 1000, -1), (2, 1025, 10, 8), (2, 4, 1000, 65), (2, 2, 3, 7), (1, 1024, 1 << 22, 8), (1 << 32, 4, 10, 4)):
        assert L.tq_beam_scratch(*bad) == -5, bad
    call = lambda dtype=2, B=2, K=4, V=1000, n=8, ptrs=(4096,) * 6, size=need: L.tq_beam_select(ptrs[0], dtype, B, K, V, K * V, V, ptrs[1], K, n, ptrs[2], ptrs[3], ptrs[4], ptrs[5], size, None)  # noqa: E731
    assert call(dtype=3) == -4 and call(n=65) == -5 and call(B=0) == 0 and call(n=0) == 0 and call(size=need - 1) == -10
    for i in range(6):
        ptrs = [4096] * 6
        ptrs[i] = None
        assert call(ptrs=ptrs) == -1
        ptrs[i] = 4097
        assert call(ptrs=ptrs) == -8
    with pytest.raises(native.TqError, match="HIP device"):
        pkg.beam_select(torch.zeros(1, 2, 3), torch.zeros(1, 2))


def test_page_numbers(pkg):
    from importlib import import_module
    pages = import_module("turboquant-pytorch_amd.paged_cache")._Pages(4)
    assert [pages.take() for _ in range(3)] == [0, 1, 2]
    pages.held[1] += 1
    assert not pages.drop(1) and pages.drop(0) and pages.drop(1) and pages.take() == 0 and pages.take() == 1 and pages.take() == 3 and not pages.free
