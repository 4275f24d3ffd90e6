"""Operators of generation over a compressed key/value store, as cases to be timed:

  chunk    PagedV3Cache.step(...).attend: new tokens of sequences of different lengths, one or many each, over packed pages and the uncompressed
           ones behind them; scores plain, capped by a tanh, with a bias by distance, or within a sliding window
  fork     PagedV3Cache.fork: sequences continued twice, whole pages shared, pages that are still filled copied
  resize   PagedV3Cache.resize: the pages in use gathered into a pool of another size
  beam     beam_select: of beams x vocabulary the best continuations by summed log probability
  reorder  V3Cache.reorder: the states of every layer follow the beams that were chosen

With `own` false, `run` computes them in elementary torch operations.
"""
import functools
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda"
PAGE = 64


def listed():
    return [
        # a decode step of one short conversation: latency counts
        {"name": "chunk 1x2k t1", "kind": "chunk", "dtype": "bf16", "seqs": 1, "heads": 8, "q_heads": 32, "tokens": 2048, "new": 1, "chunks": 1, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2, "cap": 0.0, "slopes": False, "sliding": 0},
        # a decode step of 64 conversations of 2 to 16 thousand tokens
        {"name": "chunk 64x16k t1", "kind": "chunk", "dtype": "bf16", "seqs": 64, "heads": 8, "q_heads": 32, "tokens": 16384, "new": 1, "chunks": 64, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2, "cap": 0.0, "slopes": False, "sliding": 0},
        # a chunk of a long prompt, capped scores: the largest
        {"name": "chunk 1x32k t512 cap", "kind": "chunk", "dtype": "bf16", "seqs": 1, "heads": 8, "q_heads": 32, "tokens": 32768, "new": 512, "chunks": 1, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2, "cap": 50.0, "slopes": False, "sliding": 0},
        # four prompts' chunks among twelve conversations, a sliding window, 64-wide heads
        {"name": "chunk 16x8k t256+1 d64", "kind": "chunk", "dtype": "f16", "seqs": 16, "heads": 8, "q_heads": 32, "tokens": 8191, "new": 256, "chunks": 4, "window": 128, "dim": 64, "key_bits": 6, "value_bits": 4, "cap": 0.0, "slopes": False, "sliding": 4096},
        # float32 states, a head dimension that is no multiple of 32, a bias by distance, odd counts
        {"name": "chunk 3x1003 t77 d80 f32", "kind": "chunk", "dtype": "f32", "seqs": 3, "heads": 8, "q_heads": 8, "tokens": 1003, "new": 77, "chunks": 3, "window": 128, "dim": 80, "key_bits": 4, "value_bits": 4, "cap": 0.0, "slopes": True, "sliding": 0},
        # eight sequences become beams
        {"name": "fork 8 t37", "kind": "fork", "dtype": "bf16", "seqs": 8, "copies": 3, "layers": 8, "heads": 8, "filled": 37, "dim": 128, "key_bits": 4, "value_bits": 2},
        # a cache that has become sparse: every other page is in use
        {"name": "resize 1024", "kind": "resize", "dtype": "bf16", "pages": 2048, "used": 1024, "layers": 16, "heads": 8, "dim": 128, "key_bits": 4, "value_bits": 2},
        # four beams of one sequence: latency counts
        {"name": "beam 1x4 32000", "kind": "beam", "dtype": "bf16", "batch": 1, "beams": 4, "vocab": 32000, "best": 8},
        # sixteen sequences, a large vocabulary, float32 logits
        {"name": "beam 16x8 128256 f32", "kind": "beam", "dtype": "f32", "batch": 16, "beams": 8, "vocab": 128256, "best": 16},
        # an odd vocabulary: rows that begin anywhere
        {"name": "beam 6x5 50257 f16", "kind": "beam", "dtype": "f16", "batch": 6, "beams": 5, "vocab": 50257, "best": 10},
        # four beams over a short conversation
        {"name": "reorder 1x4 1k", "kind": "reorder", "dtype": "bf16", "batch": 1, "beams": 4, "layers": 8, "heads": 8, "tokens": 1024, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2},
        # eight sequences of four beams, an odd length, 64-wide heads
        {"name": "reorder 8x4 8191 d64", "kind": "reorder", "dtype": "f16", "batch": 8, "beams": 4, "layers": 8, "heads": 8, "tokens": 8191, "window": 64, "dim": 64, "key_bits": 6, "value_bits": 4},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    kind = rng.choice(("chunk", "chunk", "chunk", "fork", "resize", "beam", "beam", "reorder"))
    if kind == "beam":
        c = {"kind": kind, "dtype": rng.choice(("bf16", "f16", "f32")), "batch": _spread(rng, 1, 32), "beams": rng.choice((1, 2, 3, 4, 5, 8, 16))}
        c["vocab"] = _spread(rng, 1000, min(262144, 16 * 8 * 128256 // (c["batch"] * c["beams"])))
        c["best"] = c["beams"] * rng.choice((1, 2, 2))
        return c
    key_bits, value_bits = rng.choice(((4, 2), (4, 2), (4, 4), (6, 4), (8, 4), (3, 2), (8, 8)))
    c = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")), "heads": rng.choice((1, 2, 4, 8, 8)), "dim": rng.choice((64, 80, 96, 128, 128, 128, 256)),
         "key_bits": key_bits, "value_bits": value_bits}
    if kind == "chunk":
        group = rng.choice((1, 2, 4, 4, 7, 8))
        c["seqs"] = _spread(rng, 1, 64)
        c["q_heads"] = c["heads"] * group
        c["new"] = rng.choice((1, 1, _spread(rng, 2, 512), _spread(rng, 2, 512)))
        c["chunks"] = c["seqs"] if c["new"] == 1 else rng.randint(1, c["seqs"])
        # (query, key) pairs no more than the largest listed case has, and no more than 2^20 tokens in all
        queries = c["q_heads"] * (c["new"] * c["chunks"] + c["seqs"] - c["chunks"])
        c["tokens"] = max(c["new"], _spread(rng, 64, max(65, min(32768, (1 << 20) // c["seqs"], 32 * 512 * 32768 // queries))))
        c.update(window=rng.choice((0, 17, 64, 128, 128)), cap=rng.choice((0.0, 0.0, 30.0, 50.0)), slopes=rng.random() < 0.25,
                 sliding=rng.choice((0, 0, _spread(rng, 16, 8192))))
        return c
    if kind == "fork":
        c.update(seqs=_spread(rng, 1, 64), copies=rng.randint(1, 3), layers=rng.choice((4, 8, 16)), filled=rng.randint(1, PAGE - 1))
        return c
    if kind == "resize":
        c["layers"] = rng.choice((4, 8, 16))
        c["used"] = max(1, min(_spread(rng, 4, 1024), 1024 * 32 * 8 * 128 // (c["layers"] * c["heads"] * c["dim"] * 3)))
        c["pages"] = c["used"] + rng.randint(0, c["used"])
        return c
    c.update(batch=_spread(rng, 1, 16), beams=rng.choice((2, 3, 4, 5, 8)), layers=rng.choice((2, 4, 8)), window=rng.choice((0, 17, 64, 128)))
    c["tokens"] = max(16, _spread(rng, 1 << 8, 1 << 17) // (c["batch"] * c["beams"]))
    return c


# ---- the codec: rotation and codebook of a head dimension, as its definition has them --------------------------------------
@functools.lru_cache(maxsize=None)
def _rotation(dim, seed):
    """Orthogonal factor of a Gaussian matrix, its columns turned so that the other factor's diagonal is positive."""
    g = torch.Generator()
    g.manual_seed(seed)
    q, r = torch.linalg.qr(torch.randn(dim, dim, generator=g))
    return (q * torch.where(torch.diagonal(r) < 0, -1.0, 1.0)).contiguous()


@functools.lru_cache(maxsize=None)
def _codebook(dim, bits):
    """Lloyd-Max levels of N(0, 1/dim): each the mean of the density between the midpoints around it."""
    levels = 1 << bits
    c = np.linspace(-3.0, 3.0, levels + 1)
    c = (c[:-1] + c[1:]) / 2
    erf = np.vectorize(math.erf)
    for _ in range(60):
        edges = np.concatenate(([-12.0], (c[:-1] + c[1:]) / 2, [12.0]))
        mass = np.diff(erf(edges / math.sqrt(2.0))) / 2
        c = -np.diff(np.exp(-edges ** 2 / 2)) / math.sqrt(2 * math.pi) / np.maximum(mass, 1e-30)
    return torch.tensor(c / math.sqrt(dim), dtype=torch.float32)


def _pages(g, pages, case, bits):
    """Pages of codes of rotated unit vectors, most significant code of a byte first, and norms, tokens spread over a factor of four."""
    shape, dim, ipb = (pages, case["heads"], PAGE), case["dim"], 8 // bits
    levels = _codebook(dim, bits)
    edges = ((levels[:-1] + levels[1:]) / 2).to(DEVICE)
    width = -(-dim // ipb)
    out = torch.empty(shape + (width,), dtype=torch.uint8, device=DEVICE)
    place = torch.arange(ipb - 1, -1, -1, device=DEVICE, dtype=torch.int32) * bits
    for lo in range(0, pages, 256):
        part = (min(256, pages - lo),) + shape[1:]
        codes = torch.zeros(part + (width * ipb,), dtype=torch.int32, device=DEVICE)
        codes[..., :dim] = torch.bucketize(torch.randn(part + (dim,), generator=g, device=DEVICE) / math.sqrt(dim), edges, out_int32=True)
        out[lo:lo + 256] = (codes.view(part + (width, ipb)) << place).sum(-1).to(torch.uint8)
    norms = 2.0 * math.sqrt(dim) * torch.exp(0.2 * torch.randn(shape, generator=g, device=DEVICE)) * (0.5 + 1.5 * torch.rand(shape, generator=g, device=DEVICE))
    return {"idx": out, "norms": norms.to(torch.float16), "Pi": _rotation(dim, 1000 + bits).to(DEVICE), "levels": levels.to(DEVICE), "bits": bits}


def _states(g, shape, dtype):
    return (2.0 * torch.randn(shape, generator=g, device=DEVICE) * (0.5 + 1.5 * torch.rand(shape[:-1] + (1,), generator=g, device=DEVICE))).to(dtype)


def _layout(case):
    """Of every sequence: tokens in all, new ones among them, and packed ones (whole pages of what is older than the window)."""
    rng = random.Random(case["tokens"] * 64 + case["seqs"])
    out = []
    for b in range(case["seqs"]):
        new = case["new"] if b < case["chunks"] else 1
        total = max(new, case["tokens"] if b == 0 else _spread(rng, max(1, case["tokens"] // 8), case["tokens"]))
        out.append((total, new, max(0, total - new - case["window"]) // PAGE * PAGE))
    return out


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], dtype=torch.float32, device=DEVICE)


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _chunk_inputs(c, seed):
    g, rng, dtype = _generator(seed), random.Random(seed), DTYPES[c["dtype"]]
    plan = _layout(c)
    pages, plain = sum(p // PAGE for _, _, p in plan), [-(-(t - p) // PAGE) for t, _, p in plan]
    x = {"kind": "chunk", "plan": plan, "k": _pages(g, max(pages, 1), c, c["key_bits"]), "v": _pages(g, max(pages, 1), c, c["value_bits"])}
    x["k_plain"], x["v_plain"] = (_states(g, (sum(plain), c["heads"], PAGE, c["dim"]), dtype) for _ in range(2))
    # a cache that has been used for a while: a sequence's pages lie anywhere
    order, order_plain = list(range(pages)), list(range(sum(plain)))
    rng.shuffle(order)
    rng.shuffle(order_plain)
    on_card = lambda ids: torch.tensor(ids, dtype=torch.int64, device=DEVICE)  # noqa: E731
    x["tables"] = [(on_card([order.pop() for _ in range(p // PAGE)]), on_card([order_plain.pop() for _ in range(n)])) for (_, _, p), n in zip(plan, plain)]
    x["q"] = torch.randn((sum(n for _, n, _ in plan), c["q_heads"], c["dim"]), generator=g, device=DEVICE).to(dtype)
    x["cap"], x["sliding"] = c["cap"], c["sliding"]
    x["slopes"] = _slopes(c["q_heads"]) if c["slopes"] else None
    return x


def _pool_inputs(c, seed):
    """A whole cache's pages, [pages, layers, ..]: raw bytes of packed pages are as good as codes to what copies them."""
    g, dtype = _generator(seed), DTYPES[c["dtype"]]
    if c["kind"] == "fork":
        filled = torch.randn((c["seqs"], c["layers"], 2, c["heads"], PAGE, c["dim"]), generator=g, device=DEVICE).to(dtype)
        pages = torch.arange(c["seqs"] * (1 + c["copies"]), device=DEVICE)
        return {"kind": "fork", "plain": torch.cat((filled, torch.zeros_like(filled).repeat(c["copies"], 1, 1, 1, 1, 1))), "filled": c["filled"],
                "source": pages[:c["seqs"]].repeat(c["copies"]), "target": pages[c["seqs"]:]}
    shape = (c["pages"], c["layers"], c["heads"], PAGE)
    x = {"kind": "resize"}
    for name, bits in (("k", c["key_bits"]), ("v", c["value_bits"])):
        x[name + "_idx"] = torch.randint(0, 256, shape + (-(-c["dim"] // (8 // bits)),), dtype=torch.uint8, generator=g, device=DEVICE)
        x[name + "_nrm"] = torch.rand(shape, generator=g, device=DEVICE).to(torch.float16)
    x["used"] = torch.tensor(sorted(random.Random(seed).sample(range(c["pages"]), c["used"])), device=DEVICE)
    x["all"] = torch.arange(c["used"], device=DEVICE)
    return x


def _beam_inputs(c, seed):
    g = _generator(seed)
    # a few likely tokens, a long tail; the sums of log probabilities of beams that have come the same way
    logits = 2.5 * torch.randn((c["batch"], c["beams"], c["vocab"]), generator=g, device=DEVICE) + 1.5 * torch.randn((1, 1, c["vocab"]), generator=g, device=DEVICE)
    return {"kind": "beam", "logits": logits.to(DTYPES[c["dtype"]]), "scores": -20.0 + 1.5 * torch.randn((c["batch"], c["beams"]), generator=g, device=DEVICE), "best": c["best"]}


def _parents(c, seed):
    """Of each sequence's beams half go on from another one, the others from themselves."""
    rng, out = random.Random(seed), []
    for b in range(c["batch"]):
        beams = list(range(c["beams"]))
        moved = set(rng.sample(beams, (c["beams"] + 1) // 2))
        out += [b * c["beams"] + (rng.choice([j for j in beams if j != i]) if i in moved else i) for i in beams]
    return out


def _reorder_inputs(c, seed):
    g, rows, dtype = _generator(seed), c["batch"] * c["beams"], DTYPES[c["dtype"]]
    x = {"kind": "reorder", "layers": [], "parents": torch.tensor(_parents(c, seed), dtype=torch.int64, device=DEVICE)}
    for _ in range(c["layers"]):
        shape, window = (rows, c["heads"], c["tokens"]), (rows, c["heads"], c["window"], c["dim"])
        idx = [torch.randint(0, 256, shape + (-(-c["dim"] // (8 // b)),), dtype=torch.uint8, generator=g, device=DEVICE) for b in (c["key_bits"], c["value_bits"])]
        nrm = [torch.rand(shape, generator=g, device=DEVICE).to(torch.float16) for _ in range(2)]
        x["layers"].append([idx[0], nrm[0], idx[1], nrm[1]] + [torch.randn(window, generator=g, device=DEVICE).to(dtype) for _ in range(2)])
    return x


def _inputs(case, seed):
    return {"chunk": _chunk_inputs, "fork": _pool_inputs, "resize": _pool_inputs, "beam": _beam_inputs, "reorder": _reorder_inputs}[case["kind"]](case, seed)


def prepare(case, seed):
    c, x = case, _inputs(case, seed)
    if not own or c["kind"] == "beam":
        return x
    import turboquant_amd as tq

    if c["kind"] == "reorder":
        cache = tq.V3Cache(key_bits=c["key_bits"], value_bits=c["value_bits"], residual_window=c["window"], n_layers=c["layers"], capacity=c["tokens"])
        n = c["tokens"]
        blank = torch.zeros((c["batch"] * c["beams"], c["heads"], n + c["window"], c["dim"]), dtype=DTYPES[c["dtype"]], device=DEVICE)
        x["views"] = []
        for i, tensors in enumerate(x.pop("layers")):
            cache.append(blank, blank, i)
            st = cache._stores[i]
            views = [t[:, :, :n] for t in (st.k_idx, st.k_nrm, st.v_idx, st.v_nrm)] + list(st.window())
            for view, t in zip(views, tensors):
                view.copy_(t)
            x["views"].append(views)
        x["cache"] = cache
        return x
    common = dict(head_dim=c["dim"], kv_heads=c["heads"], key_bits=c["key_bits"], value_bits=c["value_bits"], dtype=DTYPES[c["dtype"]], device=DEVICE, page_tokens=PAGE)
    if c["kind"] == "fork":
        count = x["plain"].shape[0]
        cache = tq.PagedV3Cache(pages=1, plain_pages=count, n_layers=c["layers"], residual_window=128, **common)
        seqs = cache.add(c["seqs"])
        cache.place(seqs, [0] * len(seqs), [c["filled"]] * len(seqs))
        cache.plain_pages().copy_(x.pop("plain"))
        return {"kind": "fork", "cache": cache, "seqs": seqs, "copies": c["copies"], "filled": c["filled"], "forks": []}
    if c["kind"] == "resize":
        cache = tq.PagedV3Cache(pages=c["pages"], plain_pages=1, n_layers=c["layers"], residual_window=0, **common)
        # every page is a sequence's; those of which the page is not in use end
        seqs = cache.add(c["pages"])
        cache.place(seqs, [PAGE] * len(seqs), [0] * len(seqs))
        for i in range(c["layers"]):
            for view, name in zip(cache.packed_pages(i), ("k_idx", "k_nrm", "v_idx", "v_nrm")):
                view.copy_(x[name][:, i])
        used = set(x["used"].tolist())
        cache.free([s for i, s in enumerate(seqs) if i not in used])
        return {"kind": "resize", "cache": cache, "layers": c["layers"]}
    pages, plain = (sum(len(t[i]) for t in x["tables"]) for i in (0, 1))
    cache = tq.PagedV3Cache(pages=max(pages, 1), plain_pages=plain, n_layers=1, residual_window=c["window"], **common)
    codec = cache.codec(0)
    codec.key_compressor, codec.val_compressor = (tq.MSECompressor.from_tensors(p["Pi"], p["levels"], p["bits"], device=DEVICE) for p in (x["k"], x["v"]))
    seqs = cache.add(c["seqs"])
    # (the step's own tokens are placed by it)
    before = [total - new for total, new, _ in x["plan"]]
    cache.place(seqs, [p for _, _, p in x["plan"]], [b - p for b, (_, _, p) in zip(before, x["plan"])])
    step = cache.step(seqs, [new for _, new, _ in x["plan"]])
    views, plain_views = cache.packed_pages(0), cache.plain_pages()[:, 0]
    for s, (table, plain_table) in zip(seqs, x["tables"]):
        ids, plain_ids = (torch.tensor(t, dtype=torch.int64, device=DEVICE) for t in cache.tables(s))
        for view, t in zip(views, (x["k"]["idx"], x["k"]["norms"], x["v"]["idx"], x["v"]["norms"])):
            view[ids] = t[table]
        plain_views[plain_ids, 0] = x["k_plain"][plain_table]
        plain_views[plain_ids, 1] = x["v_plain"][plain_table]
    return {"kind": "chunk", "cache": cache, "step": step, "q": x["q"], "cap": x["cap"], "sliding": x["sliding"], "slopes": x["slopes"]}


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _restored(p, table):
    """norm * (levels[codes] @ Pi) of a sequence's pages, float32 [H, tokens, dim]."""
    bits, ipb, dim = p["bits"], 8 // p["bits"], p["Pi"].shape[0]
    place = torch.arange(ipb - 1, -1, -1, device=DEVICE, dtype=torch.int32) * bits
    idx, norms = p["idx"][table].transpose(0, 1).flatten(1, 2), p["norms"][table].transpose(0, 1).flatten(1, 2)
    codes = (idx.to(torch.int32).unsqueeze(-1) >> place) & ((1 << bits) - 1)
    return norms.float().unsqueeze(-1) * (p["levels"][codes.flatten(-2)[..., :dim]] @ p["Pi"])


def _chunk(x):
    out, at = torch.empty_like(x["q"]), 0
    for (total, new, packed), (table, plain_table) in zip(x["plan"], x["tables"]):
        plain = lambda t: t[plain_table].transpose(0, 1).flatten(1, 2)[:, :total - packed].float()  # noqa: E731
        k, v = torch.cat((_restored(x["k"], table), plain(x["k_plain"])), 1), torch.cat((_restored(x["v"], table), plain(x["v_plain"])), 1)
        H, (Hq, D) = k.shape[0], x["q"].shape[1:]
        q = x["q"][at:at + new].float().transpose(0, 1).reshape(H, Hq // H * new, D)
        z = (q @ k.transpose(-2, -1)).reshape(Hq, new, total) * D ** -0.5
        if x["cap"]:
            z = x["cap"] * torch.tanh(z / x["cap"])
        distance = torch.arange(total - new, total, device=DEVICE).unsqueeze(1) - torch.arange(total, device=DEVICE)
        if x["slopes"] is not None:
            z = z - x["slopes"].view(Hq, 1, 1) * distance
        seen = distance >= 0
        if x["sliding"]:
            seen = seen & (distance < x["sliding"])
        z = torch.where(seen, z, float("-inf"))
        e = torch.exp(z - z.amax(-1, keepdim=True))
        probs = e / e.sum(-1, keepdim=True)
        out[at:at + new] = (probs.reshape(H, -1, total) @ v).reshape(Hq, new, D).transpose(0, 1).to(out.dtype)
        at += new
    return out


def run(state):
    x, kind = state, state["kind"]
    if kind == "chunk":
        if own:
            return x["step"].attend(x["q"], 0, softcap=x["cap"] or None, slopes=x["slopes"], sliding_window=x["sliding"] or None)
        return _chunk(x)
    if kind == "fork":
        if own:
            cache = x["cache"]
            cache.free(x["forks"])                # those of the pass before
            x["forks"] = cache.fork(x["seqs"] * x["copies"])
            return cache.plain_pages()[..., :x["filled"], :]
        part = x["plain"][..., :x["filled"], :]
        part[x["target"]] = part[x["source"]]
        return part
    if kind == "resize":
        if own:
            x["cache"].resize()
            return [x["cache"].packed_pages(i) for i in range(x["layers"])]
        # (gathered pages lie in order: what comes next takes them as they are)
        for name in ("k_idx", "k_nrm", "v_idx", "v_nrm"):
            x[name] = x[name][x["used"]]
        x["used"] = x["all"]
        return [tuple(x[name][:, i] for name in ("k_idx", "k_nrm", "v_idx", "v_nrm")) for i in range(x["k_idx"].shape[1])]
    if kind == "beam":
        if own:
            import turboquant_amd as tq

            return tq.beam_select(x["logits"], x["scores"], x["best"])
        logits, vocab = x["logits"].double(), x["logits"].shape[-1]
        top = logits.amax(-1, keepdim=True)
        sums = x["scores"].double().unsqueeze(-1) + (logits - (top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True))))
        values, order = torch.sort(sums.flatten(1), dim=-1, descending=True, stable=True)
        order = order[:, :x["best"]]
        return values[:, :x["best"]].float(), order % vocab, order // vocab
    if own:
        x["cache"].reorder(x["parents"])
        return x["views"]
    for tensors in x["layers"]:
        for t in tensors:
            t.copy_(t[x["parents"]])
    return x["layers"]


def exact(case, seed):
    """The same in float64: attention from the codes, queries turned into the codec's space and sums of levels turned back out of it, a kv head at a time."""
    x, c = _inputs(case, seed), case
    if c["kind"] == "fork":
        pool = x["plain"].double()[..., :c["filled"], :]
        return torch.cat([pool[:c["seqs"]]] * (1 + c["copies"]))
    if c["kind"] == "resize":
        kept = x["used"]
        wide = lambda t: t.double() if t.dtype == torch.float16 else t  # noqa: E731
        return [tuple(wide(torch.index_select(x[name][:, i], 0, kept)) for name in ("k_idx", "k_nrm", "v_idx", "v_nrm")) for i in range(c["layers"])]
    if c["kind"] == "reorder":
        rows = x["parents"].tolist()
        return [[torch.stack([t[r] for r in rows]) if t.dtype == torch.uint8 else torch.stack([t[r].double() for r in rows]) for t in layer] for layer in x["layers"]]
    if c["kind"] == "beam":
        logits, scores, best, vocab = x["logits"].double().cpu().numpy(), x["scores"].double().cpu().numpy(), c["best"], c["vocab"]
        values, tokens, parents = [], [], []
        for b in range(c["batch"]):
            rows = []
            for k in range(c["beams"]):
                largest = logits[b, k].max()
                rows.append(logits[b, k] - largest + (scores[b, k] - math.log(math.fsum(np.exp(logits[b, k] - largest)))))
            flat = np.concatenate(rows)
            among = np.flatnonzero(flat >= np.partition(flat, -best)[-best])
            order = among[np.argsort(-flat[among], kind="stable")][:best]
            values.append(flat[order])
            tokens.append(order % vocab)
            parents.append(order // vocab)
        return tuple(torch.from_numpy(np.stack(t)).to(DEVICE) for t in (values, tokens, parents))
    dim, wide, H = c["dim"], torch.float64, c["heads"]
    group, at = c["q_heads"] // H, 0
    out = torch.zeros(x["q"].shape, dtype=wide, device=DEVICE)

    def levels(p, table, h):
        mask, ipb = (1 << p["bits"]) - 1, 8 // p["bits"]
        raw = p["idx"][table, h].flatten(0, 1).long()
        codes = torch.stack([(raw >> (p["bits"] * (ipb - 1 - i))) & mask for i in range(ipb)], -1).flatten(1)[:, :dim]
        return p["levels"].to(wide)[codes], p["norms"][table, h].flatten().to(wide)

    for (total, new, packed), (table, plain_table) in zip(x["plan"], x["tables"]):
        where = torch.arange(total, device=DEVICE)
        own_place = where[total - new:].repeat(group)                     # of query g * new + i
        first = own_place - c["sliding"] + 1 if c["sliding"] else torch.zeros_like(own_place)
        for h in range(H):
            heads = slice(h * group, (h + 1) * group)
            mine = x["q"][at:at + new, heads].to(wide).transpose(0, 1).reshape(group * new, dim) / math.sqrt(dim)
            k_levels, k_norms = levels(x["k"], table, h)
            v_levels, v_norms = levels(x["v"], table, h)
            k_plain, v_plain = (x[n][plain_table, h].flatten(0, 1)[:total - packed].to(wide) for n in ("k_plain", "v_plain"))
            logits = torch.cat(((mine @ x["k"]["Pi"].to(wide).T @ k_levels.T) * k_norms, mine @ k_plain.T), 1)
            if c["cap"]:
                logits = c["cap"] * torch.tanh(logits / c["cap"])
            if c["slopes"]:
                logits += _slopes(c["q_heads"])[heads].to(wide).repeat_interleave(new).unsqueeze(1) * (where - own_place.unsqueeze(1))
            logits.masked_fill_((where > own_place.unsqueeze(1)) | (where < first.unsqueeze(1)), -math.inf)
            probs = torch.softmax(logits, 1)
            result = (probs[:, :packed] * v_norms) @ v_levels @ x["v"]["Pi"].to(wide) + probs[:, packed:] @ v_plain
            out[at:at + new, heads] = result.reshape(group, new, dim).transpose(0, 1)
        at += new
    return out


def work(case):
    """Every packed token, uncompressed token, query and result crosses memory once, what is copied twice; attention is its two products over the keys that are seen."""
    c = case
    if c["kind"] == "beam":
        n, elem = c["batch"] * c["beams"] * c["vocab"], 4 if c["dtype"] == "f32" else 2
        return {"bytes": n * elem + 4 * c["batch"] * c["beams"] + 20 * c["batch"] * c["best"], "flops": 4 * n}
    elem = 4 if c["dtype"] == "f32" else 2
    both = -(-c["dim"] // (8 // c["key_bits"])) - (-c["dim"] // (8 // c["value_bits"])) + 4
    plain = 2 * c["dim"] * elem
    if c["kind"] == "fork":
        return {"bytes": 2 * c["seqs"] * c["copies"] * c["layers"] * c["heads"] * c["filled"] * plain, "flops": 0}
    if c["kind"] == "resize":
        return {"bytes": 2 * c["used"] * c["layers"] * c["heads"] * PAGE * both, "flops": 0}
    if c["kind"] == "reorder":
        moved = c["batch"] * ((c["beams"] + 1) // 2)
        return {"bytes": 2 * c["layers"] * moved * c["heads"] * (c["tokens"] * both + c["window"] * plain), "flops": 0}
    size, pairs = 0, 0
    for total, new, packed in _layout(c):
        reach = c["sliding"] or total
        first = max(0, total - new + 1 - reach)
        size += c["heads"] * (max(0, packed - first) * both + (total - max(first, packed)) * plain) + new * c["q_heads"] * plain
        pairs += c["q_heads"] * sum(min(reach, at + 1) for at in range(total - new, total))
    return {"bytes": size, "flops": 4 * pairs * c["dim"]}
