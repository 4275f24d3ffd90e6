"""Operators that read or thin out a compressed key/value store, as cases to be timed:

  tree     V3Cache.attend_tree: drafted tokens, each seeing its ancestors among them, over everything cached (verification
           of a draft before any of it is accepted)
  cross    TurboQuantV3.attend_kv: queries over states compressed once (an encoder's), every sequence with a length of its own
  weigh    V3Cache.attend of a cache that keeps the attention each key has received: the output and the sums
  evict    TurboQuantV3.evict_kv: of every (sequence, kv head) the tokens with the largest sums stay

With `own` false, `run` computes them in elementary torch operations in float32.
"""
import functools
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda"


def listed():
    return [
        # a draft of eight tokens over a short conversation: latency counts
        {"name": "tree 1x2k t8", "kind": "tree", "dtype": "bf16", "batch": 1, "heads": 8, "q_heads": 32, "tokens": 2048, "window": 128, "drafts": 8, "dim": 128, "key_bits": 4, "value_bits": 2},
        # a wide draft over a long context, one sequence
        {"name": "tree 1x32k t64", "kind": "tree", "dtype": "bf16", "batch": 1, "heads": 8, "q_heads": 32, "tokens": 32768, "window": 128, "drafts": 64, "dim": 128, "key_bits": 4, "value_bits": 2},
        # sixteen sequences verified together
        {"name": "tree 16x8k t16", "kind": "tree", "dtype": "bf16", "batch": 16, "heads": 8, "q_heads": 32, "tokens": 8192, "window": 128, "drafts": 16, "dim": 128, "key_bits": 4, "value_bits": 2},
        # 64-wide heads, odd sizes, the widths recommended for generation
        {"name": "tree 4x6001 t13 d64", "kind": "tree", "dtype": "f16", "batch": 4, "heads": 8, "q_heads": 32, "tokens": 6001, "window": 128, "drafts": 13, "dim": 64, "key_bits": 6, "value_bits": 4},
        # one decoder step against encoders' states of four lengths
        {"name": "cross 4x1500 q1 d64", "kind": "cross", "dtype": "f16", "batch": 4, "heads": 16, "q_heads": 16, "tokens": 1500, "window": 0, "queries": 1, "dim": 64, "key_bits": 6, "value_bits": 4},
        # a prompt's worth of queries over eight long documents: the largest
        {"name": "cross 8x4k q512", "kind": "cross", "dtype": "bf16", "batch": 8, "heads": 8, "q_heads": 32, "tokens": 4096, "window": 128, "queries": 512, "dim": 128, "key_bits": 4, "value_bits": 4},
        # float32 states, a head dimension that is no multiple of 32, odd counts
        {"name": "cross 2x1003 q77 d80 f32", "kind": "cross", "dtype": "f32", "batch": 2, "heads": 8, "q_heads": 8, "tokens": 1003, "window": 0, "queries": 77, "dim": 80, "key_bits": 4, "value_bits": 4},
        # one long sequence that keeps count of what its keys receive
        {"name": "weigh 1x32k", "kind": "weigh", "dtype": "bf16", "batch": 1, "heads": 8, "q_heads": 32, "tokens": 32768, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2},
        # many sequences
        {"name": "weigh 32x8k", "kind": "weigh", "dtype": "bf16", "batch": 32, "heads": 8, "q_heads": 32, "tokens": 8192, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2},
        # a budget of 1024 tokens that an eighth of it has run over
        {"name": "evict 1x1152", "kind": "evict", "dtype": "bf16", "batch": 1, "heads": 8, "tokens": 1152, "keep": 1024, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2},
        # a long prompt cut to half
        {"name": "evict 1x32k", "kind": "evict", "dtype": "bf16", "batch": 1, "heads": 8, "tokens": 32768, "keep": 16384, "window": 128, "dim": 128, "key_bits": 4, "value_bits": 2},
        # a batch of prompts of an odd length, 64-wide heads
        {"name": "evict 16x8191 d64", "kind": "evict", "dtype": "f16", "batch": 16, "heads": 8, "tokens": 8191, "keep": 4097, "window": 64, "dim": 64, "key_bits": 6, "value_bits": 4},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    kind = rng.choice(("tree", "tree", "cross", "cross", "weigh", "evict"))
    key_bits, value_bits = rng.choice(((4, 2), (4, 2), (4, 4), (6, 4), (8, 4), (3, 2), (8, 8)))
    batch, heads = rng.choice((1, 1, 2, 3, 4, 8, 16)), rng.choice((1, 2, 4, 8, 8))
    group = rng.choice((1, 2, 4, 4, 7, 8))
    c = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")), "batch": batch, "heads": heads, "dim": rng.choice((64, 80, 96, 128, 128, 128, 256)),
         "key_bits": key_bits, "value_bits": value_bits, "window": rng.choice((0, 17, 64, 128, 128))}
    rows = batch * heads
    if kind == "evict":
        c["tokens"] = max(16, _spread(rng, 1 << 13, 1 << 20) // rows)
        c["keep"] = rng.randint(1, c["tokens"] - 1)
        return c
    c["q_heads"] = heads * group
    if kind == "weigh":
        c["tokens"] = max(64, _spread(rng, 1 << 13, 1 << 20) // rows)
        return c
    if kind == "tree":
        c["drafts"] = _spread(rng, 1, 64)
        count, most = c["drafts"], 1 << 20
    else:
        c["queries"] = count = rng.choice((1, 1, _spread(rng, 2, 512)))
        most = 1 << 18
    # (query, key) pairs of a row's group: no more than 2^28 over all rows
    most = max(64 * rows, min(most, (1 << 28) // (count * group)))
    c["tokens"] = max(1, _spread(rng, 64 * rows, most) // rows)
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


def _packed(g, case, bits):
    """Codes of rotated unit vectors, most significant code of a byte first, and norms: those of states with a few outlier channels and
    tokens spread over a factor of four."""
    shape, dim, ipb = (case["batch"], case["heads"], case["tokens"]), case["dim"], 8 // bits
    levels = _codebook(dim, bits)
    edges = ((levels[:-1] + levels[1:]) / 2).to(DEVICE)
    width = -(-dim // ipb)
    out = torch.empty(shape + (width,), dtype=torch.uint8, device=DEVICE)
    for b in range(shape[0]):
        codes = torch.zeros(shape[1:] + (width * ipb,), dtype=torch.int32, device=DEVICE)
        codes[..., :dim] = torch.bucketize(torch.randn(shape[1:] + (dim,), generator=g, device=DEVICE) / math.sqrt(dim), edges, out_int32=True)
        place = torch.arange(ipb - 1, -1, -1, device=DEVICE, dtype=torch.int32) * bits
        out[b] = (codes.view(shape[1:] + (width, ipb)) << place).sum(-1).to(torch.uint8)
    norms = 2.0 * math.sqrt(dim) * torch.exp(0.2 * torch.randn(shape, generator=g, device=DEVICE)) * (0.5 + 1.5 * torch.rand(shape, generator=g, device=DEVICE))
    return {"idx": out, "norms": norms.to(torch.float16), "Pi": _rotation(dim, 1000 + bits).to(DEVICE), "levels": levels.to(DEVICE), "bits": bits}


def _states(g, shape, dtype):
    return (2.0 * torch.randn(shape, generator=g, device=DEVICE) * (0.5 + 1.5 * torch.rand(shape[:-1] + (1,), generator=g, device=DEVICE))).to(dtype)


def _tree(count, seed):
    """Visibility among drafted tokens: each follows an earlier one, or the last cached token, and sees the way back."""
    rng = random.Random(seed)
    seen = []
    for i in range(count):
        parent = rng.randint(max(-1, i - 6), i - 1)
        seen.append((seen[parent] if parent >= 0 else set()) | {i})
    mask = torch.zeros(count, count, dtype=torch.bool)
    for i, s in enumerate(seen):
        mask[i, sorted(s)] = True
    return mask.to(DEVICE)


def _inputs(case, seed):
    c, dtype = case, DTYPES[case["dtype"]]
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    x = {"kind": c["kind"], "k": _packed(g, c, c["key_bits"]), "v": _packed(g, c, c["value_bits"])}
    window = (c["batch"], c["heads"], c["window"], c["dim"])
    x["k_win"], x["v_win"] = _states(g, window, dtype), _states(g, window, dtype)
    total = c["tokens"] + c["window"]
    if c["kind"] in ("weigh", "evict"):
        # what earlier steps have left: few keys hold most of it, many nothing at all
        w = torch.exp(2.0 * torch.randn(window[:2] + (total,), generator=g, device=DEVICE)) * (torch.rand(window[:2] + (total,), generator=g, device=DEVICE) > 0.2)
        if c["kind"] == "weigh":
            w *= 16.0 * c["q_heads"] / c["heads"] / w.sum(-1, keepdim=True)      # sixteen steps' attention
        x["weights"] = w
    if c["kind"] != "evict":
        count = {"tree": c.get("drafts"), "cross": c.get("queries"), "weigh": 1}[c["kind"]]
        x["q"] = torch.randn((c["batch"], c["q_heads"], count, c["dim"]), generator=g, device=DEVICE).to(dtype)
    if c["kind"] == "tree":
        fresh = window[:2] + (c["drafts"], c["dim"])
        x["k_new"], x["v_new"] = _states(g, fresh, dtype), _states(g, fresh, dtype)
        x["tree"] = _tree(c["drafts"], seed)
    if c["kind"] == "cross":
        rng = random.Random(seed)
        x["lengths"] = torch.tensor([total] + [rng.randint(1, total) for _ in range(c["batch"] - 1)], dtype=torch.int32, device=DEVICE)
    if c["kind"] == "evict":
        x["keep"] = c["keep"]
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    if own:
        import turboquant_amd as tq

        codec = tq.TurboQuantV3(case["dim"], key_bits=case["key_bits"], value_bits=case["value_bits"], residual_window=case["window"], protected_layers=0, device=DEVICE)
        codec.key_compressor, codec.val_compressor = (tq.MSECompressor.from_tensors(p["Pi"], p["levels"], p["bits"], device=DEVICE) for p in (x["k"], x["v"]))
        B, H, n, D = case["batch"], case["heads"], case["tokens"], case["dim"]
        if case["kind"] in ("cross", "evict"):
            x["codec"] = codec
            x["ck"], x["cv"] = ({"compressed": {"idx_bytes": p["idx"], "vec_norms": p["norms"], "shape": (B, H, n, D), "idx_pad": -D % (8 // p["bits"])},
                                 "fp16": w, "shape": (B, H, n + case["window"], D), "split_at": n} for p, w in ((x["k"], x["k_win"]), (x["v"], x["v_win"])))
        else:
            # a cache in the middle of a generation: its history set to the codes at hand
            cache = tq.V3Cache(key_bits=case["key_bits"], value_bits=case["value_bits"], residual_window=case["window"], n_layers=1, capacity=n, track_weights=case["kind"] == "weigh")
            cache._compressors[0] = codec
            blank = torch.zeros((B, H, n, D), dtype=x["q"].dtype, device=DEVICE)
            cache.append(torch.cat((blank, x["k_win"]), 2), torch.cat((blank, x["v_win"]), 2), 0)
            store = cache._stores[0]
            for name, p in (("k", x["k"]), ("v", x["v"])):
                getattr(store, name + "_idx")[:, :, :n].copy_(p["idx"])
                getattr(store, name + "_nrm")[:, :, :n].copy_(p["norms"])
            if case["kind"] == "weigh":
                cache.attention_weights(0).copy_(x["weights"])
            x["cache"] = cache
    return x


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _restored(p):
    """norm * (levels[codes] @ Pi), float32."""
    bits, ipb, dim = p["bits"], 8 // p["bits"], p["Pi"].shape[0]
    place = torch.arange(ipb - 1, -1, -1, device=DEVICE, dtype=torch.int32) * bits
    codes = (p["idx"].to(torch.int32).unsqueeze(-1) >> place) & ((1 << bits) - 1)
    unit = p["levels"][codes.flatten(-2)[..., :dim]]
    return p["norms"].float().unsqueeze(-1) * (unit @ p["Pi"])


def _attention(q, k, v, visible):
    """softmax(q k^T / sqrt(dim)) v where visible, and its weights [B, kv heads, group, queries, keys]; a row that sees nothing is zero."""
    B, Hq, T, D = q.shape
    H, S = k.shape[1], k.shape[2]
    scores = (q.float().reshape(B, H, (Hq // H) * T, D) @ k.transpose(-2, -1)).reshape(B, H, Hq // H, T, S) * D ** -0.5
    if visible is not None:
        scores = torch.where(visible, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    probs = e / torch.where(total == 0, 1.0, total)
    return (probs.reshape(B, H, -1, S) @ v).reshape(B, Hq, T, D).to(q.dtype), probs


def run(state):
    x, kind = state, state["kind"]
    if own:
        if kind == "tree":
            return x["cache"].attend_tree(x["q"], x["k_new"], x["v_new"], 0, x["tree"])
        if kind == "cross":
            return x["codec"].attend_kv(x["q"], x["ck"], x["cv"], lengths=x["lengths"])
        if kind == "weigh":
            return x["cache"].attend(x["q"], 0), x["cache"].attention_weights(0)
        k, v, weights, kept = x["codec"].evict_kv(x["ck"], x["cv"], x["weights"], x["keep"])
        k, v = k["compressed"], v["compressed"]
        return kept, k["idx_bytes"], k["vec_norms"], v["idx_bytes"], v["vec_norms"], weights
    if kind == "evict":
        n, keep = x["k"]["idx"].shape[2], x["keep"]
        order = torch.sort(x["weights"][:, :, :n], dim=-1, descending=True, stable=True).indices
        kept = torch.sort(order[:, :, :keep], dim=-1).values
        taken = lambda t: torch.take_along_dim(t, kept.unsqueeze(-1) if t.dim() == 4 else kept, 2)  # noqa: E731
        weights = torch.cat((taken(x["weights"][:, :, :n]), x["weights"][:, :, n:]), 2)
        return kept, taken(x["k"]["idx"]), taken(x["k"]["norms"]), taken(x["v"]["idx"]), taken(x["v"]["norms"]), weights
    k, v = torch.cat((_restored(x["k"]), x["k_win"].float()), 2), torch.cat((_restored(x["v"]), x["v_win"].float()), 2)
    if kind == "weigh":
        out, probs = _attention(x["q"], k, v, None)
        x["weights"] += probs.sum((2, 3))
        return out, x["weights"]
    if kind == "cross":
        visible = torch.arange(k.shape[2], device=DEVICE) < x["lengths"].view(-1, 1, 1, 1, 1)
        return _attention(x["q"], k, v, visible)[0]
    k, v = torch.cat((k, x["k_new"].float()), 2), torch.cat((v, x["v_new"].float()), 2)
    T = x["tree"].shape[0]
    visible = torch.cat((x["tree"].new_ones(T, k.shape[2] - T), x["tree"]), 1)
    return _attention(x["q"], k, v, visible)[0]


def exact(case, seed):
    """The same in float64, from the codes: queries turned into the codec's space and sums of levels turned back out of it, a kv head at a time."""
    x = _inputs(case, seed)
    B, H, n = x["k"]["norms"].shape
    if case["kind"] == "evict":
        w = x["weights"].cpu().numpy()
        rank = np.argsort(-w[:, :, :n].astype(np.float64), axis=-1, kind="stable")
        kept = torch.from_numpy(np.sort(rank[:, :, :x["keep"]], axis=-1)).to(DEVICE)
        rows = kept.reshape(B * H, -1)
        pick = lambda t: torch.stack([r[i] for r, i in zip(t.flatten(0, 1), rows)]).unflatten(0, (B, H))  # noqa: E731
        weights = torch.cat((pick(x["weights"][:, :, :n]), x["weights"][:, :, n:]), 2).double()
        return kept, pick(x["k"]["idx"]), pick(x["k"]["norms"]).double(), pick(x["v"]["idx"]), pick(x["v"]["norms"]).double(), weights
    dim, wide = case["dim"], torch.float64
    q = x["q"].to(wide)
    T, group = q.shape[2], q.shape[1] // H
    out = torch.zeros_like(q)
    weights = x["weights"].to(wide) if case["kind"] == "weigh" else None

    def levels(p, b, h):
        mask, ipb = (1 << p["bits"]) - 1, 8 // p["bits"]
        raw = p["idx"][b, h].long()
        codes = torch.stack([(raw >> (p["bits"] * (ipb - 1 - i))) & mask for i in range(ipb)], -1).reshape(n, -1)[:, :dim]
        return p["levels"].to(wide)[codes]

    for b in range(B):
        for h in range(H):
            mine = q[b, h * group:(h + 1) * group].reshape(group * T, dim) / math.sqrt(dim)
            turned = mine @ x["k"]["Pi"].to(wide).T
            logits = [(turned @ levels(x["k"], b, h).T) * x["k"]["norms"][b, h].to(wide), mine @ x["k_win"][b, h].to(wide).T]
            plain = [x["v_win"][b, h].to(wide)]
            if case["kind"] == "tree":
                fresh = (mine @ x["k_new"][b, h].to(wide).T).reshape(group, T, T).masked_fill(~x["tree"], -math.inf)
                logits.append(fresh.reshape(group * T, T))
                plain.append(x["v_new"][b, h].to(wide))
            logits = torch.cat(logits, 1)
            if case["kind"] == "cross":
                logits[:, int(x["lengths"][b]):] = -math.inf
            probs = torch.softmax(logits, 1)
            turned_back = (probs[:, :n] * x["v"]["norms"][b, h].to(wide)) @ levels(x["v"], b, h) @ x["v"]["Pi"].to(wide)
            out[b, h * group:(h + 1) * group] = (turned_back + probs[:, n:] @ torch.cat(plain)).reshape(group, T, dim)
            if weights is not None:
                weights[b, h] += probs.sum(0)
    return (out, weights) if weights is not None else out


def work(case):
    """Every packed token, uncompressed token, query and result crosses memory once; attention is its two products."""
    c, rows = case, case["batch"] * case["heads"]
    elem = 4 if c["dtype"] == "f32" else 2
    both = -(-c["dim"] // (8 // c["key_bits"])) - (-c["dim"] // (8 // c["value_bits"])) + 4
    if c["kind"] == "evict":
        return {"bytes": rows * (4 * (c["tokens"] + c["window"]) + c["keep"] * (2 * both + 8 + 8) + 4 * c["window"]), "flops": rows * c["tokens"]}
    count = {"tree": c.get("drafts"), "cross": c.get("queries"), "weigh": 1}[c["kind"]]
    plain = c["window"] + (count if c["kind"] == "tree" else 0)
    # (encoders' states: half of the others' longest length on average)
    share = (c["batch"] + 1) / (2 * c["batch"]) if c["kind"] == "cross" else 1.0
    queries = c["batch"] * c["q_heads"] * count
    keys = share * (c["tokens"] + plain)
    sums = 8 * rows * (c["tokens"] + c["window"]) if c["kind"] == "weigh" else 0
    return {"bytes": int(rows * share * (c["tokens"] * both + plain * 2 * c["dim"] * elem) + 2 * queries * c["dim"] * elem + sums), "flops": 4.0 * queries * keys * c["dim"]}
