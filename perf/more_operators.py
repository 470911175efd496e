"""From the QKV product to the attention's output over a 4-bit K/V cache, as calls that can be timed
and checked.

The cache holds blocks of 64 tokens: e2m1 codes, for K with one power-of-two scale for each token, KV
head and 32 channels, for V with one for each token and KV head.  Five operators, each in a plain form
(elementary torch operations in 32 bits, angles in 64) and, where ``own`` is true, as the calls that a
serving engine makes of this package:

``rotary``  norms of each query and key head and the rotation by position, out of a packed QKV
            product (``QKNormRotary``).
``store``   new keys and values into the cache, then the rows of the touched blocks read back as
            values (``Fp4TokenToKVPool.set_kv_buffer`` / ``get_rows``).
``dense``   one decode step of the dense backend over that cache.
``sparse``  one decode step of the quest backend over that cache: page bounds, page scores, selection,
            attention over the selected pages and the recent window.
``extend``  one layer of prefill: the new tokens into the cache, then causal attention over it.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 64  # tokens of a block, and of a Quest page
GROUP = 32  # channels of a key that share a scale
K_EXP, V_EXP = (-96, 125), (-50, 59)  # exponents of a scale
TOP = 6.0  # largest e2m1 value
EPS = 1e-6
DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
FAR = torch.finfo(torch.bfloat16).max  # bounds of a page that has none


def listed() -> list[dict]:
    return [
        # a decode step's layer at a 32/4-head model: 16 tokens at positions of their own, latency alone
        {"name": "rotary_decode_b16", "kind": "rotary", "n": 16, "heads": 32, "kv": 4, "dim": 128, "rot": 128,
         "dtype": "bf16", "axes": 1, "cycled": False, "neighbours": False, "norm": True, "far": 131072, "prompt": False},
        # one layer of a long prompt
        {"name": "rotary_prompt_16k", "kind": "rotary", "n": 16384, "heads": 32, "kv": 4, "dim": 128, "rot": 128,
         "dtype": "bf16", "axes": 1, "cycled": False, "neighbours": False, "norm": True, "far": 0, "prompt": True},
        # video and text: time, height and width, an odd number of tokens, narrow heads of which half turn, float32
        {"name": "rotary_axes_5001", "kind": "rotary", "n": 5001, "heads": 14, "kv": 2, "dim": 64, "rot": 32,
         "dtype": "f32", "axes": 3, "cycled": True, "neighbours": True, "norm": True, "far": 30000, "prompt": True},
        # the new tokens of a decode step, most of them into blocks begun before
        {"name": "store_decode_b32", "kind": "store", "bs": 32, "prefix_lo": 50, "prefix_hi": 400, "new_lo": 1,
         "new_hi": 1, "kv": 4, "dim": 128, "dtype": "bf16"},
        # chunks of long prompts, which begin and end inside blocks; 8 KV heads
        {"name": "store_prompts_4", "kind": "store", "bs": 4, "prefix_lo": 0, "prefix_hi": 1000, "new_lo": 1000,
         "new_hi": 30000, "kv": 8, "dim": 128, "dtype": "bf16"},
        # one interactive request: 12 layers of a 32/4-head model
        {"name": "dense_b1_2k", "kind": "dense", "bs": 1, "ctx_lo": 2000, "ctx_hi": 2000, "layers": 12, "heads": 32,
         "kv": 4, "dim": 128, "dtype": "bf16"},
        # the headline serving shape: every row of 16 long contexts
        {"name": "dense_b16_128k", "kind": "dense", "bs": 16, "ctx_lo": 131072, "ctx_hi": 131072, "layers": 1,
         "heads": 32, "kv": 4, "dim": 128, "dtype": "bf16"},
        # a mixed batch down to a single token, an odd group, narrow heads, float32 queries
        {"name": "dense_b48_ragged", "kind": "dense", "bs": 48, "ctx_lo": 1, "ctx_hi": 20000, "layers": 2, "heads": 14,
         "kv": 2, "dim": 64, "dtype": "f32"},
        # Quest decode of one request: 8 layers
        {"name": "sparse_b1_32k", "kind": "sparse", "bs": 1, "ctx_lo": 32768, "ctx_hi": 32768, "layers": 8, "heads": 32,
         "kv": 4, "dim": 128, "dtype": "bf16", "top_k": 2048, "avoid": False},
        # the headline shape of the Quest step
        {"name": "sparse_b16_128k", "kind": "sparse", "bs": 16, "ctx_lo": 131072, "ctx_hi": 131072, "layers": 2,
         "heads": 32, "kv": 4, "dim": 128, "dtype": "bf16", "top_k": 2048, "avoid": False},
        # several prompts at once, with cached prefixes
        {"name": "extend_6_ragged", "kind": "extend", "bs": 6, "prefix_lo": 0, "prefix_hi": 4000, "new_lo": 50,
         "new_hi": 1500, "heads": 32, "kv": 4, "dim": 128, "dtype": "bf16"},
        # one chunk of a long prompt
        {"name": "extend_8k_chunk", "kind": "extend", "bs": 1, "prefix_lo": 8192, "prefix_hi": 8192, "new_lo": 8192,
         "new_hi": 8192, "heads": 32, "kv": 4, "dim": 128, "dtype": "bf16"},
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotary", "rotary", "store", "dense", "dense", "sparse", "extend", "extend"])
    kv = rng.choice([1, 2, 4, 4, 4, 8])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        heads = kv * rng.choice([1, 2, 4, 5, 7, 8])
        axes = rng.choice([1, 1, 2, 3, 3])
        rot = rng.choice([dim, dim, 32, 48])
        return {"kind": kind, "n": _log(rng, 1, 4_000_000 / ((heads + 2 * kv) * dim / 16)), "heads": heads, "kv": kv, "dim": dim,
                "rot": rot, "dtype": rng.choice(["bf16", "bf16", "f32"]), "axes": axes, "cycled": axes > 1 and rng.random() < 0.5,
                "neighbours": rng.random() < 0.3, "norm": rng.random() < 0.8, "far": _log(rng, 1, 2_000_000),
                "prompt": rng.random() < 0.6}
    if kind == "store":
        bs = _log(rng, 1, 64)
        prefix = rng.choice([0, _log(rng, 1, 1000)])
        new = rng.choice([1, _log(rng, 1, 60_000 / bs)])
        return {"kind": kind, "bs": bs, "prefix_lo": prefix // rng.randint(1, 20), "prefix_hi": prefix,
                "new_lo": max(1, new // rng.randint(1, 20)), "new_hi": new, "kv": kv, "dim": rng.choice([64, 128, 128]),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "dense":
        bs = _log(rng, 1, 96)
        hi = _log(rng, 20, min(131072, 1_000_000 / bs))
        return {"kind": kind, "bs": bs, "ctx_lo": max(1, rng.choice([hi, hi // rng.randint(2, 40)])), "ctx_hi": hi,
                "layers": min(12, max(1, 400_000 // (bs * hi))), "heads": kv * rng.choice([1, 4, 5, 7, 8, 16]), "kv": kv,
                "dim": rng.choice([64, 128, 128]), "dtype": rng.choice(["bf16", "bf16", "bf16", "f32"])}
    if kind == "sparse":
        bs = _log(rng, 1, 48)
        hi = _log(rng, 1500, min(131072, 1_000_000 / bs))
        return {"kind": kind, "bs": bs, "ctx_lo": rng.choice([hi, max(500, hi // rng.randint(2, 16))]), "ctx_hi": hi,
                "layers": min(12, max(1, 400_000 // (bs * hi))), "heads": kv * rng.choice([4, 5, 7, 8]), "kv": kv,
                "dim": 128, "dtype": "bf16", "top_k": rng.choice([512, 1024, 2048, 2048]), "avoid": rng.random() < 0.5}
    bs = rng.randint(1, 8)
    new = _log(rng, 1, 8192 / bs)
    prefix = rng.choice([0, _log(rng, 1, 8192)])
    return {"kind": "extend", "bs": bs, "prefix_lo": prefix // rng.randint(1, 4), "prefix_hi": prefix,
            "new_lo": max(1, new // rng.randint(1, 8)), "new_hi": new, "heads": kv * rng.choice([1, 4, 5, 7, 8]) if kv < 8 else 32,
            "kv": kv, "dim": rng.choice([64, 128, 128]), "dtype": "bf16"}


# ---------------------------------------------------------------- lengths and work of a case


def _spread(lo: int, hi: int, n: int, salt: int) -> list[int]:
    """n lengths in [lo, hi], fixed by the case alone: both ends, the rest log-uniform."""
    r = random.Random(f"{lo} {hi} {n} {salt}")
    if lo == hi or n == 1:
        return [hi] * n
    rest = [int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1 for _ in range(n - 2)]
    out = [hi, lo, *rest]
    r.shuffle(out)
    return out


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """(cached tokens, new tokens) of each request."""
    if "ctx_hi" in case:
        ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["bs"], 1)
        return [s - 1 for s in ctx], [1] * case["bs"]
    return (_spread(case["prefix_lo"], case["prefix_hi"], case["bs"], 3),
            _spread(case["new_lo"], case["new_hi"], case["bs"], 2))


def work(case: dict) -> dict:
    kind = case["kind"]
    width = 2 if case["dtype"] == "bf16" else 4
    kv, D = case["kv"], case["dim"]
    if kind == "rotary":
        n, H = case["n"], case["heads"]
        return {"bytes": 2 * n * (H + 2 * kv) * D * width + 8 * n * case["axes"],
                "flops": n * (H + kv) * ((4 * D if case["norm"] else 0) + 3 * case["rot"])}
    prefix, new = _lens(case)
    tokens = sum(new)
    row = kv * (D + D // GROUP + 1)  # bytes of a token's K and V: codes and scales
    if kind == "store":
        back = sum((p + n) - p // BLOCK * BLOCK for p, n in zip(prefix, new))
        return {"bytes": tokens * (2 * kv * D * width + row) + back * (row + 2 * kv * D * 2), "flops": 4 * tokens * kv * D}
    H = case["heads"]
    token = 2 * H * D * width + 2 * kv * D * width + row  # q, out, the new K/V read and written
    if kind == "extend":
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, prefix))
        return {"bytes": tokens * token + row * sum(prefix), "flops": 4 * pairs * H * D}
    nbytes = flops = 0
    for p in prefix:
        s = p + 1
        rows = s if kind == "dense" else min(s, case["top_k"])
        pages = 0 if kind == "dense" or s <= case["top_k"] else s // BLOCK
        nbytes += token + row * rows + 4 * kv * D * pages
        flops += 4 * rows * H * D + 2 * pages * kv * D
    return {"bytes": case["layers"] * nbytes, "flops": case["layers"] * flops}


# ---------------------------------------------------------------- inputs


def _i64(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int64, device=DEV)


class _Layer:
    def __init__(self, layer_id: int, dim: int):
        self.layer_id = layer_id
        self.scaling = dim**-0.5


def _sections(case: dict) -> list[int]:
    """Pairs of channels that turn by each axis."""
    pairs, axes = case["rot"] // 2, case["axes"]
    rest = [pairs * 3 // (4 * (axes - 1)) if axes > 2 else pairs // 2] * (axes - 1)
    return [pairs - sum(rest), *rest]


def _positions(case: dict, seed: int) -> list[list[int]]:
    """Of each axis: a decode step's tokens anywhere, a prompt's one after the other, the tokens of
    images at their frame, row and column."""
    r = random.Random(seed)
    n, far = case["n"], case["far"]
    if not case["prompt"]:
        at = [r.randint(0, far) for _ in range(n)]
        return [at] + [[max(0, x - r.randint(0, 40)) for x in at] for _ in range(case["axes"] - 1)]
    if case["axes"] == 1:
        return [list(range(far, far + n))]
    out, at = [[] for _ in range(case["axes"])], far
    while len(out[0]) < n:  # a run of text, then frames of a picture
        text, frames, rows, cols = r.randint(1, 200), r.randint(1, 4), r.randint(2, 24), r.randint(2, 24)
        for x in out:
            x.extend(range(at, at + text))
        at += text
        sides = (frames, rows, cols) if case["axes"] == 3 else (rows, cols)
        cells = [(f, y, x) for f in range(frames) for y in range(rows) for x in range(cols)]
        for x, axis in zip(out, range(3 - case["axes"], 3)):
            x.extend(at + c[axis] for c in cells)
        at += max(sides)
    return [x[:n] for x in out]


def _rotary_source(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n, H, kv, D = case["n"], case["heads"], case["kv"], case["dim"]
    spread = torch.exp(torch.empty((H + 2 * kv) * D, device=DEV).normal_(0.0, 0.5, generator=gen))
    qkv = torch.empty((n, (H + 2 * kv) * D), device=DEV).normal_(generator=gen).mul_(spread).to(DTYPES[case["dtype"]])
    wq, wk = (1.0 + torch.empty((2, D), device=DEV).normal_(0.0, 0.3, generator=gen)).unbind(0)
    pos = _i64(_positions(case, seed))
    return {"kind": "rotary", "case": case, "qkv": qkv, "wq": wq if case["norm"] else None, "wk": wk if case["norm"] else None,
            "pos": pos if case["axes"] > 1 else pos[0]}


def _source(case: dict, seed: int):
    """What the model computes, request by request: ``q [tokens, H, D]`` of the new tokens per
    layer, and a function (layer, request) -> K, V ``[prefix + new, KV, D]`` as it hands them over.
    Keys have a mean and a spread per channel, values a spread per head, as projections leave them."""
    prefix, new = _lens(case)
    kv, D, dt = case["kv"], case["dim"], DTYPES[case["dtype"]]
    layers = case.get("layers", 1)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    mean = torch.empty((layers, kv, D), device=DEV).normal_(0.0, 0.5, generator=gen)
    spread = torch.exp(torch.empty((layers, kv, D), device=DEV).normal_(0.0, 0.4, generator=gen))
    vspread = torch.exp(torch.empty((layers, kv, 1), device=DEV).normal_(0.0, 0.5, generator=gen))
    q = None
    if "heads" in case:
        q = torch.empty((layers, sum(new), case["heads"], D), device=DEV).normal_(generator=gen).to(dt)
    hot = {}
    if case["kind"] == "sparse":  # the pages a query is after: as many as it may select
        r = random.Random(seed)
        for i, p in enumerate(prefix):
            lim = _limit(case, p + 1)
            hot[i] = sorted(r.sample(range(lim), min(case["top_k"] // BLOCK - 1, lim)))

    def kv_of(layer: int, i: int):
        g = torch.Generator(device=DEV).manual_seed(seed * 1_000_003 + layer * 4099 + i + 1)
        n = prefix[i] + new[i]
        k = torch.empty((n, kv, D), device=DEV).normal_(generator=g).mul_(spread[layer]).add_(mean[layer])
        if i in hot:
            toward = torch.sign(_mean_query(q[layer, i], kv).float()) * spread[layer]
            pages = k[: n // BLOCK * BLOCK].view(-1, BLOCK, kv, D)
            pages[hot[i]] += 1.5 * toward
        v = torch.empty((n, kv, D), device=DEV).normal_(generator=g).mul_(vspread[layer])
        return k.to(dt), v.to(dt)

    return q, kv_of, prefix, new


def _limit(case: dict, s: int) -> int:
    """Pages that a query at a context of s tokens may select: complete ones, but not the one that the
    new token completes, which has no bounds yet, nor with `avoid` any in the recent window."""
    return max(0, min(s // BLOCK - 1 if case["avoid"] else s // BLOCK, (s - 1) // BLOCK))


def _mean_query(q: torch.Tensor, kv: int) -> torch.Tensor:
    """The mean of each KV head's query heads: float32 in head order, one rounding to q's type."""
    heads, D = q.shape
    x = q.view(kv, heads // kv, D).float()
    acc = torch.zeros((kv, D), device=q.device)
    for g in range(heads // kv):
        acc = acc + x[:, g]
    return (acc / (heads // kv)).to(q.dtype)


def _blocks_of(prefix, new) -> list[int]:
    return [-(-(p + n) // BLOCK) for p, n in zip(prefix, new)]


def _scatter_blocks(prefix, new, seed: int):
    """Blocks handed out at random: the block list of each request."""
    counts = _blocks_of(prefix, new)
    ids = list(range(1, sum(counts) + 1))
    random.Random(seed).shuffle(ids)
    out, at = [], 0
    for c in counts:
        out.append(_i64(ids[at : at + c]))
        at += c
    return out


def _rows(blocks: torch.Tensor, lo: int, hi: int) -> torch.Tensor:
    pos = torch.arange(lo, hi, device=DEV)
    return blocks[pos // BLOCK] * BLOCK + pos % BLOCK


def prepare(case: dict, seed: int):
    kind = case["kind"]
    if kind == "rotary":
        return _prepare_rotary(case, seed)
    if kind == "store":
        return _prepare_store(case, seed)
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


def _prepare_rotary(case: dict, seed: int):
    st = _rotary_source(case, seed)
    if own:
        from qwenquest_amd.rotary import QKNormRotary

        st["op"] = QKNormRotary(
            case["heads"], case["kv"], case["dim"], q_weight=st["wq"], k_weight=st["wk"], eps=EPS, base=1e6,
            rotary_dim=case["rot"], sections=_sections(case) if case["axes"] > 1 else None,
            section_order="cycled" if case["cycled"] else "blocks", pairs="neighbours" if case["neighbours"] else "halves",
            device=DEV)
    return st


def _prepare_store(case: dict, seed: int):
    _, kv_of, prefix, new = _source(case, seed)
    blocks = _scatter_blocks(prefix, new, seed)
    total = sum(b.numel() for b in blocks) + 1
    kv, D = case["kv"], case["dim"]
    if own:
        from qwenquest_amd.paged import Fp4TokenToKVPool

        st = {"pool": Fp4TokenToKVPool(total, 1, kv, D, DEV)}
    else:
        st = _plain_cache(total, 1, kv, D)
    ks, vs, locs, back = [], [], [], []
    for i, (p, n) in enumerate(zip(prefix, new)):
        k, v = kv_of(0, i)
        if p:
            loc = _rows(blocks[i], 0, p)
            if own:
                st["pool"].set_kv_buffer(0, loc, k[:p], v[:p])
            else:
                _plain_store(st, 0, loc, k[:p], v[:p])
        ks.append(k[p:])
        vs.append(v[p:])
        locs.append(_rows(blocks[i], p, p + n))
        back.append(_rows(blocks[i], p // BLOCK * BLOCK, p + n))
    st.update(kind="store", k=torch.cat(ks), v=torch.cat(vs), loc=torch.cat(locs), back=torch.cat(back))
    return st


def _prepare_plain(case: dict, seed: int):
    q, kv_of, prefix, new = _source(case, seed)
    layers, kv, D = case.get("layers", 1), case["kv"], case["dim"]
    blocks = _scatter_blocks(prefix, new, seed)
    st = _plain_cache(sum(b.numel() for b in blocks) + 1, layers, kv, D)
    ks, vs = [[] for _ in range(layers)], [[] for _ in range(layers)]
    for layer in range(layers):
        for i, p in enumerate(prefix):
            k, v = kv_of(layer, i)
            if p:
                _plain_store(st, layer, _rows(blocks[i], 0, p), k[:p], v[:p])
            ks[layer].append(k[p:])
            vs[layer].append(v[p:])
    st.update(kind=case["kind"], case=case, blocks=blocks, prefix=prefix, new=new, q=q, scale=D**-0.5)
    st["k"], st["v"] = [torch.cat(x) for x in ks], [torch.cat(x) for x in vs]
    st["loc"] = torch.cat([_rows(b, p, p + n) for b, p, n in zip(blocks, prefix, new)])
    if case["kind"] == "sparse":
        pages = max(prefix) // BLOCK + 1
        st["bounds"] = torch.empty((layers, case["bs"], pages, kv, D, 2), dtype=torch.bfloat16, device=DEV)
        st["bounds"][..., 0], st["bounds"][..., 1] = FAR, -FAR
        _plain_bounds(st, [0] * len(prefix), prefix)
    return st


def _admissions(case: dict, seed: int):
    """The order in which a server's requests came to hold their cached tokens: chunk by chunk."""
    prefix, _ = _lens(case)
    r = random.Random(seed)
    at, out = [0] * len(prefix), []
    chunk = max(1, max(prefix) // 3)
    while any(a < p for a, p in zip(at, prefix)):
        rows = [i for i, p in enumerate(prefix) if at[i] < p]
        r.shuffle(rows)
        out.append((rows, [at[i] for i in rows], [min(chunk, prefix[i] - at[i]) for i in rows]))
        for i in rows:
            at[i] = min(prefix[i], at[i] + chunk)
    return out


def _prepare_own(case: dict, seed: int):
    from qwenquest_amd.attention import DenseBackend, QuestOnlyBackend
    from qwenquest_amd.batch import ForwardBatch, ForwardMode
    from qwenquest_amd.paged import BlockReqToTokenPool, Fp4TokenToKVPool

    q, kv_of, prefix, new = _source(case, seed)
    kind, bs, layers, kv, D = case["kind"], case["bs"], case.get("layers", 1), case["kv"], case["dim"]
    total = [p + n for p, n in zip(prefix, new)]
    rtp = BlockReqToTokenPool(bs, max(total) + BLOCK, sum(_blocks_of(prefix, new)) + 1, DEV)
    kvp = Fp4TokenToKVPool(rtp.num_blocks, layers, kv, D, DEV)
    for rows, a, n in _admissions(case, seed):
        rtp.assign(_i64(rows), _i64(a), _i64(n), sum(n))
    rpi, pre, ext, seq = _i64(list(range(bs))), _i64(prefix), _i64(new), _i64(total)
    loc, positions = rtp.assign(rpi, pre, ext, sum(new))
    ks, vs = [[] for _ in range(layers)], [[] for _ in range(layers)]
    for i, p in enumerate(prefix):
        rows = rtp.req_to_token[i, :p].long()
        for layer in range(layers):
            k, v = kv_of(layer, i)
            if p:
                kvp.set_kv_buffer(layer, rows, k[:p], v[:p])
            ks[layer].append(k[p:])
            vs[layer].append(v[p:])
    if kind == "sparse":
        be = QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": case["top_k"], "quest_page_size": BLOCK,
                                         "avoid_recent_overlap": case["avoid"]})
        be.quest.update_prefill_representations_blocks(rpi, pre, kvp, rtp.block_table)
    else:
        be = DenseBackend(rtp, kvp)
    k, v = [torch.cat(x) for x in ks], [torch.cat(x) for x in vs]
    mods = [_Layer(i, D) for i in range(layers)]
    if kind == "extend":
        batch = ForwardBatch(ForwardMode.EXTEND, None, positions, rpi, seq, loc, rtp, kvp, be, extend_prefix_lens=pre,
                             extend_seq_lens=ext)
        return {"kind": kind, "be": be, "q": q[0], "k": k[0], "v": v[0], "layer": mods[0], "batch": batch}
    batch = ForwardBatch(ForwardMode.DECODE, None, positions, rpi, seq, loc, rtp, kvp, be)

    def step():
        be.init_forward_metadata(batch)
        return [be.forward_decode(q[i], k[i], v[i], mods[i], batch) for i in range(layers)]

    # decode steps are captured and replayed, as a serving loop does
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return {"kind": kind, "be": be, "q": q, "k": k, "v": v, "batch": batch, "graph": graph, "out": out}


# ---------------------------------------------------------------- the plain forms


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2 ** e in float32, from its bits (e in -126 .. 127)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _axis_of_pair(case: dict) -> list[int]:
    left = _sections(case) if case["axes"] > 1 else [case["rot"] // 2]
    if not case["cycled"]:
        return [a for a, m in enumerate(left) for _ in range(m)]
    out, a = [], 0
    while sum(left):  # dealt to the axes in turn, as long as each has pairs left
        if left[a]:
            out.append(a)
            left[a] -= 1
        a = (a + 1) % len(left)
    return out


def _plain_rotary(st: dict):
    case, pos = st["case"], st["pos"].view(st["case"]["axes"], -1)
    n, H, kv, D, rot = case["n"], case["heads"], case["kv"], case["dim"], case["rot"]
    freq = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    angle = pos[_axis_of_pair(case)].T.double() * freq  # [n, rot / 2]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = st["qkv"].view(n, H + 2 * kv, D)
    out = []
    for y, w in ((x[:, :H], st["wq"]), (x[:, H : H + kv], st["wk"])):
        y = y.float()
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w
        if case["neighbours"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., : rot // 2], y[..., rot // 2 : rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([turned, y[..., rot:]], -1).to(x.dtype))
    return [*out, x[:, H + kv :].contiguous()]


def _plain_cache(blocks: int, layers: int, kv: int, D: int) -> dict:
    """The values that the codes stand for; they are exact in bfloat16."""
    return {c: torch.zeros((layers, blocks, BLOCK, kv, D), dtype=torch.bfloat16, device=DEV) for c in ("kc", "vc")}


def _quantised(x: torch.Tensor, group: int, span: tuple[int, int]) -> torch.Tensor:
    """[n, KV, D] as the cache keeps it, one scale for `group` channels."""
    y = x.float().unflatten(-1, (-1, group))
    frac, e = torch.frexp(y.abs().amax(-1, keepdim=True))  # amax <= 7 * 2 ** e: 7 = 0.875 * 2 ** 3
    e = torch.where(frac <= 0.875, e - 3, e - 2)
    e = torch.where(frac == 0, span[0], e).clamp(*span)
    half = _pow2(-(e // 2)), _pow2(-(e - e // 2))
    y = y * half[0] * half[1]
    _, ye = torch.frexp(y)
    step = _pow2((ye - 1).clamp(min=0) - 1)
    return ((torch.round(y / step) * step).clamp(-TOP, TOP) * _pow2(e)).flatten(-2).to(torch.bfloat16)


def _plain_store(st: dict, layer: int, loc: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    for a in range(0, loc.numel(), 1 << 17):  # a long prompt's in 32 bits are large
        at, x, y = (t[a : a + (1 << 17)] for t in (loc, k, v))
        # of a token and head that holds what is not finite, or too large in V, nothing is kept
        good = torch.isfinite(x).all(-1, keepdim=True) & (y.abs() <= 7 * 2.0 ** V_EXP[1]).all(-1, keepdim=True)
        for values, z, group, span in ((st["kc"], x, GROUP, K_EXP), (st["vc"], y, y.shape[-1], V_EXP)):
            z = _quantised(torch.where(good, z, 0.0), group, span)
            values[layer].view(-1, *z.shape[1:])[at] = torch.where(good, z, math.nan)


def _plain_rows(st: dict, layer: int, loc: torch.Tensor):
    return tuple(st[c][layer].view(-1, *st[c].shape[3:])[loc] for c in ("kc", "vc"))


def _plain_context(st: dict, layer: int, i: int, n: int):
    """K and V values of request i's first n tokens, as float32."""
    b = st["blocks"][i][: -(-n // BLOCK)]
    return [st[c][layer][b].float().flatten(0, 1)[:n] for c in ("kc", "vc")]


def _plain_bounds(st: dict, lo: list[int], hi: list[int]) -> None:
    """Bounds of the pages that tokens lo .. hi complete, over every layer."""
    for layer in range(st["kc"].shape[0]):
        for i, (a, b) in enumerate(zip(lo, hi)):
            p0, p1 = a // BLOCK, b // BLOCK
            if p1 > p0:
                k = st["kc"][layer][st["blocks"][i][p0:p1]].float()
                st["bounds"][layer, i, p0:p1, :, :, 0] = k.amin(1).to(torch.bfloat16)
                st["bounds"][layer, i, p0:p1, :, :, 1] = k.amax(1).to(torch.bfloat16)


def _plain_attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, first: int | None = None):
    """q [n, H, D] over k, v [m, KV, D] -> [n, H * D]; row t attends 0 .. first + t where given."""
    n, H, D = q.shape
    kv = k.shape[1]
    qh = q.float().view(n, kv, H // kv, D).permute(1, 0, 2, 3).reshape(kv, -1, D)
    s = torch.matmul(qh, k.permute(1, 2, 0).contiguous()) * scale  # [KV, n * G, m]
    if first is not None:
        seen = torch.arange(k.shape[0], device=DEV)[None] <= first + torch.arange(n, device=DEV)[:, None]
        s = s.view(kv, n, H // kv, -1).masked_fill(~seen[:, None], -math.inf).view(kv, n * (H // kv), -1)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(s, v.permute(1, 0, 2).contiguous()) / s.sum(-1, keepdim=True)
    return o.view(kv, n, H // kv, D).permute(1, 0, 2, 3).reshape(n, H * D).to(q.dtype)


def _plain_select(st: dict, layer: int, i: int, s: int) -> torch.Tensor:
    """Token positions that request i's query attends: the best pages, then the recent window."""
    case = st["case"]
    qbar = _mean_query(st["q"][layer, i], case["kv"]).float()
    lim = _limit(case, s)
    b = st["bounds"][layer, i, :lim].float()
    x = torch.where(qbar >= 0, qbar * b[..., 1], qbar * b[..., 0]).reshape(lim, -1)
    m = -(-x.shape[1] // 64)
    x = torch.nn.functional.pad(x, (0, 64 * m - x.shape[1])).view(lim, 64, m)
    acc = x[..., 0]  # the sum's order is part of the score: 64 runs of channels, then halves
    for j in range(1, m):
        acc = acc + x[..., j]
    w = 64
    while w > 1:
        w //= 2
        acc = acc[:, :w] + acc[:, w : 2 * w]
    best = torch.sort(acc[:, 0], descending=True, stable=True).indices[: case["top_k"] // BLOCK - 1]
    return torch.cat([(best[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(),
                      torch.arange(s - BLOCK, s, device=DEV)])


def _plain_decode(st: dict):
    case, outs = st["case"], []
    if case["kind"] == "sparse":  # the page that the token before the new one completed
        _plain_bounds(st, [max(p - 1, 0) for p in st["prefix"]], st["prefix"])
    for layer in range(case["layers"]):
        _plain_store(st, layer, st["loc"], st["k"][layer], st["v"][layer])
        out = []
        for i, p in enumerate(st["prefix"]):
            s = p + 1
            if case["kind"] == "sparse" and s > case["top_k"]:
                pos = _plain_select(st, layer, i, s)
                k, v = (x.float() for x in _plain_rows(st, layer, st["blocks"][i][pos // BLOCK] * BLOCK + pos % BLOCK))
            else:
                k, v = _plain_context(st, layer, i, s)
            out.append(_plain_attend(st["q"][layer, i][None], k, v, st["scale"]))
        outs.append(torch.cat(out))
    return outs


def _plain_extend(st: dict):
    _plain_store(st, 0, st["loc"], st["k"][0], st["v"][0])
    outs, at = [], 0
    for i, (p, n) in enumerate(zip(st["prefix"], st["new"])):
        k, v = _plain_context(st, 0, i, p + n)
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            outs.append(_plain_attend(st["q"][0, at + a : at + b], k[: p + b], v[: p + b], st["scale"], p + a))
        at += n
    return torch.cat(outs)


# ---------------------------------------------------------------- one pass


def run(state: dict):
    kind = state["kind"]
    if kind == "rotary":
        return list(state["op"](state["qkv"], state["pos"])) if own else _plain_rotary(state)
    if kind == "store":
        if own:
            pool = state["pool"]
            pool.set_kv_buffer(0, state["loc"], state["k"], state["v"])
            return list(pool.get_rows(0, state["back"]))
        _plain_store(state, 0, state["loc"], state["k"], state["v"])
        return list(_plain_rows(state, 0, state["back"]))
    if kind == "extend":
        if own:
            return state["be"].forward_extend(state["q"], state["k"], state["v"], state["layer"], state["batch"])
        return _plain_extend(state)
    if own:
        state["graph"].replay()
        return state["out"]
    return _plain_decode(state)


# ---------------------------------------------------------------- the same in 64 bits


def _exact_values(x: torch.Tensor, group: int, span: tuple[int, int]) -> torch.Tensor:
    """The nearest of +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} times the group's scale, ties to the even code."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    border = (grid[1:] + grid[:-1]) / 2
    out = []
    for part in x.split(1 << 16):
        y = part.double().unflatten(-1, (-1, group))
        high = y.abs().amax(-1, keepdim=True)
        e = torch.full_like(high, span[0])
        e = torch.where(high > 0, torch.ceil(torch.log2(high.clamp(min=1e-300) / 7.0)), e)
        # a logarithm may be off next to a power of two
        e = torch.where(high > 7.0 * torch.exp2(e), e + 1, e)
        e = torch.where(high <= 7.0 * torch.exp2(e - 1), e - 1, e).clamp(*span)
        y = y / torch.exp2(e)
        code = torch.bucketize(y.abs(), border)  # the lower neighbour at a border
        on_border = (code < 7) & (y.abs() == border[code.clamp(max=6)])
        code = torch.where(on_border & (code % 2 == 1), code + 1, code)
        out.append((torch.sign(y) * grid[code] * torch.exp2(e)).flatten(-2))
    return torch.cat(out)


def _attend64(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, first: int | None = None):
    n, H, D = q.shape
    G = H // k.shape[1]
    out = torch.empty((n, H, D), dtype=torch.float64, device=q.device)
    for h in range(H):
        s = (q[:, h].double() @ k[:, h // G].T) * scale
        if first is not None:
            seen = torch.arange(k.shape[0], device=q.device)[None] <= first + torch.arange(n, device=q.device)[:, None]
            s.masked_fill_(~seen, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, h // G]
    return out.view(n, H * D)


def _exact_rotary(case: dict, seed: int):
    st = _rotary_source(case, seed)
    n, H, kv, D, rot = case["n"], case["heads"], case["kv"], case["dim"], case["rot"]
    pos = st["pos"].view(case["axes"], n)
    axis = _axis_of_pair(case)
    x = st["qkv"].view(n, H + 2 * kv, D)
    outs = []
    for part, w in ((x[:, :H], st["wq"]), (x[:, H : H + kv], st["wk"])):
        y = part.double()
        if w is not None:
            y = y * w.double() * (y.square().sum(-1, keepdim=True) / D + EPS).rsqrt()
        else:
            y = y.clone()
        for j in range(rot // 2):  # one pair as a complex number, turned
            a, b = (2 * j, 2 * j + 1) if case["neighbours"] else (j, j + rot // 2)
            t = pos[axis[j]].double() * 1e6 ** (-2.0 * j / rot)
            z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(t), t)[:, None]
            y[..., a], y[..., b] = z.real, z.imag
        outs.append(y)
    return [*outs, x[:, H + kv :].double()]


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(case, seed)
    q, kv_of, prefix, new = _source(case, seed)
    layers, D = case.get("layers", 1), case["dim"]

    def values(layer: int, i: int):
        k, v = kv_of(layer, i)
        return _exact_values(k, GROUP, K_EXP), _exact_values(v, D, V_EXP)

    if kind == "store":
        rows = [], []
        for i, p in enumerate(prefix):
            for out, x in zip(rows, values(0, i)):
                out.append(x[p // BLOCK * BLOCK :])
        return [torch.cat(x) for x in rows]
    outs = []
    for layer in range(layers):
        out, at = [], 0
        for i, (p, n) in enumerate(zip(prefix, new)):
            k, v = values(layer, i)
            if kind == "extend":
                for a in range(0, n, 1024):
                    b = min(n, a + 1024)
                    out.append(_attend64(q[layer, at + a : at + b], k[: p + b], v[: p + b], D**-0.5, p + a))
            else:
                if kind == "sparse" and p + 1 > case["top_k"]:
                    pos = _exact_select(case, q[layer, i], k, p + 1)
                    k, v = k[pos], v[pos]
                out.append(_attend64(q[layer, i][None], k, v, D**-0.5))
            at += n
        outs.append(torch.cat(out))
    return outs[0] if kind == "extend" else outs


def _exact_select(case: dict, q: torch.Tensor, k: torch.Tensor, s: int) -> torch.Tensor:
    lim = _limit(case, s)
    kp = k[: lim * BLOCK].view(lim, BLOCK, *k.shape[1:])
    qbar = _mean_query(q, case["kv"]).double()  # the mean query's rounding is part of the method
    score = torch.maximum(qbar * kp.amax(1), qbar * kp.amin(1)).sum((1, 2))
    top = torch.sort(score, descending=True, stable=True).indices[: case["top_k"] // BLOCK - 1]
    return torch.cat([(top[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(),
                      torch.arange(s - BLOCK, s, device=DEV)])
