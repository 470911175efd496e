"""The operators around the 8-bit K/V cache, as calls that can be timed and checked.

The cache holds blocks of 64 tokens: e4m3 codes with one power-of-two scale for each block and KV
head, K and V apart.  Five operators, each in a plain form (elementary torch operations in 32 bits)
and, where ``own`` is true, as the calls a serving engine makes of this package:

``slots``   the pool rows of a batch's new tokens: blocks handed out, block table and request table
            written, one row and one position per token (``BlockReqToTokenPool``).
``store``   new keys and values into the cache, then the rows of the touched blocks read back as
            values (``Fp8TokenToKVPool.set_kv_buffer`` / ``get_rows``).
``dense``   one decode step of the dense backend over that cache.
``sparse``  one decode step of the quest backend over that cache: bounds, page scores, selection,
            attention over the selected pages and the recent window.
``bounds``  the page bounds of a batch of prompts over every layer, as a prefill leaves them.
``extend``  one layer of prefill: the new tokens into the cache, then causal attention over it.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 64  # tokens of a block, and of a Quest page
E_MIN = -110  # least exponent of a scale
TOP = 448.0  # largest e4m3 value
DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
FAR = torch.finfo(torch.bfloat16).max  # bounds of a page that has none


def listed() -> list[dict]:
    return [
        # a decode step of a busy server: one new token per request, latency alone
        {"name": "slots_decode_b64", "kind": "slots", "bs": 64, "prefix_lo": 100, "prefix_hi": 32768, "new_lo": 1,
         "new_hi": 1, "finish": False},
        # prompts admitted at once, and their blocks given back
        {"name": "slots_admit_16", "kind": "slots", "bs": 16, "prefix_lo": 0, "prefix_hi": 0, "new_lo": 2000,
         "new_hi": 65536, "finish": True},
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
        # bounds of two prompts over 48 layers
        {"name": "bounds_2x16k", "kind": "bounds", "bs": 2, "prefix_lo": 0, "prefix_hi": 0, "new_lo": 16000,
         "new_hi": 16384, "layers": 48, "kv": 4, "dim": 128},
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
    kind = rng.choice(["slots", "store", "dense", "dense", "sparse", "sparse", "bounds", "extend", "extend"])
    if kind == "slots":
        bs = _log(rng, 1, 256)
        prefix = rng.choice([0, _log(rng, 1, 400_000 / bs)])
        new = rng.choice([1, _log(rng, 1, 400_000 / bs)])
        return {"kind": kind, "bs": bs, "prefix_lo": prefix // rng.randint(1, 20), "prefix_hi": prefix,
                "new_lo": max(1, new // rng.randint(1, 20)), "new_hi": new, "finish": prefix == 0 and rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 4, 4, 8])
    if kind == "store":
        bs = _log(rng, 1, 64)
        prefix = rng.choice([0, _log(rng, 1, 1000)])
        new = rng.choice([1, _log(rng, 1, 60_000 / bs)])
        return {"kind": kind, "bs": bs, "prefix_lo": prefix // rng.randint(1, 20), "prefix_hi": prefix,
                "new_lo": max(1, new // rng.randint(1, 20)), "new_hi": new, "kv": kv, "dim": rng.choice([64, 128, 128]),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "bounds":
        bs, layers = rng.randint(1, 4), rng.choice([1, 12, 24, 48])
        new = _log(rng, 30, 32_000 / bs)
        return {"kind": kind, "bs": bs, "prefix_lo": 0, "prefix_hi": rng.choice([0, _log(rng, 1, 2000)]),
                "new_lo": max(1, new // rng.randint(1, 8)), "new_hi": new, "layers": layers,
                "kv": min(kv, 4), "dim": rng.choice([64, 128, 128])}
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
            "kv": kv, "dim": 128, "dtype": "bf16"}


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
    prefix, new = _lens(case)
    tokens = sum(new)
    if kind == "slots":
        blocks = sum(-(-(p + n) // BLOCK) - -(-p // BLOCK) for p, n in zip(prefix, new))
        return {"bytes": 24 * case["bs"] + 20 * tokens + 4 * blocks * (2 if case["finish"] else 1), "flops": 4 * tokens}
    row = case["kv"] * case["dim"]  # values of one K or V row, bytes of its codes
    if kind == "bounds":
        pages = [(p + n) // BLOCK - p // BLOCK for p, n in zip(prefix, new)]
        return {"bytes": case["layers"] * sum(pages) * (BLOCK * row + 4 * row), "flops": 2 * case["layers"] * sum(pages) * BLOCK * row}
    width = 2 if case.get("dtype", "bf16") == "bf16" else 4
    if kind == "store":
        back = sum((p + n) - p // BLOCK * BLOCK for p, n in zip(prefix, new))
        return {"bytes": tokens * 2 * row * (width + 1) + back * 2 * row * 3, "flops": 4 * tokens * row}
    H, D = case["heads"], case["dim"]
    token = 2 * H * D * width + 2 * row * (width + 1)  # q, out, the new K/V read and written
    if kind == "extend":
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, prefix))
        return {"bytes": tokens * token + 2 * row * sum(prefix), "flops": 4 * pairs * H * D}
    nbytes = flops = 0
    for p in prefix:
        s = p + 1
        rows = s if kind == "dense" else min(s, case["top_k"])
        pages = 0 if kind == "dense" or s <= case["top_k"] else s // BLOCK
        nbytes += token + 2 * row * rows + 4 * row * pages
        flops += 4 * rows * H * D + 2 * pages * row
    return {"bytes": case["layers"] * nbytes, "flops": case["layers"] * flops}


# ---------------------------------------------------------------- inputs


def _i64(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int64, device=DEV)


class _Layer:
    def __init__(self, layer_id: int, dim: int):
        self.layer_id = layer_id
        self.scaling = dim**-0.5


def _source(case: dict, seed: int):
    """What the model computes, request by request: ``q [tokens, H, D]`` of the new tokens per
    layer, and a function (layer, request) -> K, V ``[prefix + new, KV, D]`` as it hands them over.
    Keys have a mean and a spread per channel, values a spread per head, as projections leave them."""
    prefix, new = _lens(case)
    kv, D, dt = case["kv"], case["dim"], DTYPES[case.get("dtype", "bf16")]
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
            lim = max(0, min(p // BLOCK, (p + 1) // BLOCK - 1) if case["avoid"] else p // BLOCK)
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


def prepare(case: dict, seed: int):
    kind = case["kind"]
    if kind == "slots":
        return _prepare_slots(case, seed)
    if kind == "store":
        return _prepare_store(case, seed)
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


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


def _prepare_slots(case: dict, seed: int):
    prefix, new = _lens(case)
    bs, blocks = case["bs"], sum(_blocks_of(prefix, new)) + 8
    width = max(p + n for p, n in zip(prefix, new)) + BLOCK
    order = list(range(bs))
    random.Random(seed + 1).shuffle(order)  # the batch's order
    st = {"rpi": _i64(order), "prefix": _i64([prefix[i] for i in order]), "new": _i64([new[i] for i in order]),
          "total": sum(new), "finish": case["finish"], "kind": "slots"}
    if own:
        from qwenquest_amd.paged import BlockReqToTokenPool

        pool = BlockReqToTokenPool(bs, width, blocks + 1, DEV)
        for rows, a, n in _admissions(case, seed):
            pool.assign(_i64(rows), _i64(a), _i64(n), sum(n))
        st["pool"] = pool
        return st
    st.update(table=torch.zeros((bs, -(-width // BLOCK)), dtype=torch.int32, device=DEV),
              r2t=torch.zeros((bs, width), dtype=torch.int32, device=DEV),
              held=torch.zeros(bs, dtype=torch.int32, device=DEV),
              free=torch.arange(blocks, 0, -1, dtype=torch.int32, device=DEV),
              count=torch.full((1,), blocks, dtype=torch.int32, device=DEV))
    for rows, a, n in _admissions(case, seed):
        _plain_assign(st, _i64(rows), _i64(a), _i64(n), sum(n))
    return st


def _scatter_rows(prefix, new, seed: int):
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


def _prepare_store(case: dict, seed: int):
    _, kv_of, prefix, new = _source(case, seed)
    blocks = _scatter_rows(prefix, new, seed)
    total = sum(b.numel() for b in blocks) + 1
    kv, D = case["kv"], case["dim"]
    st = _plain_cache(total, 1, kv, D)
    if own:
        from qwenquest_amd.paged import Fp8TokenToKVPool

        st = {"pool": Fp8TokenToKVPool(total, 1, kv, D, DEV)}
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
    blocks = _scatter_rows(prefix, new, seed)
    st = _plain_cache(sum(b.numel() for b in blocks) + 1, layers, kv, D)
    held = new if case["kind"] == "bounds" else [0] * len(new)  # tokens in the cache before the pass
    ks, vs = [[] for _ in range(layers)], [[] for _ in range(layers)]
    for layer in range(layers):
        for i, (p, n) in enumerate(zip(prefix, new)):
            k, v = kv_of(layer, i)
            for lo, hi in ((0, p), (p, p + held[i])):
                if hi > lo:
                    _plain_store(st, layer, _rows(blocks[i], lo, hi), k[lo:hi], v[lo:hi])
            ks[layer].append(k[p:])
            vs[layer].append(v[p:])
    st.update(kind=case["kind"], case=case, blocks=blocks, prefix=prefix, new=new, q=q, scale=D**-0.5)
    if case["kind"] == "bounds":
        pages = -(-(max(p + n for p, n in zip(prefix, new)) + BLOCK) // BLOCK)
        st["bounds"] = torch.empty((layers, case["bs"], pages, kv, D, 2), dtype=torch.bfloat16, device=DEV)
        st["bounds"][..., 0], st["bounds"][..., 1] = FAR, -FAR
        _plain_bounds(st, [0] * len(prefix), prefix)
        return st
    st["k"], st["v"] = [torch.cat(x) for x in ks], [torch.cat(x) for x in vs]
    st["loc"] = torch.cat([_rows(b, p, p + n) for b, p, n in zip(blocks, prefix, new)])
    if case["kind"] == "sparse":
        pages = max(prefix) // BLOCK + 1
        st["bounds"] = torch.empty((layers, case["bs"], pages, kv, D, 2), dtype=torch.bfloat16, device=DEV)
        st["bounds"][..., 0], st["bounds"][..., 1] = FAR, -FAR
        _plain_bounds(st, [0] * len(prefix), prefix)
    return st


def _prepare_own(case: dict, seed: int):
    from qwenquest_amd.attention import DenseBackend, QuestOnlyBackend
    from qwenquest_amd.batch import ForwardBatch, ForwardMode
    from qwenquest_amd.paged import BlockReqToTokenPool, Fp8TokenToKVPool

    q, kv_of, prefix, new = _source(case, seed)
    kind, bs, layers, kv, D = case["kind"], case["bs"], case.get("layers", 1), case["kv"], case["dim"]
    total = [p + n for p, n in zip(prefix, new)]
    rtp = BlockReqToTokenPool(bs, max(total) + BLOCK, sum(_blocks_of(prefix, new)) + 1, DEV)
    kvp = Fp8TokenToKVPool(rtp.num_blocks, layers, kv, D, DEV)
    for rows, a, n in _admissions(case, seed):
        rtp.assign(_i64(rows), _i64(a), _i64(n), sum(n))
    rpi, pre, ext, seq = _i64(list(range(bs))), _i64(prefix), _i64(new), _i64(total)
    loc, positions = rtp.assign(rpi, pre, ext, sum(new))
    ks, vs, at = [[] for _ in range(layers)], [[] for _ in range(layers)], 0
    for i, (p, n) in enumerate(zip(prefix, new)):
        rows = rtp.req_to_token[i, :p].long()
        for layer in range(layers):
            k, v = kv_of(layer, i)
            if p:
                kvp.set_kv_buffer(layer, rows, k[:p], v[:p])
            ks[layer].append(k[p:])
            vs[layer].append(v[p:])
            if kind == "bounds":
                kvp.set_kv_buffer(layer, loc[at : at + n], k[p:], v[p:])
        at += n
    if kind in ("bounds", "sparse"):
        be = QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": case.get("top_k", 2048), "quest_page_size": BLOCK,
                                         "avoid_recent_overlap": case.get("avoid", False)})
        be.quest.update_prefill_representations_blocks(rpi, pre, kvp, rtp.block_table)
    else:
        be = DenseBackend(rtp, kvp)
    if kind == "bounds":
        return {"kind": kind, "quest": be.quest, "rpi": rpi, "prefix": pre, "seq": seq, "kvp": kvp, "rtp": rtp}
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


def _exponent(scale: torch.Tensor) -> torch.Tensor:
    return ((scale.view(torch.int32) >> 23) & 255) - 127


def _plain_cache(blocks: int, layers: int, kv: int, D: int) -> dict:
    def codes():
        return torch.zeros((layers, blocks, BLOCK, kv, D), dtype=torch.uint8, device=DEV)

    def scales():
        return torch.full((layers, blocks, kv), 2.0**E_MIN, device=DEV)

    return {"kc": codes(), "vc": codes(), "ks": scales(), "vs": scales()}


def _decode8(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).float()


def _encode8(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_store(st: dict, layer: int, loc: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    ids, at = torch.unique(loc // BLOCK, return_inverse=True)
    slot = loc % BLOCK
    for codes, scales, x in ((st["kc"][layer], st["ks"][layer], k), (st["vc"][layer], st["vs"][layer], v)):
        step = 4096  # blocks at a time: a long prompt's in 32 bits are large
        for lo in range(0, ids.numel(), step):
            part = (at >= lo) & (at < lo + step) if ids.numel() > step else None
            a, s, y = (at - lo, slot, x) if part is None else (at[part] - lo, slot[part], x[part])
            m = min(step, ids.numel() - lo)
            fresh = torch.zeros((m, BLOCK, *x.shape[1:]), device=DEV)
            mine = torch.zeros((m, BLOCK, 1, 1), dtype=torch.bool, device=DEV)
            fresh[a, s] = y.float()
            mine[a, s] = True
            good = torch.isfinite(fresh)
            frac, ex = torch.frexp((fresh.abs() * good).nan_to_num(0.0).amax((1, 3)))
            e = torch.where(frac <= TOP / 512, ex - 9, ex - 8)
            e = torch.where(frac == 0, E_MIN, e).clamp(min=E_MIN)
            begun = mine[:, 0, 0, 0][:, None]
            old = scales[ids[lo : lo + m]]
            e_old = torch.where(begun | old.isnan(), E_MIN, _exponent(old))
            bad = (~good).any(3).any(1) | (old.isnan() & ~begun)
            e = torch.maximum(e, e_old)
            now = _encode8(fresh.where(good, 0.0) * _pow2(-e)[:, None, :, None])
            kept = _decode8(codes[ids[lo : lo + m]]) * _pow2((e_old - e).clamp(min=-126))[:, None, :, None]
            kept = torch.where(begun[:, :, None, None], 0.0, kept)
            codes[ids[lo : lo + m]] = torch.where(mine, now, _encode8(kept))
            scales[ids[lo : lo + m]] = torch.where(bad, math.nan, _pow2(e))


def _plain_rows(st: dict, layer: int, loc: torch.Tensor):
    b, s = loc // BLOCK, loc % BLOCK
    return tuple(_decode8(st[c][layer][b, s]) * st[x][layer][b][:, :, None] for c, x in (("kc", "ks"), ("vc", "vs")))


def _plain_context(st: dict, layer: int, i: int, n: int, pages: torch.Tensor | None = None):
    """K and V values of request i's first n tokens (or of the listed blocks), as float32."""
    b = st["blocks"][i][: -(-n // BLOCK)] if pages is None else st["blocks"][i][pages]
    out = []
    for c, x in (("kc", "ks"), ("vc", "vs")):
        y = _decode8(st[c][layer][b]) * st[x][layer][b][:, None, :, None]
        y = y.view(-1, *y.shape[2:])
        out.append(y[:n] if pages is None else y)
    return out


def _plain_bounds(st: dict, lo: list[int], hi: list[int]) -> None:
    """Bounds of the pages that tokens lo .. hi complete, over every layer."""
    for layer in range(st["kc"].shape[0]):
        for i, (a, b) in enumerate(zip(lo, hi)):
            p0, p1 = a // BLOCK, b // BLOCK
            if p1 > p0:
                ids = st["blocks"][i][p0:p1]
                k = _decode8(st["kc"][layer][ids]) * st["ks"][layer][ids][:, None, :, None]
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
    q = st["q"][layer, i]
    qbar = _mean_query(q, case["kv"]).float()
    lim = s // BLOCK - 1 if case["avoid"] else s // BLOCK
    lim = min(lim, (s - 1) // BLOCK)  # a page that the new token completes has no bounds yet
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
                k, v = _plain_rows(st, layer, _at(st["blocks"][i], _plain_select(st, layer, i, s)))
            else:
                k, v = _plain_context(st, layer, i, s)
            out.append(_plain_attend(st["q"][layer, i][None], k, v, st["scale"]))
        outs.append(torch.cat(out))
    return outs


def _at(blocks: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    return blocks[pos // BLOCK] * BLOCK + pos % BLOCK


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


def _plain_assign(st: dict, rpi, prefix, new, total: int):
    held = st["held"][rpi].long()
    blocks = (prefix + new + BLOCK - 1) // BLOCK
    need = (blocks - held).clamp(min=0)
    first = need.cumsum(0) - need
    # the free blocks' stack, from its top
    k = torch.arange(st["free"].numel(), device=DEV)
    taken = k < need.sum()
    i = torch.searchsorted(need.cumsum(0), k, right=True).clamp(max=rpi.numel() - 1)
    block = st["free"][(st["count"] - 1 - k).clamp(min=0)]
    where = torch.where(taken, rpi[i] * st["table"].shape[1] + held[i] + k - first[i], 0)
    flat = st["table"].view(-1)
    flat.scatter_add_(0, where, torch.where(taken, block - flat[where], 0))
    st["held"][rpi] = torch.maximum(held, blocks).to(torch.int32)
    st["count"] -= need.sum()
    i = torch.repeat_interleave(torch.arange(rpi.numel(), device=DEV), new, output_size=total)
    pos = prefix[i] + torch.arange(total, device=DEV) - (new.cumsum(0) - new)[i]
    loc = st["table"][rpi[i], pos // BLOCK].long() * BLOCK + pos % BLOCK
    st["r2t"][rpi[i], pos] = loc.to(torch.int32)
    return loc, pos


def _plain_release(st: dict, rpi) -> None:
    held = st["held"][rpi].long()
    last = held.cumsum(0)
    k = torch.arange(st["free"].numel(), device=DEV)
    given = k < last[-1]
    i = torch.searchsorted(last, k, right=True).clamp(max=rpi.numel() - 1)
    block = st["table"][rpi[i], torch.where(given, k - (last - held)[i], 0)]
    where = torch.where(given, st["count"] + last[-1] - 1 - k, 0)
    st["free"].scatter_add_(0, where, torch.where(given, block - st["free"][where], 0))
    st["table"][rpi] = 0
    st["r2t"][rpi] = 0
    st["held"][rpi] = 0
    st["count"] += last[-1]


# ---------------------------------------------------------------- one pass


def run(state: dict):
    kind = state["kind"]
    if kind == "slots":
        return _run_slots(state)
    if kind == "store":
        if own:
            pool = state["pool"]
            pool.set_kv_buffer(0, state["loc"], state["k"], state["v"])
            return [*pool.get_rows(0, state["back"]), pool.k_scale[0], pool.v_scale[0]]
        _plain_store(state, 0, state["loc"], state["k"], state["v"])
        k, v = _plain_rows(state, 0, state["back"])
        return [k.to(torch.bfloat16), v.to(torch.bfloat16), state["ks"][0], state["vs"][0]]
    if kind == "bounds":
        if own:
            state["quest"].update_prefill_representations_blocks(
                state["rpi"], state["seq"], state["kvp"], state["rtp"].block_table, prefix_lens=state["prefix"])
            return state["quest"].page_k_bounds
        _plain_bounds(state, state["prefix"], [p + n for p, n in zip(state["prefix"], state["new"])])
        return state["bounds"]
    if kind == "extend":
        if own:
            return state["be"].forward_extend(state["q"], state["k"], state["v"], state["layer"], state["batch"])
        return _plain_extend(state)
    if own:
        state["graph"].replay()
        return state["out"]
    return _plain_decode(state)


def _run_slots(st: dict):
    if own:
        pool = st["pool"]
        loc, pos = pool.assign(st["rpi"], st["prefix"], st["new"], st["total"])
        if st["finish"]:
            pool.release(st["rpi"])
        return [loc, pos, pool.block_table, pool.req_to_token, pool.held, pool.free_blocks]
    loc, pos = _plain_assign(st, st["rpi"], st["prefix"], st["new"], st["total"])
    if st["finish"]:
        _plain_release(st, st["rpi"])
    return [loc, pos, st["table"], st["r2t"], st["held"], st["free"]]


# ---------------------------------------------------------------- the same in 64 bits


def _pow64(e: torch.Tensor) -> torch.Tensor:
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_cache(writes: list[torch.Tensor]):
    """Values [blocks * 64, KV, D] and scales [blocks, KV] after writing these runs of tokens one
    after the other from position 0, each element by the definition in 64 bits."""
    n = sum(w.shape[0] for w in writes)
    kv, D = writes[0].shape[1:]
    blocks = -(-n // BLOCK)
    values = torch.zeros((blocks * BLOCK, kv, D), dtype=torch.float64, device=DEV)
    expo = torch.full((blocks, kv), E_MIN, dtype=torch.int64, device=DEV)
    at = 0
    for w in writes:
        m = w.shape[0]
        if not m:
            continue
        b0, b1 = at // BLOCK, -(-(at + m) // BLOCK)
        cover = torch.zeros(((b1 - b0) * BLOCK, kv, D), dtype=torch.float64, device=DEV)
        cover[at - b0 * BLOCK : at - b0 * BLOCK + m] = w.double()
        high = cover.view(b1 - b0, BLOCK, kv, D).abs().amax((1, 3))
        mant, ex = torch.frexp(high / TOP)  # high <= 448 * 2 ** ex, with equality at a mantissa of a half
        need = torch.where(mant == 0.5, ex - 1, ex).long().masked_fill(high == 0, E_MIN).clamp(min=E_MIN)
        grown = torch.maximum(need, expo[b0:b1])
        if at % BLOCK == 0:
            grown[0] = need[0]
        expo[b0:b1] = grown
        unit = _pow64(grown).repeat_interleave(BLOCK, 0)[:, :, None]
        span = values[b0 * BLOCK : b1 * BLOCK]
        span[at - b0 * BLOCK : at - b0 * BLOCK + m] = w.double()
        y = span / unit
        _, ye = torch.frexp(y)
        fine = _pow64((ye - 1).clamp(min=-6) - 3)
        span.copy_(torch.round(y / fine) * fine * unit)
        at += m
    return values, _pow64(expo)


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


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "slots":
        return _exact_slots(case, seed)
    q, kv_of, prefix, new = _source(case, seed)
    layers, kv, D = case.get("layers", 1), case["kv"], case["dim"]
    if kind == "store":
        blocks = _scatter_rows(prefix, new, seed)
        rows, scales = ([], []), [torch.full((sum(b.numel() for b in blocks) + 1, kv), 2.0**E_MIN, dtype=torch.float64,
                                             device=DEV) for _ in range(2)]
        for i, p in enumerate(prefix):
            for j, x in enumerate(kv_of(0, i)):
                val, sc = _exact_cache([x[:p], x[p:]])
                rows[j].append(val[p // BLOCK * BLOCK : p + new[i]])
                scales[j][blocks[i]] = sc
        return [torch.cat(rows[0]), torch.cat(rows[1]), *scales]
    if kind == "bounds":
        pages = -(-(max(p + n for p, n in zip(prefix, new)) + BLOCK) // BLOCK)
        out = torch.empty((layers, case["bs"], pages, kv, D, 2), dtype=torch.float64, device=DEV)
        out[..., 0], out[..., 1] = FAR, -FAR
        for layer in range(layers):
            for i, (p, n) in enumerate(zip(prefix, new)):
                # a page that the prefix left unfinished is finished later, at its scale of then
                full = (p + n) // BLOCK
                k = _exact_cache([x for x in kv_of(layer, i)[0].split([p, n])])[0][: full * BLOCK].view(full, BLOCK, kv, D)
                out[layer, i, :full, :, :, 0], out[layer, i, :full, :, :, 1] = k.amin(1), k.amax(1)
        return out
    outs = []
    for layer in range(layers):
        out, at = [], 0
        for i, (p, n) in enumerate(zip(prefix, new)):
            src = kv_of(layer, i)
            k, v = (_exact_cache([x[:p], x[p:]])[0][: p + n] for x in src)
            if kind == "extend":
                for a in range(0, n, 1024):
                    b = min(n, a + 1024)
                    out.append(_attend64(q[layer, at + a : at + b], k[: p + b], v[: p + b], D**-0.5, p + a))
            else:
                s = p + 1
                if kind == "sparse" and s > case["top_k"]:
                    pos = _exact_select(case, q[layer, i], _exact_cache([src[0][:p]])[0], s)
                    k, v = k[pos], v[pos]
                out.append(_attend64(q[layer, i][None], k, v, D**-0.5))
            at += n
        outs.append(torch.cat(out))
    return outs[0] if kind == "extend" else outs


def _exact_select(case: dict, q: torch.Tensor, k: torch.Tensor, s: int) -> torch.Tensor:
    pages = s // BLOCK
    lim = min(pages - 1 if case["avoid"] else pages, (s - 1) // BLOCK)
    kp = k[: lim * BLOCK].view(lim, BLOCK, *k.shape[1:])
    qbar = _mean_query(q, case["kv"]).double()  # the mean query's rounding is part of the method
    score = torch.maximum(qbar * kp.amax(1), qbar * kp.amin(1)).sum((1, 2))
    top = torch.sort(score, descending=True, stable=True).indices[: case["top_k"] // BLOCK - 1]
    return torch.cat([(top[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(),
                      torch.arange(s - BLOCK, s, device=DEV)])


def _exact_slots(case: dict, seed: int):
    prefix, new = _lens(case)
    bs, width = case["bs"], max(p + n for p, n in zip(prefix, new)) + BLOCK
    free = list(range(sum(_blocks_of(prefix, new)) + 8, 0, -1))  # its memory keeps what is taken off it
    table, stack = [[] for _ in range(bs)], list(free)

    def grow(rows, lens):
        for i, n in zip(rows, lens):
            while len(table[i]) * BLOCK < n:
                table[i].append(stack.pop())

    for rows, a, n in _admissions(case, seed):
        grow(rows, [x + y for x, y in zip(a, n)])
    order = list(range(bs))
    random.Random(seed + 1).shuffle(order)
    grow(order, [prefix[i] + new[i] for i in order])
    pos = torch.cat([torch.arange(prefix[i], prefix[i] + new[i]) for i in order])
    loc = torch.cat([torch.tensor(table[i])[torch.arange(prefix[i], prefix[i] + new[i]) // BLOCK] for i in order]) * BLOCK + pos % BLOCK
    t = torch.zeros((bs, -(-width // BLOCK)), dtype=torch.int32)
    r = torch.zeros((bs, width), dtype=torch.int32)
    held = torch.zeros(bs, dtype=torch.int32)
    if not case["finish"]:
        for i in range(bs):
            t[i, : len(table[i])] = torch.tensor(table[i], dtype=torch.int32)
            held[i] = len(table[i])
            p = torch.arange(prefix[i] + new[i])
            r[i, : p.numel()] = (torch.tensor(table[i])[p // BLOCK] * BLOCK + p % BLOCK).to(torch.int32)
    out = [loc, pos, t, r, held, torch.tensor(free, dtype=torch.int32)]
    return [x.to(DEV) for x in out]
