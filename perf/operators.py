"""The paged 4-bit KV cache's operators, case by case: what each is given, its plain form in torch, and the calls a program makes.

Three kinds of case:

* ``attend``: one layer of a serving step.  The step's new K / V tokens are quantised into the pages of their
  sequences and the queries attend the pages (``PagedKVCache.write`` and ``.attend``).  With ``append`` false
  nothing is written: queries of another stream attend a stored context (``causal`` false).
* ``store``: a prompt's K / V go into the pages of one sequence and are read back as dense cells, as an evicted or
  re-used prefix is (``PagedKVCache.write`` and ``.read``).  The values read back are what the 4-bit codes stand for.
* ``copy``: pages of a paged cache of any element type are copied in every layer (``ops.copy_pages``), as forked
  sequences and compaction need.

A token's head is held as groups of ``group`` elements: ``x = zero + scale * q``, q in [-8, 7], scale = (max - min) / 15
and zero = min + 8 scale, both rounded to float16; q is rounded half to even.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LIMIT = 65024.0  # magnitudes beyond this are stored as this


def listed():
    def attend(name, B, T, tq, Hq, Hkv, d, dtype, page, *, group=0, causal=True, append=True, ragged=False):
        return {"name": name, "kind": "attend", "B": B, "T": T, "tq": tq, "Hq": Hq, "Hkv": Hkv, "d": d, "dtype": dtype, "page": page,
                "group": group or d, "causal": causal, "append": append, "ragged": ragged}

    def store(name, T, Hkv, d, dtype, page, *, group=0):
        return {"name": name, "kind": "store", "T": T, "Hkv": Hkv, "d": d, "dtype": dtype, "page": page, "group": group or d}

    def copy(name, layers, pages, pairs, page, Hkv, d, dtype):
        return {"name": name, "kind": "copy", "layers": layers, "pages": pages, "pairs": pairs, "page": page, "Hkv": Hkv, "d": d, "dtype": dtype}

    return [
        # one token of a short chat on a small model (TinyLlama's heads): the host's and the launches' latency is all there is
        attend("decode 1 x 17, d 64", 1, 17, 1, 32, 4, 64, "bf16", 16),
        # the same model's full context in its own type, fp32
        attend("decode 1 x 2048, d 64 fp32", 1, 2048, 1, 32, 4, 64, "fp32", 64),
        # a serving batch on Llama-3-8B's heads at the repository's headline context
        attend("decode 8 x 32768", 8, 32768, 1, 32, 8, 128, "bf16", 64),
        # long contexts on Qwen2-7B's heads (7 queries a KV head), few rows: the context is what is split
        attend("decode 4 x 131072, 7 a head", 4, 131072, 1, 28, 4, 128, "bf16", 128),
        # a ragged batch in fp16 with small pages and groups of 32
        attend("decode 33 ragged to 8191 fp16", 33, 8191, 1, 32, 8, 128, "fp16", 16, group=32, ragged=True),
        # four drafted tokens a sequence verified at once, Llama-3-70B's heads
        attend("verify 8 x 4 of 8192", 8, 8192, 4, 64, 8, 128, "bf16", 32, ragged=True),
        # a prompt's chunk that arrives after 6144 cached tokens
        attend("chunk 2048 of 8192", 1, 8192, 2048, 32, 8, 128, "bf16", 64),
        # 1001 decoder positions over a stored context of 1500 tokens: no causal mask, nothing written, odd sizes
        attend("cross 2 x 1001 over 1500 fp16", 2, 1500, 1001, 12, 12, 64, "fp16", 32, causal=False, append=False),
        # a short odd prompt of the fp32 model stored and read back
        store("store 37, d 64 fp32", 37, 4, 64, "fp32", 16),
        # one layer of a long prompt stored and read back (the read is what an eviction does)
        store("store 32768", 32768, 8, 128, "bf16", 64),
        # the last pages of three forked sequences of the small model, K and V of a layer
        copy("copy 3 pages", 2, 64, 3, 16, 4, 64, "fp32"),
        # a compaction's moves in all 32 layers of Llama-3-8B's heads
        copy("copy 300 pages x 32", 32, 1024, 300, 16, 8, 128, "bf16"),
    ]


HEADS = ((32, 4, 64), (12, 12, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128), (16, 1, 128))


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "prompt", "store", "copy"))
    Hq, Hkv, d = rng.choice(HEADS)
    dtype, page = rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice((16, 32, 64, 128))
    group = rng.choice((d, d, d // 2, 32))
    if kind == "attend":  # decoding and verifying: the cache's bytes are bounded by the largest listed case's
        T = _log(rng, 1, 65536)
        B = _log(rng, 1, max(1, min(64, 2 ** 28 // (T * Hkv * d))))
        tq = min(T, rng.choice((1, 1, 1, 2, 3, 5, 8)))
        return {"kind": "attend", "B": B, "T": T, "tq": tq, "Hq": Hq, "Hkv": Hkv, "d": d, "dtype": dtype, "page": page, "group": group,
                "causal": True, "append": True, "ragged": rng.random() < 0.5}
    if kind == "prompt":  # chunks of prompts, and queries over a stored context
        tq = _log(rng, 9, 1200 if dtype != "fp32" else 400)
        causal = rng.random() < 0.75
        T = _log(rng, tq if causal else 1, 6000)
        B = _log(rng, 1, max(1, min(8, 2 ** 28 // (Hq * tq * T))))
        return {"kind": "attend", "B": B, "T": T, "tq": tq, "Hq": Hq, "Hkv": Hkv, "d": d, "dtype": dtype, "page": page, "group": group,
                "causal": causal, "append": causal, "ragged": rng.random() < 0.5}
    if kind == "store":
        return {"kind": "store", "T": _log(rng, 1, 20000), "Hkv": Hkv, "d": d, "dtype": dtype, "page": page, "group": group}
    pages = _log(rng, 8, 900)
    return {"kind": "copy", "layers": rng.randint(1, 32), "pages": pages, "pairs": rng.randint(1, pages // 3), "page": page if page < 64 else 16, "Hkv": Hkv,
            "d": d, "dtype": dtype if dtype != "fp32" else "fp16"}


def _lengths(case):
    """Cached tokens of each sequence, the step's own among them."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    r = random.Random(B * 1000003 + T)
    least = min(T, case["tq"]) if case["append"] else 1
    return [T] + [r.randint(least, T) for _ in range(B - 1)]


def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["page"] * case["Hkv"] * case["d"] * DTYPES[case["dtype"]].itemsize, "flops": 0}
    d, e = case["d"], DTYPES[case["dtype"]].itemsize
    held = case["Hkv"] * (d + 8 * (d // case["group"]))  # bytes of a token's K and V in 4 bits, with their parameters
    if case["kind"] == "store":  # K and V in, the codes written and read, K and V out
        return {"bytes": case["T"] * (2 * held + 4 * case["Hkv"] * d * e), "flops": 0}
    tq, ns = case["tq"], _lengths(case)
    new = tq * case["B"]
    seen = sum(sum(max(0, n - tq + 1 + i) for i in range(tq)) if case["causal"] else n * tq for n in ns)
    moved = 2 * new * case["Hq"] * d * e + sum(ns) * held
    if case["append"]:  # the step's own K and V are read once, and their codes written; they need not be read again
        moved += new * 2 * case["Hkv"] * d * e
    return {"bytes": moved, "flops": 4 * d * case["Hq"] * seen}


def _kv(B, T, Hkv, d, dtype, g):
    """K and V with a few loud and shifted channels in K, as rotated keys have, (B, T, Hkv, d)."""
    loud = torch.ones(d, device="cuda")
    shift = torch.zeros(d, device="cuda")
    at = torch.randperm(d, generator=g, device="cuda")[: max(1, d // 16)]
    loud[at] = 8.0
    shift[at[::2]] = 4.0
    k = torch.randn(B, T, Hkv, d, generator=g, device="cuda").mul_(loud).add_(shift).to(dtype)
    v = torch.randn(B, T, Hkv, d, generator=g, device="cuda").to(dtype)
    return k, v


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "copy":
        r = random.Random(seed)
        pool = torch.randn(case["layers"], case["pages"], case["page"], case["Hkv"], case["d"], generator=g, device="cuda", dtype=dtype)
        at = r.sample(range(case["pages"]), 2 * case["pairs"])
        return pool, at[: case["pairs"]], at[case["pairs"]:]
    if case["kind"] == "store":
        return _kv(1, case["T"], case["Hkv"], case["d"], dtype, g)
    k, v = _kv(case["B"], case["T"], case["Hkv"], case["d"], dtype, g)
    q = torch.randn(case["B"] * case["tq"], case["Hq"], case["d"], generator=g, device="cuda").to(dtype)
    return k, v, q


# ---- the plain form ------------------------------------------------------


def _quantise(x, group):
    """(rows, Hkv, d) -> packed codes and (scale, zero).  In 64 bits: codes next to a border are whole numbers that have to come out right."""
    g = x.double().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15).float().half()
    zero = (lo + 8 * scale.double()).float().half()
    s = scale.double().unsqueeze(-1)
    q = torch.where(s > 0, ((g - zero.double().unsqueeze(-1)) / s).round(), 0.0).clamp(-8, 7).add(8).to(torch.uint8).flatten(-2)
    return q[..., 0::2] << 4 | q[..., 1::2], torch.stack((scale, zero), -1)


def _values(codes, params, group):
    """float32 values of packed codes."""
    q = torch.stack((codes >> 4, codes & 15), -1).flatten(-2).float() - 8
    p = params.float().unsqueeze(-2)
    return (q.unflatten(-1, (-1, group)) * p[..., 0] + p[..., 1]).flatten(-2)


def _plain_pages(case, ns, g_seed):
    """Empty pages in a shuffled order: codes and parameters by slot, the slots of each sequence's positions."""
    page, B = case["page"], len(ns)
    most = max(ns)
    each = -(-most // page)
    order = torch.randperm(B * each, generator=torch.Generator().manual_seed(g_seed)).cuda().view(B, each)
    at = torch.arange(most, device="cuda")
    slots = order[:, at // page] * page + at % page
    n, d, groups = B * each * page, case["d"], case["d"] // case["group"]
    codes = torch.zeros(2, n, case["Hkv"], d // 2, dtype=torch.uint8, device="cuda")
    params = torch.zeros(2, n, case["Hkv"], groups, 2, dtype=torch.float16, device="cuda")
    return codes, params, slots


def _plain_write(s, slots, k, v):
    for i, x in enumerate((k, v)):
        s["codes"][i][slots], s["params"][i][slots] = _quantise(x, s["group"])


def _plain_read(s, slots):
    return [_values(s["codes"][i][slots], s["params"][i][slots], s["group"]) for i in (0, 1)]


def _plain_attend(s):
    k, v = _plain_read(s, s["slots"])  # (B, T, Hkv, d)
    q, Hkv, tq = s["q"].float(), k.shape[2], s["tq"]
    B, T = k.shape[:2]
    Hq, d = q.shape[1:]
    q = q.view(B, tq, Hkv, Hq // Hkv, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, d)
    w = (q @ k.permute(0, 2, 3, 1)).mul_(d ** -0.5).view(B, Hkv, -1, tq, T)
    w.masked_fill_(~s["mask"][:, None, None], -math.inf)
    most = w.amax(-1, keepdim=True)
    w.sub_(torch.where(most > -math.inf, most, 0.0)).exp_()
    total = w.sum(-1, keepdim=True)
    out = w.view(B, Hkv, -1, T) @ v.transpose(1, 2)
    out = out.view(B, Hkv, -1, tq, d) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).reshape(B * tq, Hq, d).to(s["q"].dtype)


def _mask(case, ns):
    """(B, tq, T): which positions a query sees."""
    n = torch.tensor(ns, device="cuda").view(-1, 1, 1)
    at = torch.arange(case["T"], device="cuda")
    if not case["causal"]:
        return (at < n).expand(-1, case["tq"], -1)
    return at <= n - case["tq"] + torch.arange(case["tq"], device="cuda").view(1, -1, 1)


# ---- what a program has in hand --------------------------------------------


def _own_cache(case, ns):
    """A cache whose free pages lie far apart, as they do after some time of serving, and an empty sequence for each of `ns`."""
    from kvcompress_b200 import PagedKVCache

    page = case["page"]
    pages = sum(-(-n // page) for n in ns)
    others = min(64, pages)
    rounds = pages // others
    cache = PagedKVCache(n_layers=1, n_pages=pages, n_kv_heads=case["Hkv"], head_dim=case["d"], page_size=page, group_size=case["group"],
                         max_sequences=max(others, len(ns)), max_tokens=max(max(ns), rounds * page), device="cuda")
    held = [cache.add() for _ in range(others)]
    for _ in range(rounds):
        cache.extend(held, [page] * others)
    random.Random(pages).shuffle(held)
    for s in held:
        cache.free(s)
    return cache, [cache.add() for _ in ns]


def prepare(case, seed):
    if case["kind"] == "copy":
        pool, src, dst = _inputs(case, seed)
        if not own:
            src, dst = torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")
        return {"kind": "copy", "pool": pool, "src": src, "dst": dst}
    if case["kind"] == "store":
        k, v = _inputs(case, seed)
        s = {"kind": "store", "k": k[0], "v": v[0], "group": case["group"], "dtype": k.dtype}
        if own:
            s["cache"], (s["seq"],) = _own_cache(case, [case["T"]])
            s["step"] = s["cache"].extend([s["seq"]], [case["T"]])
        else:
            s["codes"], s["params"], slots = _plain_pages(case, [case["T"]], seed)
            s["slots"] = slots[0]
        return s
    k, v, q = _inputs(case, seed)
    ns, tq = _lengths(case), case["tq"]
    new = tq if case["append"] else 0
    n = torch.tensor(ns, device="cuda").view(-1, 1)
    at = torch.arange(case["T"], device="cuda")
    old, now = at < n - new, (at >= n - new) & (at < n)
    s = {"kind": "attend", "q": q, "k": k[now], "v": v[now], "group": case["group"], "tq": tq, "append": case["append"], "causal": case["causal"]}
    if own:
        s["cache"], seqs = _own_cache(case, ns)
        before = s["cache"].extend(seqs, [m - new for m in ns])
        if sum(ns) > new * len(ns):
            s["cache"].write(0, k[old], v[old], before)
        s["step"] = s["cache"].extend(seqs, [tq] * len(ns)) if case["append"] else s["cache"].view(seqs, [tq] * len(ns))
    else:
        s["codes"], s["params"], s["slots"] = _plain_pages(case, ns, seed)
        _plain_write(s, s["slots"][old], k[old], v[old])
        s["new"], s["mask"] = s["slots"][now], _mask(case, ns)
    return s


def run(s):
    if s["kind"] == "copy":
        if own:
            from kvcompress_b200 import ops

            ops.copy_pages(s["pool"], s["src"], s["dst"])
        else:
            s["pool"][:, s["dst"]] = s["pool"][:, s["src"]]
        return s["pool"]
    if s["kind"] == "store":
        if own:
            s["cache"].write(0, s["k"], s["v"], s["step"])
            k, v = s["cache"].read(s["seq"], dtype=s["dtype"])
            return k[0], v[0]
        _plain_write(s, s["slots"], s["k"], s["v"])
        k, v = _plain_read(s, s["slots"])
        return k.to(s["dtype"]).transpose(0, 1), v.to(s["dtype"]).transpose(0, 1)
    if own:
        if s["append"]:
            s["cache"].write(0, s["k"], s["v"], s["step"])
        return s["cache"].attend(0, s["q"], s["step"], causal=s["causal"])
    if s["append"]:
        _plain_write(s, s["new"], s["k"], s["v"])
    return _plain_attend(s)


# ---- the definition in 64 bits ----------------------------------------------


def _exact_values(x, group):
    """What a token's head is held as, in float64."""
    x = torch.clip(x.to(torch.float64), -LIMIT, LIMIT)
    parts = []
    for part in x.split(group, dim=-1):
        low, high = part.min(dim=-1, keepdim=True).values, part.max(dim=-1, keepdim=True).values
        step = torch.div(high - low, 15.0).to(torch.float32).to(torch.float16).to(torch.float64)
        mid = (low + step * 8.0).to(torch.float32).to(torch.float16).to(torch.float64)
        level = torch.clip(torch.round((part - mid) / torch.where(step == 0, math.inf, step)), -8.0, 7.0)
        parts.append(mid + step * level)
    return torch.cat(parts, dim=-1)


def exact(case, seed):
    if case["kind"] == "copy":
        return None
    if case["kind"] == "store":
        return tuple(_exact_values(x[0], case["group"]).permute(1, 0, 2) for x in _inputs(case, seed))
    k, v, q = _inputs(case, seed)
    tq, ratio = case["tq"], case["Hq"] // case["Hkv"]
    out = torch.zeros(case["B"] * tq, case["Hq"], case["d"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        for h in range(case["Hkv"]):
            keys, vals = _exact_values(k[b, :n, h], case["group"]), _exact_values(v[b, :n, h], case["group"])
            for j in range(h * ratio, (h + 1) * ratio):
                logit = torch.einsum("id,td->it", q[b * tq:(b + 1) * tq, j].double(), keys) / math.sqrt(case["d"])
                if case["causal"]:
                    i, t = torch.arange(tq, device="cuda"), torch.arange(n, device="cuda")
                    logit[t[None, :] > n - tq + i[:, None]] = -math.inf
                some = logit.max(dim=1).values > -math.inf
                out[b * tq:(b + 1) * tq, j][some] = torch.softmax(logit[some], dim=1) @ vals
    return out
