"""Performance cases of decoding with beams over a paged 16-bit key-value cache.

A case is one pass through one operator, as a serving program calls it:

  rope     rotary positions (with the per-head RMS norms where the model has them) of a
           step's queries and keys, and the writing of keys and values into the pages
  attn     attention of one new token per sequence over the pages
  reorder  beams go on from their parents: whole pages shared, the written page copied,
           pages that nobody holds freed, room for the next token
  compact  a serving loop's step that retires its oldest sequences, packs the pages that
           are left, and admits as many new ones
  beam     the n best of beams x vocabulary from the logits and the beams' scores

The page table is base_rows int32 [sequences, pages of a sequence]: the first row of the
page that holds positions [j << page_shift, (j + 1) << page_shift), or -1.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a decode step of 16 streams in a layer with 8 kv heads: norms, half pairs
        dict(name="rope_decode_16", kind="rope", seqs=_decode(16, 4096), nq=16, nkv=8, hd=256, half=128,
             stride=128, inter=False, norm=True, base=10000.0, factor=1.0, fused=False, dtype="bf16", shift=10),
        # a ragged prompt step far into two long contexts: interleaved pairs on half of the
        # head, scaled frequencies, q, k and v in one buffer
        dict(name="rope_prompt_2159_far", kind="rope", seqs="0:700,130100:411,1000003:1048", nq=32, nkv=8, hd=128,
             half=32, stride=0, inter=True, norm=False, base=500000.0, factor=32.0, fused=True, dtype="f16", shift=4),
        # one chat stream in a sliding layer
        dict(name="attn_1_sliding", kind="attn", seqs=1, ctx=1500, nq=16, nkv=8, hd=256, window=1024, cap=0.0,
             dtype="bf16", shift=10),
        # a few short streams with small pages and three query heads per kv head
        dict(name="attn_7_short", kind="attn", seqs=7, ctx=333, nq=24, nkv=8, hd=64, window=0, cap=50.0,
             dtype="f16", shift=3),
        # a full batch in a layer that sees every position
        dict(name="attn_16_full", kind="attn", seqs=16, ctx=4096, nq=16, nkv=2, hd=512, window=0, cap=0.0,
             dtype="bf16", shift=10),
        # a large batch with long contexts
        dict(name="attn_64_long", kind="attn", seqs=64, ctx=16384, nq=32, nkv=8, hd=128, window=0, cap=0.0,
             dtype="bf16", shift=4),
        # four beams of one request, an int8 cache with its scales
        dict(name="reorder_1x4_int8", kind="reorder", groups=1, beams=4, ctx=1500, layers=4, values=2048, dtype="int8",
             shift=6),
        # 32 requests of 8 beams, a 16-bit cache
        dict(name="reorder_32x8", kind="reorder", groups=32, beams=8, ctx=1000, layers=4, values=2048, dtype="bf16",
             shift=6),
        # a few sequences, of which one is replaced
        dict(name="compact_5", kind="compact", seqs=5, retire=1, ctx=333, layers=2, values=1024, dtype="bf16", shift=4),
        # a large batch, of which an eighth is replaced
        dict(name="compact_64", kind="compact", seqs=64, retire=8, ctx=2000, layers=4, values=2048, dtype="int8",
             shift=6),
        # four beams of one request over the whole vocabulary
        dict(name="beam_1x4", kind="beam", batch=1, beams=4, vocab=262144, n=4, done=False, dtype="bf16"),
        # 32 requests of 8 beams, some of them ended, twice as many candidates
        dict(name="beam_32x8", kind="beam", batch=32, beams=8, vocab=262144, n=16, done=True, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "reorder", "compact", "beam"])
    if kind == "rope":
        nq, nkv, hd, half, stride = rng.choice([(16, 8, 256, 128, 128), (16, 2, 512, 64, 256), (32, 8, 128, 64, 64),
                                                (12, 4, 64, 24, 24), (20, 20, 128, 16, 16)])
        inter = rng.random() < 0.5
        n = _log(rng, 1, 1800)
        first = rng.choice([0, rng.randrange(1, 5000), rng.randrange(100000, 1000000)])
        seqs = "%d:%d" % (first, n) if rng.random() < 0.5 else "%d:%d,%d:%d" % (first, n, rng.randrange(0, 3000), _log(rng, 1, 250))
        if rng.random() < 0.4:
            seqs = _decode(_log(rng, 1, 128), _log(rng, 200, 30000))
        return dict(kind=kind, seqs=seqs, nq=nq, nkv=nkv, hd=hd, half=half, stride=0 if inter else stride, inter=inter,
                    norm=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0, 1000000.0]),
                    factor=rng.choice([1.0, 8.0, 40.0]), fused=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16"]),
                    shift=rng.randrange(3, 11))
    if kind == "attn":
        nq, nkv, hd = rng.choice([(16, 8, 256), (16, 2, 512), (32, 8, 128), (24, 8, 64), (8, 8, 128), (20, 4, 256), (32, 1, 128)])
        seqs = _log(rng, 1, 96)
        most = 64 * 16384 * 8 * 128 // (seqs * nkv * hd)
        return dict(kind=kind, seqs=seqs, ctx=_log(rng, 1, min(60000, most)), nq=nq, nkv=nkv, hd=hd,
                    window=rng.choice([0, 0, rng.randrange(1, 5000)]), cap=rng.choice([0.0, 0.0, 30.0]),
                    dtype=rng.choice(["bf16", "f16"]), shift=rng.randrange(3, 11))
    if kind == "reorder":
        beams = rng.randrange(2, 13)
        return dict(kind=kind, groups=_log(rng, 1, 20), beams=beams, ctx=_log(rng, 1, 1100), layers=rng.randrange(1, 5),
                    values=rng.choice([256, 512, 1024, 2048]), dtype=rng.choice(["int8", "bf16"]), shift=rng.randrange(3, 8))
    if kind == "compact":
        seqs = _log(rng, 2, 64)
        return dict(kind=kind, seqs=seqs, retire=max(1, seqs // rng.randrange(2, 9)), ctx=_log(rng, 1, 1900),
                    layers=rng.randrange(1, 4), values=rng.choice([256, 512, 1024, 2048]), dtype=rng.choice(["int8", "bf16"]),
                    shift=rng.randrange(3, 9))
    beams = rng.randrange(1, 17)
    batch = _log(rng, 1, max(1, 256 // beams))
    return dict(kind=kind, batch=batch, beams=beams, vocab=_log(rng, 500, 262144), n=min(32, rng.choice([beams, 2 * beams])),
                done=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16", "f32"]))


def _decode(n, ctx):
    """n sequences of one new token each, their lengths spread below ctx."""
    return ",".join("%d:1" % (ctx - 1 - (37 * i) % max(1, ctx // 2)) for i in range(n))


def _spread(n, ctx):
    """n lengths between ctx / 2 and ctx."""
    return [ctx - (37 * i) % max(1, ctx // 2) for i in range(n)]


def _steps(case):
    return [tuple(int(v) for v in s.split(":")) for s in case["seqs"].split(",")]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pages(gen, counts, shift, spare=0):
    """Tables of counts[i] pages each (lists of page indexes that exist, and the width) at
    random places of a pool: base_rows, pages in the pool."""
    width = max(max((max(c) + 1 for c in counts if c), default=1), 1)
    total = sum(len(c) for c in counts) + spare
    order = (torch.randperm(total, device=DEV, generator=gen) << shift).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, c in enumerate(counts):
        if c:
            table[i, c[0]:c[0] + len(c)] = order[at:at + len(c)]
        at += len(c)
    return table, total


def _normal(gen, shape, dtype, scale=1.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, scale, generator=gen)


def _norm_consts(hd):
    return math.sqrt(hd), hd * 1e-6


def _frequencies(case):
    """base ** (-2 i / rotated size), the slow pairs slowed further by the context's factor with a
    ramp between, and the magnitude that goes with the factor."""
    n = case["half"]
    f = case["base"] ** (-torch.arange(n, dtype=torch.float64) / n)
    ramp = torch.clamp((torch.arange(n, dtype=torch.float64) - 0.25 * n) / (0.5 * n), 0.0, 1.0)
    f = f * (1.0 - ramp) + f / case["factor"] * ramp
    return f.to(torch.float32).to(DEV), 0.1 * math.log(case["factor"]) + 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    kind, st = case["kind"], dict(case=dict(case))
    dt = TYPES.get(case["dtype"])
    shift = case.get("shift", 0)
    if kind == "rope":
        nq, nkv, hd, steps = case["nq"], case["nkv"], case["hd"], _steps(case)
        tokens = sum(n for _, n in steps)
        table, pages = _pages(gen, [list(range(p >> shift, ((p + n - 1) >> shift) + 1)) for p, n in steps], shift)
        if case["fused"]:
            qkv = _normal(gen, (tokens, (nq + 2 * nkv) * hd), dt)
            st["q"], st["k"], st["v"] = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
        else:
            st["q"], st["k"], st["v"] = (_normal(gen, (tokens, n * hd), dt) for n in (nq, nkv, nkv))
        st["k_cache"], st["v_cache"] = (_normal(gen, (pages << shift, nkv * hd), dt) for _ in range(2))
        st["positions"] = torch.cat([torch.arange(p, p + n, dtype=torch.int32, device=DEV) for p, n in steps])
        st["seq_ids"] = torch.cat([torch.full((n,), i, dtype=torch.int32, device=DEV) for i, (_, n) in enumerate(steps)])
        st["inv_freq"], st["mscale"] = _frequencies(case)
        st["q_norm"], st["k_norm"] = ((1.0 + _normal(gen, (hd,), torch.float32, 0.2)).to(dt) if case["norm"] else None
                                      for _ in range(2))
        st["base_rows"] = table
        st["out"] = torch.zeros((tokens, nq * hd), dtype=dt, device=DEV)
    elif kind == "attn":
        nkv, hd, lens = case["nkv"], case["hd"], _spread(case["seqs"], case["ctx"])
        table, pages = _pages(gen, [list(range(((n - 1) >> shift) + 1)) for n in lens], shift)
        st["q"] = _normal(gen, (case["seqs"], case["nq"] * hd), dt)
        st["k_cache"], st["v_cache"] = (_normal(gen, (pages << shift, nkv * hd), dt) for _ in range(2))
        st["base_rows"], st["kv_lens"], st["longest"] = table, _ints(lens), max(lens)
    elif kind in ("reorder", "compact"):
        rows = 1 << shift
        if kind == "reorder":
            k = case["beams"]
            lens = [n for n in _spread(case["groups"], case["ctx"]) for _ in range(k)]
            parents = []
            for g in range(case["groups"]):  # half of a request's beams go on twice
                live = (torch.randperm(k, device=DEV, generator=gen) + g * k)[:(k + 1) // 2]
                both = torch.cat([live, live[:k // 2]])
                parents.append(both[torch.randperm(k, device=DEV, generator=gen)])
            st["parents"] = torch.cat(parents).to(torch.int32)
            st["grow"] = torch.ones(len(lens), dtype=torch.int32, device=DEV)
            spare = 2 * len(lens)
        else:
            n, r = case["seqs"], case["retire"]
            lens = [case["ctx"]] * n
            st["leave"] = _ints([i + r if i + r < n else -1 for i in range(n)])
            st["parents"] = _ints([i if i < n - r else -1 for i in range(n)])
            st["grow"] = _ints([0 if i < n - r else case["ctx"] for i in range(n)])
            spare = r + 3
        table, pages = _pages(gen, [list(range(((n - 1) >> shift) + 1)) for n in lens], shift, spare)
        width = ((max(lens) + rows) >> shift) + 1
        st["base_rows"] = torch.cat([table, torch.full((len(lens), width - table.shape[1]), -1, dtype=torch.int32, device=DEV)], 1)
        st["lens"] = _ints(lens)
        st["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
        st["refs"][(table[table >= 0] >> shift).long()] = 1
        st["arrays"] = []
        for _ in range(2 * case["layers"]):
            if case["dtype"] == "int8":
                st["arrays"].append(torch.randint(-127, 128, (pages << shift, case["values"]), dtype=torch.int8, device=DEV, generator=gen))
                st["arrays"].append(_normal(gen, (pages << shift, case["values"] // 256), torch.float32).abs_())
            else:
                st["arrays"].append(_normal(gen, (pages << shift, case["values"]), dt))
    else:
        b, k, v = case["batch"], case["beams"], case["vocab"]
        st["logits"] = _normal(gen, (b * k, v), dt, 3.0)
        st["scores"] = -torch.empty((b, k), dtype=torch.float32, device=DEV).uniform_(5.0, 12.0, generator=gen)
        st["finished"] = (torch.rand((b, k), device=DEV, generator=gen) < 0.2).to(torch.uint8) if case["done"] else None
        st["eos"] = 1 if case["done"] else -1
    return st


def work(case):
    kind, size = case["kind"], {"bf16": 2, "f16": 2, "f32": 4, "int8": 1}[case["dtype"]]
    if kind == "rope":
        tokens = sum(n for _, n in _steps(case))
        values = tokens * (case["nq"] + 2 * case["nkv"]) * case["hd"]
        return {"bytes": 2 * size * values + 12 * tokens, "flops": 6 * values}
    if kind == "attn":
        lens = [min(n, case["window"]) if case["window"] else n for n in _spread(case["seqs"], case["ctx"])]
        return {"bytes": size * case["hd"] * (2 * case["nkv"] * sum(lens) + 2 * case["nq"] * len(lens)),
                "flops": 4 * case["nq"] * case["hd"] * sum(lens)}
    if kind == "beam":
        rows = case["batch"] * case["beams"]
        return {"bytes": size * rows * case["vocab"] + 12 * case["batch"] * case["n"], "flops": 4 * rows * case["vocab"]}
    row = 2 * case["layers"] * case["values"] * size + (2 * case["layers"] * (case["values"] // 256) * 4 if case["dtype"] == "int8" else 0)
    rows = 1 << case["shift"]
    if kind == "reorder":
        lens = _spread(case["groups"], case["ctx"])
        moved = sum(n % rows for n in lens) * (case["beams"] // 2)
        table = 8 * case["beams"] * sum(-(-(n + 1) // rows) for n in lens)
    else:
        n, r, each = case["seqs"], case["retire"], -(-case["ctx"] // rows)
        moved = r * each * rows * (n - r) // n  # the freed pages below the packed size, on average
        table = 24 * n * each
    return {"bytes": 2 * moved * row + table, "flops": 0}


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        bq = _framework()
        if kind == "rope":
            bq.rope_append(st["q"], st["k"], st["v"], st["inv_freq"], st["positions"], st["base_rows"], st["k_cache"],
                           st["v_cache"], case["nq"], case["nkv"], case["hd"], case["shift"], pair_stride=case["stride"],
                           mscale=st["mscale"], seq_ids=st["seq_ids"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                           norm_v=case["norm"], out=st["out"])
            return st["out"], st["k_cache"], st["v_cache"]
        if kind == "attn":
            return bq.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["base_rows"], st["kv_lens"], case["nq"],
                                      case["nkv"], case["hd"], case["shift"], window=case["window"], softcap=case["cap"],
                                      max_kv_len=st["longest"])
        if kind == "beam":
            return bq.beam_select(st["logits"], st["scores"], case["n"], finished=st["finished"], eos_id=st["eos"])
        reorder, compact = bq.cache_reorder, bq.cache_compact
    else:
        if kind == "rope":
            return _rope(st, case)
        if kind == "attn":
            return _attention(st, case)
        if kind == "beam":
            return _beam(st, case)
        reorder, compact = _reorder, _compact
    cache = st["arrays"], st["base_rows"], st["lens"], st["refs"]
    if kind == "reorder":
        info = reorder(*cache, st["parents"], case["shift"], grow=st["grow"])
        return info, st["base_rows"], st["lens"], st["refs"], st["arrays"]
    left = reorder(*cache, st["leave"], case["shift"])
    packed = compact(st["arrays"], st["base_rows"], st["refs"], case["shift"])
    info = reorder(*cache, st["parents"], case["shift"], grow=st["grow"])
    st["lens"].add_(st["grow"])
    return left, packed, info, st["base_rows"], st["lens"], st["refs"], st["arrays"]


def _framework():
    if "bq" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mojo-gemma4-cpu_amd"))
    import bq
    return bq


# ---- the operators in their plain form ------------------------------------------


def _rope(st, case):
    hd, n, dt = case["hd"], case["half"], st["q"].dtype
    angle = st["positions"].double()[:, None] * st["inv_freq"].double()
    cos, sin = ((st["mscale"] * t).float()[:, None, :] for t in (torch.cos(angle), torch.sin(angle)))
    sqrt_n, n_eps = _norm_consts(hd)

    def heads(x, gain, normed, turned):
        x = x.float().view(x.shape[0], -1, hd)
        if normed:
            x = x * (sqrt_n / torch.sqrt((x * x).sum(-1, keepdim=True) + n_eps))
            x = x * gain.float() if gain is not None else x
        if turned:
            first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["inter"] else (
                slice(0, n), slice(case["stride"], case["stride"] + n))
            a, b = x[..., first], x[..., second]
            y = x.clone()
            y[..., first] = a * cos - b * sin
            y[..., second] = b * cos + a * sin
            x = y
        return x.to(dt).view(x.shape[0], -1)

    at = st["positions"].long()
    slots = st["base_rows"][st["seq_ids"].long(), at >> case["shift"]].long() + (at & ((1 << case["shift"]) - 1))
    st["out"].copy_(heads(st["q"], st["q_norm"], case["norm"], True))
    st["k_cache"][slots] = heads(st["k"], st["k_norm"], case["norm"], True)
    st["v_cache"][slots] = heads(st["v"], None, case["norm"], False)
    return st["out"], st["k_cache"], st["v_cache"]


def _attention(st, case):
    s, nq, nkv, hd, shift = st["q"].shape[0], case["nq"], case["nkv"], case["hd"], case["shift"]
    at = torch.arange(st["longest"], device=DEV)
    lens = st["kv_lens"].long()[:, None]
    seen = (at < lens) & (at >= (lens - case["window"] if case["window"] else 0))
    slots = st["base_rows"][:, at >> shift].long() + (at & ((1 << shift) - 1))
    slots = torch.where(seen, slots, 0)
    k = st["k_cache"][slots].float().view(s, -1, nkv, hd).permute(0, 2, 3, 1)
    scores = torch.matmul(st["q"].float().view(s, nkv, nq // nkv, hd), k) * (1.0 / math.sqrt(hd))
    del k
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    scores = scores.masked_fill(~seen[:, None, None, :], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = st["v_cache"][slots].float().masked_fill(~seen[..., None], 0.0).view(s, -1, nkv, hd).permute(0, 2, 1, 3)
    return torch.matmul(p, v).reshape(s, nq * hd).to(st["q"].dtype)


def _page_of(table, shift, pages):
    """The page numbers of a table, -1 where there is none."""
    page = table.long() >> shift
    return torch.where((table >= 0) & ((table & ((1 << shift) - 1)) == 0) & (page < pages), page, -1)


def _held(pages, count):
    """How often each page stands in a table."""
    flat = pages.reshape(-1)
    got = torch.zeros(count + 1, dtype=torch.int64, device=DEV)
    return got.index_add_(0, torch.where(flat >= 0, flat, count), torch.ones_like(flat))[:count]


def _reorder(arrays, table, lens, refs, parents, shift, grow=None):
    n, width = table.shape
    rows, pages = 1 << shift, refs.shape[0]
    old = _page_of(table, shift, pages)
    alive = (parents >= 0) & (parents < n)
    parent = torch.where(alive, parents, 0).long()
    size = torch.where(alive, lens[parent].long().clamp(0, width * rows), 0)
    more = grow.long().clamp(min=0) if grow is not None else torch.zeros_like(size)
    full = size >> shift
    end = ((size + more + rows - 1) >> shift).clamp(max=width)
    j = torch.arange(width, device=DEV)
    kept = alive[:, None] & ((j < full[:, None]) | ((j == full[:, None]) & (j < end[:, None])))
    new = torch.where(kept, old[parent], -1)
    count = refs.long() - _held(old, pages) + _held(new, pages)
    # the page that a sequence goes on writing: its own, or one that others hold as well
    has = full < end
    last = torch.where(has, new.gather(1, full.clamp(max=width - 1)[:, None])[:, 0], -1)
    earlier = ((last[:, None] == last[None, :]) & (last >= 0)[:, None]).tril(-1).sum(1)
    leaves = (last >= 0) & (count[last.clamp(min=0)] - earlier > 1)
    free = torch.argsort((count != 0).to(torch.int8), stable=True)
    count -= _held(torch.where(leaves, last, -1), pages)
    fresh = (j >= full[:, None]) & (j < end[:, None]) & ((j > full[:, None]) | leaves[:, None] | (last < 0)[:, None])
    rank = (torch.cumsum(fresh.reshape(-1).long(), 0) - 1).view(n, width)
    there = (refs.long() - _held(old, pages) + _held(new, pages) == 0).sum()
    got = fresh & (rank < there)
    new = torch.where(got, free[rank.clamp(0, pages - 1)], torch.where(fresh, -1, new))
    count += _held(torch.where(got, new, -1), pages)
    into = new.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    copied = leaves & (into >= 0) & (size % rows > 0)
    k = torch.arange(rows, device=DEV)
    wanted = copied[:, None] & (k < (size % rows)[:, None])
    src, dst = ((p[:, None] * rows + k)[wanted] for p in (last, into))
    moved = [a[src] for a in arrays]
    for a, m in zip(arrays, moved):
        a[dst] = m
    table.copy_(torch.where(new >= 0, new << shift, -1))
    lens.copy_(size)
    refs.copy_(count)
    zero = torch.zeros((), dtype=torch.int64, device=DEV)
    return torch.stack([got.sum(), copied.sum(), fresh.sum() - got.sum(), zero]).to(torch.int32)


def _compact(arrays, table, refs, shift):
    pages = refs.shape[0]
    at = torch.arange(pages, device=DEV)
    live = refs != 0
    total = live.sum()
    holes, movers = torch.nonzero(~live & (at < total))[:, 0], torch.nonzero(live & (at >= total))[:, 0]
    to = at.clone()
    to[movers] = holes
    refs[holes] = refs[movers]
    refs[movers] = 0
    page = _page_of(table, shift, pages)
    table.copy_(torch.where(page >= 0, to[page.clamp(min=0)] << shift, table.long()))
    for a in arrays:
        whole = a.view(pages, -1)
        whole[holes] = whole[movers]
    zero = torch.zeros((), dtype=torch.int64, device=DEV)
    return torch.stack([total, zero + movers.shape[0], zero, zero]).to(torch.int32)


def _beam(st, case):
    b, k, v, n = case["batch"], case["beams"], case["vocab"], case["n"]
    x = st["logits"].double()
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    scores = st["scores"].double().view(b * k, 1) + (x - lse)
    if st["finished"] is not None:  # an ended beam goes on as it is, with the end token
        done = st["finished"].view(b * k, 1) != 0
        only = torch.arange(v, device=DEV) == st["eos"]
        scores = torch.where(done, torch.where(only, st["scores"].double().view(b * k, 1), float("-inf")), scores)
    scores = scores.view(b, k * v)
    least = torch.topk(scores, n, 1).values[:, -1:]
    rows, flat = torch.nonzero((scores >= least) & (scores > float("-inf")), as_tuple=True)
    value = scores[rows, flat]
    order = torch.argsort(-value, stable=True)
    order = order[torch.argsort(rows[order], stable=True)]
    rows, flat, value = rows[order], flat[order], value[order]
    rank = torch.arange(rows.shape[0], device=DEV) - torch.searchsorted(rows, torch.arange(b, device=DEV))[rows]
    first = rank < n
    rows, flat, value, rank = rows[first], flat[first], value[first], rank[first]
    out_s = torch.full((b, n), float("-inf"), dtype=torch.float32, device=DEV)
    out_p, out_t = (torch.full((b, n), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    out_s[rows, rank] = value.float()
    out_p[rows, rank] = (rows * k + flat // v).to(torch.int32)
    out_t[rows, rank] = (flat % v).to(torch.int32)
    if st["finished"] is None:
        return out_s, out_p, out_t
    was = torch.where(out_p >= 0, st["finished"].view(-1)[out_p.clamp(min=0).long()], 0)
    return out_s, out_p, out_t, ((was != 0) | (out_t == st["eos"])).to(torch.uint8)


# ---- the same in 64 bits, from the definitions ------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _rope_exact(st, case)
    if case["kind"] == "attn":
        return _attention_exact(st, case)
    if case["kind"] == "beam":
        return _beam_exact(st, case)
    return _cache_exact(st, case)


def _rope_exact(st, case):
    hd, n = case["hd"], case["half"]
    turn = torch.polar(torch.full((), st["mscale"], dtype=torch.float64, device=DEV).expand(st["positions"].shape[0], n),
                       st["positions"].double()[:, None] * st["inv_freq"].double())
    pair = torch.arange(n, device=DEV)
    first, second = (2 * pair, 2 * pair + 1) if case["inter"] else (pair, pair + case["stride"])

    def normed(x, gain):
        x = x.double().reshape(x.shape[0], -1, hd)
        if not case["norm"]:
            return x
        x = x / torch.sqrt((x.square().sum(-1) + hd * 1e-6) / hd)[..., None]
        return x if gain is None else x * gain.double()

    def turned(x):
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None, :]
        x[..., first], x[..., second] = z.real, z.imag
        return x

    q, k, v = turned(normed(st["q"], st["q_norm"])), turned(normed(st["k"], st["k_norm"])), normed(st["v"], None)
    caches = st["k_cache"].double(), st["v_cache"].double()
    place = [int(st["base_rows"][i, p >> case["shift"]]) + p % (1 << case["shift"])
             for i, p in zip(st["seq_ids"].tolist(), st["positions"].tolist())]
    for cache, x in zip(caches, (k, v)):
        cache[torch.tensor(place, device=DEV)] = x.reshape(len(place), -1)
    return (q.reshape(q.shape[0], -1), *caches)


def _attention_exact(st, case):
    nq, nkv, hd, rows = case["nq"], case["nkv"], case["hd"], 1 << case["shift"]
    out = []
    for i, n in enumerate(st["kv_lens"].tolist()):
        start = max(0, n - case["window"]) if case["window"] else 0
        bases = st["base_rows"][i].long()
        slots = (bases[:, None] + torch.arange(rows, device=DEV)).reshape(-1)[start:n]
        k, v = (st[c][slots].double().view(-1, nkv, hd).transpose(0, 1).contiguous() for c in ("k_cache", "v_cache"))
        q = st["q"][i].double().view(nkv, nq // nkv, hd)
        s = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        if case["cap"]:
            s = torch.tanh(s / case["cap"]) * case["cap"]
        out.append(torch.matmul(torch.softmax(s, -1), v).reshape(-1))
    return torch.stack(out)


def _beam_exact(st, case):
    b, k, v = case["batch"], case["beams"], case["vocab"]
    s = torch.log_softmax(st["logits"].double(), 1) + st["scores"].double().view(-1, 1)
    if st["finished"] is not None:
        for r in torch.nonzero(st["finished"].view(-1))[:, 0].tolist():
            s[r] = float("-inf")
            s[r, st["eos"]] = float(st["scores"].view(-1)[r])
    best = torch.topk(s.view(b, k * v), case["n"], 1, sorted=True).values
    return (best, None, None) if st["finished"] is None else (best, None, None, None)


def _cache_exact(st, case):
    """The pages followed one at a time on the host; the values move with them."""
    rows, shift = 1 << case["shift"], case["shift"]
    table, lens, refs = st["base_rows"].tolist(), st["lens"].tolist(), st["refs"].tolist()
    arrays = [a.double() for a in st["arrays"]]

    def go_on(parents, grow):
        nonlocal table, lens
        before, size = [list(t) for t in table], list(lens)
        width = len(before[0])
        for t in before:
            for e in t:
                if e >= 0:
                    refs[e >> shift] -= 1
        table, lens = [], []
        for p, g in zip(parents, grow):
            n = size[p] if p >= 0 else 0
            full, end = n // rows, min(width, -(-(n + g) // rows))
            table.append([before[p][j] if p >= 0 and j < min(full + 1, end) else -1 for j in range(width)])
            lens.append(n)
            for e in table[-1]:
                if e >= 0:
                    refs[e >> shift] += 1
        free = [p for p, r in enumerate(refs) if r == 0]
        todo = []
        for i, (n, g) in enumerate(zip(lens, grow)):
            full, end = n // rows, min(width, -(-(n + g) // rows))
            for j in range(full, end):
                source = table[i][j]
                if source >= 0 and refs[source >> shift] == 1:
                    continue
                if source >= 0:
                    refs[source >> shift] -= 1
                page = free.pop(0) if free else -1
                table[i][j] = page << shift if page >= 0 else -1
                if page >= 0:
                    refs[page] += 1
                    if source >= 0 and n % rows:
                        todo.append((source, page << shift, n % rows))
        for source, to, count in todo:
            for a in arrays:
                a[to:to + count] = a[source:source + count]

    n = len(lens)
    if case["kind"] == "reorder":
        go_on(st["parents"].tolist(), st["grow"].tolist())
        return [None, None, None, None, arrays]
    go_on(st["leave"].tolist(), [0] * n)
    live = [p for p, r in enumerate(refs) if r]
    holes = [p for p, r in enumerate(refs) if not r and p < len(live)]
    to = dict(zip([p for p in live if p >= len(live)], holes))
    for source, p in to.items():
        refs[p], refs[source] = refs[source], 0
        for a in arrays:
            a[p * rows:(p + 1) * rows] = a[source * rows:(source + 1) * rows]
    table = [[to.get(e >> shift, e >> shift) << shift if e >= 0 else -1 for e in t] for t in table]
    go_on(st["parents"].tolist(), st["grow"].tolist())
    return [None, None, None, None, None, None, arrays]
