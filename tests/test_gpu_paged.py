"""The paged 16-bit cache and beams on the GPU against 64-bit references: rotary
append, attention of one token per sequence, page reorder and compaction, beam
selection; rows that take no part, bad pages, lengths of zero and one, strides,
streams, captured graphs, far offsets."""
import math

import numpy as np
import pytest
import torch

from paged_cases import EPS, Pages, attention_ref, beam_ref, rope_ref, slot_of

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dt=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dt)


def tables(g, lens, shift, width, pool, slack=0):
    """Random distinct pages for positions [0, len + slack) of each sequence, -1 past them."""
    order = torch.randperm(pool, generator=g).tolist()
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range(min(width, (n + slack + (1 << shift) - 1) >> shift)):
            t[i, j] = order.pop() << shift
    return t


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- rotary append ---------------------------------------------------------------
ROPE = [  # T, nq, nkv, hd, half, stride (0: neighbours), norms, dtype, shift, first position
    (1, 16, 8, 256, 128, 128, True, BF, 10, 4095),
    (37, 16, 2, 512, 64, 256, True, BF, 4, 1000),
    (5, 3, 1, 64, 8, 16, False, HF, 0, 0),
    (70, 12, 4, 64, 24, 24, False, HF, 3, 130000),
    (33, 6, 6, 128, 64, 64, True, HF, 5, 2**20),
    (19, 32, 8, 128, 32, 0, False, BF, 4, 2**24 - 30),
    (65, 1, 1, 256, 4, 0, True, BF, 6, 7),
    (9, 5, 5, 512, 256, 0, False, HF, 2, 77777),
    (3, 2, 2, 64, 0, 0, True, BF, 4, 3),
    (530, 7, 3, 128, 16, 64, False, BF, 4, 100),
]


def rope_case(T, nq, nkv, hd, half, stride, norm, dt, shift, first, seed=0):
    g = gen(seed + T + hd)
    seqs = 3 if T > 2 else 1
    ids = torch.arange(T, dtype=torch.int32) % seqs
    pos = first + torch.arange(T, dtype=torch.int32) // seqs
    width = (int(pos.max()) >> shift) + 1
    used = [sorted({int(p) >> shift for p, s in zip(pos, ids) if s == i}) for i in range(seqs)]
    pool = sum(map(len, used)) + 2
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    for i, u in enumerate(used):
        for j in u:
            table[i, j] = order.pop() << shift
    c = dict(q=normal(g, T, nq * hd, dt=dt), k=normal(g, T, nkv * hd, dt=dt), v=normal(g, T, nkv * hd, dt=dt),
             kc=normal(g, pool << shift, nkv * hd, dt=dt), vc=normal(g, pool << shift, nkv * hd, dt=dt),
             qn=normal(g, hd, scale=0.3).add(1).to(dt) if norm else None,
             kn=normal(g, hd, scale=0.3).add(1).to(dt) if norm else None,
             inv=(10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float() if half else None,
             table=table, ids=ids, pos=pos)
    return c


def rope_tol(ref, size, dt):
    """Half a step of the result, and 2^-18 of the pair's magnitudes for 32-bit norms, sines (from
    2^-26 turns; the instructions within 2^-19) and products."""
    return EPS[dt] * ref.abs() + 2.0 ** -18 * size + 1e-7


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("T,nq,nkv,hd,half,stride,norm,dt,shift,first", ROPE)
def test_rope_append(gpu, T, nq, nkv, hd, half, stride, norm, dt, shift, first, fused):
    c = rope_case(T, nq, nkv, hd, half, stride, norm, dt, shift, first)
    mscale = 1.0 if norm else 1.25
    d = {n: t.cuda() if t is not None else None for n, t in c.items()}
    if fused:
        qkv = torch.cat([d["q"], d["k"], d["v"]], 1)
        d["q"], d["k"], d["v"] = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    out = gpu.rope_append(d["q"], d["k"], d["v"], d["inv"], d["pos"], d["table"], d["kc"], d["vc"], nq, nkv, hd, shift,
                          pair_stride=stride, mscale=mscale, seq_ids=d["ids"], q_norm=d["qn"], k_norm=d["kn"],
                          norm_v=norm, out=d["q"] if fused else None)
    torch.cuda.synchronize()
    ne = hd * 1e-6
    ref, size = rope_ref(c["q"], hd, c["pos"], c["inv"], stride, mscale, c["qn"], norm, True, ne)
    assert bool(((out.cpu().double() - ref).abs() <= rope_tol(ref, size, dt)).all())
    written = torch.tensor([slot_of(c["table"], int(s), int(p), shift, c["kc"].shape[0]) for s, p in zip(c["ids"], c["pos"])])
    assert (written >= 0).all()
    rest = torch.ones(c["kc"].shape[0], dtype=torch.bool)
    rest[written] = False
    for name, src, gain, turned in (("kc", "k", c["kn"], True), ("vc", "v", None, False)):
        got = d[name].cpu()
        ref, size = rope_ref(c[src], hd, c["pos"], c["inv"], stride, mscale, gain, norm, turned, ne)
        assert bool(((got[written].double() - ref).abs() <= rope_tol(ref, size, dt)).all()), name
        assert same_bits(got[rest], c[name][rest]), name
        if not norm and not turned:
            assert same_bits(got[written], c[src])


def test_rope_padding_and_bad_pages(gpu):
    """Padding tokens leave their rows; a missing or foreign page leaves the cache; q is written."""
    nq, nkv, hd, shift = 4, 2, 128, 4
    c = rope_case(8, nq, nkv, hd, 64, 64, True, BF, shift, 5)
    c["pos"][2], c["ids"][4], c["ids"][5] = -1, 3, -1
    slots = c["kc"].shape[0]
    c["table"][0, 0] = slots - 15            # its last row lies past the cache
    c["pos"][7], c["ids"][7] = 2**31 - 1, 1  # past the table
    d = {n: t.cuda() if t is not None else None for n, t in c.items()}
    out = torch.full((8, nq * hd), 7.0, dtype=BF, device="cuda")
    gpu.rope_append(d["q"], d["k"], d["v"], d["inv"], d["pos"], d["table"], d["kc"], d["vc"], nq, nkv, hd, shift,
                    seq_ids=d["ids"], q_norm=d["qn"], k_norm=d["kn"], out=out)
    torch.cuda.synchronize()
    ref, size = rope_ref(c["q"], hd, c["pos"], c["inv"], 64, 1.0, c["qn"], True, True, hd * 1e-6)
    kref, ksize = rope_ref(c["k"], hd, c["pos"], c["inv"], 64, 1.0, c["kn"], True, True, hd * 1e-6)
    kc, vc = c["kc"].clone(), c["vc"].clone()
    kgot, vgot, written = d["kc"].cpu(), d["vc"].cpu(), []
    for t in range(8):
        pad = c["pos"][t] < 0 or not 0 <= c["ids"][t] < 3
        if pad:
            assert (out[t] == 7.0).all()
            continue
        assert bool(((out[t].cpu().double() - ref[t]).abs() <= rope_tol(ref[t], size[t], BF)).all()), t
        s = slot_of(c["table"], int(c["ids"][t]), int(c["pos"][t]), shift, slots)
        if s >= 0:
            written.append(s)
            assert bool(((kgot[s].double() - kref[t]).abs() <= rope_tol(kref[t], ksize[t], BF)).all()), t
            assert same_bits(vgot[s], c["v"][t]), t
    assert 0 < len(written) < 5
    rest = torch.ones(slots, dtype=torch.bool)
    rest[written] = False
    assert same_bits(kgot[rest], kc[rest]) and same_bits(vgot[rest], vc[rest])


# ---- attention -------------------------------------------------------------------
ATTN = [  # lens, nq, nkv, hd, window, softcap, dtype, shift
    ([1500], 16, 8, 256, 1024, 0.0, BF, 10),
    ([1], 1, 1, 64, 0, 0.0, HF, 0),
    ([0, 1, 2, 31, 32, 33, 0], 8, 2, 128, 0, 0.0, BF, 4),
    ([333, 64, 17, 95, 200, 1, 128], 24, 8, 64, 0, 50.0, HF, 3),
    ([700, 16, 15, 1023], 16, 2, 512, 0, 0.0, BF, 6),
    ([513, 130], 4, 4, 512, 100, 30.0, HF, 1),
    ([257, 900], 20, 4, 256, 33, 0.0, HF, 5),
    ([400, 77, 5], 32, 1, 128, 0, 0.0, BF, 2),      # 32 query heads on one kv head
    ([129], 17, 1, 64, 0, 0.0, BF, 4),              # 17: a group of 16 and one of 1
    ([2049, 1300, 2], 6, 2, 128, 1, 0.0, HF, 7),
    ([96, 96], 7, 1, 256, 0, 20.0, BF, 0),
    ([5000], 2, 1, 64, 4999, 0.0, BF, 4),
]


def attn_case(lens, nq, nkv, hd, dt, shift, seed=0, slack=0, poison=True):
    g = gen(seed + hd + len(lens))
    need = sum((n + slack + (1 << shift) - 1) >> shift for n in lens)
    width = max(1, (max(lens) + slack + (1 << shift) - 1) >> shift) + 2
    pool = need + 3
    table = tables(g, lens, shift, width, pool, slack)
    kc, vc = (normal(g, pool << shift, nkv * hd, dt=dt) for _ in range(2))
    if poison:  # whatever stands where no position is must not be looked at
        used = torch.zeros(pool << shift, dtype=torch.bool)
        for i, n in enumerate(lens):
            for p in range(n):
                used[slot_of(table, i, p, shift, pool << shift)] = True
        bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dt).min])
        for c in (kc, vc):
            c[~used] = bad[torch.arange(int((~used).sum())) % 4].to(dt)[:, None]
    return normal(g, len(lens), nq * hd, dt=dt), kc, vc, table, torch.tensor(lens, dtype=torch.int32)


def check_attn(gpu, q, kc, vc, table, lens, nq, nkv, hd, shift, window, cap, scale=None, **kw):
    lse = torch.empty(q.shape[0], nq, device="cuda")
    out = gpu.paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(), nq, nkv, hd, shift,
                              window=window, softcap=cap, scale=scale, lse=lse, **kw)
    torch.cuda.synchronize()
    ref, rl, tol = attention_ref(q, kc, vc, table, lens, nq, nkv, hd, shift, window, scale, cap)
    off = (out.cpu().double() - ref).abs()
    nan = torch.isnan(ref)  # rows that take part may hold NaN: then so does the result, and only then
    assert torch.equal(torch.isnan(out.cpu()), nan)
    assert bool((off <= tol)[~nan].all()), float((off / tol)[~nan].max())
    none, some = torch.isinf(rl), torch.isfinite(rl)
    assert torch.equal(torch.isinf(lse.cpu()) & (lse.cpu() < 0), none)
    assert torch.equal(torch.isnan(lse.cpu()), torch.isnan(rl))
    assert bool(((lse.cpu().double() - rl)[some].abs() <= 1e-4 * (1 + rl[some].abs())).all())
    assert bool((out.cpu().view(q.shape[0], nq, hd)[none] == 0).all())
    return out


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("lens,nq,nkv,hd,window,cap,dt,shift", ATTN)
def test_paged_attention(gpu, lens, nq, nkv, hd, window, cap, dt, shift, splits):
    c = attn_case(lens, nq, nkv, hd, dt, shift)
    check_attn(gpu, *c, nq, nkv, hd, shift, window, cap, max_kv_len=max(max(lens), 1), s_max=splits)


@pytest.mark.parametrize("lens,nq,nkv,hd,window,dt,shift,splits", [
    ([6000] + [40] * 9, 8, 2, 128, 0, BF, 4, 2),          # 9 shares of one, joined by its last workgroup
    ([6000] + [40] * 9, 16, 1, 128, 0, HF, 3, 4),         # capped: 16 heads' sums
    ([3, 0, 4000, 0, 700], 8, 2, 64, 0, HF, 5, 7),
    ([3000, 100, 1], 4, 2, 512, 0, BF, 4, 30),            # joined by a launch
    ([2500, 33, 1200], 32, 1, 256, 2000, BF, 6, 9),       # two groups of heads, a launch
    ([50] * 70 + [2000] + [0] * 60, 2, 1, 64, 0, BF, 0, 2),  # more sequences than lanes
    ([0] * 130, 2, 2, 128, 0, HF, 4, 3),
    ([200 + 9 * i for i in range(67)], 2, 2, 128, 0, BF, 4, None),
    ([10000], 4, 1, 128, 0, BF, 4, 256),
    ([64, 5000], 16, 1, 512, 0, HF, 4, 256),
])
def test_attention_unequal_lengths(gpu, lens, nq, nkv, hd, window, dt, shift, splits):
    """Slots are shared out by length, whatever the longest sequence was said to have; the share
    does not depend on where a sequence stands."""
    c = attn_case(lens, nq, nkv, hd, dt, shift)
    out = check_attn(gpu, *c, nq, nkv, hd, shift, window, 0.0, max_kv_len=max(max(lens), 1), s_max=splits)
    q, kc, vc, table, n = (t.flip(0) if i in (0, 3, 4) else t for i, t in enumerate(c))
    back = check_attn(gpu, q, kc, vc, table, n, nq, nkv, hd, shift, window, 0.0, max_kv_len=max(max(lens), 1), s_max=splits)
    assert same_bits(out.flip(0), back)


def test_attention_longer_than_planned(gpu):
    """max_kv_len only sizes the splits; None plans for the whole table."""
    c = attn_case([700, 3], 4, 2, 128, BF, 4)
    for longest in (1, 64, 699, None):
        for s in (None, 4):
            check_attn(gpu, *c, 4, 2, 128, 4, 0, 0.0, max_kv_len=longest, s_max=s)


def test_attention_large_scores(gpu):
    """Weights that are one key's alone, and many small ones beside it (f16 would lose them)."""
    for dt in (BF, HF):
        q, kc, vc, table, lens = attn_case([900], 2, 1, 64, dt, 4)
        q[:] = 1.0
        kc[:] = torch.where(torch.isfinite(kc), torch.zeros_like(kc), kc)
        kc[slot_of(table, 0, 450, 4, kc.shape[0])] = 1.4  # 64 * 1.4 / 8 = 11.2: the others at e^-11.2
        check_attn(gpu, q, kc, vc, table, lens, 2, 1, 64, 4, 0, 0.0)
        check_attn(gpu, q, kc, vc, table, lens, 2, 1, 64, 4, 0, 0.0, scale=8.0)
        check_attn(gpu, q, kc, vc, table, lens, 2, 1, 64, 4, 0, 0.0, scale=-0.5)


def test_attention_bad_pages(gpu):
    """Entries outside the cache are no pages: their positions take no part."""
    for hd, shift in ((128, 4), (64, 6), (512, 3)):
        q, kc, vc, table, lens = attn_case([300, 200, 90], 4, 2, hd, BF, shift)
        slots = kc.shape[0]
        table[0, 1], table[0, 2], table[0, 4] = -1, slots, slots - (1 << shift) + 1
        table[1, 0], table[1, 3] = -(2**31), 2**31 - 1
        table[2, :] = -1
        for s in (1, 3):
            check_attn(gpu, q, kc, vc, table, lens, 4, 2, hd, shift, 0, 0.0, s_max=s)
        lens[:] = 2**31 - 1  # clipped to the table
        check_attn(gpu, q, kc, vc, table, lens, 4, 2, hd, shift, 50, 0.0)


def test_attention_strided_queries_and_kept_buffers(gpu):
    q, kc, vc, table, lens = attn_case([100, 50, 7], 8, 2, 128, BF, 4)
    wide = torch.zeros(3, 8 * 128 + 40, dtype=BF)
    wide[:, 8:8 + 8 * 128] = q
    dq = wide.cuda()[:, 8:8 + 8 * 128]
    args = (kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(), 8, 2, 128, 4)
    a = gpu.paged_attention(q.cuda(), *args, s_max=2)
    out = torch.full((5, 8 * 128), 3.0, dtype=BF, device="cuda")
    ws = gpu.paged_attention_workspace(3, 8, 128, 2)
    gpu.paged_attention(dq, *args, s_max=2, workspace=ws, out=out[:3])
    assert same_bits(out[:3], a) and (out[3:] == 3.0).all()


def test_attention_far_offsets(gpu):
    """Rows past 2^32 bytes and 2^31 values of the cache."""
    nq, nkv, hd, shift, slots = 16, 8, 256, 6, 1 << 21
    g = gen(3)
    kc = torch.empty(slots, nkv * hd, dtype=BF, device="cuda")
    vc = torch.empty(slots, nkv * hd, dtype=BF, device="cuda")
    lens = torch.tensor([150, 70], dtype=torch.int32)
    table = torch.tensor([[slots - 64, 64, slots // 2 + 64], [slots - 128, 0, -1]], dtype=torch.int32)
    small_k, small_v = normal(g, 5 * 64, nkv * hd, dt=BF), normal(g, 5 * 64, nkv * hd, dt=BF)
    near = torch.tensor([[0, 64, 128], [192, 256, -1]], dtype=torch.int32)
    for t, s in zip(table.view(-1).tolist(), near.view(-1).tolist()):
        if t >= 0:
            kc[t:t + 64], vc[t:t + 64] = small_k[s:s + 64].cuda(), small_v[s:s + 64].cuda()
    q = normal(g, 2, nq * hd, dt=BF)
    far = gpu.paged_attention(q.cuda(), kc, vc, table.cuda(), lens.cuda(), nq, nkv, hd, shift, max_kv_len=150)
    want = gpu.paged_attention(q.cuda(), small_k.cuda(), small_v.cuda(), near.cuda(), lens.cuda(), nq, nkv, hd, shift,
                               max_kv_len=150)
    assert same_bits(far, want)
    pos = torch.tensor([149, 69], dtype=torch.int32, device="cuda")
    kv = normal(g, 2, 2 * nkv * hd, dt=BF).cuda()
    args = dict(q_norm=None, pair_stride=hd // 2)
    inv = gpu.rope_frequencies(hd // 2)[0]
    for cache, t in (((kc, vc), table), ((small_k.cuda(), small_v.cuda()), near)):
        gpu.rope_append(q.cuda(), kv[:, :nkv * hd], kv[:, nkv * hd:], inv, pos, t.cuda(), *cache, nq, nkv, hd, shift, **args)
        if cache[0] is kc:
            got = [cache[0][int(t[i, p >> 6]) + (p & 63)].clone() for i, p in ((0, 149), (1, 69))]
        else:
            assert all(same_bits(x, cache[0][int(t[i, p >> 6]) + (p & 63)]) for x, (i, p) in zip(got, ((0, 149), (1, 69))))


@pytest.mark.parametrize("nkv,hd", [(2, 256), (2, 512), (1, 256), (8, 64)])
def test_attention_streams_and_graph(gpu, nkv, hd):
    """Two captured graphs with a workspace each, replayed on two streams with eager work between;
    the lengths change between replays and the graph follows."""
    nq, shift = 16, 4
    cases = [attn_case([900, 333, 0], nq, nkv, hd, BF, shift, seed=s, slack=8, poison=False) for s in (1, 2)]
    dev = [[t.cuda() for t in c] for c in cases]
    outs = [torch.zeros(3, nq * hd, dtype=BF, device="cuda") for _ in cases]
    wss = [gpu.paged_attention_workspace(3, nq, hd, 8) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]

    def call(i):
        return gpu.paged_attention(*dev[i], nq, nkv, hd, shift, s_max=8, max_kv_len=910, workspace=wss[i], out=outs[i])

    graphs = []
    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i]):
            call(i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i)
        graphs.append(g)
    for rep in range(4):
        for i in range(2):
            dev[i][4].copy_(torch.tensor([900 + rep, 333 - 100 * rep, rep], dtype=torch.int32))
            outs[i].fill_(9.0)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = gpu.paged_attention(*dev[i], nq, nkv, hd, shift, s_max=8, max_kv_len=910)
            assert same_bits(outs[i], want), (rep, i)


# ---- pages -----------------------------------------------------------------------
def page_case(seed, n, width, shift, spare, dts):
    g = gen(seed)
    rng = np.random.default_rng(seed)
    rows = 1 << shift
    lens = torch.tensor([int(rng.integers(0, (width - 1) * rows + 1)) for _ in range(n)], dtype=torch.int32)
    pool = sum((int(v) + rows - 1) >> shift for v in lens) + spare
    table = tables(g, lens.tolist(), shift, width, pool)
    refs = torch.zeros(pool, dtype=torch.int32)
    refs[(table[table >= 0] >> shift).long()] = 1
    arrays = [torch.randint(-127, 128, (pool << shift, *shape), generator=g).to(dt) for dt, shape in dts]
    return table, lens, refs, arrays


def check_pages(ref, table, lens, refs, arrays, where):
    torch.cuda.synchronize()
    assert torch.equal(table.cpu(), ref.base_rows()), where
    assert lens is None or lens.tolist() == ref.lens, where
    assert refs.tolist() == ref.refs, where
    for i, (a, b) in enumerate(zip(arrays, ref.arrays)):
        assert same_bits(a.cpu(), b), (where, i)


SOME = [(torch.int8, (8, 32)), (torch.float32, (8,)), (BF, (64,)), (torch.int8, (3,)), (torch.int16, (3, 5))]


@pytest.mark.parametrize("n,width,shift,spare", [(1, 1, 0, 1), (4, 9, 4, 8), (7, 70, 2, 40), (33, 5, 6, 70), (256, 12, 3, 600),
                                                 (300, 3, 0, 900), (1024, 2, 1, 1500), (2, 3000, 1, 50),
                                                 (300, 80, 1, 900), (1000, 33, 0, 5000), (5, 4000, 0, 30000)])
def test_cache_reorder(gpu, n, width, shift, spare):
    """Several steps of forks, frees and growth, each against the page-by-page reference."""
    table, lens, refs, arrays = page_case(n + width, n, width, shift, spare, SOME)
    ref = Pages(table, lens, refs, shift, arrays)
    d = [t.cuda() for t in (table, lens, refs)]
    da = [a.cuda() for a in arrays]
    rng = np.random.default_rng(width)
    for step in range(5):
        parents = [int(rng.integers(-1, n)) if rng.random() < 0.6 else i for i in range(n)]
        if step == 3:
            parents = [0] * n  # one parent for everyone
        grow = [int(rng.integers(0, 2 << shift)) if rng.random() < 0.7 else 0 for _ in range(n)]
        grow = None if step == 1 else grow
        want = ref.reorder(parents, grow)
        info = gpu.cache_reorder(da, d[0], d[1], d[2], torch.tensor(parents, dtype=torch.int32, device="cuda"), shift,
                                 grow=None if grow is None else torch.tensor(grow, dtype=torch.int32, device="cuda"))
        check_pages(ref, *d, da, step)
        assert info.tolist() == want, step
        for i in range(n):  # positions are written: lengths move on
            more = min(max(grow[i], 0) if grow else 0, (width << shift) - ref.lens[i])
            have = sum(p >= 0 for p in ref.table[i]) << shift
            ref.lens[i] = min(ref.lens[i] + more, have)
        d[1].copy_(torch.tensor(ref.lens, dtype=torch.int32))


def test_cache_reorder_short_pool_and_bad_tables(gpu):
    """A pool that runs out, entries and parents that name nothing, lengths past the table."""
    table, lens, refs, arrays = page_case(5, 6, 6, 2, 2, SOME)
    table[0, 5], table[1, 5], table[2, 5], table[3, 5] = -7, 2, 1 << 30, -(2**31)
    lens[4] = 2**31 - 1
    lens[5] = -3
    ref = Pages(table, lens, refs, 2, arrays)
    d = [t.cuda() for t in (table, lens, refs)]
    da = [a.cuda() for a in arrays]
    short = 0
    for parents, grow in (([0, 0, 1, 9, -8, 4], [9, 9, 9, 0, 5, 0]), ([2**31 - 1, -(2**31), 2, 2, 2, 5], [0, 0, -4, 100, 7, 2**31 - 1]),
                          ([5, 4, 3, 2, 1, 0], [24] * 6), ([0, 0, 0, 3, 3, 3], [24] * 6)):
        want = ref.reorder(parents, grow)
        info = gpu.cache_reorder(da, *d, torch.tensor(parents, dtype=torch.int32, device="cuda"), 2,
                                 grow=torch.tensor(grow, dtype=torch.int32, device="cuda"))
        check_pages(ref, *d, da, parents)
        assert info.tolist() == want
        short += want[2]
    assert short > 0


@pytest.mark.parametrize("n,width,shift,spare", [(1, 1, 0, 1), (5, 9, 4, 30), (64, 33, 6, 100), (40, 120, 0, 3000), (3, 2, 10, 1),
                                                 (90, 200, 0, 9000), (300, 90, 1, 500), (6, 30, 10, 20)])
def test_cache_compact(gpu, n, width, shift, spare):
    table, lens, refs, arrays = page_case(7 * n + width, n, width, shift, spare, SOME)
    ref = Pages(table, lens, refs, shift, arrays)
    d = [t.cuda() for t in (table, lens, refs)]
    da = [a.cuda() for a in arrays]
    rng = np.random.default_rng(n)
    for step in range(3):
        parents = [int(rng.integers(-1, n)) for _ in range(n)]
        ref.reorder(parents)
        gpu.cache_reorder(da, *d, torch.tensor(parents, dtype=torch.int32, device="cuda"), shift)
        want = ref.compact()
        info = gpu.cache_compact(da, d[0], d[2], shift)
        check_pages(ref, d[0], None, d[2], da, step)
        assert info.tolist() == want
    want = ref.compact()  # packed already
    assert want[1] == 0 and gpu.cache_compact([], d[0], d[2], shift).tolist() == want
    check_pages(ref, d[0], None, d[2], da, "again")


@pytest.mark.parametrize("n,width,shift,spare", [(8, 12, 3, 40), (60, 90, 1, 1500), (200, 100, 0, 9000)])
def test_cache_graph_replays(gpu, n, width, shift, spare):
    """A captured reorder and compaction, replayed on a state that goes on: plans of one launch with
    little and with much LDS, and of several launches."""
    table, lens, refs, arrays = page_case(2, n, width, shift, spare, SOME)
    ref = Pages(table, lens, refs, shift, arrays)
    d = [t.cuda() for t in (table, lens, refs)]
    da = [a.cuda() for a in arrays]
    parents, grow = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    info, info2 = (torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2))
    ws = torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    parents.copy_(torch.arange(n, dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.cache_reorder(da, *d, parents, shift, grow=grow, workspace=ws, info=info)
    torch.cuda.synchronize()
    ref.reorder(list(range(n)), [0] * n)
    check_pages(ref, *d, da, "eager")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gpu.cache_reorder(da, *d, parents, shift, grow=grow, workspace=ws, info=info)
        gpu.cache_compact(da, d[0], d[2], shift, workspace=ws, info=info2)
    rng = np.random.default_rng(1)
    for rep in range(5):
        p, w = [int(rng.integers(-1, n)) for _ in range(n)], [int(rng.integers(0, 9)) for _ in range(n)]
        parents.copy_(torch.tensor(p, dtype=torch.int32))
        grow.copy_(torch.tensor(w, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        want = ref.reorder(p, w), ref.compact()
        check_pages(ref, *d, da, rep)
        assert (info.tolist(), info2.tolist()) == want


# ---- beams -----------------------------------------------------------------------
BEAM = [  # batch, beams, vocab, n, dtype, finished, row padding
    (1, 4, 262144, 4, BF, False, 0),
    (3, 8, 32000, 16, torch.float32, True, 0),
    (1, 1, 1, 1, BF, False, 0),
    (2, 3, 7, 64, HF, True, 1),           # fewer candidates than asked for
    (5, 2, 1025, 4, BF, True, 3),         # rows of odd alignment
    (2, 64, 500, 64, torch.float32, True, 0),
    (1, 16, 5003, 32, HF, False, 0),
    (40, 5, 2047, 5, BF, False, 0),
    (1, 2, 1 << 20, 3, HF, False, 0),
    (10, 13, 900, 13, HF, False, 0),      # a part for each beam
    (4, 10, 3756, 20, HF, True, 0),
    (2, 1, 1800, 64, torch.float32, False, 0),
    (1, 3, 130, 64, BF, True, 2),
    (2, 5, 6000, 64, BF, False, 1),
]


def check_beam(gpu, logits, scores, n, finished=None, eos=-1, dl=None):
    dl = logits.cuda() if dl is None else dl
    got = gpu.beam_select(dl, scores.cuda(), n, finished=None if finished is None else finished.cuda(), eos_id=eos)
    torch.cuda.synchronize()
    sc, pa, tk, fin = beam_ref(logits, scores, n, finished, eos)
    assert torch.equal(got[1].cpu(), pa) and torch.equal(got[2].cpu(), tk)
    none = torch.isinf(sc)
    # one rounding of a 64-bit score, and 2^-36 for the sums
    some = ~none & torch.isfinite(sc.float())
    assert torch.equal(got[0].cpu()[~some], sc.float()[~some])
    assert bool(((got[0].cpu().double() - sc)[some].abs() <= 2.0 ** -24 * sc[some].abs() + 2.0 ** -36).all())
    if finished is not None:
        assert torch.equal(got[3].cpu(), fin)
    return got


@pytest.mark.parametrize("b,k,v,n,dt,done,pad", BEAM)
def test_beam_select(gpu, b, k, v, n, dt, done, pad):
    g = gen(v + k)
    wide = normal(g, b * k, v + pad, dt=dt, scale=3.0)
    logits = wide[:, :v]
    scores = -torch.rand(b, k, generator=g) * 6 - 3
    fin = torch.rand(b, k, generator=g) < 0.3 if done else None
    check_beam(gpu, logits, scores, n, fin if fin is None or b % 2 else fin.to(torch.uint8), min(2, v - 1) if done else -1,
               dl=wide.cuda()[:, :v])


def test_beam_ties_masks_and_edges(gpu):
    v, inf = 3000, float("inf")
    for dt in (BF, torch.float32):
        flat = torch.zeros(4, v, dtype=dt)                       # everything ties
        check_beam(gpu, flat, torch.tensor([[-1.0, -1.0], [0.0, -inf]]), 40)
        check_beam(gpu, flat, torch.full((1, 4), -2.0), 64)
        few = torch.full((4, v), -inf, dtype=dt)                 # two tokens left in all
        few[1, 2999], few[3, 0] = 1.0, -5.0
        check_beam(gpu, few, torch.full((1, 4), -2.0), 4)
        low = torch.full((4, v), torch.finfo(dt).min, dtype=dt)  # masked by the lowest value, one row not
        low[2, 5], low[2, 6], low[0, 100] = 3.0, 3.0, 2.0
        check_beam(gpu, low, torch.tensor([[-1.0, -2.0, -3.0, -inf]]), 8)
        bad = normal(gen(1), 4, v, dt=dt)                        # NaN tokens, a row of NaN, a row with +inf
        bad[0, ::3], bad[1, :], bad[2, 17] = float("nan"), float("nan"), inf
        check_beam(gpu, bad, torch.tensor([[-1.0, -1.0, -1.0, -1.0]]), 16)
        check_beam(gpu, bad, torch.tensor([[float("nan"), -inf, -inf, -1.0]]), 16)
        none = torch.full((2, v), -inf, dtype=dt)
        got = check_beam(gpu, none, torch.zeros(1, 2), 3)
        assert got[1].tolist() == [[-1, -1, -1]]
        up = torch.arange(v, dtype=torch.float32).div(100).to(dt)[None].repeat(4, 1)  # sorted rows
        check_beam(gpu, up, torch.zeros(1, 4), 64)
        check_beam(gpu, up.flip(1).contiguous(), torch.zeros(2, 2), 33)
        same = normal(gen(2), 1, v, dt=dt).repeat(4, 1)          # beams that are the same
        check_beam(gpu, same, torch.full((1, 4), -3.0), 16)
    # beams put out of the way by a score that leaves little or nothing of the logits in 64 bits
    few = torch.full((4, v), -inf)
    few[0, 7], few[1, :5], few[2, 100:2000:100], few[3, 3] = 1.0, torch.arange(5.0), torch.arange(19.0), 2.0
    for low in (-1e9, -1e15, -1e30, float(torch.finfo(torch.float32).min)):
        check_beam(gpu, few, torch.tensor([[-1.0, low, low, low]]), 16)
        check_beam(gpu, normal(gen(5), 4, v), torch.tensor([[low, low, low, low]]), 40)
        check_beam(gpu, normal(gen(6), 4, v), torch.tensor([[0.0, low, low, low]]), 4)
    huge = normal(gen(7), 4, v, scale=1e30)
    check_beam(gpu, huge, torch.tensor([[-1.0, -2.0, -3.0, -4.0]]), 12)
    check_beam(gpu, huge * 1e-25, torch.tensor([[-1.0, -2.0, -3.0, -4.0]]), 12)
    fin = torch.tensor([[1, 1], [1, 0]], dtype=torch.uint8)
    x = normal(gen(3), 4, 50)
    x[0] = float("nan")                                          # a finished beam's logits are not read
    check_beam(gpu, x, torch.tensor([[-1.0, -1.0], [-50.0, -1.0]]), 3, fin, 7)
    check_beam(gpu, x, torch.tensor([[-inf, -1.0], [-2.0, -inf]]), 3, fin, 0)


def test_beam_graph_and_stream(gpu):
    g = gen(9)
    logits, scores = normal(g, 8, 5000, dt=BF).cuda(), -torch.rand(2, 4, generator=g).cuda()
    out = (torch.zeros(2, 4, device="cuda"), *(torch.zeros(2, 4, dtype=torch.int32, device="cuda") for _ in range(2)))
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.beam_select(logits, scores, workspace=ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.beam_select(logits, scores, workspace=ws, out=out)
    for rep in range(4):
        logits.copy_(normal(g, 8, 5000, dt=BF))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = gpu.beam_select(logits, scores)
        assert all(same_bits(a, b) for a, b in zip(out, want)), rep


# ---- refusals of the binding ---------------------------------------------------------
def test_binding_refusals(gpu):
    q, kc, vc, table, lens = (t.cuda() for t in attn_case([20, 5], 4, 2, 64, BF, 4, poison=False))
    ok = dict(q=q, k_cache=kc, v_cache=vc, base_rows=table, kv_lens=lens, num_q=4, num_kv=2, head_dim=64, page_shift=4)
    gpu.paged_attention(**ok)
    for kw in (dict(q=q.float()), dict(k_cache=kc.to(HF)), dict(kv_lens=lens.long()), dict(base_rows=table.long())):
        with pytest.raises(TypeError):
            gpu.paged_attention(**{**ok, **kw})
    for kw in (dict(q=q[:, :100]), dict(q=q.cpu()), dict(k_cache=kc[:, :64]), dict(k_cache=kc[:16]), dict(kv_lens=lens[:1]),
               dict(base_rows=table[:1]), dict(base_rows=table[0]), dict(q=q.t().contiguous().t()), dict(v_cache=vc[::2])):
        with pytest.raises(ValueError):
            gpu.paged_attention(**{**ok, **kw})
    with pytest.raises(gpu.BqError):
        gpu.paged_attention(**{**ok, "s_max": 3, "workspace": torch.empty(16, dtype=torch.uint8, device="cuda")})
    with pytest.raises(gpu.BqError):
        gpu.paged_attention(**{**ok, "softcap": -2.0})
    refs = torch.zeros(kc.shape[0] >> 4, dtype=torch.int32, device="cuda")
    parents = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):  # an array of another pool
        gpu.cache_reorder([kc[16:]], table, lens, refs, parents, 4)
    with pytest.raises(ValueError):
        gpu.cache_reorder([kc], table, lens, refs, parents[:1], 4)
    with pytest.raises(TypeError):
        gpu.cache_compact([kc], table, refs.long(), 4)
    x = torch.zeros(4, 100, device="cuda")
    for args, kw in (((x, torch.zeros(1, 3, device="cuda")), {}), ((x, torch.zeros(4, device="cuda")), {}),
                     ((x, torch.zeros(1, 4, device="cuda")), dict(finished=torch.zeros(3, dtype=torch.uint8, device="cuda")))):
        with pytest.raises(ValueError):
            gpu.beam_select(*args, **kw)
    with pytest.raises(gpu.BqError):
        gpu.beam_select(x, torch.zeros(1, 4, device="cuda"), n=65)


# ---- together: a decode loop with beams ----------------------------------------------
def test_beam_decoding_together(gpu):
    """Steps of beam search through the framework's calls: norm and projections, rotary append,
    attention over the pages, the output projection, a quantized head, selection, reorder.  The
    cache of every beam is its own history, its attention that of the history, and the choices
    those of the logits; then one more time as a captured graph."""
    B, K, H, V, nq, nkv, hd, shift, steps = 2, 4, 512, 2048, 8, 2, 64, 2, 11
    N, eos = B * K, 5
    g = gen(11)
    weight = lambda n, k, block=128: gpu.load_weight(normal(g, n, k, dt=BF, scale=0.06).cuda(), block)
    wq, wk, wv, head = weight(nq * hd, H), weight(nkv * hd, H), weight(nkv * hd, H), weight(V, H)
    wo = weight(H, nq * hd, 256)
    table_e = normal(g, V, H, dt=BF).cuda()
    gamma = torch.ones(H, dtype=BF, device="cuda")
    qn, kn = (normal(g, hd, scale=0.2).add(1).to(BF).cuda() for _ in range(2))
    inv, ms = gpu.rope_frequencies(hd // 2, 10000.0, factor=4.0, original_len=512)
    width, pool = 8, 80

    def state():
        return dict(kc=torch.zeros(pool << shift, nkv * hd, dtype=BF, device="cuda"),
                    vc=torch.zeros(pool << shift, nkv * hd, dtype=BF, device="cuda"),
                    table=torch.full((N, width), -1, dtype=torch.int32, device="cuda"),
                    lens=torch.zeros(N, dtype=torch.int32, device="cuda"),
                    refs=torch.zeros(pool, dtype=torch.int32, device="cuda"),
                    tokens=torch.arange(N, dtype=torch.int32, device="cuda") // K,
                    parents=torch.arange(N, dtype=torch.int32, device="cuda"),
                    scores=torch.tensor([[0.0] + [-math.inf] * (K - 1)] * B, device="cuda"),
                    fin=torch.zeros(B, K, dtype=torch.uint8, device="cuda"),
                    grow=torch.ones(N, dtype=torch.int32, device="cuda"))

    def step(s):
        gpu.cache_reorder([s["kc"], s["vc"]], s["table"], s["lens"], s["refs"], s["parents"], shift, grow=s["grow"])
        x = table_e[s["tokens"].clamp(min=0).long()]
        (q, k, v), _ = gpu.norm_qkv(x, gamma, wq, wk, wv)
        q = gpu.rope_append(q, k, v, inv, s["lens"], s["table"], s["kc"], s["vc"], nq, nkv, hd, shift, mscale=ms,
                            q_norm=qn, k_norm=kn, norm_v=True)
        s["lens"] += 1
        a = gpu.paged_attention(q, s["kc"], s["vc"], s["table"], s["lens"], nq, nkv, hd, shift, max_kv_len=width << shift)
        y = gpu.block_linear(*gpu.block_quant(a, 256, True), wo, 256)
        (_, logits), _ = gpu.norm_linear(y, gamma, head, want_f32=True)
        sc, parents, tokens, fin = gpu.beam_select(logits, s["scores"], finished=s["fin"], eos_id=eos)
        before = s["scores"].clone(), s["fin"].clone()
        s["scores"].copy_(sc)
        s["parents"].copy_(parents.view(-1))
        s["tokens"].copy_(tokens.view(-1))
        s["fin"].copy_(fin)
        return q, k, v, a, logits, before

    s = state()
    history = [[] for _ in range(N)]
    keys = []
    for t in range(steps):
        parents = s["parents"].tolist()
        q, k, v, a, logits, before = step(s)
        torch.cuda.synchronize()
        history = [list(history[p]) if p >= 0 else [] for p in parents]
        table, lens = s["table"].cpu(), s["lens"].tolist()
        pos = torch.tensor([n - 1 for n in lens])
        kr, ks = rope_ref(k.cpu(), hd, pos, inv.cpu(), hd // 2, ms, kn.cpu(), True, True, hd * 1e-6)
        kc, vc = s["kc"].cpu(), s["vc"].cpu()
        for i in range(N):
            at = slot_of(table, i, lens[i] - 1, shift, kc.shape[0])
            assert at >= 0 and lens[i] == len(history[i]) + 1
            assert bool(((kc[at].double() - kr[i]).abs() <= rope_tol(kr[i], ks[i], BF)).all())
            history[i].append((kc[at].clone(), vc[at].clone()))
            for p, (hk, hv) in enumerate(history[i]):
                at = slot_of(table, i, p, shift, kc.shape[0])
                assert same_bits(kc[at], hk) and same_bits(vc[at], hv), (t, i, p)
        ref, _, tol = attention_ref(q.cpu(), kc, vc, table, torch.tensor(lens), nq, nkv, hd, shift)
        assert bool(((a.cpu().double() - ref).abs() <= tol).all()), t
        sc, pa, tk, fin = beam_ref(logits.cpu(), before[0].cpu(), K, before[1].cpu(), eos)
        assert torch.equal(s["parents"].cpu().view(B, K), pa) and torch.equal(s["tokens"].cpu().view(B, K), tk), t
        assert torch.equal(s["fin"].cpu(), fin)
        live = torch.bincount((table[table >= 0] >> shift).long(), minlength=pool)
        assert live.tolist() == s["refs"].tolist()
        keys.append((s["tokens"].tolist(), s["parents"].tolist(), s["scores"].tolist()))
    assert len({h[0][0].sum().item() for h in history}) >= 1 and any(p != i for i, p in enumerate(keys[-1][1]))

    s = state()
    start = {n: t.clone() for n, t in s.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s)
    for n, t in s.items():
        t.copy_(start[n])
    for t in range(steps):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (s["tokens"].tolist(), s["parents"].tolist(), s["scores"].tolist()) == keys[t], t


def test_reorder_serves_the_int8_cache(gpu, O):
    """The same table under the int8 attention: beams forked on the device attend to what a
    contiguous copy of their rows gives, bit for bit."""
    nq, nkv, hd, shift, N, width = 8, 2, 128, 4, 4, 8
    g = gen(21)
    pool = 40
    slots = pool << shift
    caches = [torch.zeros(slots, nkv * hd, dtype=torch.int8, device="cuda"), torch.zeros(slots, nkv, device="cuda"),
              torch.zeros(slots, nkv * hd, dtype=torch.int8, device="cuda"), torch.zeros(slots, nkv, device="cuda")]
    table = torch.full((N, width), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(N, dtype=torch.int32, device="cuda"), torch.zeros(pool, dtype=torch.int32, device="cuda")
    ones = torch.ones(hd, dtype=BF, device="cuda")
    cos, sin = (f(torch.arange(256)[:, None] * torch.rand(64, generator=g)).float().cuda() for f in (torch.cos, torch.sin))
    parents = list(range(N))
    for t in range(40):
        gpu.cache_reorder(caches, table, lens, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"), shift,
                          grow=torch.ones(N, dtype=torch.int32, device="cuda"))
        at = lens.tolist()
        runs = torch.tensor([[i, at[i], i * width, width] for i in range(N)], dtype=torch.int32, device="cuda")
        q, k, v = (normal(g, N, n * hd, dt=BF).cuda() for n in (nq, nkv, nkv))
        qi = gpu.attn_prep(q, k, v, ones, ones, *caches, cos, sin, runs, table.view(-1), nq, nkv, hd, 64, 64, shift,
                           (1 << shift) - 1, -1)
        lens += 1
        if t % 13 == 12:
            out, _ = gpu.attention(*qi, *caches, runs, table.view(-1), nq, nkv, hd, 0, shift, (1 << shift) - 1, -1,
                                   max_kv_len=t + 1)
            rows = torch.cat([torch.stack([table[i, p >> shift] + (p & 15) for p in range(t + 1)]) for i in range(N)]).long()
            flat = [c[rows].contiguous() for c in caches]
            base = torch.tensor([i * (t + 1) for i in range(N)], dtype=torch.int32, device="cuda")
            runs2 = torch.tensor([[i, at[i], i, 1] for i in range(N)], dtype=torch.int32, device="cuda")
            want, _ = gpu.attention(*qi, *flat, runs2, base, nq, nkv, hd, 0, 20, (1 << 20) - 1, -1, max_kv_len=t + 1)
            torch.cuda.synchronize()
            assert same_bits(out, want), t
        rng = np.random.default_rng(t)
        parents = [int(rng.integers(0, N)) for _ in range(N)] if t % 3 == 2 else list(range(N))


def test_empty_calls(gpu):
    """No tokens, no sequences, no requests: nothing happens."""
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device="cuda")
    kc, table = z(64, 128), z(0, 4, dt=torch.int32)
    assert gpu.paged_attention(z(0, 256), kc, kc, table, z(0, dt=torch.int32), 4, 2, 64, 4).shape == (0, 256)
    inv = gpu.rope_frequencies(32)[0]
    assert gpu.rope_append(z(0, 256), z(0, 128), z(0, 128), inv, z(0, dt=torch.int32), table, kc, kc, 4, 2, 64, 4).shape == (0, 256)
    gpu.cache_reorder([kc], table, z(0, dt=torch.int32), z(4, dt=torch.int32), z(0, dt=torch.int32), 4)
    gpu.cache_compact([kc], table, z(4, dt=torch.int32), 4)
    assert gpu.beam_select(z(0, 50), z(0, 3, dt=torch.float32))[1].shape == (0, 3)
    torch.cuda.synchronize()
    assert not kc.any()


def test_two_streams_at_once(gpu):
    """Each operator on two streams at the same time, many times over, against one at a time."""
    g = gen(31)
    attn = [[t.cuda() for t in attn_case([3000, 100 + 900 * i], 8, 4, 128, BF, 4, seed=i, poison=False)] for i in range(2)]
    logits = [normal(g, 8, 30000, dt=BF).cuda() for _ in range(2)]
    scores = [-torch.rand(2, 4, generator=g).cuda() for _ in range(2)]
    page = [page_case(40 + i, 12, 20, 3, 200, SOME) for i in range(2)]
    parents = [torch.randint(-1, 12, (12,), generator=g, dtype=torch.int32).cuda() for _ in range(2)]
    grow = torch.full((12,), 3, dtype=torch.int32, device="cuda")
    refs = []
    for i in range(2):
        table, lens, counts, arrays = page[i]
        ref = Pages(table, lens, counts, 3, arrays)
        for _ in range(20):
            ref.reorder(parents[i].tolist(), [3] * 12)
            ref.compact()
        refs.append(ref)
    state = [[t.cuda() for t in p[:3]] for p in page]
    arrs = [[a.cuda() for a in p[3]] for p in page]
    want = [(gpu.paged_attention(*attn[i], 8, 4, 128, 4, max_kv_len=3000), gpu.beam_select(logits[i], scores[i])) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for rep in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                a = gpu.paged_attention(*attn[i], 8, 4, 128, 4, max_kv_len=3000)
                gpu.cache_reorder(arrs[i], *state[i], parents[i], 3, grow=grow)
                got[i].append((a, gpu.beam_select(logits[i], scores[i])))
                gpu.cache_compact(arrs[i], state[i][0], state[i][2], 3)
    torch.cuda.synchronize()
    for i in range(2):
        check_pages(refs[i], *state[i], arrs[i], i)
        for a, beams in got[i]:
            assert same_bits(a, want[i][0]) and all(same_bits(x, y) for x, y in zip(beams, want[i][1]))
