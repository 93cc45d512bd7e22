"""CPU checks of the paged 16-bit cache and beam operators: the refusals of their
entry points, the page arithmetic the kernels share (a CPU build of the same header)
on good and bad tables, and invariants of the page reference the GPU tests go by."""
import ctypes as C
import os
import random
import re
import shutil
import struct
import subprocess

import pytest
import torch

from paged_cases import Pages, slot_of
from test_kernel_registers import LIB, MAGIC, READELF

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = C.c_void_p(256)  # a non-null placeholder: validation fails before any use
BF16, F16, F32 = 6, 5, 9


@pytest.fixture(scope="module")
def L():
    import bq
    return bq.lib()


def rope(L, **kw):
    a = dict(q=P, k=P, v=P, qs=1024, ks=512, vs=512, qn=P, kn=P, nv=0, sq=1.0, ne=1.0, inv=P, half=64, stride=64, ms=1.0,
             pos=P, seq=P, rows=P, n=4, width=8, shift=4, slots=512, out=P, os=1024, kc=P, vc=P, nq=8, nkv=4, hd=128,
             dt=BF16, t=4, st=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return L.bq_rope_append(*a.values())


def test_rope_refusals(L):
    assert rope(L, t=0, q=None) == 0
    for name in ("q", "k", "v", "pos", "rows", "out", "kc", "vc", "inv"):
        assert rope(L, **{name: None}) == 1 and b"null" in L.bq_last_error(), name
    assert rope(L, dt=F32) == 1
    assert rope(L, q=C.c_void_p(264)) == 1 and rope(L, kn=C.c_void_p(258)) == 1
    for kw in (dict(hd=96), dict(nq=0), dict(nkv=0), dict(n=0), dict(width=0), dict(half=60), dict(stride=60),
               dict(half=72, stride=64), dict(half=64, stride=72), dict(half=66, stride=0), dict(half=68, stride=0),
               dict(half=-4, stride=0), dict(stride=-8), dict(qs=1016), dict(qs=1028), dict(ks=504), dict(os=1000),
               dict(slots=-1), dict(seq=None, t=5)):
        assert rope(L, **kw) == 2, kw
    assert rope(L, shift=-1) == 4 and rope(L, shift=21) == 4 and rope(L, nq=70000, qs=1 << 24, os=1 << 24) == 4


def attn(L, **kw):
    a = dict(q=P, qs=1024, kc=P, vc=P, slots=512, rows=P, width=8, shift=4, lens=P, out=P, lse=None, n=4, nq=8, nkv=4,
             hd=128, win=0, scale=1.0, cap=0.0, dt=BF16, s_max=2, ws=P, bytes=1 << 30, st=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return L.bq_paged_attention(*a.values())


def test_attention_refusals(L):
    assert attn(L, n=0, q=None) == 0
    for name in ("q", "kc", "vc", "rows", "lens", "out", "ws"):
        assert attn(L, **{name: None}) == 1, name
    assert attn(L, dt=F32) == 1 and attn(L, dt=77) == 1
    for name in ("q", "kc", "vc", "out", "ws"):
        assert attn(L, **{name: C.c_void_p(264)}) == 1, name
    for kw in (dict(hd=80), dict(nq=7), dict(nkv=0), dict(width=0), dict(win=-1), dict(s_max=0),
               dict(cap=-1.0), dict(cap=float("nan")), dict(scale=float("nan")), dict(qs=1023), dict(qs=1000),
               dict(bytes=4 * 8 * 2 * 132 * 4 - 1), dict(slots=-1), dict(slots=0)):
        assert attn(L, **kw) == 2, kw
    assert attn(L, s_max=257) == 4 and attn(L, shift=31) == 4


def test_attention_plan(L):
    size = L.bq_paged_attention_workspace_size
    assert size(4, 8, 128, 1) == 0 and size(4, 8, 128, 2) == 4 * 8 * 2 * 132 * 4 and size(0, 8, 128, 2) == 0
    for n, nq, nkv, hd, longest, win in ((1, 16, 8, 256, 1500, 1024), (64, 32, 8, 128, 16384, 0), (1, 1, 1, 64, 1, 0),
                                         (3, 8, 1, 512, 2**31 - 1, 0), (1, 16, 2, 512, 50, 7)):
        s = L.bq_paged_attention_splits(n, nq, nkv, hd, longest, win)
        assert 1 <= s <= 256 and s <= max(1, -(-(min(longest, win) if win else longest) // 16) + 1)
    assert L.bq_paged_attention_splits(0, 16, 8, 256, 1500, 0) == 1


class Arr(C.Structure):
    _fields_ = [("data", C.c_void_p), ("row_bytes", C.c_int64)]


def arrays(*rows, data=256):
    return (Arr * max(len(rows), 1))(*[Arr(data, r) for r in rows])


def test_cache_refusals(L):
    def reorder(**kw):
        a = dict(arr=arrays(64, 64), na=2, rows=P, lens=P, refs=P, par=P, grow=None, n=4, width=8, shift=4, pages=32,
                 info=P, ws=P, bytes=1 << 20, st=None)
        a.update(kw)
        return L.bq_cache_reorder(*a.values())

    def compact(**kw):
        a = dict(arr=arrays(64, 64), na=2, rows=P, refs=P, n=4, width=8, shift=4, pages=32, info=P, ws=P, bytes=1 << 20,
                 st=None)
        a.update({k: v for k, v in kw.items() if k in a})
        return L.bq_cache_compact(*a.values())

    assert reorder(n=0, rows=None) == 0 and compact(n=0, rows=None) == 0
    assert reorder(lens=None) == 1 and reorder(par=None) == 1
    assert reorder(bytes=L.bq_cache_reorder_workspace_size(4) - 1) == 2
    assert compact(bytes=L.bq_cache_compact_workspace_size(32) - 1) == 2
    for call in (reorder, compact):
        for name in ("rows", "refs", "info", "ws", "arr"):
            assert call(**{name: None}) == 1, name
        assert call(ws=C.c_void_p(264)) == 1
        assert call(arr=arrays(64, 64, data=0)) == 1
        for kw in (dict(width=0), dict(pages=0), dict(na=-1), dict(arr=arrays(64, 0)), dict(arr=arrays(64, 1 << 25))):
            assert call(**kw) == 2, kw
        for kw in (dict(shift=-1), dict(shift=21), dict(n=1025), dict(na=129), dict(pages=1 << 28),
                   dict(n=1024, width=1 << 21)):
            assert call(**kw) == 4, kw
    assert L.bq_cache_reorder_workspace_size(0) == 0 and L.bq_cache_compact_workspace_size(-3) == 0


def test_beam_refusals(L):
    def beam(**kw):
        a = dict(x=P, stride=1000, dt=F32, sc=C.c_void_p(512), fin=None, b=2, k=4, v=1000, n=4, eos=-1, os=P, op=P, ot=P, of=None, ws=P,
                 bytes=1 << 30, st=None)
        a.update(kw)
        return L.bq_beam_select(*a.values())

    assert beam(b=0, x=None) == 0
    for name in ("x", "sc", "os", "op", "ot", "ws"):
        assert beam(**{name: None}) == 1, name
    assert beam(dt=2) == 1 and beam(x=C.c_void_p(258)) == 1 and beam(ws=C.c_void_p(264)) == 1
    assert beam(dt=BF16, x=C.c_void_p(257)) == 1
    assert beam(sc=P) == 1 and beam(fin=P, of=P, eos=3) == 1 and b"outputs" in L.bq_last_error()
    for kw in (dict(k=0), dict(v=0), dict(n=0), dict(stride=999), dict(eos=1000), dict(eos=-2), dict(fin=P), dict(bytes=16)):
        assert beam(**kw) == 2, kw
    for kw in (dict(k=65), dict(n=65), dict(v=(1 << 20) + 1, stride=1 << 21), dict(b=1 << 20)):
        assert beam(**kw) == 4, kw
    assert L.bq_beam_select_workspace_size(0, 5) == 0 and L.bq_beam_select_workspace_size(3, 0) == 0


@pytest.fixture(scope="module")
def spills(tmp_path_factory):
    """{mangled kernel name: (scratch bytes, spilled vector registers)} of the built library"""
    if not os.path.exists(LIB) or not os.path.exists(READELF):
        pytest.skip("no built library or no tools to read it")
    data, found = open(LIB, "rb").read(), {}
    path = tmp_path_factory.mktemp("objs") / "obj"
    for at in (m.start() for m in re.finditer(MAGIC, data)):
        p = at + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", data, p - 8)[0]):
            off, size, idlen = struct.unpack_from("<QQQ", data, p)
            target, p = data[p + 24:p + 24 + idlen], p + 24 + idlen
            if b"gfx950" not in target or size == 0:
                continue
            path.write_bytes(data[at + off:at + off + size])
            notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True, text=True).stdout
            for k in re.split(r"\n\s+- \.", notes):
                name = re.search(r"\.name:\s+(_Z\S+)", k)
                if name and ".vgpr_spill_count" in k:
                    found[name[1]] = (int(re.search(r"\.private_segment_fixed_size:\s+(\d+)", k)[1]),
                                      int(re.search(r"\.vgpr_spill_count:\s+(\d+)", k)[1]))
    return found


@pytest.mark.parametrize("kernel,instances", [("k_paged_attn", 16), ("k_paged_merge", 8), ("k_rope_append", 16), ("k_beam_pick", 9),
                                              ("k_beam_parts", 3), ("k_reorder_plan", 2), ("k_compact", 2)])
def test_no_scratch(spills, kernel, instances):
    """The kernels that keep tiles and accumulators in registers spill none of them."""
    mine = {n: v for n, v in spills.items() if f"{len(kernel)}{kernel}I" in n}
    assert len(mine) == instances, sorted(mine)
    assert not {n: v for n, v in mine.items() if v != (0, 0)}


HARNESS = r"""
#include <stdio.h>
#include "bq_pages.hpp"
int main() {
  long long a, b, c, d, e, f;
  char op;
  while (scanf(" %c", &op) == 1) {
    if (op == 's') {  // shift slots width pos base: one table row of equal entries
      scanf("%lld %lld %lld %lld %lld", &a, &b, &c, &d, &e);
      int32_t rows[64];
      for (int i = 0; i < 64; ++i) rows[i] = (int32_t)e;
      printf("%lld\n", (long long)bq::page_slot(rows, (int)c, (int)a, b, d));
    } else if (op == 'n') {
      scanf("%lld %lld %lld", &a, &b, &c);
      printf("%d\n", bq::page_number((int32_t)a, (int)b, (int32_t)c));
    } else {
      scanf("%lld %lld %lld %lld %lld %lld", &a, &b, &c, &d, &e, &f);
      const bq::SeqPlan s = bq::seq_plan((int)a, (int)b, (int)c, (int)d, (int)e, (int)f);
      printf("%d %d %d %d\n", s.parent, s.len, s.full, s.end);
    }
  }
}
"""


SHARES = r"""
#include <stdio.h>
#include "bq_pages.hpp"
int main() {
  int n, s_max, most;
  while (scanf("%d %d %d", &n, &s_max, &most) == 3) {
    static int tiles[1024];
    double sum = 0.0;
    for (int i = 0; i < n; ++i) scanf("%d", tiles + i), sum += tiles[i];
    const int units = bq::attn_units(n, s_max);
    const double share = sum > 0.0 ? units / sum : 0.0;
    for (int i = 0; i < n; ++i) printf("%d ", bq::attn_splits(tiles[i], share, bq::kRoundDown, most));
    int up = 0;
    for (int i = 0; i < n; ++i)
      up += bq::attn_splits(tiles[i], sum > 0.0 ? (units - n) / sum : 0.0, bq::kRoundUp, most);
    printf("%d\n", units < n || up <= units);
  }
}
"""


def test_attention_shares(tmp_path):
    """Slots shared out by length: never more than there are, at least one each, as many as asked
    for where all are alike, most of them to the one that is long."""
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    src, exe = tmp_path / "shares.cpp", tmp_path / "shares"
    src.write_text(SHARES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unused-result", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-I", os.path.join(ROOT, "mojo-gemma4-cpu_amd", "csrc"), str(src), "-o",
                    str(exe)], check=True)
    rng, cases = random.Random(6), []
    for _ in range(2000):
        n, s_max, most = rng.choice([1, 2, 3, 17, 64, 65, 300]), rng.choice([2, 3, 9, 33, 256]), rng.choice([6, 128, 256])
        top = rng.choice([0, 5, 40, 3000, 2**27])
        tiles = [rng.randint(0, top) for _ in range(n)]
        if rng.random() < 0.3:
            tiles = [top] * n
        if rng.random() < 0.3:
            tiles[rng.randrange(n)] = 2**27
        cases.append((s_max, most, tiles))
    text = "\n".join(f"{len(t)} {s} {m} " + " ".join(map(str, t)) for s, m, t in cases)
    got = subprocess.run([str(exe)], input=text, text=True, capture_output=True, check=True).stdout.splitlines()
    assert len(got) == len(cases)
    for (s_max, most, tiles), line in zip(cases, got):
        *n, fits = (int(v) for v in line.split())
        assert fits  # where a search for the largest share that fits begins
        assert len(n) == len(tiles) and sum(n) <= len(n) * s_max
        assert all(1 <= v <= max(1, min(most, t // 6)) for v, t in zip(n, tiles))
        each = s_max if len(n) == 1 else s_max - 1
        if len(set(tiles)) == 1:
            assert set(n) == {max(1, min(each, most, tiles[0] // 6))}
        if sorted(tiles)[-1] == 2**27 and sum(tiles) < 2**27 + 2**20:
            assert max(n) >= min(most, int(each * len(n) * 0.99))


def test_page_arithmetic(tmp_path):
    """The header that the kernels use, built for the CPU: no entry leads outside the cache."""
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    src, exe = tmp_path / "pages.cpp", tmp_path / "pages"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "mojo-gemma4-cpu_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    rng, lines, want = random.Random(5), [], []
    big = 2**31 - 1
    for _ in range(3000):
        shift = rng.choice([0, 1, 4, 5, 10, 20])
        slots = rng.choice([0, 1, 1 << shift, (5 << shift) + rng.randrange(3), big])
        base = rng.choice([-1, -(2**31), 0, big, rng.randrange(0, big), 3 << shift, max(0, slots - (1 << shift)),
                           slots - (1 << shift) + 1])
        base = max(-(2**31), min(big, base))
        width, pos = rng.choice([1, 7, 64]), rng.choice([-1, 0, rng.randrange(0, 64 << shift), 64 << shift, 2**40])
        lines.append(f"s {shift} {slots} {width} {pos} {base}")
        table = torch.full((1, width), base, dtype=torch.int64)
        slot = slot_of(table, 0, pos, shift, slots)
        assert slot == -1 or 0 <= slot < slots
        want.append(str(slot))
        pages = rng.choice([1, 5, 1000])
        lines.append(f"n {base} {shift} {pages}")
        ok = base >= 0 and base % (1 << shift) == 0 and base >> shift < pages
        want.append(str(base >> shift if ok else -1))
        n, parent = rng.choice([1, 9]), rng.choice([-5, -1, 0, 3, 8, 9, big])
        length, grow = (rng.choice([-7, 0, 1, 16, 17, 4096, big]) for _ in range(2))
        lines.append(f"p {parent} {n} {length} {grow} {width} {shift}")
        p = parent if 0 <= parent < n else -1
        real = min(max(0, length), width << shift) if p >= 0 else 0
        end = min(width, (real + max(0, grow) + (1 << shift) - 1) >> shift)
        want.append(f"{p} {real} {real >> shift} {end}")
    got = subprocess.run([str(exe)], input="\n".join(lines), capture_output=True, text=True, check=True).stdout.split("\n")
    assert got[:len(want)] == want


@pytest.mark.parametrize("seed", range(12))
def test_page_reference_invariants(seed):
    """After any reorder: counts are the entries that hold a page, pages that will be written have
    one holder, every sequence reads what its parent held, and packing changes neither."""
    rng = random.Random(seed)
    shift, n, width = rng.choice([0, 1, 3]), rng.choice([1, 3, 8]), 6
    pages = n * width + rng.choice([0, 5])
    rows = 1 << shift
    cache = Pages(torch.full((n, width), -1), torch.zeros(n, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32),
                  shift, [torch.zeros(pages * rows, 2, dtype=torch.int64)])
    history = [[] for _ in range(n)]
    stamp = 0
    for step in range(30):
        parents = [rng.choice([-1] + list(range(n))) if rng.random() < 0.7 else i for i in range(n)]
        grow = [rng.choice([0, 1, rows, 2 * rows + 1]) for _ in range(n)]
        info = cache.reorder(parents, grow)
        assert info[2] == 0
        history = [list(history[p]) if p >= 0 else [] for p in parents]
        for i in range(n):
            for _ in range(rng.randrange(0, grow[i] + 1)):
                at = cache.lens[i]
                if at >= width * rows:
                    break
                stamp += 1
                cache.arrays[0][cache.table[i][at >> shift] * rows + (at & (rows - 1))] = stamp
                history[i].append(stamp)
                cache.lens[i] += 1
        if rng.random() < 0.4:
            cache.compact()
            held = sum(r != 0 for r in cache.refs)
            assert all(r != 0 for r in cache.refs[:held])
        count = [0] * pages
        for t in cache.table:
            for p in t:
                if p >= 0:
                    count[p] += 1
        assert count == cache.refs
        for i in range(n):
            got = [int(cache.arrays[0][cache.table[i][j >> shift] * rows + (j & (rows - 1)), 0]) for j in range(cache.lens[i])]
            assert got == history[i]


def test_rope_frequencies():
    import math

    import bq
    f, m = bq.rope_frequencies(64, 10000.0, device="cpu")
    assert m == 1.0 and f.shape == (64,) and f[0] == 1.0 and abs(float(f[32]) - 0.01) < 1e-9
    g, m = bq.rope_frequencies(64, 10000.0, factor=4.0, device="cpu")
    assert m == 1.0 and torch.allclose(g * 4, f, rtol=1e-6)
    g, m = bq.rope_frequencies(64, 10000.0, factor=4.0, original_len=4096, device="cpu")
    assert abs(m - (0.1 * math.log(4.0) + 1.0)) < 1e-12
    assert g[0] == f[0] and torch.allclose(g[-1] * 4, f[-1], rtol=1e-6) and bool((g <= f).all())
    for kw in (dict(rope_half=0), dict(rope_half=4, base=1.0), dict(rope_half=4, factor=0.5),
               dict(rope_half=4, factor=2.0, original_len=10, beta_fast=1.0, beta_slow=1.0)):
        with pytest.raises(ValueError):
            bq.rope_frequencies(device="cpu", **kw)
