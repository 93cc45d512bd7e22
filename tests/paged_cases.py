"""64-bit references of the paged 16-bit cache's operators, written from their
definitions: rotary append, attention of one token per sequence, the pages'
bookkeeping (followed one page at a time), and beam selection."""
import numpy as np
import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def slot_of(table, seq, pos, shift, num_slots):
    """The cache row of a position, or -1."""
    if pos < 0 or seq < 0 or seq >= table.shape[0] or (pos >> shift) >= table.shape[1]:
        return -1
    base = int(table[seq, pos >> shift])
    return base + (pos & ((1 << shift) - 1)) if 0 <= base <= num_slots - (1 << shift) else -1


def rope_ref(x, hd, positions, inv_freq, stride, mscale, gain, normed, turned, n_eps):
    """x [T, H*hd] (any float) -> f64 result and the magnitude its 32-bit error goes by."""
    t = x.shape[0]
    y = x.double().reshape(t, -1, hd).clone()
    if normed:
        y = y * (hd ** 0.5 / torch.sqrt(y.square().sum(-1, keepdim=True) + n_eps))
        if gain is not None:
            y = y * gain.double()
    size = y.abs()
    n = 0 if inv_freq is None else inv_freq.numel()
    if turned and n:
        i = torch.arange(n)
        a, b = (2 * i, 2 * i + 1) if stride == 0 else (i, i + stride)
        angle = positions.double()[:, None, None] * inv_freq.double()
        c, s = mscale * torch.cos(angle), mscale * torch.sin(angle)
        u, v = y[..., a].clone(), y[..., b].clone()
        size[..., a] = size[..., b] = abs(mscale) * (u.abs() + v.abs())
        y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y.reshape(t, -1), size.reshape(t, -1)


def attention_ref(q, k_cache, v_cache, table, lens, nq, nkv, hd, shift, window=0, scale=None, softcap=0.0):
    """-> (out f64 [S, nq*hd], lse f64 [S, nq], tolerance [S, nq*hd]); all on the CPU.

    The tolerance: half a step of the result, and for the weights half a step each
    (they are rounded for the product with v) plus what 32-bit scores are off by: a sum
    of hd products, hd + 8 roundings of 2^-24 of the sum of magnitudes, and 2^-18 for
    the exponential, tanh and the sums."""
    eps, s = EPS[q.dtype], q.shape[0]
    scale = hd ** -0.5 if scale is None else scale
    out, lse, tol = (torch.zeros(s, nq * hd, dtype=torch.float64), torch.full((s, nq), -np.inf, dtype=torch.float64),
                     torch.zeros(s, nq * hd, dtype=torch.float64))
    g = nq // nkv
    for i in range(s):
        n = min(int(lens[i]), table.shape[1] << shift)
        at = [slot_of(table, i, p, shift, k_cache.shape[0]) for p in range(max(0, n - window) if window else 0, max(n, 0))]
        at = torch.tensor([p for p in at if p >= 0], dtype=torch.long)
        if at.numel() == 0:
            continue
        k = k_cache[at].double().view(-1, nkv, hd)
        v = v_cache[at].double().view(-1, nkv, hd)
        for h in range(nq):
            qh = q[i, h * hd:(h + 1) * hd].double()
            x = (k[:, h // g] @ qh) * scale
            off = (k[:, h // g].abs() @ qh.abs()) * abs(scale) * (hd + 8) * 2.0 ** -24 + 2.0 ** -18 * (1.0 + min(softcap, 64.0))
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            lse[i, h] = torch.logsumexp(x, 0)
            w = torch.softmax(x, 0)
            o = w @ v[:, h // g]
            weight_off = eps + 2 * off.max()
            out[i, h * hd:(h + 1) * hd] = o
            tol[i, h * hd:(h + 1) * hd] = eps * o.abs() + weight_off * (w @ v[:, h // g].abs()) + 1e-7
    return out, lse, tol


class Pages:
    """A paged cache followed on the host: tables of page numbers (-1: none), lengths,
    reference counts, and arrays of rows."""

    def __init__(self, table, lens, refs, shift, arrays):
        self.rows, self.shift = 1 << shift, shift
        self.table = [[e >> shift if self._valid(e, len(refs)) else -1 for e in t] for t in table.tolist()]
        self.lens, self.refs = lens.tolist(), refs.tolist()
        self.arrays = [a.clone() for a in arrays]

    def _valid(self, base, pages):
        return base >= 0 and base % self.rows == 0 and base // self.rows < pages

    def reorder(self, parents, grow=None):
        n, width = len(self.table), len(self.table[0])
        grow = [0] * n if grow is None else [max(0, g) for g in grow]
        old, size = self.table, [min(max(0, v), width * self.rows) for v in self.lens]
        for t in old:
            for p in t:
                if p >= 0:
                    self.refs[p] -= 1
        parents = [p if 0 <= p < n else -1 for p in parents]
        self.lens = [size[p] if p >= 0 else 0 for p in parents]
        self.table = []
        for p, length, g in zip(parents, self.lens, grow):
            full, end = length // self.rows, min(width, -(-(length + g) // self.rows))
            self.table.append([old[p][j] if p >= 0 and (j < full or (j == full and j < end)) else -1
                               for j in range(width)])
            for e in self.table[-1]:
                if e >= 0:
                    self.refs[e] += 1
        free = [p for p, r in enumerate(self.refs) if r == 0]
        fresh = copied = missing = 0
        moves = []
        for i, (length, g) in enumerate(zip(self.lens, grow)):
            full, end = length // self.rows, min(width, -(-(length + g) // self.rows))
            for j in range(full, end):
                source = self.table[i][j]
                if source >= 0 and self.refs[source] == 1:
                    continue
                if source >= 0:
                    self.refs[source] -= 1
                if not free:
                    self.table[i][j] = -1
                    missing += 1
                    continue
                page = free.pop(0)
                self.table[i][j], self.refs[page] = page, 1
                fresh += 1
                if source >= 0 and length % self.rows:
                    moves.append((source, page, length % self.rows))
        for source, page, rows in moves:
            for a in self.arrays:
                a[page * self.rows:page * self.rows + rows] = a[source * self.rows:source * self.rows + rows]
        return [fresh, len(moves), missing, 0]

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p, r in enumerate(self.refs) if not r and p < len(live)]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for source, page in to.items():
            self.refs[page], self.refs[source] = self.refs[source], 0
            for a in self.arrays:
                a[page * self.rows:(page + 1) * self.rows] = a[source * self.rows:(source + 1) * self.rows]
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return [len(live), len(to), 0, 0]

    def base_rows(self):
        return torch.tensor([[p << self.shift if p >= 0 else -1 for p in t] for t in self.table], dtype=torch.int32)


def beam_ref(logits, scores, n, finished=None, eos=-1):
    """-> scores f64, parents, tokens, finished (lists per request, padded)."""
    b, k = scores.shape
    x = logits.double().clone()
    x[torch.isnan(x)] = -np.inf
    v = x.shape[1]
    out = []
    for r in range(b):
        cand = []
        for j in range(k):
            row, s = r * k + j, float(scores[r, j])
            if finished is not None and bool(finished[r, j]):
                if s > -np.inf:
                    cand.append((-s, j * v + eos))
                continue
            if torch.isinf(x[row]).all() or (x[row] == np.inf).any():
                continue
            y = s + (x[row] - torch.logsumexp(x[row], 0))
            keep = torch.nonzero(y > -np.inf)[:, 0]
            if keep.numel() > 4 * n + 64:  # no more than these can be among the n best
                least = torch.topk(y[keep], n).values[-1]
                keep = keep[y[keep] >= least]
            cand += [(-float(y[i]), j * v + int(i)) for i in keep.tolist()]
        cand = sorted(cand)[:n]
        row = [(-s, r * k + f // v, f % v) for s, f in cand] + [(-np.inf, -1, -1)] * (n - len(cand))
        out.append(row)
    sc = torch.tensor([[c[0] for c in row] for row in out], dtype=torch.float64)
    pa = torch.tensor([[c[1] for c in row] for row in out], dtype=torch.int32)
    tk = torch.tensor([[c[2] for c in row] for row in out], dtype=torch.int32)
    fin = torch.zeros(b, n, dtype=torch.uint8)
    for r in range(b):
        for i in range(n):
            p = int(pa[r, i])
            if p >= 0:
                fin[r, i] = int((finished is not None and bool(finished.reshape(-1)[p])) or int(tk[r, i]) == eos)
    return sc, pa, tk, fin
