"""Plain 64-bit forms of the attention-side operators (cache append, paged attention, page bookkeeping) and error
bounds for the kernels, derived from their arithmetic.

Unit roundoffs: 2^-8 (bf16), 2^-11 (fp16), 2^-4 (e4m3), 2^-24 (fp32)."""
from __future__ import annotations

import math

import torch

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}   # half a step below the normal range


def attend(kv, table, lens, q, *, layer=0, seqs=None, window=0, scale=None, k_scale=None, v_scale=None):
    """``(out, lse, out_tol, lse_tol)`` in 64 bits for q [B, L, Hq, D]; only positions that a token sees are touched.

    Bounds.  A score is a 32-bit sum of D exact products, off by at most d = (D + 2) 2^-23 scale sum |q k|, and
    exponentials and maxima come from such scores, so a probability is off by a factor of at most 1 + 2 d (against its
    sum: 4 d) plus 2^-20 of exponential and joins; a sum over N positions in 32 bits adds N 2^-23.  Probabilities enter
    the second product in two 16-bit parts (2^-15 left) over a 16-bit cache, in one fp16 (2^-11, and 2^-25 absolute
    below its normal range) over an 8-bit one.  The result is rounded once."""
    B, L, Hq, D = q.shape
    Hkv, ps = kv.shape[3], kv.shape[4]
    G = Hq // Hkv
    f8 = kv.dtype == torch.float8_e4m3fn
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, L, Hq, D, dtype=torch.float64)
    lse = torch.full((B, L, Hq), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    table, lens = table.cpu(), lens.cpu()
    rows = range(B) if seqs is None else seqs.tolist()
    for b, row in enumerate(rows):
        if not 0 <= row < table.shape[0]:
            continue
        n = int(lens[row])
        pages = [int(x) for x in table[row][: -(-n // ps)]]
        first = max(0, n - L + 1 - window) // ps if window else 0
        held = [p if 0 <= p < kv.shape[2] and i >= first else None for i, p in enumerate(pages)]
        ids = torch.tensor([p for p in held if p is not None], dtype=torch.long, device=kv.device)
        if not len(ids):
            continue
        where = torch.cat([torch.arange(i * ps, (i + 1) * ps) for i, p in enumerate(held) if p is not None])
        raw = kv[layer].view(torch.uint8 if f8 else torch.int16)
        k, v = (raw[i].index_select(0, ids).view(kv.dtype).double().cpu().transpose(1, 2).reshape(-1, Hkv, D)
                for i in (0, 1))
        if k_scale is not None:
            k = k * k_scale.double().cpu()[:, None]
        if v_scale is not None:
            v = v * v_scale.double().cpu()[:, None]
        for t in range(L):
            at = n - L + t
            see = (where <= at) & (where < n)
            if window:
                see &= where > at - window
            if not bool(see.any()):
                continue
            ks, vs = k[see], v[see]
            N = ks.shape[0]
            qq = q[b, t].double().cpu().view(Hkv, G, D)
            s = torch.einsum("hgd,thd->hgt", qq, ks) * scale
            d = (D + 2) * 2.0 ** -23 * scale * torch.einsum("hgd,thd->hgt", qq.abs(), ks.abs()).amax(-1)
            p = s.softmax(-1)
            o = torch.einsum("hgt,thd->hgd", p, vs)
            mass = torch.einsum("hgt,thd->hgd", p, vs.abs())
            eps = 4 * d + 2.0 ** -20 + N * 2.0 ** -23 + (2.0 ** -11 if f8 else 2.0 ** -15)
            floor = N * 2.0 ** -25 * vs.abs().amax() if f8 or q.dtype == torch.float16 else 0.0
            u = ROUND[q.dtype]
            out[b, t] = o.reshape(Hq, D)
            out_tol[b, t] = ((o.abs() + eps[..., None] * mass) * u + eps[..., None] * mass + floor
                             + TINY[q.dtype]).reshape(Hq, D)
            ls = s.logsumexp(-1)
            lse[b, t] = ls.reshape(Hq)
            lse_tol[b, t] = (2 * d + N * 2.0 ** -23 + 2.0 ** -20 + 2.0 ** -21 * ls.abs()).reshape(Hq)
    return out, lse, out_tol, lse_tol


def assert_within(got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), "finite in different places"
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin])
    over = ((got - want).abs() - tol)[fin]
    assert not over.numel() or over.max() <= 0, f"{int((over > 0).sum())} of {over.numel()} out of bounds, by up to {over.max():.3g}"


def rope(x, positions, freqs, rot, *, interleaved=False, mscale=1.0, weight=None, eps=1e-6, offset=0.0):
    """``(y, tol)`` in 64 bits before rounding: norm per head, then rotation.  tol is the 32-bit arithmetic's share:
    2^-21 from the norm, 2^-21 from sine and cosine, three roundings of 2^-24, against |a| + |b| of the pair."""
    x = x.detach().double().cpu()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.double().cpu() + offset)
    y, mag = x.clone(), x.abs()
    angle = positions.double().cpu()[:, None] * torch.tensor(freqs, dtype=torch.float64)
    cos, sin = (angle.cos() * mscale)[:, None], (angle.sin() * mscale)[:, None]
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    both = (x[..., a].abs() + x[..., b].abs()) * max(1.0, mscale)
    mag[..., a], mag[..., b] = both, both
    return y, mag * 2.0 ** -19


def rounded_tol(y, tol, dtype):
    return (y.abs() + tol) * ROUND[dtype] + tol + TINY[dtype]


def e4m3_tol(y, tol, scale):
    """Bounds of code * scale against y: the type's roundoff, or half its smallest step."""
    return torch.maximum((y.abs() + tol) * 2.0 ** -4, torch.as_tensor(scale) * 2.0 ** -10) * (1 + 2.0 ** -20) + tol


class Pages:
    """The page bookkeeping, one sequence at a time on Python lists."""

    def __init__(self, table, lens, refs, ps):
        self.table, self.lens, self.refs, self.ps = table.tolist(), lens.tolist(), refs.tolist(), ps
        self.copies = []   # (src, dst, tokens)

    def extend(self, seqs, new):
        first, todo, bad = set(), [], False
        for s, n in zip(seqs, new):
            ok = 0 <= s < len(self.lens) and s not in first and n >= 0
            first.add(s)
            ok = ok and self.lens[s] + n <= len(self.table[s]) * self.ps
            if ok and n and self.lens[s] % self.ps:
                ok = 0 <= self.table[s][self.lens[s] // self.ps] < len(self.refs)
            bad |= not ok
            todo += [(s, n)] if ok else []
        holders = {}
        for s, n in todo:
            if n and self.lens[s] % self.ps:
                p = self.table[s][self.lens[s] // self.ps]
                if self.refs[p] > 1:
                    holders.setdefault(p, []).append(s)
        keep = {v[0] for p, v in holders.items() if len(v) == self.refs[p]}
        cow = {s: p for p, v in holders.items() for s in v if s not in keep}
        need = {s: -(-(self.lens[s] + n) // self.ps) - -(-self.lens[s] // self.ps) + (s in cow) for s, n in todo}
        free = [i for i, r in enumerate(self.refs) if r == 0]
        if sum(need.values()) > len(free):
            return bad, True
        free = iter(free)
        for s, n in todo:
            have = -(-self.lens[s] // self.ps)
            if s in cow:
                to = next(free)
                self.copies.append((cow[s], to, self.lens[s] % self.ps))
                self.refs[cow[s]] -= 1
                self.refs[to] = 1
                self.table[s][have - 1] = to
            for j in range(have, -(-(self.lens[s] + n) // self.ps)):
                self.table[s][j] = next(free)
                self.refs[self.table[s][j]] = 1
            self.lens[s] += n
        return bad, False

    def fork(self, src, dst):
        bad = False
        for i, (s, d) in enumerate(zip(src, dst)):
            m = len(self.lens)
            if not (0 <= s < m and 0 <= d < m) or d in src or d in dst[:i] or self.lens[d]:
                bad = True
                continue
            have = -(-self.lens[s] // self.ps)
            self.table[d][:have] = self.table[s][:have]
            for p in self.table[s][:have]:
                self.refs[p] += 1
            self.lens[d] = self.lens[s]
        return bad

    def truncate(self, seqs, lens):
        bad, first = False, set()
        for s, n in zip(seqs, lens):
            if not 0 <= s < len(self.lens) or s in first or not 0 <= n <= self.lens[s]:
                bad = True
                first.add(s)
                continue
            first.add(s)
            for j in range(-(-n // self.ps), -(-self.lens[s] // self.ps)):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = n
        return bad

    def compact(self):
        live = [i for i, r in enumerate(self.refs) if r]
        up = [i for i in live if i >= len(live)]
        down = [i for i, r in enumerate(self.refs) if not r and i < len(live)]
        to = dict(zip(up, down))
        self.copies += [(a, b, self.ps) for a, b in to.items()]
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
