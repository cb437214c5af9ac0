"""A paged cache held in 8 bits from its definition, in 64 bits on the CPU: what
tests compare the references and the kernels with."""
import math

import torch

PAGE = 16


def e4m3(x):
    """float64 rounded to e4m3: 4 bits of mantissa from 2^-6 on, steps of 2^-9
    below, nearest even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    y = torch.round(x / step) * step
    assert not (y.abs() > 448).any()
    return y


def power(big):
    """The least power of two from 2^-126 on whose multiple of 448 is at least
    big."""
    e = -126
    while 448.0 * 2.0 ** e < big:
        e += 1
    return 2.0 ** e


class Cache:
    """Values [pages, heads, 16, dim] over their scales [pages, heads]: keys and
    values."""

    def __init__(self, pages, heads, dim):
        self.x = [torch.zeros(pages, heads, PAGE, dim, dtype=torch.float64)
                  for _ in range(2)]
        self.scale = torch.zeros(pages, heads, 2, dtype=torch.float64)

    def load(self, k_cache, v_cache, kv_scale):
        k, v = k_cache.cpu().double(), v_cache.cpu().double()
        self.x = [k.transpose(2, 3).flatten(3, 4), v.transpose(2, 3)]
        self.x = [x.contiguous() for x in self.x]
        self.scale = kv_scale.cpu().double()
        return self

    def write(self, k, v, slots):
        """Page by page, each one's tokens side by side in slots but for
        skipped ones."""
        pages = self.scale.shape[0]
        runs, last = [], -1
        for t, s in enumerate(slots):
            if not 0 <= s < pages * PAGE:
                continue
            if s // PAGE == last:
                runs[-1].append(t)
            else:
                runs.append([t])
            last = s // PAGE
        for run in runs:
            page = slots[run[0]] // PAGE
            offs = [slots[t] % PAGE for t in run]
            for i, new in enumerate((k, v)):
                for h in range(new.shape[1]):
                    x = new[run, h].cpu().double()
                    big = x[x.isfinite()].abs().max().item() \
                        if x.isfinite().any() else 0.0
                    now = power(big)
                    kept = self.x[i][page, h]
                    if 0 in offs:
                        kept.zero_()
                    else:
                        was = self.scale[page, h, i].item()
                        now = max(was, now)
                        if now != was:
                            kept.copy_(e4m3(kept * (was / now)))
                    self.scale[page, h, i] = now
                    x = torch.where(x.isfinite(), x, math.nan)
                    for o, row in zip(offs, x):
                        kept[o] = e4m3(row / now)

    def values(self, i):
        return self.x[i] * self.scale[..., i, None, None]


def same(a, b):
    """Equal, NaN where NaN."""
    a, b = a.cpu().double(), b.cpu().double()
    return torch.equal(a.isnan(), b.isnan()) and \
        torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


def attend(q, k, v, table, cu, total, scale):
    """(result, weighted sum of |v|, largest sum of |q k| of a row) in 64 bits;
    k, v [pages, heads, 16, dim]. Rows that see no key: zeros."""
    heads, dim = q.shape[1:]
    per = heads // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    big, most = torch.zeros_like(out), torch.zeros_like(out)
    for s, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        n = b - a
        L = max(min(total[s], table.shape[1] * PAGE), 0)
        if n <= 0 or L == 0:
            continue
        ids = table[s, :-(-L // PAGE)].long()
        kk, vv = (x[ids].transpose(1, 2).reshape(-1, *x.shape[1::2])[:L]
                  .repeat_interleave(per, 1) for x in (k, v))
        qq = q[a:b].cpu().double()
        z = torch.einsum("thd,lhd->htl", qq, kk) * scale
        limit = total[s] - n + 1 + torch.arange(n)
        gone = torch.arange(L)[None] >= limit[:, None]
        z = z.masked_fill(gone, -math.inf)
        p = torch.softmax(z, -1)
        p = torch.where((limit > 0)[None, :, None], p, 0.0)
        out[a:b] = torch.einsum("htl,lhd->thd", p, vv)
        big[a:b] = torch.einsum("htl,lhd->thd", p, vv.abs())
        sums = torch.einsum("thd,lhd->htl", qq.abs(), kk.abs()) * abs(scale)
        most[a:b] = sums.masked_fill(gone, 0.0).amax(-1).T[..., None]
    return out, big, most


def layout(lens, spare, seed, width=None):
    """Scattered pages for sequences of these lengths: (table, pages)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // PAGE) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).int()
    table = torch.zeros(len(lens), max(need + [1]) if width is None else width,
                        dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def slots_of(table, old, new):
    """Slots of positions [old, new) of every sequence, in their order."""
    return [int(table[i, p // PAGE]) * PAGE + p % PAGE
            for i, (a, b) in enumerate(zip(old, new)) for p in range(a, b)]
