"""A paged 8-bit cache in plain torch on the CPU: what the device's is compared with."""
import math

import torch

FLOOR = -40


def exponent(amax: float) -> int:
    """Smallest k >= -40 with amax <= 448 * 2^k, by trying."""
    k = FLOOR
    while amax > 448.0 * 2.0 ** k:
        k += 1
    return k


def rotate(x, pos, cos, sin, neox):
    """x [heads, dim] fp32 at one position: every product and sum rounded to fp32."""
    half = cos.shape[1]
    c, s, y = cos[pos], sin[pos], x.clone()
    a, b = (x[:, :half], x[:, half:2 * half]) if neox else (x[:, 0:2 * half:2], x[:, 1:2 * half:2])
    lo, hi = a * c - b * s, a * s + b * c
    if neox:
        y[:, :half], y[:, half:2 * half] = lo, hi
    else:
        y[:, 0:2 * half:2], y[:, 1:2 * half:2] = lo, hi
    return y


class PlainPages:
    def __init__(self, pages, kvh, page, dim, fill=0xFF):
        self.k = torch.full((pages, kvh, page, dim), fill, dtype=torch.uint8)  # 0xFF: undefined, where nothing was written
        self.v = torch.full((pages, kvh, dim, page), fill, dtype=torch.uint8)
        self.scales = torch.full((pages, kvh, 2), float("nan"))
        self.page, self.kvh, self.dim = page, kvh, dim

    def _put(self, raw, which, pid, h, lo, x):
        """x [n, dim] fp32 as tokens lo .. of a block; raw [page, dim] is a view of its codes."""
        bad = not bool(torch.isfinite(x).all())
        old = float(self.scales[pid, h, which]) if lo else 0.0
        if bad or math.isnan(old):
            self.scales[pid, h, which] = float("nan")
            raw[lo:lo + len(x)] = 0
            return
        new = max(old, 2.0 ** exponent(float(x.abs().max())))
        if lo and new > old:
            was = raw[:lo].contiguous().view(torch.float8_e4m3fn).float()
            raw[:lo] = (was * (old / new)).to(torch.float8_e4m3fn).view(torch.uint8)
        self.scales[pid, h, which] = new
        raw[lo:lo + len(x)] = (x / new).to(torch.float8_e4m3fn).view(torch.uint8)

    def update(self, k, v, table, lengths, rows, cos=None, sin=None, neox=True):
        """k, v [rows, kvh, dim]; `rows`: how many of them each sequence has.  Returns the rows' positions."""
        places, r0 = [], 0
        for s, (n, length) in enumerate(zip(rows, lengths)):
            pos = list(range(length - n, length))
            places += pos
            for c in sorted({p // self.page for p in pos}):
                at = [i for i, p in enumerate(pos) if p // self.page == c]
                for h in range(self.kvh):
                    lo, pid = pos[at[0]] % self.page, int(table[s][c])
                    kk = torch.stack([k[r0 + i, h].float() if cos is None else rotate(k[r0 + i, h:h + 1].float(), pos[i], cos, sin, neox)[0] for i in at])
                    self._put(self.k[pid, h], 0, pid, h, lo, kk)
                    self._put(self.v[pid, h].T, 1, pid, h, lo, torch.stack([v[r0 + i, h].float() for i in at]))
            r0 += n
        return places

    def values(self, pid):
        """(k, v) [page, kvh, dim] in fp32."""
        k = self.k[pid].view(torch.float8_e4m3fn).float() * self.scales[pid, :, 0, None, None]
        v = self.v[pid].view(torch.float8_e4m3fn).float() * self.scales[pid, :, 1, None, None]
        return k.transpose(0, 1), v.permute(2, 0, 1)

    def tokens(self, table_row, length):
        """(k, v) [length, kvh, dim] in 64 bits."""
        if length == 0:
            return (torch.zeros((0, self.kvh, self.dim), dtype=torch.float64),) * 2
        both = [self.values(int(p)) for p in table_row[:-(-length // self.page)]]
        return tuple(torch.cat([b[i] for b in both])[:length].double() for i in range(2))


def attention(pages, q, table, lengths, rows, scale, window=0, device="cpu"):
    """(out, bound) in 64 bits: the definition, and how far a result may be from it.

    Scores: operands exact in two fp16 parts up to 2^-22 of a value, sums of `dim` products in fp32: off by
    d = (2^-22 + dim 2^-24) scale sum |q_i k_i| at most, twice that after the rotation of the sum into base 2.  A weight is off by the
    factor e^d (1 + 2^-21) (exponential to 2 ulp), the sums of n weights and of n products by n 2^-24: the quotient by
    (4 d + n 2^-23 + 2^-19) max |v|.  bfloat16: weights enter the second product rounded to 11 bits, + 2^-11 max |v|, and the
    result is rounded, + 2^-8 |out|."""
    heads, dim = q.shape[1:]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    r0 = 0
    for s, (n, length) in enumerate(zip(rows, lengths)):
        k, v = (x.to(device) for x in pages.tokens(table[s], length))
        pos = torch.arange(length - n, length, device=device)
        j = torch.arange(length, device=device)
        sees = j[None] <= pos[:, None]
        if window:
            sees &= j[None] > pos[:, None] - window
        if length == 0 or n == 0:
            r0 += n
            continue
        lost = (sees[:, :, None] & (k.isnan() | v.isnan()).any(-1)[None]).any(1)  # [n, kvh]: rows that see an undefined token
        k, v = k.nan_to_num(), v.nan_to_num()
        for h in range(heads):
            g = h // (heads // pages.kvh)
            qq = q[r0:r0 + n, h].double().to(device)
            x = (qq @ k[:, g].T * scale).masked_fill(~sees, -math.inf)
            m = x.amax(-1, keepdim=True)
            w = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m)).masked_fill(~sees, 0.0)
            total = w.sum(-1, keepdim=True)
            o = (w @ v[:, g] / torch.where(total == 0, torch.ones_like(total), total)).masked_fill(lost[:, g:g + 1], math.nan)
            size = (qq.abs() @ k[:, g].abs().T * scale).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
            most = v[:, g].abs().amax()
            d = (2.0 ** -22 + dim * 2.0 ** -24) * size
            b = (4 * d + length * 2.0 ** -23 + 2.0 ** -19) * most
            if q.dtype == torch.bfloat16:
                b = b + 2.0 ** -11 * most + 2.0 ** -8 * o.abs()
            out[r0:r0 + n, h], bound[r0:r0 + n, h] = o.cpu(), b.expand_as(o).cpu()
        r0 += n
    return out, bound
