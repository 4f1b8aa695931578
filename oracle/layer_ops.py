"""Oracle: what stands between a quantized layer's products (test infrastructure only).

Norms, rotary positions and low-rank adapters in fp64 with the bound of their fp32 roundings;
page tables as lists of whole numbers.
"""
import math

import torch

from oracle.serving import TINY, UNIT

E = 2.0 ** -24  # a rounding to fp32


def rms_norm(x, weight, eps, residual=None):
    """(y, s) in fp64."""
    s = x.double() if residual is None else x.double() + residual.double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * weight.double()
    return y, s


def rms_norm_error(columns):
    """Relative error of y before its rounding: s is rounded (1) and enters twice; its squares
    are summed by at least min(columns / 8, 256) threads, so that a term passes at most
    columns / 256 + 8 sums of its thread and 10 joining threads and waves, which the root
    halves; mean, eps, root and quotient (4), the products with both factors (2)."""
    return (2 + (columns / 256 + 18) / 2 + 6) * E


def rounded(dtype, y, error):
    """Bound of a result with absolute ``error`` before it is rounded to ``dtype``."""
    return error + UNIT[dtype] * (y.abs() + error) + TINY[dtype]


def rotary(x, positions, theta, m, n, interleaved):
    """fp64 result, and the bound of its error before the last rounding.

    The position's product with the frequency in turns rounds thrice in 64 bits (3·2^-53 of the
    angle, and what the oracle loses itself); the turn left over is at most half and is rounded
    to 32 bits (2^-26 of a turn); sine and cosine have two units of 2^-23 each, and the factor
    rounds once; two products and a sum round thrice."""
    angle = positions.double()[:, None] * theta[None]
    c, s = m * torch.cos(angle)[:, None], m * torch.sin(angle)[:, None]
    x = x.double()
    a, b = (x[..., :n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    u, v = a * c - b * s, a * s + b * c
    off = abs(m) * (6 * 2.0 ** -53 * angle.abs() + 2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -23 + E)
    w = (a.abs() + b.abs()) * (off[:, None] + 3 * E * abs(m))
    out, err = x.clone(), torch.zeros_like(x)
    if interleaved:
        out[..., :n:2], out[..., 1:n:2], err[..., :n:2], err[..., 1:n:2] = u, v, w, w
    else:
        out[..., :n // 2], out[..., n // 2:n], err[..., :n // 2], err[..., n // 2:n] = u, v, w, w
    return out, err


def adapters(x, index, down, up, scale, base):
    """fp64 result, and the bound of its error before the last rounding.

    First product: a term passes at most 32 sums of a matrix instruction, one instruction for
    64 columns, and the joining of 4 waves and 8 shares.  h enters the second as two 16-bit
    numbers (bf16: 2^-16 of it is left out; fp16: 2^-22 of it, or 2^-38 of the row's largest),
    after one rounding with the scale; a term passes 32 sums and one for each 16 ranks.  Then
    the base's sum."""
    T, N = x.shape[0], up[0].shape[0]
    out = torch.zeros(T, N, dtype=torch.float64) if base is None else base.double().clone()
    err = out.abs() * E
    K = x.shape[1]
    first, lost = (32 + K / 64 + 12) * E, UNIT[x.dtype] ** 2
    for a, (d, u) in enumerate(zip(down, up)):
        t = (index == a).nonzero()[:, 0]
        if not len(t):
            continue
        d, u, xt = d.double(), u.double(), x[t].double()
        h, size = xt @ d.T, xt.abs() @ d.abs().T
        herr = (first * size + (lost + E) * h.abs() + 2.0 ** -38 * h.abs().amax(1, keepdim=True))
        part, terms = h @ u.T * scale[a], h.abs() @ u.abs().T * abs(scale[a])
        out[t] += part
        err[t] += (herr @ u.abs().T * abs(scale[a]) + (32 + d.shape[0] / 16 + 2) * E * terms
                   + 2 * E * out[t].abs())
    return out, err


class Pages:
    """Page tables one request at a time."""

    def __init__(self, pages, page, seqs, width):
        self.page, self.width, self.seqs = page, width, seqs
        self.free = list(range(pages - 1, -1, -1))
        self.rows, self.lengths = [[] for _ in range(seqs)], [0] * seqs
        self.bad = self.full = False

    def extend(self, rows, new, total):
        """(table, cu, kv_lens, slots, positions) as lists."""
        table, cu, kv, slots, positions = [], [0], [], [-1] * total, [0] * total
        seen, end, short = set(), 0, False
        for row, n in zip(rows, new):
            if n < 0:
                self.bad, n = True, 0
            start, end = end, end + n
            known = 0 <= row < self.seqs and row not in seen
            self.bad |= row >= self.seqs or row in seen
            if known:
                seen.add(row)
            if n and end > total:
                self.bad = True
            elif n and known:
                had = -(-self.lengths[row] // self.page)
                need = -(-(self.lengths[row] + n) // self.page)
                if need > self.width:
                    self.full = True
                elif need > had and (short or need - had > len(self.free)):
                    # (later requests that need pages wait for this one)
                    self.full = short = True
                else:
                    self.rows[row] += [self.free.pop() for _ in range(need - had)]
                    for j in range(n):
                        p = self.lengths[row] + j
                        slots[start + j] = self.rows[row][p // self.page] * self.page \
                            + p % self.page
                        positions[start + j] = p
                    self.lengths[row] += n
            cu.append(min(end, total))
            kv.append(self.lengths[row] if known else 0)
            mine = self.rows[row] if known else []
            table.append(mine + [-1] * (self.width - len(mine)))
        return table, cu, kv, slots, positions

    def release(self, rows, keep=None):
        seen, back = set(), []
        for i, row in enumerate(rows):
            m = 0 if keep is None else keep[i]
            if row < 0:
                continue
            if row >= self.seqs or row in seen:
                self.bad = True
                continue
            seen.add(row)
            if not 0 <= m <= self.lengths[row]:
                self.bad = True
                continue
            kept = -(-m // self.page)
            back += self.rows[row][kept:]
            self.rows[row], self.lengths[row] = self.rows[row][:kept], m
        self.free += back[::-1]

    def table(self):
        return [r + [-1] * (self.width - len(r)) for r in self.rows]
