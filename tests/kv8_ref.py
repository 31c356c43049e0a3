"""The 8-bit cache and its attention in 64 bits, cell by cell, on the CPU: what the GPU tests compare with."""
import math

import numpy as np
import torch

BLOCK, PAGE = 32, 256
E_MIN, E_MAX = -40, 40


def scale_exp(top: float) -> int:
    """The smallest exponent in range with top <= 127 * 2^e."""
    e = E_MIN
    while e < E_MAX and top > 127 * 2.0 ** e:
        e += 1
    return e


class Cells:
    """One tensor's cells: codes [streams, cells, heads, D] and exponents [streams, blocks, heads]."""

    def __init__(self, s, cells, heads, d, codes=None, exps=None):
        self.codes = np.zeros((s, cells, heads, d), np.int64) if codes is None else codes.astype(np.int64)
        self.exps = np.zeros((s, cells // BLOCK, heads), np.int64) if exps is None else exps.astype(np.int64)

    def copy(self):
        return Cells(*self.codes.shape, self.codes.copy(), self.exps.copy())

    def write(self, rows, first, count):
        """rows [streams, n, heads, D] (float64); stream s's rows j < count[s] to cells first[s] + j."""
        for s in range(rows.shape[0]):
            lo, hi = max(0, first[s]), min(self.codes.shape[1], first[s] + count[s])
            for b in range(lo // BLOCK, -(-hi // BLOCK) if hi > lo else 0):
                c0, c1 = max(lo, b * BLOCK), min(hi, (b + 1) * BLOCK)
                for h in range(rows.shape[2]):
                    new = rows[s, c0 - first[s]:c1 - first[s], h]
                    mag = np.abs(new[np.isfinite(new)])
                    e = scale_exp(float(mag.max()) if mag.size else 0.0)
                    if c0 > b * BLOCK:
                        was = int(np.clip(self.exps[s, b, h], E_MIN, E_MAX))
                        e = max(e, was)
                        kept = self.codes[s, b * BLOCK:c0, h]
                        self.codes[s, b * BLOCK:c0, h] = np.rint(kept * 2.0 ** (was - e))
                    code = np.clip(np.rint(np.where(np.isnan(new), 0.0, new) * 2.0 ** -e), -127, 127)
                    self.codes[s, c0:c1, h] = code
                    self.exps[s, b, h] = e

    def values(self):
        e = np.clip(self.exps, E_MIN, E_MAX).repeat(BLOCK, axis=1)
        return self.codes * np.exp2(e.astype(np.float64))[..., None]

    def pack_key(self):
        s, n, h, d = self.codes.shape
        x = self.codes.reshape(s, n // BLOCK, BLOCK, h, d // 16, 16).transpose(0, 3, 1, 4, 2, 5)
        return torch.from_numpy(np.ascontiguousarray(x).astype(np.int8)), self._exps()

    def pack_value(self):
        s, n, h, d = self.codes.shape
        x = self.codes.reshape(s, n // BLOCK, BLOCK, h, d).transpose(0, 3, 1, 4, 2)
        return torch.from_numpy(np.ascontiguousarray(x).astype(np.int8)), self._exps()

    def _exps(self):
        return torch.from_numpy(np.ascontiguousarray(self.exps.transpose(0, 2, 1)).astype(np.int8))

    @staticmethod
    def unpack_key(codes, exps):
        s, h, b, c = codes.shape[:4]
        x = codes.cpu().numpy().transpose(0, 2, 4, 1, 3, 5).reshape(s, b * BLOCK, h, c * 16)
        return Cells(s, b * BLOCK, h, c * 16, x, exps.cpu().numpy().transpose(0, 2, 1))

    @staticmethod
    def unpack_value(codes, exps):
        s, h, b, d = codes.shape[:4]
        x = codes.cpu().numpy().transpose(0, 2, 4, 1, 3).reshape(s, b * BLOCK, h, d)
        return Cells(s, b * BLOCK, h, d, x, exps.cpu().numpy().transpose(0, 2, 1))


def random_cells(rng, s, cells, heads, d, lo=-6, hi=-3):
    codes = np.clip(np.rint(rng.standard_normal((s, cells, heads, d)) * 28), -127, 127)
    return Cells(s, cells, heads, d, codes, rng.integers(lo, hi + 1, (s, cells // BLOCK, heads)))


def to_pages(rng, packed, n_extra=2):
    """[streams, heads, blocks, ...] as shuffled pages [n, heads, 8, ...] and the table [streams, pages]; pages that no
    stream holds are filled with ones."""
    s, h, b = packed[0].shape[:3]
    per = b // (PAGE // BLOCK)
    order = rng.permutation(s * per + n_extra)[:s * per].reshape(s, per)
    out = []
    for t in packed:
        p = torch.ones((s * per + n_extra, h, PAGE // BLOCK, *t.shape[3:]), dtype=t.dtype)
        x = t.reshape(s, h, per, PAGE // BLOCK, *t.shape[3:]).transpose(1, 2)
        p[torch.from_numpy(order.reshape(-1))] = x.reshape(s * per, h, PAGE // BLOCK, *t.shape[3:])
        out.append(p)
    return out, torch.from_numpy(order.astype(np.int32))


def attention(q, k, v, v_exp, cached, rows, scale, mode, mask=None):
    """(out, bound) for q [S, n_q, H, D] float64 (already in f16 steps) over k, v [S, cells, heads, D] float64; rows past
    rows[s] are NaN.  `bound` is how far an element may be off before the output's own rounding:
      - a weight rounded to f16 is off by at most 2^-11 of itself (half a step), and the sum of f32 products, the
        exponent and v_exp_f32 put it off by a few units of 2^-24 of the score it is the power of: together
        (2^-11 + 2^-20 (1 + |t|max)) of sum p |v|;
      - f16 weights end at steps of 2^-24 where the largest stands at 2^10: at most 2^-35 of the largest p * 2^e per
        cell, times codes of up to 127."""
    S, n_q, H, D = q.shape
    heads = k.shape[2]
    G = H // heads
    out = np.full((S, n_q, H, D), np.nan)
    tol = np.zeros((S, n_q, H, D))
    for s in range(S):
        n = cached[s] + rows[s]
        for h in range(H):
            g = h // G
            for j in range(rows[s]):
                seen = n if mode != 1 else cached[s] + j + 1
                t = scale * (k[s, :seen, g] @ q[s, j, h])
                if mask is not None:
                    t = t + mask[s if mask.shape[0] > 1 else 0, 0, j, :seen]
                top = t.max() if seen else -math.inf
                if top == -math.inf:
                    out[s, j, h] = 0.0
                    continue
                p = np.exp(t - top)
                p /= p.sum()
                out[s, j, h] = p @ v[s, :seen, g]
                finite = np.abs(t[np.isfinite(t)]).max()
                step = np.exp2(np.clip(v_exp[s, :, g], E_MIN, E_MAX).astype(np.float64)).repeat(BLOCK)[:seen]
                tol[s, j, h] = (2.0 ** -11 + 2.0 ** -20 * (1 + finite * 1.4427)) * (p @ np.abs(v[s, :seen, g])) \
                    + seen * 2.0 ** -28 * (p * step).max()
    return out, tol
