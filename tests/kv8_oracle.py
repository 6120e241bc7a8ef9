"""The paged 8-bit cache and its attention from their definitions, on the CPU: rows as fp32 / fp16 arithmetic says, softmax in 64 bits."""
import math

import torch

D, BLOCK = 128, 64
PLACE = [((r >> 2) & 3) * 16 + (r >> 5) * 8 + ((r >> 4) & 1) * 4 + (r & 3) for r in range(BLOCK)]      # of each row in a line of V


def tables(n, theta=1e6):
    angle = torch.outer(torch.arange(n, dtype=torch.float64), theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    return angle.cos().half(), angle.sin().half()


def rotate(x, cos, sin, place):
    """x [n, heads, 128] fp16, place [n]: fp32 from fp16 (the products are exact), then fp16"""
    c, s = cos[place].float()[:, None], sin[place].float()[:, None]
    a, b = x[..., :64].float(), x[..., 64:].float()
    return torch.cat((a * c - b * s, b * c + a * s), -1).half()


class Sequence:
    """The rows of one sequence, as they entered: k rotated, v, fp16 [n, Hkv, 128]"""

    def __init__(self, Hkv):
        self.k = torch.empty((0, Hkv, D), dtype=torch.float16)
        self.v = torch.empty((0, Hkv, D), dtype=torch.float16)

    def add(self, k, v):
        self.k, self.v = torch.cat((self.k, k)), torch.cat((self.v, v))

    def block(self, j):
        """codes [2][Hkv, 64, 128] (K, V by row) and scales [2][Hkv] of whole block j"""
        codes, scales = [], []
        for x in (self.k, self.v):
            x = x[j * BLOCK:(j + 1) * BLOCK].float().transpose(0, 1)
            amax = x.abs().amax((1, 2))
            inv = torch.where(amax > 0, torch.div(torch.full_like(amax, 127.0), amax), torch.zeros_like(amax))      # (127.0 / x is 127.0 times a rounded 1 / x)
            codes.append((x * inv[:, None, None]).round().add(128).to(torch.uint8))
            scales.append(torch.div(amax, torch.full_like(amax, 127.0)))
        return codes, scales

    def held(self):
        """K and V as the cache gives them back, float64 [n, Hkv, 128]"""
        out = []
        for i, x in enumerate((self.k, self.v)):
            x = x.double()
            for j in range(x.shape[0] // BLOCK):
                codes, scales = self.block(j)
                x[j * BLOCK:(j + 1) * BLOCK] = ((codes[i].double() - 128) * scales[i].double()[:, None, None]).transpose(0, 1)
            out.append(x)
        return out


def attention(q, k, v, old, window=0, sinks=0):
    """q [n, H, 128] at places old .., k and v float64 [old + n, Hkv, 128] -> (o, the weighted mean of |v|), float64 [n, H, 128]"""
    n, H, _ = q.shape
    rep = H // k.shape[1]
    at, key = torch.arange(old, old + n)[:, None], torch.arange(k.shape[0])[None]
    hide = key > at
    if window:
        hide |= (key <= at - window) & (key >= sinks)
    x = torch.einsum("nhd,khd->hnk", q.double(), k.repeat_interleave(rep, 1)) / math.sqrt(D)
    w = torch.softmax(x.masked_fill(hide, -math.inf), -1)
    v = v.repeat_interleave(rep, 1)
    return torch.einsum("hnk,khd->nhd", w, v), torch.einsum("hnk,khd->nhd", w, v.abs())


def attention_bound(o, mean_abs, keys, vmax):
    """How far fp16 outputs may be: weights are rounded to fp16 (half a step, 2^-11 of each; below 2^-14 half of 2^-24, and the largest weight is 1), the
    scores' fp32 sums and exponentials are good to 2^-16 of a weight for scores up to 64 (2^-22 x 64), the output is rounded once."""
    return (2.0 ** -11 + 2.0 ** -16) * mean_abs + keys * 2.0 ** -25 * vmax + 2.0 ** -11 * o.abs() + 2.0 ** -25
