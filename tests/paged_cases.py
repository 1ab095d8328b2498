"""Batches over a paged cache and their float64 attention, for the tests of q38_paged_append and
q38_paged_attention (CPU tensors; the tests move them to the device)."""
from __future__ import annotations

import math

import torch

BF16 = torch.bfloat16
HALF_BF16 = torch.finfo(BF16).eps / 2   # the largest relative error of one rounding to bf16
HALF_F32 = torch.finfo(torch.float32).eps / 2
HALF_16 = 2.0 ** -17                    # of a rounding to two bf16 parts, 16 bits


class Batch:
    """rows[i] new rows of sequence i, tokens[i] tokens with them; pages in a random order with
    spare ones between; `gap` rows in front of the first sequence and behind the last that belong
    to nobody."""

    def __init__(self, rows, tokens, page=16, hkv=2, dim=64, seed=0, gap=0, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page, self.hkv, self.dim = g, page, hkv, dim
        self.lens, self.ctx = list(rows), list(tokens)
        off = [gap]
        for r in rows:
            off.append(off[-1] + r)
        self.rows = off[-1] + gap
        self.off = torch.tensor(off, dtype=torch.int32)
        self.tokens = torch.tensor(tokens, dtype=torch.int32)
        used = [-(-max(t, 0) // page) for t in tokens]
        self.width = width or max(1, *used) + 1
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        # unused table entries are out of range on purpose: nobody may follow them
        self.table = torch.full((len(rows), self.width), -7, dtype=torch.int32)
        self.table[:, 1::2] = 1 << 30
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        self.max_rows = max(1, *rows)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g)

    def places(self, i):
        """(pages, positions in them) of sequence i's tokens."""
        t = torch.arange(self.ctx[i])
        return self.table[i].long()[t // self.page], t % self.page

    def cache(self, q8, poison=float("nan")):
        """keys, values [pages, hkv, page, dim] and scales (or None): random where a sequence has a
        token, `poison` everywhere else."""
        shape = (self.pages, self.hkv, self.page, self.dim)
        live = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for i in range(len(self.ctx)):
            p, o = self.places(i)
            live[p, o] = True
        live = live[:, None, :]
        if q8:
            out = [torch.randint(-127, 128, shape, generator=self.g, dtype=torch.int8) for _ in range(2)]
            scales = [(torch.rand(shape[:3], generator=self.g) * 0.02 + 0.005).where(live, torch.tensor(poison))
                      for _ in range(2)]
            return out[0], out[1], scales[0], scales[1]
        out = [self.randn(*shape).where(live[..., None], torch.tensor(poison)).to(BF16) for _ in range(2)]
        return out[0], out[1], None, None


def values64(x, scales):
    return x.double() if scales is None else x.double() * scales.double()[..., None]


def attention64(b: Batch, keys, values, ks, vs, q, scale, half=HALF_BF16):
    """(out, bound) in float64 for every row of the batch, NaN for rows that no sequence owns.
    half: the probabilities' half step, HALF_16 where a sequence has few queries.
    bound: half a bf16 step of the result, half a step of every probability against what it
    multiplies, and the float sums (D products per score, relative in the probabilities; one
    sum over the tokens)."""
    hq, D = q.shape[1], b.dim
    G = hq // b.hkv
    out = torch.full((b.rows, hq, D), math.nan, dtype=torch.float64)
    bound = out.clone()
    for i, n in enumerate(b.lens):
        p, o = b.places(i)
        K = values64(keys[p, :, o], None if ks is None else ks[p, :, o])    # [tokens, hkv, D]
        V = values64(values[p, :, o], None if vs is None else vs[p, :, o])
        for r in range(n):
            row, see = int(b.off[i]) + r, b.ctx[i] - n + r + 1
            for h in range(hq):
                if see <= 0:
                    out[row, h], bound[row, h] = 0, 0
                    continue
                x = q[row, h].double()
                k, v = K[:see, h // G], V[:see, h // G]
                s = (k @ x) * scale
                w = torch.softmax(s, 0)
                out[row, h] = w @ v
                # (twice the first-order float error of a score: its own and that of the maximum)
                err = 2 * abs(scale) * (k.abs() @ x.abs()).max() * (D + 8) * 2 * HALF_F32 + 2 * s.abs().max() * HALF_F32 * 4
                size = w @ v.abs()
                bound[row, h] = HALF_BF16 * out[row, h].abs() + size * (half * 1.01 + 2 * err + (see + 64) * HALF_F32)
    return out, bound


def cancel_values(b: Batch, cache, q, scale):
    """Sets the value of every sequence's last token so that the outputs of its last row nearly vanish beside
    the terms that they are sums of (exactly, but for its own rounding, for the first query of each kv
    head; the others' probabilities are close where the scale is small): then the rounding of an output hides
    nothing of the probabilities'."""
    keys, values, ks, vs = cache
    G = q.shape[1] // b.hkv
    for i in range(len(b.lens)):
        p, o = b.places(i)
        if b.lens[i] == 0 or len(p) < 2:
            continue
        K = values64(keys[p, :, o], None if ks is None else ks[p, :, o])
        V = values64(values[p, :, o], None if vs is None else vs[p, :, o])
        for h in range(b.hkv):
            w = torch.softmax((K[:, h] @ q[int(b.off[i + 1]) - 1, h * G].double()) * scale, 0)
            v = -(w[:-1] @ V[:-1, h]) / w[-1]
            if vs is not None:
                vs[p[-1], h, o[-1]] = v.abs().max() / 127
                v = torch.round(v / vs[p[-1], h, o[-1]].double())
            values[p[-1], h, o[-1]] = v.to(values.dtype)
