"""Ragged batches of the gated delta rule and their float64 recurrence, for the tests of
q38_delta_rule (CPU tensors)."""
from __future__ import annotations

import math

import torch

BF16 = torch.bfloat16
HALF_BF16 = torch.finfo(BF16).eps / 2
HALF_F32 = torch.finfo(torch.float32).eps / 2


class DeltaCase:
    def __init__(self, rows, hk=2, hv=4, dk=64, dv=64, seed=0, gap=0, spare=2, checkpoints=False, decay=0.05,
                 origin="random", unit=True):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens = g, list(rows)
        self.hk, self.hv, self.dk, self.dv = hk, hv, dk, dv
        off = [gap]
        for r in rows:
            off.append(off[-1] + r)
        n, R = len(rows), off[-1] + gap
        self.rows, self.off = R, torch.tensor(off, dtype=torch.int32)
        self.max_rows = max(1, *rows)
        # projections beside each other, as a convolution leaves them
        x = torch.nn.functional.silu(torch.randn(R, 2 * hk * dk + hv * dv, generator=g))
        qk = x[:, :2 * hk * dk].view(R, 2 * hk, dk)
        if unit:
            qk /= qk.norm(dim=-1, keepdim=True)
        self.qkv = x.to(BF16)
        self.g_log = -decay * torch.exp(torch.randn(R, hv, generator=g))
        self.beta = torch.sigmoid(torch.randn(R, hv, generator=g))
        self.scale = dk ** -0.5
        kept = R if checkpoints else 0
        self.slots = 2 * n + kept + spare
        order = torch.randperm(self.slots, generator=g).to(torch.int32)
        self.states = torch.full((self.slots, hv, dv, dk), math.nan)
        self.origin = order[:n].clone()
        self.states[self.origin.long()] = torch.randn(n, hv, dv, dk, generator=g) * 0.2
        if origin == "zero":
            self.origin[:] = -1
        self.last = order[n:2 * n].clone()
        self.ckpt = order[2 * n:2 * n + kept].clone() if checkpoints else None

    def operands(self, device):
        """q, k, v as slices of one tensor, then log decay and beta."""
        x = self.qkv.to(device)
        kw = self.hk * self.dk
        return (x[:, :kw].view(-1, self.hk, self.dk), x[:, kw:2 * kw].view(-1, self.hk, self.dk),
                x[:, 2 * kw:].view(-1, self.hv, self.dv), self.g_log.to(device), self.beta.to(device))

    def exact(self, chunk=0):
        """(out, out bound, states after every row, their bound) in float64 by row, NaN where no
        sequence owns a row; states and bounds per row [rows, hv, dv, dk] / [rows, hv, dv].

        State bound, per value row in the 2-norm: a step makes an error of at most
        (DK + 8) 2^-24 (|S| + |v|) (its dot product of DK terms, three roundings per element,
        beta |k| <= 1) and the rule contracts what was there by exp(g). In the chunked form
        (chunk > 0) a row's update comes from a triangular system of the chunk instead: the
        backward error of the substitution, `chunk` half steps, reaches the updates through
        |T| |A|, which `system` measures, and its dot products are DK and `chunk` terms long.
        Output bound: half a bf16 step, the state's error and a dot product against q; in the
        chunked form also half a bf16 step of every term (state, scores, updates: three)."""
        q, k, v, g, beta = (t.double() for t in self.operands("cpu"))
        rep = self.hv // self.hk
        q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
        R, hv, dv, dk = self.rows, self.hv, self.dv, self.dk
        out = torch.full((R, hv, dv), math.nan, dtype=torch.float64)
        ob, S_all = out.clone(), torch.full((R, hv, dv, dk), math.nan, dtype=torch.float64)
        sb = out.clone()
        for i, n in enumerate(self.lens):
            S = self.states[int(self.origin[i])].double() if self.origin[i] >= 0 else torch.zeros(hv, dv, dk).double()
            E = S.norm(dim=-1) * HALF_F32
            size = torch.zeros(hv, dv).double()
            for t in range(n):
                r = int(self.off[i]) + t
                if chunk and t % chunk == 0:
                    c = slice(r, r + min(chunk, n - t))
                    steps = dk + 8 + 2 * chunk + chunk * self.system(k[c], g[c], beta[c])[:, None]
                    size, base = torch.zeros(hv, dv).double(), S.norm(dim=-1)
                elif not chunk:
                    steps = dk + 8
                d = torch.exp(g[r])[:, None]
                S = S * d[..., None]
                u = beta[r][:, None] * (v[r] - (S @ k[r][..., None])[..., 0])
                S = S + u[..., None] * k[r][:, None, :]
                E = E * d + steps * 2 * HALF_F32 * (S.norm(dim=-1) + v[r].abs() + (base if chunk else 0))
                qn = q[r].norm(dim=-1)[:, None]
                out[r] = (S @ q[r][..., None])[..., 0] * self.scale
                ob[r] = HALF_BF16 * out[r].abs() + self.scale * qn * (E + (dk + 8) * 2 * HALF_F32 * S.norm(dim=-1))
                if chunk:
                    base = base * d
                    size = size * d + u.abs() * k[r].norm(dim=-1)[:, None]
                    ob[r] += 3 * HALF_BF16 * self.scale * qn * (base + size)
                S_all[r], sb[r] = S, E
        return out, ob, S_all, sb

    @staticmethod
    def system(k, g, beta):
        """Per head, the norm of |T| |A| of a chunk's triangular system (I + A) u = x, T its inverse."""
        G = g.clamp_min(-1e4).cumsum(0).T
        kk = torch.einsum("ihd,jhd->hij", k, k)
        A = (beta.T[..., None] * kk * torch.exp((G[:, :, None] - G[:, None, :]).clamp_max(0))).tril(-1)
        T = torch.linalg.inv(torch.eye(A.shape[-1], dtype=A.dtype) + A)
        return torch.linalg.matrix_norm(T.abs() @ A.abs(), 2)


def final_states(c, dt):
    """The states after the last rows by the recurrence in one type, on the CPU: [sequences, hv, dv, dk]."""
    q, k, v, g, beta = (t.to(dt) for t in c.operands("cpu"))
    k = k.repeat_interleave(c.hv // c.hk, 1)
    out = []
    for i, n in enumerate(c.lens):
        S = c.states[int(c.origin[i])].to(dt)
        for r in range(int(c.off[i]), int(c.off[i]) + n):
            S = S * torch.exp(g[r])[:, None, None]
            u = beta[r][:, None] * (v[r] - (S * k[r][:, None, :]).sum(-1))
            S = S + u[..., None] * k[r][:, None, :]
        out.append(S)
    return torch.stack(out)


def concentrate_keys(c):
    """Keys with all their weight on one of four dims: a row's error in them meets no other that cancels it."""
    at = torch.randint(0, 4, (c.rows, c.hk), generator=c.g)
    c.qkv[:, c.hk * c.dk:2 * c.hk * c.dk] = torch.nn.functional.one_hot(at, c.dk).view(c.rows, -1).to(BF16)


def state_error(states, exact):
    """[sequences, hv]: the error relative in a head's norm."""
    return (states.double() - exact).flatten(2).norm(dim=-1) / exact.flatten(2).norm(dim=-1)


def state_limit(c, exact):
    """The error that the chunked form may make in a head's norm. It rounds an element of the state
    once per chunk and product of operand parts (24 bits) where the recurrence in float rounds it
    twice per row: twice the recurrence's error covers it, with two float steps where the recurrence
    happens to be exact (keys of one dim make exact products)."""
    return 2 * state_error(final_states(c, torch.float32), exact) + 2 * 2 * HALF_F32


def output_error(out, want):
    """[hv]: the norm of a head's error over all rows."""
    return (out.double() - want).transpose(0, 1).flatten(1).norm(dim=-1)


def output_limit(want):
    """The norm of the error that rounding the exact outputs makes, and 5% for what is off before it:
    16-bit operands, 2^-9 of a rounding, turn a few roundings the other way."""
    return 1.05 * output_error(want.to(BF16), want)
