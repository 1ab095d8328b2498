"""Performance cases of the batched token mixers: the paged KV cache (append and attention) and
the gated delta rule over pooled states, for many requests of ragged lengths at once.

Operators (the "op" of a case):
  append  q38_paged_append: the new keys and values of a batch into a paged cache, bf16 or 8 bits
          with one scale per (token, kv head)
  attend  q38_paged_attention: causal attention of each sequence's new rows over its paged cache
  delta   q38_delta_rule: S <- exp(g) S, S <- S + beta (v - S k) k^T, o = scale S q per row

Where `own` is false, run() computes the same in elementary torch operations (32 bits, decay sums
in 64); exact() computes it in 64 bits, per sequence and, for the delta rule, row by row.

Head counts and sizes are those of the other performance cases (16 + 2 attention heads of 256,
16 / 32 delta-rule heads of 128) or common ones (32 + 8 heads of 128, 64-dim heads). Lengths of
the sequences of a batch are spread evenly over the logarithm of the case's range, in an order
of their own; they go by the case alone, values and page order by the seed.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_contexts = {}  # of the framework, one per device


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of 64 requests: the smallest call, bound by its launch
        {"name": "append_decode_b64", "op": "append", "format": "bf16", "seqs": 64, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 64, "ctx_hi": 1024, "page": 64, "hkv": 2, "dim": 256},
        # prompts of several requests entering an 8-bit cache
        {"name": "append_prompt_q8", "op": "append", "format": "q8", "seqs": 6, "rows_lo": 500, "rows_hi": 5000,
         "ctx_lo": 5000, "ctx_hi": 5000, "page": 64, "hkv": 2, "dim": 256},
        # one request decoding alone: latency, its cache split over the chip
        {"name": "attend_one_4k", "op": "attend", "format": "bf16", "seqs": 1, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 4001, "ctx_hi": 4001, "page": 64, "hq": 16, "hkv": 2, "dim": 256},
        # a decode step of 64 requests with contexts between a short chat and a document
        {"name": "attend_decode_b64", "op": "attend", "format": "bf16", "seqs": 64, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 100, "ctx_hi": 16000, "page": 64, "hq": 16, "hkv": 2, "dim": 256},
        # a few very long contexts in an 8-bit cache
        {"name": "attend_long_q8", "op": "attend", "format": "q8", "seqs": 3, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 40000, "ctx_hi": 131072, "page": 128, "hq": 16, "hkv": 2, "dim": 256},
        # speculative verification: 16 requests, a token and three drafts each
        {"name": "attend_verify_b16", "op": "attend", "format": "bf16", "seqs": 16, "rows_lo": 4, "rows_hi": 4,
         "ctx_lo": 500, "ctx_hi": 12000, "page": 16, "hq": 16, "hkv": 2, "dim": 256},
        # ragged prompts behind cached prefixes, heads of 128
        {"name": "attend_prompt", "op": "attend", "format": "bf16", "seqs": 5, "rows_lo": 300, "rows_hi": 2500,
         "ctx_lo": 2500, "ctx_hi": 6000, "page": 64, "hq": 32, "hkv": 8, "dim": 128},
        # one request decoding alone
        {"name": "delta_one", "op": "delta", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "hk": 16, "hv": 32, "dk": 128,
         "dv": 128, "checkpoints": False},
        # a decode step of 128 requests: the states' traffic
        {"name": "delta_decode_b128", "op": "delta", "seqs": 128, "rows_lo": 1, "rows_hi": 1, "hk": 16, "hv": 32,
         "dk": 128, "dv": 128, "checkpoints": False},
        # speculative verification: the state after every row is kept
        {"name": "delta_verify_b16", "op": "delta", "seqs": 16, "rows_lo": 4, "rows_hi": 4, "hk": 16, "hv": 32,
         "dk": 128, "dv": 128, "checkpoints": True},
        # one prompt: a single chain of chunks per head
        {"name": "delta_prompt_4k", "op": "delta", "seqs": 1, "rows_lo": 4001, "rows_hi": 4001, "hk": 16, "hv": 32,
         "dk": 128, "dv": 128, "checkpoints": False},
        # ragged prompts of several requests
        {"name": "delta_prompt_b8", "op": "delta", "seqs": 8, "rows_lo": 600, "rows_hi": 4500, "hk": 16, "hv": 32,
         "dk": 128, "dv": 128, "checkpoints": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "delta", "delta"))
    if op == "delta":
        dk, dv = rng.choice(((128, 128), (128, 128), (64, 64), (256, 256), (128, 64)))
        hk = rng.choice((4, 8, 16))
        c = {"op": op, "hk": hk, "hv": hk * rng.choice((1, 2, 4) if hk < 16 else (1, 2)), "dk": dk, "dv": dv,
             "checkpoints": False}
        kind = rng.choice(("decode", "verify", "prompt"))
        if kind == "prompt":
            seqs = _log(rng, 1, 12)
            hi = min(_log(rng, 20, 4500), int(8e9 // (c["hv"] * dk * dv)))
            seqs = max(1, min(seqs, int(8e9 // (hi * c["hv"] * dk * dv))))
            c.update(seqs=seqs, rows_lo=max(1, hi // rng.choice((1, 3, 8))), rows_hi=hi)
        elif kind == "verify":
            c.update(seqs=_log(rng, 1, 32), rows_lo=1, rows_hi=rng.randint(2, 9), checkpoints=True)
        else:
            c.update(seqs=_log(rng, 1, 160), rows_lo=1, rows_hi=1)
        state = c["hv"] * dk * dv * 4  # the pool holds an origin and a result (or one per row) for each
        c["seqs"] = max(1, min(c["seqs"], int(6e8 // (state * (1 + (c["rows_hi"] if c["checkpoints"] else 1))))))
        return c
    fmt, page = rng.choice(("bf16", "q8")), rng.choice((16, 32, 64, 128, 256))
    hkv, group, dim = rng.choice(((2, 8, 256), (2, 8, 256), (8, 4, 128), (4, 7, 128), (1, 16, 64), (4, 1, 256)))
    c = {"op": op, "format": fmt, "page": page, "hkv": hkv, "dim": dim}
    if op == "append":
        seqs, hi = _log(rng, 1, 128), _log(rng, 1, 4000)
        hi = min(hi, max(1, 16000 // seqs))
        c.update(seqs=seqs, rows_lo=max(1, hi // 4), rows_hi=hi, ctx_lo=hi, ctx_hi=hi + _log(rng, 1, 800))
        return c
    kind = rng.choice(("decode", "decode", "verify", "prompt"))
    c["hq"] = hkv * group
    if kind == "decode":
        rows = (1, 1)
    elif kind == "verify":
        rows = (1, rng.randint(2, 16))
    else:
        hi = _log(rng, 17, 2000)
        rows = (max(1, hi // 5), hi)
    ctx = _log(rng, rows[1], 60000 if kind != "prompt" else 6000)
    # bounded by the cache and by the scores of the largest listed cases
    seqs = _log(rng, 1, 128 if kind != "prompt" else 6)
    seqs = max(1, min(seqs, int(1.3e8 // (ctx * hkv * dim)), int(8e10 // (ctx * rows[1] * hkv * group * dim))))
    c.update(seqs=seqs, rows_lo=rows[0], rows_hi=rows[1], ctx_lo=max(rows[1], ctx // rng.choice((1, 4, 50))), ctx_hi=ctx)
    return c


# ------------------------------------------------------------------ lengths
def _spread(lo, hi, n, salt):
    """n lengths from lo to hi, even over the logarithm, in an order of their own."""
    v = [hi] if n == 1 else [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    random.Random(salt).shuffle(v)
    return v


def _lengths(case):
    """(rows, tokens after the call) of each sequence."""
    rows = _spread(case["rows_lo"], case["rows_hi"], case["seqs"], 1)
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"], 2) if "ctx_hi" in case else rows
    return rows, [max(r, c) for r, c in zip(rows, ctx)]


def _visible(rows, ctx):
    """Pairs of a row and a token that it sees, over all sequences."""
    return sum(r * (c - r) + r * (r + 1) // 2 for r, c in zip(rows, ctx))


def work(case):
    rows, ctx = _lengths(case)
    R = sum(rows)
    if case["op"] == "delta":
        hk, hv, dk, dv = (case[k] for k in ("hk", "hv", "dk", "dv"))
        states = case["seqs"] + (R if case["checkpoints"] else case["seqs"])
        b = R * (2 * hk * dk * 2 + 2 * hv * dv * 2 + 2 * hv * 4) + states * hv * dv * dk * 4
        return {"bytes": b, "flops": 7 * R * hv * dk * dv}
    el, sc = (2, 0) if case["format"] == "bf16" else (1, 4)
    token = 2 * case["hkv"] * (case["dim"] * el + sc)  # a token's keys and values in the cache
    if case["op"] == "append":
        return {"bytes": R * (2 * case["hkv"] * case["dim"] * 2 + token), "flops": 0}
    return {"bytes": sum(ctx) * token + 2 * R * case["hq"] * case["dim"] * 2,
            "flops": 4 * case["hq"] * case["dim"] * _visible(rows, ctx)}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rows, ctx = _lengths(case)
    n, R = case["seqs"], sum(rows)
    off = [0]
    for r in rows:
        off.append(off[-1] + r)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    s = {"case": dict(case), "rows": R, "max_rows": max(rows), "off": ints(off)}
    if case["op"] == "delta":
        hk, hv, dk, dv = (case[k] for k in ("hk", "hv", "dk", "dv"))
        silu = torch.nn.functional.silu
        # the convolved and activated projections, side by side as the convolution leaves them;
        # q and k normalised per head
        qkv = silu(randn(R, 2 * hk * dk + hv * dv))
        qk = qkv[:, : 2 * hk * dk].view(R, 2 * hk, dk)
        qk /= qk.norm(dim=-1, keepdim=True)
        qkv = qkv.to(torch.bfloat16)
        s["q"] = qkv[:, : hk * dk].view(R, hk, dk)
        s["k"] = qkv[:, hk * dk: 2 * hk * dk].view(R, hk, dk)
        s["v"] = qkv[:, 2 * hk * dk:].view(R, hv, dv)
        rate = torch.rand(hv, generator=g, device=dev) * 15 + 1
        s["g"] = -rate * torch.nn.functional.softplus(randn(R, hv) - 4.0)
        s["beta"] = torch.sigmoid(randn(R, hv))
        s["scale"] = dk ** -0.5
        # slots: the origins, then the results (a verification keeps both until it commits)
        states = n + (R if case["checkpoints"] else n)
        order = torch.randperm(states, generator=g, device=dev).to(torch.int32)
        s["states"] = torch.zeros(states, hv, dv, dk, device=dev)
        s["origin"] = order[:n].contiguous()
        s["states"][s["origin"].long()] = randn(n, hv, dv, dk) * 0.1
        s["out"] = torch.zeros(R, hv, dv, dtype=torch.bfloat16, device=dev)
        if case["checkpoints"]:  # the last row's checkpoint is the sequence's result
            s["checkpoints"], s["final"] = order[n:].contiguous(), torch.full((n,), -1, dtype=torch.int32, device=dev)
            s["written"] = s["checkpoints"].long()
        else:
            s["checkpoints"], s["final"] = None, order[n:].contiguous()
            s["written"] = s["final"].long()
        return s
    hkv, D, P = case["hkv"], case["dim"], case["page"]
    used = [-(-c // P) for c in ctx]
    width, pages = max(used), sum(used) + 1
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32, device=dev)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at: at + u]
        at += u
    s.update(tokens=ints(ctx), table=table, page=P, scale=D ** -0.5)
    shape = (pages, hkv, P, D)
    for name in ("keys", "values"):
        if case["format"] == "bf16":
            s[name], s[name + "_scale"] = randn(*shape).to(torch.bfloat16), None
        else:
            s[name] = torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)
            s[name + "_scale"] = torch.rand(pages, hkv, P, generator=g, device=dev) * 0.01 + 0.015
    if case["op"] == "append":  # the rows' slices of the projections' output
        kv = randn(R, 2 * hkv * D).to(torch.bfloat16)
        s["k"], s["v"] = kv[:, : hkv * D].view(R, hkv, D), kv[:, hkv * D:].view(R, hkv, D)
        return s
    # normalised and rotated queries; a few tokens carry most of a softmax in trained layers
    s["q"] = (randn(R, case["hq"], D) * 2.0).to(torch.bfloat16)
    s["out"] = torch.zeros(R, case["hq"], D, dtype=torch.bfloat16, device=dev)
    return s


# ------------------------------------------------------------------ the framework's calls
def _framework(device):
    path = os.path.join(os.getcwd(), "qwen38-flash.cpp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q38
    if device.index not in _contexts:
        _contexts[device.index] = q38.Ctx(device.index)
    return q38, _contexts[device.index]


def _workspace(s, nbytes):
    """A prepared state's own: passes of other states may overlap, and a graph of this one keeps its address."""
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=s["off"].device)


def _own(s):
    st = torch.cuda.current_stream(s["off"].device).cuda_stream
    op = s["case"]["op"]
    if "call" not in s:  # the handles and descriptions that a program keeps beside its buffers
        q38, ctx = _framework(s["off"].device)
        if op == "delta":
            rule = q38.DeltaRule(ctx, s["case"]["hk"], s["case"]["hv"], s["case"]["dk"], s["case"]["dv"], s["scale"])
            batch = q38.DeltaBatch(s["states"], s["off"], s["origin"], s["final"], s["rows"], s["max_rows"],
                                   s["checkpoints"])
            s["call"] = rule, batch, _workspace(s, rule.workspace_size(batch))
        else:
            cache = q38.PagedCache(ctx, s["keys"], s["values"], s["keys_scale"], s["values_scale"])
            batch = q38.PagedBatch(s["off"], s["tokens"], s["table"], s["rows"], s["max_rows"])
            ws = _workspace(s, cache.workspace_size(batch, s["case"]["hq"])) if op == "attend" else None
            s["call"] = cache, batch, ws
    handle, batch, ws = s["call"]
    if op == "delta":
        handle.run(batch, s["q"], s["k"], s["v"], s["g"], s["beta"], s["out"], ws, st)
    elif op == "append":
        handle.append(batch, s["k"], s["v"], st)
    else:
        handle.attend(batch, s["q"], s["out"], s["scale"], ws, st)


# ------------------------------------------------------------------ the plain forms
def _row_places(s):
    """Of every row of the batch: its sequence, and its number within it."""
    r = torch.arange(s["rows"], device=s["off"].device, dtype=torch.int32)
    seq = torch.searchsorted(s["off"], r, right=True) - 1
    return seq, (r - s["off"][seq]).long()


def _plain_append(s):
    seq, r = _row_places(s)
    n = (s["off"][1:] - s["off"][:-1])[seq]
    t = s["tokens"][seq].long() - n + r
    page = s["table"][seq, t // s["page"]].long()
    for name, x in (("keys", s["k"]), ("values", s["v"])):
        if s[name + "_scale"] is None:
            s[name][page, :, t % s["page"]] = x
        else:
            x = x.float()
            top = x.abs().amax(-1, keepdim=True)
            code = torch.where(top > 0, torch.round(x * 127 / top), 0)
            s[name][page, :, t % s["page"]] = code.to(torch.int8)
            s[name + "_scale"][page, :, t % s["page"]] = (top / 127).squeeze(-1)


def _plain_attend(s):
    c = s["case"]
    hkv, D, G = c["hkv"], c["dim"], c["hq"] // c["hkv"]
    seq, r = _row_places(s)
    n, width, most = c["seqs"], s["table"].shape[1] * s["page"], s["max_rows"]
    q = torch.zeros(n, most, hkv, G, D, device=s["q"].device)
    q[seq, r] = s["q"].view(-1, hkv, G, D).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(n * hkv, most * G, D).contiguous()
    table = s["table"].long()

    def cached(name):
        x = s[name][table].float()
        if s[name + "_scale"] is not None:
            x *= s[name + "_scale"][table].unsqueeze(-1)
        return x.permute(0, 2, 1, 3, 4).reshape(n * hkv, width, D)

    score = torch.bmm(q, cached("keys").transpose(1, 2).contiguous()) * s["scale"]
    rows = s["off"][1:] - s["off"][:-1]
    last = (s["tokens"] - rows)[:, None] + torch.arange(most, device=rows.device)  # [n, most]
    t = torch.arange(width, device=rows.device)
    score = score.view(n, hkv, most, G, width)
    score.masked_fill_((t > last[..., None])[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp_(score.sub_(torch.where(top > -math.inf, top, 0)))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(n * hkv, most * G, width), cached("values")).view(n, hkv, most, G, D)
    o = torch.where(total > 0, o / total, 0)
    s["out"].copy_(o.permute(0, 2, 1, 3, 4)[seq, r].reshape(s["out"].shape))


def _plain_delta(s):
    c = s["case"]
    n, most, hv, dk, dv = c["seqs"], s["max_rows"], c["hv"], c["dk"], c["dv"]
    seq, r = _row_places(s)

    def padded(x):  # [rows, heads, ...] -> [n, hv, most, ...] in 32 bits, zeros behind a sequence's rows
        y = torch.zeros(n, most, *x.shape[1:], device=x.device)
        y[seq, r] = x.float()
        y = y.transpose(1, 2)
        return y if x.shape[1] == hv else y.repeat_interleave(hv // x.shape[1], dim=1)

    q, k, v, g, beta = (padded(s[x]) for x in ("q", "k", "v", "g", "beta"))
    S = s["states"][s["origin"].long()]
    out = torch.zeros(n, hv, most, dv, device=S.device)
    if most <= 16:  # row by row
        kept = []
        for t in range(most):
            S = S * torch.exp(g[:, :, t])[..., None, None]
            u = beta[:, :, t, None] * (v[:, :, t] - (S * k[:, :, t, None]).sum(-1))
            S = S + u[..., None] * k[:, :, t, None]
            out[:, :, t] = (S * q[:, :, t, None]).sum(-1)
            kept.append(S)
        if s["checkpoints"] is not None:
            s["states"][s["checkpoints"].long()] = torch.stack(kept)[r, seq]
    else:  # chunk by chunk: within a chunk the rows' updates solve a unit lower triangular system
        C = 64
        pad = -most % C
        q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)).view(n, hv, -1, C, x.shape[-1]) for x in (q, k, v))
        g, beta = (torch.nn.functional.pad(x, (0, pad)).view(n, hv, -1, C) for x in (g, beta))
        G = g.double().cumsum(-1)
        low = torch.ones(C, C, dtype=torch.bool, device=S.device).tril()
        decay = torch.where(low, torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, 0)), 0).float()
        A = beta[..., None] * torch.matmul(k, k.transpose(-1, -2).contiguous()) * decay
        T = torch.zeros_like(A)
        for i in range(C):  # row i of (I + A)^-1
            T[..., i, :] = -torch.matmul(A[..., i: i + 1, :i], T[..., :i, :]).squeeze(-2) if i else 0
            T[..., i, i] += 1
        M = torch.matmul(q, k.transpose(-1, -2).contiguous()) * decay
        into, left = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
        outs = []
        for j in range(q.shape[2]):
            St = S.transpose(-1, -2).contiguous()
            U = torch.matmul(T[:, :, j], beta[:, :, j, :, None] * (v[:, :, j] - into[:, :, j] * torch.matmul(k[:, :, j], St)))
            outs.append(into[:, :, j] * torch.matmul(q[:, :, j], St) + torch.matmul(M[:, :, j], U))
            S = into[:, :, j, -1:] * S + torch.matmul((left[:, :, j] * U).transpose(-1, -2).contiguous(), k[:, :, j])
        out = torch.cat(outs, 2)
    s["out"].copy_(out.transpose(1, 2)[seq, r] * s["scale"])
    if s["checkpoints"] is None:
        s["states"][s["final"].long()] = S


def run(state):
    op = state["case"]["op"]
    if own:
        _own(state)
    else:
        {"append": _plain_append, "attend": _plain_attend, "delta": _plain_delta}[op](state)
    if op == "delta":
        return {"out": state["out"], "states": state["states"][state["written"]]}
    if op == "attend":
        return {"out": state["out"]}
    if state["case"]["format"] == "bf16":
        return {"keys": state["keys"], "values": state["values"]}
    return {"keys": state["keys"] * state["keys_scale"][..., None],
            "values": state["values"] * state["values_scale"][..., None]}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    rows, ctx = _lengths(case)
    off = s["off"].tolist()
    if case["op"] == "delta":
        rep = case["hv"] // case["hk"]
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        S = s["states"][s["origin"].long()].double()
        kept = [None] * (s["rows"] if case["checkpoints"] else 0)
        order = sorted(range(len(rows)), key=lambda i: -rows[i])
        back = sorted(range(len(rows)), key=lambda i: order[i])
        S = S[torch.tensor(order, device="cuda")]
        first = torch.tensor([off[i] for i in order], device="cuda")
        for t in range(max(rows)):  # the sequences that still have a row t come first
            live = sum(rows[i] > t for i in order)
            at = first[:live] + t
            k, q = (s[x][at].double().repeat_interleave(rep, 1)[..., None] for x in ("k", "q"))
            H = S[:live] * torch.exp(s["g"][at].double())[..., None, None]
            miss = s["v"][at].double()[..., None] - H @ k
            H = H + (s["beta"][at].double()[..., None, None] * miss) @ k.transpose(-1, -2)
            S[:live] = H
            out[at] = (H @ q)[..., 0] * s["scale"]
            if kept:
                for j, i in enumerate(order[:live]):
                    kept[off[i] + t] = H[j].clone()
        return {"out": out, "states": torch.stack(kept) if kept else S[torch.tensor(back, device="cuda")]}
    P, D, hkv = case["page"], case["dim"], case["hkv"]
    if case["op"] == "append":
        result = {}
        for name, x in (("keys", s["k"]), ("values", s["v"])):
            now = s[name].double()
            if case["format"] == "q8":
                now *= s[name + "_scale"].double()[..., None]
                x = x.double()
                top = x.abs().amax(-1, keepdim=True)
                x = torch.round(x * 127 / top).nan_to_num(0) * (top / 127)
            for i, (r, c) in enumerate(zip(rows, ctx)):
                t = torch.arange(c - r, c, device="cuda")
                now[s["table"][i].long()[t // P], :, t % P] = x[off[i]: off[i + 1]].double()
            result[name] = now
        return result
    if _visible(rows, ctx) * case["hq"] * D > 4e12:
        return None
    G = case["hq"] // hkv
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for i, (r, c) in enumerate(zip(rows, ctx)):
        pages = s["table"][i, : -(-c // P)].long()
        see = torch.arange(c, device="cuda")[None] <= torch.arange(c - r, c, device="cuda")[:, None]
        for h in range(hkv):
            K, V = (s[x][pages, h].double() if s[x + "_scale"] is None else
                    s[x][pages, h].double() * s[x + "_scale"][pages, h].double()[..., None] for x in ("keys", "values"))
            K, V = K.reshape(-1, D)[:c], V.reshape(-1, D)[:c]
            for j in range(G):
                w = (s["q"][off[i]: off[i + 1], h * G + j].double() @ K.T) * s["scale"]
                w = torch.softmax(w.masked_fill(~see, -math.inf), -1)
                out[off[i]: off[i + 1], h * G + j] = w @ V
    return {"out": out}
