"""The batched token mixers together, as a server runs them: an attention layer over a paged cache
and a delta-rule layer over pooled states for the same requests, which enter with prompts, decode,
verify drafts, drop some and leave. Every step against float64 over what the layers hold."""
import pytest
import torch

import gpu_util as G
from delta_cases import BF16, DeltaCase
from paged_cases import Batch, attention64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
def test_requests_enter_decode_verify_and_leave(gpu, q38, q8):
    hkv, hq, dim, hk, hv, dk = 2, 8, 128, 2, 4, 64
    width, page, slots = 12, 16, 12
    g = torch.Generator().manual_seed(51)
    pages = 40
    shape = (pages, hkv, page, dim)
    if q8:
        dev = [torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2)]
        dev += [torch.full(shape[:3], float("nan"), device="cuda") for _ in range(2)]
    else:
        dev = [torch.full(shape, float("nan"), dtype=BF16, device="cuda") for _ in range(2)]
    cache = q38.PagedCache(gpu, *dev)
    pool = torch.full((slots, hv, dk, dk), float("nan"), device="cuda")
    rule = q38.DeltaRule(gpu, hk, hv, dk, dk, dk ** -0.5)
    ws = G.workspace(1 << 27)
    free = torch.randperm(pages, generator=g).tolist()
    tables, have, state = {}, {}, {}  # request -> its pages, tokens, slot of its state (-1: none yet)

    def step(rows, keep=None):
        """rows: request -> its new rows; keep: request -> how many of them stay (a verification)."""
        ids = sorted(rows)
        for r in ids:
            tables.setdefault(r, [])
            have.setdefault(r, 0)
            state.setdefault(r, -1)
            while len(tables[r]) * page < have[r] + rows[r]:
                tables[r].append(free.pop())
        b = Batch([rows[r] for r in ids], [have[r] + rows[r] for r in ids], page=page, hkv=hkv, dim=dim, width=width)
        for i, r in enumerate(ids):
            b.table[i] = -1
            b.table[i, :len(tables[r])] = torch.tensor(tables[r], dtype=torch.int32)
        d = DeltaCase([rows[r] for r in ids], hk, hv, dk, dk, seed=int(torch.randint(1 << 30, (1,), generator=g)),
                      checkpoints=keep is not None)
        spare = [s for s in range(slots) if s not in state.values()]
        d.slots, d.states = slots, pool.cpu()
        d.origin = torch.tensor([state[r] for r in ids], dtype=torch.int32)
        if keep is None:
            d.last = torch.tensor([state[r] if state[r] >= 0 else spare.pop() for r in ids], dtype=torch.int32)
        else:
            d.last[:] = -1
            d.ckpt = torch.tensor([spare.pop() for _ in range(d.rows)], dtype=torch.int32)
        q, k, v = (torch.randn(b.rows, h, dim, generator=g).to(BF16) for h in (hq, hkv, hkv))
        off = b.off.cuda()
        B = q38.PagedBatch(off, b.tokens.cuda(), b.table.cuda(), b.rows, b.max_rows)
        D = q38.DeltaBatch(pool, off, d.origin.cuda(), d.last.cuda(), b.rows, b.max_rows, None if keep is None else d.ckpt.cuda())
        out = torch.zeros(b.rows, hq, dim, dtype=BF16, device="cuda")
        mixed = torch.zeros(b.rows, hv, dk, dtype=BF16, device="cuda")
        assert max(cache.workspace_size(B, hq), rule.workspace_size(D)) <= ws.numel()
        cache.append(B, k.cuda(), v.cuda(), G.stream())
        cache.attend(B, q.cuda(), out, dim ** -0.5, ws, G.stream())
        rule.run(D, *d.operands("cuda"), mixed, ws, G.stream())
        torch.cuda.synchronize()
        want, bound = attention64(b, *(t.cpu() for t in dev), *([] if q8 else [None, None]), q, dim ** -0.5)
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
        want, ob, S, sb = d.exact(32 if keep is None else 0)
        assert bool(((mixed.cpu().double() - want).abs() <= ob).all())
        for i, r in enumerate(ids):
            n = rows[r] if keep is None else keep[r]
            at, slot = int(b.off[i]) + n - 1, int(d.last[i]) if keep is None else int(d.ckpt[int(b.off[i]) + n - 1])
            assert bool(((pool[slot].cpu().double() - S[at]).norm(dim=-1) <= sb[at]).all())
            state[r] = slot
            have[r] += n

    step({0: 40, 1: 7})
    step({0: 1, 1: 1, 2: 90})          # two decode while one enters
    step({0: 1, 1: 1, 2: 1})
    step({0: 3, 1: 4, 2: 2}, keep={0: 1, 1: 4, 2: 2})
    step({0: 1, 1: 1, 2: 1})           # over the places of dropped drafts
    free += tables.pop(1)
    have.pop(1), state.pop(1)
    step({0: 1, 2: 1, 3: 33})          # a request in the pages and the state of the one that left
    step({0: 2, 2: 1, 3: 3}, keep={0: 2, 2: 1, 3: 1})
    step({0: 1, 2: 1, 3: 1})
