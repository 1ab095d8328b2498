"""The gated delta rule on the GPU (q38_delta_rule) against its float64 recurrence, bounds from
delta_cases.DeltaCase.exact. Slots that a call does not read hold NaN."""
import math

import pytest
import torch

import gpu_util as G
from delta_cases import (BF16, DeltaCase, concentrate_keys, final_states, output_error, output_limit, state_error,
                         state_limit)

pytestmark = pytest.mark.gpu

CHUNK = 32  # rows of a chunk of the long form


def run(q38, gpu, c, states=None, ws=None, out=None, max_rows=None):
    states = c.states.cuda() if states is None else states
    rule = q38.DeltaRule(gpu, c.hk, c.hv, c.dk, c.dv, c.scale)
    batch = q38.DeltaBatch(states, c.off.cuda(), c.origin.cuda(), c.last.cuda(), c.rows, max_rows or c.max_rows,
                           None if c.ckpt is None else c.ckpt.cuda())
    if ws is None:  # dirty
        ws = torch.full((max(16, rule.workspace_size(batch)),), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full((c.rows, c.hv, c.dv), 7.0, dtype=BF16, device="cuda") if out is None else out
    rule.run(batch, *c.operands("cuda"), out, ws, G.stream())
    torch.cuda.synchronize()
    return out.cpu(), states.cpu()


def check(c, out, states):
    # (either form may run: the bounds are the larger ones of the chunked form for long sequences)
    want, ob, S, sb = c.exact(CHUNK if c.max_rows > 8 and c.ckpt is None else 0)
    lo, hi = int(c.off[0]), int(c.off[-1])
    owned = torch.zeros(c.rows, dtype=torch.bool)
    owned[lo:hi] = True
    assert (out[~owned] == 7.0).all(), "rows of nobody were written"
    err = (out.double() - want)[owned].abs()
    assert bool((err <= ob[owned]).all()), float((err / ob[owned]).max())
    touched = torch.zeros(c.slots, dtype=torch.bool)
    for i, n in enumerate(c.lens):
        got = states[int(c.last[i])].double()
        touched[int(c.last[i])] = True
        if n == 0:
            o = int(c.origin[i])
            assert torch.equal(got.float(), c.states[o] if o >= 0 else torch.zeros_like(c.states[0]))
            continue
        r = int(c.off[i + 1]) - 1
        off = (got - S[r]).norm(dim=-1)
        assert bool((off <= sb[r]).all()), float((off / sb[r]).max())
    if c.ckpt is not None:
        for r in range(lo, hi):
            off = (states[int(c.ckpt[r])].double() - S[r]).norm(dim=-1)
            touched[int(c.ckpt[r])] = True
            assert bool((off <= sb[r]).all()), (r, float((off / sb[r]).max()))
    assert torch.equal(states[~touched].nan_to_num(123.0), c.states[~touched].nan_to_num(123.0))


HEADS = {"family": (2, 4, 128, 128), "small": (1, 1, 64, 64), "wide": (2, 2, 256, 256), "uneven": (1, 3, 128, 64),
         "tall": (2, 2, 64, 256), "many": (4, 16, 64, 128)}
LENGTHS = {"one": [1], "decode": [1] * 9, "verify": [4, 1, 3, 7], "empty": [0, 2, 0, 0, 5, 0],
           "prompt_33": [33], "prompt": [70, 1, 0, 129, 32, 64], "prompt_long": [515, 40], "edge": [31, 32, 33, 63, 64, 65]}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("heads", list(HEADS))
def test_delta(gpu, q38, heads, lengths):
    hk, hv, dk, dv = HEADS[heads]
    c = DeltaCase(LENGTHS[lengths], hk, hv, dk, dv, seed=len(heads) * 7 + len(lengths), gap=2)
    check(c, *run(q38, gpu, c))


@pytest.mark.parametrize("lengths", ["one", "verify", "empty", "prompt_33"])
def test_checkpoints(gpu, q38, lengths):
    c = DeltaCase(LENGTHS[lengths], 2, 4, 128, 128, seed=3, checkpoints=True)
    check(c, *run(q38, gpu, c))


@pytest.mark.parametrize("rows", [[3, 1], [90, 40, 33]])
def test_zero_origin_and_no_results(gpu, q38, rows):
    c = DeltaCase(rows, 2, 2, 64, 64, seed=4, origin="zero")
    out, states = run(q38, gpu, c)
    check(c, out, states)
    rule = q38.DeltaRule(gpu, 2, 2, 64, 64, c.scale)
    for pool in (None, torch.full((1, 2, 64, 64), math.nan, device="cuda")):  # null arrays: no slot is read or written
        batch = q38.DeltaBatch(pool, c.off.cuda(), None, None, c.rows, c.max_rows)
        o2 = torch.zeros(c.rows, 2, 64, dtype=BF16, device="cuda")
        rule.run(batch, *c.operands("cuda"), o2, G.workspace(max(16, rule.workspace_size(batch))), G.stream())
        torch.cuda.synchronize()
        assert torch.equal(o2.cpu(), out)


@pytest.mark.parametrize("rows", [[2, 5], [70, 140]])
@pytest.mark.parametrize("decay", [0.0, 1.0, 40.0, math.inf])
def test_decays(gpu, q38, rows, decay):
    """No decay, strong decay (sums of a chunk far below the smallest exponent) and rows that clear
    the state (log decay -inf)."""
    c = DeltaCase(rows, 1, 2, 64, 64, seed=5, decay=0.05 if decay == math.inf else decay)
    if decay == math.inf:
        c.g_log[3::7] = -math.inf
    if decay == 40.0:  # one strong row among weak ones: the weak ones' differences must survive its size
        c.g_log[torch.arange(c.rows) % 9 != 4] *= 1e-3
    check(c, *run(q38, gpu, c))


def test_in_place_and_shared_origins(gpu, q38):
    c = DeltaCase([3, 40, 2], 2, 4, 64, 64, seed=6)
    want_out, want = run(q38, gpu, c)
    d = DeltaCase([3, 40, 2], 2, 4, 64, 64, seed=6)
    d.last = d.origin.clone()
    out, states = run(q38, gpu, d)
    assert torch.equal(out, want_out)
    assert torch.equal(states[d.origin.long()], want[c.last.long()])
    e = DeltaCase([3, 40, 2], 2, 4, 64, 64, seed=6)
    e.origin[:] = e.origin[0]
    check(e, *run(q38, gpu, e))


@pytest.mark.parametrize("rows", [[2, 1, 3], [50, 40, 90]])
def test_bad_slots(gpu, q38, rows):
    c = DeltaCase(rows, 1, 2, 64, 64, seed=7)
    clean_out, clean = run(q38, gpu, c)
    c.origin[1] = c.slots
    last = c.last.clone()
    c.last[2] = c.slots + 5
    out, states = run(q38, gpu, c)
    a, b = int(c.off[1]), int(c.off[2])
    assert torch.isnan(out[a:b].float()).all() and torch.isnan(states[int(last[1])]).all()
    assert torch.equal(out[:a], clean_out[:a]) and torch.equal(out[b:], clean_out[b:])
    assert torch.equal(states[int(last[0])], clean[int(last[0])])
    assert torch.isnan(states[int(last[2])]).all()  # as it was


@pytest.mark.parametrize("hint", [1, 3, 200, 10 ** 9])
def test_max_rows_is_a_hint(gpu, q38, hint):
    c = DeltaCase([200, 1, 3, 50], 2, 4, 128, 128, seed=8)
    check(c, *run(q38, gpu, c, max_rows=min(hint, c.rows)))


def test_offsets_outside_the_rows_are_clamped(gpu, q38):
    c = DeltaCase([40, 50], 1, 2, 64, 64, seed=9)
    want = run(q38, gpu, c)
    c.off[2] = 10 ** 6
    got = run(q38, gpu, c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][c.last.long()], want[1][c.last.long()])


def test_prompt_in_pieces_then_tokens(gpu, q38):
    """A prompt in two calls, then single tokens, then a verification of four rows committed at its
    second: the same as the rows in one float64 recurrence."""
    n = 150
    c = DeltaCase([n], 2, 4, 128, 128, seed=10, origin="zero", spare=8)
    want, ob, S, sb = c.exact(CHUNK)
    pool = c.states.cuda()
    at, origin = 0, -1
    for size in (97, 45, 1, 1, 1, 1, 4):
        d = DeltaCase([size], 2, 4, 128, 128, checkpoints=size == 4)
        d.qkv, d.g_log, d.beta = c.qkv[at:at + size], c.g_log[at:at + size], c.beta[at:at + size]
        d.origin, d.last = torch.tensor([origin], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)
        if size == 4:
            d.ckpt = torch.arange(1, 5, dtype=torch.int32)
            d.last[:] = -1
        out, states = run(q38, gpu, d, states=pool)
        assert bool(((out.double() - want[at:at + size]).abs() <= 2 * ob[at:at + size]).all())
        at, origin = at + size, 0
    assert at == n
    for r in range(4):
        off = (states[1 + r].double() - S[n - 4 + r]).norm(dim=-1)
        assert bool((off <= 2 * sb[n - 4 + r]).all())


def test_captured_and_on_streams(gpu, q38):
    """Graphs of the long and the short form over one pool, replayed with new values, against eager
    calls on another stream with another workspace."""
    for rows in ([1, 1, 1], [64, 33, 100]):
        c = DeltaCase(rows, 2, 4, 128, 128, seed=11)
        rule = q38.DeltaRule(gpu, 2, 4, 128, 128, c.scale)
        pool = c.states.cuda()
        batch = q38.DeltaBatch(pool, c.off.cuda(), c.origin.cuda(), c.last.cuda(), c.rows, c.max_rows)
        q, k, v, g, beta = c.operands("cuda")
        qkv = q._base if q._base is not None else q
        out = torch.zeros(c.rows, 4, 128, dtype=BF16, device="cuda")
        ws = G.workspace(max(16, rule.workspace_size(batch)))
        rule.run(batch, q, k, v, g, beta, out, ws, G.stream())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rule.run(batch, q, k, v, g, beta, out, ws, torch.cuda.current_stream().cuda_stream)
        side = torch.cuda.Stream()
        for i in range(3):
            d = DeltaCase(rows, 2, 4, 128, 128, seed=20 + i)
            qkv.copy_(d.qkv)
            g.copy_(d.g_log)
            beta.copy_(d.beta)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got, st = out.clone(), pool[c.last.long().cuda()].clone()
            with torch.cuda.stream(side):
                o2, w2 = torch.zeros_like(out), torch.zeros_like(ws)
                rule.run(batch, q, k, v, g, beta, o2, w2, side.cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(got, o2) and torch.equal(st, pool[c.last.long().cuda()])


def test_rows_of_a_batch_do_not_depend_on_each_other(gpu, q38):
    """A sequence's bits are the same alone and beside others of its own form."""
    for rows in ([3, 1, 5], [200, 70, 41]):
        c = DeltaCase(rows, 2, 4, 128, 128, seed=12)
        out, states = run(q38, gpu, c)
        for i, n in enumerate(rows):
            d = DeltaCase([n], 2, 4, 128, 128, spare=c.slots - 2)
            a = int(c.off[i])
            d.qkv, d.g_log, d.beta = c.qkv[a:a + n], c.g_log[a:a + n], c.beta[a:a + n]
            d.states, d.slots, d.origin, d.last = c.states, c.slots, c.origin[i:i + 1], c.last[i:i + 1]
            o, s = run(q38, gpu, d)
            assert torch.equal(o, out[a:a + n]) and torch.equal(s[int(c.last[i])], states[int(c.last[i])])


@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("dv", [64, 128, 256])
@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 2), (2, 6)])
def test_head_sizes_of_the_long_form(gpu, q38, dk, dv, hk, hv):
    c = DeltaCase([45, 20, 1], hk, hv, dk, dv, seed=dk + dv + hv)
    check(c, *run(q38, gpu, c))


@pytest.mark.parametrize("seqs,rows", [(65, 20), (64, 33), (130, 3), (200, 17), (65, 30), (130, 29), (31, 17), (32, 28)])
def test_many_sequences(gpu, q38, seqs, rows):
    """More sequences than a wave has lanes, some of no rows."""
    lens = [i * 7 % (rows + 1) if i % 5 else rows for i in range(seqs)]
    c = DeltaCase(lens, 1, 2, 64, 64, seed=seqs)
    check(c, *run(q38, gpu, c))


def test_most_sequences(gpu, q38):
    """4096 sequences: as many alone in small batches, bit for bit."""
    for max_rows in (2, 20, 40):
        lens = [i % 3 for i in range(4096)]
        lens[1000] = max_rows
        c = DeltaCase(lens, 1, 1, 64, 64, seed=13, spare=0)
        out, states = run(q38, gpu, c)
        for a in (0, 960, 4060):
            d = DeltaCase(lens[a:a + 41], 1, 1, 64, 64, spare=c.slots - 82)
            r0, r1 = int(c.off[a]), int(c.off[a + 41] if a + 41 < 4097 else c.off[-1])
            d.qkv, d.g_log, d.beta = c.qkv[r0:r1], c.g_log[r0:r1], c.beta[r0:r1]
            d.rows = r1 - r0
            d.states, d.origin, d.last = c.states, c.origin[a:a + 41], c.last[a:a + 41]
            d.off = c.off[a:a + 1 + len(d.last)] - r0
            o, s = run(q38, gpu, d, max_rows=min(max_rows, d.rows))
            assert torch.equal(o, out[r0:r1])
            at = d.last.long()
            assert torch.equal(s[at], states[at])


def test_most_rows(gpu, q38):
    """A prompt of 2^19 rows: the bits of the same rows in sixteen calls (whole chunks each)."""
    n, parts = 1 << 19, 16
    c = DeltaCase([n], 1, 1, 64, 64, seed=18)
    out, states = run(q38, gpu, c)
    assert torch.isfinite(out.float()).all()
    pool = c.states.cuda()
    at = c.origin.clone()
    for i in range(parts):
        m = n // parts
        d = DeltaCase([m], 1, 1, 64, 64)
        d.qkv, d.g_log, d.beta = c.qkv[i * m:i * m + m], c.g_log[i * m:i * m + m], c.beta[i * m:i * m + m]
        d.origin, d.last = at, c.last
        o, s = run(q38, gpu, d, states=pool)
        assert torch.equal(o, out[i * m:i * m + m]), i
        at = c.last
    assert torch.equal(s[int(c.last[0])], states[int(c.last[0])])


def test_no_rows_copies_states(gpu, q38):
    c = DeltaCase([0, 0, 0], 2, 4, 64, 128, seed=14)
    c.origin[1] = -1
    rule = q38.DeltaRule(gpu, 2, 4, 64, 128, c.scale)
    pool = c.states.cuda()
    batch = q38.DeltaBatch(pool, c.off.cuda(), c.origin.cuda(), c.last.cuda(), 0, 0)
    e = lambda *s, dt=BF16: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
    rule.run(batch, e(0, 2, 64), e(0, 2, 64), e(0, 4, 128), e(0, 4, dt=torch.float32), e(0, 4, dt=torch.float32),
             e(0, 4, 128), None, G.stream())
    torch.cuda.synchronize()
    want = c.states.clone()
    want[c.last.long()] = want[c.origin.long()]
    want[int(c.last[1])] = 0
    assert torch.equal(pool.cpu().nan_to_num(123.0), want.nan_to_num(123.0))


@pytest.mark.parametrize("rows", [[2, 1], [40, 3]])
def test_slots_beyond_32_bits(gpu, q38, rows):
    """A pool of more than 2^31 floats whose last slots are the batch's."""
    c = DeltaCase(rows, 8, 32, 128, 128, seed=15)
    want_out, want = run(q38, gpu, c)
    slots = (1 << 31) // (32 * 128 * 128) + 16
    shift = slots - c.slots
    pool = torch.empty(slots, 32, 128, 128, device="cuda")
    pool[shift:] = c.states.cuda()
    rule = q38.DeltaRule(gpu, 8, 32, 128, 128, c.scale)
    batch = q38.DeltaBatch(pool, c.off.cuda(), c.origin.cuda() + shift, c.last.cuda() + shift, c.rows, c.max_rows)
    out = torch.zeros(c.rows, 32, 128, dtype=BF16, device="cuda")
    rule.run(batch, *c.operands("cuda"), out, G.workspace(max(16, rule.workspace_size(batch))), G.stream())
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want_out)
    at = c.last.long()
    assert torch.equal(pool[shift:].cpu()[at], want[at])


@pytest.mark.parametrize("rows", [[2], [40]])
def test_row_offsets_beyond_32_bits(gpu, q38, rows):
    """Operands of more than 2^31 elements whose last rows are the batch's."""
    stride = 1 << 20
    c = DeltaCase(rows, 2, 4, 64, 64, seed=16)
    want_out, want = run(q38, gpu, c)
    before = (1 << 31) // stride + 5
    wide = torch.zeros(before + c.rows, stride, dtype=BF16, device="cuda")
    qkv = [t.cuda() for t in c.operands("cpu")[:3]]
    views = []
    for i, x in enumerate(qkv):
        v = wide[:, 4096 * i:4096 * i + x[0].numel()].unflatten(1, tuple(x.shape[1:]))
        v[before:] = x
        views.append(v)
    pad = lambda t: torch.cat([torch.zeros(before, 4), t]).cuda()  # noqa: E731
    pool = c.states.cuda()
    rule = q38.DeltaRule(gpu, 2, 4, 64, 64, c.scale)
    batch = q38.DeltaBatch(pool, (c.off + before).cuda(), c.origin.cuda(), c.last.cuda(), before + c.rows, c.max_rows)
    out = torch.zeros(before + c.rows, 4, 64, dtype=BF16, device="cuda")
    rule.run(batch, *views, pad(c.g_log), pad(c.beta), out, G.workspace(max(16, rule.workspace_size(batch))), G.stream())
    torch.cuda.synchronize()
    assert torch.equal(out[before:].cpu(), want_out) and (out[:before] == 0).all()
    at = c.last.long()
    assert torch.equal(pool.cpu()[at], want[at])


def test_two_calls_at_once(gpu, q38):
    """The long and the short form on two streams over one pool, other slots: the same bits as alone."""
    jobs = []
    for rows in ([300, 65, 129], [1, 2, 1, 7]):
        c = DeltaCase(rows, 2, 4, 128, 128, seed=17)
        want = run(q38, gpu, c)
        jobs.append((c, want))
    n = jobs[0][0].slots
    pool = torch.cat([c.states for c, _ in jobs]).cuda()
    calls = []
    for i, (c, _) in enumerate(jobs):
        rule = q38.DeltaRule(gpu, 2, 4, 128, 128, c.scale)
        batch = q38.DeltaBatch(pool, c.off.cuda(), c.origin.cuda() + i * n, c.last.cuda() + i * n, c.rows, c.max_rows)
        out = torch.zeros(c.rows, 4, 128, dtype=BF16, device="cuda")
        calls.append((rule, batch, c.operands("cuda"), out, G.workspace(max(16, rule.workspace_size(batch))), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(4):
        for rule, batch, ops, out, ws, st in calls:
            rule.run(batch, *ops, out, ws, st.cuda_stream)
    torch.cuda.synchronize()
    for i, ((c, (o, s)), call) in enumerate(zip(jobs, calls)):
        at = c.last.long()
        assert torch.equal(call[3].cpu(), o) and torch.equal(pool.cpu()[at + i * n], s[at])


@pytest.mark.parametrize("rows", [[3, 1, 5, 2], [40, 70, 33, 5]])
def test_nan_stays_in_its_sequence(gpu, q38, rows):
    """NaN in every operand of one sequence and in the rows of nobody: the others' bits stay."""
    c = DeltaCase(rows, 2, 4, 64, 128, seed=19, gap=3)
    want_out, want = run(q38, gpu, c)
    a, b = int(c.off[1]), int(c.off[2])
    bad = torch.ones(c.rows, dtype=torch.bool)
    bad[int(c.off[0]):a] = False
    bad[b:int(c.off[-1])] = False
    for t in (c.qkv, c.g_log, c.beta):
        t[bad] = math.nan
    c.states[int(c.origin[1])] = math.nan
    out, states = run(q38, gpu, c)
    assert torch.equal(out[:a], want_out[:a]) and torch.equal(out[b:], want_out[b:])
    for i in (0, 2, 3):
        assert torch.equal(states[int(c.last[i])], want[int(c.last[i])])
    assert torch.isnan(out[a:b].float()).all()


@pytest.mark.parametrize("rows", [[5], [100]])
def test_zero_beta_and_zero_rows_leave_the_state(gpu, q38, rows):
    """beta 0 and no decay: the state as it was, bit for bit in both forms; the outputs S q."""
    c = DeltaCase(rows, 1, 2, 64, 64, seed=20, decay=0.0)
    c.beta[:] = 0
    out, states = run(q38, gpu, c)
    check(c, out, states)
    assert torch.equal(states[int(c.last[0])], c.states[int(c.origin[0])])


def test_workspace_is_aligned_to_16_bytes_only(gpu, q38):
    c = DeltaCase([90, 40], 2, 4, 128, 128, seed=21)
    want = run(q38, gpu, c)
    need = q38.DeltaRule(gpu, 2, 4, 128, 128, c.scale).workspace_size(
        q38.DeltaBatch(c.states.cuda(), c.off.cuda(), c.origin.cuda(), c.last.cuda(), c.rows, c.max_rows))
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device="cuda")
    at = 48 - ws.data_ptr() % 32
    got = run(q38, gpu, c, ws=ws[at:at + need])
    last = c.last.long()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][last], want[1][last])
    assert (ws[:at] == 0xff).all() and (ws[at + need:] == 0xff).all()


@pytest.mark.parametrize("decay", [0.0, 0.001, 0.05, 1.0])
@pytest.mark.parametrize("keys", ["spread", "concentrated"])
@pytest.mark.parametrize("heads", list(HEADS))
def test_chunked_states_are_as_exact_as_float_rows(gpu, q38, heads, keys, decay):
    """The final states against the recurrence's in 64 bits: delta_cases.state_limit."""
    hk, hv, dk, dv = HEADS[heads]
    c = DeltaCase([128, 70], hk, hv, dk, dv, seed=22, decay=decay)
    if keys == "concentrated":
        concentrate_keys(c)
    _, states = run(q38, gpu, c)
    exact = final_states(c, torch.float64)
    got = state_error(states[c.last.long()], exact)
    limit = state_limit(c, exact)
    assert bool((got <= limit).all()), (got.max().item(), (got / limit).max().item())


@pytest.mark.parametrize("at", [0, 20, 45, 69])
@pytest.mark.parametrize("what", ["q nan", "q inf", "k nan", "k inf", "v nan", "v inf", "g nan", "beta nan", "beta inf"])
@pytest.mark.parametrize("in_place", [False, True])
def test_non_finite_operands_reach_only_later_rows(gpu, q38, what, at, in_place):
    """One element of one row of a prompt is infinite or NaN: what the recurrence in 64 bits keeps finite, the rows
    before it, other heads and, for a value, other value dims, is as exact as without it, also among the rows
    of its chunk; the rest is not finite. The other sequence's bits stay."""
    hk, hv, dk, dv = 2, 4, 64, 128
    c = DeltaCase([70, 40], hk, hv, dk, dv, seed=23)
    if in_place:
        c.last = c.origin.clone()
    clean_out, clean = run(q38, gpu, c)
    _, ob, _, sb = c.exact(CHUNK)
    x = math.nan if what.endswith("nan") else math.inf
    if what[0] == "q":
        c.qkv[at, dk + 5] = x                   # of key head 1
    elif what[0] == "k":
        c.qkv[at, hk * dk + 5] = x              # of key head 0
    elif what[0] == "v":
        c.qkv[at, 2 * hk * dk + dv + 9] = x     # of value head 1
    elif what[0] == "g":
        c.g_log[at, 2] = x
    else:
        c.beta[at, 3] = x
    want, _, S, _ = c.exact()
    out, states = run(q38, gpu, c)
    assert torch.equal(out[70:], clean_out[70:]) and torch.equal(states[int(c.last[1])], clean[int(c.last[1])])
    fine = torch.isfinite(want[:70])
    assert bool(fine.any()) and not bool(fine.all())
    assert torch.equal(torch.isfinite(out[:70]), fine)
    assert bool(((out[:70].double() - want[:70]).abs() <= ob[:70])[fine].all())
    got, want = states[int(c.last[0])].double(), S[69]
    whole = torch.isfinite(want).all(-1)
    assert not bool(torch.isfinite(got[~whole]).any())
    assert bool(((got - want).norm(dim=-1) <= sb[69])[whole].all())


def test_non_finite_origin_stays_in_its_value_rows(gpu, q38):
    c = DeltaCase([50, 33], 1, 2, 64, 64, seed=24)
    want, ob, S, sb = c.exact(CHUNK)
    c.states[int(c.origin[0]), 1, 7, 3] = math.nan
    out, states = run(q38, gpu, c)
    bad = torch.zeros(c.rows, 2, 64, dtype=torch.bool)
    bad[:50, 1, 7] = True
    assert torch.isnan(out[bad].float()).all()
    assert bool(((out.double() - want).abs() <= ob)[~bad].all())
    for i, r in ((0, 49), (1, 82)):
        off = (states[int(c.last[i])].double() - S[r]).norm(dim=-1)
        assert bool((off <= sb[r])[~bad[r]].all()) and torch.isnan(off[bad[r]]).all()


@pytest.mark.parametrize("decay", [0.0, 0.05, 1.0])
@pytest.mark.parametrize("keys", ["spread", "concentrated"])
@pytest.mark.parametrize("heads", list(HEADS))
def test_chunked_outputs_are_off_by_their_rounding(gpu, q38, heads, keys, decay):
    c = DeltaCase([128, 70], *HEADS[heads], seed=25, decay=decay)
    if keys == "concentrated":
        concentrate_keys(c)
    out, _ = run(q38, gpu, c)
    want = c.exact()[0]
    got, limit = output_error(out, want), output_limit(want)
    assert bool((got <= limit).all()), float((got / limit).max())


@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("dv", [64, 128, 256])
def test_sequences_run_again_at_every_size(gpu, q38, dk, dv):
    """A NaN value and, in another sequence, an infinite key: rows before them as without them, whatever the
    sizes; captured, and replayed over the same slots."""
    c = DeltaCase([50, 33, 90], 2, 4, dk, dv, seed=26)
    want, ob, S, sb = c.exact(CHUNK)
    clean_out, clean = run(q38, gpu, c)
    c.qkv[40, 2 * 2 * dk + 3 * dv + dv - 1] = math.nan
    c.qkv[50 + 33 + 77, 2 * dk + dk - 1] = math.inf        # of key head 0: value heads 0 and 1
    bad = torch.zeros(c.rows, 4, dv, dtype=torch.bool)
    bad[40:50, 3, dv - 1] = True
    bad[160:, :2] = True
    states = c.states.cuda()
    rule = q38.DeltaRule(gpu, 2, 4, dk, dv, c.scale)
    batch = q38.DeltaBatch(states, c.off.cuda(), c.origin.cuda(), c.last.cuda(), c.rows, c.max_rows)
    ops, out = c.operands("cuda"), torch.zeros(c.rows, 4, dv, dtype=BF16, device="cuda")
    ws = G.workspace(max(16, rule.workspace_size(batch)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rule.run(batch, *ops, out, ws, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.fill_(3.0)
        states[c.last.long().cuda()] = 5.0
        graph.replay()
        torch.cuda.synchronize()
        got, now = out.cpu(), states.cpu()
        assert torch.equal(torch.isfinite(got), ~bad)
        assert bool(((got.double() - want).abs() <= ob)[~bad].all())
        for i, r in enumerate((49, 82, 172)):
            off = (now[int(c.last[i])].double() - S[r]).norm(dim=-1)
            assert bool((off <= sb[r])[~bad[r]].all()) and not bool(torch.isfinite(off[bad[r]]).any())
        assert torch.equal(got[50:83], clean_out[50:83]) and torch.equal(now[int(c.last[1])], clean[int(c.last[1])])
