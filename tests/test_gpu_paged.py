"""The paged cache on the GPU: q38_paged_append and q38_paged_attention against float64.

Places of the cache that no token holds are NaN (bf16) or have NaN scales (Q8), and unused page
numbers are out of range, so a read of either shows. Tolerances: paged_cases.attention64."""
import math

import pytest
import torch

import gpu_util as G
from paged_cases import BF16, HALF_16, HALF_F32, Batch, attention64, cancel_values

pytestmark = pytest.mark.gpu


def batch_on_gpu(q38, b):
    return q38.PagedBatch(b.off.cuda(), b.tokens.cuda(), b.table.cuda(), b.rows, b.max_rows)


def run_attend(q38, gpu, b, cache, q, scale, out=None, ws=None):
    dev = [None if t is None else t.cuda() for t in cache]
    C = q38.PagedCache(gpu, *dev)
    B = batch_on_gpu(q38, b)
    qd = q.cuda()
    out = torch.full(q.shape, 7.0, dtype=BF16, device="cuda") if out is None else out
    if ws is None:  # a dirty workspace: what it holds must not matter
        ws = torch.full((max(16, C.workspace_size(B, q.shape[1])),), 0xff, dtype=torch.uint8, device="cuda")
    C.attend(B, qd, out, scale, ws, G.stream())
    torch.cuda.synchronize()
    return out.cpu()


def check_attend(b, cache, q, scale, got):
    want, bound = attention64(b, *cache, q, scale)
    owned = torch.zeros(b.rows, dtype=torch.bool)
    owned[int(b.off[0]):int(b.off[-1])] = True
    assert (got[~owned] == 7.0).all(), "rows of nobody were written"
    err = (got.double() - want)[owned].abs()
    worst = (err / bound[owned].clamp_min(1e-300)).nan_to_num(nan=math.inf, posinf=math.inf)
    worst = worst.where(err > 0, 0)
    assert worst.max() <= 1.0 if worst.numel() else True, float(worst.max())


GEOS = {  # kv heads, queries per kv head, head dim
    "family": (2, 8, 256), "gqa4_128": (4, 4, 128), "mha_64": (3, 1, 64), "odd_group": (2, 7, 128),
    "mqa16_64": (1, 16, 64), "mqa_wide": (1, 24, 256),
}
LENGTHS = {  # rows, tokens after the call
    "one": ([1], [1]),
    "decode": ([1] * 7, [1, 2, 15, 16, 17, 33, 200]),
    "decode_long": ([1, 1], [3001, 517]),
    "empty_between": ([0, 1, 0, 0, 2, 0], [0, 5, 40, 0, 129, 64]),
    "verify": ([4, 3, 1, 5], [300, 3, 64, 1029]),
    "verify_wide": ([16, 9, 33], [800, 9, 70]),
    "prompt": ([130, 67, 1, 260], [130, 200, 90, 700]),
    "row_sees_nothing": ([3, 2], [1, 0]),
}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("geo", list(GEOS))
@pytest.mark.parametrize("q8", [False, True])
def test_attention(gpu, q38, geo, lengths, q8):
    hkv, group, dim = GEOS[geo]
    rows, tokens = LENGTHS[lengths]
    b = Batch(rows, tokens, page=16, hkv=hkv, dim=dim, seed=len(geo) + len(lengths), gap=2)
    cache = b.cache(q8)
    q = (b.randn(b.rows, hkv * group, dim) * 1.5).to(BF16)
    scale = dim ** -0.5
    check_attend(b, cache, q, scale, run_attend(q38, gpu, b, cache, q, scale))


@pytest.mark.parametrize("rows", [16, 17, 32, 33, 128, 129, 256, 257])
@pytest.mark.parametrize("dim", [64, 256])
def test_attention_rows_around_a_tile(gpu, q38, rows, dim):
    b = Batch([rows, 1], [rows + 30, 90], hkv=1, dim=dim, seed=rows)
    cache = b.cache(False)
    q = b.randn(b.rows, 1, dim).to(BF16)
    check_attend(b, cache, q, 0.1, run_attend(q38, gpu, b, cache, q, 0.1))


@pytest.mark.parametrize("rows,tokens", [([1, 2], [300, 77]), ([5], [700])])
@pytest.mark.parametrize("hkv,group,dim", [(1, 128, 64), (2, 128, 128), (1, 128, 256), (2, 100, 256), (64, 4, 64), (64, 1, 128),
                                           (5, 3, 128)])
@pytest.mark.parametrize("q8", [False, True])
def test_attention_many_heads(gpu, q38, rows, tokens, hkv, group, dim, q8):
    b = Batch(rows, tokens, hkv=hkv, dim=dim, seed=hkv + group)
    cache = b.cache(q8)
    q = b.randn(b.rows, hkv * group, dim).to(BF16)
    check_attend(b, cache, q, dim ** -0.5, run_attend(q38, gpu, b, cache, q, dim ** -0.5))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q8", [False, True])
def test_long_tiles_are_cut_and_joined(gpu, q38, dim, q8):
    """Few tiles over long contexts: every workgroup takes a part of one."""
    b = Batch([70, 3, 41], [6000, 2500, 41], page=32, hkv=1, dim=dim, seed=dim)
    cache = b.cache(q8)
    q = b.randn(b.rows, 2, dim).to(BF16)
    check_attend(b, cache, q, dim ** -0.5, run_attend(q38, gpu, b, cache, q, dim ** -0.5))


@pytest.mark.parametrize("seqs,rows", [(65, 1), (150, 3), (4096, 1), (130, 40)])
def test_attention_many_sequences(gpu, q38, seqs, rows):
    """More sequences than a wave has lanes; some without rows or tokens."""
    lens = [(i * 7 % (rows + 1)) if i % 5 else rows for i in range(seqs)]
    tokens = [n + i * 13 % 90 for i, n in enumerate(lens)]
    tokens[3], tokens[64] = 2000, 777
    b = Batch(lens, tokens, hkv=1, dim=64, seed=seqs)
    cache = b.cache(False)
    q = b.randn(b.rows, 2, 64).to(BF16)
    check_attend(b, cache, q, 0.125, run_attend(q38, gpu, b, cache, q, 0.125))


@pytest.mark.parametrize("rows", [1, 50])
def test_attention_scale_zero(gpu, q38, rows):
    b = Batch([rows], [rows + 200], hkv=2, dim=64, seed=17)
    cache = b.cache(False)
    q = b.randn(b.rows, 8, 64).to(BF16)
    check_attend(b, cache, q, 0.0, run_attend(q38, gpu, b, cache, q, 0.0))


@pytest.mark.parametrize("rows", [1, 40])
def test_row_offsets_beyond_32_bits(gpu, q38, rows):
    """Row tensors of more than 2^31 elements whose last rows are the batch's."""
    hkv, hq, dim = 2, 8, 64
    stride = 1 << 20
    b = Batch([rows], [rows + 100], hkv=hkv, dim=dim, seed=18)
    before = (1 << 31) // stride + 5
    dev = [t.cuda() for t in b.cache(False)[:2]]
    wide = torch.zeros(before + rows, stride, dtype=BF16, device="cuda")
    w = hkv * dim
    q, k, v = b.randn(rows, hq, dim).to(BF16), b.randn(rows, hkv, dim).to(BF16), b.randn(rows, hkv, dim).to(BF16)
    wide[before:, :hq * dim] = q.view(rows, -1).cuda()
    wide[before:, 4096:4096 + w] = k.view(rows, -1).cuda()
    wide[before:, 8192:8192 + w] = v.view(rows, -1).cuda()
    view = lambda at, heads: wide[:, at:at + heads * dim].unflatten(1, (heads, dim))  # noqa: E731
    B = q38.PagedBatch((b.off + before).cuda(), b.tokens.cuda(), b.table.cuda(), before + rows, rows)
    C = q38.PagedCache(gpu, *dev)
    C.append(B, view(4096, hkv), view(8192, hkv), G.stream())
    C.attend(B, view(0, hq), view(16384, hq), 0.1, G.workspace(max(16, C.workspace_size(B, hq))), G.stream())
    torch.cuda.synchronize()
    p, o = b.places(0)
    cache = [t.cpu() for t in dev] + [None, None]
    assert torch.equal(cache[0][p, :, o][100:], k) and torch.equal(cache[1][p, :, o][100:], v)
    check_attend(b, cache, q, 0.1, view(16384, hq)[before:].cpu())


@pytest.mark.parametrize("page", [32, 64, 256, 1024])
@pytest.mark.parametrize("q8", [False, True])
def test_attention_page_sizes(gpu, q38, page, q8):
    b = Batch([1, 40, 2], [1500, 333, page + 1], page=page, hkv=2, dim=128, seed=page)
    cache = b.cache(q8)
    q = b.randn(b.rows, 8, 128).to(BF16)
    check_attend(b, cache, q, 0.1, run_attend(q38, gpu, b, cache, q, 0.1))


@pytest.mark.parametrize("rows,tokens", [([1], [900]), ([3, 1], [500, 40]), ([70], [400])])
def test_attention_peaked_scores(gpu, q38, rows, tokens):
    """Scores of thousands: all weight on one token (a running maximum that jumps), and a negative
    scale, which turns the order around."""
    b = Batch(rows, tokens, hkv=2, dim=128, seed=9)
    cache = b.cache(False)
    q = (b.randn(b.rows, 8, 128) * 64).to(BF16)
    for scale in (1.0, -0.5):
        check_attend(b, cache, q, scale, run_attend(q38, gpu, b, cache, q, scale))


@pytest.mark.parametrize("rows,group", [([6], 2), ([3], 8), ([40], 4), ([90], 8)])
@pytest.mark.parametrize("what", [math.inf, math.nan])
def test_non_finite_tokens_reach_only_the_rows_that_see_them(gpu, q38, rows, group, what):
    """The last new token's value (then its key) is infinite or NaN: the rows before it do not see it."""
    n = rows[0]
    b = Batch(rows, [n + 45], hkv=2, dim=128, seed=11)
    for which in (0, 1):
        cache = b.cache(False)
        q = b.randn(b.rows, 2 * group, 128).to(BF16)
        clean = run_attend(q38, gpu, b, cache, q, 0.1)
        page, at = b.places(0)
        cache[which][page[-1], :, at[-1], 3] = what
        got = run_attend(q38, gpu, b, cache, q, 0.1)
        assert torch.equal(got[:-1], clean[:-1])
        last = got[-1].float()
        if which == 1:  # a value: its own dim only
            assert not torch.isfinite(last[:, 3]).any()
            keep = [i for i in range(128) if i != 3]
            assert torch.equal(got[-1][:, keep], clean[-1][:, keep])
        elif math.isnan(what):
            assert torch.isnan(last).all()


def test_bad_lengths_and_pages_give_nan_and_nothing_else(gpu, q38):
    b = Batch([1, 2, 1, 1], [40, 50, 60, 20], hkv=2, dim=64, seed=12)
    cache = b.cache(False)
    q = b.randn(b.rows, 4, 64).to(BF16)
    clean = run_attend(q38, gpu, b, cache, q, 0.125)
    b.table[1, 2] = b.pages          # a seen page out of range
    b.table[2, 0] = -1
    b.tokens[3] = b.width * b.page + 1  # tokens behind the table
    got = run_attend(q38, gpu, b, cache, q, 0.125)
    assert torch.equal(got[0], clean[0])
    assert torch.isnan(got[1:].float()).all()
    b.tokens[3] = -5                 # no token: rows that see nothing
    got = run_attend(q38, gpu, b, cache, q, 0.125)
    assert (got[4] == 0).all()


def test_offsets_outside_the_rows_are_clamped(gpu, q38):
    b = Batch([2, 3], [20, 30], hkv=2, dim=64, seed=13)
    cache = b.cache(False)
    q = b.randn(b.rows, 4, 64).to(BF16)
    b.off[2] = 1000
    got = run_attend(q38, gpu, b, cache, q, 0.125)
    b.off[2] = 5
    assert torch.equal(got, run_attend(q38, gpu, b, cache, q, 0.125))


def test_attention_strided_rows_and_shared_prefix(gpu, q38):
    """q and out as slices of wider rows; two sequences over the same prefix pages."""
    b = Batch([2, 3], [50, 67], hkv=2, dim=64, seed=14)
    b.table[1, :3] = b.table[0, :3]   # 48 shared tokens of 16-token pages
    cache = b.cache(False)
    wide = b.randn(b.rows, 3, 8, 64).to(BF16)
    q = wide[:, 1]
    want = run_attend(q38, gpu, b, cache, q.contiguous(), 0.125)
    check_attend(b, cache, q, 0.125, want)
    dev = [None if t is None else t.cuda() for t in cache]
    C, B = q38.PagedCache(gpu, *dev), batch_on_gpu(q38, b)
    wd = wide.cuda()
    od = torch.full_like(wd, 5.0)
    ws = G.workspace(max(16, C.workspace_size(B, 8)))
    C.attend(B, wd[:, 1], od[:, 2], 0.125, ws, G.stream())
    torch.cuda.synchronize()
    assert torch.equal(od[:, 2].cpu(), want)
    assert (od[:, :2] == 5.0).all()


def test_attention_does_not_depend_on_max_rows(gpu, q38):
    """max_rows is a hint: a wrong one costs time, not results."""
    b = Batch([20, 1, 7], [400, 90, 30], hkv=2, dim=128, seed=15)
    cache = b.cache(False)
    q = b.randn(b.rows, 16, 128).to(BF16)
    for hint in (1, 2, 20, b.rows):
        b.max_rows = hint
        check_attend(b, cache, q, 0.09, run_attend(q38, gpu, b, cache, q, 0.09))


def test_offsets_beyond_32_bits(gpu, q38):
    """A pool of more than 2^31 elements whose last pages hold the tokens."""
    page, hkv, dim = 64, 2, 256
    pages = (1 << 31) // (page * hkv * dim) + 8
    b = Batch([1, 2], [150, 70], page=page, hkv=hkv, dim=dim, seed=16)
    cache = b.cache(False)
    shift = pages - b.pages
    big = [torch.zeros(pages, hkv, page, dim, dtype=BF16, device="cuda") for _ in range(2)]
    for t, s in zip(big, cache):
        t[shift:] = s.cuda()
    table = b.table.clone()
    table[(table >= 0) & (table < b.pages)] += shift
    C = q38.PagedCache(gpu, *big)
    B = q38.PagedBatch(b.off.cuda(), b.tokens.cuda(), table.cuda(), b.rows, 2)
    q = b.randn(b.rows, 16, dim).to(BF16)
    out = torch.full(q.shape, 7.0, dtype=BF16, device="cuda")
    ws = G.workspace(max(16, C.workspace_size(B, 16)))
    C.attend(B, q.cuda(), out, 0.06, ws, G.stream())
    torch.cuda.synchronize()
    check_attend(b, cache, q, 0.06, out.cpu())
    k = b.randn(b.rows, hkv, dim).to(BF16)
    C.append(B, k.cuda(), k.cuda(), G.stream())
    torch.cuda.synchronize()
    p, o = b.places(0)
    assert torch.equal(big[0][shift + p[-1], :, o[-1]].cpu(), k[0])


def test_most_rows(gpu, q38):
    """A prompt of 2^19 rows: a few of its rows against float64."""
    n = 1 << 19
    b = Batch([n], [n], page=1024, hkv=1, dim=64, seed=19)
    cache = b.cache(False)
    q = b.randn(n, 1, 64).to(BF16)
    got = run_attend(q38, gpu, b, cache, q, 0.125)
    assert torch.isfinite(got.float()).all()
    rows = [0, 1, 255, 256, 131071, 300000, n - 257, n - 1]
    for r in rows:  # each as the last row of a sequence of its own
        one = Batch([1], [r + 1], page=1024, hkv=1, dim=64)
        one.table, one.pages = b.table, b.pages
        check_attend(one, cache, q[r:r + 1], 0.125, got[r:r + 1])


# ------------------------------------------------------------------ append
def quantised(x):
    """Codes and scales of head rows [..., dim] by exact arithmetic (integers in float64)."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    code = torch.where(top > 0, torch.round(x * 127 / top), 0)
    return code, top.squeeze(-1) / 127


@pytest.mark.parametrize("rows,tokens", [([1], [1]), ([1] * 70, list(range(1, 71))), ([37, 0, 200, 5], [37, 9, 260, 5])])
@pytest.mark.parametrize("hkv,dim", [(2, 256), (3, 128), (5, 64)])
@pytest.mark.parametrize("q8", [False, True])
def test_append(gpu, q38, rows, tokens, hkv, dim, q8):
    b = Batch(rows, tokens, page=16, hkv=hkv, dim=dim, seed=21, gap=1)
    cache = b.cache(q8, poison=3.0)
    kv = b.randn(b.rows, 2, hkv, dim)
    kv[::3] *= torch.exp2(torch.randint(-30, 30, (kv[::3].shape[0], 2, hkv, 1), generator=b.g).float())
    kv = kv.to(BF16)
    want = [None if t is None else t.clone() for t in cache]
    for i, n in enumerate(rows):
        p, o = (t[tokens[i] - n:] for t in b.places(i))
        for j in range(2):
            x = kv[int(b.off[i]):int(b.off[i]) + n, j]
            if q8:
                code, scale = quantised(x)
                want[j][p, :, o] = code.to(torch.int8)
                want[2 + j][p, :, o] = scale.float()
            else:
                want[j][p, :, o] = x
    dev = [None if t is None else t.cuda() for t in cache]
    C = q38.PagedCache(gpu, *dev)
    kvd = kv.cuda()
    C.append(batch_on_gpu(q38, b), kvd[:, 0], kvd[:, 1], G.stream())
    torch.cuda.synchronize()
    for got, w in zip(dev, want):
        if w is not None and w.dtype == torch.float32:
            assert ((got.cpu().double() - w.double()).abs() <= w.double().abs() * 2 * HALF_F32).all()
        elif w is not None:
            assert torch.equal(got.cpu(), w)


def test_append_many_sequences(gpu, q38):
    lens = [i % 3 for i in range(4096)]
    tokens = [n + i % 20 for i, n in enumerate(lens)]
    b = Batch(lens, tokens, hkv=2, dim=64, seed=24)
    want = list(b.cache(False, poison=3.0)[:2])
    dev = [t.cuda() for t in want]
    kv = b.randn(b.rows, 2, 2, 64).to(BF16)
    for i, n in enumerate(lens):
        if n:
            p, o = (t[tokens[i] - n:] for t in b.places(i))
            for j in range(2):
                want[j][p, :, o] = kv[int(b.off[i]):int(b.off[i]) + n, j]
    kvd = kv.cuda()
    q38.PagedCache(gpu, *dev).append(batch_on_gpu(q38, b), kvd[:, 0], kvd[:, 1], G.stream())
    torch.cuda.synchronize()
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu(), w)


def test_append_q8_extremes(gpu, q38):
    """Zeros, ties, the largest bf16, infinities and NaN."""
    big = torch.finfo(BF16).max
    x = torch.zeros(6, 1, 64)
    x[1, 0, 0], x[1, 0, 1:4] = 1.0, torch.tensor([0.5, -0.5, 0.25])   # 63.5 and -63.5: to the even 64
    x[2, 0, :3] = torch.tensor([big, -big, big / 2])
    x[3, 0, 5] = math.inf
    x[4, 0, 6] = math.nan
    x[5, 0, :2] = torch.tensor([2.0 ** -126, 2.0 ** -127])
    x = x.to(BF16)
    b = Batch([6], [6], hkv=1, dim=64, seed=22)
    dev = [t.cuda() for t in b.cache(True)]
    q38.PagedCache(gpu, *dev).append(batch_on_gpu(q38, b), x.cuda(), x.cuda(), G.stream())
    torch.cuda.synchronize()
    p, o = b.places(0)
    code, scale = dev[0].cpu()[p, :, o][:, 0], dev[2].cpu()[p, :, o][:, 0]
    assert (code[0] == 0).all() and scale[0] == 0
    assert code[1, :4].tolist() == [127, 64, -64, 32] and scale[1] == torch.tensor(1.0) / 127
    assert code[2, :2].tolist() == [127, -127] and torch.isfinite(scale[2])
    assert torch.isnan(scale[3]) and torch.isnan(scale[4])
    assert code[5, :2].tolist() == [127, 64]


def test_append_skips_bad_places(gpu, q38):
    b = Batch([2, 2, 2, 1], [20, 30, 1, 9], hkv=2, dim=64, seed=23)
    cache = b.cache(False, poison=3.0)
    b.table[0, 1] = b.pages         # the last tokens of sequence 0: not written
    b.tokens[1] = b.width * b.page + 1  # its last row is behind the table
    b.table[1, b.width - 1] = -1
    k = b.randn(b.rows, 2, 64).to(BF16)
    dev = [t.cuda() for t in cache[:2]]
    q38.PagedCache(gpu, *dev).append(batch_on_gpu(q38, b), k.cuda(), k.cuda(), G.stream())
    torch.cuda.synchronize()
    want = [t.clone() for t in cache[:2]]
    for t in want:
        t[b.table[2, 0], :, 0] = k[5]  # sequence 2: its first row is token -1
        t[b.table[3, 0], :, 8] = k[6]
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu(), w)


# ------------------------------------------------------------------ together, captured, on streams
@pytest.mark.parametrize("q8", [False, True])
def test_prompt_then_decode(gpu, q38, q8):
    """Prompts of three requests entered in two calls, then decode steps: every step's attention
    against float64 over what the cache holds."""
    hkv, hq, dim, page = 2, 8, 128, 16
    final = [90, 33, 7]
    b = Batch(final, final, page=page, hkv=hkv, dim=dim, seed=31)
    dev = [None if t is None else t.cuda() for t in b.cache(q8)]
    C = q38.PagedCache(gpu, *dev)
    ws = G.workspace(1 << 24)
    steps = [[40, 30, 0], [46, 0, 3]] + [[1, 1, 1]] * 3 + [[1, 0, 1]]
    assert [sum(s[i] for s in steps) for i in range(3)] == [90, 33, 7]
    at = [0, 0, 0]
    for step in steps:
        at = [a + n for a, n in zip(at, step)]
        now = Batch(step, at, page=page, hkv=hkv, dim=dim, width=b.width)
        now.table = b.table
        k, v = (b.randn(now.rows, hkv, dim).to(BF16) for _ in range(2))
        q = b.randn(now.rows, hq, dim).to(BF16)
        B = batch_on_gpu(q38, now)
        out = torch.full(q.shape, 7.0, dtype=BF16, device="cuda")
        C.append(B, k.cuda(), v.cuda(), G.stream())
        assert C.workspace_size(B, hq) <= ws.numel()
        C.attend(B, q.cuda(), out, dim ** -0.5, ws, G.stream())
        torch.cuda.synchronize()
        check_attend(now, [None if t is None else t.cpu() for t in dev], q, dim ** -0.5, out.cpu())


def test_captured_step_replayed_with_new_lengths(gpu, q38):
    """A decode step in a graph: lengths, pages and operands change between the replays; every
    replay equals the eager call on another stream with a workspace of its own."""
    hkv, hq, dim = 2, 16, 256
    b = Batch([1] * 5, [300, 20, 129, 64, 7], hkv=hkv, dim=dim, seed=32)
    dev = [t.cuda() for t in b.cache(False)[:2]]
    C, B = q38.PagedCache(gpu, *dev), batch_on_gpu(q38, b)
    tokens, q = B._keep[1], torch.zeros(5, hq, dim, dtype=BF16, device="cuda")
    k = torch.zeros(5, hkv, dim, dtype=BF16, device="cuda")
    out = torch.zeros_like(q)
    ws = G.workspace(max(16, C.workspace_size(B, hq)))
    side = torch.cuda.Stream()

    def step(o, w):
        st = torch.cuda.current_stream().cuda_stream
        C.append(B, k, k, st)
        C.attend(B, q, o, 0.06, w, st)

    step(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, ws)
    for i in range(4):
        tokens.copy_(torch.tensor([300 - 70 * i, 20 + i, 129 - i, 64, 7 - i], dtype=torch.int32))
        q.copy_(b.randn(5, hq, dim).to(BF16))
        k.copy_(b.randn(5, hkv, dim).to(BF16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        with torch.cuda.stream(side):
            o2 = torch.zeros_like(q)
            step(o2, torch.zeros_like(ws))
        torch.cuda.synchronize()
        assert torch.equal(got, o2), i


def test_repeated_calls_are_bit_identical(gpu, q38):
    b = Batch([1, 4, 30], [2000, 700, 300], hkv=2, dim=256, seed=33)
    cache = b.cache(False)
    q = b.randn(b.rows, 16, 256).to(BF16)
    first = run_attend(q38, gpu, b, cache, q, 0.06)
    for _ in range(3):
        assert torch.equal(run_attend(q38, gpu, b, cache, q, 0.06), first)


def test_two_calls_at_once(gpu, q38):
    """Calls on two streams with a workspace each: the same bits as one after the other."""
    jobs = []
    for seed, rows, tokens in ((41, [1] * 6, [4000, 700, 90, 1500, 3, 2222]), (42, [90, 33], [1200, 400])):
        b = Batch(rows, tokens, hkv=2, dim=128, seed=seed)
        C, B = q38.PagedCache(gpu, *[t.cuda() for t in b.cache(False)[:2]]), batch_on_gpu(q38, b)
        q = b.randn(b.rows, 16, 128).to(BF16).cuda()
        outs = [torch.zeros_like(q) for _ in range(2)]
        jobs.append((C, B, q, outs, G.workspace(max(16, C.workspace_size(B, 16))), torch.cuda.Stream()))
    for C, B, q, outs, ws, _ in jobs:
        C.attend(B, q, outs[0], 0.09, ws, G.stream())
        torch.cuda.synchronize()
    for _ in range(5):
        for C, B, q, outs, ws, st in jobs:
            C.attend(B, q, outs[1], 0.09, ws, st.cuda_stream)
    torch.cuda.synchronize()
    for _, _, _, outs, _, _ in jobs:
        assert torch.equal(*outs)


@pytest.mark.parametrize("rows", [[3, 1, 2], [40, 70, 33]])
@pytest.mark.parametrize("q8", [False, True])
def test_nan_stays_in_its_sequence(gpu, q38, rows, q8):
    """NaN queries of one sequence and of the rows of nobody, NaN keys and values of its tokens: the
    others' bits stay."""
    b = Batch(rows, [200, 300, 90], hkv=2, dim=128, seed=43, gap=3)
    cache = b.cache(q8)
    q = b.randn(b.rows, 8, 128).to(BF16)
    want = run_attend(q38, gpu, b, cache, q, 0.09)
    a, e = int(b.off[1]), int(b.off[2])
    q[:3], q[-3:], q[a:e] = math.nan, math.nan, math.nan
    p, o = b.places(1)
    for t in cache[2:] if q8 else cache[:2]:
        t[p, :, o] = math.nan
    got = run_attend(q38, gpu, b, cache, q, 0.09)
    assert torch.equal(got[:a], want[:a]) and torch.equal(got[e:], want[e:])
    assert torch.isnan(got[a:e].float()).all()


@pytest.mark.parametrize("rows", [1, 60])
def test_one_token_is_its_value(gpu, q38, rows):
    """Rows that see one token, or tokens of one value, give that value exactly (softmax sums to 1)."""
    b = Batch([rows], [rows], hkv=2, dim=64, seed=44)
    cache = b.cache(False)
    p, o = b.places(0)
    cache[1][p, :, o] = cache[1][p[:1], :, o[:1]].clone()
    q = b.randn(b.rows, 4, 64).to(BF16)
    got = run_attend(q38, gpu, b, cache, q, 0.125)
    v = cache[1][p[0], :, o[0]].repeat_interleave(2, 0)
    assert torch.equal(got[0], v)
    check_attend(b, cache, q, 0.125, got)


@pytest.mark.parametrize("rows,tokens", [([1, 2], [3000, 700]), ([60, 1], [2500, 900])])
def test_workspace_is_aligned_to_16_bytes_only(gpu, q38, rows, tokens):
    """A workspace 16 bytes behind a multiple of 32 (what the call asks for and no more), with items cut across
    workgroups: the bits of any other workspace."""
    b = Batch(rows, tokens, hkv=2, dim=128, seed=45)
    cache = b.cache(False)
    q = b.randn(b.rows, 8, 128).to(BF16)
    want = run_attend(q38, gpu, b, cache, q, 0.09)
    need = q38.PagedCache(gpu, *[t.cuda() for t in cache[:2]]).workspace_size(batch_on_gpu(q38, b), 8)
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device="cuda")
    view = ws[48 - ws.data_ptr() % 32:][:need]
    assert view.data_ptr() % 32 == 16
    assert torch.equal(run_attend(q38, gpu, b, cache, q, 0.09, ws=view), want)
    assert (ws[:48 - ws.data_ptr() % 32] == 0xff).all() and (ws[48 - ws.data_ptr() % 32 + need:] == 0xff).all()


@pytest.mark.parametrize("lengths", ["decode", "verify", "beside_a_prompt", "hint"])
@pytest.mark.parametrize("geo", ["family", "gqa4_128", "mha_64", "mqa_wide"])
@pytest.mark.parametrize("q8", [False, True])
def test_few_queries_have_16_bit_probabilities(gpu, q38, geo, lengths, q8):
    """Sequences of up to 32 queries per kv head, alone and where a prompt of the batch (or a hint of one)
    brings the kernel for many queries: outputs that nearly cancel show the probabilities' rounding."""
    hkv, group, dim = GEOS[geo]
    few = 32 // group
    rows = {"decode": [1, 1, 1], "verify": [few, 1, few], "beside_a_prompt": [1, few, 150, 1], "hint": [few, 1, 1]}[lengths]
    tokens = [30, 200, 777, 1500][:len(rows)]
    b = Batch(rows, tokens, hkv=hkv, dim=dim, seed=62)
    if lengths == "hint":
        b.max_rows = b.rows
    cache, scale = b.cache(q8), 0.005
    q = b.randn(b.rows, hkv * group, dim).to(BF16)
    cancel_values(b, cache, q, scale)
    got = run_attend(q38, gpu, b, cache, q, scale).double()
    for i, n in enumerate(rows):
        if n * group > 32:
            continue
        a, e = int(b.off[i]), int(b.off[i + 1])
        one = Batch([n], [tokens[i]], hkv=hkv, dim=dim)
        one.table = b.table[i:i + 1]
        want, bound = attention64(one, *cache, q[a:e], scale, HALF_16)
        assert bool(((got[a:e] - want).abs() <= bound).all()), (i, float(((got[a:e] - want).abs() / bound).max()))


@pytest.mark.parametrize("rows,tokens", [([6], 3000), ([1], 1700), ([16], 1029), ([90], 4000)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("back", [0, 1, 5, 200, 600])
def test_non_finite_values_in_pieces(gpu, q38, rows, tokens, dim, back):
    """An infinite and a NaN value, `back` tokens before the last one, of a sequence whose tokens are cut into
    many workgroups' pieces: in the last step, among the new rows, and in pieces that every row sees whole."""
    n = rows[0]
    b = Batch(rows, [tokens], hkv=2, dim=dim, seed=46)
    cache = b.cache(False)
    q = b.randn(b.rows, 4, dim).to(BF16)
    clean = run_attend(q38, gpu, b, cache, q, 0.1)
    page, at = b.places(0)
    cache[1][page[-1 - back], :, at[-1 - back], 3] = math.inf
    cache[1][page[-1 - back], :, at[-1 - back], dim - 1] = math.nan
    got = run_attend(q38, gpu, b, cache, q, 0.1)
    sees = torch.arange(n) >= n - 1 - back  # the rows that see the token
    assert torch.equal(got[~sees], clean[~sees])
    assert not torch.isfinite(got[sees][..., [3, dim - 1]].float()).any()
    keep = [i for i in range(dim) if i not in (3, dim - 1)]
    assert torch.equal(got[sees][..., keep], clean[sees][..., keep])


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 8), (256, 8), (256, 16)])
@pytest.mark.parametrize("q8", [False, True])
def test_few_queries_beside_a_prompt_with_bad_tokens(gpu, q38, dim, group, q8):
    """Sequences of few queries in the kernel for many: an infinity that only the last row sees, a NaN that all
    see, a page out of range and tokens behind the table; over several pieces."""
    n = 32 // group
    b = Batch([n, n, n, n, 120, 1], [900, 700, 800, 30, 300, 5], hkv=2, dim=dim, seed=47)
    cache = b.cache(q8)
    q = b.randn(b.rows, 2 * group, dim).to(BF16)
    clean = run_attend(q38, gpu, b, cache, q, 0.1)
    check_attend(b, cache, q, 0.1, clean)
    bad = cache[3] if q8 else cache[1][..., 7]   # a token's value scales, or one dim of its values
    p, o = b.places(0)
    bad[p[-1], :, o[-1]] = math.inf
    p, o = b.places(1)
    bad[p[40], :, o[40]] = math.nan
    b.table[2, 3] = b.pages
    b.tokens[3] = b.width * b.page + 1
    got = run_attend(q38, gpu, b, cache, q, 0.1)
    off = b.off.tolist()
    dims = list(range(dim)) if q8 else [7]
    keep = [] if q8 else [i for i in range(dim) if i != 7]
    assert torch.equal(got[:n - 1], clean[:n - 1]) and torch.equal(got[off[4]:], clean[off[4]:])
    for rows in (slice(n - 1, n), slice(off[1], off[2])):
        assert not torch.isfinite(got[rows][..., dims].float()).any()
        assert torch.equal(got[rows][..., keep], clean[rows][..., keep])
    assert torch.isnan(got[off[2]:off[4]].float()).all()
