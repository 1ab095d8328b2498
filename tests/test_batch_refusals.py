"""The refusals of the batched token mixers (q38_paged_append, q38_paged_attention,
q38_delta_rule): no GPU is needed, every argument is checked before the context is."""
import ctypes as C

import pytest

X = 1 << 20  # a 16-byte aligned address that is never followed


def cache(q38, **kw):
    f = dict(keys=X, values=X, key_scales=None, value_scales=None, format=q38.Q38_KV_BF16, pages=4, page_tokens=16,
             kv_heads=2, head_dim=64)
    f.update(kw)
    return q38.PagedCacheDesc(**f)


def batch(q38, **kw):
    f = dict(sequences=2, rows=3, max_rows=2, table_pages=4, row_offsets=X, tokens=X, page_table=X)
    f.update(kw)
    return q38.PagedBatchDesc(**f)


def append(q38, c, b, k=X, ks=128, v=X, vs=128):
    return q38.lib.q38_paged_append(None, C.byref(c) if c else None, C.byref(b) if b else None, k, ks, v, vs, None)


def attend(q38, c, b, q=X, qs=512, heads=8, scale=0.1, out=X, os=512, ws=X, ws_bytes=1 << 40):
    return q38.lib.q38_paged_attention(None, C.byref(c) if c else None, C.byref(b) if b else None, q, qs, heads, scale,
                                       out, os, ws, ws_bytes, None)


BAD_CACHE = [dict(format=2), dict(format=-1), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=2048),
             dict(pages=0), dict(kv_heads=0), dict(kv_heads=65), dict(head_dim=96), dict(keys=None), dict(values=None),
             dict(keys=X + 8), dict(values=X + 2), dict(key_scales=X), dict(format=1), dict(format=1, key_scales=X),
             dict(format=1, key_scales=X + 4, value_scales=X), dict(format=1, key_scales=X, value_scales=X + 8)]
BAD_BATCH = [dict(sequences=-1), dict(sequences=4097), dict(rows=-1), dict(rows=(1 << 19) + 1), dict(max_rows=0),
             dict(max_rows=4), dict(table_pages=0), dict(table_pages=1 << 26), dict(row_offsets=None),
             dict(tokens=None), dict(page_table=None)]


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_cache(q38, kw):
    assert append(q38, cache(q38, **kw), batch(q38)) == q38.Q38_EINVAL
    assert "q38_paged_append: " in q38.last_error() and "context" not in q38.last_error()
    assert attend(q38, cache(q38, **kw), batch(q38)) == q38.Q38_EINVAL
    assert "q38_paged_attention: " in q38.last_error() and "context" not in q38.last_error()


@pytest.mark.parametrize("kw", BAD_BATCH)
def test_bad_batch(q38, kw):
    for rc in (append(q38, cache(q38), batch(q38, **kw)), attend(q38, cache(q38), batch(q38, **kw))):
        assert rc == q38.Q38_EINVAL and "context" not in q38.last_error()


def test_null_descriptions_and_context(q38):
    assert append(q38, None, batch(q38)) == q38.Q38_EINVAL
    assert attend(q38, cache(q38), None) == q38.Q38_EINVAL
    assert append(q38, cache(q38), batch(q38)) == q38.Q38_EINVAL and "null context" in q38.last_error()
    assert attend(q38, cache(q38), batch(q38)) == q38.Q38_EINVAL and "null context" in q38.last_error()


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(k=X + 8), dict(ks=120), dict(vs=132), dict(ks=-128)])
def test_bad_append_operands(q38, kw):
    assert append(q38, cache(q38), batch(q38), **kw) == q38.Q38_EINVAL
    assert "context" not in q38.last_error()


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(q=X + 4), dict(out=X + 8), dict(qs=504), dict(os=516),
                                dict(heads=0), dict(heads=7), dict(heads=258), dict(qs=1 << 24), dict(scale=float("nan")),
                                dict(scale=float("inf"))])
def test_bad_attention_operands(q38, kw):
    assert attend(q38, cache(q38), batch(q38), **kw) == q38.Q38_EINVAL
    assert "context" not in q38.last_error()


def test_too_many_queries_per_kv_head(q38):
    c = cache(q38, kv_heads=1)
    assert attend(q38, c, batch(q38), qs=129 * 64, heads=129, os=129 * 64) == q38.Q38_EINVAL
    assert "128 per kv head" in q38.last_error()
    assert attend(q38, c, batch(q38), qs=128 * 64, heads=128, os=128 * 64) == q38.Q38_EINVAL
    assert "null context" in q38.last_error()


def test_attention_workspace(q38):
    c, b = cache(q38), batch(q38, table_pages=4096)
    need = q38.lib.q38_paged_attention_workspace_size(C.byref(c), C.byref(b), 8)
    if need:
        assert attend(q38, c, b, ws_bytes=need - 1) == q38.Q38_ESPACE
        assert attend(q38, c, b, ws=None) == q38.Q38_ESPACE
        assert attend(q38, c, b, ws=X + 8) == q38.Q38_ESPACE
    assert attend(q38, c, b, ws_bytes=need) == q38.Q38_EINVAL and "null context" in q38.last_error()
    assert q38.lib.q38_paged_attention_workspace_size(C.byref(c), C.byref(b), 7) == 0
    assert q38.lib.q38_paged_attention_workspace_size(None, C.byref(b), 8) == 0


def test_empty_batches_are_done(q38):
    for kw in (dict(rows=0), dict(sequences=0), dict(rows=0, row_offsets=None, tokens=None, page_table=None)):
        assert append(q38, cache(q38), batch(q38, **kw)) == q38.Q38_OK
        assert attend(q38, cache(q38), batch(q38, **kw)) == q38.Q38_OK


def ddesc(q38, **kw):
    f = dict(key_heads=2, value_heads=4, key_dim=64, value_dim=64, scale=0.125)
    f.update(kw)
    return q38.DeltaDesc(**f)


def dbatch(q38, **kw):
    f = dict(sequences=2, rows=3, max_rows=2, slots=4, row_offsets=X, origin=X, final_slots=X, checkpoints=None, states=X)
    f.update(kw)
    return q38.DeltaBatchDesc(**f)


def delta(q38, d, b, q=X, qs=512, k=X, ks=512, v=X, vs=512, g=X, beta=X, out=X, ws=X, ws_bytes=1 << 40):
    return q38.lib.q38_delta_rule(None, C.byref(d) if d else None, C.byref(b) if b else None, q, qs, k, ks, v, vs, g,
                                  beta, out, ws, ws_bytes, None)


@pytest.mark.parametrize("kw", [dict(key_heads=0), dict(value_heads=3), dict(value_heads=258), dict(key_dim=96),
                                dict(value_dim=512), dict(scale=float("nan"))])
def test_bad_delta_desc(q38, kw):
    assert delta(q38, ddesc(q38, **kw), dbatch(q38)) == q38.Q38_EINVAL
    assert "context" not in q38.last_error()


@pytest.mark.parametrize("kw", [dict(sequences=-1), dict(sequences=4097), dict(rows=-1), dict(rows=(1 << 19) + 1),
                                dict(max_rows=0), dict(max_rows=4), dict(slots=-1), dict(row_offsets=None),
                                dict(states=None), dict(states=X + 4)])
def test_bad_delta_batch(q38, kw):
    assert delta(q38, ddesc(q38), dbatch(q38, **kw)) == q38.Q38_EINVAL
    assert "context" not in q38.last_error()


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=X + 2), dict(v=None), dict(qs=120), dict(ks=130), dict(vs=248),
                                dict(g=None), dict(beta=None), dict(out=None), dict(out=X + 8)])
def test_bad_delta_operands(q38, kw):
    assert delta(q38, ddesc(q38), dbatch(q38), **kw) == q38.Q38_EINVAL
    assert "context" not in q38.last_error()


def test_delta_workspace_and_context(q38):
    d, b = ddesc(q38), dbatch(q38, rows=5000, max_rows=5000)
    need = q38.lib.q38_delta_workspace_size(C.byref(d), C.byref(b))
    if need:
        assert delta(q38, d, b, ws_bytes=need - 1) == q38.Q38_ESPACE
        assert delta(q38, d, b, ws=None) == q38.Q38_ESPACE
    assert delta(q38, d, b, ws_bytes=need) == q38.Q38_EINVAL and "null context" in q38.last_error()
    assert delta(q38, None, b) == q38.Q38_EINVAL
    assert delta(q38, d, None) == q38.Q38_EINVAL
    assert delta(q38, d, dbatch(q38, sequences=0)) == q38.Q38_OK


def test_binding_refuses_what_the_abi_cannot_see(q38):
    import torch
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32 = lambda *s: t(*s, dt=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        q38.PagedCache(None, t(4, 2, 16, 64), t(4, 2, 16, 32))
    with pytest.raises(ValueError):
        q38.PagedCache(None, t(4, 2, 16, 64, dt=torch.int8), t(4, 2, 16, 64, dt=torch.int8))
    with pytest.raises(ValueError):
        q38.PagedCache(None, t(4, 2, 16, 64, dt=torch.int8), t(4, 2, 16, 64, dt=torch.int8), t(4, 2, 16, dt=torch.float32),
                       t(4, 2, 15, dt=torch.float32))
    with pytest.raises(ValueError):
        q38.PagedBatch(i32(3), i32(3), i32(3, 4), 3, 1)
    with pytest.raises(ValueError):
        q38.PagedBatch(t(4, dt=torch.int64), i32(3), i32(3, 4), 3, 1)
    c, b = q38.PagedCache(None, t(4, 2, 16, 64), t(4, 2, 16, 64)), q38.PagedBatch(i32(4), i32(3), i32(3, 4), 3, 1)
    with pytest.raises(ValueError):
        c.append(b, t(2, 2, 64), t(3, 2, 64))
    with pytest.raises(ValueError):
        c.append(b, t(3, 2, 64).transpose(1, 2), t(3, 2, 64))
    with pytest.raises(ValueError):
        c.attend(b, t(3, 4, 64, dt=torch.float32), t(3, 4, 64), 0.1, None)
    with pytest.raises(ValueError):
        q38.DeltaBatch(t(4, 2, 64, 64), i32(3), i32(2), i32(2), 3, 1)
    with pytest.raises(ValueError):
        q38.DeltaBatch(t(4, 2, 64, 64, dt=torch.float32), i32(3), i32(3), i32(2), 3, 1)
    rule = q38.DeltaRule(None, 1, 2, 64, 64, 1.0)
    db = q38.DeltaBatch(t(4, 2, 64, 32, dt=torch.float32), i32(3), i32(2), i32(2), 3, 1)
    f = t(3, 2, dt=torch.float32)
    with pytest.raises(ValueError):
        rule.run(db, t(3, 1, 64), t(3, 1, 64), t(3, 2, 64), f, f, t(3, 2, 64), None)


def test_binding_refuses_tensors_of_another_device(q38):
    """Host tensors (here for every operand in turn) never reach a kernel: the binding refuses them before the
    library is called. A context of the host's "device" -1 stands for tensors that are where they should be."""
    import types

    import torch
    gpu, here = (types.SimpleNamespace(h=None, device=d) for d in (0, -1))
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32 = lambda *s: t(*s, dt=torch.int32)  # noqa: E731

    class Elsewhere:  # a tensor that names device 0 as its own
        def __init__(self, x):
            self.x = x

        def __getattr__(self, name):
            return getattr(self.x, name)

        def get_device(self):
            return 0

    keys = t(4, 2, 16, 64)
    with pytest.raises(ValueError, match="device"):
        q38.PagedCache(gpu, keys, keys)
    with pytest.raises(ValueError, match="device"):
        q38.PagedCache(gpu, Elsewhere(keys), keys)
    with pytest.raises(ValueError, match="device"):
        q38.PagedBatch(Elsewhere(i32(4)), i32(3), i32(3, 4), 3, 1)
    batch, cache = q38.PagedBatch(i32(4), i32(3), i32(3, 4), 3, 1), q38.PagedCache(here, keys, keys)
    ws = t(1 << 22, dt=torch.uint8)
    k, q = t(3, 2, 64), t(3, 4, 64)
    for bad in range(2):
        ops = [Elsewhere(k) if i == bad else k for i in range(2)]
        with pytest.raises(ValueError, match="device"):
            cache.append(batch, *ops)
    for bad in range(3):
        ops = [Elsewhere(x) if i == bad else x for i, x in enumerate((q, q, ws))]
        with pytest.raises(ValueError, match="device"):
            cache.attend(batch, ops[0], ops[1], 0.1, ops[2])
    moved = q38.PagedBatch(Elsewhere(i32(4)), Elsewhere(i32(3)), Elsewhere(i32(3, 4)), 3, 1)
    with pytest.raises(ValueError, match="device"):
        cache.append(moved, k, k)
    with pytest.raises(q38.Q38Error, match="null context"):  # nothing else is wrong with the call
        cache.append(batch, k, k)

    f, pool = t(3, 2, dt=torch.float32), t(4, 2, 64, 64, dt=torch.float32)
    with pytest.raises(ValueError, match="device"):
        q38.DeltaBatch(Elsewhere(pool), i32(3), i32(2), i32(2), 3, 1)
    rule, db = q38.DeltaRule(here, 1, 2, 64, 64, 1.0), q38.DeltaBatch(pool, i32(3), i32(2), i32(2), 3, 1)
    good = (t(3, 1, 64), t(3, 1, 64), t(3, 2, 64), f, f, t(3, 2, 64), ws)
    for bad in range(len(good)):
        with pytest.raises(ValueError, match="device"):
            rule.run(db, *(Elsewhere(x) if i == bad else x for i, x in enumerate(good)))
    with pytest.raises(ValueError, match="device"):
        q38.DeltaRule(gpu, 1, 2, 64, 64, 1.0).run(db, *good)
    with pytest.raises(q38.Q38Error, match="null context"):
        rule.run(db, *good)
