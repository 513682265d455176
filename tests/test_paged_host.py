"""Refusals of the paged cache and of rotary positions that need no GPU: the
Python classes' checks and the C ABI's, all before any launch."""

import ctypes
import math

import pytest
import torch

from unicache_amd import _native as nat
from unicache_amd.operators import MultiAxisRotary
from unicache_amd.storage import PagedKVCache


def _tensors(layers=2, pages=5, h=2, b=64, d=128, s=3, m=4, dtype=torch.bfloat16):
    return (torch.zeros(layers, pages, h, b, d, dtype=dtype), torch.zeros(layers, pages, h, b, d, dtype=dtype),
            torch.full((s, m), -1, dtype=torch.int32), torch.zeros(s, dtype=torch.int32))


def _books(pages=5, s=3):
    return dict(granted=torch.zeros(s, dtype=torch.int32), references=torch.zeros(pages, dtype=torch.int32),
                free_pages=torch.zeros(-(-pages // 32), dtype=torch.int32))


def _on_host(**kw):
    """A cache of CPU tensors, which the constructor refuses: calls on it must be refused before they launch."""

    cache = PagedKVCache.__new__(PagedKVCache)
    key, value, table, lengths = _tensors(**kw)
    books = _books(key.shape[1], table.shape[0])
    cache._set(key, value, table, lengths, books["granted"], books["references"], books["free_pages"], None)
    return cache


def test_cpu_tensors_fail_closed():
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKVCache(*_tensors())
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKVCache.empty(1, 4, 2, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        MultiAxisRotary(64, (32,), device="cpu")


def test_tensor_checks():
    good = list(_tensors())
    for i, bad, match in (
            (0, good[0].float(), "bf16 or fp16"), (0, good[0][0], "layers, pages"), (0, good[0][..., :96], "head_dim"),
            (0, good[0][:, :, :, :48], "pages of"), (0, good[0].transpose(2, 3), "pages of|contiguous"),
            (1, good[1][:, :4], "value"), (1, good[1].half(), "value"), (2, good[2].long(), "table"),
            (2, good[2][0], "table"), (2, good[2][:, ::2], "table"), (3, good[3][:2], "lengths"),
            (3, good[3].long(), "lengths"), (2, good[2][:, :0], "a page per sequence"), (0, good[0][:0], "needs a layer")):
        with pytest.raises(ValueError, match=match):
            PagedKVCache(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError, match="gradient"):
        PagedKVCache(good[0].clone().requires_grad_(), *good[1:])
    books = _books()
    for name, bad in (("granted", None), ("references", None), ("free_pages", None)):
        with pytest.raises(ValueError, match="belong together"):
            PagedKVCache(*good, **{**books, name: bad})
    for name, bad in (("granted", books["granted"][:2]), ("references", books["references"].long()),
                      ("free_pages", torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match=name):
            PagedKVCache(*good, **{**books, name: bad})


def test_empty_checks():
    for args, kw, match in (((0, 4, 2, 64), {}, "needs a layer"), ((1, 0, 2, 64), {}, "needs a layer"),
                            ((1, 4, 0, 64), {}, "needs a layer"), ((1, 4, 2, 96), {}, "head_dim"),
                            ((1, 4, 2, 64), dict(page_tokens=8), "pages of"), ((1, 4, 2, 64), dict(layers=0), "needs a layer"),
                            ((1, 4, 2, 64), dict(sequence_pages=0), "needs a layer"),
                            ((1, 4, 2, 64), dict(dtype=torch.float32), "bf16 or fp16")):
        with pytest.raises(ValueError, match=match):
            PagedKVCache.empty(*args, **kw)


def test_call_checks():
    cache = _on_host()
    rows = torch.zeros(3, 2, 2, 128, dtype=torch.bfloat16)
    q = torch.zeros(3, 2, 4, 128, dtype=torch.bfloat16)
    for call, match in (
            (lambda: cache.reserve(-1), "negative"), (lambda: cache.reserve(1 << 30), "2\\^30"),
            (lambda: cache.reserve(1, counts=torch.zeros(3)), "counts"),
            (lambda: cache.reserve(1, counts=torch.zeros(2, dtype=torch.int32)), "counts"),
            (lambda: cache.reorder(torch.zeros(3, dtype=torch.int64)), "parents"),
            (lambda: cache.reorder(torch.zeros(3, dtype=torch.int32), lengths=torch.zeros(4, dtype=torch.int32)), "lengths"),
            (lambda: cache.truncate(torch.zeros(6, dtype=torch.int32)[::2]), "lengths"),
            (lambda: cache.compact(torch.zeros(3, 8)), "keep"), (lambda: cache.compact(torch.zeros(2, 8, dtype=torch.bool)), "keep"),
            (lambda: cache.compact(torch.zeros(3, dtype=torch.bool)), "keep"),
            (lambda: cache.write(rows, rows[:, :1]), "one shape"), (lambda: cache.write(rows.half(), rows), "dtype"),
            (lambda: cache.write(rows[:2], rows[:2]), "keys"), (lambda: cache.write(rows, q), "values"),
            (lambda: cache.write(rows, rows, layer=2), "layers 0"), (lambda: cache.write(rows, rows, layer=-1), "layers 0"),
            (lambda: cache.write(rows, rows, query=q), "rotary"),
            (lambda: cache.write(rows, rows, positions=torch.zeros(1, 3, 2, dtype=torch.int32)), "rotary"),
            (lambda: cache.write(rows, rows, counts=torch.zeros(3, dtype=torch.int64)), "counts"),
            (lambda: cache.write(rows.clone().requires_grad_(), rows), "gradient"),
            (lambda: cache.attention(q[..., :64]), "queries"), (lambda: cache.attention(q[0]), "queries"),
            (lambda: cache.attention(q[:, :, :3]), "divisible"), (lambda: cache.attention(q.half()), "dtype"),
            (lambda: cache.attention(q.float()), "dtype"), (lambda: cache.attention(q[:, :, :0]), "queries"),
            (lambda: cache.attention(q, layer=5), "layers 0"), (lambda: cache.attention(q, sm_scale=0.0), "sm_scale"),
            (lambda: cache.attention(q, sm_scale=-1.0), "sm_scale"), (lambda: cache.attention(q, sm_scale=math.nan), "sm_scale"),
            (lambda: cache.attention(q, sm_scale=math.inf), "sm_scale"), (lambda: cache.attention(q, sm_scale=1e-39), "sm_scale"),
            (lambda: cache.attention(q, query_lengths=torch.zeros(3)), "query_lengths"),
            (lambda: cache.attention(q.clone().requires_grad_()), "gradient"), (lambda: cache.dense(layer=2), "layers 0"),
            (lambda: cache.layer(2), "layers 0"), (lambda: cache.layer(0, sequence=3), "sequences 0"),
            (lambda: cache.layer(0, sequence=-1), "sequences 0")):
        with pytest.raises(ValueError, match=match):
            call()
    view = cache.layer(1)
    numbers = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: view.reserve(1), lambda: view.reorder(numbers), lambda: view.truncate(numbers),
                 lambda: view.compact(torch.zeros(3, 8, dtype=torch.bool))):
        with pytest.raises(RuntimeError, match="references"):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, q)
        with pytest.raises(ValueError, match="forward-mode"):
            cache.attention(dual)


def test_rotary_checks():
    for args, kw, match in (
            ((64, ()), {}, "an axis"), ((64, (-8, 16)), {}, "negative"), ((64, (4,)), {}, "multiple of 8"),
            ((64, (40,)), {}, "half of head_dim"), ((60, (16,)), {}, "head_dim"), ((528, (16,)), {}, "head_dim"),
            ((0, (8,)), {}, "head_dim"), ((64, (32,)), dict(pairing="both"), "pairing"),
            ((64, (16, 16)), dict(axes=[0] * 32), "axes"), ((64, (16, 16)), dict(axes=[0, 1]), "axes"),
            ((64, (16, 16)), dict(axes=[0] * 15 + [1] * 16 + [2]), "axes"),
            ((64, (32,)), dict(theta=0.0), "theta"), ((64, (32,)), dict(theta=math.nan), "theta"),
            ((64, (32,)), dict(frequencies=[1.0]), "frequencies"),
            ((64, (32,)), dict(frequencies=[math.inf] * 32), "frequencies")):
        with pytest.raises(ValueError, match=match):
            MultiAxisRotary(*args, **kw)
    rotary = _rotary()
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    positions = torch.zeros(2, 2, 3, dtype=torch.int64)
    for call, match in (
            (lambda: rotary.rotate(q.float(), positions=positions), "bf16 or fp16"),
            (lambda: rotary.rotate(q[..., :32], positions=positions), "expected"),
            (lambda: rotary.rotate(q, q[:, :2], positions=positions), "expected"),
            (lambda: rotary.rotate(q, q.half(), positions=positions), "one dtype"),
            (lambda: rotary.rotate(q[:, :, :0], positions=positions), "expected"),
            (lambda: rotary.rotate(q[0, 0], positions=positions), "expected"),
            (lambda: rotary.rotate(q, positions=None), "need positions"),
            (lambda: rotary.rotate(q.clone().requires_grad_(), positions=positions), "gradient"),
            (lambda: rotary.plan(positions.float(), 2, 3), "int32 or int64"),
            (lambda: rotary.plan(positions[:1], 2, 3), "positions must be"),
            (lambda: rotary.plan(positions[:, 0], 2, 3), "positions must be"),
            (lambda: rotary.plan(positions, 2, 4), "positions must be")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.rotate(q, positions=positions)
    cache = _on_host(d=128)
    rows = torch.zeros(3, 2, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="head_dim 64"):
        cache.write(rows, rows, rotary=rotary)
    cache = _on_host(d=64)
    rows = torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="as many queries"):
        cache.write(rows, rows, rotary=rotary, query=rows[:, :1])
    with pytest.raises(ValueError, match="positions must be"):
        cache.write(rows, rows, rotary=rotary, positions=positions)


def _rotary():
    rotary = MultiAxisRotary.__new__(MultiAxisRotary)
    rotary.head_dim, rotary.pairs, rotary.num_axes, rotary.pairing = 64, 32, 2, "halves"
    rotary._turns, rotary._axis = torch.zeros(32, dtype=torch.float64), torch.zeros(32, dtype=torch.int32)
    rotary._tables, rotary._adjacent = (16, 16), 0
    rotary.device = rotary._turns.device
    return rotary


# --------------------------------------------------------------------- ABI --
def _cache(**kw):
    f = dict(key=16, value=16, table=16, lengths=16, granted=16, references=16, free_pages=16, layers=2, pages=100,
             sequences=3, sequence_pages=10, heads_kv=4, head_dim=128, page_tokens=64, dtype=nat.UC_BF16)
    f.update(kw)
    return nat.PagedCache(**f)


def _query(**kw):
    f = dict(query=16, q_ss=0, q_st=0, q_sh=0, query_len=2, heads_q=28, query_lengths=None, max_tokens=640,
             dtype=nat.UC_BF16, causal=0)
    f.update(kw)
    return nat.Block8Query(**f)


def _plan(**kw):
    f = dict(turns=16, axis=16, positions=16, axes=3, pairs=64, position_bytes=8, adjacent=0, inverse=0, reserved=0)
    f.update(kw)
    return nat.RotaryPlan(**f)


BIG = 1 << 50


def _calls(c, layer=0):
    return [
        lambda: nat.call("uc_paged_attn", c, layer, _query(), 0.1, 16, None, 16, BIG, None),
        lambda: nat.call("uc_paged_write", c, layer, 16, 0, 0, 0, 16, 0, 0, 0, 1, None, None, None, 0, 0, 0, 0, None, None),
        lambda: nat.call("uc_paged_dense", c, layer, 16, 16, 1, None),
        lambda: nat.call("uc_paged_reserve", c, 1, None, None),
        lambda: nat.call("uc_paged_reorder", c, None, None, 640, 16, BIG, None),
        lambda: nat.call("uc_paged_compact", c, 16, 0, 1, 640, 16, BIG, None),
    ]


@pytest.mark.parametrize("fields,match", [
    (dict(dtype=nat.UC_FP32), "bf16 or fp16"), (dict(head_dim=96), "head_dim"), (dict(page_tokens=8), "pages must have"),
    (dict(page_tokens=48), "pages must have"), (dict(sequences=0), "sequences"), (dict(sequences=4097), "sequences"),
    (dict(layers=0), "layer"), (dict(pages=0), "number of pages"), (dict(pages=1 << 30), "number of pages"),
    (dict(sequence_pages=0), "per sequence"), (dict(sequence_pages=(1 << 24) + 1), "per sequence"),
    (dict(sequences=4096, sequence_pages=1 << 18, page_tokens=16), "table is too large"),
    (dict(heads_kv=0), "KV heads"), (dict(heads_kv=1 << 20), "KV heads"), (dict(key=None), "aligned"),
    (dict(value=24), "aligned"), (dict(table=None), "aligned"), (dict(lengths=18), "aligned"),
    (dict(granted=None), "belong together"), (dict(references=2), "belong together"), (dict(free_pages=None), "belong together"),
    (dict(pages=(1 << 30) - 1, layers=(1 << 20) - 1, heads_kv=4096), "too large"),
])
def test_cache_validation(fields, match):
    c = _cache(**fields)
    for call in _calls(c):
        with pytest.raises(ValueError, match=match):
            call()
    lib = nat.lib()
    assert lib.uc_paged_attn_workspace_bytes(c, _query()) == -1
    assert lib.uc_paged_reorder_workspace_bytes(c) == -1 and lib.uc_paged_compact_workspace_bytes(c) == -1


def test_layers_and_pools():
    for layer in (-1, 2):
        for call in _calls(_cache(), layer)[:3]:
            with pytest.raises(ValueError, match="layer"):
                call()
    bare = _cache(granted=None, references=None, free_pages=None)
    for call in _calls(bare)[3:]:
        with pytest.raises(ValueError, match="no references"):
            call()
    with pytest.raises(ValueError, match="cache is NULL"):
        nat.call("uc_paged_reserve", None, 1, None, None)


@pytest.mark.parametrize("fields,match", [
    (dict(dtype=nat.UC_FP16), "the cache's dtype"), (dict(heads_q=30), "multiple of KV heads"), (dict(heads_q=0), "multiple"),
    (dict(query_len=-1), "query_len"), (dict(query_len=1 << 24), "query_len"), (dict(max_tokens=-1), "max_tokens"),
    (dict(query_len=(1 << 24) - 1), "too many query rows"), (dict(query=None), "16-byte aligned"), (dict(query=8), "16-byte aligned"),
    (dict(q_ss=4), "multiples of 8"), (dict(q_st=7), "multiples of 8"), (dict(q_sh=1), "multiples of 8"),
])
def test_query_validation(fields, match):
    with pytest.raises(ValueError, match=match):
        nat.call("uc_paged_attn", _cache(), 0, _query(**fields), 0.1, 16, None, 16, BIG, None)


def test_attention_validation():
    c, q = _cache(), _query()
    need = nat.lib().uc_paged_attn_workspace_bytes(c, q)
    assert need > 0
    for args, match in (((0.0, 16, None, 16, need), "sm_scale"), ((float("nan"), 16, None, 16, need), "sm_scale"),
                        ((float("inf"), 16, None, 16, need), "sm_scale"), ((0.1, None, None, 16, need), "out"),
                        ((0.1, 24, None, 16, need), "out"), ((0.1, 16, None, 16, need - 1), "workspace"),
                        ((0.1, 16, None, None, need), "workspace"), ((0.1, 16, None, 8, need), "workspace")):
        with pytest.raises(ValueError, match=match):
            nat.call("uc_paged_attn", c, 0, q, *args, None)
    with pytest.raises(ValueError, match="query is NULL"):
        nat.call("uc_paged_attn", c, 0, None, 0.1, 16, None, 16, need, None)
    # no queries: nothing to do
    nat.call("uc_paged_attn", c, 0, _query(query_len=0, query=None), 0.1, None, None, None, 0, None)
    assert nat.lib().uc_paged_attn_workspace_bytes(c, _query(query_len=0)) == 0


@pytest.mark.parametrize("fields,match", [
    (dict(turns=None), "turns and axes"), (dict(axis=None), "turns and axes"), (dict(pairs=0), "multiple of 8"),
    (dict(pairs=12), "multiple of 8"), (dict(pairs=72), "multiple of 8"), (dict(axes=0), "axes"), (dict(axes=1 << 16), "axes"),
    (dict(position_bytes=2), "4 or 8 bytes"),
])
def test_plan_validation(fields, match):
    p = _plan(**fields)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_rotary", ctypes.byref(p), 2, 3, 128, nat.UC_BF16, 16, 0, 0, 0, 4, 16, None, 0, 0, 0, 0, None, None)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_paged_write", _cache(), 0, 16, 0, 0, 0, 16, 0, 0, 0, 1, None, ctypes.byref(p), None, 0, 0, 0, 0, None,
                 None)


def test_rotary_and_write_validation():
    p = ctypes.byref(_plan())
    good = dict(plan=p, s=2, n=3, d=128, dtype=nat.UC_BF16, q=(16, 0, 0, 0, 4, 16), k=(16, 0, 0, 0, 2, 16))
    for change, match in ((dict(plan=None), "plan is NULL"), (dict(dtype=nat.UC_FP32), "bf16 or fp16"), (dict(d=120), "head_dim"),
                          (dict(d=1024), "head_dim"), (dict(q=(16, 0, 0, 0, 0, 16)), "number of heads"),
                          (dict(k=(16, 0, 0, 0, -1, 16)), "number of heads"), (dict(s=1 << 23), "too many rows"),
                          (dict(n=-1), "too many rows"), (dict(q=(8, 0, 0, 0, 4, 16)), "query must be"),
                          (dict(q=(16, 1, 0, 0, 4, 16)), "query must be"), (dict(q=(16, 0, 0, 0, 4, None)), "out must be"),
                          (dict(k=(None, 0, 0, 0, 2, 16)), "key must be"), (dict(k=(16, 0, 0, 0, 2, 8)), "out must be"),
                          (dict(q=(16, 0, 0, 0, 1 << 20, 16)), "too many heads"),
                          (dict(plan=ctypes.byref(_plan(positions=None))), "positions are NULL")):
        a = {**good, **change}
        with pytest.raises(ValueError, match=match):
            nat.call("uc_rotary", a["plan"], a["s"], a["n"], a["d"], a["dtype"], *a["q"], *a["k"], None)
    c = _cache()
    base = dict(k=(16, 0, 0, 0), v=(16, 0, 0, 0), n=3, plan=p, q=(16, 0, 0, 0, 4, 16))
    for change, match in ((dict(k=(8, 0, 0, 0)), "key must be"), (dict(v=(16, 0, 4, 0)), "value must be"),
                          (dict(q=(24, 0, 0, 0, 4, 16)), "query must be"), (dict(q=(16, 0, 0, 0, 4, None)), "out must be"),
                          (dict(plan=None), "without a plan"), (dict(q=(16, 0, 0, 0, 0, 16)), "query heads"),
                          (dict(n=-1), "too many rows"), (dict(n=1 << 24), "too many rows")):
        a = {**base, **change}
        with pytest.raises(ValueError, match=match):
            nat.call("uc_paged_write", c, 0, *a["k"], *a["v"], a["n"], None, a["plan"], *a["q"], None)
    # no rows: nothing to do
    nat.call("uc_paged_write", c, 0, None, 0, 0, 0, None, 0, 0, 0, 0, None, None, None, 0, 0, 0, 0, None, None)


def test_page_call_validation():
    c = _cache()
    lib = nat.lib()
    for entry, args in (("uc_paged_reorder", (None, None, 640)), ("uc_paged_compact", (16, 0, 1, 640))):
        need = getattr(lib, entry + "_workspace_bytes")(c)
        assert need > 0 and need % 16 == 0
        with pytest.raises(ValueError, match="max_tokens"):
            nat.call(entry, c, *args[:-1], -1, 16, need, None)
        for ws, size in ((16, need - 1), (None, need), (8, need)):
            with pytest.raises(ValueError, match="workspace"):
                nat.call(entry, c, *args, ws, size, None)
    for tokens in (-1, 1 << 30):
        with pytest.raises(ValueError, match="number of tokens"):
            nat.call("uc_paged_reserve", c, tokens, None, None)
        with pytest.raises(ValueError, match="number of tokens"):
            nat.call("uc_paged_compact", c, 16, 0, tokens, 640, 16, BIG, None)
    with pytest.raises(ValueError, match="keep is NULL"):
        nat.call("uc_paged_compact", c, None, 0, 5, 640, 16, BIG, None)
    with pytest.raises(ValueError, match="number of tokens"):
        nat.call("uc_paged_dense", c, 0, 16, 16, 641, None)
    with pytest.raises(ValueError, match="aligned"):
        nat.call("uc_paged_dense", c, 0, 16, 24, 640, None)
    nat.call("uc_paged_dense", c, 0, None, None, 0, None)


# -------------------------------------------------------- tensors that change --
_NAMES = ("key", "value", "table", "lengths", "granted", "references", "free_pages")


def _built(monkeypatch):
    """A cache of CPU tensors whose C struct stands."""

    cache = _on_host()
    with monkeypatch.context() as m:
        m.setattr(PagedKVCache, "_check", staticmethod(lambda *tensors: None))
        cache._struct()
    return cache


@pytest.mark.parametrize("name", _NAMES)
@pytest.mark.parametrize("how", ["data", "set"])
def test_the_struct_follows_storage_that_was_swapped(monkeypatch, name, how):
    cache = _built(monkeypatch)
    t = getattr(cache, name)
    old = t.detach()  # (keeps the first memory, so that the addresses differ)
    if how == "data":
        t.data = t.clone()
    else:
        t.set_(t.clone())
    monkeypatch.setattr(PagedKVCache, "_check", staticmethod(lambda *tensors: None))
    assert {n: getattr(cache._struct(True), n) for n in _NAMES} == {n: getattr(cache, n).data_ptr() for n in _NAMES}
    del old


def test_swapped_storage_is_checked(monkeypatch):
    # (attention and writes do without the last three)
    for name, bad in (("key", lambda t: t.half()), ("value", lambda t: t[:, :2].contiguous()), ("table", lambda t: t.long()),
                      ("lengths", lambda t: torch.zeros(9, dtype=torch.int32)), ("references", lambda t: t[:2].clone())):
        cache = _built(monkeypatch)
        t = getattr(cache, name)
        old, t.data = t.detach(), bad(t)
        with pytest.raises(ValueError, match="Paged cache"):
            cache._struct(True)
        del old


def test_a_used_cache_is_copied_with_its_addresses_made_anew(monkeypatch):
    import copy
    import pickle

    cache = _built(monkeypatch)
    monkeypatch.setattr(PagedKVCache, "_check", staticmethod(lambda *tensors: None))
    for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert other.key.data_ptr() != cache.key.data_ptr() and torch.equal(other.table, cache.table)
        assert {n: getattr(other._struct(True), n) for n in _NAMES} == {n: getattr(other, n).data_ptr() for n in _NAMES}


def test_a_plan_follows_its_tables():
    import copy
    import pickle

    rotary = _rotary()
    positions = torch.zeros(2, 1, 3, dtype=torch.int64)
    for other in (rotary, copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary))):
        struct, _ = other.plan(positions, 1, 3)
        assert struct.turns == other._turns.data_ptr() and struct.axis == other._axis.data_ptr()


def test_tensors_that_came_to_track_a_gradient(monkeypatch):
    # under no_grad, or after the cache was made
    for name in ("key", "value"):
        cache = _built(monkeypatch)
        getattr(cache, name).requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            cache._struct()
        with torch.no_grad():
            cache._struct()


def test_a_replaced_tensor_is_let_go(monkeypatch):
    import gc
    import weakref

    for name in _NAMES:
        cache = _built(monkeypatch)
        old = weakref.ref(getattr(cache, name))
        setattr(cache, name, getattr(cache, name).clone())
        gc.collect()
        assert old() is None


def test_dense_tokens():
    cache = _on_host()
    for tokens in (-1, cache.capacity + 1):
        with pytest.raises(ValueError, match="tokens must be 0 .. 256"):
            cache.dense(tokens=tokens)
