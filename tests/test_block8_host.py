"""Refusals of the 8-bit block-scaled cache that need no GPU: the Python
class's checks and the C ABI's, all before any launch."""

import ctypes

import pytest
import torch

from unicache_amd import _native as nat
from unicache_amd.storage import Block8KVCache


def test_cpu_tensors_fail_closed():
    key = torch.randn(1, 64, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        Block8KVCache.from_dense(key, key)
    with pytest.raises(RuntimeError, match="GPU"):
        Block8KVCache.empty(1, 64, 4, 128, device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        Block8KVCache(*_tensors())


def _tensors(s=2, h=2, n=3, b=64, d=128, code=torch.int8):
    return (torch.zeros(s, h, n * b, d, dtype=code), torch.zeros(s, h, n, d, b, dtype=code), torch.zeros(s, h, n),
            torch.zeros(s, h, n), torch.zeros(s, h, n, 2, d, dtype=torch.int8), torch.zeros(s, dtype=torch.int32))


def test_tensor_checks():
    good = list(_tensors())
    for i, bad, match in (
            (0, good[0].float(), "codes must be"), (0, good[0][:, :, :-1], "key_code"), (1, good[1][..., :48], "blocks of"),
            (1, good[1].transpose(3, 4), "blocks of|contiguous|expected"), (2, good[2].double(), "key_scale"),
            (3, good[3][:, :1], "value_scale"), (4, good[4].to(torch.uint8), "key_bounds"),
            (5, good[5].long(), "lengths"), (0, good[0][0], "expects"), (0, good[0][..., ::2], "blocks of|key_code|supports")):
        with pytest.raises(ValueError, match=match):
            Block8KVCache(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError, match="tail"):
        Block8KVCache(*good, tail=torch.zeros(2, 2, 2, 64, 128))
    with pytest.raises(ValueError, match="tail"):
        Block8KVCache(*good, tail=torch.zeros(2, 2, 2, 32, 128, dtype=torch.float16))


def test_dense_checks():
    key = torch.randn(1, 64, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="matching"):
        Block8KVCache.from_dense(key, key[:, :32])
    with pytest.raises(ValueError, match="one dtype"):
        Block8KVCache.from_dense(key, key.half())
    with pytest.raises(ValueError, match="bf16 or fp16"):
        Block8KVCache.from_dense(key.float(), key.float())
    with pytest.raises(ValueError, match="gradient"):
        Block8KVCache.from_dense(key.requires_grad_(), key)


def _cache(**kw):
    f = dict(key_code=16, value_code=16, key_scale=16, value_scale=16, key_bounds=16, lengths=16, sequences=2,
             heads_kv=4, head_dim=128, blocks=10, block_tokens=64, code_dtype=nat.UC_INT8)
    f.update(kw)
    return nat.Block8Cache(**f)


def _query(**kw):
    f = dict(query=16, q_ss=0, q_st=0, q_sh=0, query_len=2, heads_q=28, query_lengths=None, max_tokens=640,
             dtype=nat.UC_BF16, causal=0)
    f.update(kw)
    return nat.Block8Query(**f)


BAD_CACHES = [(dict(head_dim=96), "head_dim"), (dict(block_tokens=48), "block_tokens"), (dict(block_tokens=16), "block_tokens"),
              (dict(code_dtype=nat.UC_FP16), "int8 or e4m3"), (dict(sequences=0), "empty"), (dict(blocks=0), "empty"),
              (dict(heads_kv=-1), "empty"), (dict(blocks=1 << 40), "too large"), (dict(key_code=None), "NULL"),
              (dict(value_code=24), "aligned"), (dict(lengths=2), "aligned"), (dict(sequences=1 << 23), "too many")]


@pytest.mark.parametrize("fields,match", BAD_CACHES)
def test_cache_validation(fields, match):
    c, q = _cache(**fields), _query()
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_pack", c, 16, 0, 0, 0, 16, 0, 0, 0, nat.UC_BF16, 64, None, None, None)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_append", c, 16, 16, 0, 0, 0, 16, 0, 0, 0, nat.UC_BF16, 1, None, None)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_dequant", c, 16, 16, nat.UC_BF16, 64, None)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_attn", c, q, None, 0, 0, 0.1, 16, None, 16, 1 << 40, None)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_select", c, q, 4, 1, 1, 1, 16, 16, 1 << 40, None)
    assert nat.lib().uc_block8_attn_workspace_bytes(c, q, 0, 0) == -1
    assert nat.lib().uc_block8_select_workspace_bytes(c, q, 1) == -1


def test_row_validation():
    c = _cache()
    for bad in ((8, 0, 0, 0), (None, 0, 0, 0), (16, 4, 0, 0), (16, 0, 12, 0), (16, 0, 0, 1)):
        with pytest.raises(ValueError, match="16-byte aligned"):
            nat.call("uc_block8_pack", c, *bad, 16, 0, 0, 0, nat.UC_BF16, 64, None, None, None)
        with pytest.raises(ValueError, match="16-byte aligned"):
            nat.call("uc_block8_append", c, 16, 16, 0, 0, 0, *bad, nat.UC_BF16, 64, None, None)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        nat.call("uc_block8_pack", c, 16, 0, 0, 0, 16, 0, 0, 0, nat.UC_FP32, 64, None, None, None)
    with pytest.raises(ValueError, match="capacity"):
        nat.call("uc_block8_pack", c, 16, 0, 0, 0, 16, 0, 0, 0, nat.UC_BF16, 641, None, None, None)
    with pytest.raises(ValueError, match="capacity"):
        nat.call("uc_block8_dequant", c, 16, 16, nat.UC_BF16, 641, None)
    with pytest.raises(ValueError, match="tail"):
        nat.call("uc_block8_append", c, None, 16, 0, 0, 0, 16, 0, 0, 0, nat.UC_BF16, 1, None, None)
    with pytest.raises(ValueError, match="outputs"):
        nat.call("uc_block8_dequant", c, 16, 24, nat.UC_BF16, 64, None)
    nat.call("uc_block8_pack", c, None, 0, 0, 0, None, 0, 0, 0, nat.UC_BF16, 0, None, None, None)  # nothing to do


BAD_QUERIES = [(dict(dtype=nat.UC_FP32), "bf16 or fp16"), (dict(heads_q=30), "multiple of KV heads"), (dict(heads_q=0), "multiple"),
               (dict(query_len=-1), "query_len"), (dict(query_len=1 << 30), "query_len"), (dict(max_tokens=-1), "max_tokens")]


@pytest.mark.parametrize("fields,match", BAD_QUERIES)
def test_query_validation(fields, match):
    c, q = _cache(), _query(**fields)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_attn", c, q, None, 0, 0, 0.1, 16, None, 16, 1 << 40, None)
    with pytest.raises(ValueError, match=match):
        nat.call("uc_block8_select", c, q, 4, 1, 1, 1, 16, 16, 1 << 40, None)


def test_attention_and_selection_validation():
    c = _cache()
    for q, match in ((_query(query=8), "aligned"), (_query(q_st=4), "aligned")):
        with pytest.raises(ValueError, match=match):
            nat.call("uc_block8_attn", c, q, None, 0, 0, 0.1, 16, None, 16, 1 << 40, None)
        with pytest.raises(ValueError, match=match):
            nat.call("uc_block8_select", c, q, 4, 1, 1, 1, 16, 16, 1 << 40, None)
    q = _query()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="sm_scale"):
            nat.call("uc_block8_attn", c, q, None, 0, 0, scale, 16, None, 16, 1 << 40, None)
    with pytest.raises(ValueError, match="belong together"):
        nat.call("uc_block8_attn", c, q, 16, 0, 1, 0.1, 16, None, 16, 1 << 40, None)
    with pytest.raises(ValueError, match="belong together"):
        nat.call("uc_block8_attn", c, q, None, 4, 1, 0.1, 16, None, 16, 1 << 40, None)
    with pytest.raises(ValueError, match="query_block"):
        nat.call("uc_block8_attn", c, q, 16, 4, 0, 0.1, 16, None, 16, 1 << 40, None)
    with pytest.raises(ValueError, match="out must be"):
        nat.call("uc_block8_attn", c, q, None, 0, 0, 0.1, 8, None, 16, 1 << 40, None)
    need = nat.lib().uc_block8_attn_workspace_bytes(c, q, 0, 0)
    assert need > 0
    with pytest.raises(ValueError, match="workspace"):
        nat.call("uc_block8_attn", c, q, None, 0, 0, 0.1, 16, None, 16, need - 1, None)
    need = nat.lib().uc_block8_select_workspace_bytes(c, q, 1)
    with pytest.raises(ValueError, match="workspace"):
        nat.call("uc_block8_select", c, q, 4, 1, 1, 1, 16, 16, need - 1, None)
    for budget, sink, recent, block, match in ((0, 1, 1, 1, "budget"), (4, -1, 1, 1, "sink"), (4, 1, 0, 1, "recent"),
                                               (4, 1, 1, 0, "query_block"), (4, 2, 3, 1, "always chosen")):
        with pytest.raises(ValueError, match=match):
            nat.call("uc_block8_select", c, q, budget, sink, recent, block, 16, 16, 1 << 40, None)
    causal = _query(causal=1, query_len=200)  # 200 queries cover up to 1 + ceil(199 / 64) blocks
    with pytest.raises(ValueError, match="6 blocks always chosen"):
        nat.call("uc_block8_select", c, causal, 5, 1, 1, 200, 16, 16, 1 << 40, None)
    with pytest.raises(ValueError, match="NULL"):
        nat.call("uc_block8_attn", c, None, None, 0, 0, 0.1, 16, None, 16, 1 << 40, None)
    assert ctypes.sizeof(nat.Block8Cache) == 88 and ctypes.sizeof(nat.Block8Query) == 72


def test_launches_that_are_too_large():
    many = _query(query_len=1 << 21, heads_q=4)  # 2 x 4 x 2^21 runs of one query, a workgroup each
    with pytest.raises(ValueError, match="too many query rows"):
        nat.call("uc_block8_select", _cache(), many, 4, 1, 1, 1, 16, 16, 1 << 50, None)
    with pytest.raises(ValueError, match="too many query rows"):
        nat.call("uc_block8_attn", _cache(), many, 16, 4, 1, 0.1, 16, None, 16, 1 << 50, None)
    # 2^28 rows of 16 lanes
    with pytest.raises(ValueError, match="too many query rows"):
        nat.call("uc_block8_select", _cache(heads_kv=16), _query(query_len=1 << 23, heads_q=16), 4, 1, 1, 1 << 23, 16, 16,
                 1 << 50, None)
    # one workgroup of 128 rows a head, and each head's dealt to eight XCDs
    with pytest.raises(ValueError, match="too many query rows"):
        nat.call("uc_block8_attn", _cache(sequences=(1 << 22) - 1, heads_kv=1), _query(query_len=64, heads_q=2), None, 0,
                 0, 0.1, 16, None, 16, 1 << 50, None)
    with pytest.raises(ValueError, match="budget"):
        nat.call("uc_block8_attn", _cache(), _query(), 16, (1 << 24) + 1, 1, 0.1, 16, None, 16, 1 << 50, None)
    with pytest.raises(ValueError, match="budget"):
        nat.call("uc_block8_select", _cache(), _query(), (1 << 24) + 1, 1, 1, 1, 16, 16, 1 << 50, None)
    with pytest.raises(ValueError, match="too many keys"):
        nat.call("uc_block8_attn", _cache(), _query(query_len=100), 16, 1 << 24, 1, 0.1, 16, None, 16, 1 << 50, None)
    with pytest.raises(ValueError, match="too many rows"):  # 2^13 x 8 x 257 workgroups
        nat.call("uc_block8_append", _cache(sequences=1 << 13, heads_kv=8, blocks=300), 16, 16, 0, 0, 0, 16, 0, 0, 0,
                 nat.UC_BF16, 1 << 14, None, None)


def test_decode_selection_asks_for_scores_where_it_keeps_them_in_memory():
    need = nat.lib().uc_block8_select_workspace_bytes
    one = _query(query_len=1)
    assert need(_cache(blocks=512), one, 1) == 256
    for sequences, blocks in ((2, 513), (32, 513), (33, 8193)):  # 8, 128 and 132 runs
        assert need(_cache(sequences=sequences, blocks=blocks), one, 1) >= sequences * 4 * blocks * 4
    assert need(_cache(sequences=33, blocks=8192), one, 1) == 256


@pytest.mark.parametrize("sink,recent", [(1 << 62, 1 << 62), ((1 << 62) + 100, (1 << 62) + 100), ((1 << 63) - 1, 1),
                                         (1, (1 << 63) - 1), (5, 1), (0, 5)])
def test_always_chosen_blocks_whose_sum_passes_64_bits(sink, recent):
    with pytest.raises(ValueError, match="always chosen"):
        nat.call("uc_block8_select", _cache(), _query(), 4, sink, recent, 1, 16, 16, 1 << 40, None)


def _cpu_cache(monkeypatch):
    """A cache object over CPU tensors, and the calls that it would make."""

    tensors = _tensors()
    cache = Block8KVCache.__new__(Block8KVCache)
    cache._set(*tensors, None, (2, 2, 128, 3, 64), None)
    calls = []
    monkeypatch.setattr(cache, "_call", lambda entry, *args: calls.append((entry, args)))
    return cache, calls


def test_sparse_attention_numbers_that_do_not_fit_the_c_types(monkeypatch):
    # ctypes cuts whole numbers to 64 bits without a word
    cache, calls = _cpu_cache(monkeypatch)
    q = torch.randn(2, 10, 4, 128, dtype=torch.bfloat16)
    for kw in (dict(budget=(1 << 64) + 5), dict(budget=1 << 40), dict(budget=(1 << 24) + 1), dict(budget=4, sink=1 << 64),
               dict(budget=4, sink=-1), dict(budget=4, recent=(1 << 64) + 1), dict(budget=4, recent=0)):
        with pytest.raises(ValueError):
            cache.sparse_attention(q, **kw)
    assert not calls
    for block in (10, 11, (1 << 64) + 3):
        _, _, blocks = cache.sparse_attention(q, budget=4, query_block=block)
        assert blocks.shape == (2, 1, 2, 4)
    assert [c[1][5] for c in calls if c[0] == "uc_block8_select"] == [10] * 3
    assert [c[1][4] for c in calls if c[0] == "uc_block8_attn"] == [10] * 3
    cache.sparse_attention(q[:, :0], budget=4, query_block=1 << 64)


@pytest.mark.parametrize("heads,lq", [(1 << 62, 4), (1 << 61, 8), (1 << 32, 1 << 20), (1 << 34, 0)])
def test_query_heads_whose_rows_pass_64_bits(heads, lq):
    # heads_q x query_len is 2^64: as a 64-bit number no row at all
    q = _query(heads_q=heads, query_len=lq)
    with pytest.raises(ValueError, match="query heads|query rows"):
        nat.call("uc_block8_attn", _cache(), q, None, 0, 0, 0.1, 16, None, 16, 1 << 50, None)
    with pytest.raises(ValueError, match="query heads|query rows"):
        nat.call("uc_block8_select", _cache(), q, 4, 1, 1, 1, 16, 16, 1 << 50, None)
    assert nat.lib().uc_block8_attn_workspace_bytes(_cache(), q, 0, 0) == -1
    assert nat.lib().uc_block8_select_workspace_bytes(_cache(), q, 1) == -1


@pytest.mark.parametrize("scale", [3e38, 2.4e38, 1e39, 1e-46, 0.0, -1.0, float("nan"), float("inf")])
def test_logit_scales_that_fp32_does_not_hold(monkeypatch, scale):
    # times log2(e), as the kernels take them; before any launch
    with pytest.raises(ValueError, match="sm_scale"):
        nat.call("uc_block8_attn", _cache(), _query(), None, 0, 0, scale, 16, None, 16, 1 << 40, None)
    cache, calls = _cpu_cache(monkeypatch)
    q = torch.randn(2, 3, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="sm_scale"):
        cache.attention(q, sm_scale=scale)
    with pytest.raises(ValueError, match="sm_scale"):
        cache.sparse_attention(q, budget=3, sm_scale=scale)
    assert not calls


def test_tracked_tensors_are_refused(monkeypatch):
    # by autograd or by forward mode: a gradient would be lost without a word
    from torch.autograd import forward_ad

    dense = torch.randn(2, 64, 2, 128, dtype=torch.bfloat16)
    q = torch.randn(2, 3, 4, 128, dtype=torch.bfloat16)
    cache, calls = _cpu_cache(monkeypatch)
    cache.tail = torch.zeros(2, 2, 2, 64, 128, dtype=torch.bfloat16)

    def refuses(track):
        for call in (lambda t: Block8KVCache.from_dense(t, dense), lambda t: Block8KVCache.from_dense(dense, t),
                     lambda t: cache.append(t, dense), lambda t: cache.append(dense, t)):
            with pytest.raises(ValueError, match="gradient"):
                call(track(dense))
        for call in (cache.attention, lambda t: cache.sparse_attention(t, budget=3)):
            with pytest.raises(ValueError, match="gradient"):
                call(track(q))
        for i in (2, 3):  # another program's scales
            tensors = list(_tensors())
            tensors[i] = track(tensors[i])
            with pytest.raises(ValueError, match="gradient"):
                Block8KVCache(*tensors)
        with pytest.raises(ValueError, match="gradient"):
            Block8KVCache(*_tensors(), tail=track(cache.tail))

    refuses(lambda t: t.clone().requires_grad_())
    with forward_ad.dual_level():
        refuses(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        cache.attention(q)  # no tangent of its own
    with torch.no_grad():
        cache.attention(q.clone().requires_grad_())
    assert [c[0] for c in calls] == ["uc_block8_attn"] * 2
