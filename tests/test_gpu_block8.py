"""The 8-bit block-scaled KV cache (Block8KVCache) against 64-bit arithmetic:
codes, scales and bounds exactly, attention within the roundings it makes,
block selection exactly."""

import math

import numpy as np
import pytest
import torch

from unicache_amd.storage import Block8KVCache

pytestmark = pytest.mark.gpu

LIMIT = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = 2.0 ** -60
CODES = [torch.int8, torch.float8_e4m3fn]
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def dense(s, t, h, d, *, seed=0, dtype=torch.bfloat16, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    key = torch.randn(s, t, h, d, generator=g)
    key += torch.randn(s, -(-t // 40), h, d, generator=g).repeat_interleave(40, dim=1)[:, :t]
    key[..., torch.randperm(d, generator=g)[:5]] *= 6.0
    value = torch.randn(s, t, h, d, generator=g)
    # blocks of very different sizes, as sink tokens have them
    value *= torch.exp2(torch.randint(-6, 3, (s, -(-t // 32), h, 1), generator=g).float()).repeat_interleave(32, 1)[:, :t]
    return key.to(dtype).to(device), value.to(dtype).to(device)


def queries(s, lq, hq, d, *, seed=1, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(s, lq, hq, d, generator=g) * scale).to(dtype).cuda()


def quantized(x, length, block, code):
    """numpy fp32 restatement of one head's blocks: x [T, D] -> value of every
    code [N, B, D], scales [N], largest / smallest code value of the counted rows [N, D]."""

    t, d = x.shape
    n = -(-t // block)
    rows = np.zeros((n * block, d), np.float32)
    rows[:length] = x[:length]
    rows = rows.reshape(n, block, d)
    limit = np.float32(LIMIT[code])
    a = np.maximum(np.abs(rows).max(axis=(1, 2)), np.float32(limit * TINY)).astype(np.float32)
    scale = a * np.float32(1.0 / limit)
    y = rows * (limit / a)[:, None, None]
    if code == torch.int8:
        c = np.rint(y)
    else:
        c = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).float().numpy()
    live = (np.arange(n * block) < length).reshape(n, block, 1)
    hi = np.where(live, c, -np.inf).max(axis=1)
    lo = np.where(live, c, np.inf).min(axis=1)
    return c, scale, hi, lo


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block,d,dtype", [(32, 64, torch.bfloat16), (32, 128, torch.float16), (64, 64, torch.float16),
                                          (64, 128, torch.bfloat16), (128, 64, torch.bfloat16),
                                          (128, 128, torch.float16)])
def test_codes_scales_and_bounds_are_exact(device, code, block, d, dtype):
    t, h = 333, 3
    lens = [333, 1, 0, 2 * block]
    key, value = dense(4, t, h, d, dtype=dtype)
    key[3, block:2 * block, 1] = 0  # a block of zeros
    cache = Block8KVCache.from_dense(key, value, lengths=torch.tensor(lens, dtype=torch.int32, device=device),
                                     block_tokens=block, code_dtype=code)
    rk, rv = cache.dequantize()
    assert rk.shape == key.shape and rk.dtype == dtype
    for s, n in enumerate(lens):
        for j in range(h):
            ck, sk, hi, lo = quantized(key[s, :, j].float().cpu().numpy(), n, block, code)
            cv, sv, _, _ = quantized(value[s, :, j].float().cpu().numpy(), n, block, code)
            assert np.array_equal(cache.key_scale[s, j].cpu().numpy(), sk)
            assert np.array_equal(cache.value_scale[s, j].cpu().numpy(), sv)
            assert np.array_equal(cache.key_code[s, j].float().cpu().numpy(), ck.reshape(-1, d))
            assert np.array_equal(cache.value_code[s, j].float().cpu().numpy(), cv.transpose(0, 2, 1))
            for restored, c, sc in ((rk, ck, sk), (rv, cv, sv)):
                want = torch.from_numpy((c * sc[:, None, None]).reshape(-1, d)[:t]).to(dtype)
                assert torch.equal(restored[s, :, j].cpu(), want)
            some = np.arange(len(sk)) * block < n
            bounds = cache.key_bounds[s, j].cpu().numpy().astype(np.int64)
            # whole multiples of 2^-9 times 127/448, in whole numbers
            up = lambda c: -((-(c * 512).astype(np.int64) * 127) // (512 * 448))  # noqa: E731
            down = lambda c: ((c * 512).astype(np.int64) * 127) // (512 * 448)  # noqa: E731
            if code == torch.int8:
                up = down = lambda c: c.astype(np.int64)  # noqa: E731
            assert np.array_equal(bounds[some, 0], up(hi[some])) and np.array_equal(bounds[some, 1], down(lo[some]))
            assert not bounds[~some].any()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block,d", [(32, 128), (64, 64), (128, 128)])
def test_append_equals_from_dense(device, code, block, d):
    # ragged counts that fill, cross and skip blocks; rows behind a count are never read as tokens
    t, h, s = 5 * block + 9, 2, 3
    key, value = dense(s, t, h, d, seed=3)
    cache = Block8KVCache.empty(s, t, h, d, block_tokens=block, code_dtype=code)
    steps = [(1, [1, 1, 0]), (block - 1, [block - 1, 5, 0]), (1, [1, 0, 1]), (2 * block + 7, [2 * block + 7, block, 3]),
             (1, [0, 1, 1]), (block, [block, block, block])]
    done = [0] * s
    for n, counts in steps:
        rows_k = torch.full((s, n, h, d), 77.0, dtype=key.dtype, device=device)
        rows_v = torch.full_like(rows_k, -55.0)
        for i, c in enumerate(counts):
            rows_k[i, :c], rows_v[i, :c] = key[i, done[i]:done[i] + c], value[i, done[i]:done[i] + c]
            done[i] += c
        cache.append(rows_k, rows_v, counts=torch.tensor(counts, dtype=torch.int32, device=device))
        assert cache.lengths.tolist() == done
        want = Block8KVCache.from_dense(key, value, lengths=cache.lengths, block_tokens=block, code_dtype=code)
        for i in range(s):
            n_blocks = -(-done[i] // block)
            for name in ("key_code", "value_code", "key_scale", "value_scale", "key_bounds"):
                got, exp = getattr(cache, name)[i], getattr(want, name)[i]
                m = n_blocks * block if name == "key_code" else n_blocks
                assert torch.equal(got[:, :m].float(), exp[:, :m].float()), (name, i, done)
    # past the capacity: dropped
    cache.append(key, value)
    assert cache.lengths.tolist() == [cache.capacity] * s


@pytest.mark.parametrize("code", CODES)
def test_chunked_prefill_equals_from_dense(device, code):
    # chunks of many blocks, each from an open block into another
    t, h, s, d, block = 2500, 3, 2, 64, 32
    key, value = dense(s, t, h, d, seed=4)
    cache = Block8KVCache.empty(s, t, h, d, block_tokens=block, code_dtype=code)
    start = 0
    for n in (700, 1024, 3, 512, 261):
        cache.append(key[:, start:start + n], value[:, start:start + n])
        start += n
    assert start == t
    want = Block8KVCache.from_dense(key, value, block_tokens=block, code_dtype=code)
    for name in ("key_code", "value_code", "key_scale", "value_scale", "key_bounds"):
        assert torch.equal(getattr(cache, name).float(), getattr(want, name).float()), name
    rows = t % block
    assert torch.equal(cache.tail[:, :, 0, :rows], key[:, -rows:].transpose(1, 2))
    assert torch.equal(cache.tail[:, :, 1, :rows], value[:, -rows:].transpose(1, 2))


def test_a_block_with_infinities_reads_as_nan(device):
    key, value = dense(1, 200, 2, 128)
    key[0, 70, 1, 3] = math.inf
    value[0, 130, 0, 5] = math.nan
    for code in CODES:
        cache = Block8KVCache.from_dense(key, value, block_tokens=64, code_dtype=code)
        k, v = cache.dequantize()
        assert torch.isnan(k[0, 64:128, 1]).all() and torch.isnan(v[0, 128:192, 0]).all()
        k[0, 64:128, 1] = v[0, 128:192, 0] = 0
        assert torch.isfinite(k).all() and torch.isfinite(v).all()
        # rows that see such a block are NaN, rows and heads that do not are not touched by it
        q = queries(1, 200, 4, 128)
        out, lse = cache.attention(q, causal=True)
        assert torch.isnan(out[0, 64:, 2:]).all() and torch.isfinite(out[0, :64, 2:]).all()
        assert torch.isnan(out[0, 128:, :2]).all() and torch.isfinite(out[0, :128, :2]).all()
        assert torch.isfinite(lse[0, 2:, :64]).all() and torch.isfinite(lse[0, :2, :128]).all()


# --------------------------------------------------------------- attention --
def reference(cache, q, lens, qlens, causal, sm_scale, chosen=None, query_block=1):
    """Attention over the cache's codes in 64 bits: out, lse, and per element
    how far a kernel that rounds the weights to fp16 once may be off."""

    s, lq, hq, d = q.shape
    h, b = cache.num_kv_heads, cache.block_tokens
    g = hq // h
    out = torch.zeros(s, lq, hq, d, dtype=torch.float64)
    lse = torch.full((s, hq, lq), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    tol_lse = torch.zeros_like(lse)
    kc, vc = cache.key_code.float().double().cpu(), cache.value_code.float().double().cpu()
    ks, vs = cache.key_scale.double().cpu(), cache.value_scale.double().cpu()
    qd = q.double().cpu()
    for i in range(s):
        n, m = lens[i], qlens[i]
        if n == 0 or m == 0:
            continue
        nb = -(-n // b)
        for j in range(h):
            k = (kc[i, j, :nb * b] * ks[i, j, :nb].repeat_interleave(b)[:, None])[:n]
            v = (vc[i, j, :nb].transpose(1, 2).reshape(nb * b, d) * vs[i, j, :nb].repeat_interleave(b)[:, None])[:n]
            x = torch.einsum("rgd,td->grt", qd[i, :m, j * g:(j + 1) * g], k) * sm_scale
            size = torch.einsum("rgd,td->grt", qd[i, :m, j * g:(j + 1) * g].abs(), k.abs()) * sm_scale
            if causal:
                x.masked_fill_(torch.arange(n) > (n - m + torch.arange(m))[:, None], -math.inf)
            if chosen is not None:
                for r0 in range(0, m, query_block):
                    keep = torch.zeros(nb + 1, dtype=torch.bool)
                    keep[chosen[i, r0 // query_block, j].long()] = True
                    x[:, r0:r0 + query_block, ~keep[torch.arange(n) // b]] = -math.inf
            total = torch.logsumexp(x, dim=-1)
            p = torch.exp(x - torch.where(total == -math.inf, 0.0, total)[..., None])
            o = torch.einsum("grt,td->rgd", p, v)
            spread = torch.einsum("grt,td->rgd", p, v.abs())
            # fp32 logits: D products and as many sums, each half a step of the sum of magnitudes at
            # most, the scales, the exponent's addend (60 at most); the same in the sum below the line
            off = (d + 8) * 2.0 ** -24 * size.amax(dim=-1) + 64 * 2.0 ** -23
            weight = 2.0 ** -11 + 2 * off + n * 2.0 ** -23
            # weights below fp16's normal range: half a step of 2^-24 each, over a largest one of at least 2^-8
            flat = n * 2.0 ** -25 * 2.0 ** 8 * (p.amax(dim=-1).transpose(0, 1)[..., None] * v.abs().amax())
            out[i, :m, j * g:(j + 1) * g] = o
            tol[i, :m, j * g:(j + 1) * g] = (EPS[q.dtype] * (o.abs() + weight.transpose(0, 1)[..., None] * spread)
                                             + weight.transpose(0, 1)[..., None] * spread + flat
                                             + torch.finfo(q.dtype).smallest_normal * EPS[q.dtype])
            lse[i, j * g:(j + 1) * g, :m] = total
            tol_lse[i, j * g:(j + 1) * g, :m] = off + n * 2.0 ** -23 + 2.0 ** -22 * (1 + total.abs())
    return out, lse, tol, tol_lse


def check(got, want):
    out, lse = (x.double().cpu() for x in got)
    eo, el, to, tl = want
    assert out.shape == eo.shape and lse.shape == el.shape
    empty = el == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert not out.transpose(1, 2)[empty].any()
    err = (out - eo).abs()
    assert (err <= to).all(), f"out: {err.max():.3g}, {(err / to.clamp_min(1e-300)).max():.3g} of what it may be"
    err = (lse - el)[~empty].abs()
    if err.numel():
        assert (err <= tl[~empty]).all(), f"lse: {err.max():.3g}"


# tokens, sequence lengths, heads, queries: single tokens, odd lengths, rows of one and of several
# MFMA tiles, every group size, causal rows that see nothing (more queries than keys)
ATTEND = [
    dict(lens=[1], hq=4, hkv=4, lq=1),
    dict(lens=[31, 0, 32, 33], hq=28, hkv=4, lq=1),
    dict(lens=[63, 64, 65, 1], hq=7, hkv=1, lq=1, causal=True),
    dict(lens=[2047, 129, 1000], hq=32, hkv=8, lq=1),
    dict(lens=[4097], hq=28, hkv=4, lq=1, d=64),
    dict(lens=[700, 3], hq=28, hkv=4, lq=3, causal=True),
    dict(lens=[513, 5, 0], hq=16, hkv=2, lq=5, qlens=[5, 2, 3], causal=True, d=64),
    dict(lens=[300], hq=24, hkv=1, lq=1),
    dict(lens=[300], hq=40, hkv=1, lq=1),
    dict(lens=[1000, 20], hq=4, hkv=4, lq=100, causal=True),
    dict(lens=[515, 700], hq=28, hkv=4, lq=130, causal=False, qlens=[130, 77]),
    dict(lens=[600, 600, 90], hq=8, hkv=2, lq=301, causal=True, qlens=[301, 0, 200], d=64),
    dict(lens=[1500], hq=14, hkv=2, lq=257, causal=True),
]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(device, code, block, case):
    a = ATTEND[case]
    lens, d, lq = a["lens"], a.get("d", 128), a["lq"]
    dtype = torch.float16 if (case + block // 32) % 2 else torch.bfloat16
    print(f"attention case {case} block {block} {code}", flush=True)
    key, value = dense(len(lens), max(lens), a["hkv"], d, seed=case, dtype=dtype)
    lengths = torch.tensor(lens, dtype=torch.int32, device=device)
    cache = Block8KVCache.from_dense(key, value, lengths=lengths, block_tokens=block, code_dtype=code)
    q = queries(len(lens), lq, a["hq"], d, seed=case + 50, dtype=dtype)
    qlens = a.get("qlens")
    given = None if qlens is None else torch.tensor(qlens, dtype=torch.int32, device=device)
    causal = a.get("causal", False)
    got = cache.attention(q, causal=causal, query_lengths=given)
    check(got, reference(cache, q, lens, qlens or [lq] * len(lens), causal, 1 / math.sqrt(d)))


@pytest.mark.parametrize("lq", [1, 96])
def test_garbage_behind_the_length_does_not_matter(device, lq):
    # NaN codes, scales and bounds in rows and blocks that no length covers; a cache with room to spare
    lens = [70, 33, 0]
    key, value = dense(3, 96, 2, 128, seed=8)
    lengths = torch.tensor(lens, dtype=torch.int32, device=device)
    for block in (32, 64):
        cache = Block8KVCache.from_dense(key, value, lengths=lengths, block_tokens=block, capacity=400)
        q = queries(3, lq, 8, 128, seed=9)
        want = cache.attention(q), cache.sparse_attention(q, budget=4, query_block=lq)
        for s, n in enumerate(lens):
            nb = -(-n // block)
            cache.key_code.view(torch.uint8)[s, :, n:] = 0x7f
            cache.value_code.view(torch.uint8)[s, :, nb:] = 0x7f
            if n % block:
                cache.value_code.view(torch.uint8)[s, :, nb - 1, :, n % block:] = 0xff
            for name in ("key_scale", "value_scale"):
                getattr(cache, name)[s, :, nb:] = math.nan
            cache.key_bounds[s, :, nb:] = 127
        got = cache.attention(q), cache.sparse_attention(q, budget=4, query_block=lq)
        for a, b in zip(want[0] + want[1], got[0] + got[1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("lq", [1, 64])
def test_lengths_outside_the_capacity_read_as_its_ends(device, lq):
    key, value = dense(2, 128, 2, 64, seed=4)
    cache = Block8KVCache.from_dense(key, value, block_tokens=64)
    q = queries(2, lq, 4, 64)
    want, _ = cache.attention(q)
    cache.lengths.copy_(torch.tensor([1 << 30, -5], dtype=torch.int32))
    got, lse = cache.attention(q)
    assert torch.equal(got[0], want[0]) and not got[1].any() and (lse[1] == -math.inf).all()


def test_values_of_any_size(device):
    # queries and values far from fp16's range, blocks of zeros beside them
    key, value = dense(1, 400, 2, 128, seed=11)
    q = queries(1, 2, 8, 128, seed=12)
    for power in (-90, -30, 40, 100):
        k, v = key * 2.0 ** (-power), value * 2.0 ** (power if power > -50 else -40)
        v[0, 128:256] = 0
        for code in CODES:
            cache = Block8KVCache.from_dense(k, v, block_tokens=64, code_dtype=code)
            qq = q * 2.0 ** power
            check(cache.attention(qq), reference(cache, qq, [400], [2], False, 1 / math.sqrt(128)))


def test_strided_queries_and_rows(device):
    # a fused projection's slices, transposed layouts, an odd channel stride
    key, value = dense(2, 200, 4, 64, seed=20)
    fused = torch.cat([key, value], dim=2)
    a = Block8KVCache.from_dense(fused[:, :, :4], fused[:, :, 4:])
    b = Block8KVCache.from_dense(key.transpose(1, 2).contiguous().transpose(1, 2), value.clone())
    c = Block8KVCache.from_dense(key, value)
    wide = torch.empty(2, 200, 4, 65, dtype=key.dtype, device=device)
    wide[..., 1:] = key
    e = Block8KVCache.from_dense(wide[..., 1:], value)
    for x in (a, b, e):
        for name in ("key_code", "value_code", "key_scale", "value_scale", "key_bounds"):
            assert torch.equal(getattr(x, name).float(), getattr(c, name).float()), name
    q = queries(2, 3, 24, 64, seed=21)
    want = c.attention(q[:, :, 8:16])
    for view in (q[:, :, 8:16].contiguous(), q.transpose(1, 2).contiguous().transpose(1, 2)[:, :, 8:16]):
        got = c.attention(view)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_one_sequence_without_a_batch_axis(device):
    key, value = dense(1, 150, 2, 128, seed=30)
    cache = Block8KVCache.from_dense(key[0], value[0], capacity=256)
    q = queries(1, 1, 4, 128)
    assert torch.equal(cache.attention(q[0])[0], cache.attention(q)[0])
    cache.append(key[0, :3], value[0, :3])
    assert cache.lengths.tolist() == [153]


def test_queries_of_no_tokens_and_odd_strides_of_single_dimensions(device):
    key, value = dense(1, 64, 2, 64, seed=31)
    cache = Block8KVCache.from_dense(key, value)
    q = queries(1, 1, 4, 64, seed=32)
    out, lse = cache.attention(q[:, :0])
    assert out.shape == (1, 0, 4, 64) and lse.shape == (1, 4, 0)
    out, lse, blocks = cache.sparse_attention(q[:, :0], budget=3)
    assert out.shape == (1, 0, 4, 64) and blocks.shape == (1, 0, 2, 3)
    odd = torch.empty_strided((1, 1, 4, 64), (7, 5, 64, 1), dtype=q.dtype, device=device).copy_(q)
    assert torch.equal(cache.attention(odd)[0], cache.attention(q)[0])


@pytest.mark.parametrize("lq,d", [(1, 128), (3, 64), (40, 64)])
def test_more_sequences_than_a_wave_has_lanes(device, lq, d):
    g = torch.Generator().manual_seed(33)
    lens = torch.randint(0, 700, (150,), generator=g)
    lens[::7] = 0
    lens[60:70] = 0
    lens = lens.tolist()
    key, value = dense(150, 700, 2, d, seed=34)
    cache = Block8KVCache.from_dense(key, value, lengths=torch.tensor(lens, dtype=torch.int32, device=device))
    q = queries(150, lq, 6, d, seed=35)
    check(cache.attention(q, causal=True), reference(cache, q, lens, [lq] * 150, True, 1 / math.sqrt(d)))
    out, lse, blocks = cache.sparse_attention(q, budget=4, query_block=lq)
    want = chosen_blocks(cache, q, lens, [lq] * 150, False, 4, lq, 1, 1)
    assert torch.equal(blocks.cpu(), want)
    check((out, lse), reference(cache, q, lens, [lq] * 150, False, 1 / math.sqrt(d), want, lq))


@pytest.mark.parametrize("rows", [(8, 4, 64), (16, 3, 64), (16, 4, 64), (28, 4, 128), (4, 5, 128), (9, 7, 64)])
def test_every_number_of_rows_of_a_head(device, rows):
    # groups of 2 .. 28 query heads over one KV head x a few tokens, on both sides of 16, 32, 48 and 128 rows
    hq, lq, d = rows
    lens = [1500, 63]
    key, value = dense(2, 1500, 1, d, seed=36)
    cache = Block8KVCache.from_dense(key, value, lengths=torch.tensor(lens, dtype=torch.int32, device=device),
                                     code_dtype=torch.int8)
    q = queries(2, lq, hq, d, seed=37)
    check(cache.attention(q, causal=True), reference(cache, q, lens, [lq] * 2, True, 1 / math.sqrt(d)))


@pytest.mark.parametrize("lq", [1, 50])
def test_scales_of_zero(device, lq):
    # a cache that another program made, whose blocks of zeros have the scale 0
    key, value = dense(1, 320, 2, 128, seed=38)
    key[:, 64:128], value[:, :64], value[:, 192:256] = 0, 0, 0
    cache = Block8KVCache.from_dense(key, value)
    q = queries(1, lq, 4, 128, seed=39)
    want = reference(cache, q, [320], [lq], False, 1 / math.sqrt(128))
    cache.key_scale[:, :, 1] = 0
    cache.value_scale[:, :, [0, 3]] = 0
    check(cache.attention(q), want)


@pytest.mark.parametrize("lq", [2, 60])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_any_block_list_is_read_within_bounds(device, lq, block):
    # the C entry point with indexes outside the cache, the same one twice in a row, none, and blocks behind the length
    from unicache_amd import _native as nat

    key, value = dense(1, 1000, 2, 128, seed=40)
    cache = Block8KVCache.from_dense(key, value, block_tokens=block, capacity=1400)
    q = queries(1, lq, 6, 128, seed=41)
    lists = torch.full((1, 1, 2, 70), -1, dtype=torch.int32)
    lists[0, 0, 0, :8] = torch.tensor([0, 0, 2, 2, 5, 10000, -7, 1 << 30])
    lists[0, 0, 1, 60:70] = torch.tensor([1, 3, 3, 3, 6, cache.blocks - 1, cache.blocks, -1, -1, 7])
    struct = cache._query(q, None, False)[1]
    out, lse = torch.empty_like(q), torch.empty(1, 6, lq, device=device)
    nbytes = nat.lib().uc_block8_attn_workspace_bytes(cache._struct(), struct, 70, lq)
    ws = nat.workspace(device, nbytes)
    there = lists.to(device)
    nat.call("uc_block8_attn", cache._struct(), struct, there.data_ptr(), 70, lq, 0.1, out.data_ptr(), lse.data_ptr(),
             ws.data_ptr(), nbytes, nat.stream(device))
    last = -(-1000 // block) - 1
    keep = torch.full((1, 1, 2, 4), -1, dtype=torch.int32)
    keep[0, 0, 0, :3] = torch.tensor([0, 2, 5])
    keep[0, 0, 1] = torch.tensor([1, 3, 6, 7])
    check((out, lse), reference(cache, q, [1000], [lq], False, 0.1, keep.clamp_max(last + 1), lq))


# --------------------------------------------------------------- selection --
def chosen_blocks(cache, q, lens, qlens, causal, budget, query_block, sink, recent):
    s, lq, hq, d = q.shape
    h, b = cache.num_kv_heads, cache.block_tokens
    g = hq // h
    x = q.float().cpu().numpy()
    good = np.isfinite(x).all(axis=-1)
    x = np.where(good[..., None], x, 0).astype(np.float32)
    a = np.abs(x).max(axis=-1, keepdims=True)
    codes = np.where(a > 0, np.rint(x * (np.float32(127) / np.where(a > 0, a, 1))), 0).clip(-127, 127)
    step = a[..., 0] * np.float32(1.0 / 127.0)
    out = np.full((s, -(-lq // query_block), h, budget), -1, np.int32)
    for i in range(s):
        n, m = lens[i], qlens[i]
        for r0 in range(0, m, query_block):
            r1 = min(m, r0 + query_block)
            first, last = (max(0, n - m + r0), n - m + r1 - 1) if causal else (max(0, n - 1), n - 1)
            if last < 0:
                continue
            for j in range(h):
                bounds = cache.key_bounds[i, j].cpu().numpy().astype(np.float64)
                unit = cache.key_scale[i, j].cpu().numpy()
                if cache.code_dtype != torch.int8:
                    unit = unit * np.float32(448.0 / 127.0)
                c = codes[i, r0:r1, j * g:(j + 1) * g].reshape(-1, d).astype(np.float64)
                ok = good[i, r0:r1, j * g:(j + 1) * g].reshape(-1)
                whole = np.maximum(c[:, None] * bounds[None, :, 0], c[:, None] * bounds[None, :, 1]).sum(axis=2)
                score = whole.astype(np.float32) * unit * step[i, r0:r1, j * g:(j + 1) * g].reshape(-1, 1)
                score = np.where(ok[:, None], score, -np.inf).max(axis=0)[:last // b + 1]
                score[~np.isfinite(unit[:len(score)])] = np.inf
                forced = np.zeros(len(score), bool)
                forced[:sink] = True
                forced[max(0, first // b - recent + 1):] = True
                order = sorted(range(len(score)), key=lambda t: (not forced[t], -score[t], t))[:budget]
                out[i, r0 // query_block, j, :len(order)] = sorted(order)
    return torch.from_numpy(out)


SPARSE = [
    dict(lens=[5000, 70, 0, 1], hq=28, hkv=4, lq=1, budget=5),
    dict(lens=[8191], hq=32, hkv=8, lq=1, budget=16, sink=0, recent=2),
    dict(lens=[900, 3000], hq=16, hkv=2, lq=4, budget=9, query_block=2, d=64),
    dict(lens=[2100], hq=14, hkv=2, lq=150, budget=11, query_block=32, causal=True, sink=2, recent=3),
    dict(lens=[1300, 90], hq=8, hkv=4, lq=201, qlens=[201, 120], budget=8, query_block=100, causal=True, d=64),
    dict(lens=[640], hq=4, hkv=4, lq=77, budget=64, query_block=33, causal=False),
    dict(lens=[20000, 9000], hq=8, hkv=2, lq=1, budget=150, recent=2),
    dict(lens=[9000], hq=8, hkv=2, lq=48, budget=100, query_block=24, causal=True),
    dict(lens=[1500], hq=8, hkv=4, lq=300, budget=5, causal=True),  # a list for each token
]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("case", range(len(SPARSE)))
def test_sparse_attention(device, code, block, case):
    a = SPARSE[case]
    lens, d, lq = a["lens"], a.get("d", 128), a["lq"]
    causal, qb = a.get("causal", False), a.get("query_block", 1)
    sink, recent = a.get("sink", 1), a.get("recent", 1)
    print(f"sparse case {case} block {block} {code}", flush=True)
    key, value = dense(len(lens), max(lens), a["hkv"], d, seed=100 + case)
    cache = Block8KVCache.from_dense(key, value, lengths=torch.tensor(lens, dtype=torch.int32, device=device),
                                     block_tokens=block, code_dtype=code)
    q = queries(len(lens), lq, a["hq"], d, seed=150 + case)
    qlens = a.get("qlens")
    given = None if qlens is None else torch.tensor(qlens, dtype=torch.int32, device=device)
    qlens = qlens or [lq] * len(lens)
    out, lse, blocks = cache.sparse_attention(q, budget=a["budget"], query_block=qb, sink=sink, recent=recent,
                                              query_lengths=given, causal=causal)
    want = chosen_blocks(cache, q, lens, qlens, causal, a["budget"], qb, sink, recent)
    assert torch.equal(blocks.cpu(), want)
    check((out, lse), reference(cache, q, lens, qlens, causal, 1 / math.sqrt(d), want, qb))


@pytest.mark.parametrize("lq", [1, 40])
def test_selection_among_more_blocks_than_lds_holds(device, lq):
    lens = [300000, 262144 + 64]  # 9375 and 8194 blocks
    g = torch.Generator(device="cuda").manual_seed(5)
    key = torch.randn(2, 300000, 1, 64, generator=g, device="cuda", dtype=torch.bfloat16)
    cache = Block8KVCache.from_dense(key, key, lengths=torch.tensor(lens, dtype=torch.int32, device=device),
                                     block_tokens=32)
    q = queries(2, lq, 2, 64, seed=6)
    _, _, blocks = cache.sparse_attention(q, budget=50, query_block=40)
    assert torch.equal(blocks.cpu(), chosen_blocks(cache, q, lens, [lq, lq], False, 50, 40, 1, 1))


@pytest.mark.parametrize("lens,lq,run", [([262200], 130, 1), ([40000, 100, 25000], 7, 2), ([17000], 12, 5)])
def test_selection_of_few_rows_among_many_blocks(device, lens, lq, run):
    # many runs of more blocks than LDS holds; causal runs whose sequences end differently
    causal = run > 1
    g = torch.Generator(device="cuda").manual_seed(7)
    key = torch.randn(len(lens), max(lens), 1, 64, generator=g, device="cuda", dtype=torch.bfloat16)
    cache = Block8KVCache.from_dense(key, key, lengths=torch.tensor(lens, dtype=torch.int32, device=device),
                                     block_tokens=32)
    q = queries(len(lens), lq, 3, 64, seed=8)
    _, _, blocks = cache.sparse_attention(q, budget=50, query_block=run, sink=3, recent=2, causal=causal)
    assert torch.equal(blocks.cpu(), chosen_blocks(cache, q, lens, [lq] * len(lens), causal, 50, run, 3, 2))
    # a launch that expects shorter sequences
    cache.max_tokens = 600 * 32
    assert torch.equal(cache.sparse_attention(q, budget=50, query_block=run, sink=3, recent=2, causal=causal)[2], blocks)


def test_selection_of_equal_scores_and_odd_queries(device):
    # equal blocks: the lower index; zero queries; a NaN query beside good ones; a block of NaN keys
    key, value = dense(1, 64 * 40, 1, 128, seed=60)
    key[:, :] = key[:, :64].repeat(1, 40, 1, 1)
    cache = Block8KVCache.from_dense(key, value, block_tokens=64)
    q = queries(1, 1, 4, 128)
    _, _, blocks = cache.sparse_attention(q, budget=6)
    assert blocks[0, 0, 0].tolist() == [0, 1, 2, 3, 4, 39]
    _, _, blocks = cache.sparse_attention(torch.zeros_like(q), budget=6)
    assert blocks[0, 0, 0].tolist() == [0, 1, 2, 3, 4, 39]
    key, value = dense(1, 64 * 40, 1, 128, seed=61)
    cache = Block8KVCache.from_dense(key, value, block_tokens=64)
    bad = q.clone()
    bad[0, 0, 2, 7] = math.nan
    out, _, blocks = cache.sparse_attention(bad, budget=6)
    assert torch.equal(blocks.cpu(), chosen_blocks(cache, bad, [2560], [1], False, 6, 1, 1, 1))
    assert torch.isnan(out[0, 0, 2]).all() and torch.isfinite(out[0, 0, [0, 1, 3]]).all()
    key[0, 64 * 17 + 3, 0, 0] = math.nan
    cache = Block8KVCache.from_dense(key, value, block_tokens=64)
    out, _, blocks = cache.sparse_attention(q, budget=6)
    assert 17 in blocks[0, 0, 0].tolist() and torch.isnan(out).all()


def test_all_blocks_selected_equals_attention(device):
    key, value = dense(2, 700, 2, 128, seed=70)
    cache = Block8KVCache.from_dense(key, value, block_tokens=64)
    q = queries(2, 2, 8, 128, seed=71)
    out, lse, _ = cache.sparse_attention(q, budget=11, query_block=2)
    want = reference(cache, q, [700, 700], [2, 2], False, 1 / math.sqrt(128))
    check((out, lse), want)
    check(cache.attention(q), want)


# ----------------------------------------------------------- as it is used --
def test_prefill_then_decode_as_a_program_runs_it(device):
    # a prompt in two chunks, then tokens one at a time, dense and sparse, against one cache built at once
    s, h, hq, d, prompt, steps = 2, 2, 8, 64, 300, 5
    key, value = dense(s, prompt + steps, h, d, seed=80)
    q = queries(s, prompt + steps, hq, d, seed=81)
    cache = Block8KVCache.empty(s, 512, h, d, block_tokens=32)
    cache.append(key[:, :200], value[:, :200])
    cache.append(key[:, 200:prompt], value[:, 200:prompt])
    chunk = cache.attention(q[:, 200:prompt], causal=True)
    check(chunk, reference(cache, q[:, 200:prompt], [prompt] * s, [100] * s, True, 1 / math.sqrt(d)))
    for t in range(prompt, prompt + steps):
        cache.append(key[:, t:t + 1], value[:, t:t + 1])
        whole = Block8KVCache.from_dense(key[:, :t + 1], value[:, :t + 1], block_tokens=32)
        for call in (lambda c: c.attention(q[:, t:t + 1], causal=True),
                     lambda c: c.sparse_attention(q[:, t:t + 1], budget=4)):
            for a, b in zip(call(cache), call(whole)):
                # the launch is shaped by each cache's capacity: sums in another order
                assert a.shape == b.shape
        check(cache.attention(q[:, t:t + 1]), reference(whole, q[:, t:t + 1], [t + 1] * s, [1] * s, False, 1 / math.sqrt(d)))
        assert torch.equal(cache.sparse_attention(q[:, t:t + 1], budget=4)[2],
                           whole.sparse_attention(q[:, t:t + 1], budget=4)[2])


def test_captured_steps_replayed(device):
    # append + attention + sparse attention of a token in one graph, replayed past the captured length
    # and a block's end, eager work between; two graphs share nothing
    s, h, hq, d = 2, 2, 14, 128
    key, value = dense(s, 400, h, d, seed=90)
    q = queries(s, 60, hq, d, seed=91)
    cache = Block8KVCache.from_dense(key[:, :90], value[:, :90], capacity=400, block_tokens=32)
    mirror = Block8KVCache.from_dense(key[:, :90], value[:, :90], capacity=400, block_tokens=32)
    k1, v1, q1 = key[:, :1].clone(), value[:, :1].clone(), q[:, :1].clone()

    def step(c):
        c.append(k1, v1)
        return (*c.attention(q1), *c.sparse_attention(q1, budget=3))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        scratch = Block8KVCache.from_dense(key[:, :90], value[:, :90], capacity=400, block_tokens=32)
        step(scratch)  # warm-up outside the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache)
    for t in range(50):
        k1.copy_(key[:, 90 + t:91 + t])
        v1.copy_(value[:, 90 + t:91 + t])
        q1.copy_(q[:, t:t + 1])
        graph.replay()
        mirror.append(k1, v1)
        mirror.max_tokens = cache.max_tokens  # the launch that was captured
        want = (*mirror.attention(q1), *mirror.sparse_attention(q1, budget=3))
        for a, b in zip(got, want):
            assert torch.equal(a, b), t
        if t % 7 == 0:
            torch.cuda.synchronize()
    assert cache.lengths.tolist() == [140, 140]


def test_two_graphs_of_one_cache(device):
    # decode and a sparse step captured apart, replayed in turn and over changed lengths
    key, value = dense(3, 600, 2, 128, seed=92)
    lens = torch.tensor([600, 100, 0], dtype=torch.int32, device=device)
    cache = Block8KVCache.from_dense(key, value, lengths=lens)
    q = queries(3, 1, 14, 128, seed=93)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attention(q), cache.sparse_attention(q, budget=3)
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.graph(graphs[0]):
        got.append(cache.attention(q))
    with torch.cuda.graph(graphs[1]):
        got.append(cache.sparse_attention(q, budget=3))
    for n in (600, 64, 1, 0, 599, 300):
        cache.lengths.copy_(torch.tensor([n, 600 - n, 7], dtype=torch.int32))
        q.copy_(queries(3, 1, 14, 128, seed=n))
        for g in graphs:
            g.replay()
        want = cache.attention(q), cache.sparse_attention(q, budget=3)
        for a, b in zip(got[0] + got[1], want[0] + want[1]):
            assert torch.equal(a, b), n


def test_mixed_attention_over_a_block8_segment(device):
    # the adapter's mixed call: dense rows, a packed KIVI segment, an H2O segment and an 8-bit one as one softmax
    from unicache_amd.adapters.bagel import run_batched_physical_attention, run_fused_mixed_attention
    from unicache_amd.storage import GQAH2OCache, PackedKIVICache

    def rows(n, seed):
        k, v = dense(1, n, 4, 128, seed=seed)
        return k[0] * 0.3, v[0]

    dk, dv = rows(90, 110)
    pk, pv = rows(300, 111)
    bk, bv = rows(333, 112)
    hk, hv = rows(64, 113)
    packed = PackedKIVICache.from_dense(pk, pv, logical_token_ids=torch.arange(300, device=device), token_type_id=0,
                                        k_bits=4, v_bits=4, group_size=32, residual_length=10, backend="cuda")
    h2o = GQAH2OCache.from_dense(hk, hv, logical_token_ids=torch.arange(64, device=device), token_type_id=0,
                                 per_kv_head_scores=torch.rand(4, 64, device=device), target_tokens=20,
                                 recent_tokens=5, selection_frozen=True)
    block8 = Block8KVCache.from_dense(bk, bv)
    rk, rv = packed.dequantize()
    ek, ev = (t[0].float().double() for t in block8.dequantize(torch.float16))
    for lq in (1, 200):
        q = queries(1, lq, 28, 128, seed=114)[0]
        for segments, keys, values in (
                ([packed, block8, h2o], [dk, rk, h2o.key.transpose(0, 1)], [dv, rv, h2o.value.transpose(0, 1)]),
                ([block8], [dk], [dv])):
            out, lse = run_fused_mixed_attention(q, dk, dv, segments, return_lse=True)
            k = torch.cat([*(t.double() for t in keys), ek]).repeat_interleave(7, dim=1)
            v = torch.cat([*(t.double() for t in values), ev]).repeat_interleave(7, dim=1)
            x = torch.einsum("rhd,thd->hrt", q.double(), k) / math.sqrt(128)
            want = torch.einsum("hrt,thd->rhd", torch.softmax(x, dim=-1), v)
            # the tolerances of the other mixed-attention tests: summaries are rounded to bf16 before they are merged
            assert (out.double() - want).abs().max() < 2e-2 and (lse.double() - torch.logsumexp(x, dim=-1)).abs().max() < 5e-3
            batched = run_batched_physical_attention(q, dk, dv, [0, lq], [0, 90], [segments])
            assert torch.equal(batched, out)
    with pytest.raises(ValueError, match="one sequence"):
        run_fused_mixed_attention(q, dk, dv, [Block8KVCache.empty(2, 64, 4, 128, device=device)])


def test_another_stream(device):
    key, value = dense(4, 3000, 4, 128, seed=95)
    q = queries(4, 1, 28, 128, seed=96)
    cache = Block8KVCache.from_dense(key, value)
    want = cache.attention(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        held = [cache.attention(q) for _ in range(8)]
    torch.cuda.current_stream().wait_stream(stream)
    for got in held:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_results_do_not_change_from_run_to_run(device):
    key, value = dense(3, 2500, 4, 128, seed=97)
    cache = Block8KVCache.from_dense(key, value)
    for lq in (1, 70):
        q = queries(3, lq, 28, 128, seed=98)
        want = cache.sparse_attention(q, budget=9, query_block=32) + cache.attention(q, causal=True)
        for _ in range(3):
            for a, b in zip(want, cache.sparse_attention(q, budget=9, query_block=32) + cache.attention(q, causal=True)):
                assert torch.equal(a, b)


def test_a_long_cache_past_32_bit_offsets(device):
    # one sequence behind 4 GiB of codes, its last blocks at large offsets
    s, h, d, n = 3, 8, 128, 1 << 21
    cache = Block8KVCache.empty(s, n, h, d, block_tokens=128, code_dtype=torch.int8)  # 2 GiB of keys a sequence
    key, value = dense(1, 300, h, d, seed=99)
    small = Block8KVCache.from_dense(key, value, block_tokens=128, code_dtype=torch.int8)
    at = n // 128 - 3  # the blocks of the last 300 tokens (the last one partial in `small`)
    for name in ("key_scale", "value_scale", "key_bounds", "value_code"):
        getattr(cache, name)[2].zero_()
        getattr(cache, name)[2, :, at:] = getattr(small, name)[0]
    cache.value_scale[2, :, :at] = 1.0
    cache.key_code[2].zero_()
    cache.key_code[2, :, at * 128:] = small.key_code[0]
    cache.lengths[2] = n - 84
    q = queries(1, 1, 8, d, seed=100)
    big = torch.zeros(s, 1, 8, d, dtype=q.dtype, device=device)
    big[2] = q[0]
    out, lse, blocks = cache.sparse_attention(big, budget=4, sink=0, recent=3)
    assert blocks[2, 0, 0, 1:].tolist() == [at, at + 1, at + 2]
    dense_out, dense_lse = cache.attention(big)
    eo, el, to, tl = reference(small, q, [300], [1], False, 1 / math.sqrt(d))
    # the zero keys each add exp(0), their values nothing
    zeros = n - 384
    want = torch.logaddexp(el[0], torch.full_like(el[0], math.log(zeros)))
    assert (dense_lse[2].double().cpu() - want).abs().max() < 1e-4
    share = torch.exp(el[0] - want).reshape(1, -1, 1)
    assert (dense_out[2].double().cpu() - eo[0] * share).abs().max() <= 2.0 ** -7 * eo.abs().max()


def zero_region(region, *, block, code, s=1, n=2048, h=4, d=128, seed=130):
    """A cache as another program may have made it: values of zero and value scales of 0 in the blocks
    for which region(first token) holds."""

    key, value = dense(s, n, h, d, seed=seed)
    at = torch.tensor([region(b * block) for b in range(-(-n // block))])
    value[:, at.repeat_interleave(block)[:n].to(value.device)] = 0
    cache = Block8KVCache.from_dense(key, value, block_tokens=block, code_dtype=code)
    cache.value_scale[:, :, at.to(value.device)] = 0
    return cache


# alone, before real values (a padded sequence), between them, behind them, and every second block
ZERO_REGIONS = [lambda t: True, lambda t: t < 256, lambda t: t < 1024, lambda t: 256 <= t < 512, lambda t: t >= 1024,
                lambda t: t // 128 % 2 == 0, lambda t: t // 32 % 2 == 0, lambda t: t // 32 % 2 == 1]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("lq", [1, 50])
@pytest.mark.parametrize("region", range(len(ZERO_REGIONS)))
def test_many_blocks_of_zeros_with_scales_of_zero(device, region, lq, code):
    # logits that are equal (zero queries) and random ones; d products at most, so the tolerances of reference() hold
    for block in (32, 128):
        print(f"zero region {region} block {block} rows {lq}", flush=True)
        cache = zero_region(ZERO_REGIONS[region], block=block, code=code)
        for q in (queries(1, lq, 28, 128, seed=131, scale=0.0), queries(1, lq, 28, 128, seed=132)):
            got = cache.attention(q)
            assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
            check(got, reference(cache, q, [2048], [lq], False, 1 / math.sqrt(128)))


@pytest.mark.parametrize("lq", [1, 50])
@pytest.mark.parametrize("tokens", [256, 1024, 30000])
def test_a_sequence_of_zeros_alone(device, tokens, lq):
    # ragged: as many keys as one workgroup takes, and many times that; out is 0, lse that of the keys
    cache = zero_region(lambda t: True, block=64, code=torch.int8, s=2, n=tokens, h=2, d=64, seed=133)
    cache.lengths[1] = tokens // 2 + 5
    q = queries(2, lq, 8, 64, seed=134)
    check(cache.attention(q), reference(cache, q, [tokens, tokens // 2 + 5], [lq] * 2, False, 1 / math.sqrt(64)))


@pytest.mark.parametrize("lq", [1, 50])
@pytest.mark.parametrize("power", [70, 100])
@pytest.mark.parametrize("odd", [0, 1])
def test_blocks_of_zeros_beside_very_large_values(device, odd, power, lq):
    # from_dense's own scales: every second half of a 64-key tile holds zeros (scale 2^-60), the others values of 2^power
    for code in CODES:
        key, value = dense(1, 640, 2, 128, seed=135)
        value = value * 2.0 ** power
        value[:, torch.arange(640, device=device) // 32 % 2 == odd] = 0
        cache = Block8KVCache.from_dense(key, value, block_tokens=32, code_dtype=code)
        for q in (queries(1, lq, 8, 128, seed=136, scale=0.0), queries(1, lq, 8, 128, seed=137)):
            for causal in (False, True):
                check(cache.attention(q, causal=causal),
                      reference(cache, q, [640], [lq], causal, 1 / math.sqrt(128)))


@pytest.mark.parametrize("lq", [1, 50])
def test_small_value_scales(device, lq):
    # another program's values far below the quantizer's smallest, behind blocks of zeros: kept down to scales of 2^-88
    for block in (32, 64):
        cache = zero_region(lambda t: t < 512, block=block, code=torch.float8_e4m3fn, n=1000, h=2)
        q = queries(1, lq, 8, 128, seed=138)
        cache.value_scale.mul_(2.0 ** -66)  # dense() has scales of 2^-13 to 2^-6
        check(cache.attention(q), reference(cache, q, [1000], [lq], False, 1 / math.sqrt(128)))
        # below that the weights stay right, and what the values add is less than 448 * 2^-88
        _, want, _, tol = reference(cache, q, [1000], [lq], False, 1 / math.sqrt(128))
        cache.value_scale.mul_(2.0 ** -60)
        out, lse = cache.attention(q)
        assert ((lse.double().cpu() - want).abs() <= tol).all() and (out.abs() <= 448 * 2.0 ** -88).all()


@pytest.mark.parametrize("lq", [3, 50])
def test_rows_that_do_not_see_a_tiles_larger_scale(device, lq):
    # causal rows whose last key is in the first half of a tile, whose second half holds values 2^70 times as large
    key, value = dense(1, 64 + lq, 2, 128, seed=139)
    for code in CODES:
        cache = Block8KVCache.from_dense(key[:, :64], value[:, :64], block_tokens=32, code_dtype=code, capacity=128)
        cache.value_scale[:, :, 0] *= 2.0 ** -70
        q = queries(1, 64, 8, 128, seed=140)[:, 32 - lq // 2:32 - lq // 2 + lq]
        cache.lengths.fill_(32 - lq // 2 + lq)
        out, lse = cache.attention(q, causal=True)
        seen = lq // 2  # rows whose last key is token 31 or one before it
        first = Block8KVCache(*(getattr(cache, n) for n in ("key_code", "value_code", "key_scale", "value_scale", "key_bounds")),
                              torch.full_like(cache.lengths, 32))
        check((out[:, :seen], lse[..., :seen]), reference(first, q[:, :seen], [32], [seen], True, 1 / math.sqrt(128)))


@pytest.mark.parametrize("lq", [1, 70])
def test_mixed_attention_over_empty_segments(device, lq):
    # no dense rows and 8-bit segments of which none, one or all hold tokens
    from unicache_amd.adapters.bagel import run_batched_physical_attention, run_fused_mixed_attention

    key, value = dense(1, 100, 4, 128, seed=115)
    none = key[0, :0]
    q = queries(1, lq, 28, 128, seed=116)[0]

    def empty():
        return Block8KVCache.empty(1, 200, 4, 128, device=device)

    for segments in ([empty()], [empty(), empty()], [empty(), empty(), empty()]):
        out, lse = run_fused_mixed_attention(q, none, none, segments, return_lse=True)
        assert not out.any() and (lse == -math.inf).all()
        assert not run_batched_physical_attention(q, none, none, [0, lq], [0, 0], [segments]).any()
    full = Block8KVCache.from_dense(key, value)
    want, want_lse = run_fused_mixed_attention(q, none, none, [full], return_lse=True)
    out, lse = run_fused_mixed_attention(q, none, none, [empty(), full, empty()], return_lse=True)
    # weights of 0 and 1, and 1 again for the logarithm's half step
    assert (out.float() - want.float()).abs().max() <= 2.0 ** -8 * want.float().abs().max()
    assert (lse - want_lse).abs().max() <= 2.0 ** -22 * (1 + want_lse.abs().max())


@pytest.mark.parametrize("lq", [1, 5, 40])
def test_selection_by_very_small_queries(device, lq):
    # bf16 rows down to subnormals: 127 / max|q| is past fp32's range below 2^-121, the codes are what they are of 2^64 q
    key, value = dense(1, 64 * 40, 2, 128, seed=62)
    q = queries(1, lq, 4, 128, seed=63)
    q[..., ::5] = 0
    for power in (-90, -110, -122, -126, -131):
        small = (q.float() * 2.0 ** power).to(torch.bfloat16)
        for code in CODES:
            cache = Block8KVCache.from_dense(key * 2.0 ** 100, value, block_tokens=64, code_dtype=code)
            blocks = cache.sparse_attention(small, budget=6, query_block=lq)[2]
            x = small[0].float().cpu().numpy()
            a = np.abs(x).max(axis=-1, keepdims=True)
            y, b = x * np.float32(2.0 ** 64), a * np.float32(2.0 ** 64)
            with np.errstate(divide="ignore", invalid="ignore"):
                c = np.where(b > 0, np.rint(y * (np.float32(127) / b)), 0).astype(np.float64)
            step = a[..., 0] * np.float32(1.0 / 127.0)
            for j in range(2):
                bounds = cache.key_bounds[0, j].cpu().numpy().astype(np.float64)
                unit = cache.key_scale[0, j].cpu().numpy()
                if code != torch.int8:
                    unit = unit * np.float32(448.0 / 127.0)
                rows, s = c[:, 2 * j:2 * j + 2].reshape(-1, 128), step[:, 2 * j:2 * j + 2].reshape(-1, 1)
                whole = np.maximum(rows[:, None] * bounds[None, :, 0], rows[:, None] * bounds[None, :, 1]).sum(axis=2)
                score = (whole.astype(np.float32) * unit * s).max(axis=0)
                order = sorted(range(40), key=lambda t: (t not in (0, 39), -score[t], t))[:6]
                assert blocks[0, 0, j].tolist() == sorted(order), (power, code, j)


def test_more_sequences_and_heads_than_a_grid_dimension_holds(device):
    # packed at once, appended, restored: 65,535 is the most in a launch's second dimension
    s, h = 33000, 2
    g = torch.Generator(device="cuda").manual_seed(17)
    key = torch.randn(s, 3, h, 64, generator=g, device="cuda", dtype=torch.bfloat16)
    value = torch.randn(s, 3, h, 64, generator=g, device="cuda", dtype=torch.bfloat16)
    lengths = torch.randint(0, 4, (s,), generator=g, device="cuda", dtype=torch.int32)
    packed = Block8KVCache.from_dense(key, value, lengths=lengths, block_tokens=32, code_dtype=torch.int8)
    grown = Block8KVCache.empty(s, 3, h, 64, block_tokens=32, code_dtype=torch.int8)
    grown.append(key, value, counts=lengths)
    assert torch.equal(packed.lengths, lengths) and torch.equal(grown.lengths, lengths)
    some = lengths > 0
    for name in ("key_code", "value_code", "key_scale", "value_scale", "key_bounds"):
        assert torch.equal(getattr(packed, name)[some], getattr(grown, name)[some]), name
    small = Block8KVCache.from_dense(key[-9:], value[-9:], lengths=lengths[-9:].clone(), block_tokens=32, code_dtype=torch.int8)
    want = small.dequantize()
    for cache in (packed, grown):
        k, v = cache.dequantize()
        assert torch.equal(k[-9:, :3], want[0]) and torch.equal(v[-9:, :3], want[1])
        # codes are within half a step of the rows: amax / 254, and half a step of bf16
        live = torch.arange(3, device=device) < lengths[:, None]
        for rows, restored in ((key, k), (value, v)):
            bound = rows.float().abs().amax(dim=(1, 3), keepdim=True) * (1 / 254 + 2.0 ** -8)
            assert ((rows.float() - restored[:, :3].float()).abs()[live] <= bound.expand_as(rows)[live]).all()
            assert not restored[:, :3][~live].any()


@pytest.mark.parametrize("lq", [1, 3, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mixed_attention_over_heads_of_64_channels(device, lq, dtype):
    # dense rows and 8-bit segments, few and many query rows of a KV head
    from unicache_amd.adapters.bagel import run_batched_physical_attention, run_fused_mixed_attention

    dk, dv = (t[0] for t in dense(1, 130, 4, 64, seed=117, dtype=dtype))
    bk, bv = dense(1, 200, 4, 64, seed=118, dtype=dtype)
    block8 = Block8KVCache.from_dense(bk, bv)
    ek, ev = ((c.float().double() * sc.double().repeat_interleave(64, dim=2)[..., None])[0, :, :200].transpose(0, 1)
              for c, sc in ((block8.key_code, block8.key_scale),
                            (block8.value_code.float().transpose(3, 4).reshape(1, 4, -1, 64), block8.value_scale)))
    q = queries(1, lq, 28, 64, seed=119, dtype=dtype)[0] * 0.3
    out, lse = run_fused_mixed_attention(q, dk, dv, [block8], return_lse=True)
    k = torch.cat([dk.double(), ek]).repeat_interleave(7, dim=1)
    v = torch.cat([dv.double(), ev]).repeat_interleave(7, dim=1)
    x = torch.einsum("rhd,thd->hrt", q.double(), k) / 8
    p = torch.softmax(x, dim=-1)
    want, spread = (torch.einsum("hrt,thd->rhd", p, t) for t in (v, v.abs()))
    # weights rounded to 16 bits (half a step of the type at most), each summary's output and the merged one
    # likewise, and fp32 sums: three roundings relative to the sum of magnitudes, and a fourth for their products
    assert ((out.double() - want).abs() <= 4 * EPS[dtype] * spread + 1e-6).all()
    # logits: 64 products and as many sums in fp32, over the largest sum of magnitudes; the sums of weights.  Of many
    # rows the dense kernel sums the weights that it has rounded to the rows' type, (1 + e) p with |e| <= EPS for each:
    # their sum is within EPS of the exact one, relatively, so its logarithm within -log(1 - EPS) <= 1.01 EPS, and the
    # merged one, in which the dense part weighs 1 at most, no farther
    size = (torch.einsum("rhd,thd->hrt", q.double().abs(), k.abs()) / 8).amax(dim=-1)
    off = 72 * 2.0 ** -24 * size + 400 * 2.0 ** -23 + 64 * 2.0 ** -23 + (1.01 * EPS[dtype] if lq * 7 > 16 else 0)
    assert ((lse.double() - torch.logsumexp(x, dim=-1)).abs() <= off).all()
    assert torch.equal(run_batched_physical_attention(q, dk, dv, [0, lq], [0, 130], [[block8]]), out)


@pytest.mark.parametrize("lq", [1, 40])
def test_a_long_context_of_zeros_before_a_few_values(device, lq):
    # 2^21 keys in blocks whose value scale is 0, then 64 real ones; zero queries, so that every key weighs the same
    n, d = (1 << 21) + 64, 64
    cache = Block8KVCache.empty(1, n, 1, d, block_tokens=64, code_dtype=torch.int8)
    key, value = dense(1, 64, 1, d, seed=141)
    last = Block8KVCache.from_dense(key, value, block_tokens=64, code_dtype=torch.int8)
    for name in ("key_code", "value_code", "key_scale", "value_scale", "key_bounds"):
        getattr(cache, name).zero_()
    cache.key_code[:, :, -64:] = last.key_code
    for name in ("value_code", "key_scale", "value_scale", "key_bounds"):
        getattr(cache, name)[:, :, -1] = getattr(last, name)[:, :, 0]
    q = torch.zeros(1, lq, 8, d, dtype=torch.bfloat16, device=device)
    values = (last.value_code[0, 0, 0].double() * last.value_scale[0, 0, 0].double()).cpu()  # [D, 64]
    for tokens in (n, n - 64):
        cache.lengths.fill_(tokens)
        out, lse = cache.attention(q)
        # fp32 sums in one lane: 2^15 tiles at most, and 2^10 terms of a tile and of the joins; the logarithm's half steps
        off = (2 ** 15 + 2 ** 10) * 2.0 ** -24 + 2.0 ** -16
        assert (lse.double() - math.log(tokens)).abs().max() <= off
        want, size = (t.sum(dim=1) / tokens if tokens == n else torch.zeros(d).double() for t in (values, values.abs()))
        err = (out.double().cpu() - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + (off + 2.0 ** -11) * size + 448 * 2.0 ** -88).all()
