"""The paged KV cache (PagedKVCache) and rotary positions of several axes
(MultiAxisRotary) against 64-bit arithmetic: attention and rotation within the
roundings they make, pages, copies and tables exactly."""

import math

import pytest
import torch

from unicache_amd.operators import MultiAxisRotary
from unicache_amd.storage import PagedKVCache

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}    # half a step, relative
WEIGHT = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}  # of a weight held as two such numbers


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def randn(*shape, seed, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ------------------------------------------------------------- a model of it --
class Model:
    """The pool's bookkeeping on lists; `rows` gives each page's rows an id for what was written there."""

    def __init__(self, sequences, pages, width, b):
        self.b, self.width, self.p = b, width, pages
        self.pages = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.refs = [0] * pages
        self.rows = [[None] * b for _ in range(pages)]

    def take(self):
        free = [p for p in range(self.p) if self.refs[p] == 0]
        if not free:
            return None
        self.refs[free[0]] = 1
        return free[0]

    def drop(self, page):
        self.refs[page] -= 1

    def need(self, n):
        return -(-n // self.b)

    def reserve(self, counts):
        granted = []
        before = list(self.lengths)
        for s, c in enumerate(counts):
            n = min(before[s] + c, self.width * self.b)
            while len(self.pages[s]) < self.need(n):
                page = self.take()
                if page is None:
                    break
                self.pages[s].append(page)
            self.lengths[s] = min(n, len(self.pages[s]) * self.b)
            granted.append(self.lengths[s] - before[s])
        return granted

    def write(self, granted, ids):
        for s, n in enumerate(granted):
            for i in range(n):
                t = self.lengths[s] - n + i
                self.rows[self.pages[s][t // self.b]][t % self.b] = ids[s][i]

    def contents(self, s):
        return [self.rows[self.pages[s][t // self.b]][t % self.b] for t in range(self.lengths[s])]

    def reorder(self, parents, cut=None):
        n = len(parents)
        old, lengths = [list(p) for p in self.pages], list(self.lengths)
        for s, p in enumerate(parents):
            there = 0 <= p < n
            self.lengths[s] = min(lengths[p], max(cut[s], 0)) if there and cut else lengths[p] if there else 0
            self.pages[s] = old[p][:self.need(self.lengths[s])] if there else []
        self.refs = [sum(x in pages for pages in self.pages) for x in range(self.p)]
        opens = [self.pages[s][-1] if self.lengths[s] % self.b else None for s in range(n)]
        copies = []
        for s in range(n):
            if opens[s] is None:
                continue
            holders = [x for x in range(n) if opens[s] in self.pages[x]]
            whole = any(opens[x] != opens[s] for x in holders)
            if whole or min(holders) != s:
                copies.append(s)
        for s in copies:
            page = self.take()
            self.drop(opens[s])
            if page is None:
                self.pages[s].pop()
                self.lengths[s] -= self.lengths[s] % self.b
            else:
                r = self.lengths[s] % self.b
                self.rows[page][:r] = self.rows[opens[s]][:r]
                self.pages[s][-1] = page

    def compact(self, keep):
        free = self.refs.count(0)
        plans = []
        for s in range(len(self.pages)):
            kept = [t for t in range(self.lengths[s]) if t >= len(keep[s]) or keep[s][t]]
            if len(kept) == self.lengths[s]:
                continue
            whole = next(i for i, t in enumerate([*kept, -1]) if t != i) // self.b
            free -= max(self.need(len(kept)) - whole, 0)
            if free < 0:
                break
            plans.append((s, kept, whole))
        moved = []
        for s, kept, whole in plans:
            contents = self.contents(s)
            new = [self.take() for _ in range(whole, self.need(len(kept)))]
            moved.append((s, whole, new))
            for j in range(whole * self.b, len(kept)):
                self.rows[new[j // self.b - whole]][j % self.b] = contents[kept[j]]
            self.lengths[s] = len(kept)
        for s, whole, new in moved:
            for page in self.pages[s][whole:]:
                self.drop(page)
            self.pages[s] = self.pages[s][:whole] + new


def agrees(cache, model, store):
    """The device's state is the model's; store: id -> (key rows, value rows) [L, Hkv, D]."""

    assert cache.lengths.tolist() == model.lengths
    want = [p + [-1] * (model.width - len(p)) for p in model.pages]
    assert cache.table.tolist() == want
    assert cache.references.tolist() == model.refs
    bits = [(w >> i) & 1 for w in cache.free_pages.tolist() for i in range(32)][:model.p]
    assert bits == [int(r == 0) for r in model.refs]
    longest = max(model.lengths)
    if store is None or not longest:
        return
    cache.max_tokens = max(cache.max_tokens, longest)
    for layer in range(cache.layers):
        key, value = (t.cpu() for t in cache.dense(layer=layer))
        for s, n in enumerate(model.lengths):
            ids = model.contents(s)
            if n:
                assert torch.equal(key[s, :n], torch.stack([store[i][0][layer] for i in ids]))
                assert torch.equal(value[s, :n], torch.stack([store[i][1][layer] for i in ids]))
            assert not key[s, n:].any() and not value[s, n:].any()


def filled(lengths, *, hkv=2, d=64, b=16, layers=1, pages=None, width=None, dtype=torch.bfloat16, seed=0, shuffle=True):
    """A cache with sequences of these lengths in scattered pages, NaN everywhere else, and their rows [S, T, Hkv, D] of layer 0."""

    need = [-(-n // b) for n in lengths]
    pages = sum(need) + 3 if pages is None else pages
    width = max(max(need), 1) + 1 if width is None else width
    g = torch.Generator().manual_seed(seed)
    order = (torch.randperm(pages, generator=g) if shuffle else torch.arange(pages)).tolist()
    key = torch.full((layers, pages, hkv, b, d), float("nan"), dtype=dtype)
    value = key.clone()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    t_max = max(max(lengths), 1)
    rows_k = torch.randn(len(lengths), t_max, hkv, d, generator=g).to(dtype)
    rows_k[..., :4] *= 6
    rows_v = torch.randn(len(lengths), t_max, hkv, d, generator=g).to(dtype)
    at = 0
    for s, n in enumerate(lengths):
        for i in range(need[s]):
            page = order[at]
            at += 1
            table[s, i] = page
            r = min(b, n - i * b)
            key[:, page, :, :r] = rows_k[s, i * b:i * b + r].transpose(0, 1)
            value[:, page, :, :r] = rows_v[s, i * b:i * b + r].transpose(0, 1)
    cache = PagedKVCache(key.cuda(), value.cuda(), table.cuda(), i32(lengths), max_tokens=t_max)
    return cache, rows_k, rows_v


def attend64(q, rows_k, rows_v, seen, sm_scale, dtype):
    """One sequence in 64 bits, and what the kernel's roundings may add: q [Lq, Hq, D], rows [T, Hkv, D],
    seen [Lq, T] of booleans."""

    lq, hq, d = q.shape
    group = hq // rows_k.shape[1]
    # more than 64 rows of a KV head: each weight is rounded to one 16-bit number
    weight = EPS[dtype] if lq * group > 64 else WEIGHT[dtype]
    out, lse = torch.zeros(lq, hq, d, dtype=torch.float64), torch.full((hq, lq), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    t = rows_k.shape[0]
    for h in range(hq):
        k, v = rows_k[:, h // group].double(), rows_v[:, h // group].double()
        for i in range(lq):
            at = seen[i].nonzero().view(-1)
            if not len(at):
                continue
            x = (k[at] @ q[i, h].double()) * sm_scale
            # products summed in fp32 in any order, the scale, and the exponent's own rounding
            delta = ((d + 4) * 2.0 ** -24 * (k[at].abs() @ q[i, h].double().abs()) * sm_scale + 2.0 ** -22 * x.abs()).max()
            lse[h, i] = torch.logsumexp(x, 0)
            w = torch.exp(x - lse[h, i])
            out[i, h] = w @ v[at]
            spread = w @ v[at].abs()
            # weights as one or two 16-bit numbers (fp16: and half of 2^-24 where they are below its steps, the
            # largest being 2^6 at least), 1 ulp of the exponential, sums of t terms and their joins
            out_tol[i, h] = (EPS[dtype] * out[i, h].abs() + (weight + 2 * delta + (t + 64) * 2.0 ** -23) * spread
                             + 2.0 ** (-31 if lq * group <= 64 else -30) * v[at].abs().sum(0))
            lse_tol[h, i] = delta + (t + 64) * 2.0 ** -24 + 2.0 ** -21 * (1 + lse[h, i].abs())
    return out, lse, out_tol, lse_tol


def check_attention(cache, rows_k, rows_v, lengths, q, counts, causal, sm_scale=None, result=None, hidden=None):
    lq, d = q.shape[1], q.shape[3]
    query_lengths = None if counts is None else i32(counts)
    out, lse = result or cache.attention(q, query_lengths=query_lengths, causal=causal, sm_scale=sm_scale)
    scale = float(torch.tensor(sm_scale or 1 / math.sqrt(d), dtype=torch.float32))
    assert out.shape == q.shape and out.dtype == q.dtype and lse.dtype == torch.float32
    for s, n in enumerate(lengths):
        c = lq if counts is None else min(max(counts[s], 0), lq)
        seen = torch.zeros(lq, max(rows_k.shape[1], 1), dtype=torch.bool)
        for i in range(c):
            seen[i, :max(n - c + i + 1, 0) if causal else n] = True
        if hidden is not None:
            seen &= ~hidden[s]
        want, want_lse, tol, lse_tol = attend64(q[s].cpu(), rows_k[s], rows_v[s], seen, scale, q.dtype)
        got, got_lse = out[s].double().cpu(), lse[s].double().cpu()
        none = want_lse == -math.inf
        assert torch.equal(got_lse == -math.inf, none)
        assert not got[none.t()].any()
        over, over_lse = ((got - want).abs() - tol).max(), ((got_lse - want_lse).abs() - lse_tol)[~none]
        assert float(over) <= 0.0, s
        assert not len(over_lse) or float(over_lse.max()) <= 0.0, s


# --------------------------------------------------------------- attention --
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,d", [(16, 64), (16, 128), (32, 128), (64, 64), (128, 128), (256, 64)])
def test_decode_of_any_length(device, b, d, dtype):
    lengths = [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300, 2 * b, 2 * b + 1]
    cache, k, v = filled(lengths, d=d, b=b, dtype=dtype)
    q = randn(len(lengths), 1, 6, d, seed=1, dtype=dtype)
    check_attention(cache, k, v, lengths, q, None, False)


@pytest.mark.parametrize("hq,hkv,lq", [(7, 1, 1), (28, 4, 1), (8, 8, 1), (16, 1, 1), (16, 2, 3), (28, 4, 3), (8, 1, 5),
                                     (14, 2, 9), (64, 1, 1), (8, 2, 17), (40, 1, 2), (5, 5, 33), (96, 2, 3), (28, 4, 19),
                                     (4, 1, 33), (8, 2, 70), (64, 1, 5)])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_of_any_number(device, hq, hkv, lq, causal):
    # units of 16, 32 and 64 rows, one and several a head
    lengths, counts = [200, lq, 77, 5], [lq, lq, lq // 2, 0]
    for d, dtype, b in ((128, torch.bfloat16, 32), (64, torch.float16, 16)):
        cache, k, v = filled(lengths, hkv=hkv, d=d, b=b, dtype=dtype, seed=hq)
        q = randn(len(lengths), lq, hq, d, seed=2, dtype=dtype)
        check_attention(cache, k, v, lengths, q, counts, causal)
        check_attention(cache, k, v, lengths, q, None, causal)


@pytest.mark.parametrize("d,dtype,b,causal", [(128, torch.bfloat16, 16, True), (64, torch.float16, 64, True),
                                             (128, torch.float16, 32, False), (64, torch.bfloat16, 256, False)])
def test_chunks_of_prompts(device, d, dtype, b, causal):
    lengths, counts = [1500, 141, 700], [141, 141, 50]
    cache, k, v = filled(lengths, hkv=2, d=d, b=b, dtype=dtype)
    q = randn(3, 141, 4, d, seed=3, dtype=dtype)
    check_attention(cache, k, v, lengths, q, counts, causal)
    for hint in (1, 300):  # one split of the keys, and as many as a shorter sequence would have
        cache.max_tokens = hint
        check_attention(cache, k, v, lengths, q, counts, causal)


def test_few_rows_over_many_keys_in_tiles(device):
    # a short chunk behind a long prefix: the keys are split
    lengths = [9000, 30]
    cache, k, v = filled(lengths, hkv=1, d=128, b=64)
    q = randn(2, 11, 7, 128, seed=3)
    check_attention(cache, k, v, lengths, q, None, True)


def test_many_row_groups_of_many_sequences(device):
    # more row groups than the workgroups share out: one workgroup each
    s, lq = 2100, 130
    lengths = [(37 * i) % 190 for i in range(s)]
    cache, k, v = filled(lengths, hkv=1, d=64, b=16)
    q = randn(s, lq, 1, 64, seed=3)
    counts = [n % (lq + 1) for n in lengths]
    out, lse = cache.attention(q, query_lengths=i32(counts), causal=True)
    some = [0, 1, 5, 700, 2099]
    few = [lengths[i] for i in some]
    check_attention(cache, k[some], v[some], few, q[some], [counts[i] for i in some], True, result=(out[some], lse[some]))


def test_many_sequences_share_the_workgroups(device):
    # more sequences than a wave has lanes, empty ones among them; max_tokens far from the truth
    lengths = [(37 * i) % 260 if i % 3 else 0 for i in range(131)]
    cache, k, v = filled(lengths, hkv=1, d=64, b=16)
    q = randn(len(lengths), 1, 2, 64, seed=3)
    for hint in (1, 260, 100000):
        cache.max_tokens = min(hint, cache.capacity)
        check_attention(cache, k, v, lengths, q, None, True)


def test_long_sequence_split_and_joined(device):
    lengths = [20011, 9]
    cache, k, v = filled(lengths, hkv=1, d=128, b=64)
    q = randn(2, 1, 4, 128, seed=4)
    check_attention(cache, k, v, lengths, q, None, False)
    for hint in (1, 700, 5000):  # one workgroup, few, many
        cache.max_tokens = hint
        check_attention(cache, k, v, lengths, q, None, False)


@pytest.mark.parametrize("b", [16, 32, 128])
def test_entries_that_are_no_pages_hide_their_tokens(device, b):
    lengths = [5 * b + 3, 4 * b]
    cache, k, v = filled(lengths, hkv=2, d=64, b=b)
    hidden = torch.zeros(2, k.shape[1], dtype=torch.bool)
    # (few rows, and tiles of many)
    for s, i, entry in ((0, 1, -1), (0, 4, cache.pages), (1, 0, 2 ** 31 - 1), (1, 1, -7), (1, 2, -2 ** 31), (1, 3, -1)):
        cache.table[s, i] = entry
        hidden[s, i * b:(i + 1) * b] = True
    for lq in (3, 40):
        q = randn(2, lq, 4, 64, seed=5)
        check_attention(cache, k, v, lengths, q, None, True, hidden=hidden)
    cache.lengths.copy_(i32([-5, 2 ** 31 - 1]))  # read as 0 and as the capacity
    out, lse = cache.attention(q)
    assert not out[0].any() and (lse[0] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,lq", [(2, 5), (4, 21), (7, 30)])
def test_what_a_row_does_not_see_never_reaches_it(device, dtype, hq, lq):
    # the newest keys and values are not finite: rows before them are as if they were zeros
    lengths = [100, 64]
    cache, k, v = filled(lengths, hkv=1, d=64, b=16, dtype=dtype)
    bad_k, bad_v = k.clone(), v.clone()
    for s, n in enumerate(lengths):
        bad_k[s, n - 1, 0, 3] = math.nan
        bad_v[s, n - 1, 0, :] = math.inf
        bad_v[s, n - 1, 0, 5] = math.nan
        bad_v[s, n - 2, 0, 7] = -math.inf
    rewritten, _, _ = filled([0, 0], hkv=1, d=64, b=16, dtype=dtype)
    table = cache.table.cpu()
    key, value = cache.key.clone(), cache.value.clone()
    for s, n in enumerate(lengths):
        for t in (n - 2, n - 1):
            key[0, table[s, t // 16], :, t % 16], value[0, table[s, t // 16], :, t % 16] = bad_k[s, t], bad_v[s, t]
    dirty = PagedKVCache(key, value, cache.table, cache.lengths, max_tokens=100)
    q = randn(2, lq, hq, 64, seed=6, dtype=dtype)
    out, lse = dirty.attention(q, causal=True)
    clean, clean_lse = cache.attention(q, causal=True)
    assert torch.equal(out[:, :lq - 2], clean[:, :lq - 2]) and torch.equal(lse[:, :, :lq - 2], clean_lse[:, :, :lq - 2])
    # the row that sees the infinite value has it, and its other channels; the last row sees a key that is NaN
    assert (out[:, lq - 2, :, 7] == -math.inf).all()
    other = [c for c in range(64) if c != 7]
    want = torch.isfinite(out[:, lq - 2][..., other].float())
    assert want.all()
    assert out[:, lq - 1].isnan().all() and lse[:, :, lq - 1].isnan().all()
    assert torch.equal(lse[:, :, lq - 2], clean_lse[:, :, lq - 2])


def test_large_logits_and_scales(device):
    lengths = [333]
    cache, k, v = filled(lengths, hkv=1, d=128, b=32, dtype=torch.float16)
    q = randn(1, 2, 3, 128, seed=7, dtype=torch.float16, scale=40.0)
    check_attention(cache, k, v, lengths, q, None, False, sm_scale=0.5)
    check_attention(cache, k, v, lengths, q * 0, None, False, sm_scale=1e-3)
    check_attention(cache, k, v, lengths, q, None, False, sm_scale=1e-30)
    # logits past fp32's range are no numbers, and no zeros
    for lq in (2, 40):
        out, lse = cache.attention(randn(1, lq, 3, 128, seed=7, dtype=torch.float16, scale=40.0), sm_scale=2.0 ** 127)
        assert out.isnan().all() and lse.isnan().all()


def test_strides_offsets_and_views(device):
    lengths = [130, 40]
    cache, k, v = filled(lengths, hkv=2, d=64, b=32)
    big = randn(2, 4, 3, 5, 64, seed=8)
    for q in (big[:, :, 1], big[:, 1:3, :, 4].transpose(1, 2)[:, :, :2], big[:, ::2, 2, 1:5], big.transpose(1, 2)[:, 1, :3, :4],
              randn(2, 2, 4, 72, seed=9)[..., 3:67]):
        if q.shape[2] % 2:
            q = q[:, :, :2]
        check_attention(cache, k, v, lengths, q, None, True)


def test_pool_larger_than_32_bits(device):
    # pages whose rows lie past 2^32 elements
    pages, b, hkv, d = 70000, 64, 8, 128
    key = torch.zeros(1, pages, hkv, b, d, dtype=torch.bfloat16, device=device)
    value = torch.zeros_like(key)
    ids = [69999, 3, 65537, 69001]
    g = torch.Generator(device=device).manual_seed(0)
    for page in ids:
        key[0, page] = torch.randn(hkv, b, d, generator=g, device=device)
        value[0, page] = torch.randn(hkv, b, d, generator=g, device=device)
    cache = PagedKVCache(key, value, i32([ids]), i32([250]), max_tokens=256)
    k = key[0, ids].transpose(1, 2).reshape(1, -1, hkv, d)[:, :250].cpu()
    v = value[0, ids].transpose(1, 2).reshape(1, -1, hkv, d)[:, :250].cpu()
    q = randn(1, 1, 8, d, seed=10)
    check_attention(cache, k, v, [250], q, None, False)
    rows = randn(1, 2, hkv, d, seed=11)
    cache.write(rows, rows * 2, counts=i32([2]))
    assert torch.equal(cache.key[0, 69001, :, 56:58], rows[0].transpose(0, 1))
    assert torch.equal(cache.value[0, 69001, :, 56:58], rows[0].transpose(0, 1) * 2)


# ------------------------------------------------------------------ rotary --
def turned64(x, positions, sections, pairing, frequencies=None, theta=10000.0, axes=None):
    pairs = sum(sections)
    freq = [theta ** (-i / pairs) for i in range(pairs)] if frequencies is None else frequencies
    axes = axes or [a for a, n in enumerate(sections) for _ in range(n)]
    y = x.double().cpu()
    out, size = y.clone(), torch.zeros_like(y)
    for i in range(pairs):
        a, b = (i, i + pairs) if pairing == "halves" else (2 * i, 2 * i + 1)
        angle = (positions[axes[i]].cpu().double() * freq[i])[..., None]
        out[..., a] = y[..., a] * angle.cos() - y[..., b] * angle.sin()
        out[..., b] = y[..., b] * angle.cos() + y[..., a] * angle.sin()
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def check_turned(got, x, positions, sections, pairing, **kwargs):
    want, size = turned64(x, positions, sections, pairing, **kwargs)
    # sines, cosines and the products in fp32 (2^-21 of both channels), one rounding.  The oracle's own angles are
    # doubles: below 2^21 radians to 2^-31
    over = ((got.double().cpu() - want).abs() - EPS[x.dtype] * want.abs() - 2.0 ** -21 * size).max()
    assert float(over) <= 0.0
    assert torch.equal(got[..., 2 * sum(sections):], x[..., 2 * sum(sections):])


@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("d,sections", [(128, (16, 24, 24)), (64, (16, 16)), (64, (32,)), (128, (8, 0, 16)), (16, (3, 5)),
                                       (80, (5, 20, 7)), (512, (100, 56, 100)), (48, (8,))])
def test_rotary_turns_pairs_by_their_axis(device, d, sections, pairing):
    for dtype, int_type, s, n in ((torch.bfloat16, torch.int64, 2, 37), (torch.float16, torch.int32, 1, 1)):
        g = torch.Generator().manual_seed(d)
        positions = torch.randint(-500, 40000, (len(sections), s, n), generator=g).to(int_type).cuda()
        q, k = randn(s, n, 5, d, seed=1, dtype=dtype), randn(s, n, 2, d, seed=2, dtype=dtype)
        rotary = MultiAxisRotary(d, sections, pairing=pairing)
        a, b = rotary.rotate(q, k, positions=positions)
        check_turned(a, q, positions, sections, pairing)
        check_turned(b, k, positions, sections, pairing)
        assert torch.equal(rotary.rotate(q, positions=positions), a)
        if s == 1:
            flat = rotary.rotate(q[0], k[0], positions=positions[:, 0])
            assert torch.equal(flat[0], a[0]) and torch.equal(flat[1], b[0])


def test_rotary_far_positions_and_long_inputs(device):
    sections = (16, 24, 24)
    # more tokens than one launch's short form takes; places at which fp32 angles would be useless
    positions = torch.stack([torch.arange(3001) * 331 % 1009, torch.arange(3001) + 2 ** 20, torch.arange(3001) % 7 - 3])[:, None].cuda()
    q, k = randn(1, 3001, 3, 128, seed=3), randn(1, 3001, 1, 128, seed=4)
    a, b = MultiAxisRotary(128, sections, theta=1e6).rotate(q, k, positions=positions)
    check_turned(a, q, positions, sections, "halves", theta=1e6)
    check_turned(b, k, positions, sections, "halves", theta=1e6)
    far = torch.full((3, 1, 1), 2 ** 31 - 1, dtype=torch.int64, device=device)
    ones = torch.ones(1, 1, 1, 128, dtype=torch.float16, device=device)
    # whole turns come off exactly where the frequency is a power of two of a turn
    freq = [2.0 * math.pi / 4.0] * 64
    out = MultiAxisRotary(128, sections, frequencies=freq).rotate(ones, positions=far)  # 2^31 - 1 = -1 quarters
    assert torch.allclose(out[..., :64].float(), torch.ones(64, device=device)) and torch.allclose(
        out[..., 64:].float(), -torch.ones(64, device=device))


def test_rotary_axes_frequencies_inverse_and_gradient(device):
    sections, axes = (4, 4), [0, 1] * 4
    freq = [0.5 * i for i in range(8)]
    positions = torch.randint(0, 300, (2, 1, 33), generator=torch.Generator().manual_seed(0)).cuda()
    q = randn(1, 33, 4, 32, seed=5, dtype=torch.float16)
    rotary = MultiAxisRotary(32, sections, frequencies=freq, axes=axes)
    out = rotary.rotate(q, positions=positions)
    check_turned(out, q, positions, sections, "halves", frequencies=freq, axes=axes)
    back = rotary.rotate(q, positions=positions, inverse=True)
    check_turned(back, q, -positions, sections, "halves", frequencies=freq, axes=axes)
    # the turn back is the transpose: <turn x, y> = <x, turn back y> to the roundings of both
    y = randn(1, 33, 4, 32, seed=6, dtype=torch.float16)
    left = (out.double() * y.double()).sum(-1)
    right = (q.double() * rotary.rotate(y, positions=positions, inverse=True).double()).sum(-1)
    bound = 4 * EPS[torch.float16] * (q.double().norm(dim=-1) * y.double().norm(dim=-1)) * math.sqrt(2)
    assert ((left - right).abs() <= bound).all()


def test_rotary_views(device):
    positions = torch.arange(24, device=device).view(2, 2, 6)
    big = randn(2, 6, 4, 3, 64, seed=7)
    rotary = MultiAxisRotary(64, (16, 16))
    for x in (big[:, :, 1], big[:, :, ::2, 1], big.transpose(1, 2)[:, 1], randn(2, 6, 2, 72, seed=8)[..., 3:67]):
        check_turned(rotary.rotate(x, positions=positions), x, positions, (16, 16), "halves")
    some = positions.transpose(1, 2).contiguous().transpose(1, 2)  # not contiguous
    assert torch.equal(rotary.rotate(big[:, :, 1], positions=some), rotary.rotate(big[:, :, 1], positions=positions))


# ------------------------------------------------------------------- write --
@pytest.mark.parametrize("b,d", [(16, 64), (32, 128), (256, 64)])
@pytest.mark.parametrize("with_query", [False, True])
def test_write_puts_turned_rows_in_their_places(device, b, d, with_query):
    s, n, hkv, hq = 4, 2 * b + 5, 2, 6
    lengths, counts = [n + 40, n, 3 * b, 7], [n, n - 1, 0, 5]
    cache, k, v = filled(lengths, hkv=hkv, d=d, b=b, layers=3)
    before = cache.key.clone(), cache.value.clone()
    key, value = randn(s, n, hkv, d, seed=1), randn(s, n, hkv, d, seed=2)
    query = randn(s, n, hq, d, seed=3) if with_query else None
    sections = (d // 8, d // 8, d // 4)
    rotary = MultiAxisRotary(d, sections)
    positions = torch.randint(0, 9000, (3, s, n), generator=torch.Generator().manual_seed(0)).cuda()
    for where in (positions, None):
        if where is None:  # each token's place
            where = torch.stack([torch.arange(n) + lengths[i] - counts[i] for i in range(s)]).cuda().expand(3, s, n)
        out = cache.write(key, value, layer=1, query=query, rotary=rotary, counts=i32(counts),
                          positions=positions if where is positions else None)
        if with_query:
            check_turned(out, query, where, sections, "halves")
        else:
            assert out is None
        want = rotary.rotate(key, positions=where)
        check_turned(want, key, where, sections, "halves")
        want_k, want_v = before[0].clone(), before[1].clone()
        for i in range(s):
            for j in range(counts[i]):
                t = lengths[i] - counts[i] + j
                page = int(cache.table[i, t // b])
                want_k[1, page, :, t % b], want_v[1, page, :, t % b] = want[i, j], value[i, j]
        # (bits, since unused rows are NaN)
        assert torch.equal(cache.key.view(torch.int16), want_k.view(torch.int16))
        assert torch.equal(cache.value.view(torch.int16), want_v.view(torch.int16))


def test_write_skips_what_has_no_place(device):
    # counts past the rows, past the length, entries that are no page; no rotary
    b, n = 16, 20
    cache, _, _ = filled([50, 10, 40], b=b, hkv=1)
    before = cache.key.clone()
    cache.table[2, 1] = -1
    cache.table[2, 2] = cache.pages
    rows = randn(3, n, 1, 64, seed=1)
    cache.write(rows, rows, counts=i32([99, 15, 20]))
    want = before.clone()
    for s, length, count in ((0, 50, 20), (1, 10, 15), (2, 40, 20)):
        for j in range(count):
            t = length - count + j
            page = int(cache.table[s, t // b]) if t >= 0 else -1
            if 0 <= page < cache.pages:
                want[0, page, :, t % b] = rows[s, j]
    assert torch.equal(cache.key.view(torch.int16), want.view(torch.int16))


# ------------------------------------------------------------------- pages --
def test_reserve_write_and_the_end_of_the_pool(device):
    cache = PagedKVCache.empty(3, 7, 2, 64, layers=2, page_tokens=16, sequence_pages=4)
    model, store = Model(3, 7, 4, 16), {}
    agrees(cache, model, None)
    for step, counts in enumerate([[5, 0, 16], [12, 33, 0], [0, 0, 20], [1, 1, 1], [60, 60, 60], [0, 0, 0], [3, 3, 3]]):
        n = max(max(counts), 1)
        got = cache.reserve(n, counts=i32(counts)).tolist()
        granted = model.reserve(counts)
        assert got == granted
        ids = [[(step, s, i) for i in range(n)] for s in range(3)]
        k, v = randn(2, 3, n, 2, 64, seed=step), randn(2, 3, n, 2, 64, seed=100 + step)
        for layer in range(2):
            cache.write(k[layer], v[layer], layer=layer)
        for s in range(3):
            for i in range(n):
                store[(step, s, i)] = k[:, s, i].cpu(), v[:, s, i].cpu()
        model.write(granted, ids)
        agrees(cache, model, store)
    cache.reserve(4)
    model.reserve([4, 4, 4])
    agrees(cache, model, None)


@pytest.mark.parametrize("seed,b,pages,room", [(0, 16, 40, 0), (1, 16, 9, 0), (2, 32, 16, 0), (3, 16, 70, 0), (4, 64, 12, 0),
                                               (5, 16, 40, 900), (6, 32, 20, 900)])
def test_any_order_of_calls_keeps_the_books(device, seed, b, pages, room):
    # (with room the table is more than one workgroup takes in reorder)
    import random

    rng = random.Random(seed)
    s, width = 5, 6 + room
    cache = PagedKVCache.empty(s, pages, 1, 64, layers=2, page_tokens=b, sequence_pages=width, dtype=torch.float16)
    hints = (1, 4096, cache.capacity)
    model, store = Model(s, pages, width, b), {}
    for step in range(30):
        cache.max_tokens = hints[step % 3] if room else cache.max_tokens
        call = rng.choice(["reserve", "reserve", "reserve", "reorder", "truncate", "compact", "cut"])
        if call == "reserve":
            counts = [rng.choice([0, 1, b // 2, b, 2 * b + 3]) for _ in range(s)]
            n = max(max(counts), 1)
            assert cache.reserve(n, counts=i32(counts)).tolist() == (granted := model.reserve(counts))
            k = randn(2, s, n, 1, 64, seed=1000 * seed + step, dtype=torch.float16)
            for layer in range(2):
                cache.write(k[layer], -k[layer], layer=layer)
            host = k.cpu()
            for i in range(s):
                for j in range(n):
                    store[(step, i, j)] = host[:, i, j], -host[:, i, j]
            model.write(granted, [[(step, i, j) for j in range(n)] for i in range(s)])
        elif call in ("reorder", "cut"):
            parents = [rng.choice([i, i, rng.randrange(s), rng.randrange(s), -1, s]) for i in range(s)]
            cut = [rng.choice([-1, 0, rng.randrange(6 * b), width * b]) for _ in range(s)] if call == "cut" else None
            cache.reorder(i32(parents), lengths=None if cut is None else i32(cut))
            model.reorder(parents, cut)
        elif call == "truncate":
            cut = [max(0, n - rng.choice([0, 0, 1, 3, b])) for n in model.lengths]
            cache.truncate(i32(cut))
            model.reorder(list(range(s)), cut)
        else:
            t = rng.choice([0, b, 3 * b, 6 * b])
            p = rng.choice([0.0, 0.5, 0.95, 1.0])
            keep = [[rng.random() < p if i != 2 else True for _ in range(t)] for i in range(s)]
            cache.compact(torch.tensor(keep, dtype=torch.bool, device=device).view(s, t))
            model.compact(keep)
        agrees(cache, model, store)


def test_fork_then_grow_leaves_the_parent_alone(device):
    b = 16
    cache = PagedKVCache.empty(4, 64, 2, 64, page_tokens=b)
    model, store = Model(4, 64, 64, b), {}

    def grow(counts, seed):
        n = max(counts)
        granted = cache.reserve(n, counts=i32(counts))
        assert granted.tolist() == model.reserve(counts) == counts
        k = randn(4, n, 2, 64, seed=seed)
        cache.write(k, -k)
        for s in range(4):
            for i in range(n):
                store[(seed, s, i)] = k[s, i].cpu()[None], -k[s, i].cpu()[None]
        model.write(counts, [[(seed, s, i) for i in range(n)] for s in range(4)])

    grow([40, 0, 0, 32], 1)
    for parents in ([0, 0, 0, 3], [2, 1, 0, 3], [3, 3, 0, 3], [0, 1, 2, -1]):
        cache.reorder(i32(parents))
        model.reorder(parents)
        agrees(cache, model, store)
        grow([3, 5, 1, 2], 10 + sum(parents))
        agrees(cache, model, store)
    # a shared whole page cut open again is copied before anyone writes there
    cache.reorder(i32([1, 1, 1, 1]))
    model.reorder([1, 1, 1, 1])
    cache.truncate(i32([20, 1000, 20, 5]))
    model.reorder([0, 1, 2, 3], [20, 1000, 20, 5])
    agrees(cache, model, store)
    grow([2, 2, 2, 2], 99)
    agrees(cache, model, store)


def test_compact_with_uint8_strided_and_short_masks(device):
    b = 16
    cache = PagedKVCache.empty(2, 40, 1, 64, page_tokens=b)
    k = randn(2, 90, 1, 64, seed=1)
    cache.reserve(90, counts=i32([90, 77]))
    cache.write(k, -k)
    mask = torch.zeros(2, 128, dtype=torch.uint8, device=device)
    mask[0, :17], mask[0, 30:60], mask[1, 3::5] = 1, 255, 7
    keep = mask[:, :64]  # tokens from 64 on stay
    want = [[*range(17), *range(30, 60), *range(64, 90)], [*range(3, 64, 5), *range(64, 77)]]
    cache.compact(keep)
    assert cache.lengths.tolist() == [len(w) for w in want]
    key, value = cache.dense()
    for s in range(2):
        assert torch.equal(key[s, :len(want[s])], k[s, want[s]]) and torch.equal(value[s, :len(want[s])], -k[s, want[s]])
    cache.compact(keep.t().contiguous().t()[:, :0])  # no column: all stay
    assert cache.lengths.tolist() == [len(w) for w in want]


def test_pool_of_many_pages(device):
    # more words of free pages, and more pages at a time, than one round of the workgroup takes
    pages = 33 * 1024 + 77
    cache = PagedKVCache.empty(3, pages, 1, 64, page_tokens=16)
    counts = [12000 * 16, 9000 * 16, 20000 * 16]
    got = cache.reserve(max(counts), counts=i32(counts)).tolist()
    assert got == [12000 * 16, 9000 * 16, (pages - 21000) * 16]
    table = cache.table.cpu()
    assert torch.equal(table[0, :12000], torch.arange(12000, dtype=torch.int32))
    assert torch.equal(table[1, :9000], torch.arange(12000, 21000, dtype=torch.int32))
    assert torch.equal(table[2, :pages - 21000], torch.arange(21000, pages, dtype=torch.int32))
    assert not cache.free_pages.any() and (cache.references == 1).all()
    cache.reorder(i32([0, -1, 2]))
    cache.truncate(i32([2 ** 31 - 1, 0, 16 * 5]))
    assert cache.reserve(16 * 3, counts=i32([0, 48, 48])).tolist() == [0, 48, 48]
    assert cache.table[1, :4].tolist() == [12000, 12001, 12002, -1]
    assert cache.table[2, :9].tolist() == [21000, 21001, 21002, 21003, 21004, 12003, 12004, 12005, -1]


# ---------------------------------------------------------------- together --
def test_steps_of_a_decode_loop_under_a_graph(device):
    """Reserve, write and attend for two layers, then refuse half of the tokens: captured once, replayed over changing
    rows with eager work between, and equal to the same calls made eagerly."""

    s, n, hkv, hq, d, b, layers = 3, 3, 2, 6, 128, 16, 2
    rotary = MultiAxisRotary(d, (16, 24, 24))

    def fresh():
        cache = PagedKVCache.empty(s, 60, hkv, d, layers=layers, page_tokens=b, sequence_pages=20)
        cache.reserve(20, counts=i32([20, 7, 0]))
        for layer in range(layers):
            rows = randn(s, 20, hkv, d, seed=50 + layer)
            cache.write(rows, -rows, layer=layer, rotary=rotary)
        return cache

    def step(cache, rows, query, cut):
        cache.reserve(n)
        outs = []
        for layer in range(layers):
            q = cache.write(rows[layer], -rows[layer], layer=layer, query=query[layer], rotary=rotary)
            outs.append(cache.attention(q, layer=layer, causal=True, query_lengths=cache.granted))
        torch.sub(cache.lengths, cut, out=cut)
        cache.truncate(cut)
        return outs

    eager, graphed = fresh(), fresh()
    rows, query = randn(layers, s, n, hkv, d, seed=1), randn(layers, s, n, hq, d, seed=2)
    cut = i32([1, 2, 0])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        warm = fresh()
        step(warm, rows, query, cut.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(graphed, rows, query, cut)
    for t in range(8):
        rows.copy_(randn(layers, s, n, hkv, d, seed=10 + t))
        query.copy_(randn(layers, s, n, hq, d, seed=30 + t))
        cut.copy_(i32([t % 3, (t + 1) % 4, 1]))
        want = step(eager, rows, query, cut.clone())
        graph.replay()
        torch.cuda.synchronize()
        for (o, l), (wo, wl) in zip(results, want):
            assert torch.equal(o, wo) and torch.equal(l, wl)
        for name in ("table", "lengths", "granted", "references", "free_pages"):
            assert torch.equal(getattr(eager, name), getattr(graphed, name)), name


def test_other_streams_and_determinism(device):
    lengths = [3000, 500]
    cache, k, v = filled(lengths, hkv=2, d=128, b=64)
    q = randn(2, 1, 14, 128, seed=1)
    want = cache.attention(q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for stream in streams * 2:
        with torch.cuda.stream(stream):
            got.append(cache.attention(q))
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])


def test_layer_views_and_rows_behind_the_end(device):
    cache = PagedKVCache.empty(2, 10, 2, 64, layers=3, page_tokens=32)
    cache.reserve(33, counts=i32([33, 2]))
    rows = randn(3, 2, 33, 2, 64, seed=1)
    for layer in range(3):
        view = cache.layer(layer)
        assert view.layers == 1 and view.max_tokens == 33
        view.write(rows[layer], -rows[layer], counts=cache.granted)
    for layer in range(3):
        key, value = cache.dense(layer=layer)
        assert torch.equal(key[0], rows[layer, 0]) and torch.equal(key[1, :2], rows[layer, 1, :2]) and not key[1, 2:].any()
        q = randn(2, 1, 4, 64, seed=2)
        a, b = cache.attention(q, layer=layer), cache.layer(layer).attention(q)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(RuntimeError, match="references"):
        cache.layer(0).reserve(1)
    # rows of one sequence without their first dimension
    one, want = cache.layer(2, sequence=0), cache.attention(q, layer=2)
    out, lse = one.attention(q[0])
    assert out.shape == (1, 4, 64) and lse.shape == (4, 1)
    assert torch.equal(out, want[0][0]) and torch.equal(lse, want[1][0])
    rotary = MultiAxisRotary(64, (32,))
    new = randn(2, 2, 64, seed=3)
    turned = one.write(new, -new, query=new, rotary=rotary)
    where = torch.tensor([[31, 32]], device=device)
    assert torch.equal(turned, rotary.rotate(new, positions=where))
    assert torch.equal(cache.dense(layer=2)[0][0, 31:33], turned) and torch.equal(cache.dense(layer=2)[1][0, 31:33], -new)


def test_tensors_may_be_replaced_by_their_like(device):
    cache, k, v = filled([100, 37], d=64, b=16)
    q = randn(2, 1, 4, 64, seed=1)
    want = cache.attention(q)
    cache.key, cache.value = cache.key.clone(), cache.value.clone()
    cache.table = cache.table.clone()
    again = cache.attention(q)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    lengths, cache.lengths = cache.lengths, i32([50, 37])
    check_attention(cache, k, v, [50, 37], q, None, False)
    cache.lengths, table = lengths, cache.table
    for name, bad, match in (("table", table[:, :2].contiguous(), "same sizes"), ("table", table.long(), "table"),
                             ("lengths", i32([1]), "lengths"), ("key", cache.key.half(), "value"),
                             ("key", cache.key[:, :2].contiguous(), "value")):
        good = getattr(cache, name)
        setattr(cache, name, bad)
        with pytest.raises(ValueError, match=match):
            cache.attention(q)
        setattr(cache, name, good)
    assert torch.equal(cache.attention(q)[0], want[0])


def test_empty_calls(device):
    cache = PagedKVCache.empty(2, 4, 1, 64, page_tokens=16)
    out, lse = cache.attention(randn(2, 0, 3, 64, seed=0))
    assert out.shape == (2, 0, 3, 64) and lse.shape == (2, 3, 0)
    out, lse = cache.attention(randn(2, 2, 3, 64, seed=0), causal=True)
    assert not out.any() and (lse == -math.inf).all()
    none = torch.empty(2, 0, 1, 64, dtype=torch.bfloat16, device=device)
    assert cache.write(none, none) is None
    assert cache.reserve(0).tolist() == [0, 0]
    rotary = MultiAxisRotary(64, (16, 16))
    q, k = rotary.rotate(none, none, positions=torch.empty(2, 2, 0, dtype=torch.int64, device=device))
    assert q.shape == k.shape == none.shape
    key, value = cache.dense()
    assert key.shape == (2, 0, 1, 64)
    cache.compact(torch.ones(2, 5, dtype=torch.bool, device=device))
    cache.truncate(i32([0, 0]))
    cache.reorder(i32([1, 0]))
    assert cache.lengths.tolist() == [0, 0] and (cache.table == -1).all()


@pytest.mark.parametrize("lq", [1, 3, 60])
def test_mixed_attention_over_paged_segments(device, lq):
    # the adapter's mixed call: dense rows, a packed KIVI segment and two sequences' pages as one softmax
    from unicache_amd.adapters.bagel import run_batched_physical_attention, run_fused_mixed_attention
    from unicache_amd.storage import PackedKIVICache

    dk, dv = randn(90, 4, 128, seed=1, scale=0.3), randn(90, 4, 128, seed=2)
    pk, pv = randn(300, 4, 128, seed=3, scale=0.3), randn(300, 4, 128, seed=4)
    packed = PackedKIVICache.from_dense(pk, pv, logical_token_ids=torch.arange(300, device=device), token_type_id=0,
                                        k_bits=4, v_bits=4, group_size=32, residual_length=10, backend="cuda")
    cache = PagedKVCache.empty(2, 20, 4, 128, layers=2, page_tokens=32)
    cache.reserve(150, counts=i32([150, 33]))
    rows = randn(2, 2, 150, 4, 128, seed=5, scale=0.3)
    values = randn(2, 2, 150, 4, 128, seed=6)
    for layer in range(2):
        cache.write(rows[layer], values[layer], layer=layer)
    first, second = cache.layer(1, sequence=0), cache.layer(1, sequence=1)
    rk, rv = packed.dequantize()
    q = randn(lq, 28, 128, seed=7)
    for segments, keys, vals in (([packed, first, second], [dk, rk, rows[1, 0], rows[1, 1, :33]],
                                  [dv, rv, values[1, 0], values[1, 1, :33]]), ([second], [dk, rows[1, 1, :33]], [dv, values[1, 1, :33]])):
        out, lse = run_fused_mixed_attention(q, dk, dv, segments, return_lse=True)
        k, v = (torch.cat([t.double().cpu() for t in ts]).repeat_interleave(7, dim=1) for ts in (keys, vals))
        x = torch.einsum("rhd,thd->hrt", q.double().cpu(), k) / math.sqrt(128)
        want = torch.einsum("hrt,thd->rhd", torch.softmax(x, dim=-1), v)
        # the tolerances of the other mixed-attention tests: summaries are rounded to bf16 before they are merged
        assert float((out.double().cpu() - want).abs().max()) < 2e-2
        assert float((lse.double().cpu() - torch.logsumexp(x, dim=-1)).abs().max()) < 5e-3
        batched = run_batched_physical_attention(q, dk, dv, [0, lq], [0, 90], [segments])
        assert torch.equal(batched, out)
    none = dk[:0]
    cache.truncate(i32([0, 5]))
    out, lse = run_fused_mixed_attention(q, none, none, [cache.layer(0, sequence=0)], return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    for bad in (cache, cache.layer(0)):
        with pytest.raises(ValueError, match="one layer of one sequence"):
            run_fused_mixed_attention(q, dk, dv, [bad])


# ----------------------------------------------------------- what lies hidden --
def booked(lengths, *, spare=6, b=16, d=64, layers=2, seed=0):
    """filled() over a pool with its books, `spare` pages free, and what free pages hold finite and large."""

    need = sum(-(-n // b) for n in lengths)
    bare, _, _ = filled(lengths, hkv=2, d=d, b=b, layers=layers, pages=need + spare, seed=seed)
    held = bare.table[bare.table >= 0].long()
    references = torch.zeros(bare.pages, dtype=torch.int32, device="cuda").scatter_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    bits = [sum((int(references[w * 32 + i]) == 0) << i for i in range(min(32, bare.pages - w * 32)))
            for w in range(-(-bare.pages // 32))]
    words = i32([x - (1 << 32) if x >> 31 else x for x in bits])
    key, value = torch.nan_to_num(bare.key, nan=500.0), torch.nan_to_num(bare.value, nan=500.0)
    return PagedKVCache(key, value, bare.table, bare.lengths, granted=i32([0] * len(lengths)), references=references,
                        free_pages=words, max_tokens=max(lengths))


@pytest.mark.parametrize("b", [16, 64])
def test_compact_drops_tokens_without_a_page(device, b):
    """Tokens whose table entries are no page have no rows: they do not come back as those of whoever had the page before."""

    n = 5 * b
    lengths = [n + 3, n, n + 7, 2 * b, n]
    cache = booked(lengths, b=b, spare=40)
    hidden = [{1}, {0, 4}, {5}, {0, 1}, set()]  # a page between, at both ends, the open one, all, none
    odd = [-1, cache.pages, -2 ** 31]
    for s, entries in enumerate(hidden):
        for i in entries:
            page = int(cache.table[s, i])
            cache.references[page] -= 1  # (it went to somebody else, and is free again)
            word = int(cache.free_pages[page // 32]) | (1 << page % 32) - (1 << 32 if page % 32 == 31 else 0)
            cache.free_pages[page // 32] = word
            cache.table[s, i] = odd[(s + i) % 3]
    key, value = cache.dense(layer=1)
    g = torch.Generator().manual_seed(b)
    keep = torch.rand(5, n, generator=g) < 0.7
    keep[2] = True  # (loses nothing but the page that is not there)
    keep[4] = True
    want = [[t for t in range(length) if t // b not in hidden[s] and (t >= n or bool(keep[s, t]))]
            for s, length in enumerate(lengths)]
    q = randn(5, 1, 4, 64, seed=1)
    before = cache.attention(q, layer=1)
    cache.compact(keep.cuda())
    assert cache.lengths.tolist() == [len(w) for w in want]
    after_k, after_v = cache.dense(layer=1)
    for s, w in enumerate(want):
        assert torch.equal(after_k[s, :len(w)], key[s, w]) and torch.equal(after_v[s, :len(w)], value[s, w])
        assert not after_k[s, len(w):].any()
        pages = -(-len(w) // b)
        row = cache.table[s].tolist()
        assert all(0 <= p < cache.pages for p in row[:pages]) and row[pages:] == [-1] * (cache.sequence_pages - pages)
    held = [p for row in cache.table.tolist() for p in row if p >= 0]
    assert cache.references.tolist() == [held.count(p) for p in range(cache.pages)]
    bits = [(w >> i) & 1 for w in cache.free_pages.tolist() for i in range(32)][:cache.pages]
    assert bits == [int(p not in held) for p in range(cache.pages)]
    # a mask that keeps all drops what was hidden, and what attention sees stays
    again = booked(lengths, b=b, spare=40)
    for s, entries in enumerate(hidden):
        for i in entries:
            again.table[s, i] = -1
    again.compact(torch.ones(5, 1, dtype=torch.bool, device=device))
    assert again.lengths.tolist() == [sum(t // b not in hidden[s] for t in range(x)) for s, x in enumerate(lengths)]
    out, lse = again.attention(q, layer=1)
    # (sums of the same weights over tiles cut otherwise: two roundings of the output, 64 steps of a sum of 5 b terms)
    assert ((out.float() - before[0].float()).abs() <= 2 * EPS[q.dtype] * before[0].float().abs() + 2.0 ** -10).all()
    seen = lse != -math.inf
    assert torch.equal(seen, before[1] != -math.inf)
    assert ((lse - before[1])[seen].abs() <= 2.0 ** -16 * (1 + lse[seen].abs())).all()


@pytest.mark.parametrize("dtype,d,b", [(torch.bfloat16, 64, 16), (torch.float16, 128, 64)])
@pytest.mark.parametrize("hq,lq", [(128, 3), (200, 4), (400, 2)])
def test_a_tile_of_one_token_hides_what_follows_it(device, dtype, d, b, hq, lq):
    # all rows of a workgroup's unit are of one query token: they all see less than the sequence holds
    lengths = [100, 70]
    cache, _, _ = filled(lengths, hkv=1, d=d, b=b, dtype=dtype)
    key, value = cache.key.clone(), cache.value.clone()
    table = cache.table.cpu()
    for s, n in enumerate(lengths):
        page, t = table[s, (n - 1) // b], (n - 1) % b
        key[0, page, :, t, 3], value[0, page, :, t] = math.nan, math.inf
        value[0, page, :, t, 5] = math.nan
    dirty = PagedKVCache(key, value, cache.table, cache.lengths, max_tokens=100)
    q = randn(2, lq, hq, d, seed=6, dtype=dtype)
    out, lse = dirty.attention(q, causal=True)
    clean, clean_lse = cache.attention(q, causal=True)
    assert torch.equal(out[:, :lq - 1], clean[:, :lq - 1]) and torch.equal(lse[:, :, :lq - 1], clean_lse[:, :, :lq - 1])
    assert out[:, lq - 1].isnan().all() and lse[:, :, lq - 1].isnan().all()


def test_storage_that_was_swapped_is_read_where_it_is(device):
    import copy

    cache, _, _ = filled([100, 37], d=64, b=16)
    q = randn(2, 1, 4, 64, seed=1)
    want = cache.attention(q)
    kept = cache.key.clone(), cache.value.clone(), cache.table.clone(), cache.lengths.clone()
    old = [t.detach() for t in (cache.key, cache.value, cache.table, cache.lengths)]
    cache.key.data, cache.value.data = kept[0], kept[1]
    cache.table.set_(kept[2])
    cache.lengths.data = kept[3]
    for t in old:
        t.zero_()
    got = cache.attention(q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    other = copy.deepcopy(cache)
    cache.key.zero_(), cache.lengths.zero_()
    got = other.attention(q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_copied_rotary_reads_its_own_tables(device):
    import copy

    q = randn(2, 1, 4, 64, seed=1)
    rotary = MultiAxisRotary(64, (16, 16))
    positions = torch.arange(4, device=device).view(2, 2, 1)
    want = rotary.rotate(q, positions=positions)
    other = copy.deepcopy(rotary)
    rotary._turns.zero_()
    assert torch.equal(other.rotate(q, positions=positions), want)


# ------------------------------------------------------------ ends of the range --
@pytest.mark.parametrize("hq,lq", [(3, 1), (3, 9), (2, 17), (2, 40), (130, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_logits_that_all_overflow_downwards_give_nan(device, hq, lq, d):
    """A row that sees keys, all of whose logits are below fp32's range, is no row without keys; a logit within the range beside
    them takes all the weight, as exp(-inf) = 0 says."""

    far, b = 700, 16
    lengths = [lq, far, far, far, 2 * b]
    key = torch.full((5, far, 1, d), -1.0, dtype=torch.float16)
    key[2, 650] = 0.0    # the only logit in range, in the last steps
    key[3, :300] = 0.0   # and many, in the first
    value = randn(5, far, 1, d, seed=3, dtype=torch.float16).cpu()
    cache, _, _ = filled(lengths, hkv=1, d=d, b=b, dtype=torch.float16)
    table = cache.table.cpu()
    for s, n in enumerate(lengths):
        for i in range(-(-n // b)):
            r = min(b, n - i * b)
            cache.key[0, table[s, i], :, :r] = key[s, i * b:i * b + r].transpose(0, 1).cuda()
            cache.value[0, table[s, i], :, :r] = value[s, i * b:i * b + r].transpose(0, 1).cuda()
    cache.table[4] = -1  # no page: these rows see no key, and get 0 and -inf
    q = torch.ones(5, lq, hq, d, dtype=torch.float16, device=device)
    for hint in (1, far):
        cache.max_tokens = hint
        for causal in (False, True):
            out, lse = cache.attention(q, causal=causal, sm_scale=2.0 ** 127 if causal else 1.1e38)
            assert out[:2].isnan().all() and lse[:2].isnan().all()
            assert not out[4].any() and (lse[4] == -math.inf).all()
            want = value[2, 650, 0].double()
            assert ((out[2].double().cpu() - want).abs() <= 2 * EPS[q.dtype] * want.abs()).all()
            assert (lse[2].abs() <= 2.0 ** -20).all()
            # equal weights of 300 values: their roundings to 16 bits and the sum's
            want, size = value[3, :300, 0].double().mean(0), value[3, :300, 0].double().abs().mean(0)
            assert ((out[3].double().cpu() - want).abs() <= EPS[q.dtype] * (want.abs() + size) + 2.0 ** -14 * size).all()
            assert ((lse[3] - math.log(300)).abs() <= 2.0 ** -18).all()
    # the one in range may lie as low as fp32 goes
    cache.key.mul_(4)
    cache.key[0, table[2, 650 // b], :, 650 % b] = -1.125
    out, lse = cache.attention(q, sm_scale=2.9e38 / (1.125 * d * math.log2(math.e)))
    want = value[2, 650, 0].double()
    assert ((out[2].double().cpu() - want).abs() <= 2 * EPS[q.dtype] * want.abs()).all()
    assert ((lse[2] / (-2.9e38 * math.log(2)) - 1).abs() <= 2.0 ** -18).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,lq", [(7, 6), (4, 16), (4, 70), (16, 40)])
def test_a_hidden_key_changes_no_bit_of_a_row(device, dtype, hq, lq):
    # the newest key is finite and far larger than all others: only the last row sees it
    lengths = [1000, 517]
    for seed in range(3):
        cache, _, _ = filled(lengths, hkv=1, d=64, b=32, dtype=dtype, seed=seed)
        key, table = cache.key.clone(), cache.table.cpu()
        q = randn(2, lq, hq, 64, seed=seed, dtype=dtype)
        for s, n in enumerate(lengths):
            key[0, table[s, (n - 1) // 32], :, (n - 1) % 32] = 30 * q[s, lq - 1, 0]
        other = PagedKVCache(key, cache.value, cache.table, cache.lengths, max_tokens=1000)
        out, lse = other.attention(q, causal=True)
        want, want_lse = cache.attention(q, causal=True)
        assert torch.equal(out[:, :lq - 1], want[:, :lq - 1]) and torch.equal(lse[:, :, :lq - 1], want_lse[:, :, :lq - 1])
        assert not torch.equal(lse[:, :, lq - 1], want_lse[:, :, lq - 1])


# ------------------------------------------------------------ rows that are held --
def test_dense_after_replays_of_a_captured_reserve(device):
    cache = PagedKVCache.empty(2, 12, 1, 64, page_tokens=16, sequence_pages=6)
    view, one = cache.layer(0), cache.layer(0, sequence=1)
    cache.reserve(5)
    rows = randn(2, 90, 1, 64, seed=1)
    cache.write(rows[:, :5], -rows[:, :5])
    for v, s in ((view, slice(0, 2)), (one, slice(1, 2))):  # views know of what was reserved after they were made
        key, value = v.dense()
        assert torch.equal(key, rows[s, :5]) and torch.equal(value, -rows[s, :5])
    new = torch.empty(2, 10, 1, 64, dtype=torch.bfloat16, device=device)

    def step():
        cache.reserve(10)
        cache.write(new, -new)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        new.copy_(rows[:, 5:15])
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        new.copy_(rows[:, 15 + 10 * i:25 + 10 * i])
        graph.replay()
        torch.cuda.synchronize()
        n = 25 + 10 * i
        assert cache.lengths.tolist() == [n, n]
        key, value = cache.dense()
        assert key.shape[1] >= n and torch.equal(key[:, :n], rows[:, :n]) and torch.equal(value[:, :n], -rows[:, :n])
        assert not key[:, n:].any() and not value[:, n:].any()
        key, _ = one.dense()
        assert torch.equal(key[:, :n], rows[1:, :n]) and not key[:, n:].any()
        key, value = cache.dense(tokens=n - 3)
        assert torch.equal(key, rows[:, :n - 3]) and torch.equal(value, -rows[:, :n - 3])
    key, _ = cache.dense(tokens=0)
    assert key.shape == (2, 0, 1, 64)
    for tokens in (-1, cache.capacity + 1):
        with pytest.raises(ValueError, match="tokens"):
            cache.dense(tokens=tokens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,lq,causal", [(1, 1, False), (7, 1, True), (8, 5, True), (4, 60, False), (4, 60, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(device, dtype, hq, lq, causal, d):
    """Weights are positive: a visible infinity makes its channel that infinity, two of both signs or a NaN make it NaN, however
    small the weight, in whole tiles and in parts that are joined; the other channels are as without it."""

    b, lengths = 16, [40, 700, 9000]
    for hint in (1, 9000):
        cache, _, _ = filled(lengths, hkv=1, d=d, b=b, dtype=dtype)
        cache.max_tokens = hint
        table, rows = cache.table.cpu(), {}
        q = randn(3, lq, hq, d, seed=1, dtype=dtype)
        q[..., 0] = 4.0
        far = math.sqrt(d) * 40.0  # a logit 160 below the others': fp32 holds no e^-160
        for s, n in enumerate(lengths):
            for t, channel, x, small in ((2, 7, math.inf, False), (n // 2, 8, -math.inf, False), (3, 9, math.inf, False),
                                         (n // 3, 9, -math.inf, False), (1, 10, math.nan, False), (0, 11, math.inf, True),
                                         (n // 4, 12, -math.inf, True)):
                at = 0, table[s, t // b], 0, t % b
                if small:
                    cache.key[at][0] = -far
                rows[s, t, channel] = at, x
        clean = cache.attention(q, causal=causal)
        for (s, t, channel), (at, x) in rows.items():
            cache.value[at][channel] = x
        zeros = PagedKVCache(cache.key, torch.nan_to_num(cache.value, nan=0.0, posinf=0.0, neginf=0.0), cache.table, cache.lengths,
                             max_tokens=hint)
        out, lse = cache.attention(q, causal=causal)
        want, want_lse = zeros.attention(q, causal=causal)
        assert torch.equal(lse, want_lse) and torch.equal(lse, clean[1])
        for s, n in enumerate(lengths):
            if causal and lq > n:
                continue  # (rows that see few keys or none)
            got = out[s].float()
            assert (got[..., 7] == math.inf).all() and (got[..., 8] == -math.inf).all()
            assert got[..., 9].isnan().all() and got[..., 10].isnan().all()
            assert (got[..., 11] == math.inf).all() and (got[..., 12] == -math.inf).all()
            others = [c for c in range(d) if not 7 <= c <= 12]
            assert torch.equal(out[s][..., others], want[s][..., others])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,lq", [(1, 1), (3, 9), (4, 40)])
@pytest.mark.parametrize("d", [64, 128])
def test_logits_whose_steps_pass_one_take_the_largest(device, dtype, hq, lq, d):
    """Logits so large that fp32 holds them in steps above 1: those that are the largest share the weight, whichever way they, the
    scale and the reference were rounded."""

    lengths, b = [40, 700], 16
    cache, k, v = filled(lengths, hkv=1, d=d, b=b, dtype=dtype)
    table = cache.table.cpu()
    q = torch.full((2, lq, hq, d), 64.0, dtype=dtype, device=device)
    for sign in (1.0, -1.0):
        for s, n in enumerate(lengths):
            # a key's channels are all alike, so that products and sums are exact: d * 64 * size
            sizes = sign * (torch.arange(n) * 7 % 31 + 32.0)
            for i in range(-(-n // b)):
                r = min(b, n - i * b)
                cache.key[0, table[s, i], :, :r] = sizes[i * b:i * b + r].to(dtype)[:, None].cuda()
        for scale in (300.0, 4000.0, 4321.0, 33333.0, 5e5, 7.7e5, 3.3e9, 1.7e17, 2.9e30):
            for hint in (1, 700):
                cache.max_tokens = hint
                out, lse = cache.attention(q, sm_scale=scale)
                for s, n in enumerate(lengths):
                    sizes = sign * (torch.arange(n) * 7 % 31 + 32.0)
                    at = sizes == sizes.max()
                    top = v[s, :n, 0][at].double()
                    want, size = top.mean(0), top.abs().mean(0)
                    # equal weights, each rounded the same way, the sum's terms and the output's rounding
                    tol = EPS[dtype] * (want.abs() + size) + 2.0 ** -14 * size
                    assert ((out[s].double().cpu() - want).abs() <= tol).all(), (sign, scale)
                    x = d * 64.0 * float(sizes.max()) * float(torch.tensor(scale, dtype=torch.float32))
                    assert ((lse[s].double() - x - math.log(int(at.sum()))).abs() <= 2.0 ** -21 * abs(x)).all()


@pytest.mark.parametrize("hq,lq", [(3, 5), (4, 40)])
@pytest.mark.parametrize("d", [64, 128])
def test_log_sum_exp_is_rounded_once(device, hq, lq, d):
    """One key a row, whose product with the query fp32 holds exactly: what is left are the logarithm's last rounding and, of the
    weight, a few units of numbers below 16."""

    cache, _, _ = filled([1] * 8, hkv=1, d=d, b=16)
    g = torch.Generator().manual_seed(d)
    k = torch.randint(-8, 9, (8, d), generator=g)
    q = torch.randint(-8, 9, (8, lq, hq, d), generator=g) * 64
    for s in range(8):
        cache.key[0, int(cache.table[s, 0]), 0, 0] = k[s].to(torch.bfloat16).cuda()
    product = torch.einsum("slhd,sd->shl", q.double(), k.double())
    for scale in (0.07, 0.1, 1 / math.sqrt(128), 0.77):
        _, lse = cache.attention(q.to(torch.bfloat16).cuda(), sm_scale=scale)
        want = product * float(torch.tensor(scale, dtype=torch.float32))
        assert ((lse.double().cpu() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -19).all()


@pytest.mark.parametrize("hq,lq", [(7, 6), (4, 70)])
def test_a_far_hidden_key_changes_no_bit_of_a_row(device, hq, lq):
    # the newest key's logits pass 2^24: its row's unit is gone over again, and the other rows come out as they were
    lengths = [1000, 517]
    cache, _, _ = filled(lengths, hkv=1, d=64, b=32)
    key, table = cache.key.clone(), cache.table.cpu()
    q = randn(2, lq, hq, 64, seed=1)
    for s, n in enumerate(lengths):
        key[0, table[s, (n - 1) // 32], :, (n - 1) % 32] = 1e12 * q[s, lq - 1, 0]
    other = PagedKVCache(key, cache.value, cache.table, cache.lengths, max_tokens=1000)
    out, lse = other.attention(q, causal=True)
    want, want_lse = cache.attention(q, causal=True)
    assert torch.equal(out[:, :lq - 1], want[:, :lq - 1]) and torch.equal(lse[:, :, :lq - 1], want_lse[:, :, :lq - 1])
    # the last row's first head has all its weight there, and all of its logits' size
    for s, n in enumerate(lengths):
        value = cache.value[0, table[s, (n - 1) // 32], 0, (n - 1) % 32]
        assert torch.equal(out[s, lq - 1, 0], value)
        x = float((key[0, table[s, (n - 1) // 32], 0, (n - 1) % 32].double() * q[s, lq - 1, 0].double()).sum()) / 8
        assert abs(float(lse[s, 0, lq - 1]) - x) <= 70 * 2.0 ** -24 * x
