"""The paged KV cache, what writes it, what reads it and what moves its pages:
what their calls are timed on, with the same calls in plain torch.

A cache of L layers holds the 16-bit keys and values of up to S sequences in
pages of B tokens from a common pool of P pages:

    key, value  [L, P, Hkv, B, D]      table       [S, M] int32, -1 for none
    lengths     [S] int32              references  [P] int32, holders of each page
    granted     [S] int32              free_pages  [ceil(P / 32)] int32, a bit for each free page

Token t of sequence s is row t % B of page table[s, t / B] in every layer.
Whole pages may be held by several sequences; the last, partly filled page of
a sequence (its open page) by no other.

Kinds of cases:

- ``attend``  attention of [S, Lq, Hq, D] queries over one layer
              (PagedKVCache.attention): one new token per sequence, a few
              (verification of drafted tokens), or a prompt's chunk.
- ``write``   new rows into the pages of one layer, queries and keys rotated
              by positions of several axes on the way (PagedKVCache.write).
- ``rotate``  the rotation alone (MultiAxisRotary.rotate).
- ``pages``   children forked from running sequences (PagedKVCache.reorder)
              and, with `keep` below 1, the children's tokens thinned out
              (PagedKVCache.compact).
- ``step``    a step of speculative decoding over all layers: room for the
              drafted tokens (reserve), each layer's write and attention, and
              the drafted tokens taken back (truncate).

Head counts and lengths come from this repository's configurations (28/4 heads
of 128 channels, 28 layers, 2k to 32k tokens) and from common layouts of 16 and
32 heads.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------- cases --
def _cache(kind, *, tokens, seqs=1, hq=28, hkv=4, d=128, page=64, dtype="bf16", ragged=0.0, layers=1):
    return dict(kind=kind, tokens=tokens, seqs=seqs, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, ragged=ragged,
                layers=layers)


def _attend_case(*, lq=1, short=0, causal=False, shared=0.0, **cache):
    return dict(_cache("attend", **cache), lq=lq, short=short, causal=causal, shared=shared)


def _write_case(*, new, short=0, sections=(16, 24, 24), pairing="halves", far=0, kind="write", **cache):
    axes = ",".join(map(str, sections))
    return dict(_cache(kind, **cache), new=new, short=short, sections=axes, pairing=pairing, far=far)


def _pages_case(*, children=1, keep=1.0, **cache):
    return dict(_cache("pages", **cache), children=children, keep=keep)


def _step_case(*, new, **cache):
    return dict(_cache("step", **cache), new=new)


def listed():
    return [
        # one layer of a short chat turn: the smallest read, bound by latency
        dict(_attend_case(tokens=2048), name="attend_2k"),
        # one layer of a batched decode loop over long contexts
        dict(_attend_case(tokens=32768, seqs=8), name="attend_8x32k"),
        # a large batch of sequences of every length down to one token, small pages
        dict(_attend_case(tokens=8191, seqs=64, hq=32, hkv=8, page=16, dtype="fp16", ragged=1.0),
             name="attend_64x8k_ragged"),
        # drafted tokens verified in one pass, heads of 64 channels
        dict(_attend_case(tokens=4099, seqs=16, hq=16, hkv=2, d=64, page=32, ragged=0.5, lq=5, causal=True),
             name="attend_16x5tok"),
        # the next chunk of two prompts behind a prefix that both share: the most products
        dict(_attend_case(tokens=13001, seqs=2, hq=32, hkv=8, page=128, lq=1999, short=700, causal=True, shared=0.8),
             name="attend_chunk_2x2k_of_13k"),
        # the new token of each sequence of a batch, text positions behind images
        dict(_write_case(tokens=4000, seqs=32, new=1, ragged=0.9), name="write_32x1"),
        # the prompt of a video: frames, rows and columns as positions
        dict(_write_case(tokens=0, new=16384, sections=(16, 24, 24)), name="write_video_16k"),
        # the patches of a batch of images in an encoder: rows and columns, neighbours as pairs
        dict(_write_case(kind="rotate", tokens=0, seqs=4, new=1089, hq=16, hkv=16, d=64, dtype="fp16",
                         sections=(16, 16), pairing="adjacent"), name="rotate_4x1089"),
        # far positions of a long video, half of the channels rotated
        dict(_write_case(kind="rotate", tokens=0, new=7001, hq=32, hkv=8, sections=(8, 12, 12), far=1000000),
             name="rotate_far_7k"),
        # three samples each of the answers to eight prompts: whole pages shared, open pages copied
        dict(_pages_case(tokens=1000, seqs=8, children=3, layers=28, ragged=0.4), name="fork_8x3"),
        # children of long contexts keep every second token
        dict(_pages_case(tokens=8192, seqs=4, layers=4, keep=0.5, ragged=0.2), name="compact_4x8k"),
        # drafted tokens of a small batch through the layers, and back
        dict(_step_case(tokens=2050, seqs=6, new=4, layers=6, ragged=0.3, page=32), name="step_6x4tok"),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of its range; every third one a multiple of 64."""

    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, n // 64 * 64) if rng.random() < 0.34 and n >= 64 else n


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "chunk", "write", "write", "rotate", "fork", "compact", "step"])
    hq, hkv = rng.choice([(28, 4), (28, 4), (32, 8), (16, 2), (16, 4), (8, 8), (16, 1)])
    d = rng.choice([128, 128, 64])
    common = dict(hq=hq, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 64, 128, 256]),
                  dtype=rng.choice(["bf16", "bf16", "fp16"]))
    ragged = rng.choice([0.0, 0.3, 1.0])
    if kind == "decode":
        seqs = rng.choice([1, 1, 2, 7, 8, 24, 32])
        return _attend_case(tokens=_log(rng, 100, min(65536, 131072 // seqs)), seqs=seqs, ragged=ragged,
                            lq=rng.choice([1, 1, 1, 2, 4, 6]), causal=rng.random() < 0.5,
                            shared=rng.choice([0.0, 0.0, 0.5]), **common)
    if kind == "chunk":
        seqs = rng.choice([1, 1, 2, 3])
        lq = _log(rng, 20, 2048 // seqs)
        return _attend_case(tokens=max(lq, _log(rng, 200, 12000 // seqs)), seqs=seqs, ragged=min(ragged, 0.3), lq=lq,
                            short=rng.choice([0, lq // 3]), causal=rng.random() < 0.7, **common)
    if kind in ("write", "rotate"):
        seqs = rng.choice([1, 1, 2, 5, 16])
        new = rng.choice([1, 2, 5]) if rng.random() < 0.4 else _log(rng, 20, 16384 // seqs)
        half = d // 2
        sections = rng.choice([(half,), (half // 2, half // 2), (half // 4, 3 * half // 8, 3 * half // 8),
                               (half // 8, half // 8, half // 4), (half // 2,)])
        return _write_case(kind=kind, tokens=0 if kind == "rotate" else _log(rng, 1, 5000), seqs=seqs, new=new,
                           short=rng.choice([0, new // 3]), ragged=min(ragged, 0.9), sections=sections,
                           pairing=rng.choice(["halves", "halves", "adjacent"]), far=rng.choice([0, 0, 4096, 1000000]),
                           **common)
    if kind == "step":
        seqs = rng.choice([1, 2, 5, 8])
        return _step_case(tokens=_log(rng, 50, 8192 // seqs), seqs=seqs, new=rng.choice([1, 1, 3, 5]),
                          layers=rng.choice([1, 2, 4]), ragged=min(ragged, 0.5), **common)
    seqs = rng.choice([1, 2, 4, 7])
    tokens = _log(rng, 30, 8192 // seqs)
    return _pages_case(tokens=tokens, seqs=seqs, layers=rng.choice([1, 2, 4]), ragged=min(ragged, 0.5),
                       children=rng.choice([1, 2]), keep=1.0 if kind == "fork" else rng.choice([0.1, 0.5, 0.9]), **common)


def _lengths(case):
    """Tokens of each sequence: `tokens` down to (1 - ragged) of it, one at least."""

    s, t = case["seqs"], case["tokens"]
    return [max(min(t, 1), t - int(case["ragged"] * t * i / max(1, s - 1))) for i in range(s)]


def _counts(case, rows):
    """New rows of each sequence: `rows`, and `short` fewer for every second one."""

    return [rows - (case.get("short", 0) if i % 2 else 0) for i in range(case["seqs"])]


# ------------------------------------------------------------------ inputs --
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, case, gen):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=_DTYPES[case["dtype"]])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bits(mask):
    """Bit p % 32 of word p / 32 for each p of the mask, as int32."""

    mask = torch.nn.functional.pad(mask, (0, -mask.numel() % 32)).view(-1, 32).to(torch.int64)
    words = (mask << torch.arange(32, device=mask.device)).sum(dim=1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _pool(case, lengths, slots, spare, gen, shared=0, room=0):
    """A cache whose sequences lie scattered over the pool, as after a while of use; `shared`: leading pages that every
    sequence holds.  Sequences past len(lengths) are empty, `spare` pages are free, and the longest sequence has room for
    `room` more pages."""

    b = case["page"]
    held = [-(-n // b) for n in lengths]
    used = sum(held) - shared * (len(held) - 1)
    pages, width = used + spare, max(max(held), 1) + room
    order = torch.randperm(pages, generator=gen, device="cuda")[:used].tolist()
    table = torch.full((slots, width), -1, dtype=torch.int32)
    references = torch.zeros(pages, dtype=torch.int32)
    at = shared
    for s, n in enumerate(held):
        own_pages = order[:shared] + order[at:at + n - shared]
        at += n - shared
        table[s, :n] = torch.tensor(own_pages, dtype=torch.int32)
        references[own_pages] += 1
    shape = (case["layers"], pages, case["hkv"], b, case["d"])
    key = _randn(shape, case, gen)
    # eight outlier channels per head
    gain = torch.full((case["hkv"], 1, case["d"]), 0.75, device="cuda", dtype=key.dtype)
    gain.scatter_(2, torch.rand(case["hkv"], 1, case["d"], generator=gen, device="cuda").topk(8, dim=2).indices, 4.5)
    key *= gain
    references = references.cuda()
    return {"key": key, "value": _randn(shape, case, gen), "table": table.cuda(),
            "lengths": _int32(list(lengths) + [0] * (slots - len(lengths))),
            "granted": torch.zeros(slots, dtype=torch.int32, device="cuda"),
            "references": references, "free_pages": _bits(references == 0)}


def _positions(case, gen):
    """Positions [axes, S, rows]: frames of 32 x 33 patches, counted from `far` on; one axis: the tokens in turn.  A
    single new row per sequence has the same place on every axis, as text has."""

    s, n, axes = case["seqs"], case["new"], len(case["sections"].split(","))
    start = torch.randint(0, 500, (s, 1), generator=gen, device="cuda") + case["far"]
    i = torch.arange(n, device="cuda")[None]
    if n == 1 or axes == 1:
        return (start + i).expand(axes, s, n).contiguous()
    grid = [i // (32 * 33), i // 33 % 32, i % 33][3 - axes:]
    return torch.stack([start + g for g in grid])


def _frequencies(case):
    pairs = sum(map(int, case["sections"].split(",")))
    return [10000.0 ** (-i / pairs) for i in range(pairs)]


def _axis_of_pair(case):
    return [a for a, n in enumerate(map(int, case["sections"].split(","))) for _ in range(n)]


def prepare(case, seed):
    gen = _generator(seed)
    kind, s = case["kind"], case["seqs"]
    state = {"case": case}
    if kind == "attend":
        lengths = [max(n, c) for n, c in zip(_lengths(case), _counts(case, case["lq"]))]
        shared = int(min(lengths) * case["shared"]) // case["page"] if s > 1 else 0
        state.update(_pool(case, lengths, s, 0, gen, shared))
        state["query"] = _randn((s, case["lq"], case["hq"], case["d"]), case, gen)
        state["query_lengths"] = _int32(_counts(case, case["lq"])) if case["short"] else None
    elif kind in ("write", "rotate"):
        n, counts = case["new"], _counts(case, case["new"])
        if kind == "write":
            state.update(_pool(case, [a + c for a, c in zip(_lengths(case), counts)], s, 0, gen))
            state["granted"] = _int32(counts)
            state["new_value"] = _randn((s, n, case["hkv"], case["d"]), case, gen)
        state["new_key"] = _randn((s, n, case["hkv"], case["d"]), case, gen)
        state["query"] = _randn((s, n, case["hq"], case["d"]), case, gen)
        state["positions"] = _positions(case, gen)
    elif kind == "pages":
        lengths = _lengths(case)
        slots = s * (1 + case["children"])
        b = case["page"]
        spare = slots + (case["children"] * sum(-(-n // b) for n in lengths) if case["keep"] < 1.0 else 0)
        state.update(_pool(case, lengths, slots, spare, gen))
        # slots behind the parents become their children, in turn
        state["parents"] = torch.arange(slots, dtype=torch.int32, device="cuda") % s
        if case["keep"] < 1.0:
            keep = torch.rand(slots, max(lengths), generator=gen, device="cuda") < case["keep"]
            keep[:s] = True
            state["keep"] = keep
    else:
        lengths = _lengths(case)
        more = 1 + -(-case["new"] // case["page"])
        state.update(_pool(case, lengths, s, s * more, gen, room=more))
        shape = (case["layers"], s, case["new"])
        state["before"] = state["lengths"].clone()
        state["new_key"] = _randn((*shape, case["hkv"], case["d"]), case, gen)
        state["new_value"] = _randn((*shape, case["hkv"], case["d"]), case, gen)
        state["query"] = _randn((*shape, case["hq"], case["d"]), case, gen)
    if kind in ("write", "rotate", "step"):
        state["frequencies"] = torch.tensor(_frequencies(_rotary_case(case)), dtype=torch.float64, device="cuda")
        state["axis"] = torch.tensor(_axis_of_pair(_rotary_case(case)), device="cuda")
    if own:
        from unicache_amd.operators import MultiAxisRotary
        from unicache_amd.storage import PagedKVCache

        if kind != "rotate":
            state["cache"] = PagedKVCache(*(state[n] for n in ("key", "value", "table", "lengths")),
                                          granted=state["granted"], references=state["references"],
                                          free_pages=state["free_pages"], max_tokens=max(_lengths_of(state)))
        if kind in ("write", "rotate", "step"):
            spec = _rotary_case(case)
            state["rotary"] = MultiAxisRotary(case["d"], [int(n) for n in spec["sections"].split(",")],
                                              pairing=spec["pairing"])
    return state


def _rotary_case(case):
    """A step rotates whole heads by the token's place on one axis."""

    return case if "sections" in case else {**case, "sections": str(case["d"] // 2), "pairing": "halves"}


def _lengths_of(state):
    return state["lengths"].tolist()


# ------------------------------------------------------------- plain forms --
def _rows_of(pool, table, tokens):
    """The first `tokens` rows of every sequence as fp32 [S, Hkv, tokens, D]; pool [P, Hkv, B, D]."""

    b = pool.shape[2]
    x = pool[table[:, :-(-tokens // b)].clamp_min(0).long()]  # [S, n, Hkv, B, D]
    x = x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])
    return x[:, :, :tokens].float()


def _softmax(logits, visible):
    """Weights and log-sum-exp over the visible keys; zeros and -inf where there are none."""

    logits = torch.where(visible, logits, -math.inf)
    top = logits.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = (logits - top).exp()
    total = e.sum(dim=-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1)
    return e / torch.where(total == 0, 1.0, total), lse


def _attention(key, value, table, lengths, q, query_lengths, causal, tokens):
    s, lq, hq, d = q.shape
    hkv = key.shape[1]
    i = torch.arange(lq, device=q.device)[None]
    count = torch.full_like(lengths, lq) if query_lengths is None else query_lengths
    end = lengths[:, None] - count[:, None] + i + 1 if causal else lengths[:, None].expand(-1, lq)
    end = torch.where(i < count[:, None], end, 0)
    visible = torch.arange(tokens, device=q.device) < end[:, :, None]  # [S, Lq, T]
    visible = visible.repeat_interleave(hq // hkv, dim=1)[:, None]
    # rows of a KV head: [S, Hkv, Lq * group, D]
    x = q.float().view(s, lq, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(s, hkv, -1, d)
    logits = torch.matmul(x, _rows_of(key, table, tokens).transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    weights, lse = _softmax(logits, visible)
    del logits
    out = torch.matmul(weights, _rows_of(value, table, tokens)).view(s, hkv, lq, -1, d)
    out = out.permute(0, 2, 1, 3, 4).reshape(s, lq, hq, d)
    return out.to(q.dtype), lse.view(s, hkv, lq, -1).permute(0, 1, 3, 2).reshape(s, hq, lq)


def _rotate(x, positions, axis, frequencies, pairing):
    """Rows [S, n, H, D] turned: pair i by the angle positions[axis[i]] * frequencies[i]."""

    angle = positions.double()[axis] * frequencies[:, None, None]  # [pairs, S, n]
    cos, sin = (f(angle).permute(1, 2, 0)[:, :, None].float() for f in (torch.cos, torch.sin))
    pairs, y = axis.numel(), x.float()
    if pairing == "halves":
        a, b = y[..., :pairs], y[..., pairs:2 * pairs]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = y[..., :2 * pairs:2], y[..., 1:2 * pairs:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, y[..., 2 * pairs:]], dim=-1).to(x.dtype)


def _put(pool, table, lengths, granted, rows):
    """New rows [S, n, Hkv, D] into a layer's pages, as the sequences' last granted[s] tokens."""

    b = pool.shape[2]
    # rows behind a sequence's last new one stand for that
    i = torch.minimum(torch.arange(rows.shape[1], device=rows.device)[None], granted[:, None].long() - 1)
    token = (lengths - granted)[:, None].long() + i
    page = torch.gather(table.long(), 1, token // b)
    pool[page, :, token % b] = torch.gather(rows, 1, i[:, :, None, None].expand(-1, -1, *rows.shape[2:]))


def _free_rank(references):
    """Pages in the order in which they are given out: the free ones, the lowest first."""

    return torch.sort((references > 0).to(torch.int32), stable=True).indices


def _reserve(state, rows):
    """Pages for `rows` more tokens of every sequence (of which there are enough)."""

    table, lengths, references = state["table"], state["lengths"], state["references"]
    b = state["key"].shape[3]
    held, wanted = (lengths + b - 1) // b, (lengths + rows + b - 1) // b
    first = torch.cumsum(wanted - held, 0) - (wanted - held)
    entry = torch.arange(table.shape[1], device=table.device)[None]
    new = (entry >= held[:, None]) & (entry < wanted[:, None])
    rank = (first[:, None] + entry - held[:, None]).clamp(0, references.numel() - 1).long()
    table.copy_(torch.where(new, _free_rank(references)[rank].to(torch.int32), table))
    lengths += rows
    state["granted"].fill_(rows)
    _count_holders(state)


def _count_holders(state):
    table, references = state["table"], state["references"]
    references.zero_()
    references.scatter_add_(0, table.clamp_min(0).long().view(-1), (table >= 0).to(torch.int32).view(-1))
    state["free_pages"].copy_(_bits(references == 0))


def _truncate(state, most):
    """Cut the sequences to most[s] tokens (whose open pages are their own)."""

    table, lengths, b = state["table"], state["lengths"], state["key"].shape[3]
    lengths.copy_(torch.minimum(lengths, most))
    entry = torch.arange(table.shape[1], device=table.device)[None]
    table.copy_(torch.where(entry < (lengths[:, None] + b - 1) // b, table, -1))
    _count_holders(state)


def _fork(state):
    """Slot s becomes slot parents[s]; of the holders of an open page the first keeps it, the others get copies."""

    table, lengths, parents, b = state["table"], state["lengths"], state["parents"].long(), state["key"].shape[3]
    table.copy_(table[parents])
    lengths.copy_(lengths[parents])
    _count_holders(state)
    slot = torch.arange(len(parents), device=table.device)
    first = torch.full_like(slot, len(parents)).scatter_reduce(0, parents, slot, "amin")[parents]
    copied = (slot != first) & (lengths % b > 0)
    entry = ((lengths + b - 1) // b - 1).clamp_min(0).long()
    source = table[slot, entry].long()
    rank = (torch.cumsum(copied.long(), 0) - 1).clamp_min(0)
    target = torch.where(copied, _free_rank(state["references"])[rank], source)
    # slots that copy nothing repeat the first copy, if there is one
    one = copied.to(torch.int32).argmax()
    source, to = torch.where(copied, source, source[one]), torch.where(copied, target, target[one])
    rows = torch.arange(b, device=table.device)[None] < torch.where(copied, lengths % b, lengths[one] % b)[:, None]
    for pool in (state["key"], state["value"]):
        pool[:, to] = torch.where(rows[None, :, None, :, None], pool[:, source], pool[:, to])
    table[slot, entry] = target.to(torch.int32)
    _count_holders(state)


def _compact(state):
    """Sequences keep the tokens that the mask keeps: from the first page that loses one on, in new pages."""

    table, lengths, b = state["table"], state["lengths"], state["key"].shape[3]
    slots, t = state["keep"].shape
    token = torch.arange(t, device=table.device)[None]
    there = token < lengths[:, None]
    keep = state["keep"] & there
    dropped = there & ~keep
    changed = dropped.any(dim=1)
    whole = torch.where(changed, dropped.to(torch.int32).argmax(dim=1), lengths) // b  # pages that stay
    kept = keep.sum(dim=1)
    need = torch.where(changed, (kept + b - 1) // b - whole, 0).clamp_min(0)
    start = torch.cumsum(need, 0) - need
    entry = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (entry >= whole[:, None]) & (entry < (whole + need)[:, None]) & changed[:, None]
    rank = (start[:, None] + entry - whole[:, None]).clamp(0, state["references"].numel() - 1)
    stays = (entry < whole[:, None]) | ~changed[:, None]
    new = torch.where(fresh, _free_rank(state["references"])[rank].to(torch.int32), torch.where(stays, table, -1))
    # row j of a sequence's kept tokens comes from token source[j]
    source = torch.sort((~keep).to(torch.int32), dim=1, stable=True).indices
    moved = changed[:, None] & (token >= (whole * b)[:, None]) & (token < kept[:, None])
    fill = moved.view(-1).to(torch.int32).argmax()  # what moves nothing repeats the first that does
    page_from = torch.gather(table.long(), 1, source // b)
    page_to = torch.gather(new.long(), 1, token.expand(slots, -1) // b)
    where = [torch.where(moved.view(-1), x.reshape(-1), x.reshape(-1)[fill])
             for x in (page_from, source % b, page_to, (token % b).expand(slots, -1))]
    for pool in (state["key"], state["value"]):
        for layer in pool:
            layer[where[2], :, where[3]] = layer[where[0], :, where[1]]
    table.copy_(new)
    lengths.copy_(kept.to(torch.int32))
    _count_holders(state)


def _whole_state(state):
    return {n: state[n] for n in ("key", "value", "table", "lengths", "references", "free_pages")}


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "attend":
        out, lse = _attention(state["key"][0], state["value"][0], state["table"], state["lengths"], state["query"],
                              state["query_lengths"], case["causal"], case["tokens"])
        return {"out": out, "lse": lse}
    if kind in ("write", "rotate"):
        turn = (state["positions"], state["axis"], state["frequencies"], case["pairing"])
        query, key = _rotate(state["query"], *turn), _rotate(state["new_key"], *turn)
        if kind == "rotate":
            return {"query": query, "key": key}
        place = (state["table"], state["lengths"], state["granted"])
        _put(state["key"][0], *place, key)
        _put(state["value"][0], *place, state["new_value"])
        return {"query": query, "key": state["key"], "value": state["value"]}
    if kind == "pages":
        _fork(state)
        if "keep" in state:
            _compact(state)
        return _whole_state(state)
    rows, outs, lses = case["new"], [], []
    _reserve(state, rows)
    place = (state["table"], state["lengths"], state["granted"])
    positions = ((state["lengths"] - rows)[:, None] + torch.arange(rows, device="cuda"))[None]
    turn = (positions, state["axis"], state["frequencies"], "halves")
    for layer in range(case["layers"]):
        _put(state["key"][layer], *place, _rotate(state["new_key"][layer], *turn))
        _put(state["value"][layer], *place, state["new_value"][layer])
        out, lse = _attention(state["key"][layer], state["value"][layer], state["table"], state["lengths"],
                              _rotate(state["query"][layer], *turn), None, True, case["tokens"] + rows)
        outs.append(out)
        lses.append(lse)
    _truncate(state, state["before"])
    return {"out": outs, "lse": lses, **_whole_state(state)}


# ------------------------------------------------------------- the kernels --
def _kernels(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "rotate":
        query, key = state["rotary"].rotate(state["query"], state["new_key"], positions=state["positions"])
        return {"query": query, "key": key}
    cache = state["cache"]
    if kind == "attend":
        out, lse = cache.attention(state["query"], query_lengths=state["query_lengths"], causal=case["causal"])
        return {"out": out, "lse": lse}
    if kind == "write":
        query = cache.write(state["new_key"], state["new_value"], query=state["query"], rotary=state["rotary"],
                            positions=state["positions"])
        return {"query": query, "key": cache.key, "value": cache.value}
    if kind == "pages":
        cache.reorder(state["parents"])
        if "keep" in state:
            cache.compact(state["keep"])
        return _whole_state(state)
    outs, lses = [], []
    cache.reserve(case["new"])
    for layer in range(case["layers"]):
        query = cache.write(state["new_key"][layer], state["new_value"][layer], layer=layer,
                            query=state["query"][layer], rotary=state["rotary"])
        out, lse = cache.attention(query, layer=layer, causal=True)
        outs.append(out)
        lses.append(lse)
    cache.truncate(state["before"])
    return {"out": outs, "lse": lses, **_whole_state(state)}


def run(state):
    return _kernels(state) if own else _plain(state)


# -------------------------------------------------------------------- work --
def work(case):
    kind, s, d, hq, hkv, b = (case[n] for n in ("kind", "seqs", "d", "hq", "hkv", "page"))
    row = 2 * hkv * d * 2  # a token's key and value
    if kind == "attend":
        counts = _counts(case, case["lq"])
        lengths = [max(n, c) for n, c in zip(_lengths(case), counts)]
        shared = int(min(lengths) * case["shared"]) // b * b if s > 1 else 0
        seen = sum(c * n - (c * (c - 1) // 2 if case["causal"] else 0) for n, c in zip(lengths, counts))
        held = sum(-(-n // b) for n in lengths)
        io = s * case["lq"] * hq * (2 * d * 2 + 4)
        return {"bytes": (sum(lengths) - shared * (s - 1)) * row + io + 4 * (held + s), "flops": 4 * seen * hq * d}
    if kind in ("write", "rotate"):
        rows, counts = s * case["new"], sum(_counts(case, case["new"]))
        axes = len(case["sections"].split(","))
        pairs = sum(map(int, case["sections"].split(",")))
        moved = rows * hq * d * 2 * 2 + rows * axes * 8
        moved += counts * row * 2 if kind == "write" else rows * hkv * d * 2 * 2
        return {"bytes": moved, "flops": 6 * pairs * rows * (hq + hkv)}
    lengths = _lengths(case)
    if kind == "pages":
        n = case["children"]
        entries = sum(-(-t // b) for t in lengths) * (1 + n)
        copied = sum(t % b for t in lengths) * n
        if case["keep"] < 1.0:
            copied += int(case["keep"] * sum(lengths) * n)
        mask = s * (1 + n) * max(lengths) if case["keep"] < 1.0 else 0
        return {"bytes": copied * case["layers"] * row * 2 + 8 * entries + mask, "flops": 0}
    new, layers = case["new"], case["layers"]
    seen = sum(new * (t + new) - new * (new - 1) // 2 for t in lengths)
    each = (sum(lengths) + 2 * s * new) * row + s * new * hq * (2 * d * 2 + 4)
    return {"bytes": layers * each, "flops": layers * 4 * seen * hq * d}


# ------------------------------------------------------------------- exact --
def _exact_attention(rows_k, rows_v, q, ends):
    """One sequence in 64 bits: rows [T, Hkv, D], queries [Lq, Hq, D], keys that each query sees."""

    lq, hq, d = q.shape
    group = hq // rows_k.shape[1]
    out = torch.zeros(lq, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((hq, lq), -math.inf, dtype=torch.float64, device=q.device)
    hidden = torch.arange(rows_k.shape[0], device=q.device)[None] >= torch.tensor(ends, device=q.device)[:, None]
    for h in range(hq):
        k, v = rows_k[:, h // group].double(), rows_v[:, h // group].double()
        x = (q[:, h].double() @ k.t()) / d ** 0.5
        x = x.masked_fill(hidden, -math.inf)
        lse[h] = torch.logsumexp(x, dim=1)
        some = torch.tensor(ends, device=q.device) > 0
        out[some, h] = torch.exp(x[some] - lse[h][some][:, None]) @ v
    return out, lse


def _sequence(pool, pages, tokens):
    """[tokens, Hkv, D] of a sequence's pages (a list) of [P, Hkv, B, D]."""

    return torch.cat([pool[p].transpose(0, 1) for p in pages])[:tokens]


def _exact_turn(x, positions, case):
    """Rows [S, n, H, D] in 64 bits, turned as complex numbers."""

    spec = _rotary_case(case)
    frequency = torch.tensor(_frequencies(spec), dtype=torch.float64, device=x.device)
    place = positions.to(torch.float64)
    angle = torch.stack([place[a] * f for a, f in zip(_axis_of_pair(spec), frequency)], dim=-1)[:, :, None]
    turn = torch.complex(angle.cos(), angle.sin())
    y, pairs = x.double(), len(frequency)
    at = list(range(pairs)), list(range(pairs, 2 * pairs))
    if spec["pairing"] == "adjacent":
        at = list(range(0, 2 * pairs, 2)), list(range(1, 2 * pairs, 2))
    z = torch.complex(y[..., at[0]], y[..., at[1]]) * turn
    out = y.clone()
    out[..., at[0]], out[..., at[1]] = z.real, z.imag
    return out


def _exact_pages(state, case):
    """The pool after the fork (and the thinning out), slot by slot; the whole numbers have no such value."""

    s, b = case["seqs"], case["page"]
    key, value = state["key"].clone(), state["value"].clone()
    pages, lengths = state["table"].tolist(), _lengths_of(state)
    slots = len(pages)
    free = sorted(set(range(key.shape[1])) - {p for row in pages for p in row if p >= 0})
    for slot in range(s, slots):
        n = lengths[slot] = lengths[slot % s]
        pages[slot] = list(pages[slot % s])
        if n % b:
            last, new = n // b, free.pop(0)
            for pool in (key, value):
                pool[:, new, :, :n % b] = pool[:, pages[slot][last], :, :n % b]
            pages[slot][last] = new
    if case["keep"] < 1.0:
        for slot in range(s, slots):
            kept = torch.nonzero(state["keep"][slot, :lengths[slot]]).view(-1).tolist()
            if len(kept) == lengths[slot]:
                continue
            whole = next(i for i, t in enumerate([*kept, -1]) if t != i) // b
            new = {j: free.pop(0) for j in range(whole, -(-len(kept) // b))}
            rows = range(whole * b, len(kept))
            source = [pages[slot][kept[j] // b] for j in rows], [kept[j] % b for j in rows]
            target = [new[j // b] for j in rows], [j % b for j in rows]
            for pool in (key, value):
                pool[:, target[0], :, target[1]] = pool[:, source[0], :, source[1]]
    return {"key": key, "value": value, **{n: None for n in ("table", "lengths", "references", "free_pages")}}


def exact(case, seed):
    kind = case["kind"]
    state = prepare(case, seed)
    s, b = case["seqs"], case["page"]
    if kind == "pages":
        return _exact_pages(state, case)
    if kind == "rotate":
        return {n: _exact_turn(state[x], state["positions"], case) for n, x in (("query", "query"), ("key", "new_key"))}
    pages, lengths = state["table"].tolist(), _lengths_of(state)
    if kind == "attend":
        counts = _counts(case, case["lq"])
        outs, lses = [], []
        for i in range(s):
            rows = [_sequence(state[n][0], pages[i][:-(-lengths[i] // b)], lengths[i]) for n in ("key", "value")]
            ends = [(lengths[i] - counts[i] + j + 1 if case["causal"] else lengths[i]) if j < counts[i] else 0
                    for j in range(case["lq"])]
            out, lse = _exact_attention(*rows, state["query"][i], ends)
            outs.append(out)
            lses.append(lse)
        return {"out": torch.stack(outs), "lse": torch.stack(lses)}
    if kind == "write":
        key, value = state["key"].double(), state["value"].double()
        turned = _exact_turn(state["new_key"], state["positions"], case)
        for i, count in enumerate(_counts(case, case["new"])):
            for j in range(0, count):
                if j and (lengths[i] - count + j) % b:
                    continue
                # the rows from j on that lie in one page
                t = lengths[i] - count + j
                n = min(b - t % b, count - j)
                page = pages[i][t // b]
                key[0, page, :, t % b:t % b + n] = turned[i, j:j + n].transpose(0, 1)
                value[0, page, :, t % b:t % b + n] = state["new_value"][i, j:j + n].double().transpose(0, 1)
        return {"query": _exact_turn(state["query"], state["positions"], case), "key": key, "value": value}
    new, dtype = case["new"], _DTYPES[case["dtype"]]
    outs, lses = [], []
    positions = torch.tensor([[list(range(n, n + new)) for n in lengths]], device="cuda")
    for layer in range(case["layers"]):
        turned = _exact_turn(state["new_key"][layer], positions, case).to(dtype)  # as they are held
        # (the kernels attend with rotated queries of the cache's type)
        query = _exact_turn(state["query"][layer], positions, case).to(dtype)
        out, lse = [], []
        for i in range(s):
            held = pages[i][:-(-lengths[i] // b)]
            k, v = (_sequence(state[n][layer], held, lengths[i]) for n in ("key", "value"))
            k, v = torch.cat([k, turned[i]]), torch.cat([v, state["new_value"][layer, i]])
            o, l = _exact_attention(k, v, query[i], [lengths[i] + j + 1 for j in range(new)])
            out.append(o)
            lse.append(l)
        outs.append(torch.stack(out))
        lses.append(torch.stack(lse))
    return {"out": outs, "lse": lses,
            **{n: None for n in ("key", "value", "table", "lengths", "references", "free_pages")}}
