"""The 4-bit row cache's work as measured cases: writing rows and reading them back, attention over
the cached rows, attention over the pages that a score selects for each query.

A row is one token's Key or Value of one kv head.  It is kept as 4-bit codes with a scale and a
minimum (float16) per group of channels, quantised when it is written.  Kinds of case:

* ``write``  -- ``new`` tokens per sequence are written behind ``tokens`` cached ones (0: prompts
  into an empty cache) and read back; a full page's per-channel Key bounds are part of what a write
  leaves behind.
* ``attend`` -- attention of the last ``q_len`` tokens' queries over every cached row.
* ``sparse`` -- the pages of highest score are selected for each query token and kv head, and
  attended together with the query's own page.

Keys are N(0, 1) times a log-normal scale per channel with four outlier channels per head, Values
N(0, 1), queries N(0, 1) / sqrt(head_dim).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(kind, batch, heads, tokens, *, low=None, head_dim=128, page=128, group=128, new=0, q_len=1, top=0,
          dtype="bf16", name=None):
    """``tokens``: the longest context; ``low``: contexts are spread from it to ``tokens`` (None: all equal)."""
    case = {"kind": kind, "batch": batch, "n_q": heads[0], "n_kv": heads[1], "tokens": tokens,
            "low": tokens if low is None else low, "head_dim": head_dim, "page": page, "group": group, "new": new,
            "q_len": q_len, "top": top, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # A decode step's write: one token for each of 8 contexts, some of which fill a page with it.
        _case("write", 8, (12, 2), 8191, low=8000, new=1, name="write_one_token"),
        # The next turn of a chat with a small-head float16 model: 515 tokens behind what is there,
        # starting and ending inside pages.
        _case("write", 2, (14, 2), 1003, low=700, head_dim=64, page=64, group=32, new=515, dtype="fp16",
              name="write_next_turn"),
        # Prompts of four requests enter an empty cache, ragged up to 16K tokens.
        _case("write", 4, (28, 4), 0, new=16300, group=64, name="write_prompts"),
        # One user, a short chat: pure latency.
        _case("attend", 1, (28, 4), 1061, name="attend_one_1k"),
        # A small model's decode step at batch 8 and 8K context.
        _case("attend", 8, (12, 2), 8229, name="attend_small_8k"),
        # The 7B-shaped decode: batch 16, 32K context.
        _case("attend", 16, (28, 4), 32868, group=64, name="attend_batch_32k"),
        # A server's mixed batch of long contexts, the finest groups.
        _case("attend", 32, (40, 8), 65536, low=4096, group=32, name="attend_ragged_64k"),
        # A small-head float16 model, ragged.
        _case("attend", 8, (14, 2), 5003, low=1500, head_dim=64, page=64, group=32, dtype="fp16",
              name="attend_head_64"),
        # Speculative decoding: four drafted tokens per sequence are scored in one call.
        _case("attend", 16, (28, 4), 8192, low=2000, q_len=4, name="attend_verify_4"),
        # A long prompt fed in chunks: the last 512 of 16.9K tokens attend causally.
        _case("attend", 1, (28, 4), 16896, q_len=512, name="attend_chunk_512"),
        # The 7B-shaped decode over 32 selected pages of 256.
        _case("sparse", 16, (28, 4), 32868, group=64, top=32, name="sparse_batch_32k"),
        # One user with a very long document: 64 selected pages of 4 096, small pages.
        _case("sparse", 1, (28, 4), 262207, page=64, top=64, name="sparse_one_256k"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choices(("write", "attend", "chunk", "sparse"), (3, 5, 2, 3))[0]
    heads = rng.choice(((28, 4), (12, 2), (40, 8), (14, 2), (32, 8), (8, 8), (32, 4), (16, 1)))
    head_dim = rng.choice((64, 128, 128, 256))
    shape = {"head_dim": head_dim, "page": rng.choice((32, 64, 128, 128, 256)),
             "group": rng.choice([g for g in (32, 64, 128) if g <= head_dim]),
             "dtype": rng.choice(("bf16", "bf16", "bf16", "fp16", "fp16", "fp32"))}
    batch = _log_int(rng, 1, 32)
    tokens = _log_int(rng, 40, 65536)
    low = tokens if rng.random() < 0.4 else max(8, int(tokens * rng.uniform(0.1, 0.9)))
    if kind == "write":
        new = rng.choice((1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 16384)))
        if rng.random() < 0.5:
            tokens = low = 0
        case = _case("write", batch, heads, min(tokens, 8192), low=min(low, 8192), new=new, **shape)
    elif kind == "attend":
        case = _case("attend", batch, heads, tokens, low=low, q_len=rng.choice((1, 1, 1, 2, 3, 5, 8)), **shape)
    elif kind == "chunk":
        case = _case("attend", min(batch, 4), heads, tokens, low=low, q_len=_log_int(rng, 9, 600), **shape)
    else:
        case = _case("sparse", batch, heads, tokens, low=low, q_len=rng.choice((1, 1, 1, 2, 3)),
                     top=_log_int(rng, 1, 64), **shape)
    # no larger than the largest listed case of its kind
    same = [work(c) for c in listed() if c["kind"] == case["kind"]]
    top_bytes, top_flops = max(w["bytes"] for w in same), max(w["flops"] for w in same)
    while work(case)["bytes"] > top_bytes or work(case)["flops"] > top_flops:
        if case["batch"] > 1:
            case["batch"] = (case["batch"] + 1) // 2
        elif case["tokens"] > 1400:
            case["tokens"] = case["tokens"] * 2 // 3
            case["low"] = min(case["low"], case["tokens"])
        elif case["new"] > 1:
            case["new"] = (case["new"] + 1) // 2
        else:
            case["q_len"] = max(1, case["q_len"] // 2)
    return case


# ---- inputs -------------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens of every sequence: the longest first, the others spread over [low, tokens]."""
    n, lo, hi = case["batch"], case["low"], case["tokens"]
    if lo == hi:
        return [hi] * n
    rng = random.Random(f"{n} {lo} {hi}")
    return [hi] + [rng.randint(lo, hi) for _ in range(n - 1)]


def _new_lengths(case):
    """Tokens that a write adds: prompts into an empty cache are ragged, later turns alike."""
    n, new = case["batch"], case["new"]
    if case["tokens"] or new < 16:
        return [new] * n
    rng = random.Random(f"{n} {new}")
    return [new] + [rng.randint(max(1, new // 8), new) for _ in range(n - 1)]


def _rows(case, seed, which, tokens):
    """Key, Value ``[batch, n_kv, tokens, head_dim]``: the cached rows (``which`` 0) or the written ones (1)."""
    device = torch.device("cuda", torch.cuda.current_device())
    B, H, D = case["batch"], case["n_kv"], case["head_dim"]
    g = torch.Generator(device=device).manual_seed(seed)
    sigma = torch.exp(torch.randn(H, 1, D, generator=g, device=device))
    outlier = torch.rand(H, 1, D, generator=g, device=device).argsort(dim=-1) < 4
    sigma = torch.where(outlier, 20.0 * sigma, sigma)
    g = torch.Generator(device=device).manual_seed(seed * 2 + which + (1 << 40))
    key = torch.empty(B, H, tokens, D, dtype=DTYPES[case["dtype"]], device=device)
    value = torch.empty_like(key)
    for b in range(B):
        key[b] = torch.randn(H, tokens, D, generator=g, device=device).mul_(sigma)
        value[b] = torch.randn(H, tokens, D, generator=g, device=device)
    return key, value


def _query(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed + (1 << 41))
    D = case["head_dim"]
    q = torch.randn(case["batch"], case["n_q"], case["q_len"], D, generator=g, device=device) / math.sqrt(D)
    return q.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    lengths = _lengths(case)
    state = {"case": case, "lengths": lengths, "scaling": case["head_dim"] ** -0.5}
    key, value = _rows(case, seed, 0, case["tokens"])
    if own:
        from logitfill_amd.packed import Int4KVManager

        mgr = Int4KVManager(1, case["n_q"], case["n_kv"], case["head_dim"], case["page"], case["group"], key.device,
                            batch_size=case["batch"], capacity_tokens=case["tokens"] + case["new"])
        if case["tokens"]:
            mgr.commit(0, key, value, lengths)
        state["mgr"] = mgr
    else:
        rows = _quantise(key, case["group"]) + _quantise(value, case["group"])
        state["rows"] = rows
        state["bounds"] = _bounds(case, rows[:3], lengths) if case["kind"] == "sparse" else None
    del key, value
    if case["kind"] == "write":
        state["new"] = _rows(case, seed, 1, case["new"])
        state["new_lengths"] = _new_lengths(case)
        # what a pass may find of an earlier one: the first page it completes and the last
        state["first_page"] = min(lengths) // case["page"]
        state["last_page"] = max(n + m for n, m in zip(lengths, state["new_lengths"])) // case["page"]
    else:
        state["query"] = _query(case, seed)
    return state


# ---- the operators in their plain form --------------------------------------------------------------
def _quantise(x, group):
    """Codes (uint8), scales and minima (float16) of ``x [..., D]`` per ``group`` channels.  The two
    quotients are formed in 64 bits and rounded to 32: a code is decided next to the border of two."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo).double() / 15).float().clamp(1e-5, 1e5)
    codes = ((g - lo).double() / scale.double()).float().round().clamp(0, 15).to(torch.uint8)
    return [codes.flatten(-2), scale.squeeze(-1).half(), lo.squeeze(-1).half()]


def _values(rows, at=...):
    """The float32 values that codes, scales and minima stand for."""
    codes, scale, lo = (r[at] for r in rows)
    g = codes.float().unflatten(-1, (scale.shape[-1], -1))
    return (g * scale.float()[..., None] + lo.float()[..., None]).flatten(-2)


def _upward(x):
    """float32 rounded up to the next bfloat16."""
    bits = x.contiguous().view(torch.int32)
    return (torch.where(bits >= 0, bits + 0xFFFF, bits) >> 16 << 16).view(torch.float32)


def _bounds(case, key_rows, lengths, first=0, last=None):
    """Outward bfloat16 bounds ``[batch, n_kv, pages, 2, D]`` of every full page's Keys (zeros where a
    sequence has no such page)."""
    P, D = case["page"], case["head_dim"]
    last = max(lengths) // P if last is None else last
    out = torch.zeros(case["batch"], case["n_kv"], last - first, 2, D, device=key_rows[0].device)
    for b, n in enumerate(lengths):
        full = n // P
        if full > first:
            v = _values(key_rows, (b, slice(None), slice(first * P, full * P))).unflatten(1, (-1, P))
            out[b, :, : full - first, 0] = -_upward(-v.amin(2))
            out[b, :, : full - first, 1] = _upward(v.amax(2))
    return out.bfloat16()


def _softmax_rows(scores, value):
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.bmm(p, value) / p.sum(-1, keepdim=True)


def _plain_write(state):
    case = state["case"]
    out, cached = [], []
    for x, rows in zip(state["new"], (state["rows"][:3], state["rows"][3:])):
        new = _quantise(x, case["group"])
        out.append(_values(new).to(x.dtype))
        cached.append((rows, new))
    for t in out:  # rows behind a sequence's last one are no rows
        for b, m in enumerate(state["new_lengths"]):
            t[b, :, m:] = 0
    P, first = case["page"], state["first_page"]
    ends = [n + m for n, m in zip(state["lengths"], state["new_lengths"])]
    bounds = torch.zeros(case["batch"], case["n_kv"], state["last_page"] - first, 2, case["head_dim"],
                         dtype=torch.bfloat16, device=out[0].device)
    (old, new) = cached[0]
    for b, (n, end) in enumerate(zip(state["lengths"], ends)):
        if end // P > first:
            # the rows of the pages that this write may complete, old ones first
            rows = [torch.cat([o[b : b + 1, :, first * P : n], w[b : b + 1, :, : end - n]], 2)
                    for o, w in zip(old, new)]
            one = {**case, "batch": 1}
            bounds[b, :, : end // P - first] = _bounds(one, rows, [end - first * P])[0]
    return {"key": out[0], "value": out[1], "bounds": bounds}


def _plain_attend(state):
    case, query = state["case"], state["query"]
    H, n, D = case["n_kv"], case["q_len"], case["head_dim"]
    out = torch.zeros_like(query)
    for b, total in enumerate(state["lengths"]):
        key = _values(state["rows"][:3], (b, slice(None), slice(0, total)))
        value = _values(state["rows"][3:], (b, slice(None), slice(0, total)))
        q = query[b].float().reshape(H, -1, D)  # row = head of the group x token
        scores = torch.bmm(q, key.transpose(1, 2).contiguous()) * state["scaling"]
        if n > 1:
            last = torch.arange(n, device=q.device).repeat(case["n_q"] // H) + total - n
            scores.masked_fill_(torch.arange(total, device=q.device)[None, None, :] > last[None, :, None], -math.inf)
            blind = last < 0  # a query in front of the first token sees nothing
            scores[:, blind] = 0
            o = _softmax_rows(scores, value)
            o[:, blind] = 0
        else:
            o = _softmax_rows(scores, value)
        out[b] = o.reshape(case["n_q"], n, D).to(query.dtype)
    return out


def _plain_sparse(state):
    case, query = state["case"], state["query"]
    H, n, D, P, top = case["n_kv"], case["q_len"], case["head_dim"], case["page"], case["top"]
    device = query.device
    pages = torch.full((case["batch"], H, n, top), -1, dtype=torch.int32, device=device)
    out = torch.zeros_like(query)
    head = torch.arange(H, device=device)[:, None]
    for b, total in enumerate(state["lengths"]):
        q = query[b].reshape(H, -1, n, D)
        for j in range(n):
            last = total - n + j
            if last < 0:
                continue
            own_page = last // P
            qj = q[:, :, j]
            picked = torch.zeros(H, 0, dtype=torch.int64, device=device)
            if own_page:
                # 64 bits: a page is chosen next to the border of the last one that is not
                lo, hi = (state["bounds"][b, :, :own_page, i].double()[:, None] for i in (0, 1))
                wide = qj.double()[:, :, None]
                score = torch.maximum(wide * lo, wide * hi).sum(-1).amax(1)
                order = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :top]
                picked = order.sort(-1).values
                pages[b, :, j, : picked.shape[1]] = picked.int()
            rows = (picked[:, :, None] * P + torch.arange(P, device=device)).flatten(1)
            local = torch.arange(own_page * P, last + 1, device=device).expand(H, -1)
            rows = torch.cat([rows, local], 1)
            key = _values([r[b] for r in state["rows"][:3]], (head, rows))
            value = _values([r[b] for r in state["rows"][3:]], (head, rows))
            scores = torch.bmm(qj.float(), key.transpose(1, 2).contiguous()) * state["scaling"]
            out[b].view(H, -1, n, D)[:, :, j] = _softmax_rows(scores, value).to(query.dtype)
    return {"pages": pages, "out": out}


def run(state):
    case = state["case"]
    if not own:
        return {"write": _plain_write, "attend": _plain_attend, "sparse": _plain_sparse}[case["kind"]](state)
    from logitfill_amd.packed import int4_attention, select_pages

    mgr = state["mgr"]
    if case["kind"] == "write":
        mgr.truncate(state["lengths"])
        mgr.commit(0, *state["new"], state["new_lengths"])
        key, value = mgr.layers[0].read(state["lengths"], case["new"], state["new"][0].dtype)
        bounds = mgr.layers[0].page_bounds()[:, :, state["first_page"] : state["last_page"]]
        return {"key": key, "value": value, "bounds": bounds}
    if case["kind"] == "attend":
        return int4_attention(mgr, 0, state["query"], None, None, state["scaling"])
    pages = select_pages(mgr, 0, state["query"], case["top"])
    return {"pages": pages, "out": int4_attention(mgr, 0, state["query"], None, None, state["scaling"], pages=pages)}


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    """Bytes: codes at 4 bits, a float16 scale and minimum per group, rows of the model's type, page
    bounds, each once; flops: the products of the attention and of the scores, 8 per element written."""
    D, H, P, B = case["head_dim"], case["n_kv"], case["page"], case["batch"]
    size = 4 if case["dtype"] == "fp32" else 2
    row = D + 8 * (D // case["group"])  # Key and Value of one token and kv head
    raw = 2 * size * D
    n_bytes = flops = 0
    if case["kind"] == "write":
        for n, m in zip(_lengths(case), _new_lengths(case)):
            pages = (n + m) // P - n // P
            # read, written as codes, read back, written as rows; the bounds of completed pages
            n_bytes += H * (m * (raw + 2 * row + raw) + pages * 4 * D)
            flops += 16 * H * m * D
        return {"bytes": n_bytes, "flops": flops}
    n = case["q_len"]
    n_bytes = 2 * B * case["n_q"] * n * D * size
    for total in _lengths(case):
        if case["kind"] == "attend":
            n_bytes += H * total * row
            flops += 4 * case["n_q"] * D * sum(max(0, total - n + j + 1) for j in range(n))
            continue
        n_bytes += H * max(0, total - 1) // P * 4 * D
        seen = 0
        for j in range(n):
            last = total - n + j
            if last < 0:
                continue
            rows = min(case["top"], last // P) * P + last % P + 1
            seen += rows
            flops += case["n_q"] * D * (4 * rows + 3 * (last // P))
        n_bytes += H * min(seen, total) * row + B * H * n * case["top"] * 4
    return {"bytes": int(n_bytes), "flops": int(flops)}


# ---- the same in 64 bits ---------------------------------------------------------------------------
def _dense(x, group):
    """Float64 of what the cache holds of ``x [..., D]``: the code rule's steps rounded to float32 as the
    format says (differences, scale, quotient), scale and minimum to float16."""
    shape = x.shape
    x = x.double().reshape(*shape[:-1], shape[-1] // group, group)
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values

    def step(t):
        return t.float().double()

    scale = step(torch.clamp(step(step(hi - lo) / 15), step(torch.tensor(1e-5)).item(), 1e5))
    codes = torch.clamp(torch.round(step(step(x - lo) / scale)), 0, 15)
    return (codes * scale.half().double() + lo.half().double()).reshape(shape)


def _outward(dense, P):
    """Float64 ``[n_kv, pages, 2, D]``: per-channel bounds of every full page of ``dense [n_kv, T, D]``,
    taken from the float32 values, moved outward to bfloat16."""
    H, T, D = dense.shape
    v = dense[:, : T // P * P].float().reshape(H, T // P, P, D)
    out = []
    for t, sign in ((v.min(2).values, -1), (v.max(2).values, 1)):
        near = t.bfloat16()
        step = torch.nextafter(near.cpu(), torch.full_like(near.cpu(), sign * math.inf)).to(t.device)
        short = (t - near.float()) * sign > 0
        out.append(torch.where(short, step, near).double())
    return torch.stack(out, 2)


def _attention64(q, key, value, scaling, hidden=None):
    s = (q @ key.t()) * scaling
    if hidden is not None:
        s = s.masked_fill(hidden, -math.inf)
    return torch.softmax(s, -1) @ value


def exact(case, seed):
    lengths, P, n, top = _lengths(case), case["page"], case["q_len"], case["top"]
    key, value = _rows(case, seed, 0, case["tokens"])
    H, D, B = case["n_kv"], case["head_dim"], case["batch"]
    if case["kind"] == "write":
        new_k, new_v = _rows(case, seed, 1, case["new"])
        added = _new_lengths(case)
        first = min(lengths) // P
        last = max(a + m for a, m in zip(lengths, added)) // P
        out = {"key": torch.zeros(new_k.shape, dtype=torch.float64, device=key.device),
               "value": torch.zeros(new_k.shape, dtype=torch.float64, device=key.device),
               "bounds": torch.zeros(B, H, last - first, 2, D, dtype=torch.float64, device=key.device)}
        for b, (a, m) in enumerate(zip(lengths, added)):
            k = _dense(new_k[b, :, :m], case["group"])
            out["key"][b, :, :m] = k
            out["value"][b, :, :m] = _dense(new_v[b, :, :m], case["group"])
            k = torch.cat([_dense(key[b, :, first * P : a], case["group"]), k], 1)
            if k.shape[1] >= P:
                bounds = _outward(k, P)
                out["bounds"][b, :, : bounds.shape[1]] = bounds
        return out
    query = _query(case, seed)
    group = case["n_q"] // H
    out = torch.zeros(query.shape, dtype=torch.float64, device=key.device)
    for b, total in enumerate(lengths):
        for h in range(H):
            k, v = _dense(key[b, h, :total], case["group"]), _dense(value[b, h, :total], case["group"])
            bounds = _outward(k[None], P)[0] if case["kind"] == "sparse" and total >= P else None
            for j in range(n) if case["kind"] == "sparse" else (None,):
                if j is None:
                    at = torch.arange(total, device=k.device)[None, :]
                    seen = torch.arange(n, device=k.device)[:, None] + total - n
                    for i in range(h * group, (h + 1) * group):
                        o = _attention64(query[b, i].double(), k, v, D ** -0.5, at > seen)
                        out[b, i] = torch.where(seen < 0, 0.0, o)
                    continue
                last = total - n + j
                if last < 0:
                    continue
                q = query[b, h * group : (h + 1) * group, j].double()
                keep = torch.arange(total, device=k.device) // P == last // P
                if last // P:
                    above = bounds[: last // P]
                    score = torch.stack([torch.maximum(r * above[:, 0], r * above[:, 1]).sum(-1) for r in q])
                    score = score.max(0).values
                    # a page's place: how many pages come before it
                    index = torch.arange(score.numel(), device=k.device)
                    place = torch.empty_like(index)
                    for at in index.split(512):
                        ahead = (score[None, :] > score[at, None]) | (
                            (score[None, :] == score[at, None]) & (index[None, :] < at[:, None]))
                        place[at] = ahead.sum(1)
                    chosen = torch.zeros(total // P + 1, dtype=torch.bool, device=k.device)
                    chosen[: last // P] = place < top
                    keep = keep | chosen[torch.arange(total, device=k.device) // P]
                keep = keep & (torch.arange(total, device=k.device) <= last)
                out[b, h * group : (h + 1) * group, j] = _attention64(q, k[keep], v[keep], D ** -0.5)
    # the selected pages are whole numbers, compared between implementations
    return {"pages": None, "out": out} if case["kind"] == "sparse" else out
