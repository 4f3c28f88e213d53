"""The way of a prompt as measured cases: positions turned into its queries and Keys, causal attention
over whole prompts, and the decode of a batch whose sequences continue one prompt.

* ``rotary`` -- query and Key rows are rotated by their tokens' positions (pairs of channels of both
  halves, or neighbouring ones; the whole head or its front part; frequencies stretched for long
  contexts).
* ``prompt`` -- causal attention of prompts of unlike lengths, grouped heads, packed one behind another
  in one row or padded to a batch; with ``history`` tokens whose Keys and Values are there already, the
  queries are the last ones (a long prompt fed in pieces, a single token).
* ``shared`` -- decode attention over the 4-bit row cache where groups of sequences share a prefix that
  is cached once, in front of each one's own rows.

Keys are N(0, 1) times a log-normal scale per channel with four outlier channels per head, Values
N(0, 1), queries N(0, 1) / sqrt(head_dim).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotary(batch, heads, tokens, *, low=None, packed=False, start=0, head_dim=128, rotary_dim=None, layout="half",
            base=10000.0, scaling="none", factor=1.0, original=4096, dtype="bf16", name=None):
    """``start``: the first token's position in every sequence (decode steps and later turns)."""
    case = {"kind": "rotary", "batch": batch, "n_q": heads[0], "n_kv": heads[1], "tokens": tokens,
            "low": tokens if low is None else low, "packed": packed, "start": start, "head_dim": head_dim,
            "rotary_dim": head_dim if rotary_dim is None else rotary_dim, "layout": layout, "base": base,
            "scaling": scaling, "factor": factor, "original": original, "dtype": dtype}
    return {**case, "name": name} if name else case


def _prompt(batch, heads, tokens, *, low=None, packed=True, history=0, head_dim=128, dtype="bf16", name=None):
    """``tokens``: the longest sequence's queries; ``history``: the most Keys in front of a sequence's own tokens."""
    case = {"kind": "prompt", "batch": batch, "n_q": heads[0], "n_kv": heads[1], "tokens": tokens,
            "low": tokens if low is None else low, "packed": packed, "history": history, "head_dim": head_dim,
            "dtype": dtype}
    return {**case, "name": name} if name else case


def _shared(prefixes, batch, heads, prefix, tokens, *, prefix_low=None, low=None, head_dim=128, page=128, group=128,
            q_len=1, dtype="bf16", name=None):
    """``prefix``: tokens of the longest shared prefix; ``tokens``: of the longest sequence behind its own."""
    case = {"kind": "shared", "prefixes": prefixes, "batch": batch, "n_q": heads[0], "n_kv": heads[1],
            "prefix": prefix, "prefix_low": prefix if prefix_low is None else prefix_low, "tokens": tokens,
            "low": tokens if low is None else low, "head_dim": head_dim, "page": page, "group": group,
            "q_len": q_len, "dtype": dtype}
    return {**case, "name": name} if name else case


def listed():
    return [
        # A decode step of a small model, 8 contexts around 8K tokens: latency.
        _rotary(8, (12, 2), 1, start=8191, name="rotary_one_token"),
        # Four requests' prompts packed behind one another, frequencies stretched fourfold for long contexts.
        _rotary(4, (28, 4), 16300, low=2000, packed=True, base=1e6, scaling="yarn", factor=4.0, original=32768,
                name="rotary_prompts"),
        # A later turn far into a document: neighbouring pairs, the front quarter of the head, float16.
        _rotary(3, (14, 2), 515, low=300, start=250001, head_dim=64, rotary_dim=16, layout="interleaved",
                scaling="linear", factor=8.0, dtype="fp16", name="rotary_part_far"),
        # One user's short prompt.
        _prompt(1, (28, 4), 1061, name="prompt_one_1k"),
        # A server's batch of prompts, packed.
        _prompt(8, (28, 4), 8190, low=300, name="prompt_packed_8k"),
        # Many short prompts for a small-head float16 model, padded to a batch.
        _prompt(16, (14, 2), 1500, low=1, packed=False, head_dim=64, dtype="fp16", name="prompt_padded_64"),
        # A long prompt fed in pieces: 512 tokens behind 16 384.
        _prompt(1, (28, 4), 512, history=16384, name="prompt_piece_512"),
        # A float32 model with one kv head per query head, wide heads.
        _prompt(2, (8, 8), 1500, low=900, head_dim=256, dtype="fp32", name="prompt_fp32_256"),
        # One long document, 14B-shaped heads.
        _prompt(1, (40, 8), 16384, name="prompt_one_16k"),
        # Eight samples of one chat behind a 1K system prompt: latency.
        _shared(1, 8, (12, 2), 1061, 200, low=20, name="shared_chat_1k"),
        # Sixteen samples of one 32K document, 7B-shaped heads.
        _shared(1, 16, (28, 4), 32768, 600, low=100, group=64, name="shared_batch_32k"),
        # Four documents with eight samples each, three drafted tokens to verify, float16.
        _shared(4, 32, (40, 8), 16300, 900, prefix_low=4000, low=64, q_len=3, dtype="fp16", name="shared_four_16k"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choices(("rotary", "prompt", "shared"), (3, 5, 4))[0]
    heads = rng.choice(((28, 4), (12, 2), (40, 8), (14, 2), (32, 8), (8, 8), (32, 4), (16, 1)))
    head_dim = rng.choice((64, 128, 128, 256))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp16", "fp32"))
    batch = _log_int(rng, 1, 32)
    spread = rng.random() < 0.6
    if kind == "rotary":
        tokens = rng.choice((1, _log_int(rng, 2, 32), _log_int(rng, 32, 16384)))
        scaling = rng.choice(("none", "linear", "ntk", "yarn"))
        case = _rotary(batch, heads, tokens, low=max(1, int(tokens * rng.uniform(0.1, 0.9))) if spread else None,
                       packed=rng.random() < 0.5, start=rng.choice((0, _log_int(rng, 1, 1000000))),
                       head_dim=head_dim, rotary_dim=rng.choice((head_dim, head_dim, head_dim // 2, head_dim // 4)),
                       layout=rng.choice(("half", "half", "interleaved")), base=rng.choice((1e4, 5e5, 1e6)),
                       scaling=scaling, factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                       original=rng.choice((4096, 32768)), dtype=dtype)
    elif kind == "prompt":
        tokens = rng.choice((1, _log_int(rng, 2, 64), _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)))
        history = rng.choice((0, 0, _log_int(rng, 1, 32768)))
        case = _prompt(batch, heads, tokens, low=max(1, int(tokens * rng.uniform(0.05, 0.9))) if spread else None,
                       packed=rng.random() < 0.7, history=history, head_dim=head_dim, dtype=dtype)
    else:
        prefixes = rng.choice((1, 1, 1, 2, 4))
        each = _log_int(rng, 1, 32 // prefixes)
        prefix, tokens = _log_int(rng, 64, 32768), _log_int(rng, 4, 2048)
        case = _shared(prefixes, prefixes * each, heads, prefix, tokens,
                       prefix_low=max(1, int(prefix * rng.uniform(0.1, 0.9))) if spread else None,
                       low=max(1, int(tokens * rng.uniform(0.1, 0.9))) if spread else None, head_dim=head_dim,
                       page=rng.choice((32, 64, 128, 128, 256)),
                       group=rng.choice([g for g in (32, 64, 128) if g <= head_dim]),
                       q_len=rng.choice((1, 1, 1, 2, 3, 5)), dtype=dtype)
    # no larger than the largest listed case of its kind
    same = [work(c) for c in listed() if c["kind"] == kind]
    top_bytes, top_flops = max(w["bytes"] for w in same), max(w["flops"] for w in same)
    while work(case)["bytes"] > top_bytes or work(case)["flops"] > top_flops:
        longest = "prefix" if kind == "shared" else "history" if case.get("history", 0) > case["tokens"] else "tokens"
        if case["batch"] > case.get("prefixes", 1):
            case["batch"] = (case["batch"] + 1) // 2
            if kind == "shared":
                case["batch"] = max(1, case["batch"] // case["prefixes"]) * case["prefixes"]
        elif case[longest] > 64:
            case[longest] = case[longest] * 2 // 3
            case["low"] = min(case["low"], case["tokens"])
            if kind == "shared":
                case["prefix_low"] = min(case["prefix_low"], case["prefix"])
        else:
            case["tokens"] = case["low"] = max(1, case["tokens"] // 2)
    return case


# ---- inputs -------------------------------------------------------------------------------------
def _spread(n, lo, hi):
    """``n`` lengths: the longest first, the others spread over [lo, hi]."""
    if lo == hi:
        return [hi] * n
    rng = random.Random(f"{n} {lo} {hi}")
    return [hi] + [rng.randint(lo, hi) for _ in range(n - 1)]


def _lengths(case):
    return _spread(case["batch"], case["low"], case["tokens"])


def _histories(case):
    return _spread(case["batch"], case["history"] // 4, case["history"])


def _prefixes(case):
    return _spread(case["prefixes"], case["prefix_low"], case["prefix"])


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _normal(shape, seed, dtype):
    g = torch.Generator(device=_device()).manual_seed(seed)
    return torch.randn(shape, generator=g, device=_device()).to(DTYPES[dtype])


def _scales(case, seed):
    """A Key channel's scale, ``[n_kv, head_dim]``."""
    g = torch.Generator(device=_device()).manual_seed(seed)
    sigma = torch.exp(torch.randn(case["n_kv"], case["head_dim"], generator=g, device=_device()))
    outlier = torch.rand(sigma.shape, generator=g, device=_device()).argsort(dim=-1) < 4
    return torch.where(outlier, 20.0 * sigma, sigma)


def _keys(shape, case, seed, which):
    """Keys ``[..., tokens, n_kv, head_dim]``."""
    g = torch.Generator(device=_device()).manual_seed(seed * 8 + which + (1 << 40))
    return (torch.randn(shape, generator=g, device=_device()) * _scales(case, seed)).to(DTYPES[case["dtype"]])


def _values(shape, case, seed, which):
    return _normal(shape, seed * 8 + which + (1 << 41), case["dtype"])


def _queries(shape, case, seed):
    g = torch.Generator(device=_device()).manual_seed(seed + (1 << 42))
    return (torch.randn(shape, generator=g, device=_device()) / math.sqrt(case["head_dim"])).to(DTYPES[case["dtype"]])


def _rows(case, lengths):
    """``(batch, tokens)`` of the tensors that hold sequences of ``lengths``."""
    return (1, sum(lengths)) if case["packed"] else (len(lengths), max(lengths))


def _places(case, lengths):
    """Where every sequence's rows are: ``(row of the batch, first token, tokens)``."""
    out, at = [], 0
    for b, n in enumerate(lengths):
        out.append((0, at, n) if case["packed"] else (b, 0, n))
        at += n
    return out


def _rotary_inputs(case, seed):
    """Query, Key ``[B, heads, T, D]`` as a projection leaves them (tokens outermost) and positions ``[B, T]``."""
    lengths = _lengths(case)
    B, T = _rows(case, lengths)
    query = _queries((B, T, case["n_q"], case["head_dim"]), case, seed).transpose(1, 2)
    key = _keys((B, T, case["n_kv"], case["head_dim"]), case, seed, 0).transpose(1, 2)
    positions = torch.zeros(B, T, dtype=torch.int64)
    for b, at, n in _places(case, lengths):
        positions[b, at : at + n] = case["start"] + torch.arange(n)
    return query, key, positions.to(_device())


def _prompt_inputs(case, seed):
    """Query ``[B, n_q, T, D]``, Key and Value ``[B, n_kv, S, D]``, tokens outermost in memory."""
    lengths = _lengths(case)
    total = [n + h for n, h in zip(lengths, _histories(case))]
    (B, T), (_, S) = _rows(case, lengths), _rows(case, total)
    query = _queries((B, T, case["n_q"], case["head_dim"]), case, seed).transpose(1, 2)
    key = _keys((B, S, case["n_kv"], case["head_dim"]), case, seed, 0).transpose(1, 2)
    value = _values((B, S, case["n_kv"], case["head_dim"]), case, seed, 0).transpose(1, 2)
    return query, key, value, lengths, total


def _shared_inputs(case, seed):
    """Rows of the prefixes and of the sequences ``[B, n_kv, T, D]``, queries ``[B, n_q, q_len, D]``."""
    H, D = case["n_kv"], case["head_dim"]
    out = []
    for which, (n, tokens) in enumerate(((case["prefixes"], case["prefix"]), (case["batch"], case["tokens"]))):
        out.append((_keys((n, tokens, H, D), case, seed, which).transpose(1, 2),
                    _values((n, tokens, H, D), case, seed, which).transpose(1, 2)))
    return (*out, _queries((case["batch"], case["n_q"], case["q_len"], D), case, seed))


def _stretch(case):
    """The argument that names a case's stretched frequencies, or None."""
    return None if case["scaling"] == "none" else {"type": case["scaling"], "factor": case["factor"],
                                                   "original_positions": case["original"]}


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "rotary":
        state["query"], state["key"], state["positions"] = _rotary_inputs(case, seed)
        if own:
            from logitfill_amd.packed import Rotary

            state["rotary"] = Rotary(case["head_dim"], case["base"], rotary_dim=case["rotary_dim"],
                                     layout=case["layout"], scaling=_stretch(case), device=_device())
        else:
            state["frequencies"] = [torch.tensor(x, dtype=torch.float64, device=_device()) for x in _frequencies(case)]
    elif case["kind"] == "prompt":
        state["query"], state["key"], state["value"], state["lengths"], state["total"] = _prompt_inputs(case, seed)
        if own:
            from logitfill_amd.packed import PromptPlan

            state["plan"] = PromptPlan(state["lengths"], state["total"], device=_device())
    else:
        before, behind, state["query"] = _shared_inputs(case, seed)
        if own:
            from logitfill_amd.packed import Int4KVManager

            shape = (1, case["n_q"], case["n_kv"], case["head_dim"], case["page"], case["group"], _device())
            prefix = Int4KVManager(*shape, batch_size=case["prefixes"], capacity_tokens=case["prefix"])
            prefix.commit(0, *before, _prefixes(case))
            manager = Int4KVManager(*shape, batch_size=case["batch"], capacity_tokens=case["tokens"], prefix=prefix)
            manager.commit(0, *behind, _lengths(case))
            state["manager"] = manager
        else:
            state["before"], state["behind"] = ([_quantise(x, case["group"]) for x in pair] for pair in (before, behind))
    return state


# ---- the operators in their plain form ------------------------------------------------------------
def _frequencies(case):
    """Angles per position of every pair of channels, and the factor on the rotated ones (float64)."""
    dim, base, s = case["rotary_dim"], case["base"], case["factor"]
    if case["scaling"] == "ntk":
        base = base * s ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if case["scaling"] == "linear":
        return [f / s for f in freq], 1.0
    if case["scaling"] != "yarn":
        return freq, 1.0

    def pair_of(turns):  # the pair that turns this often over the original context
        return dim * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))

    first, last = max(math.floor(pair_of(32)), 0), min(math.ceil(pair_of(1)), dim - 1)
    slow = [min(max((i - first) / max(last - first, 0.001), 0.0), 1.0) for i in range(dim // 2)]
    return [f / s * m + f * (1 - m) for f, m in zip(freq, slow)], 0.1 * math.log(s) + 1


def _plain_rotary(state):
    case, (freq, factor) = state["case"], state["frequencies"]
    # angles in 64 bits: of far positions, 32 lose them
    angle = state["positions"].double()[:, None, :, None] * freq
    cos, sin = ((f(angle) * factor).float() for f in (torch.cos, torch.sin))
    R, out = case["rotary_dim"], {}
    for name in ("query", "key"):
        x = state[name].float()
        y = torch.empty_like(x)
        y[..., R:] = x[..., R:]
        one, two = (slice(0, R // 2), slice(R // 2, R)) if case["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
        y[..., one] = x[..., one] * cos - x[..., two] * sin
        y[..., two] = x[..., two] * cos + x[..., one] * sin
        out[name] = y.to(state[name].dtype)
    return out


def _softmax_rows(scores, value):
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.bmm(p, value) / p.sum(-1, keepdim=True)


def _plain_prompt(state):
    case, query = state["case"], state["query"]
    H, D, g = case["n_kv"], case["head_dim"], case["n_q"] // case["n_kv"]
    B, T = query.shape[0], query.shape[2]
    out = torch.zeros(B, T, case["n_q"], D, dtype=query.dtype, device=query.device).transpose(1, 2)
    for (qb, qt, n), (kb, kt, total) in zip(_places(case, state["lengths"]), _places(case, state["total"])):
        key, value = (state[name][kb, :, kt : kt + total].float().contiguous() for name in ("key", "value"))
        for at in range(0, n, 1024):  # (blocks of queries, so that their scores fit)
            m = min(1024, n - at)
            seen = total - n + at + m  # rows that the block's last query sees
            q = query[qb, :, qt + at : qt + at + m].float().reshape(H, g * m, D)
            s = torch.bmm(q, key[:, :seen].transpose(1, 2).contiguous()) * D ** -0.5
            last = total - n + at + torch.arange(m, device=s.device).repeat(g)
            s.masked_fill_(torch.arange(seen, device=s.device)[None, None] > last[None, :, None], -math.inf)
            o = _softmax_rows(s, value[:, :seen])
            out[qb, :, qt + at : qt + at + m] = o.reshape(case["n_q"], m, D).to(query.dtype)
    return out


def _quantise(x, group):
    """Codes (uint8), scales and minima (float16) of ``x [..., D]`` per ``group`` channels; quotients in 64 bits,
    rounded to 32: a code is decided next to the border of two."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo).double() / 15).float().clamp(1e-5, 1e5)
    codes = ((g - lo).double() / scale.double()).float().round().clamp(0, 15).to(torch.uint8)
    return [codes.flatten(-2), scale.squeeze(-1).half(), lo.squeeze(-1).half()]


def _read(rows, at):
    """The float32 values that codes, scales and minima stand for."""
    codes, scale, lo = (r[at] for r in rows)
    g = codes.float().unflatten(-1, (scale.shape[-1], -1))
    return (g * scale.float()[..., None] + lo.float()[..., None]).flatten(-2)


def _plain_shared(state):
    case, query = state["case"], state["query"]
    H, n, D = case["n_kv"], case["q_len"], case["head_dim"]
    g, each = case["n_q"] // H, case["batch"] // case["prefixes"]
    out = torch.zeros_like(query)
    for p, common in enumerate(_prefixes(case)):
        key, value = (_read(rows, (p, slice(None), slice(0, common))) for rows in state["before"])
        # the scores of all the sequences' queries over their prefix at once
        q = query[p * each : (p + 1) * each].float().reshape(each, H, g * n, D).transpose(0, 1).reshape(H, -1, D)
        first = (torch.bmm(q, key.transpose(1, 2).contiguous()) * D ** -0.5).view(H, each, g * n, common)
        weights, sums = [], []
        for i in range(each):
            b = p * each + i
            total = _lengths(case)[b]
            k, v = (_read(rows, (b, slice(None), slice(0, total))) for rows in state["behind"])
            s = torch.bmm(q.view(H, each, g * n, D)[:, i].contiguous(), k.transpose(1, 2).contiguous()) * D ** -0.5
            last = (torch.arange(n, device=s.device).repeat(g) + total - n)[None, :, None]
            s = s.masked_fill(torch.arange(total, device=s.device) > last, -math.inf)
            w = first[:, i]
            if total < n:  # (the first queries stand inside the prefix)
                w = w.masked_fill(torch.arange(common, device=s.device) > common + last, -math.inf)
            most = torch.maximum(w.amax(-1, keepdim=True), s.amax(-1, keepdim=True))
            w, s = torch.exp(w - most), torch.exp(s - most)
            weights.append(w)
            sums.append((torch.bmm(s, v), w.sum(-1, keepdim=True) + s.sum(-1, keepdim=True)))
        o = torch.bmm(torch.cat(weights, 1), value).view(H, each, g * n, D)
        for i, (rest, total) in enumerate(sums):
            out[p * each + i] = ((o[:, i] + rest) / total).reshape(case["n_q"], n, D).to(query.dtype)
    return out


def run(state):
    case = state["case"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "shared": _plain_shared}[case["kind"]](state)
    if case["kind"] == "rotary":
        query, key = state["rotary"].rotate(state["query"], state["key"], state["positions"])
        return {"query": query, "key": key}
    from logitfill_amd.packed import int4_attention, prompt_attention

    scaling = case["head_dim"] ** -0.5
    if case["kind"] == "prompt":
        return prompt_attention(state["query"], state["key"], state["value"], scaling, state["plan"])
    return int4_attention(state["manager"], 0, state["query"], None, None, scaling)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    """Bytes: every row of the model's type read and written once, 4-bit rows as codes with a float16 scale and
    minimum per group; flops: six per rotated pair, the products of the attention."""
    D, H, size = case["head_dim"], case["n_kv"], 4 if case["dtype"] == "fp32" else 2
    lengths = _lengths(case)
    if case["kind"] == "rotary":
        B, T = _rows(case, lengths)
        return {"bytes": B * T * (2 * (case["n_q"] + H) * D * size + 8),
                "flops": B * T * (case["n_q"] + H) * 3 * case["rotary_dim"]}
    n_bytes = flops = 0
    if case["kind"] == "prompt":
        for n, h in zip(lengths, _histories(case)):
            n_bytes += size * D * (2 * case["n_q"] * n + 2 * H * (n + h))
            flops += 4 * case["n_q"] * D * (n * h + n * (n + 1) // 2)
        return {"bytes": n_bytes, "flops": flops}
    n = case["q_len"]
    row = D + 8 * (D // case["group"])  # Key and Value of one token and kv head
    each = case["batch"] // case["prefixes"]
    n_bytes = H * row * (sum(lengths) + sum(_prefixes(case))) + 2 * case["batch"] * case["n_q"] * n * D * size
    for p, common in enumerate(_prefixes(case)):
        for total in lengths[p * each : (p + 1) * each]:
            flops += 4 * case["n_q"] * D * sum(max(0, common + total - n + j + 1) for j in range(n))
    return {"bytes": n_bytes, "flops": flops}


# ---- the same in 64 bits ---------------------------------------------------------------------------
def _turn64(x, positions, case):
    """``x [B, heads, T, D]`` in float64, pair by pair multiplied by e^(i angle)."""
    R = case["rotary_dim"]
    freq, factor = _frequencies(case)
    angle = positions.double()[:, None, :, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    turned = x.double().clone()
    part = turned[..., :R]
    pairs = part.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (R // 2, 2))
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, factor), angle)
    pairs = torch.view_as_real(z)
    turned[..., :R] = (pairs.transpose(-1, -2) if case["layout"] == "half" else pairs).flatten(-2)
    return turned


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


def _attend64(q, k, v, last):
    """Causal attention of one head in float64: query i sees rows 0 .. ``last[i]``."""
    s = (q.double() @ k.t()) * q.shape[-1] ** -0.5
    s = s.masked_fill(torch.arange(k.shape[0], device=k.device)[None, :] > last[:, None], -math.inf)
    return torch.softmax(s, -1) @ v


def exact(case, seed):
    if case["kind"] == "rotary":
        query, key, positions = _rotary_inputs(case, seed)
        return {"query": _turn64(query, positions, case), "key": _turn64(key, positions, case)}
    g = case["n_q"] // case["n_kv"]
    if case["kind"] == "prompt":
        query, key, value, lengths, total = _prompt_inputs(case, seed)
        out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
        for (qb, qt, n), (kb, kt, m) in zip(_places(case, lengths), _places(case, total)):
            for h in range(case["n_q"]):
                k, v = (t[kb, h // g, kt : kt + m].double() for t in (key, value))
                for at in range(0, n, 4096):
                    end = min(n, at + 4096)
                    last = torch.arange(m - n + at, m - n + end, device=k.device)
                    seen = m - n + end
                    out[qb, h, qt + at : qt + end] = _attend64(query[qb, h, qt + at : qt + end], k[:seen], v[:seen], last)
        return out
    before, behind, query = _shared_inputs(case, seed)
    n, each = case["q_len"], case["batch"] // case["prefixes"]
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    for p, common in enumerate(_prefixes(case)):
        first = [_dense(x[p, :, :common], case["group"]) for x in before]
        for b in range(p * each, (p + 1) * each):
            total = _lengths(case)[b]
            k, v = (torch.cat([f, _dense(x[b, :, :total], case["group"])], 1) for f, x in zip(first, behind))
            last = torch.arange(n, device=k.device) + common + total - n
            for h in range(case["n_q"]):
                out[b, h] = _attend64(query[b, h], k[h // g], v[h // g], last)
    return out
