"""The operators that a decoder serves tokens with, as cases that can be timed: rotary positions of heads (with a norm of
each head in the same pass), keys and values appended to a paged cache, and attention that reads such a cache.

    listed()           the cases
    draw(rng)          one more case of the same ranges
    prepare(case, s)   inputs made from the seed `s`, and the descriptions of cache and batch that a program keeps
    run(state)         one pass: in elementary torch operations, or (own) by this package's operators; the outputs whole
    work(case)         bytes (inputs and outputs once) and operations of one pass
    exact(case, s)     the outputs by the operators' definitions, in 64 bits

Definitions.  A head's channels (i, i + r/2), or (2 i, 2 i + 1) where interleaved, of its first r turn by position x
frequency i; a norm in front divides the head by its root mean square and multiplies it by weights.  Token t of a sequence
with n tokens in the call and a length L after them stands at place L - n + t, in slot place % page_size of the sequence's
page place / page_size.  It sees the keys [low, high): high = L, or place + 1 where causal, at least the sequence's prefix;
low = place - window + 1 where there is a window, at least the token's first key.  Scores are q k scale, then
cap tanh(score / cap), then less slope |place - key|; a row that sees nothing is zero.
"""
import functools
import math

import numpy as np
import torch

own = False

HALVES, INTERLEAVED = "halves", "interleaved"


# ---- the cases -------------------------------------------------------------------------------------------------------

def _rotary(name, batch, tokens, heads, size, turned, layout, norm, order, far):
    return {"name": name, "kind": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "size": size, "turned": turned,
            "layout": layout, "norm": norm, "order": order, "far": far}


def _append(name, sequences, least, most, before, heads, kv, size, turned, layout, norm, type_, page, order, spare):
    return {"name": name, "kind": "append", "sequences": sequences, "least": least, "most": most, "before": before, "heads": heads,
            "kv": kv, "size": size, "turned": turned, "layout": layout, "norm": norm, "type": type_, "page": page, "order": order, "spare": spare}


def _attend(name, sequences, least, most, before_least, before, heads, kv, size, type_, page, order, causal=True, window=0, cap=0.0,
            slopes=False, prefix=False, documents=0, spare=0):
    return {"name": name, "kind": "attend", "sequences": sequences, "least": least, "most": most, "before_least": before_least,
            "before": before, "heads": heads, "kv": kv, "size": size, "type": type_, "page": page, "order": order, "causal": causal,
            "window": window, "cap": cap, "slopes": slopes, "prefix": prefix, "documents": documents, "spare": spare}


def listed():
    return [
        # The queries of one new token in a small decoder: the smallest call, all launch and latency.
        _rotary("rotary_token", 1, 1, 12, 64, 64, HALVES, False, "token", 900),
        # Four prompts of 1024 tokens, each head normed first, in frequencies stretched for long contexts.
        _rotary("rotary_prompt_norm", 4, 1024, 16, 128, 128, HALVES, True, "token", 0),
        # Odd sizes: half of each head turns, neighbours in pairs, heads in front of tokens, far into a long context.
        _rotary("rotary_odd_far", 3, 1777, 9, 80, 40, INTERLEAVED, False, "head", 120000),
        # One new token of each of 64 sequences, out of one packed product; eight query heads for two of keys.
        _append("append_tokens_64", 64, 1, 1, 4000, 32, 8, 128, 128, HALVES, False, "f32", 16, "head", 0),
        # Ragged prompts into a cache in bf16, heads normed, with rows of padding behind the last prompt.
        _append("append_prompts_bf16", 9, 100, 1024, 0, 16, 4, 128, 128, HALVES, True, "bf16", 64, "slot", 61),
        # One new token behind a prompt of 76: the smallest attention, all latency.
        _attend("attend_token_77", 1, 1, 1, 76, 76, 12, 12, 64, "f32", 16, "head"),
        # One new token of one sequence behind a long document: few rows, a long axis.
        _attend("attend_token_long", 1, 1, 1, 65535, 65535, 32, 8, 128, "f32", 16, "head"),
        # One new token of each of 48 sequences of all lengths, cache in bf16, capped scores.
        _attend("attend_tokens_ragged_bf16", 48, 1, 1, 100, 8191, 32, 4, 128, "bf16", 16, "slot", cap=50.0),
        # Four prompts of a small decoder's whole context.
        _attend("attend_prompts", 4, 1024, 1024, 0, 0, 12, 12, 64, "f32", 64, "head"),
        # A long prompt over a window, capped scores, cache in bf16.
        _attend("attend_prompt_window_bf16", 1, 4096, 4096, 0, 0, 16, 4, 128, "bf16", 64, "head", window=1500, cap=30.0),
        # Pieces of prompts on top of what earlier pieces left, a bias by distance, pages that end inside a tile.
        _attend("attend_pieces_bias", 5, 57, 333, 500, 4801, 8, 8, 96, "f32", 24, "head", slopes=True),
        # Training-style rows: documents packed into one, the first part of each row open to all; padding behind.
        _attend("attend_documents", 3, 1500, 2048, 0, 0, 16, 4, 128, "f32", 32, "slot", documents=190, prefix=True, spare=7),
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most = [_cost(c) for c in listed()]
    most = [max(c[i] for c in most) for i in range(3)]
    while True:
        case = _drawn(rng)
        if all(mine <= m for mine, m in zip(_cost(case), most)):
            return case


def _cost(case):
    """Bytes, operations and, for attention with all sequences as long as the longest, the number of scores."""
    w, scores = work(case), 0
    if case["kind"] == "attend":
        n, length = _lengths(case)
        scores = case["sequences"] * case["heads"] * int(n.max()) * int(length.max())
    return w["bytes"], w["flops"], scores


def _drawn(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend"])
    layout, order, type_ = rng.choice([HALVES, INTERLEAVED]), rng.choice(["head", "slot"]), rng.choice(["f32", "bf16"])
    size = rng.choice([64, 64, 80, 96, 128, 128, 128])
    turned = size if rng.random() < 0.6 else size // 2
    if kind == "rotary":
        return _rotary_case(rng, size, turned, layout)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    page = rng.choice([8, 16, 16, 24, 64, 128, 250])
    if kind == "append":
        most = _log(rng, 1, 1500)
        case = _append("", _log(rng, 1, 64 if most < 200 else 8), max(1, most // rng.choice([1, 1, 3])), most, _log(rng, 1, 3000) - 1, heads, kv, size, turned,
                       layout, rng.random() < 0.5, type_, page, order, rng.choice([0, 0, 5, 64]))
    elif rng.random() < 0.5:
        most = _log(rng, 16, 20000)
        case = _attend("", _log(rng, 1, max(1, min(64, 300000 // most))), 1, rng.choice([1, 1, 1, 3]), max(8, most // rng.choice([1, 4, 50])), most, heads, kv, size,
                       type_, page, order, window=rng.choice([0, 0, 0, 700]), cap=rng.choice([0.0, 0.0, 50.0]), slopes=rng.random() < 0.3)
    else:
        most = _log(rng, 17, 2500)
        before = rng.choice([0, 0, _log(rng, 1, 3000)])
        case = _attend("", _log(rng, 1, 4 if most < 1000 else 2), max(1, most // rng.choice([1, 1, 3])), most, before // 2, before, heads, kv, size, type_, page,
                       order, causal=rng.random() < 0.8, window=rng.choice([0, 0, 0, 300]), cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3,
                       prefix=rng.random() < 0.25, documents=rng.choice([0, 0, 130]), spare=rng.choice([0, 0, 9]))
    del case["name"]
    return case


def _rotary_case(rng, size, turned, layout):
    tokens = _log(rng, 1, 4000)
    case = _rotary("", _log(rng, 1, max(1, min(16, 16000 // tokens))), tokens, rng.randint(1, 32), size, turned, layout, rng.random() < 0.5,
                   rng.choice(["token", "head"]), rng.choice([0, 0, 3000, 120000]))
    del case["name"]
    return case


# ---- sizes that follow from a case -----------------------------------------------------------------------------------

def _spread(low, high, count):
    """`count` whole numbers from low to high, the two ends among them, in no order of size (steps of the golden section)."""
    part = (0.6180339887498949 * np.arange(1, count + 1)) % 1.0
    values = low + np.floor(part * (high - low + 1)).astype(np.int64)
    values[0] = high
    if count > 1:
        values[-1] = low
    return values


def _lengths(case):
    """(tokens of each sequence in the call, its length after them)."""
    n = _spread(case["least"], case["most"], case["sequences"])
    low = case.get("before_least", case["before"] // 3)
    return n, n + _spread(low, case["before"], case["sequences"])[::-1]


def _prefix_and_first(case, n, length):
    """What a batch of packed rows brings along: keys in front that all see, and the first key of each token's document."""
    prefix = np.maximum(1, length // 5) if case["prefix"] else None
    first = None
    if case["documents"]:
        places = [np.arange(l - m, l) for m, l in zip(n, length)]
        first = np.concatenate([p // case["documents"] * case["documents"] for p in places] + [np.zeros(case["spare"], np.int64)])
    return prefix, first


def _ranges(case, n, length):
    """[low, high) of each token's keys, one pair of arrays for each sequence."""
    prefix, first = _prefix_and_first(case, n, length)
    out, at = [], 0
    for s, (m, l) in enumerate(zip(n, length)):
        place = np.arange(l - m, l)
        high = place + 1 if case["causal"] else np.full(m, l)
        if prefix is not None:
            high = np.maximum(high, min(prefix[s], l))
        low = np.maximum(0, place - case["window"] + 1) if case["window"] else np.zeros(m, np.int64)
        if first is not None:
            low = np.maximum(low, first[at:at + m])
        out.append((low, np.maximum(low, high)))
        at += m
    return out


def _frequencies(turned, stretched):
    """Radians by which each pair turns per position, base 10000; stretched: pairs with less than one turn in 1024 positions
    eight times slower, those with more than four as they are, between the two in proportion."""
    f = 10000.0 ** (-np.arange(0, turned, 2, dtype=np.float64) / turned)
    if stretched:
        turns = 1024 * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / 8.0)
    return f


EPSILON = 1e-6
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- what a program has in hand --------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=1)
def _context():
    from altius_amd import device
    return device.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)  # noqa: E731
    whole = lambda values: torch.tensor(np.asarray(values), device="cuda", dtype=torch.int32)  # noqa: E731
    s = {"case": dict(case)}
    d = case["size"]
    if case["kind"] == "rotary":
        b, t, h = case["batch"], case["tokens"], case["heads"]
        s["x"] = normal(b, t, h, d) if case["order"] == "token" else normal(b, h, t, d).transpose(1, 2)
        s["out"] = torch.empty_like(s["x"])  # laid out as x is
        s["positions"] = torch.randint(0, 64, (b, 1), generator=gen, device="cuda", dtype=torch.int32) + whole(np.arange(t) + case["far"])
        s["gamma"] = 1 + 0.1 * normal(d) if case["norm"] else None
        s["frequencies"] = torch.tensor(_frequencies(case["turned"], case["norm"]), device="cuda")
        s["call"] = None
        if own:
            _rotary_call(s)
        return s
    n, length = _lengths(case)
    q, kv, page = case["heads"], case["kv"], case["page"]
    s["starts"] = whole(np.concatenate([[0], np.cumsum(n)]))
    s["lengths"] = whole(length)
    s["most"], s["longest"] = int(n.max()), int(length.max())
    tokens = int(n.sum()) + case["spare"]
    per = -(-s["longest"] // page)
    pages = case["sequences"] * per + 3
    s["table"] = torch.randperm(pages, generator=gen, device="cuda")[:case["sequences"] * per].to(torch.int32).reshape(case["sequences"], per)
    shape = (pages, kv, page, d) if case["order"] == "head" else (pages, page, kv, d)
    for name in ("keys", "values"):
        cache = normal(*shape).to(_TORCH[case["type"]]) if case["kind"] == "attend" else torch.zeros(shape, device="cuda", dtype=_TORCH[case["type"]])
        s[name + "_whole"] = cache
        s[name] = cache if case["order"] == "head" else cache.transpose(1, 2)  # [pages, kv, page, d] either way
    if case["kind"] == "append":
        packed = normal(tokens, q + 2 * kv, d)
        s["q"], s["k"], s["v"] = packed[:, :q], packed[:, q:q + kv], packed[:, q + kv:]
        s["q_out"] = torch.zeros((tokens, q, d), device="cuda")
        s["q_gamma"], s["k_gamma"] = (1 + 0.1 * normal(d), 1 + 0.1 * normal(d)) if case["norm"] else (None, None)
        s["frequencies"] = torch.tensor(_frequencies(case["turned"], case["norm"]), device="cuda")
    else:
        prefix, first = _prefix_and_first(case, n, length)
        s["q"] = 1.5 * normal(tokens, q, d)
        s["out"] = torch.zeros((tokens, q, d), device="cuda")
        s["scale"] = 1.0 / math.sqrt(d)
        s["prefix"] = None if prefix is None else whole(prefix)
        s["first"] = None if first is None else whole(first)
        s["slopes"] = torch.tensor(2.0 ** (-8.0 * np.arange(1, q + 1) / q), device="cuda", dtype=torch.float32) if case["slopes"] else None
    if own:
        _cache_call(s)
    return s


# ---- the package's operators -----------------------------------------------------------------------------------------

def _turning(s):
    from altius_amd import device as D
    return D.Rotary(s["frequencies"].data_ptr(), s["case"]["turned"], D.ROTARY_INTERLEAVED if s["case"]["layout"] == INTERLEAVED else D.ROTARY_HALVES)


def _pointer(x):
    return None if x is None else x.data_ptr()


def _rotary_call(s):
    from altius_amd import device as D
    b, t, h, d = s["x"].shape
    s["call"] = D.HeadRows(out=s["out"].data_ptr(), x=s["x"].data_ptr(), batch=b, tokens=t, heads=h, head_size=d, out_strides=s["out"].stride()[:3],
                           x_strides=s["x"].stride()[:3], positions=s["positions"].data_ptr(), position_stride=t, gamma=_pointer(s["gamma"]), epsilon=EPSILON)
    s["turning"], s["context"] = _turning(s), _context()


def _cache_call(s):
    from altius_amd import device as D
    case, strides = s["case"], s["keys"].stride()
    s["context"] = _context()
    s["cache"] = D.KvCache(keys=s["keys"].data_ptr(), values=s["values"].data_ptr(), elem=D.KV_BF16 if case["type"] == "bf16" else D.KV_F32, kv_heads=case["kv"],
                           head_size=case["size"], page_size=case["page"], pages=s["keys"].shape[0], page_stride=strides[0], head_stride=strides[1],
                           slot_stride=strides[2])
    s["batch"] = D.KvBatch(sequences=case["sequences"], query_starts=s["starts"].data_ptr(), lengths=s["lengths"].data_ptr(), page_table=s["table"].data_ptr(),
                           table_pages=s["table"].shape[1], table_stride=s["table"].shape[1])
    if case["kind"] == "append":
        s["turning"] = _turning(s)
        s["call"] = D.KvTokens(tokens=s["q"].shape[0], q_heads=case["heads"], q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), q_out=s["q_out"].data_ptr(),
                               q_strides=s["q"].stride()[:2], k_strides=s["k"].stride()[:2], v_strides=s["v"].stride()[:2], q_out_strides=s["q_out"].stride()[:2],
                               q_gamma=_pointer(s["q_gamma"]), k_gamma=_pointer(s["k_gamma"]), epsilon=EPSILON)
        return
    s["call"] = D.KvAttend(tokens=s["q"].shape[0], q_heads=case["heads"], q=s["q"].data_ptr(), out=s["out"].data_ptr(), q_strides=s["q"].stride()[:2],
                           out_strides=s["out"].stride()[:2], scale=s["scale"], softcap=case["cap"], causal=case["causal"], window=case["window"],
                           slopes=_pointer(s["slopes"]), prefix=_pointer(s["prefix"]), first_keys=_pointer(s["first"]), max_tokens=s["most"], max_keys=s["longest"])
    room = D.kv_attention_workspace(s["context"], s["cache"], s["batch"], s["call"])
    s["workspace"] = torch.empty(max(room, 16), device="cuda", dtype=torch.uint8)
    s["call"].workspace, s["call"].workspace_bytes = s["workspace"].data_ptr(), room


def _run_own(s):
    kind = s["case"]["kind"]
    if kind == "rotary":
        s["context"].rotary_raw(s["call"], s["turning"])
        return s["out"]
    if kind == "append":
        s["context"].kv_append_raw(s["cache"], s["batch"], s["call"], s["turning"])
        return {"q": s["q_out"], "keys": s["keys_whole"], "values": s["values_whole"]}
    s["context"].kv_attention_raw(s["cache"], s["batch"], s["call"])
    return s["out"]


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _turn(x, positions, frequencies, interleaved):
    """x [..., heads, size] at `positions` [...]; angles in 64 bits, the rest in 32."""
    angle = (positions.to(torch.float64)[..., None] * frequencies)[..., None, :]
    cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    half = frequencies.shape[0]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _normed(x, gamma):
    return x if gamma is None else x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPSILON) * gamma


def _places(s, tokens):
    """(sequence of each token, or the number of sequences behind the last; its place in the sequence)."""
    at = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], at, right=True)
    inside = seq.clamp(max=s["lengths"].shape[0] - 1)
    return seq, s["lengths"][inside] - s["starts"][1:][inside] + at


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "rotary":
        s["out"].copy_(_turn(_normed(s["x"], s["gamma"]), s["positions"], s["frequencies"], case["layout"] == INTERLEAVED))
        return s["out"]
    if case["kind"] == "append":
        count = s["q"].shape[0] - case["spare"]
        seq, place = (x[:count].to(torch.int64) for x in _places(s, s["q"].shape[0]))
        interleaved, page = case["layout"] == INTERLEAVED, s["table"][seq, place // case["page"]].to(torch.int64)
        slot = place % case["page"]
        s["q_out"][:count] = _turn(_normed(s["q"][:count], s["q_gamma"]), place, s["frequencies"], interleaved)
        s["keys"].transpose(1, 2)[page, slot] = _turn(_normed(s["k"][:count], s["k_gamma"]), place, s["frequencies"], interleaved).to(s["keys"].dtype)
        s["values"].transpose(1, 2)[page, slot] = s["v"][:count].to(s["values"].dtype)
        return {"q": s["q_out"], "keys": s["keys_whole"], "values": s["values_whole"]}
    return _attend_plain(s)


def _attend_plain(s):
    """Every sequence padded to the longest: [sequences, kv heads, query heads of each x tokens, keys]."""
    case = s["case"]
    sequences, kv, d, longest, most = case["sequences"], case["kv"], case["size"], s["longest"], s["most"]
    group = case["heads"] // kv
    table = s["table"].to(torch.int64)
    gathered = lambda c: c[table].to(torch.float32).permute(0, 2, 1, 3, 4).reshape(sequences, kv, -1, d)[:, :, :longest]  # noqa: E731
    k, v = gathered(s["keys"]), gathered(s["values"])
    starts, lengths = s["starts"].to(torch.int64), s["lengths"].to(torch.int64)
    t = torch.arange(most, device="cuda")
    token = (starts[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)
    place = (lengths - (starts[1:] - starts[:-1]))[:, None] + t
    key = torch.arange(longest, device="cuda")
    high = place + 1 if case["causal"] else lengths[:, None].expand(-1, most)
    if s["prefix"] is not None:
        high = torch.maximum(high, s["prefix"].to(torch.int64)[:, None])
    high = torch.minimum(high, lengths[:, None])
    low = place - case["window"] + 1 if case["window"] else torch.zeros_like(place)
    if s["first"] is not None:
        low = torch.maximum(low, s["first"].to(torch.int64)[token])
    seen = ((key >= low[..., None]) & (key < high[..., None]))[:, None, None]
    q = s["q"][token].reshape(sequences, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(sequences, kv, group * most, d)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).reshape(sequences, kv, group, most, longest) * s["scale"]
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    if s["slopes"] is not None:
        score = score - s["slopes"].reshape(1, kv, group, 1, 1) * (place[..., None] - key).abs().to(torch.float32)[:, None, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(dim=-1, keepdim=True)
    out = torch.matmul(weight.reshape(sequences, kv, group * most, longest), v).reshape(sequences, kv, group, most, d)
    out = out / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(sequences, most, case["heads"], d)
    seq, _ = _places(s, s["q"].shape[0])
    inside = seq.clamp(max=sequences - 1)
    mine = out[inside, (torch.arange(s["q"].shape[0], device="cuda") - starts[:-1][inside]).clamp(max=most - 1)]
    s["out"].copy_(torch.where((seq < sequences)[:, None, None], mine, s["out"]))
    return s["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    d = case["size"]
    if case["kind"] == "rotary":
        rows = case["batch"] * case["tokens"] * case["heads"]
        return {"bytes": 8 * rows * d + 4 * case["batch"] * case["tokens"] + 4 * case["turned"], "flops": rows * (3 * case["turned"] + (4 * d if case["norm"] else 0))}
    n, length = _lengths(case)
    tokens, held = int(n.sum()), 4 if case["type"] == "f32" else 2
    if case["kind"] == "append":
        q, kv = case["heads"], case["kv"]
        return {"bytes": tokens * d * (8 * q + 2 * kv * (4 + held)) + 8 * case["sequences"] + 4 * case["turned"],
                "flops": tokens * (q + kv) * (3 * case["turned"] + (4 * d if case["norm"] else 0))}
    pairs = keys = 0
    for low, high in _ranges(case, n, length):
        pairs += int((high - low).sum())
        some = high > low
        keys += int(high[some].max() - low[some].min()) if some.any() else 0
    return {"bytes": 8 * tokens * case["heads"] * d + 2 * keys * case["kv"] * d * held + 8 * case["sequences"], "flops": 4 * pairs * case["heads"] * d}


# ---- by definition, in 64 bits ---------------------------------------------------------------------------------------

def _rotated_exactly(x, place, frequencies, interleaved, gamma):
    """x [tokens, heads, size] at `place` [tokens], as products with e^(i place frequency)."""
    x = x.double()
    if gamma is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPSILON) * gamma.double()
    half = frequencies.shape[0]
    angle = torch.outer(place.double(), frequencies)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2].contiguous(), x[..., 1:2 * half:2].contiguous()) * turn
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        rows = [_rotated_exactly(s["x"][b], s["positions"][b], s["frequencies"], case["layout"] == INTERLEAVED, s["gamma"]) for b in range(case["batch"])]
        return torch.stack(rows)
    n, length = _lengths(case)
    begin, table = np.concatenate([[0], np.cumsum(n)]), s["table"].long()
    if case["kind"] == "append":
        q_out, keys, values = s["q_out"].double(), s["keys_whole"].double(), s["values_whole"].double()
        by_slot = (lambda c: c.transpose(1, 2)) if case["order"] == "head" else (lambda c: c)
        for i in range(case["sequences"]):
            rows = slice(int(begin[i]), int(begin[i + 1]))
            place = torch.arange(int(length[i] - n[i]), int(length[i]), device="cuda")
            page, slot = table[i][torch.div(place, case["page"], rounding_mode="floor")], place.remainder(case["page"])
            turned = lambda x, gamma: _rotated_exactly(x[rows], place, s["frequencies"], case["layout"] == INTERLEAVED, gamma)  # noqa: E731
            q_out[rows] = turned(s["q"], s["q_gamma"])
            by_slot(keys)[page, slot] = turned(s["k"], s["k_gamma"])
            by_slot(values)[page, slot] = s["v"][rows].double()
        return {"q": q_out, "keys": keys, "values": values}
    out, group = s["out"].double(), case["heads"] // case["kv"]
    for i, (low, high) in enumerate(_ranges(case, n, length)):
        key = torch.arange(int(length[i]), device="cuda")
        page, slot = table[i][torch.div(key, case["page"], rounding_mode="floor")], key.remainder(case["page"])
        place = torch.arange(int(length[i] - n[i]), int(length[i]), device="cuda")
        hidden = (key[None] < torch.tensor(low, device="cuda")[:, None]) | (key[None] >= torch.tensor(high, device="cuda")[:, None])
        rows = slice(int(begin[i]), int(begin[i + 1]))
        for h in range(case["heads"]):
            k, v = s["keys"][page, h // group, slot].double(), s["values"][page, h // group, slot].double()
            score = s["q"][rows, h].double() @ k.t().contiguous() * s["scale"]
            if case["cap"]:
                score = torch.tanh(score / case["cap"]) * case["cap"]
            if s["slopes"] is not None:
                score = score - s["slopes"][h].double() * (place[:, None] - key[None]).abs()
            score = score.masked_fill(hidden, -math.inf)
            weight = torch.exp(score - torch.logsumexp(score, dim=-1, keepdim=True)).masked_fill(hidden, 0.0)
            out[rows, h] = weight @ v
    return out
