"""What a decoder does with its paged cache beyond a plain step, as cases that can be timed: attention of a tree of drafted
tokens, attention over the pages that a cheap score selects, attention that adds up what each key was given, the choice of the
keys that stay when a cache is full, and the moves that follow from either.

    listed()           the cases
    draw(rng)          one more case of the same ranges
    prepare(case, s)   inputs made from the seed `s`, and the descriptions of cache and batch that a program keeps
    run(state)         one pass: in elementary torch operations, or (own) by this package's operators; the outputs whole
    work(case)         bytes (inputs and outputs once) and operations of one pass
    exact(case, s)     the outputs by the operators' definitions, in 64 bits

Definitions.  A sequence with n tokens in the call and a length L after them has its token t in slot L - n + t, slot j being
slot j % page_size of the sequence's page j / page_size.  Scores are q k scale, then cap tanh(score / cap).

tree   Token t follows token parents[t] < t of the call, or (-1) the last slot in front of them; its depth is the number of those
       before it in the call.  It sees the slots in front of the call and, of the call's, its own and those of the tokens it follows,
       all of them less than `window` positions away where there is a window; less slope x distance, where slots in front of the
       call are at their place and the call's at L - n + depth.
mass   Causal attention.  Then, for each kv head, the mass of slot j becomes decay x mass (0 for the call's own slots) plus the
       sum of its weights over all tokens of the call and query heads of the group; positions of the call's own slots are noted.
evict  For each kv head of a sequence longer than `budget`, `budget` slots stay: those at positions below `first` or of the
       `recent` newest, then those of the largest mass, the lowest slot where masses are equal.  The i-th slot from `budget` on
       that stays is to go to the i-th slot below that does not.
move   Keys, values, masses and positions of slots `sources` go to slots `targets`, a list for each sequence, or for each of its kv heads.
sparse A token at place p sees the slots up to p in `most` pages (all where there are no more): the first `first`, the `last`
       newest up to its own, then those with the largest score, the lowest where they are equal.  A page's score is the largest
       q . mean over the query heads of the group, mean being the mean of the page's keys (held in 32 bits) once it is full.
"""
import functools
import math

import numpy as np
import torch

own = False


# ---- the cases -------------------------------------------------------------------------------------------------------

def _tree(name, sequences, least, most, before_least, before, heads, kv, size, type_, page, order, cap=0.0, window=0, slopes=False, spare=0):
    return {"name": name, "kind": "tree", "sequences": sequences, "least": least, "most": most, "before_least": before_least, "before": before,
            "heads": heads, "kv": kv, "size": size, "type": type_, "page": page, "order": order, "cap": cap, "window": window, "slopes": slopes, "spare": spare}


def _mass(name, sequences, least, most, before_least, before, heads, kv, size, type_, page, order, decay=1.0, cap=0.0, spare=0):
    return {"name": name, "kind": "mass", "sequences": sequences, "least": least, "most": most, "before_least": before_least, "before": before,
            "heads": heads, "kv": kv, "size": size, "type": type_, "page": page, "order": order, "decay": decay, "cap": cap, "spare": spare}


def _sparse(name, sequences, least, most, before_least, before, heads, kv, size, type_, page, order, pages, first=1, last=2, cap=0.0, spare=0):
    return {"name": name, "kind": "sparse", "sequences": sequences, "least": least, "most": most, "before_least": before_least, "before": before,
            "heads": heads, "kv": kv, "size": size, "type": type_, "page": page, "order": order, "pages": pages, "first": first, "last": last, "cap": cap, "spare": spare}


def _evict(name, sequences, longest, shortest, budget, recent, first, kv, page):
    return {"name": name, "kind": "evict", "sequences": sequences, "longest": longest, "shortest": shortest, "budget": budget, "recent": recent, "first": first,
            "kv": kv, "page": page}


def _move(name, sequences, moves_least, moves, slots, kv, size, type_, page, order, by_head):
    return {"name": name, "kind": "move", "sequences": sequences, "moves_least": moves_least, "moves": moves, "slots": slots, "kv": kv, "size": size, "type": type_,
            "page": page, "order": order, "by_head": by_head}


def listed():
    return [
        # Eight tokens drafted for one short text of a small decoder: the smallest attention here, all latency.
        _tree("tree_small", 1, 8, 8, 500, 500, 12, 12, 64, "f32", 16, "head"),
        # Trees of 16 to 48 drafted tokens for each of 16 texts of all lengths, cache in bf16, eight heads of keys.
        _tree("tree_batch_bf16", 16, 16, 48, 300, 8000, 32, 8, 128, "bf16", 16, "slot", spare=5),
        # A large tree behind two long documents, a bias by distance, pages that end inside a tile.
        _tree("tree_long_bias", 2, 40, 61, 20011, 30000, 16, 4, 96, "f32", 24, "head", slopes=True),
        # One new token of each of 24 texts whose cache is to be thinned out later.
        _mass("mass_tokens", 24, 1, 1, 1000, 4095, 32, 8, 128, "f32", 16, "head"),
        # Two prompts of up to 2048 tokens, cache in bf16, older masses fading.
        _mass("mass_prompts_bf16", 2, 1500, 2048, 0, 300, 16, 4, 128, "bf16", 64, "slot", decay=0.9, spare=3),
        # Every text one token over its budget: what a server asks after each step.
        _evict("evict_step", 48, 1025, 1025, 1024, 256, 4, 8, 16),
        # Four long documents that are to be thinned out at once.
        _evict("evict_long", 4, 50000, 20011, 4096, 512, 16, 8, 64),
        # The accepted branch of each of 64 trees goes to the front, the same for all heads: all latency.
        _move("move_accepted", 64, 0, 7, 24, 8, 128, "f32", 16, "head", False),
        # What stays of eight caches goes where others went, for each head its own, cache in bf16.
        _move("move_survivors_bf16", 8, 1100, 2000, 4096, 8, 128, "bf16", 16, "slot", True),
        # One new token behind a long document, 32 pages of 64 of the thousand that there are.
        _sparse("sparse_token_long", 1, 1, 1, 65535, 65535, 32, 8, 128, "f32", 64, "head", 32),
        # One new token of each of 48 texts of all lengths, cache in bf16, capped scores.
        _sparse("sparse_tokens_bf16", 48, 1, 1, 100, 16000, 32, 4, 128, "bf16", 32, "slot", 40, cap=50.0),
        # A piece of a prompt behind what earlier pieces left, small pages, heads of 80 channels.
        _sparse("sparse_piece", 2, 100, 207, 6001, 12000, 16, 4, 80, "f32", 16, "head", 61, first=2, last=4, spare=2),
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["tree", "mass", "evict", "move", "sparse"])
    most = [_cost(c) for c in listed() if c["kind"] == kind]
    most = [max(c[i] for c in most) for i in range(3)]
    while True:
        case = _drawn(rng, kind)
        if all(mine <= m for mine, m in zip(_cost(case), most)):
            return case


def _cost(case):
    """Bytes, operations, and how much the plain form holds: all sequences as long as the longest."""
    w, held, kind = work(case), 0, case["kind"]
    if "heads" in case:
        n, length = _lengths(case)
        keys = int(length.max())
        if kind == "sparse":  # the chosen keys and values of each token
            keys = min(keys, case["pages"] * case["page"]) * case["size"] * case["kv"] // case["heads"]
        held = case["sequences"] * case["heads"] * int(n.max()) * keys
    return w["bytes"], w["flops"], held


def _drawn(rng, kind):
    order, type_ = rng.choice(["head", "slot"]), rng.choice(["f32", "bf16"])
    size = rng.choice([64, 64, 80, 96, 128, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    page = rng.choice([8, 16, 16, 24, 64, 128, 250])
    if kind == "tree":
        most, before = _log(rng, 2, 64), _log(rng, 1, 30000)
        case = _tree("", _log(rng, 1, 32), max(1, most // rng.choice([1, 1, 3])), most, max(0, before // rng.choice([1, 4, 50])), before, heads, kv, size, type_, page, order,
                     cap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, 0, 5, 700]), slopes=rng.random() < 0.3, spare=rng.choice([0, 0, 9]))
    elif kind == "mass":
        if rng.random() < 0.5:
            before, most = _log(rng, 8, 16000), rng.choice([1, 1, 1, 3])
            case = _mass("", _log(rng, 1, 48), 1, most, max(1, before // rng.choice([1, 4, 50])), before, heads, kv, size, type_, page, order,
                         decay=rng.choice([1.0, 1.0, 0.5, 0.0]), cap=rng.choice([0.0, 0.0, 50.0]))
        else:
            most, before = _log(rng, 17, 2000), rng.choice([0, 0, _log(rng, 1, 2000)])
            case = _mass("", _log(rng, 1, 4), max(1, most // rng.choice([1, 1, 3])), most, before // 2, before, heads, kv, size, type_, page, order,
                         decay=rng.choice([1.0, 1.0, 0.9, 0.0]), cap=rng.choice([0.0, 0.0, 50.0]), spare=rng.choice([0, 0, 9]))
    elif kind == "evict":
        budget = _log(rng, 16, 4096)
        longest = _log(rng, budget + 1, 50000)
        case = _evict("", _log(rng, 1, 64), longest, max(1, longest // rng.choice([1, 1, 2, 5])), budget, budget // rng.choice([2, 4, 9]), rng.choice([0, 1, 4]), kv, page)
    elif kind == "move":
        slots = _log(rng, 8, 8192)
        moves = max(1, slots // rng.choice([2, 2, 5]))
        case = _move("", _log(rng, 1, 64), moves // rng.choice([1, 2, 9]), moves, slots, kv, size, type_, page, order, rng.random() < 0.6)
    else:
        page = rng.choice([16, 16, 24, 32, 64, 128])
        before, most = _log(rng, 8, 65535), rng.choice([1, 1, 1, 3, _log(rng, 4, 200)])
        first, last = rng.choice([0, 1, 2]), rng.choice([1, 2, 4])
        case = _sparse("", _log(rng, 1, 48), max(1, most // rng.choice([1, 2])), most, max(1, before // rng.choice([1, 4, 50])), before, heads, kv, size, type_, page, order,
                       first + last + _log(rng, 1, 80), first=first, last=last, cap=rng.choice([0.0, 0.0, 50.0]), spare=rng.choice([0, 0, 9]))
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
    if case["kind"] == "evict":
        length = _spread(case["shortest"], case["longest"], case["sequences"])
        return np.zeros_like(length), length
    if case["kind"] == "move":
        length = np.full(case["sequences"], case["slots"], np.int64)
        return np.zeros_like(length), length
    n = _spread(case["least"], case["most"], case["sequences"])
    return n, n + _spread(case["before_least"], case["before"], case["sequences"])[::-1]


def _moves(case):
    """How many slots each sequence (or head of one) moves."""
    return _spread(case["moves_least"], case["moves"], case["sequences"] * (case["kv"] if case["by_head"] else 1))


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_HELD = {"f32": 4, "bf16": 2}


# ---- what a program has in hand --------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=1)
def _context():
    from altius_amd import device
    return device.Context(0, stream=torch.cuda.current_stream().cuda_stream)


def _slots(s, length):
    """Page and slot of each of a sequence's places, for all sequences: [sequences, longest]."""
    place = torch.arange(length, device="cuda")
    return s["table"].long()[:, place // s["case"]["page"]], (place % s["case"]["page"])[None].expand(s["table"].shape[0], -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32)  # noqa: E731
    whole = lambda values: torch.tensor(np.asarray(values), device="cuda", dtype=torch.int32)  # noqa: E731
    s = {"case": dict(case)}
    n, length = _lengths(case)
    kind, kv, page, sequences = case["kind"], case["kv"], case["page"], case["sequences"]
    s["starts"], s["lengths"] = whole(np.concatenate([[0], np.cumsum(n)])), whole(length)
    s["most"], s["longest"] = int(n.max()), int(length.max())
    per = -(-s["longest"] // page)
    pages = sequences * per + 3
    s["table"] = torch.randperm(pages, generator=gen, device="cuda")[:sequences * per].to(torch.int32).reshape(sequences, per)
    if kind != "evict":
        d = case["size"]
        shape = (pages, kv, page, d) if case["order"] == "head" else (pages, page, kv, d)
        for name in ("keys", "values"):
            cache = normal(*shape)
            if kind == "sparse" and name == "keys":  # what stands together is alike
                cache += 0.7 * (normal(pages, kv, 1, d) if case["order"] == "head" else normal(pages, 1, kv, d))
            cache = cache.to(_TORCH[case["type"]])
            s[name + "_whole"] = cache
            s[name] = cache if case["order"] == "head" else cache.transpose(1, 2)  # [pages, kv, page, d] either way
    if kind in ("tree", "mass", "sparse"):
        tokens = int(n.sum()) + case["spare"]
        s["q"] = 1.5 * normal(tokens, case["heads"], d)
        s["out"] = torch.zeros((tokens, case["heads"], d), device="cuda")
        s["scale"] = 1.0 / math.sqrt(d)
    if kind == "tree":
        # Token t follows one of the few before it, now and then the text itself.
        t = torch.cat([torch.arange(int(m), device="cuda") for m in n] + [torch.zeros(case["spare"], device="cuda", dtype=torch.int64)])
        back = 1 + (uniform(tokens).square() * 6).long()
        s["parents"] = torch.where(back > t, torch.full_like(t, -1), t - back).to(torch.int32)
        s["slopes"] = torch.tensor(2.0 ** (-8.0 * np.arange(1, case["heads"] + 1) / case["heads"]), device="cuda", dtype=torch.float32) if case["slopes"] else None
    if kind == "sparse":
        s["chosen"] = torch.full((tokens, kv, case["pages"]), -7, device="cuda", dtype=torch.int32)
        s["means"] = s["keys"].double().mean(dim=2).float()  # [pages, kv, d]: those of the call's own pages are made by the call
        begin = [int(length[i] - n[i]) // page for i in range(sequences)]
        for i in range(sequences):
            s["means"][s["table"][i, begin[i]:].long()] = 0.0
    if kind in ("mass", "evict", "move"):
        # A few slots hold most of the mass, some none of it; a slot's position is its place but for the first half, which has been mixed.
        s["mass"] = torch.exp(2.5 * normal(pages, kv, page)) * (uniform(pages, kv, page) > 0.1)
        position = torch.zeros((pages, kv, page), device="cuda", dtype=torch.int32)
        at, slot = _slots(s, s["longest"])
        half = s["longest"] // 2
        mixed = torch.arange(s["longest"], device="cuda", dtype=torch.int32)[None, None].repeat(sequences, kv, 1) * 2
        if half > 1:
            order = torch.argsort(uniform(sequences, kv, half), dim=-1)
            mixed[:, :, :half] = mixed[:, :, :half].gather(-1, order)
        position[at, :, slot] = mixed.transpose(1, 2)
        s["positions"] = position
    if kind == "mass":
        s["row_positions"] = whole(2 * np.concatenate([np.arange(l - m, l) for m, l in zip(n, length)] + [np.zeros(case["spare"], np.int64)]))
    if kind == "evict":
        s["room"] = max(1, min(case["budget"], s["longest"] - case["budget"]))
        for name in ("sources", "targets"):
            s[name] = torch.full((sequences, kv, s["room"]), -7, device="cuda", dtype=torch.int32)
        s["counts"], s["kept"] = torch.zeros((sequences, kv), device="cuda", dtype=torch.int32), torch.zeros(sequences, device="cuda", dtype=torch.int32)
    if kind == "move":
        counts = _moves(case)
        lists = (sequences, kv if case["by_head"] else 1)
        s["room"] = int(counts.max())
        s["counts"] = whole(counts.reshape(lists))
        low = case["slots"] // 2  # sources from there on, targets below: each in order, no slot twice
        pick = lambda m: torch.sort(torch.argsort(uniform(*lists, m), dim=-1)[..., :max(1, s["room"])], dim=-1).values  # noqa: E731
        s["targets"], s["sources"] = pick(low).to(torch.int32), (low + pick(case["slots"] - low)).to(torch.int32)
    if own:
        _calls(s)
    return s


# ---- the package's operators -----------------------------------------------------------------------------------------

def _pointer(x):
    return None if x is None else x.data_ptr()


def _calls(s):
    from altius_amd import device as D
    case, kind = s["case"], s["case"]["kind"]
    ctx = s["context"] = _context()
    pages, kv, page = s["table"].numel() + 3, case["kv"], case["page"]
    held = {}
    if kind != "evict":
        strides = s["keys"].stride()
        held = dict(keys=s["keys"].data_ptr(), values=s["values"].data_ptr(), elem=D.KV_BF16 if case["type"] == "bf16" else D.KV_F32, head_size=case["size"],
                    page_stride=strides[0], head_stride=strides[1], slot_stride=strides[2])
    cache = s["cache"] = D.KvCache(**{**dict(kv_heads=kv, page_size=page, pages=pages, head_size=1), **held})
    batch = s["batch"] = D.KvBatch(sequences=case["sequences"], query_starts=s["starts"].data_ptr(), lengths=s["lengths"].data_ptr(), page_table=s["table"].data_ptr(),
                                   table_pages=s["table"].shape[1], table_stride=s["table"].shape[1])
    if "mass" in s:
        s["history"] = D.KvHistory(mass=s["mass"].data_ptr(), positions=s["positions"].data_ptr(), page_stride=kv * page, head_stride=page)
    if kind == "evict":
        s["call"] = D.KvEviction(budget=case["budget"], recent=case["recent"], first=case["first"], most=s["room"], max_keys=s["longest"], sources=s["sources"].data_ptr(),
                                 targets=s["targets"].data_ptr(), counts=s["counts"].data_ptr(), lengths=s["kept"].data_ptr())
        return
    if kind == "move":
        by_head = case["by_head"]
        lists = s["sources"].shape
        s["call"] = D.KvMoves(sources=s["sources"].data_ptr(), targets=s["targets"].data_ptr(), counts=s["counts"].data_ptr(), most=s["room"], apart=1,
                              strides=(lists[1] * lists[2], lists[2] if by_head else 0), count_strides=(lists[1], 1 if by_head else 0))
        return
    call = s["call"] = D.KvAttend(tokens=s["q"].shape[0], q_heads=case["heads"], q=s["q"].data_ptr(), out=s["out"].data_ptr(), q_strides=s["q"].stride()[:2],
                                  out_strides=s["out"].stride()[:2], scale=s["scale"], softcap=case["cap"], causal=1, window=case.get("window", 0),
                                  slopes=_pointer(s.get("slopes")), max_tokens=s["most"], max_keys=s["longest"])
    if kind == "tree":
        room = D.kv_attention_workspace(ctx, cache, batch, call)
    elif kind == "mass":
        room = D.kv_attention_mass_workspace(ctx, cache, batch, call)
    else:
        s["sparse"] = D.KvSparse(means=s["means"].data_ptr(), chosen=s["chosen"].data_ptr(), most=case["pages"], first=case["first"], last=case["last"],
                                 page_stride=kv * case["size"], head_stride=case["size"])
        room = D.kv_attention_sparse_workspace(ctx, cache, batch, call, s["sparse"])
    s["workspace"] = torch.empty(max(room, 16), device="cuda", dtype=torch.uint8)
    call.workspace, call.workspace_bytes = s["workspace"].data_ptr(), room


def _run_own(s):
    kind, ctx = s["case"]["kind"], s["context"]
    if kind == "tree":
        ctx.kv_attention_tree_raw(s["cache"], s["batch"], s["call"], s["parents"].data_ptr())
    elif kind == "mass":
        ctx.kv_attention_mass_raw(s["cache"], s["batch"], s["call"], s["history"], s["case"]["decay"], s["row_positions"].data_ptr())
    elif kind == "sparse":
        ctx.kv_attention_sparse_raw(s["cache"], s["batch"], s["call"], s["sparse"])
    elif kind == "evict":
        ctx.kv_evict_raw(s["cache"], s["batch"], s["history"], s["call"])
    else:
        ctx.kv_move_raw(s["cache"], s["batch"], s["call"], s["history"])
    return _outputs(s)


def _outputs(s):
    names = {"tree": ("out",), "mass": ("out", "mass", "positions"), "sparse": ("out", "chosen", "means"), "evict": ("sources", "targets", "counts", "kept"),
             "move": ("keys_whole", "values_whole", "mass", "positions")}[s["case"]["kind"]]
    return {name: s[name] for name in names}


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _rows(s):
    """Each sequence's tokens padded to the most: (row in the tensors, place, whether it is there), [sequences, most]."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    t = torch.arange(s["most"], device="cuda")
    there = t < (starts[1:] - starts[:-1])[:, None]
    return (starts[:-1, None] + t).clamp(max=s["q"].shape[0] - 1), (lengths - (starts[1:] - starts[:-1]))[:, None] + t, there


def _gathered(s, cache):
    """[sequences, kv, longest, size] in 32 bits."""
    table = s["table"].long()
    return cache[table].float().permute(0, 2, 1, 3, 4).reshape(table.shape[0], cache.shape[1], -1, cache.shape[3])[:, :, :s["longest"]]


def _weights(s, score, seen, bias=None):
    """Softmax of capped scores over what is seen of the last axis, zero where that is nothing."""
    if s["case"]["cap"]:
        score = s["case"]["cap"] * torch.tanh(score / s["case"]["cap"])
    if bias is not None:
        score = score - bias
    score = torch.where(seen, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(dim=-1, keepdim=True)
    return weight / torch.where(total == 0, 1.0, total)


def _attend_plain(s, seen, bias=None):
    """Every sequence padded to the longest.  seen [sequences, most, longest]; returns the weights [sequences, kv, group, most, longest]."""
    case = s["case"]
    sequences, kv, d, most, group = case["sequences"], case["kv"], case["size"], s["most"], case["heads"] // case["kv"]
    token, _, there = _rows(s)
    k, v = _gathered(s, s["keys"]), _gathered(s, s["values"])
    q = s["q"][token].reshape(sequences, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(sequences, kv, group * most, d)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).reshape(sequences, kv, group, most, -1) * s["scale"]
    if bias is not None:
        bias = s["slopes"].reshape(1, kv, group, 1, 1) * bias[:, None, None].float()
    weight = _weights(s, score, seen[:, None, None], bias)
    out = torch.matmul(weight.reshape(sequences, kv, group * most, -1), v).reshape(sequences, kv, group, most, d)
    s["out"][token[there]] = out.permute(0, 3, 1, 2, 4).reshape(sequences, most, case["heads"], d)[there]
    return weight


def _tree_plain(s):
    token, place, there = _rows(s)
    most, base = s["most"], place[:, :1]
    parent = torch.where(there, s["parents"].long()[token], -1)
    t = torch.arange(most, device="cuda")
    above = ((parent[..., None] == t) | (t[:, None] == t)).float()  # itself and the one it follows
    for _ in range(max(1, (most - 1).bit_length())):  # then those that these follow, twice as far each time
        above = (torch.matmul(above, above) > 0).float()
    depth = above.sum(-1).long() - 1
    key = torch.arange(s["longest"], device="cuda")
    u = (key - base)  # [sequences, longest]
    drafted = (u >= 0) & (u < most)
    at = u.clamp(0, most - 1)
    key_position = torch.where(drafted, base + depth.gather(1, at), key)
    distance = (base + depth)[..., None] - key_position[:, None]
    mine = above.gather(2, at[:, None].expand(-1, most, -1)) > 0
    seen = torch.where(drafted[:, None], mine, (key < base)[:, None]) & there[..., None]
    if s["case"]["window"]:
        seen = seen & (distance < s["case"]["window"])
    _attend_plain(s, seen, distance.abs() if s["slopes"] is not None else None)


def _mass_plain(s):
    token, place, there = _rows(s)
    key = torch.arange(s["longest"], device="cuda")
    weight = _attend_plain(s, (key <= place[..., None]) & there[..., None])
    given = weight.sum(dim=(2, 3))  # [sequences, kv, longest]
    lengths, first = s["lengths"].long()[:, None], place[:, :1]
    page, slot = _slots(s, s["longest"])
    inside, fresh = key < lengths, key >= first
    before = s["mass"][page, :, slot].transpose(1, 2)
    after = torch.where(fresh[:, None], 0.0, s["case"]["decay"] * before if s["case"]["decay"] else 0.0) + given
    s["mass"][page[inside], :, slot[inside]] = after.transpose(1, 2)[inside]
    new = inside & fresh
    row = (s["starts"].long()[:-1, None] + key - first)[new]
    s["positions"][page[new], :, slot[new]] = s["row_positions"][row][:, None]


def _sparse_plain(s):
    case = s["case"]
    page, kv, d, group, most = case["page"], case["kv"], case["size"], case["heads"] // case["kv"], case["pages"]
    token, place, there = _rows(s)
    table = s["table"].long()
    number = torch.arange(table.shape[1], device="cuda")
    # Means of the pages that the call's tokens have filled.
    full = (number + 1) * page
    filled = (full <= s["lengths"].long()[:, None]) & (full > place[:, :1])
    s["means"][table[filled]] = s["keys"][table[filled]].double().mean(dim=2).float()
    row, at = token[there], place[there]
    seq = torch.arange(case["sequences"], device="cuda")[:, None].expand_as(token)[there]
    q = s["q"][row].reshape(-1, kv, group, d)
    mine = at // page
    score = torch.matmul(s["means"][table].double().permute(0, 2, 1, 3)[seq], q.double().transpose(-1, -2).contiguous()).amax(dim=-1)  # [rows, kv, pages]
    there_yet = number <= mine[:, None]
    always = there_yet & ((number < case["first"]) | (number > mine[:, None] - case["last"]))
    score = torch.where(always[:, None], math.inf, torch.where(there_yet[:, None], score, -math.inf))
    count = min(most, number.shape[0])
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :count]
    kept = torch.arange(count, device="cuda") < (mine + 1)[:, None]
    best = torch.sort(torch.where(kept[:, None], best, table.shape[1]), dim=-1).values
    s["chosen"][row] = -1
    s["chosen"][row, :, :count] = torch.where(kept[:, None], best, -1).to(torch.int32)
    physical = table[seq[:, None, None], best.clamp(max=table.shape[1] - 1)]  # [rows, kv, count]
    heads = torch.arange(kv, device="cuda")[None, :, None]
    k, v = (s[name][physical, heads].float().reshape(-1, kv, count * page, d) for name in ("keys", "values"))
    key = (best[..., None] * page + torch.arange(page, device="cuda")).reshape(-1, kv, 1, count * page)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    weight = _weights(s, score, (key <= at[:, None, None, None]) & (best < table.shape[1])[..., None].expand(-1, -1, -1, page).reshape(key.shape))
    s["out"][row] = torch.matmul(weight, v).reshape(-1, case["heads"], d)


def _evict_plain(s):
    case = s["case"]
    budget = case["budget"]
    page, slot = _slots(s, s["longest"])
    place = torch.arange(s["longest"], device="cuda")
    inside = (place < s["lengths"].long()[:, None])[:, None]
    mass, position = s["mass"][page, :, slot].transpose(1, 2), s["positions"][page, :, slot].transpose(1, 2)
    newest = torch.where(inside, position, -1).amax(dim=-1, keepdim=True)
    kept_anyway = (position < case["first"]) | (position > newest - case["recent"])
    value = torch.where(inside, torch.where(kept_anyway, math.inf, mass), -math.inf)
    rank = torch.sort(value, dim=-1, descending=True, stable=True).indices
    stays = torch.zeros_like(inside.expand_as(value)).scatter(-1, rank[..., :budget], True) & inside
    long = (s["lengths"] > budget)[:, None, None]
    hole, mover = ~stays & (place < budget) & inside & long, stays & (place >= budget) & long
    for name, which in (("targets", hole), ("sources", mover)):
        number = which.cumsum(-1) - 1
        seq, head, at = which.nonzero(as_tuple=True)
        s[name][seq, head, number[seq, head, at]] = at.to(torch.int32)
    s["counts"].copy_(mover.sum(-1))
    s["kept"].copy_(s["lengths"].clamp(max=budget))


def _move_plain(s):
    case = s["case"]
    lists = s["sources"].expand(-1, case["kv"], -1).long(), s["targets"].expand(-1, case["kv"], -1).long()
    seq, head, i = (torch.arange(lists[0].shape[-1], device="cuda") < s["counts"][..., None]).expand(-1, case["kv"], -1).nonzero(as_tuple=True)
    (source, source_slot), (target, target_slot) = ((s["table"].long()[seq, x[seq, head, i] // case["page"]], x[seq, head, i] % case["page"]) for x in lists)
    for name in ("keys", "values", "mass", "positions"):
        s[name][target, head, target_slot] = s[name][source, head, source_slot]


def run(state):
    if own:
        return _run_own(state)
    {"tree": _tree_plain, "mass": _mass_plain, "sparse": _sparse_plain, "evict": _evict_plain, "move": _move_plain}[state["case"]["kind"]](state)
    return _outputs(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind, kv = case["kind"], case["kv"]
    n, length = _lengths(case)
    if kind == "evict":
        long = length[length > case["budget"]]
        # Masses and positions; as many moves as slots from the budget on would stay if it went by chance.
        moves = (np.minimum(long, case["budget"]) * (long - case["budget"]) / np.maximum(long, 1)).sum()
        return {"bytes": float(kv * (8 * long.sum() + 8 * moves) + 4 * kv * len(length) + 8 * len(length)), "flops": float(kv * long.sum())}
    d, held = case["size"], _HELD[case["type"]]
    if kind == "move":
        count = int(_moves(case).sum())
        moved = count * (1 if case["by_head"] else kv)
        return {"bytes": moved * (4 * d * held + 16) + 8 * count, "flops": 0}
    tokens, keys, pairs = int(n.sum()), int(length.sum()), 0
    rows = 8 * tokens * case["heads"] * d
    if kind == "sparse":
        page, most, seen, read = case["page"], case["pages"], 0, 0
        for m, l in zip(n, length):
            place = np.arange(l - m, l)
            mine = np.minimum(place // page, most - 1) * page + place % page + 1
            seen += int(mine.sum())
            read += min(int(mine.sum()), int(l))
        scored = int((np.maximum(0, length // page)).sum())
        return {"bytes": rows + 2 * read * kv * d * held + 4 * scored * kv * d + 4 * tokens * kv * most, "flops": 4 * seen * case["heads"] * d}
    for m, l in zip(n, length):
        pairs += int(np.arange(l - m + 1, l + 1).sum()) if kind == "mass" else int(m * (l - m + 3))
    more = 8 * keys * kv if kind == "mass" else 4 * tokens
    return {"bytes": rows + 2 * keys * kv * d * held + more, "flops": (6 if kind == "mass" and case["most"] > 1 else 4) * pairs * case["heads"] * d}


# ---- by definition, in 64 bits ---------------------------------------------------------------------------------------

def _exact_rows(s, i, h, q, key, seen, bias=None):
    """Weights [rows, keys] and results of query head h over the places `key` of sequence i."""
    case = s["case"]
    page, slot, g = s["table"][i].long()[key // case["page"]], key % case["page"], h // (case["heads"] // case["kv"])
    k, v = s["keys"][page, g, slot].double(), s["values"][page, g, slot].double()
    score = q.double() @ k.t().contiguous() * s["scale"]
    if case["cap"]:
        score = torch.tanh(score / case["cap"]) * case["cap"]
    if bias is not None:
        score = score - s["slopes"][h].double() * bias
    score = score.masked_fill(~seen, -math.inf)
    weight = torch.exp(score - torch.logsumexp(score, dim=-1, keepdim=True)).masked_fill(~seen, 0.0)
    return weight, weight @ v


def _exact_tree(s, i, start, m, l):
    case, base = s["case"], l - m
    parent = s["parents"][start:start + m].cpu().numpy()
    depth, seen = np.zeros(m, np.int64), np.zeros((m, l), bool)
    for t in range(m):
        depth[t] = 0 if parent[t] < 0 else depth[parent[t]] + 1
    position = np.concatenate([np.arange(base), base + depth])
    for t in range(m):
        seen[t, :base] = True
        u = t
        while u >= 0:
            seen[t, base + u] = True
            u = parent[u]
    distance = (base + depth)[:, None] - position[None]
    if case["window"]:
        seen &= distance < case["window"]
    return torch.tensor(seen, device="cuda"), torch.tensor(np.abs(distance), device="cuda") if case["slopes"] else None


def exact(case, seed):
    s = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    n, length = _lengths(case)
    if kind == "evict":
        lists = [torch.full_like(s["sources"], -7).cpu() for _ in range(2)]
        counts = np.zeros((case["sequences"], case["kv"]), np.int64)
        for i, l in enumerate(length):
            at = np.arange(l)
            pages, slot = s["table"][i].cpu().numpy()[at // page], at % page
            for g in range(case["kv"] if l > case["budget"] else 0):
                mass, position = (s[x][:, g].cpu().numpy()[pages, slot].astype(np.float64) for x in ("mass", "positions"))
                safe = (position < case["first"]) | (position > position.max() - case["recent"])
                order = np.lexsort((at, -mass, ~safe))
                stays = np.zeros(l, bool)
                stays[order[:case["budget"]]] = True
                move, hole = np.flatnonzero(stays[case["budget"]:]) + case["budget"], np.flatnonzero(~stays[:case["budget"]])
                counts[i, g] = len(move)
                for which, places in zip(lists, (move, hole)):
                    which[i, g, :len(places)] = torch.tensor(places, dtype=torch.int32)
        return {"sources": lists[0], "targets": lists[1], "counts": torch.tensor(counts, dtype=torch.int32), "kept": torch.tensor(np.minimum(length, case["budget"]), dtype=torch.int32)}
    if kind == "move":
        held = {name: s[name].clone() for name in ("keys", "values", "mass", "positions")}
        for i in range(case["sequences"]):
            for g in range(case["kv"]):
                j = g if case["by_head"] else 0
                count = int(s["counts"][i, j])
                a, b = s["sources"][i, j, :count].long(), s["targets"][i, j, :count].long()
                table = s["table"][i].long()
                for name in held:
                    held[name][table[b // page], g, b % page] = s[name][table[a // page], g, a % page]
        by_order = lambda x: x if case["order"] == "head" else x.transpose(1, 2)  # noqa: E731
        return {"keys_whole": by_order(held["keys"]).double(), "values_whole": by_order(held["values"]).double(), "mass": held["mass"].double(), "positions": held["positions"]}
    out, begin, heads, group = s["out"].double(), np.concatenate([[0], np.cumsum(n)]), case["heads"], case["heads"] // case["kv"]
    mass, positions = (s["mass"].double(), s["positions"].clone()) if kind == "mass" else (None, None)
    chosen, means = (s["chosen"].clone(), s["means"].double()) if kind == "sparse" else (None, None)
    for i in range(case["sequences"]):
        m, l, start = int(n[i]), int(length[i]), int(begin[i])
        rows, key, place = slice(start, start + m), torch.arange(l, device="cuda"), torch.arange(l - m, l, device="cuda")
        bias = None
        if kind == "tree":
            seen, bias = _exact_tree(s, i, start, m, l)
        elif kind == "mass":
            seen, given = key[None] <= place[:, None], torch.zeros((case["kv"], l), device="cuda", dtype=torch.float64)
        else:
            table = s["table"][i].long()
            for b in range((l - m) // page, l // page):
                means[table[b]] = (s["keys"][table[b]].double().sum(dim=1) / page).float().double()
            pages = -(-l // page)
            for r in range(m):
                p = l - m + r
                mine = p // page
                for g in range(case["kv"]):
                    score = (means[table[:mine + 1], g] @ s["q"][start + r, g * group:(g + 1) * group].double().t().contiguous()).amax(dim=1)
                    score[:case["first"]] = math.inf
                    score[max(0, mine + 1 - case["last"]):] = math.inf
                    best = torch.sort(torch.argsort(-score, stable=True)[:case["pages"]]).values
                    chosen[start + r, g] = -1
                    chosen[start + r, g, :len(best)] = best.to(torch.int32)
            seen = None
        for h in range(heads):
            if kind == "sparse":
                mine = chosen[rows, h // group].long()
                seen = torch.zeros((m, pages + 1), device="cuda", dtype=torch.bool).scatter(1, torch.where(mine < 0, pages, mine), True)
                seen = seen[:, :pages].repeat_interleave(page, dim=1)[:, :l] & (key[None] <= place[:, None])
            weight, out[rows, h] = _exact_rows(s, i, h, s["q"][rows, h], key, seen, bias)
            if kind == "mass":
                given[h // group] += weight.sum(dim=0)
        if kind == "mass":
            at, slot = s["table"][i].long()[key // page], key % page
            before = torch.where(key < l - m, mass[at, :, slot].t() * case["decay"], 0.0)
            mass[at, :, slot] = (before + given).t()
            positions[at[l - m:], :, slot[l - m:]] = s["row_positions"][rows][:, None].expand(-1, case["kv"])
    if kind == "mass":
        return {"out": out, "mass": mass, "positions": positions}
    return {"out": out, "chosen": chosen, "means": means} if kind == "sparse" else {"out": out}
