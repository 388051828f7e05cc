"""Keys and values appended to a paged cache (ahip_kv_append) and attention over it (ahip_kv_attention) against their
definitions in float64: ragged batches, pages of any size, masks that leave rows empty, whatever lies in slots not seen."""
import math

import numpy as np
import pytest
import torch

from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_UNSUPPORTED, AltiusHipError
from decoder_oracle import attended, bf16, normed, ranges, turned, turned_bound
from decoder_precision import WINDOWS, expected, keys, queries, values

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture
def here():
    with D.Context(0, stream=torch.cuda.current_stream().cuda_stream) as c:
        yield c


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Paged:
    """A cache on the GPU with pages in random order, and the sequences of one call.  order: how [pages, heads, slots, d] lies."""

    def __init__(self, rng, n, lengths, kv_heads, d, page, elem="f32", order="head", spare_pages=2, table_pages=None, fill=None):
        self.n, self.lengths, self.kv_heads, self.d, self.page, self.elem = list(n), list(lengths), kv_heads, d, page, elem
        self.per = table_pages or max(1, max(-(-max(l, 1) // page) for l in lengths))
        used = self.per * len(n)
        self.pages = used + spare_pages
        self.table = rng.permutation(self.pages)[:used].reshape(len(n), self.per).astype(np.int32)
        shape = (self.pages, kv_heads, page, d) if order == "head" else (self.pages, page, kv_heads, d)
        self.order = order
        self.on = []
        for _ in range(2):
            x = rng.standard_normal(shape).astype(np.float32) if fill is None else np.full(shape, fill, np.float32)
            self.on.append(gpu(x).to(torch.bfloat16 if elem == "bf16" else torch.float32))
        self.starts_on, self.lengths_on, self.table_on = gpu(np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)), gpu(np.array(self.lengths, np.int32)), gpu(self.table)

    def views(self):
        return [x if self.order == "head" else x.transpose(1, 2) for x in self.on]

    def cache(self):
        k = self.views()[0].stride()
        return D.KvCache(keys=self.on[0].data_ptr(), values=self.on[1].data_ptr(), elem=D.KV_BF16 if self.elem == "bf16" else D.KV_F32, kv_heads=self.kv_heads,
                         head_size=self.d, page_size=self.page, pages=self.pages, page_stride=k[0], head_stride=k[1], slot_stride=k[2])

    def batch(self):
        return D.KvBatch(sequences=len(self.n), table_pages=self.per, table_stride=self.per, query_starts=self.starts_on.data_ptr(), lengths=self.lengths_on.data_ptr(),
                         page_table=self.table_on.data_ptr())

    def dense(self, s):
        """Keys and values of sequence s, [length, heads, d] as fp32."""
        at = np.arange(self.lengths[s])
        page, slot = self.table[s][at // self.page], at % self.page
        page, slot = torch.from_numpy(page.astype(np.int64)).cuda(), torch.from_numpy(slot).cuda()
        return [v[page, :, slot].float().cpu().numpy() for v in self.views()]


# ---- appending -------------------------------------------------------------------------------------------------------

def append(ctx, paged, q, k, v, rotary=None, q_out=None, **more):
    """q / k / v: [tokens, heads, d] on the GPU (q may be None)."""
    fields = dict(tokens=k.shape[0], k=k.data_ptr(), v=v.data_ptr(), k_strides=k.stride()[:2], v_strides=v.stride()[:2], epsilon=EPS)
    if q is not None:
        fields.update(q_heads=q.shape[1], q=q.data_ptr(), q_out=q_out.data_ptr(), q_strides=q.stride()[:2], q_out_strides=q_out.stride()[:2])
    torch.cuda.synchronize()
    ctx.kv_append_raw(paged.cache(), paged.batch(), D.KvTokens(**{**fields, **more}), rotary)


APPENDS = [  # n, lengths, q heads, kv heads, d, dim, page, type, order, interleaved, norm
    ([1], [1], 12, 12, 64, 64, 16, "f32", "head", False, False),
    ([1, 1, 1, 1, 1], [9, 1, 300, 17, 16], 32, 8, 128, 128, 16, "f32", "head", False, True),
    ([1] * 70, list(range(1, 71)), 4, 2, 64, 32, 8, "bf16", "slot", True, False),
    ([3, 0, 7, 1, 0], [3, 9, 30, 1, 0], 6, 3, 96, 96, 5, "f32", "slot", False, True),
    ([0, 0, 65, 2], [0, 4, 65, 100], 7, 1, 80, 40, 24, "bf16", "head", True, True),
    ([200, 31], [400, 31], 0, 4, 128, 64, 64, "bf16", "slot", False, False),
    ([5, 6], [5, 60], 3, 1, 20, 12, 3, "f32", "head", False, True),
    ([5, 6], [5, 60], 3, 2, 7, 6, 1, "bf16", "head", True, False),
    ([40], [1000], 2, 2, 256, 0, 250, "f32", "slot", False, False),
]


@pytest.mark.parametrize("n,lengths,heads,kv,d,dim,page,elem,order,interleaved,norm", APPENDS)
def test_tokens_land_in_their_slots(here, case, n, lengths, heads, kv, d, dim, page, elem, order, interleaved, norm):
    case(f"append n {n[:5]} lengths {lengths[:5]} heads {heads}/{kv} d {d} dim {dim} page {page} {elem} {order}")
    rng = np.random.default_rng(d + page)
    paged = Paged(rng, n, lengths, kv, d, page, elem, order, fill=7.0)
    tokens = sum(n) + 3  # three rows of padding behind the last sequence
    packed = rng.standard_normal((tokens, heads + 2 * kv, d)).astype(np.float32)
    on = gpu(packed)
    q, k, v = on[:, :heads], on[:, heads:heads + kv], on[:, heads + kv:]
    q_out = torch.full((tokens, heads, d), 5.0, device="cuda")
    f = gpu(D.rotary_frequencies(dim)) if dim else None
    gammas = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) if norm else None for _ in range(2)]
    held = [gpu(x) if norm else None for x in gammas]
    more = dict(q_gamma=held[0].data_ptr(), k_gamma=held[1].data_ptr()) if norm else {}
    rotary = D.Rotary(f.data_ptr(), dim, int(interleaved), 0.75) if dim else None
    append(here, paged, q if heads else None, k, v, rotary, q_out if heads else None, **more)
    here.sync()
    places = np.concatenate([np.arange(l - m, l) for m, l in zip(n, lengths)]) if sum(n) else np.empty(0)
    seq = np.repeat(np.arange(len(n)), n)
    live = slice(0, sum(n))
    frequencies, magnitude = (D.rotary_frequencies(dim), 0.75) if dim else (np.empty(0), 1.0)

    def check(got, x, gamma, extra=0.0):
        y = normed(x, gamma, EPS)
        want, bound = turned(y, places, frequencies, interleaved, magnitude), turned_bound(y, dim // 2, interleaved, gamma, magnitude)
        off = np.abs(got - want)
        assert (off <= bound + extra * (np.abs(want) + bound) + 1e-37).all(), (off / (bound + extra * np.abs(want) + 1e-37)).max()

    rounding = 2.0 ** -8 if elem == "bf16" else 0.0
    if heads:
        got = q_out.cpu().numpy()
        check(got[live], packed[live, :heads], gammas[0])
        assert (got[sum(n):] == 5.0).all()
    keys, values = (x.float().cpu().numpy() for x in paged.views())
    page_of, slot = paged.table[seq, places.astype(int) // page], places.astype(int) % page
    check(keys[page_of, :, slot], packed[live, heads:heads + kv], gammas[1], rounding)
    want = packed[live, heads + kv:]
    np.testing.assert_array_equal(values[page_of, :, slot], bf16(want) if elem == "bf16" else want)
    for x in (keys, values):  # no other slot was written
        mask = np.ones(x.shape, bool)
        mask[page_of, :, slot] = False
        assert (x[mask] == 7.0).all()


def test_queries_turn_in_place_and_positions_may_be_given(here, case):
    case("append in place, own positions")
    rng = np.random.default_rng(3)
    paged = Paged(rng, [2, 3], [10, 3], 2, 64, 4, fill=0.0)
    packed = rng.standard_normal((5, 8, 64)).astype(np.float32)
    on, f, positions = gpu(packed), gpu(D.rotary_frequencies(64)), gpu(np.array([5, 900, 70000, 1, 2], np.int64))
    append(here, paged, on[:, :4], on[:, 4:6], on[:, 6:], D.Rotary(f.data_ptr(), 64), on[:, :4], positions=positions.data_ptr(), position_size=8)
    here.sync()
    got = on.cpu().numpy()
    y = packed[:, :4].astype(np.float64)
    assert (np.abs(got[:, :4] - turned(y, positions.cpu().numpy(), D.rotary_frequencies(64), False)) <= turned_bound(y, 32, False, None)).all()
    assert (got[:, 4:] == packed[:, 4:]).all()


def test_values_that_bf16_does_not_hold(here, case):
    case("append, special values")
    rng = np.random.default_rng(4)
    special = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 3.3895e38, 3.4e38, 1e-40, 1.00390625, 1.01171875, -1.00390625, 65536.0], np.float32)
    for elem in ("f32", "bf16"):
        paged = Paged(rng, [1], [1], 1, 16, 2, elem, fill=0.0)
        x = np.zeros((1, 1, 16), np.float32)
        x[0, 0, :12] = special
        append(here, paged, None, gpu(x), gpu(x))
        here.sync()
        got = paged.views()[1][paged.table[0, 0], 0, 0].float().cpu().numpy()
        want = gpu(x).to(torch.bfloat16).float().cpu().numpy()[0, 0] if elem == "bf16" else x[0, 0]
        np.testing.assert_array_equal(got, want)


def raises_at_sync(ctx, code=ERR_ARG):
    with pytest.raises(AltiusHipError) as e:
        ctx.sync()
    assert e.value.code == code and "paged cache" in str(e.value)
    ctx.sync()  # told once


@pytest.mark.parametrize("what", ["page", "page_negative", "length", "length_short", "starts", "starts_past"])
def test_a_batch_that_does_not_fit_is_told_and_writes_nowhere_else(here, case, what):
    case(f"append, bad {what}")
    rng = np.random.default_rng(5)
    paged = Paged(rng, [2, 2, 2], [8, 8, 8], 1, 16, 4, fill=7.0)
    x = gpu(rng.standard_normal((6, 1, 16)).astype(np.float32))
    if what == "page":
        paged.table_on[1, 1] = paged.pages
    elif what == "page_negative":
        paged.table_on[1, 1] = -1
    elif what == "length":
        paged.lengths_on[1] = 9
    elif what == "length_short":
        paged.lengths_on[1] = 0
    elif what == "starts":
        paged.starts_on[1] = 5  # sequence 1 then has -1 rows, sequence 0 five
        paged.lengths_on[0] = 2
    else:
        paged.starts_on[3] = 9
    append(here, paged, None, x, x)
    raises_at_sync(here)
    got = paged.views()[0].float().cpu().numpy()
    if what in ("page", "page_negative", "length", "length_short"):
        for s in (0, 2):
            np.testing.assert_array_equal(got[paged.table[s, 1], 0, 2:], x.cpu().numpy()[2 * s:2 * s + 2, 0])
        assert (got[paged.table[1]] == 7.0).all() and (got != 7.0).sum() <= 4 * 16
    assert (got == 7.0).sum() >= (paged.pages * 4 - 6) * 16


# ---- attention -------------------------------------------------------------------------------------------------------

def attend(ctx, paged, q, causal=True, window=0, cap=0.0, slopes=None, prefix=None, first=None, scale=None, out=None, max_tokens=0, max_keys=0):
    """q [tokens, heads, d] on the GPU; the workspace is filled with NaN before the call."""
    out = torch.full_like(q, 5.0, memory_format=torch.contiguous_format) if out is None else out
    call = D.KvAttend(tokens=q.shape[0], q_heads=q.shape[1], q=q.data_ptr(), out=out.data_ptr(), q_strides=q.stride()[:2], out_strides=out.stride()[:2],
                      scale=scale if scale is not None else 1 / math.sqrt(paged.d), softcap=cap, causal=int(causal), window=window, max_tokens=max_tokens, max_keys=max_keys)
    keep = {}
    for name, x in (("slopes", slopes), ("prefix", prefix), ("first_keys", first)):
        if x is not None:
            keep[name] = gpu(x)
            setattr(call, name, keep[name].data_ptr())
    room = D.kv_attention_workspace(ctx, paged.cache(), paged.batch(), call)
    space = torch.full((room // 4 + 4,), math.nan, device="cuda")
    call.workspace, call.workspace_bytes = space.data_ptr(), room
    torch.cuda.synchronize()
    ctx.kv_attention_raw(paged.cache(), paged.batch(), call)
    torch.cuda.synchronize()
    assert torch.isnan(space[room // 4:]).all()
    return out


def held_to_definition(got, paged, q, causal=True, window=0, cap=0.0, slopes=None, prefix=None, first=None, scale=None):
    at = 0
    for s, (m, l) in enumerate(zip(paged.n, paged.lengths)):
        k, v = paged.dense(s)
        low, high, place = ranges(m, l, causal, window, None if prefix is None else prefix[s], None if first is None else first[at:at + m])
        want, bound = attended(q[at:at + m], k, v, low, high, place, scale if scale is not None else 1 / math.sqrt(paged.d), cap, slopes)
        mine = got[at:at + m]
        nan, finite = np.isnan(want), np.isfinite(want)
        assert (np.isnan(mine) == nan).all(), f"sequence {s}: NaN elsewhere"
        np.testing.assert_array_equal(mine[~finite & ~nan], want[~finite & ~nan])
        with np.errstate(invalid="ignore"):
            off = np.where(finite, np.abs(mine - want), 0.0)
        assert (off <= np.where(finite, bound, 0) + 1e-37).all(), f"sequence {s}: {np.nanmax(off / np.where(finite, bound + 1e-37, 1)):.3g} times the bound, {off.max():.3g}"
        at += m
    assert (got[at:] == 5.0).all(), "padding was written"


SHAPES = [  # n, lengths, heads, kv heads, d, page, type, order
    ([1], [1], 1, 1, 64, 16, "f32", "head"),
    ([1], [77], 12, 12, 64, 16, "f32", "head"),
    ([1, 1, 1], [1, 300, 33], 8, 2, 128, 16, "f32", "slot"),
    ([1, 1, 1], [5, 31, 1000], 8, 1, 128, 32, "bf16", "head"),
    ([1], [5000], 4, 2, 64, 64, "f32", "head"),
    ([1], [9000], 7, 1, 128, 48, "bf16", "slot"),
    ([1, 0, 2, 0], [40, 12, 41, 0], 32, 1, 64, 16, "bf16", "slot"),
    ([3, 1], [70, 500], 40, 2, 96, 24, "f32", "head"),
    ([2, 5], [19, 300], 6, 3, 80, 8, "bf16", "head"),
    ([1, 1], [100, 64], 4, 4, 256, 16, "f32", "head"),
    ([4, 1], [200, 129], 16, 2, 256, 64, "bf16", "slot"),
    ([1, 3], [1000, 700], 4, 4, 256, 16, "f32", "head"),
    ([1, 3], [1000, 700], 8, 1, 256, 48, "f32", "slot"),
    ([2], [3000], 4, 2, 256, 16, "bf16", "slot"),
    ([1, 1], [2500, 90], 2, 1, 256, 20, "bf16", "head"),
    ([1], [1111], 6, 6, 132, 16, "f32", "head"),
    ([1] * 70, [5 * i + 1 for i in range(69)] + [1500], 8, 4, 64, 16, "f32", "slot"),
    ([1] * 66 + [0, 3], [1700] + [330 - 5 * i for i in range(65)] + [5, 900], 6, 6, 64, 16, "bf16", "head"),
    ([70, 1], [400, 3000], 2, 2, 256, 16, "f32", "slot"),
    ([1, 2], [33, 50], 3, 1, 200, 7, "bf16", "head"),
    ([1, 2], [33, 50], 3, 1, 20, 5, "f32", "slot"),
    ([17], [17], 2, 2, 64, 16, "f32", "head"),
    ([65, 1, 130], [65, 700, 200], 4, 2, 64, 16, "f32", "head"),
    ([100], [300], 8, 2, 128, 64, "bf16", "slot"),
    ([128, 3], [128, 260], 2, 1, 96, 24, "bf16", "head"),
    ([257], [400], 1, 1, 128, 250, "f32", "slot"),
    ([70], [90], 2, 2, 256, 32, "f32", "head"),
    ([1, 66], [4100, 66], 2, 2, 64, 64, "bf16", "head"),
]


@pytest.mark.parametrize("n,lengths,heads,kv,d,page,elem,order", SHAPES)
@pytest.mark.parametrize("plain", [True, False])
def test_rows_attend_to_their_keys(here, case, n, lengths, heads, kv, d, page, elem, order, plain):
    case(f"attend n {n} lengths {lengths} heads {heads}/{kv} d {d} page {page} {elem} {order} plain {plain}")
    rng = np.random.default_rng(d + page + len(n))
    paged = Paged(rng, n, lengths, kv, d, page, elem, order)
    q = (1.5 * rng.standard_normal((sum(n) + 2, heads, d))).astype(np.float32)
    options = {} if plain else dict(window=max(2, max(lengths) // 3), cap=20.0, slopes=(2.0 ** -np.arange(1, heads + 1).astype(np.float32) * 0.5).astype(np.float32),
                                    first=rng.integers(-3, max(lengths), sum(n) + 2).astype(np.int32), prefix=rng.integers(0, 30, len(n)).astype(np.int32))
    got = attend(here, paged, gpu(q), **options).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q, **options)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("options", [dict(causal=False), dict(window=1), dict(window=40), dict(causal=False, window=9), dict(prefix=np.array([0, 60, 1000], np.int32)),
                                     dict(cap=2.0), dict(scale=0.0), dict(scale=-0.2), dict(slopes=np.array([0.0, 0.5, 0.01, -0.02], np.float32)),
                                     dict(causal=False, prefix=np.array([-5, 3, 9], np.int32))])
@pytest.mark.parametrize("n", [[1, 2, 1], [90, 33, 64]])
def test_each_mask_and_bias(here, case, elem, options, n):
    case(f"attend {elem} {sorted(options)} n {n}")
    rng = np.random.default_rng(17)
    paged = Paged(rng, n, [99, 50, 64], 2, 64, 16, elem)
    q = rng.standard_normal((sum(n), 4, 64)).astype(np.float32)
    got = attend(here, paged, gpu(q), **options).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q, **options)


MIXED = [  # n, lengths: few and many rows in one batch, whose keys are cut into parts
    ([57, 20, 16, 33, 200, 0, 1, 9], [600, 900, 700, 64, 1500, 10, 333, 9]),
    ([1, 40, 1, 300], [2100, 1000, 1, 300]),
    ([300] + [1] * 60 + [17] * 9 + [34] * 2, [900] + [7 * i + 1 for i in range(60)] + [40 * i + 17 for i in range(9)] + [800, 34]),
]


@pytest.mark.parametrize("n,lengths", MIXED)
@pytest.mark.parametrize("heads,kv,d,page,elem", [(2, 1, 128, 24, "f32"), (1, 1, 64, 16, "f32"), (2, 2, 96, 16, "f32"), (1, 1, 96, 40, "bf16"), (3, 1, 128, 32, "bf16"), (1, 1, 256, 16, "f32")])
@pytest.mark.parametrize("options", [dict(), dict(window=130, cap=9.0), dict(causal=False, prefix=True), dict(first=True, slopes=True, prefix=True)])
def test_batches_of_all_lengths(here, case, n, lengths, heads, kv, d, page, elem, options):
    case(f"attend mixed {len(n)} heads {heads}/{kv} d {d} page {page} {elem} {sorted(options)}")
    rng = np.random.default_rng(len(n) + d)
    paged = Paged(rng, n, lengths, kv, d, page, elem)
    q = rng.standard_normal((sum(n) + 3, heads, d)).astype(np.float32)
    options = dict(options)
    if "prefix" in options: options["prefix"] = rng.integers(-2, 500, len(n)).astype(np.int32)
    if "first" in options: options["first"] = rng.integers(-3, 700, len(q)).astype(np.int32)
    if "slopes" in options: options["slopes"] = np.full(heads, 0.03, np.float32)
    got = attend(here, paged, gpu(q), max_tokens=max(n), max_keys=max(lengths), **options).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q, **options)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n", [[1, 1, 2], [80, 5, 30]])
def test_rows_that_see_nothing_are_zero(here, case, elem, n):
    """First keys behind the token, and sequences shorter than their rows: such rows are 0, the others what they were."""
    case(f"attend empty rows {elem} n {n}")
    rng = np.random.default_rng(18)
    lengths = [100, 5, 0 if n[2] == 2 else 11]
    paged = Paged(rng, n, lengths, 1, 64, 16, elem)
    q = rng.standard_normal((sum(n), 4, 64)).astype(np.float32)
    first = np.zeros(sum(n), np.int32)
    first[0] = 5000
    first[n[0] - 1] = 100
    got = attend(here, paged, gpu(q), first=first).cpu().numpy()
    here.sync()
    assert (got[0] == 0).all() and (got[n[0] - 1] == 0).all() and (got[n[0] + n[1]] == 0).all()
    held_to_definition(got, paged, q, first=first)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("page", [16, 32, 24])
@pytest.mark.parametrize("n", [[3, 1], [70, 40]])
def test_slots_that_are_not_seen_may_hold_anything(here, case, elem, bad, page, n):
    """NaN and infinities behind a sequence's end, in front of a window, in pages of nobody, and in keys that only later rows see."""
    case(f"attend unseen {bad} {elem} page {page} n {n}")
    rng = np.random.default_rng(19)
    lengths = [100, 67]
    paged = Paged(rng, n, lengths, 2, 64, page, elem)
    for x in paged.views():
        seen = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
        for s, (m, l) in enumerate(zip(n, lengths)):
            at = np.arange(max(0, l - m - 20), l)
            seen[torch.from_numpy(paged.table[s][at // page].astype(np.int64)).cuda(), :, torch.from_numpy(at % page).cuda()] = True
        x[~seen] = bad
    q = rng.standard_normal((sum(n), 4, 64)).astype(np.float32)
    got = attend(here, paged, gpu(q), window=20).cpu().numpy()
    assert np.isfinite(got).all()
    held_to_definition(got, paged, q, window=20)
    # the newest token's key and value: only its own row sees them
    for x in paged.views():
        x[paged.table[0, (lengths[0] - 1) // page], :, (lengths[0] - 1) % page] = bad
    got = attend(here, paged, gpu(q), window=20).cpu().numpy()
    rows = np.isfinite(got).all((1, 2))
    assert rows[np.arange(sum(n)) != n[0] - 1].all() and not rows[n[0] - 1]
    held_to_definition(np.where(np.arange(sum(n))[:, None, None] == n[0] - 1, np.nan, got), paged, np.where(np.arange(sum(n))[:, None, None] == n[0] - 1, np.nan, q).astype(np.float32),
                       window=20)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n", [[2], [70]])
def test_infinite_values_and_keys_that_are_seen(here, case, elem, n):
    """An infinite value makes its channel infinite; a key that gives minus infinity has no weight."""
    case(f"attend seen infinities {elem} n {n}")
    rng = np.random.default_rng(20)
    paged = Paged(rng, n, [90], 1, 64, 16, elem)
    keys, values = paged.views()
    values[paged.table[0, 0], 0, 3, 5] = math.inf
    values[paged.table[0, 1], 0, 2, 6] = -math.inf
    keys[paged.table[0, 0], 0, 7, 0] = -math.inf
    q = rng.standard_normal((n[0], 2, 64)).astype(np.float32)
    q[..., 0] = np.abs(q[..., 0]) + 0.1
    got = attend(here, paged, gpu(q)).cpu().numpy()
    held_to_definition(got, paged, q)
    assert (got[..., 5] == np.inf).all() and (got[..., 6] == -np.inf).all() and np.isfinite(got[..., :5]).all()


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d,page", [(64, 16), (96, 24), (128, 32), (256, 16)])
@pytest.mark.parametrize("n,lengths", [([3, 2], [40, 700]), ([70, 30], [70, 900])])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_queries_that_are_not_finite(here, case, elem, d, page, n, lengths, cap):
    """Infinity and NaN among the queries reach their own rows and no other."""
    case(f"attend queries not finite {elem} d {d} page {page} n {n} cap {cap}")
    rng = np.random.default_rng(21)
    paged = Paged(rng, n, lengths, 1, d, page, elem)
    q = rng.standard_normal((sum(n), 2, d)).astype(np.float32)
    for at, (channel, value) in enumerate([(0, math.inf), (d - 1, -math.inf), (3, math.nan), (d - 4, math.inf)]):
        q[at % n[0], at % 2, channel] = value
        q[n[0] + at % n[1], at % 2, channel] = value
    got = attend(here, paged, gpu(q), cap=cap, max_tokens=max(n)).cpu().numpy()
    held_to_definition(got, paged, q, cap=cap)


def test_a_large_range_of_scores(here, case):
    case("attend peaked scores")
    rng = np.random.default_rng(21)
    for elem, n in (("f32", [1]), ("bf16", [1]), ("f32", [100]), ("bf16", [100])):
        paged = Paged(rng, n, [300], 1, 64, 16, elem)
        q = (30 * rng.standard_normal((n[0], 1, 64))).astype(np.float32)
        got = attend(here, paged, gpu(q), scale=1.0).cpu().numpy()
        held_to_definition(got, paged, q, scale=1.0)


def test_a_page_outside_the_cache_is_told(here, case):
    case("attend bad pages")
    rng = np.random.default_rng(22)
    for page, n in ((16, [1, 1]), (24, [1, 1]), (16, [80, 70]), (24, [80, 70])):
        for bad in (-1, 1 << 30):
            paged = Paged(rng, n, [90, 80], 1, 64, page)
            q = rng.standard_normal((sum(n), 2, 64)).astype(np.float32)
            paged.table_on[1, 0] = bad
            got = attend(here, paged, gpu(q)).cpu().numpy()
            raises_at_sync(here)
            k, v = paged.dense(0)
            low, high, place = ranges(n[0], 90, True, 0, None, None)
            want, bound = attended(q[:n[0]], k, v, low, high, place, 1 / 8, 0.0, None)
            assert (np.abs(got[:n[0]] - want) <= bound).all()


@pytest.mark.parametrize("what", ["length", "length_negative", "starts", "starts_past", "max_tokens", "max_keys"])
def test_a_batch_that_does_not_fit_the_call_is_told_and_its_rows_stay(here, case, what):
    case(f"attend, bad {what}")
    rng = np.random.default_rng(23)
    paged = Paged(rng, [2, 2], [30, 30], 1, 64, 16)
    q = gpu(rng.standard_normal((4, 2, 64)).astype(np.float32))
    more = {}
    if what == "length":
        paged.lengths_on[1] = 33
    elif what == "length_negative":
        paged.lengths_on[1] = -1
    elif what == "starts":
        paged.starts_on[2] = 1
    elif what == "starts_past":
        paged.starts_on[2] = 5
    elif what == "max_tokens":
        more = dict(max_tokens=1)
    else:
        more = dict(max_keys=29)
    got = attend(here, paged, q, **more).cpu().numpy()
    raises_at_sync(here)
    assert (got[2:] == 5.0).all()


def test_the_call_is_refused_without_its_workspace(here, case):
    case("attend refusals")
    rng = np.random.default_rng(24)
    paged = Paged(rng, [1], [4000], 1, 64, 16)
    q = gpu(rng.standard_normal((1, 2, 64)).astype(np.float32))
    call = D.KvAttend(tokens=1, q_heads=2, q=q.data_ptr(), out=q.data_ptr(), q_strides=(128, 64), out_strides=(128, 64))
    room = D.kv_attention_workspace(here, paged.cache(), paged.batch(), call)
    assert room > 0
    space = torch.zeros(room, dtype=torch.uint8, device="cuda")

    def code(cache=None, batch=None, **more):
        for name, value in {**dict(workspace=space.data_ptr(), workspace_bytes=room, q=q.data_ptr(), out=space.data_ptr(), tokens=1), **more}.items():
            setattr(call, name, value)
        try:
            here.kv_attention_raw(cache or paged.cache(), batch or paged.batch(), call)
        except AltiusHipError as e:
            return e.code
        return 0

    assert code(workspace_bytes=room - 4) == ERR_ARG and code(workspace=None) == ERR_ARG
    assert code(q=None) == ERR_ARG and code(out=None) == ERR_ARG
    empty = paged.cache()
    empty.pages = 0
    assert code(cache=empty) == ERR_ARG
    batch = paged.batch()
    batch.lengths = None
    assert code(batch=batch) == ERR_ARG
    batch = paged.batch()
    batch.sequences = 0
    assert code(batch=batch, q=None, out=None) == 0 and code(tokens=0, q=None) == 0
    odd = paged.cache()
    odd.slot_stride = 66
    assert code(cache=odd) == ERR_UNSUPPORTED
    here.sync()


def test_strided_queries_and_results(here, case):
    """Queries read out of a packed product; results written between other columns."""
    case("attend strided")
    rng = np.random.default_rng(25)
    for n in ([1, 1], [70, 4]):
        paged = Paged(rng, n, [90, 20], 2, 64, 16)
        packed = rng.standard_normal((sum(n), 10, 64)).astype(np.float32)
        wide = torch.full((sum(n), 6, 80), 9.0, device="cuda")
        attend(here, paged, gpu(packed)[:, 3:7], out=wide[:, 1:5, 8:72])
        got = wide.cpu().numpy()
        held_to_definition(got[:, 1:5, 8:72], paged, packed[:, 3:7])
        mask = np.ones(got.shape, bool)
        mask[:, 1:5, 8:72] = False
        assert (got[mask] == 9.0).all()


def test_a_cache_past_32_bits(here, case):
    """Pages more than 2^33 bytes apart."""
    case("attend far pages")
    rng = np.random.default_rng(26)
    stride = (1 << 31) + 64 * 3
    whole = [torch.empty(2 * stride + 16 * 64, device="cuda") for _ in range(2)]
    for n in ([1], [70]):
        paged = Paged(rng, n, [100], 1, 64, 48, spare_pages=0)
        assert paged.pages == 3
        for x, y in zip(whole, paged.on):
            far = x.as_strided((3, 1, 16, 64), (stride, 1024, 64, 1))
            far.copy_(y[:, :, :16])
        small = Paged(rng, n, [40], 1, 64, 16, spare_pages=0)
        small.on = [x.as_strided((3, 1, 16, 64), (stride, 1024, 64, 1)) for x in whole]
        q = rng.standard_normal((n[0], 2, 64)).astype(np.float32)
        held_to_definition(attend(here, small, gpu(q)).cpu().numpy(), small, q)
        k, v = gpu(rng.standard_normal((n[0], 1, 64)).astype(np.float32)), gpu(rng.standard_normal((n[0], 1, 64)).astype(np.float32))
        if n[0] == 1:
            append(here, small, None, k, v)
            here.sync()
            np.testing.assert_array_equal(small.dense(0)[1][39], v.cpu().numpy()[0])


def test_recorded_and_replayed_with_other_lengths(here, case):
    """One recorded pass -- append, then attention -- replayed while the sequences grow on the device, beside eager calls of the same
    context between the replays."""
    case("decode replay")
    rng = np.random.default_rng(27)
    stream = torch.cuda.Stream()
    for elem in ("f32", "bf16"):
        paged = Paged(rng, [1, 1, 1], [1, 1, 1], 2, 64, 16, elem, table_pages=40, fill=0.0)
        q = torch.zeros((3, 8, 64), device="cuda")
        packed, out, f = torch.zeros((3, 12, 64), device="cuda"), torch.full((3, 8, 64), 5.0, device="cuda"), gpu(D.rotary_frequencies(64))
        with D.Context(0, stream=stream.cuda_stream) as c:
            tokens = D.KvTokens(tokens=3, q_heads=8, q=packed.data_ptr(), k=packed[:, 8:].data_ptr(), v=packed[:, 10:].data_ptr(), q_out=q.data_ptr(),
                                q_strides=(768, 64), k_strides=(768, 64), v_strides=(768, 64), q_out_strides=(512, 64))
            call = D.KvAttend(tokens=3, q_heads=8, q=q.data_ptr(), out=out.data_ptr(), q_strides=(512, 64), out_strides=(512, 64), scale=0.125, max_tokens=1)
            room = D.kv_attention_workspace(c, paged.cache(), paged.batch(), call)
            space = torch.zeros(max(room, 16), dtype=torch.uint8, device="cuda")
            call.workspace, call.workspace_bytes = space.data_ptr(), room
            rotary = D.Rotary(f.data_ptr(), 64)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                c.kv_append_raw(paged.cache(), paged.batch(), tokens, rotary)
                c.kv_attention_raw(paged.cache(), paged.batch(), call)
            for step in range(40):
                x = rng.standard_normal((3, 12, 64)).astype(np.float32)
                grown = [1 + step, 1 + 2 * (step // 2), 600 - 40 + step + 1]
                paged.lengths_on.copy_(torch.tensor(grown, dtype=torch.int32))
                packed.copy_(gpu(x))
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                c.sync()
                paged.lengths = grown
                if step % 13 == 0:
                    held_to_definition(out.cpu().numpy(), paged, q.cpu().numpy(), scale=0.125)
                    again = attend(c, paged, q, scale=0.125).cpu().numpy()
                    np.testing.assert_allclose(again, out.cpu().numpy(), rtol=1e-4, atol=1e-5)
            # a replay's bad page is told like a call's
            paged.table_on[0, 0] = -1
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            raises_at_sync(c)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_a_prompt_in_pieces_then_token_by_token(here, case, elem, norm):
    """What serving does: prompts appended whole or in pieces, tokens one by one, each attended to as it comes; every row is what one
    attention over the whole sequence gives, from the same keys rounded to the cache's type."""
    case(f"serving {elem} norm {norm}")
    rng = np.random.default_rng(28)
    heads, kv, d, total = 4, 2, 64, [150, 40]
    paged = Paged(rng, [0, 0], total, kv, d, 16, elem, fill=math.nan)
    x = [rng.standard_normal((t, heads + 2 * kv, d)).astype(np.float32) for t in total]
    f = gpu(D.rotary_frequencies(d))
    gamma = gpu((1 + 0.2 * rng.standard_normal(d)).astype(np.float32))
    more = dict(q_gamma=gamma.data_ptr(), k_gamma=gamma.data_ptr()) if norm else {}
    results, turned_q = [np.zeros((t, heads, d), np.float32) for t in total], [np.zeros((t, heads, d), np.float32) for t in total]
    done = [0, 0]
    for n in [[100, 7], [40, 1], [0, 1]] + [[1, 1]] * 10:
        paged.n, paged.lengths = n, [a + b for a, b in zip(done, n)]
        paged.starts_on.copy_(torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32))
        paged.lengths_on.copy_(torch.tensor(paged.lengths, dtype=torch.int32))
        on = gpu(np.concatenate([x[s][done[s]:done[s] + n[s]] for s in range(2)]))
        q = torch.empty((sum(n), heads, d), device="cuda")
        append(here, paged, on[:, :heads], on[:, heads:heads + kv], on[:, heads + kv:], D.Rotary(f.data_ptr(), d), q, **more)
        out = attend(here, paged, q).cpu().numpy()
        here.sync()
        at = 0
        for s in range(2):
            results[s][done[s]:done[s] + n[s]], turned_q[s][done[s]:done[s] + n[s]] = out[at:at + n[s]], q.cpu().numpy()[at:at + n[s]]
            at += n[s]
        done = list(paged.lengths)
    assert done == [150, 19]
    paged.n = paged.lengths = done
    held_to_definition(np.concatenate([results[0], results[1][:19]]), paged, np.concatenate([turned_q[0], turned_q[1][:19]]))
    for s in range(2):
        keys, values = paged.dense(s)
        y = normed(x[s][:done[s], heads:heads + kv], gamma.cpu().numpy() if norm else None, EPS)
        want = turned(y, np.arange(done[s]), D.rotary_frequencies(d), False)
        bound = turned_bound(y, d // 2, False, gamma if norm else None)
        assert (np.abs(keys - want) <= bound + (2.0 ** -8 if elem == "bf16" else 0) * (np.abs(want) + bound)).all()
        raw = x[s][:done[s], heads + kv:]
        np.testing.assert_array_equal(values, bf16(raw) if elem == "bf16" else raw)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("sequences,n,lengths,kv", [(40, 300, 500, 2), (40, 70, 4000, 8), (300, 40, 100, 1)])
def test_starts_that_jump_back_are_told(here, case, elem, sequences, n, lengths, kv):
    """Every other sequence takes the first rows once more: more rows in all than the call has."""
    case(f"attend starts that jump back {elem} {sequences} of {n}")
    rng = np.random.default_rng(32)
    paged = Paged(rng, [0] * sequences, [lengths] * sequences, kv, 64, 64, elem)
    paged.starts_on.copy_(torch.tensor([n if s % 2 else 0 for s in range(sequences + 1)], dtype=torch.int32))
    q = gpu(rng.standard_normal((n + 2, kv, 64)).astype(np.float32))
    got = attend(here, paged, q, max_tokens=n, max_keys=lengths)
    assert (got[n:] == 5.0).all()
    raises_at_sync(here)
    paged.n, paged.lengths = [n] + [0] * (sequences - 1), [lengths] * sequences  # the context goes on
    paged.starts_on.copy_(torch.tensor([0] + [n] * sequences, dtype=torch.int32))
    got = attend(here, paged, q, max_tokens=n, max_keys=lengths).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q.cpu().numpy())


def test_a_piece_beside_many_tokens(here, case):
    """Blocks for the row tiles that there are, not for as many as the longest sequence has in each."""
    case("attend a piece beside tokens")
    rng = np.random.default_rng(33)
    for elem, d, kv, options in (("f32", 64, 8, {}), ("bf16", 128, 8, dict(window=100)), ("f32", 96, 4, dict(first=True, prefix=True))):
        n, lengths = [1] * 380 + [150] + [3, 0] * 10 + [90, 1], [60 + s % 50 for s in range(380)] + [350] + [40, 7] * 10 + [90, 1]
        paged = Paged(rng, n, lengths, kv, d, 16, elem)
        q = rng.standard_normal((sum(n) + 1, 4 * kv, d)).astype(np.float32)
        options = dict(options)
        if "first" in options: options.update(first=rng.integers(0, 60, len(q)).astype(np.int32), prefix=rng.integers(0, 200, len(n)).astype(np.int32))
        got = attend(here, paged, gpu(q), max_tokens=150, max_keys=350, **options).cpu().numpy()
        here.sync()
        held_to_definition(got, paged, q, **options)


def test_replayed_with_other_rows(here, case):
    """One recorded attention whose sequences change from prompts to single tokens and back on the device."""
    case("attend replayed with other rows")
    rng = np.random.default_rng(31)
    stream = torch.cuda.Stream()
    for d, elem in ((128, "f32"), (64, "bf16")):
        paged = Paged(rng, [200, 30, 1], [900, 500, 700], 1, d, 16, elem)
        q, out = gpu(rng.standard_normal((240, 2, d)).astype(np.float32)), torch.full((240, 2, d), 5.0, device="cuda")
        with D.Context(0, stream=stream.cuda_stream) as c:
            call = D.KvAttend(tokens=240, q_heads=2, q=q.data_ptr(), out=out.data_ptr(), q_strides=(2 * d, d), out_strides=(2 * d, d), scale=0.125, causal=1, max_tokens=200)
            room = D.kv_attention_workspace(c, paged.cache(), paged.batch(), call)
            assert room > 0
            space = torch.full((room // 4,), math.nan, device="cuda")
            call.workspace, call.workspace_bytes = space.data_ptr(), room
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                c.kv_attention_raw(paged.cache(), paged.batch(), call)
            for n, lengths in (([200, 30, 1], [900, 500, 700]), ([1, 1, 1], [900, 1, 12]), ([0, 200, 8], [5, 200, 880]), ([16, 17, 33], [16, 400, 33]), ([200, 0, 40], [201, 0, 40])):
                paged.n, paged.lengths = n, lengths
                paged.starts_on.copy_(torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32))
                paged.lengths_on.copy_(torch.tensor(lengths, dtype=torch.int32))
                out.fill_(5.0), space.fill_(math.nan)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                c.sync()
                held_to_definition(out.cpu().numpy(), paged, q.cpu().numpy(), scale=0.125)


def test_two_contexts_at_once(here, case):
    """Two streams at work on one cache, each with a workspace of its own."""
    case("two contexts")
    rng = np.random.default_rng(29)
    paged = Paged(rng, [1, 1], [3000, 2500], 2, 64, 16)
    q = [gpu(rng.standard_normal((2, 8, 64)).astype(np.float32)) for _ in range(2)]
    out = [torch.full((2, 8, 64), 5.0, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [D.Context(0, stream=s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    spaces, calls = [], []
    for i in range(2):
        call = D.KvAttend(tokens=2, q_heads=8, q=q[i].data_ptr(), out=out[i].data_ptr(), q_strides=(512, 64), out_strides=(512, 64), scale=0.125, max_tokens=1)
        room = D.kv_attention_workspace(contexts[i], paged.cache(), paged.batch(), call)
        spaces.append(torch.zeros(max(16, room), dtype=torch.uint8, device="cuda"))
        call.workspace, call.workspace_bytes = spaces[-1].data_ptr(), room
        calls.append(call)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            contexts[i].kv_attention_raw(paged.cache(), paged.batch(), calls[i])
    for i in range(2):
        contexts[i].sync()
        held_to_definition(out[i].cpu().numpy(), paged, q[i].cpu().numpy(), scale=0.125)
        contexts[i].close()


def test_the_same_call_gives_the_same_bits(here, case):
    case("attend bits")
    rng = np.random.default_rng(30)
    for n, elem in (([1, 1], "f32"), ([1, 1], "bf16"), ([70, 90], "f32"), ([70, 90], "bf16")):
        paged = Paged(rng, n, [3000, 2500], 2, 128, 16, elem)
        q = gpu(rng.standard_normal((sum(n), 8, 128)).astype(np.float32))
        first = attend(here, paged, q).cpu().numpy()
        for _ in range(3):
            np.testing.assert_array_equal(attend(here, paged, q).cpu().numpy().view(np.uint32), first.view(np.uint32))


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d,page", [(64, 8), (64, 16), (64, 24), (64, 64), (128, 16), (96, 8), (256, 8), (256, 24)])
@pytest.mark.parametrize("n,lengths", [([1, 3], [1000, 500]), ([100, 70], [1000, 700])])
@pytest.mark.parametrize("mask", ["window", "first"])
def test_pages_in_front_of_the_first_key_seen_may_be_gone(here, case, elem, d, page, n, lengths, mask):
    """A window has left them, or no document reaches back to them: their entries, and those behind the end, hold nothing that is a page."""
    case(f"attend released pages {elem} d {d} page {page} n {n} {mask}")
    rng = np.random.default_rng(34)
    paged = Paged(rng, n, lengths, 1, d, page, elem, table_pages=1008 // page + 3)
    options = dict(window=300) if mask == "window" else dict(first=np.concatenate([np.full(m, max(0, l - m - 250), np.int32) for m, l in zip(n, lengths)]))
    for s, (m, l) in enumerate(zip(n, lengths)):
        low = ranges(m, l, True, options.get("window", 0), None, options["first"][sum(n[:s]):][:m] if mask == "first" else None)[0].min()
        assert low > 100
        paged.table_on[s, :low // page] = -1 if s else paged.pages + 7
        paged.table_on[s, -(-l // page):] = -1
    q = rng.standard_normal((sum(n), 2, d)).astype(np.float32)
    got = attend(here, paged, gpu(q), **options).cpu().numpy()
    here.sync()  # nothing to tell
    held_to_definition(got, paged, q, **options)


def test_a_bad_page_and_a_bad_index_are_both_told(here, case):
    """Two kernels raise their flags in front of one synchronisation."""
    case("bad page beside a bad index")
    rng = np.random.default_rng(35)
    paged = Paged(rng, [1], [20], 1, 64, 16)
    x = gpu(rng.standard_normal((1, 1, 64)).astype(np.float32))
    table, index, out = torch.zeros(6, device="cuda"), torch.tensor([6], device="cuda"), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    assert here.L.ahip_gather(here.handle, out.data_ptr(), table.data_ptr(), index.data_ptr(), 8, 4, 1, 6, 1, 1) == 0
    paged.table_on[0, 1] = -1
    append(here, paged, None, x, x)
    with pytest.raises(AltiusHipError) as e:
        here.sync()
    assert e.value.code == ERR_ARG and "paged cache" in str(e.value) and "Gather" in str(e.value)
    here.sync()  # told once


@pytest.mark.parametrize("n,lengths,left", [([4, 2, 70], [20, 9, 100], 1), ([3, 0, 2], [5, 7, 40], 2), ([2] * 80, list(range(10, 90)), 7), ([5, 1], [9, 3], 2)])
def test_some_of_a_batchs_sequences(here, case, n, lengths, left):
    """A call whose first sequence's rows do not start at row 0: the rows in front are padding, for either operator."""
    case(f"sequences {left} on of {len(n)}")
    rng = np.random.default_rng(36)
    paged = Paged(rng, n, lengths, 1, 64, 16, fill=7.0)
    packed = rng.standard_normal((sum(n) + 2, 4, 64)).astype(np.float32)
    on, q = gpu(packed), torch.full((sum(n) + 2, 2, 64), 5.0, device="cuda")
    some = paged.batch()
    some.sequences = len(n) - left
    some.query_starts, some.lengths, some.page_table = paged.starts_on[left:].data_ptr(), paged.lengths_on[left:].data_ptr(), paged.table_on[left:].data_ptr()
    paged.batch = lambda: some
    append(here, paged, on[:, :2], on[:, 2:3], on[:, 3:], None, q)
    here.sync()
    at, end = sum(n[:left]), sum(n)
    got = q.cpu().numpy()
    assert (got[:at] == 5.0).all() and (got[end:] == 5.0).all()
    np.testing.assert_array_equal(got[at:end], packed[at:end, :2])
    for s, (m, l) in enumerate(zip(n, lengths)):
        values = paged.dense(s)[1]
        assert (values[:l - m] == 7.0).all()
        np.testing.assert_array_equal(values[l - m:, 0], packed[sum(n[:s]):sum(n[:s + 1]), 3] if s >= left else np.full((m, 64), 7.0))
    for x in paged.views():
        x.copy_(gpu(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
    got = attend(here, paged, q).cpu().numpy()
    here.sync()
    assert (got[:at] == 5.0).all()
    paged.n, paged.lengths, paged.table = n[left:], lengths[left:], paged.table[left:]
    held_to_definition(got[at:], paged, packed[at:, :2])


def test_results_in_the_place_of_queries_are_refused(here, case):
    case("attend out is q")
    rng = np.random.default_rng(37)
    paged = Paged(rng, [1], [40], 1, 64, 16)
    q = rng.standard_normal((1, 2, 64)).astype(np.float32)
    on = gpu(q)
    with pytest.raises(AltiusHipError) as e:
        attend(here, paged, on, out=on)
    assert e.value.code == ERR_ARG
    here.sync()
    np.testing.assert_array_equal(on.cpu().numpy(), q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n", [[2], [70]])
@pytest.mark.parametrize("cap", [1e-18, 1e-3, 1e6, 1e18])
def test_caps_far_from_the_scores(here, case, elem, n, cap):
    """The smallest make all weights alike, the largest do nothing."""
    case(f"attend cap {cap} {elem} n {n}")
    rng = np.random.default_rng(38)
    paged = Paged(rng, n, [90], 1, 64, 16, elem)
    q = rng.standard_normal((n[0], 2, 64)).astype(np.float32)
    got = attend(here, paged, gpu(q), cap=float(np.float32(cap))).cpu().numpy()
    k, v = paged.dense(0)
    low, high, place = ranges(n[0], 90, True, 0, None, None)
    # A cap of 1000 times the scores and more changes them by less than 2^-21 of themselves; 8 steps of a large cap are not 8 of the score.
    want, bound = attended(q, k, v, low, high, place, 0.125, 0.0 if cap > 1e3 else cap, None)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("what", sorted(WINDOWS))
@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("n,lengths,heads,kv", [([2] * 12, [30 + 9 * i for i in range(12)], 16, 4), ([70, 40, 1], [200, 40, 300], 4, 2), ([2, 1], [1500, 700], 16, 1)])
def test_no_part_of_a_number_is_lost(here, case, what, elem, d, page, n, lengths, heads, kv):
    """Held to bounds that a dropped third part or product of parts exceeds (decoder_precision.py)."""
    case(f"attend precision {what} {elem} d {d} page {page} n {n[:3]}")
    rng = np.random.default_rng(d + page)
    paged = Paged(rng, n, lengths, kv, d, page, elem)
    for x, make in zip(paged.on, (keys, values)):
        x.copy_(gpu(make(rng, what, tuple(x.shape), elem)))
    q = queries(rng, what, sum(n) * heads, d).reshape(sum(n), heads, d)
    got = attend(here, paged, gpu(q), window=WINDOWS[what], scale=1.0).cpu().numpy()
    here.sync()
    at = 0
    for s, (m, l) in enumerate(zip(n, lengths)):
        k, v = paged.dense(s)
        low, high, _ = ranges(m, l, True, WINDOWS[what], None, None)
        seen = (np.arange(l) >= low[:, None]) & (np.arange(l) < high[:, None])
        for h in range(heads):
            want, bound = expected(what, q[at:at + m, h], k[:, h // (heads // kv)], v[:, h // (heads // kv)], seen)
            off = np.abs(got[at:at + m, h] - want)
            assert (off <= bound).all(), f"sequence {s} head {h}: off by {off.max():.3g}, {(off / np.maximum(bound, 1e-30)).max():.3g} times the bound"
        at += m


def sharing_pages(rng, n, lengths, kv_heads, d, page, elem):
    """Long sequences out of few pages, which several of them read."""
    paged = Paged(rng, [0], [1], kv_heads, d, page, elem, table_pages=60)
    paged.n, paged.lengths, paged.per = n, lengths, -(-max(lengths) // page)
    paged.table = rng.integers(0, paged.pages, (len(n), paged.per)).astype(np.int32)
    paged.starts_on, paged.lengths_on, paged.table_on = gpu(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)), gpu(np.array(lengths, np.int32)), gpu(paged.table)
    return paged


@pytest.mark.parametrize("d,page,elem,sequences,kv", [(64, 16, "f32", 200, 8), (64, 32, "bf16", 200, 8), (64, 24, "f32", 200, 8), (128, 16, "f32", 130, 8), (128, 64, "bf16", 200, 8),
                                                      (256, 16, "f32", 66, 8), (256, 20, "f32", 66, 8), (256, 16, "bf16", 66, 8), (200, 48, "f32", 66, 8)])
def test_long_sequences_among_many(here, case, d, page, elem, sequences, kv):
    """So many sequences that no keys are cut: a wavefront goes through up to 140 tiles of 16 keys, and the starts of its pages, 64 tiles at a
    time, are looked up anew."""
    case(f"attend long among many d {d} page {page} {elem}")
    rng = np.random.default_rng(39)
    lengths = [1 + 37 * s % 90 for s in range(sequences)]
    lengths[3], lengths[40], lengths[-1] = 8999, 4097, 5000
    paged = sharing_pages(rng, [1] * sequences, lengths, kv, d, page, elem)
    q = rng.standard_normal((sequences, kv, d)).astype(np.float32)
    got = attend(here, paged, gpu(q), max_tokens=1, max_keys=9000).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q)


@pytest.mark.parametrize("page,elem", [(16, "f32"), (48, "f32"), (24, "f32"), (16, "bf16"), (20, "bf16")])
@pytest.mark.parametrize("sequences,lengths", [(16, 1000), (16, 4000), (3, 20000)])
@pytest.mark.parametrize("d", [132, 256])
def test_many_tiles_of_wide_heads(here, case, page, elem, sequences, lengths, d):
    """Heads of more than 128 channels whose keys are cut into parts of 4 and more tiles a wavefront."""
    case(f"attend wide heads d {d} page {page} {elem} {sequences} of {lengths}")
    if elem == "bf16" and d == 132:
        d = 136  # a multiple of 8
    rng = np.random.default_rng(40)
    paged = sharing_pages(rng, [1] * sequences, [lengths - 31 * s for s in range(sequences)], 4, d, page, elem)
    q = rng.standard_normal((sequences, 8, d)).astype(np.float32)
    got = attend(here, paged, gpu(q), max_tokens=1, max_keys=lengths).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q)


@pytest.mark.parametrize("d,page,elem,kv", [(64, 16, "f32", 8), (64, 24, "f32", 8), (64, 64, "bf16", 8), (96, 16, "f32", 8), (128, 32, "f32", 8), (128, 16, "bf16", 8), (256, 16, "f32", 2),
                                            (256, 24, "bf16", 2)])
def test_pieces_behind_long_sequences_among_many(here, case, d, page, elem, kv):
    """Pieces whose blocks are enough uncut: a block of 128 rows goes through up to 125 tiles of 32 keys, and the starts of its pages, 32 tiles
    at a time, are looked up anew; so does one of 16 rows of wide heads."""
    case(f"attend pieces behind long sequences d {d} page {page} {elem}")
    rng = np.random.default_rng(41)
    n, lengths = [40] * 32, [45 + s for s in range(32)]
    lengths[5], lengths[20], lengths[-1] = 1100, 4000, 2500
    paged = sharing_pages(rng, n, lengths, kv, d, page, elem)
    q = rng.standard_normal((sum(n), kv, d)).astype(np.float32)
    got = attend(here, paged, gpu(q), max_tokens=40, max_keys=4000).cpu().numpy()
    here.sync()
    held_to_definition(got, paged, q)


@pytest.mark.parametrize("sequences,most", [(65, 3), (66, 1), (100, 9), (513, 4), (1000, 2)])
@pytest.mark.parametrize("d,elem", [(64, "f32"), (20, "bf16"), (7, "f32")])
def test_tokens_of_many_sequences_land_in_their_slots(here, case, sequences, most, d, elem):
    """More than 64 sequences with none to several rows each: a row's sequence is searched for."""
    rng = np.random.default_rng(sequences + most)
    n = [int(m) for m in rng.integers(0, most + 1, sequences)]
    lengths = [m + int(x) if m else int(x) for m, x in zip(n, rng.integers(0, 30, sequences))]
    test_tokens_land_in_their_slots(here, case, n, lengths, 3, 1, d, 6, 8, elem, "head", False, d == 64)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [[3], [70]])
@pytest.mark.parametrize("size", [1.5e38, 2.0 ** -90])
def test_values_near_the_ends_of_fp32(here, case, elem, d, n, size):
    """Two keys a row: their weights relative to the larger one add up to 2 at most, and 2 x 1.5e38 is finite."""
    case(f"attend values of {size:.3g} {elem} d {d} n {n}")
    rng = np.random.default_rng(42)
    paged = Paged(rng, n, [120], 1, d, 16, elem)
    paged.on[1].copy_(size * (2 * torch.rand(paged.on[1].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(42)) - 1))
    q = rng.standard_normal((n[0], 4, d)).astype(np.float32)
    got = attend(here, paged, gpu(q), window=2, scale=3.0 / d).cpu().numpy()
    here.sync()
    assert np.isfinite(got).all()
    held_to_definition(got, paged, q, window=2, scale=3.0 / d)
