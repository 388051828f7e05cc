"""Attention that adds up what it gave each key (ahip_kv_attention_mass) and the choice of the keys that stay (ahip_kv_evict) against their definitions."""
import math

import numpy as np
import pytest
import torch

from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_UNSUPPORTED, AltiusHipError
from decoder_more_oracle import attended_where, stays
from decoder_oracle import STEP, ranges
from test_gpu_kv_cache import Paged, attend, gpu, here, raises_at_sync  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


class Mass:
    """The history of a cache (masses spread over ten powers of two, positions -3 where nothing was written) and one call."""

    def __init__(self, ctx, paged, q, rng, decay=1.0, own_positions=True, max_tokens=0, max_keys=0, causal=True, window=0, cap=0.0, slopes=None, prefix=None, first=None, scale=None):
        self.paged, self.q, self.decay = paged, q, decay
        shape = (paged.pages, paged.kv_heads, paged.page)
        self.before = np.exp2(10 * rng.random(shape) - 5).astype(np.float32)
        self.mass, self.positions = gpu(self.before), torch.full(shape, -3, device="cuda", dtype=torch.int32)
        self.rows = gpu(rng.integers(0, 1 << 30, q.shape[0]).astype(np.int32)) if own_positions else None
        self.history = D.KvHistory(mass=self.mass.data_ptr(), positions=self.positions.data_ptr(), page_stride=paged.kv_heads * paged.page, head_stride=paged.page)
        self.out = torch.full_like(q, 5.0, memory_format=torch.contiguous_format)
        self.masks = dict(causal=causal, window=window, prefix=prefix, first=first)
        self.scores = dict(cap=cap, slopes=slopes, scale=scale if scale is not None else 1 / math.sqrt(paged.d))
        self.call = D.KvAttend(tokens=q.shape[0], q_heads=q.shape[1], q=q.data_ptr(), out=self.out.data_ptr(), q_strides=q.stride()[:2], out_strides=self.out.stride()[:2],
                               scale=self.scores["scale"], softcap=cap, causal=int(causal), window=window, max_tokens=max_tokens, max_keys=max_keys)
        self.keep = [None if x is None else gpu(x) for x in (slopes, prefix, first)]
        self.call.slopes, self.call.prefix, self.call.first_keys = (None if x is None else x.data_ptr() for x in self.keep)
        self.room = D.kv_attention_mass_workspace(ctx, paged.cache(), paged.batch(), self.call)
        self.space = torch.full((self.room // 4 + 4,), math.nan, device="cuda")
        self.call.workspace, self.call.workspace_bytes = self.space.data_ptr(), self.room

    def run(self, ctx):
        torch.cuda.synchronize()
        ctx.kv_attention_mass_raw(self.paged.cache(), self.paged.batch(), self.call, self.history, self.decay, None if self.rows is None else self.rows.data_ptr())
        torch.cuda.synchronize()
        assert torch.isnan(self.space[self.room // 4:]).all()
        return self


def held_to_masses(got, q, but=()):
    paged = got.paged
    group = q.shape[1] // paged.kv_heads
    out, mass, positions = got.out.cpu().numpy(), got.mass.cpu().numpy(), got.positions.cpu().numpy()
    rows = None if got.rows is None else got.rows.cpu().numpy()
    touched, placed = np.zeros(mass.shape, bool), np.zeros(mass.shape, bool)
    at = 0
    for s, (m, l) in enumerate(zip(paged.n, paged.lengths)):
        mine = slice(at, at + m)
        at += m
        if m == 0 or s in but:
            continue
        k, v = paged.dense(s)
        low, high, place = ranges(m, l, got.masks["causal"], got.masks["window"], None if got.masks["prefix"] is None else got.masks["prefix"][s],
                                  None if got.masks["first"] is None else got.masks["first"][mine])
        key = np.arange(l)
        seen = (key >= low[:, None]) & (key < high[:, None])
        want, bound, weights, off = attended_where(q[mine], k, v, seen, place[:, None] - key, got.scores["scale"], got.scores["cap"], got.scores["slopes"])
        assert (np.abs(out[mine] - want) <= bound + 1e-37).all()
        page, slot = paged.table[s][key // paged.page], key % paged.page
        fresh = key >= l - m
        for g in range(paged.kv_heads):
            given = weights[:, g * group:(g + 1) * group].sum((0, 1))
            kept = np.where(fresh, 0.0, got.decay * got.before[page, g, slot].astype(np.float64) if got.decay else 0.0)
            # Each weight's own error, a step for each of the sum's terms, the decay's product and the last sum; weights that fp32 flushes.
            most = off[:, g * group:(g + 1) * group].sum((0, 1)) + (m * group + 4) * STEP * (given + kept) + m * group * 2.0 ** -120
            error = np.abs(mass[page, g, slot] - (given + kept))
            assert (error <= most).all(), f"sequence {s} head {g}: {(error / most).max():.3g} times the bound"
            touched[page, g, slot] = True
            placed[page[fresh], g, slot[fresh]] = True
            np.testing.assert_array_equal(positions[page[fresh], g, slot[fresh]], key[fresh] if rows is None else rows[mine][key[fresh] - (l - m)])
    if not but:
        np.testing.assert_array_equal(mass[~touched], got.before[~touched])
        assert (positions[~placed] == -3).all() and (out[at:] == 5.0).all()


SHAPES = [  # n, lengths, heads, kv heads, d, page, type, order
    ([1], [1], 1, 1, 64, 16, "f32", "head"),
    ([1], [77], 12, 12, 64, 16, "f32", "head"),
    ([1, 1, 1], [1, 300, 33], 8, 2, 128, 16, "f32", "slot"),
    ([1, 1, 1], [5, 31, 1000], 8, 1, 128, 32, "bf16", "head"),
    ([1], [9000], 7, 1, 128, 48, "bf16", "slot"),
    ([1, 0, 2, 0], [40, 12, 41, 0], 40, 1, 64, 16, "bf16", "slot"),
    ([3, 1], [70, 500], 40, 2, 96, 24, "f32", "head"),
    ([1, 1], [100, 64], 4, 4, 256, 16, "f32", "head"),
    ([20, 1], [200, 129], 16, 2, 256, 64, "bf16", "slot"),
    ([1] * 70, [5 * i + 1 for i in range(69)] + [1500], 8, 4, 64, 16, "f32", "slot"),
    ([1, 2], [33, 50], 3, 1, 20, 5, "f32", "slot"),
    ([65, 1, 130], [65, 700, 200], 4, 2, 64, 16, "f32", "head"),
    ([128, 3], [128, 260], 2, 1, 96, 24, "bf16", "head"),
    ([257], [400], 8, 1, 128, 250, "f32", "slot"),
    ([600], [600], 4, 1, 64, 16, "bf16", "head"),
    ([70], [90], 2, 2, 200, 32, "f32", "head"),
    ([5, 40, 1], [3, 25, 0], 4, 2, 64, 16, "f32", "slot"),
    ([300, 2], [280, 1], 8, 2, 128, 16, "bf16", "head"),
]


@pytest.mark.parametrize("n,lengths,heads,kv,d,page,elem,order", SHAPES)
@pytest.mark.parametrize("plain", [True, False])
def test_keys_are_given_their_weights(here, case, n, lengths, heads, kv, d, page, elem, order, plain):  # noqa: F811
    case(f"mass n {n[:5]} lengths {lengths[:5]} heads {heads}/{kv} d {d} page {page} {elem} {order} plain {plain}")
    rng = np.random.default_rng(d + page + len(n))
    paged = Paged(rng, n, lengths, kv, d, page, elem, order)
    q = (1.5 * rng.standard_normal((sum(n) + 2, heads, d))).astype(np.float32)
    options = dict(decay=0.0, max_tokens=max(n), max_keys=max(lengths)) if plain else dict(
        decay=0.75, own_positions=False, window=max(2, max(lengths) // 3), cap=20.0, slopes=(2.0 ** -np.arange(1, heads + 1) * 0.5).astype(np.float32),
        first=rng.integers(-3, max(lengths), sum(n) + 2).astype(np.int32), prefix=rng.integers(0, 30, len(n)).astype(np.int32))
    got = Mass(here, paged, gpu(q), rng, **options).run(here)
    here.sync()
    held_to_masses(got, q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("options", [dict(causal=False), dict(window=1), dict(window=40), dict(causal=False, window=9), dict(prefix=np.array([0, 60, 1000], np.int32)),
                                     dict(cap=2.0), dict(scale=0.0), dict(scale=-0.2), dict(slopes=np.array([0.0, 0.5, 0.01, -0.02], np.float32))])
@pytest.mark.parametrize("n", [[1, 2, 1], [90, 33, 64]])
def test_each_mask_and_bias_of_masses(here, case, elem, options, n):  # noqa: F811
    case(f"mass {elem} {sorted(options)} n {n}")
    rng = np.random.default_rng(17)
    paged = Paged(rng, n, [99, 50, 64], 2, 64, 16, elem)
    q = rng.standard_normal((sum(n), 4, 64)).astype(np.float32)
    got = Mass(here, paged, gpu(q), rng, **options).run(here)
    here.sync()
    held_to_masses(got, q)


@pytest.mark.parametrize("n,lengths", [([1], [50000]), ([1, 1], [7000, 300]), ([40, 300], [900, 1200]), ([1000], [1000])])
@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_long_sums_of_weights(here, case, n, lengths, elem):  # noqa: F811
    """The weights of each row add up to 1, whatever its keys; the same call twice gives the same bits, and attention those of ahip_kv_attention."""
    case(f"mass n {n} lengths {lengths} {elem}")
    rng = np.random.default_rng(18)
    paged = Paged(rng, n, lengths, 2, 64, 16, elem)
    q = gpu(rng.standard_normal((sum(n), 6, 64)).astype(np.float32))
    got, again = (Mass(here, paged, q, np.random.default_rng(1), decay=0.0).run(here) for _ in range(2))
    here.sync()
    assert torch.equal(got.mass, again.mass)
    assert torch.equal(got.out, attend(here, paged, q))
    mass = got.mass.cpu().numpy().astype(np.float64)
    for s, (m, l) in enumerate(zip(n, lengths)):
        key = np.arange(l)
        total = mass[paged.table[s][key // 16], :, key % 16].sum(0)
        # A row's weights are off by (2 x its worst score + 2 x its keys + 8) steps at most: scores here stay below 8.
        assert (np.abs(total - 3 * m) <= 3 * m * (2 * 68 * 64 + 2 * l + 8) * STEP).all()


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n", [[1, 1], [40, 70]])
def test_slots_that_no_row_sees_do_not_matter(here, case, elem, n):  # noqa: F811
    """Infinities and NaN in slots behind the sequences, in masked keys, and in masses that a decay of 0 does not read."""
    case(f"mass, slots not seen {elem} n {n}")
    rng = np.random.default_rng(19)
    paged = Paged(rng, n, [95, 75], 1, 64, 16, elem)
    q = rng.standard_normal((sum(n), 2, 64)).astype(np.float32)
    first = np.full(sum(n), 20, np.int32)
    for x in paged.views():
        for s, l in enumerate(paged.lengths):
            x[int(paged.table[s, l // 16]), :, l % 16:] = math.nan
            x[int(paged.table[s, 0]), :, 3] = math.inf
            x[int(paged.table[s, 0]), :, 4] = math.nan
    got = Mass(here, paged, gpu(q), rng, decay=0.0, first=first)
    got.mass.fill_(math.nan)
    got.run(here)
    here.sync()
    mass, at = got.mass.cpu().numpy(), 0
    for s, (m, l) in enumerate(zip(n, paged.lengths)):
        k, v = paged.dense(s)
        low, high, place = ranges(m, l, True, 0, None, first[at:at + m])
        key = np.arange(l)
        _, _, weights, off = attended_where(q[at:at + m], k, v, (key >= low[:, None]) & (key < high[:, None]), None, 1 / 8, 0.0, None)
        given = weights.sum((0, 1))
        mine = mass[paged.table[s][key // 16], 0, key % 16]
        assert (np.abs(mine - given) <= off.sum((0, 1)) + (2 * m + 4) * STEP * given + 1e-30).all() and (mine[:20] == 0).all()
        at += m


@pytest.mark.parametrize("n", [[1], [50]])
def test_infinite_keys_that_are_seen(here, case, n):  # noqa: F811
    """A score of minus infinity gives a weight of 0, one of infinity makes all of its row's NaN, as the softmax has it."""
    case(f"mass, infinite keys n {n}")
    rng = np.random.default_rng(20)
    for elem in ("f32", "bf16"):
        paged = Paged(rng, n, [90], 1, 64, 16, elem)
        paged.views()[0][int(paged.table[0, 1]), 0, 2, 5] = math.inf
        q = rng.standard_normal((n[0], 2, 64)).astype(np.float32)
        q[..., 5] = -np.abs(q[..., 5]) - 0.1
        got = Mass(here, paged, gpu(q), rng, decay=0.0).run(here)
        here.sync()
        mass = got.mass.cpu().numpy()
        assert mass[paged.table[0, 1], 0, 2] == 0 and abs(mass[paged.table[0][np.arange(90) // 16], 0, np.arange(90) % 16].sum() - 2 * n[0]) < 1e-3
        q[..., 5] *= -1
        got = Mass(here, paged, gpu(q), rng, decay=0.0).run(here)
        here.sync()
        assert np.isnan(got.mass.cpu().numpy()[paged.table[0][np.arange(90 - n[0]) // 16], 0, np.arange(90 - n[0]) % 16]).all()


def test_masses_that_are_refused_and_batches_that_do_not_fit(here, case):  # noqa: F811
    case("mass refusals")
    rng = np.random.default_rng(21)
    paged = Paged(rng, [1, 2], [100, 40], 1, 64, 16)
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    q = gpu(x)
    for decay in (-0.1, 1.5, math.nan):
        got = Mass(here, paged, q, rng, decay=decay)
        with pytest.raises(AltiusHipError) as e:
            got.run(here)
        assert e.value.code == ERR_ARG
    for on, change, code in (("history", dict(mass=None), ERR_ARG), ("history", dict(page_stride=-1), ERR_ARG), ("call", dict(workspace_bytes=8), ERR_ARG), ("call", dict(workspace=None), ERR_ARG),
                             ("call", dict(out=None), ERR_ARG), ("call", dict(q=q.data_ptr() + 4), ERR_UNSUPPORTED)):
        got = Mass(here, paged, q, rng)
        for name, v in change.items():
            setattr(getattr(got, on), name, v)
        with pytest.raises(AltiusHipError) as e:
            got.run(here)
        assert e.value.code == code
        here.sync()
        assert (got.out == 5.0).all() and (got.mass == gpu(got.before)).all()
    for what in ("length", "page"):
        paged = Paged(rng, [1, 2], [100, 40], 1, 64, 16)
        got = Mass(here, paged, q, rng, decay=0.5)
        if what == "length":
            paged.lengths_on[1] = 16 * paged.per + 1
        else:
            paged.table_on[1, 1] = -1
        got.run(here)
        raises_at_sync(here)
        held_to_masses(got, x, but=(1,))


def test_a_history_without_positions(here, case):  # noqa: F811
    case("mass without positions")
    rng = np.random.default_rng(22)
    paged = Paged(rng, [2], [40], 2, 64, 16)
    got = Mass(here, paged, gpu(rng.standard_normal((2, 2, 64)).astype(np.float32)), rng)
    got.history.positions = None
    got.run(here)
    here.sync()
    assert (got.positions == -3).all()


# ---- eviction --------------------------------------------------------------------------------------------------------

class Evict:
    def __init__(self, rng, lengths, kv, page, budget, recent, first, most=None, max_keys=0, spare=2):
        per = max(1, -(-max(lengths) // page))
        self.lengths, self.kv, self.page, self.budget, self.recent, self.first = lengths, kv, page, budget, recent, first
        pages = per * len(lengths) + spare
        self.pages = pages
        self.table = rng.permutation(pages)[:per * len(lengths)].reshape(len(lengths), per).astype(np.int32)
        self.mass = np.exp2(20 * rng.random((pages, kv, page)) - 10).astype(np.float32)
        self.positions = rng.permutation(pages * kv * page).reshape(pages, kv, page).astype(np.int32)
        self.most = most if most is not None else max(0, min(budget, (max_keys or per * page) - budget))
        self.max_keys = max_keys

    in_place = False

    def run(self, ctx, overlap=0):
        on = dict(mass=gpu(self.mass), positions=gpu(self.positions), table=gpu(self.table), lengths=gpu(np.array(self.lengths, np.int32)))
        self.lists = [torch.full((len(self.lengths), self.kv, max(1, self.most)), -9, device="cuda", dtype=torch.int32) for _ in range(2)]
        self.counts, self.kept = torch.full((len(self.lengths), self.kv), -9, device="cuda", dtype=torch.int32), torch.full((len(self.lengths),), -9, device="cuda", dtype=torch.int32)
        if self.in_place:
            self.kept = on["lengths"]
        cache = D.KvCache(kv_heads=self.kv, head_size=8, page_size=self.page, pages=self.pages)
        batch = D.KvBatch(sequences=len(self.lengths), table_pages=self.table.shape[1], table_stride=self.table.shape[1], lengths=on["lengths"].data_ptr(), page_table=on["table"].data_ptr())
        history = D.KvHistory(mass=on["mass"].data_ptr(), positions=on["positions"].data_ptr(), page_stride=self.kv * self.page, head_stride=self.page)
        eviction = D.KvEviction(budget=self.budget, recent=self.recent, first=self.first, most=self.most, max_keys=self.max_keys, sources=self.lists[0].data_ptr(),
                                targets=self.lists[1].data_ptr(), counts=self.counts.data_ptr(), lengths=self.kept.data_ptr() + overlap)
        torch.cuda.synchronize()
        ctx.kv_evict_raw(cache, batch, history, eviction)
        torch.cuda.synchronize()
        return self

    def held(self, but=()):
        sources, targets, counts, kept = (x.cpu().numpy() for x in (*self.lists, self.counts, self.kept))
        for s, l in enumerate(self.lengths):
            if s in but:
                assert (counts[s] == 0).all() and kept[s] == -9
                continue
            assert kept[s] == min(l, self.budget)
            at = np.arange(l)
            page, slot = self.table[s][at // self.page], at % self.page
            for g in range(self.kv):
                keep = stays(self.mass[page, g, slot], self.positions[page, g, slot], self.budget, self.recent, self.first) if l > self.budget else np.ones(l, bool)
                movers, holes = np.flatnonzero(keep[self.budget:]) + self.budget, np.flatnonzero(~keep[:self.budget])
                assert counts[s, g] == len(movers) == len(holes)
                np.testing.assert_array_equal(sources[s, g, :len(movers)], movers)
                np.testing.assert_array_equal(targets[s, g, :len(holes)], holes)
                assert (sources[s, g, len(movers):] == -9).all() and (targets[s, g, len(holes):] == -9).all()


EVICTIONS = [  # lengths, kv heads, page, budget, recent, first
    ([10], 1, 4, 5, 0, 0),
    ([1, 2, 3, 0, 64, 65, 63], 2, 16, 64, 8, 2),
    ([1025] * 9, 4, 16, 1024, 256, 4),
    ([2000, 700, 701, 5], 2, 24, 700, 350, 350),
    ([5000], 3, 250, 1, 0, 0),
    ([5000], 1, 1, 1, 1, 0),
    ([5000, 4097], 2, 64, 4096, 0, 0),
    ([40000, 33000], 2, 64, 3000, 100, 4),
    ([70000], 1, 16, 35000, 100, 4),
    ([100] * 70, 2, 8, 50, 10, 1),
]


@pytest.mark.parametrize("lengths,kv,page,budget,recent,first", EVICTIONS)
@pytest.mark.parametrize("masses", ["spread", "few", "equal", "odd"])
def test_who_stays(here, case, lengths, kv, page, budget, recent, first, masses):  # noqa: F811
    case(f"evict lengths {lengths[:5]} kv {kv} page {page} budget {budget} recent {recent} first {first} masses {masses}")
    rng = np.random.default_rng(budget + page)
    e = Evict(rng, lengths, kv, page, budget, recent, first, max_keys=max(lengths))
    if masses == "few":  # many equal ones
        e.mass = rng.integers(0, 5, e.mass.shape).astype(np.float32)
    elif masses == "equal":
        e.mass[:] = 0.25
    elif masses == "odd":
        values = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -np.nan, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0, np.nextafter(np.float32(1), np.float32(2))], np.float32)
        e.mass = values[rng.integers(0, len(values), e.mass.shape)]
    e.run(here)
    here.sync()
    e.held()


def test_positions_at_the_ends_of_32_bits_and_equal_ones(here, case):  # noqa: F811
    case("evict, positions")
    rng = np.random.default_rng(1)
    for values in ([-(1 << 31), (1 << 31) - 1, 0, 5], [7], [-5, -4]):
        e = Evict(rng, [300, 301], 2, 16, 100, 60, 40)
        e.positions = np.array(values, np.int64)[rng.integers(0, len(values), e.positions.shape)].astype(np.int32)
        e.run(here)
        here.sync()
        e.held()


@pytest.mark.parametrize("what", ["length", "length_negative", "bound", "page"])
def test_evictions_that_do_not_fit_are_told(here, case, what):  # noqa: F811
    case(f"evict, bad {what}")
    rng = np.random.default_rng(2)
    e = Evict(rng, [300, 301, 250], 2, 16, 100, 20, 4, max_keys=300 if what == "bound" else 0)
    if what == "length":
        e.lengths = [300, 16 * 19 + 1, 250]
    elif what == "length_negative":
        e.lengths = [300, -1, 250]
    elif what == "page":
        e.table[1, 3] = e.pages
    e.run(here)
    raises_at_sync(here)
    if what != "page":
        e.held(but=(1,))


def test_evictions_that_are_refused(here, case):  # noqa: F811
    case("evict refusals")
    rng = np.random.default_rng(3)
    for change in (dict(budget=0), dict(budget=-5), dict(recent=-1), dict(first=-1), dict(recent=60, first=41), dict(most=99)):
        e = Evict(rng, [300], 2, 16, 100, 20, 4)
        for name, x in change.items():
            setattr(e, name, x)
        with pytest.raises(AltiusHipError) as error:
            e.run(here)
        assert error.value.code == ERR_ARG
    here.sync()


@pytest.mark.parametrize("longest", [150, 5000])
def test_new_lengths_in_the_place_of_the_old_ones(here, case, longest):  # noqa: F811
    """Every head of a sequence goes by the old length, however late its block starts: many more blocks than run at once."""
    case(f"evict in place, {longest}")
    rng = np.random.default_rng(5)
    lengths = [int(x) for x in rng.integers(90, longest + 1, 150)]
    e = Evict(rng, lengths, 32, 50, 100, 20, 4, max_keys=longest)
    e.in_place = True
    e.run(here)
    here.sync()
    e.held()
    with pytest.raises(AltiusHipError) as error:
        e.in_place = 1
        e.run(here, overlap=4)
    assert error.value.code == ERR_ARG


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_a_cache_that_is_kept_within_its_budget(here, case, elem):  # noqa: F811
    """Tokens are appended at their positions and attend with masses, and whenever a text is longer than its budget its slots are chosen and moved; recorded once and
    replayed.  A model of the same cache on the host holds what each head should hold: keys, values, masses and positions, and attention over them."""
    case(f"evict, recorded {elem}")
    rng = np.random.default_rng(4)
    kv, heads, d, page, budget, recent, first, texts = 2, 4, 64, 8, 40, 12, 2, 2
    paged = Paged(rng, [1] * texts, [0] * texts, kv, d, page, elem, table_pages=6, fill=0.0)
    packed, q, out = torch.zeros((texts, heads + 2 * kv, d), device="cuda"), torch.zeros((texts, heads, d), device="cuda"), torch.zeros((texts, heads, d), device="cuda")
    positions = torch.zeros(texts, dtype=torch.int32, device="cuda")
    shape = (paged.pages, kv, page)
    mass, slots = torch.full(shape, math.nan, device="cuda"), torch.full(shape, -3, device="cuda", dtype=torch.int32)
    history = D.KvHistory(mass=mass.data_ptr(), positions=slots.data_ptr(), page_stride=kv * page, head_stride=page)
    call = D.KvAttend(tokens=texts, q_heads=heads, q=q.data_ptr(), out=out.data_ptr(), q_strides=q.stride()[:2], out_strides=out.stride()[:2], scale=1 / 8, max_tokens=1, max_keys=48)
    room = D.kv_attention_mass_workspace(here, paged.cache(), paged.batch(), call)
    space = torch.full((room // 4 + 4,), math.nan, device="cuda")
    call.workspace, call.workspace_bytes = space.data_ptr(), room
    fields = D.KvTokens(tokens=texts, k=packed[:, heads:].data_ptr(), v=packed[:, heads + kv:].data_ptr(), k_strides=packed.stride()[:2], v_strides=packed.stride()[:2], q_heads=heads,
                        q=packed.data_ptr(), q_out=q.data_ptr(), q_strides=packed.stride()[:2], q_out_strides=q.stride()[:2], positions=positions.data_ptr())
    sources, targets = (torch.zeros((texts, kv, 8), dtype=torch.int32, device="cuda") for _ in range(2))
    counts = torch.zeros((texts, kv), dtype=torch.int32, device="cuda")
    eviction = D.KvEviction(budget=budget, recent=recent, first=first, most=8, max_keys=48, sources=sources.data_ptr(), targets=targets.data_ptr(), counts=counts.data_ptr(),
                            lengths=paged.lengths_on.data_ptr())
    moves = D.KvMoves(sources=sources.data_ptr(), targets=targets.data_ptr(), counts=counts.data_ptr(), strides=(kv * 8, 8), count_strides=(kv, 1), most=8, apart=1)
    model = [[[] for _ in range(kv)] for _ in range(texts)]  # of each head: (position, key, value, mass) by place
    stream = torch.cuda.Stream()
    with D.Context(0, stream=stream.cuda_stream) as recorded:
        torch.cuda.synchronize()
        step, thin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(step, stream=stream):
            recorded.kv_append_raw(paged.cache(), paged.batch(), fields)
            recorded.kv_attention_mass_raw(paged.cache(), paged.batch(), call, history, 1.0, positions.data_ptr())
        with torch.cuda.graph(thin, stream=stream):
            recorded.kv_evict_raw(paged.cache(), paged.batch(), history, eviction)
            recorded.kv_move_raw(paged.cache(), paged.batch(), moves, history)
        for position in range(90):
            x = rng.standard_normal((texts, heads + 2 * kv, d)).astype(np.float32)
            packed.copy_(gpu(x)), positions.fill_(position)
            paged.lengths_on += 1
            torch.cuda.synchronize()
            step.replay()
            torch.cuda.synchronize()
            results, masses = out.cpu().numpy(), mass.cpu().numpy()
            for s in range(texts):
                for g in range(kv):
                    held = gpu(x[s, heads + g::kv][:2]).to(torch.bfloat16 if elem == "bf16" else torch.float32).float().cpu().numpy()
                    model[s][g].append([position, held[0], held[1], 0.0])
                    k, v = (np.stack([t[i] for t in model[s][g]])[:, None] for i in (1, 2))
                    want, bound, weights, off = attended_where(x[s:s + 1, g * 2:g * 2 + 2], k, v, np.ones((1, len(k)), bool), None, 1 / 8, 0.0, None)
                    assert (np.abs(results[s, g * 2:g * 2 + 2] - want[0]) <= bound[0]).all()
                    at = np.arange(len(k))
                    mine = masses[paged.table[s][at // page], g, at % page]
                    then = np.array([t[3] for t in model[s][g]]) + weights.sum((0, 1))
                    assert (np.abs(mine - then) <= off.sum((0, 1)) + 6 * STEP * then).all()
                    for t, m in zip(model[s][g], mine):
                        t[3] = m  # the model goes on from the kernel's own
            if len(model[0][0]) < budget + (5 if position % 2 else 1):
                continue
            thin.replay()
            torch.cuda.synchronize()
            remembered, keys = slots.cpu().numpy(), paged.views()[0].float().cpu().numpy()
            assert (paged.lengths_on.cpu().numpy() == budget).all()
            for s in range(texts):
                for g in range(kv):
                    tokens = model[s][g]
                    keep = stays(np.array([t[3] for t in tokens], np.float32), np.array([t[0] for t in tokens]), budget, recent, first)
                    movers, holes = np.flatnonzero(keep[budget:]) + budget, np.flatnonzero(~keep[:budget])
                    for a, b in zip(movers, holes):
                        tokens[b] = list(tokens[a])
                    del tokens[budget:]
                    at = np.arange(budget)
                    np.testing.assert_array_equal(remembered[paged.table[s][at // page], g, at % page], [t[0] for t in tokens])
                    np.testing.assert_array_equal(keys[paged.table[s][at // page], g, at % page], np.stack([t[1] for t in tokens]))
                    assert {0, 1} | set(range(position - recent + 1, position + 1)) <= {t[0] for t in tokens}
        recorded.sync()
