"""Attention over the pages of a cache that their means select (ahip_kv_attention_sparse, ahip_kv_page_means) against its definition: the chosen pages exactly,
results within the bound of their sums."""
import math

import numpy as np
import pytest
import torch

from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_UNSUPPORTED, AltiusHipError
from decoder_more_oracle import attended_where, chosen_pages
from test_gpu_kv_cache import Paged, attend, gpu, here, raises_at_sync  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def page_means(paged):
    """The mean of every page's keys, rounded to fp32: [pages, heads, d]."""
    k = paged.views()[0].double()
    return k.sum(dim=2).div(paged.page).float()


class Sparse:
    """The means (NaN where a page is not full yet), the list of chosen pages and the call."""

    def __init__(self, ctx, paged, q, most, first=0, last=1, cap=0.0, max_tokens=0, max_keys=0, scale=None):
        self.paged, self.q, self.most, self.first, self.last = paged, q, most, first, last
        self.scale, self.cap = scale if scale is not None else 1 / math.sqrt(paged.d), cap
        self.means = torch.full((paged.pages, paged.kv_heads, paged.d), math.nan, device="cuda")
        full = page_means(paged)
        for s, (m, l) in enumerate(zip(paged.n, paged.lengths)):
            before = max(0, l - m) // paged.page
            pages = torch.from_numpy(paged.table[s, :before].astype(np.int64)).cuda()
            self.means[pages] = full[pages]
        self.chosen = torch.full((q.shape[0], paged.kv_heads, most), -5, device="cuda", dtype=torch.int32)
        self.out = torch.full_like(q, 5.0, memory_format=torch.contiguous_format)
        self.call = D.KvAttend(tokens=q.shape[0], q_heads=q.shape[1], q=q.data_ptr(), out=self.out.data_ptr(), q_strides=q.stride()[:2], out_strides=self.out.stride()[:2],
                               scale=self.scale, softcap=cap, max_tokens=max_tokens, max_keys=max_keys)
        self.sparse = D.KvSparse(means=self.means.data_ptr(), chosen=self.chosen.data_ptr(), most=most, first=first, last=last, page_stride=paged.kv_heads * paged.d,
                                 head_stride=paged.d)
        self.room = D.kv_attention_sparse_workspace(ctx, paged.cache(), paged.batch(), self.call, self.sparse)
        self.space = torch.full((self.room // 4 + 4,), math.nan, device="cuda")
        self.call.workspace, self.call.workspace_bytes = self.space.data_ptr(), self.room

    def run(self, ctx):
        torch.cuda.synchronize()
        ctx.kv_attention_sparse_raw(self.paged.cache(), self.paged.batch(), self.call, self.sparse)
        torch.cuda.synchronize()
        assert torch.isnan(self.space[self.room // 4:]).all()
        return self


def held_to_choice(got, q, but=()):
    paged, page = got.paged, got.paged.page
    out, chosen, means, full = got.out.cpu().numpy(), got.chosen.cpu().numpy(), got.means.cpu().numpy(), page_means(paged).cpu().numpy()
    at, group = 0, q.shape[1] // paged.kv_heads
    written = np.zeros(paged.pages, bool)
    for s, (m, l) in enumerate(zip(paged.n, paged.lengths)):
        rows = slice(at, at + m)
        at += m
        if s in but:
            continue
        of = paged.table[s][:l // page]
        written[of] = True
        np.testing.assert_array_equal(means[of], full[of])
        seen = np.zeros((m, paged.kv_heads, l), bool)
        for t in range(m):
            place = l - m + t
            for g in range(paged.kv_heads):
                want = chosen_pages(q[rows][t, g * group:(g + 1) * group], full[paged.table[s], g], place, page, got.most, got.first, got.last) if place >= 0 else np.empty(0, int)
                mine = chosen[rows][t, g]
                np.testing.assert_array_equal(mine[:len(want)], want, err_msg=f"sequence {s} row {t} head {g}")
                assert (mine[len(want):] == -1).all()
                for b in want:
                    seen[t, g, b * page:min(place + 1, (b + 1) * page)] = True
        k, v = paged.dense(s)
        want, bound, _, _ = attended_where(q[rows], k, v, seen, None, got.scale, got.cap, None)
        off = np.abs(out[rows] - want)
        assert (off <= bound + 1e-37).all(), f"sequence {s}: {(off / (bound + 1e-37)).max():.3g} times the bound"
    if not but:
        assert np.isnan(means[~written]).all(), "the mean of a page that is not full was written"
        assert (out[at:] == 5.0).all() and (chosen[at:] == -5).all(), "padding was written"


SHAPES = [  # n, lengths, heads, kv heads, d, page, type, order, most, first, last
    ([1], [1], 1, 1, 64, 16, "f32", "head", 1, 0, 1),
    ([1], [33], 4, 4, 64, 16, "f32", "head", 2, 0, 1),
    ([1, 1, 1], [16, 300, 1000], 8, 2, 128, 16, "f32", "slot", 5, 1, 2),
    ([1], [5000], 12, 2, 128, 16, "bf16", "head", 20, 1, 1),
    ([1], [40000], 4, 2, 64, 16, "f32", "head", 30, 2, 3),
    ([1, 1], [9001, 8], 32, 2, 128, 8, "bf16", "slot", 100, 0, 4),
    ([1, 0, 2, 0], [400, 12, 410, 0], 40, 1, 64, 16, "bf16", "slot", 7, 1, 2),
    ([3, 1], [70, 500], 40, 2, 96, 24, "f32", "head", 3, 0, 1),
    ([20, 5], [200, 300], 6, 3, 80, 8, "bf16", "head", 9, 2, 3),
    ([17], [17], 2, 2, 64, 4, "f32", "head", 3, 1, 1),
    ([1, 3], [1000, 700], 8, 1, 256, 48, "f32", "slot", 5, 1, 1),
    ([2], [3000], 4, 2, 200, 16, "bf16", "head", 11, 1, 1),
    ([40, 1], [333, 100], 5, 1, 20, 5, "f32", "slot", 6, 1, 2),
    ([130], [130], 4, 2, 64, 16, "f32", "head", 3, 1, 1),
    ([1] * 70, [15 * i + 1 for i in range(70)], 8, 4, 64, 16, "f32", "slot", 4, 1, 1),
    ([2] * 66 + [0, 5], [40 + 9 * i for i in range(66)] + [5, 900], 6, 6, 64, 16, "bf16", "head", 6, 0, 2),
    ([1, 1], [640, 640], 4, 1, 64, 64, "f32", "head", 4, 0, 4),
    ([1], [700], 7, 1, 64, 250, "f32", "slot", 2, 1, 1),
    ([1], [20000], 4, 1, 64, 1, "f32", "head", 64, 4, 8),
    ([1], [9000], 2, 1, 64, 1, "f32", "head", 8700, 4, 8),
    ([1, 2], [17000, 20], 1, 1, 8, 1, "bf16", "slot", 16384, 0, 3),
]


@pytest.mark.parametrize("n,lengths,heads,kv,d,page,elem,order,most,first,last", SHAPES)
@pytest.mark.parametrize("bounded", [False, True])
def test_rows_attend_to_chosen_pages(here, case, n, lengths, heads, kv, d, page, elem, order, most, first, last, bounded):  # noqa: F811
    case(f"sparse n {n[:5]} lengths {lengths[:5]} heads {heads}/{kv} d {d} page {page} {elem} {order} most {most} {first} {last} bounded {bounded}")
    rng = np.random.default_rng(d + page + len(n))
    paged = Paged(rng, n, lengths, kv, d, page, elem, order)
    q = (1.5 * rng.standard_normal((sum(n) + 2, heads, d))).astype(np.float32)
    bounds = dict(max_tokens=max(n), max_keys=max(lengths)) if bounded else {}
    got = Sparse(here, paged, gpu(q), most, first, last, cap=0.0 if bounded else 9.0, **bounds).run(here)
    here.sync()
    held_to_choice(got, q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n,length", [(1, 900), (1, 9000), (30, 700)])
def test_equal_scores_go_to_the_lowest_page(here, case, elem, n, length):  # noqa: F811
    """Pages of the same keys, in eight kinds; and one kind alone."""
    case(f"sparse, equal scores {elem} n {n} length {length}")
    rng = np.random.default_rng(3)
    for kinds in (8, 1):
        paged = Paged(rng, [n], [length], 2, 64, 16, elem)
        kind = rng.standard_normal((kinds, 2, 16, 64)).astype(np.float32)
        pages = gpu(kind[rng.integers(0, kinds, paged.per)]).to(paged.on[0].dtype)
        paged.views()[0][torch.from_numpy(paged.table[0].astype(np.int64)).cuda()] = pages
        q = rng.standard_normal((n, 4, 64)).astype(np.float32)
        got = Sparse(here, paged, gpu(q), 9, 1, 2).run(here)
        here.sync()
        held_to_choice(got, q)


@pytest.mark.parametrize("length", [600, 9000])
def test_scores_that_are_no_numbers_come_last(here, case, length):  # noqa: F811
    """Means of infinity and NaN, queries that are 0; what is not chosen does not reach the row."""
    case(f"sparse, NaN scores {length}")
    rng = np.random.default_rng(4)
    paged = Paged(rng, [1], [length], 1, 64, 16)
    k = paged.views()[0]
    for b, value in ((3, math.nan), (5, math.inf), (7, -math.inf), (11, math.nan)):
        k[int(paged.table[0, b]), 0, 4, 9] = value
    q = rng.standard_normal((1, 2, 64)).astype(np.float32)
    q[0, :, 9] = [-1.0, -2.0]  # page 5 scores minus infinity, page 7 infinity
    got = Sparse(here, paged, gpu(q), 6, 1, 1).run(here)
    here.sync()
    mine = got.chosen.cpu().numpy()[0, 0]
    full = page_means(paged).cpu().numpy()
    np.testing.assert_array_equal(mine, chosen_pages(q[0], full[paged.table[0], 0], length - 1, 16, 6, 1, 1))
    assert 7 in mine and not {3, 5, 11} & set(mine)
    q[:] = 0.0  # 0 x infinity is no number either: the others are all equal
    got = Sparse(here, paged, gpu(q), 6, 1, 1).run(here)
    here.sync()
    np.testing.assert_array_equal(got.chosen.cpu().numpy()[0, 0], [0, 1, 2, 4, 6, (length - 1) // 16])


def test_all_pages_are_plain_attention(here, case):  # noqa: F811
    case("sparse over all pages")
    rng = np.random.default_rng(5)
    for n, lengths in (([1, 1], [700, 50]), ([20, 3], [300, 90])):
        paged = Paged(rng, n, lengths, 2, 64, 16)
        q = gpu(rng.standard_normal((sum(n), 4, 64)).astype(np.float32))
        got, want = Sparse(here, paged, q, 50).run(here).out, attend(here, paged, q)
        here.sync()
        assert (got - want).abs().max() < 1e-5


@pytest.mark.parametrize("elem,d,page", [("f32", 64, 16), ("bf16", 128, 24), ("f32", 20, 5), ("bf16", 256, 1)])
def test_means_behind_a_prompt(here, case, elem, d, page):  # noqa: F811
    """ahip_kv_page_means writes the means of the pages that the rows fill, and no others."""
    case(f"page means {elem} d {d} page {page}")
    rng = np.random.default_rng(6)
    n, lengths = [100, 0, 3, 7], [130, 40, 48, 7]
    paged = Paged(rng, n, lengths, 2, d, page, elem)
    means = torch.full((paged.pages, 2, d), math.nan, device="cuda")
    torch.cuda.synchronize()
    here.kv_page_means_raw(paged.cache(), paged.batch(), D.KvSparse(means=means.data_ptr(), page_stride=2 * d, head_stride=d), sum(n), 100)
    here.sync()
    got, full, written = means.cpu().numpy(), page_means(paged).cpu().numpy(), np.zeros(paged.pages, bool)
    for s, (m, l) in enumerate(zip(n, lengths)):
        written[paged.table[s, (l - m) // page:l // page]] = m > 0
    np.testing.assert_array_equal(got[written], full[written])
    assert np.isnan(got[~written]).all()


@pytest.mark.parametrize("what", ["page", "length", "starts", "tokens", "keys", "short"])
def test_a_batch_that_does_not_fit_is_told_by_sparse_attention(here, case, what):  # noqa: F811
    case(f"sparse, bad {what}")
    rng = np.random.default_rng(7)
    n = [1, 3, 1]
    paged = Paged(rng, n, [100, 203, 60], 1, 64, 16)
    q = rng.standard_normal((5, 2, 64)).astype(np.float32)
    got = Sparse(here, paged, gpu(q), 4, max_tokens=2 if what == "tokens" else 0, max_keys=150 if what == "keys" else 0)
    if what == "page":
        paged.table_on[1, 2] = paged.pages
    elif what == "length":
        paged.lengths_on[1] = paged.per * 16 + 1
    elif what == "starts":
        paged.starts_on[2] = 0
    elif what == "short":
        paged.lengths_on[1] = 2  # fewer tokens than rows: the first row sees nothing
    got.run(here)
    if what == "short":
        here.sync()
        assert (got.out[1] == 0).all() and (got.chosen[1] == -1).all()
        paged.lengths[1] = 2
        held_to_choice(got, q, but=(1,))
        return
    raises_at_sync(here)
    if what != "starts":
        held_to_choice(got, q, but=(1,))
    if what not in ("page", "starts"):
        assert (got.out[1:4] == 5.0).all() and (got.chosen[1:4] == -5).all()


def test_sparse_attention_that_is_refused(here, case):  # noqa: F811
    case("sparse refusals")
    rng = np.random.default_rng(8)
    paged = Paged(rng, [1], [100], 1, 64, 16)
    q = gpu(rng.standard_normal((1, 2, 64)).astype(np.float32))
    for code, on, change in ((ERR_UNSUPPORTED, "call", dict(causal=0)), (ERR_UNSUPPORTED, "call", dict(window=5)), (ERR_UNSUPPORTED, "call", dict(slopes=q.data_ptr())),
                             (ERR_UNSUPPORTED, "call", dict(prefix=q.data_ptr())), (ERR_UNSUPPORTED, "call", dict(first_keys=q.data_ptr())), (ERR_ARG, "sparse", dict(last=0)),
                             (ERR_ARG, "sparse", dict(first=-1)), (ERR_ARG, "sparse", dict(first=4)), (ERR_ARG, "sparse", dict(most=0)), (ERR_ARG, "sparse", dict(means=None)),
                             (ERR_ARG, "sparse", dict(chosen=None)), (ERR_ARG, "sparse", dict(page_stride=-4)), (ERR_UNSUPPORTED, "sparse", dict(head_stride=62)),
                             (ERR_UNSUPPORTED, "sparse", dict(most=1 << 30)), (ERR_ARG, "call", dict(workspace_bytes=0)), (ERR_ARG, "call", dict(q=None))):
        got = Sparse(here, paged, q, 4)
        for name, x in change.items():
            setattr(getattr(got, on), name, x)
        with pytest.raises(AltiusHipError) as e:
            here.kv_attention_sparse_raw(paged.cache(), paged.batch(), got.call, got.sparse)
        assert e.value.code == code, change
        here.sync()
        assert (got.out == 5.0).all() and (got.chosen == -5).all()


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("start", [30, 9000])
def test_recorded_steps_over_chosen_pages(here, case, elem, start):  # noqa: F811
    """One recorded call, replayed while two sequences grow token by token past the ends of their pages, the means kept by the calls alone."""
    case(f"sparse, recorded {elem} start {start}")
    rng = np.random.default_rng(9)
    paged = Paged(rng, [1, 1], [start, start - 9], 2, 64, 8, elem, table_pages=start // 8 + 5)
    q = torch.zeros((2, 4, 64), device="cuda")
    stream = torch.cuda.Stream()
    got = Sparse(here, paged, q, 6, 1, 1, max_tokens=1, max_keys=start + 32)
    with D.Context(0, stream=stream.cuda_stream) as recorded:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            recorded.kv_attention_sparse_raw(paged.cache(), paged.batch(), got.call, got.sparse)
        for turn in range(20):
            new = rng.standard_normal((2, 4, 64)).astype(np.float32)
            q.copy_(gpu(new))
            paged.lengths_on.copy_(gpu(np.array(paged.lengths, np.int32)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            recorded.sync()
            held_to_choice(got, new)
            paged.lengths = [l + 1 for l in paged.lengths]
