"""The operators around a paged cache at sizes that choose among their kernels or that a sum feels: sums of many weights, more rows than a grid of
large blocks has twice, positions at the ends of 32 bits; weights of few rows that are computed again because their scores would not fit the workspace, scores of many
pages for wide heads."""
import math

import numpy as np
import pytest
import torch

from altius_amd import device as D
from altius_amd._lib import ERR_ARG, AltiusHipError
from decoder_oracle import STEP
from test_gpu_kv_cache import Paged, gpu, held_to_definition, here  # noqa: F401 (a fixture)
from test_gpu_kv_mass import Evict, Mass, held_to_masses
from test_gpu_kv_sparse import Sparse, held_to_choice, page_means

pytestmark = pytest.mark.gpu


def test_masses_of_many_rows_are_summed_to_fp32(here, case):  # noqa: F811
    """A prompt of 4096 tokens, 4 heads a head of keys.  Key 0 is given a weight of 1 by the first 8800 rows and 1 / p by each row at place p - 1 from then on, between a
    quarter of a step and a step of what it has by then: a sum in fp32 that takes one weight after the other rounds each of them to nothing or to a whole step, 2300 steps
    of the sum in all.  (All other scores are 0, so that weights are off by 2 steps at most.)"""
    case("sums of 16384 weights a key")
    tokens, early, kv, heads, d = 4096, 2200, 48, 192, 4
    rng = np.random.default_rng(40)
    paged = Paged(rng, [tokens], [tokens], kv, d, 16, fill=0.0, spare_pages=0)
    paged.on[0][int(paged.table[0, 0]), :, 0, 0] = 1.0
    q = torch.zeros((tokens, heads, d), device="cuda")
    q[:early, :, 0] = 40.0
    got = Mass(here, paged, q, rng, decay=0.0, scale=1.0).run(here)
    here.sync()
    # Key 0 of the first rows has a weight of 1 / (1 + (p - 1) e^-40), which is 1 to 2e-14; the other keys 2e-14 together, which is nothing beside what follows.
    late = 4.0 / np.arange(early + 1, tokens + 1)
    behind = np.concatenate([np.cumsum(late[::-1])[::-1], [0.0]])  # of the late rows from this one on
    want = np.array([behind[max(0, key - early)] for key in range(tokens)])
    want[0] += 4 * early
    mass = got.mass.cpu().numpy()[paged.table[0][np.arange(tokens) // 16], :, np.arange(tokens) % 16].astype(np.float64)
    # 2 steps a weight; 16 for a partial sum of as many weights, 2 for a sum that carries its rounding along, 1 for the two halves of a row tile and up to 15 for parts
    # of the rows.
    assert (np.abs(mass - want[:, None]) <= (2 + 16 + 2 + 1 + 15) * STEP * want[:, None] + 1e-9).all(), (np.abs(mass - want[:, None]) / want[:, None]).max() / STEP


def test_more_rows_than_twice_a_grid_of_large_blocks(here, case):  # noqa: F811
    """129 single tokens of 32767 heads, each the sixth of its text, in pages of two: the page that it fills, and the better one of the two in front."""
    case("chosen pages of 129 x 32767 rows")
    tokens, heads, d, page, pages = 129, 32767, 4, 2, 3
    gen = torch.Generator(device="cuda").manual_seed(44)
    k, v = (torch.randn((tokens * pages, heads, page, d), device="cuda", generator=gen) for _ in range(2))
    q, out = torch.randn((tokens, heads, d), device="cuda", generator=gen), torch.empty((tokens, heads, d), device="cuda")
    table = torch.randperm(tokens * pages, device="cuda", generator=gen).int().reshape(tokens, pages)
    at = table.long()
    means = torch.full((tokens * pages, heads, d), math.nan, device="cuda")
    full = k.double().sum(2).div(page).float()
    means[at[:, :2].flatten()] = full[at[:, :2].flatten()]
    chosen = torch.full((tokens, heads, 2), -5, device="cuda", dtype=torch.int32)
    starts, lengths = torch.arange(tokens + 1, device="cuda", dtype=torch.int32), torch.full((tokens,), 6, device="cuda", dtype=torch.int32)
    cache = D.KvCache(keys=k.data_ptr(), values=v.data_ptr(), elem=D.KV_F32, kv_heads=heads, head_size=d, page_size=page, pages=tokens * pages, page_stride=heads * page * d,
                      head_stride=page * d, slot_stride=d)
    batch = D.KvBatch(sequences=tokens, table_pages=pages, table_stride=pages, query_starts=starts.data_ptr(), lengths=lengths.data_ptr(), page_table=table.data_ptr())
    call = D.KvAttend(tokens=tokens, q_heads=heads, q=q.data_ptr(), out=out.data_ptr(), q_strides=(heads * d, d), out_strides=(heads * d, d), scale=0.5, max_tokens=1)
    sparse = D.KvSparse(means=means.data_ptr(), page_stride=heads * d, head_stride=d, chosen=chosen.data_ptr(), most=2, first=0, last=1)
    room = D.kv_attention_sparse_workspace(here, cache, batch, call, sparse)
    space = torch.empty(room, device="cuda", dtype=torch.uint8)
    call.workspace, call.workspace_bytes = space.data_ptr(), room
    torch.cuda.synchronize()
    here.kv_attention_sparse_raw(cache, batch, call, sparse)
    here.sync()
    assert torch.equal(means, full)
    score = (full[at[:, :2]].double() * q[:, None].double()).sum(-1)  # [tokens, page, heads]
    best = (score[:, 1] > score[:, 0]).int()
    assert torch.equal(chosen[..., 0], best) and (chosen[..., 1] == 2).all()
    take = torch.stack([torch.gather(at[:, None, :].expand(-1, heads, -1), 2, best[..., None].long())[..., 0], at[:, 2:3].expand(-1, heads)], 2)
    number = torch.arange(heads, device="cuda")[None, :, None]
    keys, values = (x[take, number].reshape(tokens, heads, 2 * page, d).double() for x in (k, v))
    x = (keys * q[:, :, None].double()).sum(-1) * 0.5
    p = torch.softmax(x, -1)
    want = (p[..., None] * values).sum(2)
    # A score is off by (d + 4) steps of its terms; a weight by what the worst score and its own are, the sum of 4 and 8 more: twice that with the values' sum.
    worst = (2 * (d + 4) * ((keys.abs() * q[:, :, None].double().abs()).sum(-1) * 0.5).amax(-1) + 2 * 4 + 8) * STEP
    assert ((out - want).abs() <= worst[..., None] * (p[..., None] * values.abs()).sum(2) + 1e-37).all()


@pytest.mark.parametrize("longest", [300, 3000, 60000])
def test_evictions_that_keep_no_recent_position(here, case, longest):  # noqa: F811
    """Positions at both ends of 32 bits, and none of them kept for being new."""
    case(f"evict, recent 0, {longest}")
    rng = np.random.default_rng(43)
    for values in ([-(1 << 31), (1 << 31) - 1, 0, 5], [(1 << 31) - 1], [-(1 << 31)]):
        for recent, first in ((0, 40), (0, 0), (1, 0)):
            e = Evict(rng, [longest, longest - 9], 2, 16, longest // 3, recent, first, max_keys=longest)
            e.positions = np.array(values, np.int64)[rng.integers(0, len(values), e.positions.shape)].astype(np.int32)
            e.run(here)
            here.sync()
            e.held()


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n,lengths,heads,kv,d", [([1, 1, 1], [1, 300, 77], 8, 2, 64), ([1, 2, 40], [700, 33, 90], 8, 2, 128), ([3, 1, 1], [2, 50, 400], 12, 3, 80),
                                                  ([1, 1, 9], [600, 5, 130], 8, 2, 256)])
@pytest.mark.parametrize("plain", [True, False])
def test_masses_whose_scores_are_not_kept(here, case, elem, n, lengths, heads, kv, d, plain):  # noqa: F811
    """Short sequences whose page table has room for 2^24 tokens, and no bound on their keys: their scores would take more than the workspace has for them."""
    case(f"mass, scores not kept {elem} n {n} lengths {lengths} heads {heads}/{kv} d {d} plain {plain}")
    rng = np.random.default_rng(41 + d)
    paged = Paged(rng, n, lengths, kv, d, 16, elem)
    table = np.full((len(n), 1 << 20), -1, np.int32)
    table[:, :paged.per] = paged.table
    paged.per, paged.table_on = table.shape[1], gpu(table)
    q = rng.standard_normal((sum(n) + 2, heads, d)).astype(np.float32)
    options = dict(decay=0.0) if plain else dict(decay=0.75, own_positions=False, window=100, cap=20.0, slopes=(2.0 ** -np.arange(1, heads + 1)).astype(np.float32),
                                                 first=rng.integers(-3, 60, sum(n) + 2).astype(np.int32))
    got = Mass(here, paged, gpu(q), rng, **options)
    assert got.room < 1 << 29
    got.run(here)
    here.sync()
    held_to_masses(got, q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n,lengths,heads,kv,d,page", [([20, 3], [1500, 900], 4, 2, 256, 8), ([9, 1, 30], [700, 800, 1300], 7, 1, 136, 12), ([11], [600], 3, 3, 200, 8),
                                                       ([1], [9000], 4, 2, 256, 16), ([1, 2], [5000, 8000], 6, 1, 200, 9), ([2], [5300], 2, 2, 136, 8)])
def test_many_pages_of_wide_heads(here, case, elem, n, lengths, heads, kv, d, page):  # noqa: F811
    """Scores by launches of their own: of rows next to each other, and of few rows of more than 512 pages."""
    case(f"sparse, wide heads {elem} n {n} lengths {lengths} heads {heads}/{kv} d {d} page {page}")
    rng = np.random.default_rng(42 + d)
    paged = Paged(rng, n, lengths, kv, d, page, elem)
    q = (1.5 * rng.standard_normal((sum(n) + 2, heads, d))).astype(np.float32)
    got = Sparse(here, paged, gpu(q), 12, 1, 2).run(here)
    here.sync()
    held_to_choice(got, q)


def widened(paged, sequences, table_pages):
    """The same sequences with others behind them that hold nothing, and a page table with room for more."""
    table = np.full((sequences, table_pages), -1, np.int32)
    table[:len(paged.n), :paged.per] = paged.table
    more = sequences - len(paged.n)
    paged.n, paged.lengths = paged.n + [0] * more, paged.lengths + [0] * more
    paged.table, paged.per, paged.table_on = table[:, :paged.per], table_pages, gpu(table)
    paged.starts_on, paged.lengths_on = gpu(np.concatenate([[0], np.cumsum(paged.n)]).astype(np.int32)), gpu(np.array(paged.lengths, np.int32))
    return paged


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("n", [[1], [40, 2]])
@pytest.mark.parametrize("room", [2512, 1 << 20])
def test_masses_of_more_keys_than_blocks_are_launched_for(here, case, elem, d, n, room):  # noqa: F811
    """1024 sequences, of which few hold anything, 2 heads of keys: 8 blocks a head, which go on with the keys behind their own."""
    case(f"mass, long {elem} d {d} n {n} room {room}")
    rng = np.random.default_rng(45)
    lengths = [2500, 1100][:len(n)]
    paged = widened(Paged(rng, n, lengths, 2, d, 16, elem), 1024, room // 16)
    q = rng.standard_normal((sum(n) + 2, 4, d)).astype(np.float32)
    got = Mass(here, paged, gpu(q), rng, decay=0.5).run(here)
    here.sync()
    held_to_masses(got, q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_masses_are_taken_whatever_the_page_table_has_room_for(here, case, elem):  # noqa: F811
    """32 sequences of 8 heads, whose table has room for 2^24 tokens each: a block for each 256 of those would be more than a grid holds."""
    case(f"mass, long table {elem}")
    rng = np.random.default_rng(46)
    paged = widened(Paged(rng, [1, 3, 1], [500, 70, 1], 8, 64, 16, elem), 32, 1 << 20)
    q = rng.standard_normal((5, 16, 64)).astype(np.float32)
    got = Mass(here, paged, gpu(q), rng).run(here)
    here.sync()
    held_to_masses(got, q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,tokens", [([1, 2, 1], 128), ([9, 3, 20], 2048)])
@pytest.mark.parametrize("room", [1280, 1 << 14])
def test_more_pages_than_blocks_are_launched_for(here, case, elem, d, n, tokens, room):  # noqa: F811
    """Three sequences among rows of padding, 8 heads of keys: blocks for 1024 pages of a row, which go on with the pages behind their own."""
    case(f"sparse, long {elem} d {d} n {n} tokens {tokens} room {room}")
    rng = np.random.default_rng(47)
    paged = widened(Paged(rng, n, [5000, 4300, 30], 8, d, 4, elem), 3, room)
    q = rng.standard_normal((tokens, 16, d)).astype(np.float32)
    got = Sparse(here, paged, gpu(q), 20, 3, 2, max_tokens=max(n)).run(here)
    here.sync()
    held_to_choice(got, q)


def test_chosen_pages_are_taken_whatever_the_page_table_has_room_for(here, case):  # noqa: F811
    """1024 rows times heads, and a table of 2^20 pages: a block for each 64 of those would be more than a grid holds."""
    case("sparse, long table")
    rng = np.random.default_rng(48)
    paged = widened(Paged(rng, [1, 2, 1], [900, 77, 9], 8, 64, 4), 3, 1 << 20)
    q = rng.standard_normal((128, 16, 64)).astype(np.float32)
    got = Sparse(here, paged, gpu(q), 20, 3, 2, max_tokens=2).run(here)
    here.sync()
    held_to_choice(got, q)


@pytest.mark.parametrize("page", [1, 4, 16])
def test_means_of_more_pages_than_blocks_are_launched_for(here, case, page):  # noqa: F811
    """1024 sequences, of which three hold anything, 8 heads of keys: two blocks a head."""
    case(f"page means, long, pages of {page}")
    rng = np.random.default_rng(49)
    n, lengths = [100, 3, 70], [130, 48, 70]
    paged = widened(Paged(rng, n, lengths, 8, 64, page), 1024, 200)
    means = torch.full((paged.pages, 8, 64), math.nan, device="cuda")
    torch.cuda.synchronize()
    here.kv_page_means_raw(paged.cache(), paged.batch(), D.KvSparse(means=means.data_ptr(), page_stride=8 * 64, head_stride=64), sum(n))
    here.sync()
    got, full, written = means.cpu().numpy(), page_means(paged).cpu().numpy(), np.zeros(paged.pages, bool)
    for s, (m, l) in enumerate(zip(n, lengths)):
        written[paged.table[s, (l - m) // page:l // page]] = True
    np.testing.assert_array_equal(got[written], full[written])
    assert np.isnan(got[~written]).all()


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_the_workspace_that_plain_attention_wants_is_told(here, case, elem):  # noqa: F811
    """Where trees want more, the query without `causal` answers for ahip_kv_attention alone, whatever its masks."""
    case(f"workspace of plain attention {elem}")
    rng = np.random.default_rng(50)
    n, lengths = [40] * 16, [int(x) for x in rng.integers(40, 700, 16)]
    paged = Paged(rng, n, lengths, 8, 64, 16, elem)
    q = rng.standard_normal((sum(n), 32, 64)).astype(np.float32)
    on, out, prefix = gpu(q), torch.empty((sum(n), 32, 64), device="cuda"), rng.integers(0, 300, 16).astype(np.int32)
    call = D.KvAttend(tokens=sum(n), q_heads=32, q=on.data_ptr(), out=out.data_ptr(), q_strides=on.stride()[:2], out_strides=out.stride()[:2], scale=1 / 8, max_tokens=40)
    asked = D.kv_attention_workspace(here, paged.cache(), paged.batch(), call)
    call.causal = 0
    room = D.kv_attention_workspace(here, paged.cache(), paged.batch(), call)
    assert room < asked
    space = torch.full((room // 4 + 4,), math.nan, device="cuda")
    call.workspace, call.workspace_bytes, on_prefix = space.data_ptr(), room, gpu(prefix)
    for masks in (dict(), dict(causal=False), dict(window=90), dict(prefix=prefix)):
        call.causal, call.window, call.prefix = int(masks.get("causal", True)), masks.get("window", 0), on_prefix.data_ptr() if "prefix" in masks else None
        torch.cuda.synchronize()
        here.kv_attention_raw(paged.cache(), paged.batch(), call)
        here.sync()
        held_to_definition(out.cpu().numpy(), paged, q, **masks)
    assert torch.isnan(space[room // 4:]).all()
    if room:
        call.workspace_bytes = room - 4
        with pytest.raises(AltiusHipError) as e:
            here.kv_attention_raw(paged.cache(), paged.batch(), call)
        assert e.value.code == ERR_ARG
