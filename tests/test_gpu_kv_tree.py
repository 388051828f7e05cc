"""Attention of trees of drafted tokens over a paged cache (ahip_kv_attention_tree), and the moves (ahip_kv_move) that follow, against their definitions."""
import math

import numpy as np
import pytest
import torch

from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_UNSUPPORTED, AltiusHipError
from decoder_more_oracle import attended_where, tree
from decoder_oracle import turned, turned_bound
from test_gpu_kv_cache import Paged, attend, gpu, here, raises_at_sync  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def tree_call(ctx, paged, q, options, out, max_tokens=0, max_keys=0):
    call = D.KvAttend(tokens=q.shape[0], q_heads=q.shape[1], q=q.data_ptr(), out=out.data_ptr(), q_strides=q.stride()[:2], out_strides=out.stride()[:2],
                      scale=options.get("scale", 1 / math.sqrt(paged.d)), softcap=options.get("cap", 0.0), window=options.get("window", 0), max_tokens=max_tokens, max_keys=max_keys)
    keep = [gpu(options[x]) if options.get(x) is not None else None for x in ("slopes", "first")]
    call.slopes, call.first_keys = (None if x is None else x.data_ptr() for x in keep)
    room = D.kv_attention_workspace(ctx, paged.cache(), paged.batch(), call)
    space = torch.full((room // 4 + 4,), math.nan, device="cuda")
    call.workspace, call.workspace_bytes = space.data_ptr(), room
    return call, (keep, space, room)


def attend_tree(ctx, paged, q, parents, out=None, max_tokens=0, max_keys=0, **options):
    out = torch.full_like(q, 5.0, memory_format=torch.contiguous_format) if out is None else out
    call, keep = tree_call(ctx, paged, q, options, out, max_tokens, max_keys)
    on = gpu(parents.astype(np.int32))
    torch.cuda.synchronize()
    ctx.kv_attention_tree_raw(paged.cache(), paged.batch(), call, on.data_ptr())
    torch.cuda.synchronize()
    assert torch.isnan(keep[1][keep[2] // 4:]).all()
    return out


def held_to_tree(got, paged, q, parents, window=0, cap=0.0, slopes=None, first=None, scale=None, but=()):
    at = 0
    for s, (m, l) in enumerate(zip(paged.n, paged.lengths)):
        rows = slice(at, at + m)
        at += m
        if s in but or m == 0:
            continue
        k, v = paged.dense(s)
        seen, distance = tree(parents[rows], l, window, None if first is None else first[rows])
        want, bound, _, _ = attended_where(q[rows], k, v, seen, distance, scale if scale is not None else 1 / math.sqrt(paged.d), cap, slopes)
        assert np.isfinite(got[rows]).all()
        off = np.abs(got[rows] - want)
        assert (off <= bound + 1e-37).all(), f"sequence {s}: {(off / (bound + 1e-37)).max():.3g} times the bound, {off.max():.3g}"
    assert (got[at:] == 5.0).all(), "padding was written"


def random_tree(rng, n, back=6):
    """Each row follows one of a few in front of it, or none."""
    parents = np.arange(n) - 1 - (rng.random(n) ** 2 * back).astype(np.int64)
    return np.where(parents < 0, -1, parents)


TREES = [  # n, before, heads, kv heads, d, page, type, order
    ([1], [0], 1, 1, 64, 16, "f32", "head"),
    ([8], [500], 12, 12, 64, 16, "f32", "head"),
    ([4, 1, 7], [0, 300, 33], 8, 2, 128, 16, "f32", "slot"),
    ([5, 3], [31, 1000], 8, 1, 128, 32, "bf16", "head"),
    ([31, 2, 32], [100, 5, 64], 4, 4, 64, 16, "bf16", "slot"),
    ([33, 0, 60], [7, 12, 250], 4, 2, 96, 24, "f32", "head"),
    ([64], [3000], 8, 2, 128, 64, "f32", "slot"),
    ([63, 17], [1700, 40], 14, 2, 80, 16, "bf16", "head"),
    ([256, 9], [70, 400], 2, 1, 64, 16, "f32", "head"),
    ([255, 130], [10, 1], 3, 1, 128, 48, "bf16", "slot"),
    ([200], [1], 1, 1, 128, 16, "f32", "head"),
    ([20, 9], [90, 3], 4, 2, 256, 16, "f32", "head"),
    ([100], [333], 2, 1, 256, 24, "bf16", "slot"),
    ([6, 40], [50, 33], 3, 1, 20, 5, "f32", "slot"),
    ([3] * 70, [5 * i for i in range(70)], 4, 2, 64, 16, "f32", "head"),
]


@pytest.mark.parametrize("n,before,heads,kv,d,page,elem,order", TREES)
@pytest.mark.parametrize("plain", [True, False])
def test_drafted_tokens_see_what_they_follow(here, case, n, before, heads, kv, d, page, elem, order, plain):  # noqa: F811
    case(f"tree n {n[:5]} before {before[:5]} heads {heads}/{kv} d {d} page {page} {elem} {order} plain {plain}")
    rng = np.random.default_rng(d + page + len(n) + n[0])
    lengths = [a + b for a, b in zip(n, before)]
    paged = Paged(rng, n, lengths, kv, d, page, elem, order)
    parents = np.concatenate([random_tree(rng, m) for m in n] + [np.full(3, 1000)])  # what stands beside padding is not read
    q = (1.5 * rng.standard_normal((sum(n) + 3, heads, d))).astype(np.float32)
    options = {} if plain else dict(window=max(3, max(lengths) // 3), cap=20.0, slopes=(2.0 ** -np.arange(1, heads + 1)).astype(np.float32),
                                    first=rng.integers(-3, max(before) + 9, sum(n) + 3).astype(np.int32))
    got = attend_tree(here, paged, gpu(q), parents, **options).cpu().numpy()
    here.sync()
    held_to_tree(got, paged, q, parents, **options)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n", [[6, 20], [90, 64]])
@pytest.mark.parametrize("options", [dict(window=1), dict(window=2), dict(window=40), dict(cap=2.0), dict(scale=0.0), dict(slopes=np.array([0.0, 0.5, 0.01, -0.02], np.float32)),
                                     dict(slopes=np.full(4, 0.3, np.float32), window=7), dict(first=True)])
def test_each_mask_and_bias_of_trees(here, case, elem, options, n):  # noqa: F811
    case(f"tree {elem} {sorted(options)} n {n}")
    rng = np.random.default_rng(19)
    paged = Paged(rng, n, [n[0] + 77, n[1] + 5], 2, 64, 16, elem)
    parents = np.concatenate([random_tree(rng, m, 3) for m in n])
    q = rng.standard_normal((sum(n), 4, 64)).astype(np.float32)
    options = {**options, **({"first": rng.integers(0, 90, sum(n)).astype(np.int32)} if "first" in options else {})}
    got = attend_tree(here, paged, gpu(q), parents, **options).cpu().numpy()
    here.sync()
    held_to_tree(got, paged, q, parents, **options)


@pytest.mark.parametrize("n,before", [([5, 9], [40, 700]), ([100, 7, 64], [300, 1, 2000]), ([256], [5000])])
@pytest.mark.parametrize("d,elem", [(64, "f32"), (128, "bf16"), (96, "f32"), (256, "f32")])
def test_a_chain_is_a_prompt(here, case, n, before, d, elem):  # noqa: F811
    """Each row follows the one in front of it: what ahip_kv_attention gives, within the bounds of both (the sums are made in another order)."""
    case(f"tree chain n {n} d {d} {elem}")
    rng = np.random.default_rng(5)
    paged = Paged(rng, n, [a + b for a, b in zip(n, before)], 2, d, 16, elem)
    x = rng.standard_normal((sum(n), 4, d)).astype(np.float32)
    q, chain = gpu(x), np.concatenate([np.arange(m) - 1 for m in n])
    for options in (dict(), dict(cap=9.0, slopes=np.full(4, 0.1, np.float32)), dict(window=60)):
        want, got = attend(here, paged, q, **options).cpu().numpy(), attend_tree(here, paged, q, chain, **options).cpu().numpy()
        here.sync()
        held_to_tree(got, paged, x, chain, **options)
        held_to_tree(want, paged, x, chain, **options)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("n", [6, 80])
def test_other_branches_do_not_reach_a_row(here, case, elem, n):  # noqa: F811
    """Two branches from the root, turn about; what one holds is not finite."""
    case(f"tree branches {elem} n {n}")
    rng = np.random.default_rng(6)
    paged = Paged(rng, [n], [50 + n], 1, 64, 16, elem)
    parents = np.maximum(np.arange(n) - 2, -1)
    odd = np.arange(51, 50 + n, 2)
    for x, bad in zip(paged.views(), (math.inf, math.nan)):
        x[torch.from_numpy(paged.table[0, odd // 16]).long().cuda(), 0, torch.from_numpy(odd % 16).cuda()] = bad
    q = rng.standard_normal((n, 2, 64)).astype(np.float32)
    got = attend_tree(here, paged, gpu(q), parents).cpu().numpy()
    here.sync()
    k, v = paged.dense(0)
    seen, distance = tree(parents, 50 + n)
    even = np.arange(0, n, 2)
    want, bound, _, _ = attended_where(q[even], k, v, seen[even], distance[even], 1 / 8, 0.0, None)
    assert (np.abs(got[even] - want) <= bound).all() and np.isnan(got[1::2]).all()


def test_a_sequence_that_is_shorter_than_its_rows(here, case):  # noqa: F811
    case("tree, short sequence")
    rng = np.random.default_rng(7)
    for n, length in (([5, 3], [3, 40]), ([90, 3], [60, 40])):
        paged = Paged(rng, n, length, 1, 64, 16)
        parents = np.concatenate([np.maximum(np.arange(m) - 2, -1) for m in n])
        q = rng.standard_normal((sum(n), 2, 64)).astype(np.float32)
        got = attend_tree(here, paged, gpu(q), parents).cpu().numpy()
        here.sync()
        held_to_tree(got, paged, q, parents)
        assert (got[:n[0] - length[0]] == 0).all()


@pytest.mark.parametrize("n", [[7, 7], [100, 90]])
@pytest.mark.parametrize("bad", [3, 4, -2, 1 << 30, -(1 << 31)])
def test_parents_that_are_not_in_front_are_told(here, case, n, bad):  # noqa: F811
    case(f"tree, bad parent {bad} n {n}")
    rng = np.random.default_rng(8)
    paged = Paged(rng, n, [40 + m for m in n], 2, 64, 16)
    parents = np.concatenate([random_tree(rng, m) for m in n])
    q = rng.standard_normal((sum(n), 2, 64)).astype(np.float32)
    wrong, taken = parents.copy(), parents.copy()
    wrong[3], taken[3] = bad, -1
    got = attend_tree(here, paged, gpu(q), wrong).cpu().numpy()
    raises_at_sync(here)
    held_to_tree(got, paged, q, taken)


def test_more_rows_than_a_tree_has_are_left_out(here, case):  # noqa: F811
    case("tree of 257 rows")
    rng = np.random.default_rng(9)
    paged = Paged(rng, [257, 4], [300, 90], 1, 64, 16)
    parents = np.concatenate([np.arange(257) - 1, np.arange(4) - 1])
    q = rng.standard_normal((261, 1, 64)).astype(np.float32)
    got = attend_tree(here, paged, gpu(q), parents).cpu().numpy()
    raises_at_sync(here)
    assert (got[:257] == 5.0).all()
    held_to_tree(got, paged, q, parents, but=(0,))


def test_trees_that_are_refused(here, case):  # noqa: F811
    case("tree refusals")
    rng = np.random.default_rng(10)
    paged = Paged(rng, [2], [20], 1, 64, 16)
    q, parents = gpu(rng.standard_normal((2, 1, 64)).astype(np.float32)), gpu(np.array([-1, 0], np.int32))
    out = torch.full_like(q, 5.0)
    for code, change in ((ERR_ARG, dict(causal=0)), (ERR_ARG, dict(prefix=parents.data_ptr())), (ERR_UNSUPPORTED, dict(max_tokens=257)), (ERR_ARG, dict(out=q.data_ptr())),
                         (ERR_ARG, dict(q=None)), (ERR_UNSUPPORTED, dict(q=q.data_ptr() + 4))):
        call, keep = tree_call(here, paged, q, {}, out)
        for name, x in change.items():
            setattr(call, name, x)
        with pytest.raises(AltiusHipError) as e:
            here.kv_attention_tree_raw(paged.cache(), paged.batch(), call, parents.data_ptr())
        assert e.value.code == code
    call, keep = tree_call(here, paged, q, {}, out)
    with pytest.raises(AltiusHipError) as e:
        here.kv_attention_tree_raw(paged.cache(), paged.batch(), call, None)
    assert e.value.code == ERR_ARG
    here.sync()
    assert (out == 5.0).all()


# ---- moves -----------------------------------------------------------------------------------------------------------

def lists(rng, sequences, heads, slots, counts, kind):
    """Sources and targets [sequences, heads, most], padded with places that are none."""
    most = max(1, max(counts))
    sources, targets = (np.full((sequences, heads, most), 1 << 30, np.int32) for _ in range(2))
    for i, c in enumerate(counts):
        s, h = divmod(i, heads)
        if kind == "apart":
            places = rng.permutation(slots)[:2 * c]
            sources[s, h, :c], targets[s, h, :c] = places[:c], places[c:]
        else:  # an accepted branch: ascending, to the front
            base = slots - 2 * c if c else 0
            sources[s, h, :c] = base + np.sort(rng.permutation(2 * c)[:c])
            targets[s, h, :c] = base + np.arange(c)
    return sources, targets, most


MOVES = [  # sequences, kv heads, d, page, type, order, slots, most moves, by head, kind, history
    (1, 1, 64, 16, "f32", "head", 8, 3, False, "order", False),
    (3, 2, 128, 16, "f32", "slot", 60, 25, False, "order", True),
    (5, 4, 128, 16, "bf16", "head", 90, 40, True, "apart", True),
    (2, 2, 96, 24, "f32", "head", 3000, 1400, True, "apart", True),
    (2, 3, 80, 5, "bf16", "slot", 600, 290, False, "apart", False),
    (2, 1, 256, 16, "f32", "head", 700, 340, True, "order", True),
    (70, 2, 64, 8, "f32", "head", 20, 9, True, "order", True),
    (2, 2, 7, 3, "bf16", "head", 50, 24, True, "apart", True),
    (2, 2, 20, 3, "bf16", "slot", 50, 24, False, "order", True),
    (1, 2, 5, 4, "f32", "head", 50, 24, True, "order", True),
    (1, 1, 1100, 4, "f32", "slot", 20, 9, True, "order", True),
    (1, 1, 4099, 4, "bf16", "head", 20, 9, True, "apart", False),
    (1, 1, 5000, 4, "f32", "head", 20, 9, False, "order", False),
]


@pytest.mark.parametrize("sequences,kv,d,page,elem,order,slots,most,by_head,kind,history", MOVES)
def test_slots_move(here, case, sequences, kv, d, page, elem, order, slots, most, by_head, kind, history):  # noqa: F811
    case(f"move {sequences} x {kv} d {d} page {page} {elem} {order} slots {slots} most {most} {kind}")
    rng = np.random.default_rng(d + page + slots)
    paged = Paged(rng, [0] * sequences, [slots] * sequences, kv, d, page, elem, order)
    heads = kv if by_head else 1
    counts = rng.integers(0, most + 1, sequences * heads)
    counts[0] = most
    sources, targets, room = lists(rng, sequences, heads, slots, counts, kind)
    on = [gpu(x) for x in (sources, targets, counts.astype(np.int32))]
    mass, positions = gpu(rng.random((paged.pages, kv, page)).astype(np.float32)), gpu(rng.integers(0, 1 << 30, (paged.pages, kv, page)).astype(np.int32))
    state = [x.float().cpu().numpy() for x in paged.views()] + [mass.cpu().numpy(), positions.cpu().numpy()]
    want = [x.copy() for x in state]
    for s in range(sequences):
        for h in range(kv):
            i = h if by_head else 0
            c = counts[s * heads + i]
            a, b = sources[s, i, :c], targets[s, i, :c]
            for w, x in zip(want, state):
                w[paged.table[s][b // page], h, b % page] = x[paged.table[s][a // page], h, a % page]
    moves = D.KvMoves(sources=on[0].data_ptr(), targets=on[1].data_ptr(), counts=on[2].data_ptr(), strides=(heads * room, room if by_head else 0),
                      count_strides=(heads, 1 if by_head else 0), most=room, apart=int(kind == "apart"))
    remembered = D.KvHistory(mass=mass.data_ptr(), positions=positions.data_ptr(), page_stride=kv * page, head_stride=page) if history else None
    torch.cuda.synchronize()
    here.kv_move_raw(paged.cache(), paged.batch(), moves, remembered)
    here.sync()
    got = [x.float().cpu().numpy() for x in paged.views()] + [mass.cpu().numpy(), positions.cpu().numpy()]
    for i, (x, y) in enumerate(zip(got, want)):
        np.testing.assert_array_equal(x, y if i < 2 or history else state[i])


@pytest.mark.parametrize("apart", [0, 1])
@pytest.mark.parametrize("what", ["source", "source_negative", "target", "page", "count", "count_negative"])
def test_moves_that_do_not_fit_are_told(here, case, what, apart):  # noqa: F811
    case(f"move, bad {what} apart {apart}")
    rng = np.random.default_rng(12)
    paged = Paged(rng, [0, 0], [16, 16], 1, 64, 4)
    sources, targets, counts = (np.array(x, np.int32) for x in ([[8, 9, 10], [8, 9, 10]], [[0, 1, 2], [0, 1, 2]], [3, 3]))
    bad = {(0, 1)}
    if what == "source":
        sources[0, 1] = 16
    elif what == "source_negative":
        sources[0, 1] = -1
    elif what == "target":
        targets[0, 1] = 1 << 30
    elif what == "page":
        paged.table_on[0, 2] = paged.pages
        bad = {(0, 0), (0, 1), (0, 2)}
    else:
        counts[0] = 4 if what == "count" else -1
        bad = {(0, 0), (0, 1), (0, 2)}
    before = paged.views()[0].cpu().numpy()
    want = before.copy()
    for s in range(2):
        for i in range(3):
            if (s, i) not in bad:
                want[paged.table[s, i // 4], 0, i] = before[paged.table[s, (8 + i) // 4], 0, i]
    on = [gpu(x) for x in (sources, targets, counts)]
    torch.cuda.synchronize()
    here.kv_move_raw(paged.cache(), paged.batch(), D.KvMoves(sources=on[0].data_ptr(), targets=on[1].data_ptr(), counts=on[2].data_ptr(), strides=(3, 0), count_strides=(1, 0),
                                                             most=3, apart=apart))
    raises_at_sync(here)
    np.testing.assert_array_equal(paged.views()[0].cpu().numpy(), want)


def test_moves_that_are_refused(here, case):  # noqa: F811
    case("move refusals")
    rng = np.random.default_rng(13)
    paged = Paged(rng, [0], [16], 1, 64, 4)
    on = gpu(np.zeros(4, np.int32))
    fine = dict(sources=on.data_ptr(), targets=on.data_ptr(), counts=on.data_ptr(), strides=(4, 0), count_strides=(1, 0), most=4, apart=1)
    history = dict(page_stride=4, head_stride=4)
    for change in (dict(sources=None), dict(targets=None), dict(counts=None), dict(strides=(-1, 0)), dict(count_strides=(0, -1)), dict(most=-1)):
        with pytest.raises(AltiusHipError) as e:
            here.kv_move_raw(paged.cache(), paged.batch(), D.KvMoves(**{**fine, **change}))
        assert e.value.code == ERR_ARG
    with pytest.raises(AltiusHipError) as e:
        here.kv_move_raw(paged.cache(), paged.batch(), D.KvMoves(**fine), D.KvHistory(**{**history, "page_stride": -1}))
    assert e.value.code == ERR_ARG
    here.kv_move_raw(paged.cache(), paged.batch(), D.KvMoves(**{**fine, "most": 0, "sources": None}))  # nothing to do
    here.sync()


# ---- together --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_a_recorded_step_of_drafted_tokens(here, case, elem):  # noqa: F811
    """Drafted tokens are appended at their positions, attend as a tree, and one branch of each is moved to the front: recorded once, replayed while the texts
    grow and the trees change, each replay held to the same steps on another cache without a recording."""
    case(f"tree step, recorded {elem}")
    rng = np.random.default_rng(14)
    n, kv, heads, d, page = [9, 5, 12], 2, 8, 64, 16
    lengths = [30, 100, 12]
    caches = [Paged(np.random.default_rng(1), n, lengths, kv, d, page, elem, table_pages=20) for _ in range(2)]
    f = gpu(D.rotary_frequencies(d))
    tokens = sum(n)
    starts = np.concatenate([[0], np.cumsum(n)])
    held = []
    stream = torch.cuda.Stream()
    for which, paged in enumerate(caches):
        s = dict(packed=torch.zeros((tokens, heads + 2 * kv, d), device="cuda"), q=torch.zeros((tokens, heads, d), device="cuda"), out=torch.zeros((tokens, heads, d), device="cuda"),
                 parents=torch.zeros(tokens, dtype=torch.int32, device="cuda"), positions=torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                 sources=torch.zeros((3, 12), dtype=torch.int32, device="cuda"), targets=torch.zeros((3, 12), dtype=torch.int32, device="cuda"),
                 counts=torch.zeros(3, dtype=torch.int32, device="cuda"))
        call, keep = tree_call(here, paged, s["q"], {}, s["out"], max_tokens=12, max_keys=300)
        p = s["packed"]
        fields = D.KvTokens(tokens=tokens, k=p[:, heads:].data_ptr(), v=p[:, heads + kv:].data_ptr(), k_strides=p.stride()[:2], v_strides=p.stride()[:2], q_heads=heads, q=p.data_ptr(),
                            q_out=s["q"].data_ptr(), q_strides=p.stride()[:2], q_out_strides=s["q"].stride()[:2], positions=s["positions"].data_ptr())
        moves = D.KvMoves(sources=s["sources"].data_ptr(), targets=s["targets"].data_ptr(), counts=s["counts"].data_ptr(), strides=(12, 0), count_strides=(1, 0), most=12)
        s.update(paged=paged, call=call, keep=keep, fields=fields, moves=moves)
        held.append(s)

    def step(ctx, s):
        ctx.kv_append_raw(s["paged"].cache(), s["paged"].batch(), s["fields"], D.Rotary(f.data_ptr(), d))
        ctx.kv_attention_tree_raw(s["paged"].cache(), s["paged"].batch(), s["call"], s["parents"].data_ptr())
        ctx.kv_move_raw(s["paged"].cache(), s["paged"].batch(), s["moves"])

    with D.Context(0, stream=stream.cuda_stream) as recorded:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step(recorded, held[0])
        base = np.array(lengths) - n
        for turn in range(5):
            new = rng.standard_normal((tokens, heads + 2 * kv, d)).astype(np.float32)
            parents, positions, accepted = [], [], []
            for i, m in enumerate(n):
                mine = random_tree(rng, m)
                depth = np.zeros(m, int)
                for t in range(m):
                    depth[t] = depth[mine[t]] + 1 if mine[t] >= 0 else 0
                branch, at = [], int(rng.integers(0, m))
                while at >= 0:
                    branch.insert(0, at)
                    at = mine[at]
                parents.append(mine), positions.append(base[i] + depth), accepted.append(np.array(branch))
            for s in held:
                s["packed"].copy_(gpu(new)), s["parents"].copy_(gpu(np.concatenate(parents).astype(np.int32))), s["positions"].copy_(gpu(np.concatenate(positions).astype(np.int32)))
                s["paged"].lengths_on.copy_(gpu((base + n).astype(np.int32)))
                for i, a in enumerate(accepted):
                    s["sources"][i, :len(a)] = gpu((base[i] + a).astype(np.int32))
                    s["targets"][i, :len(a)] = gpu((base[i] + np.arange(len(a))).astype(np.int32))
                s["counts"].copy_(gpu(np.array([len(a) for a in accepted], np.int32)))
            torch.cuda.synchronize()
            graph.replay()
            step(here, held[1])
            torch.cuda.synchronize()
            here.sync(), recorded.sync()
            np.testing.assert_array_equal(held[0]["out"].cpu().numpy(), held[1]["out"].cpu().numpy())
            for x, y in zip(held[0]["paged"].on, held[1]["paged"].on):
                assert torch.equal(x, y)
            # The branch's rows against what they are: a text that grows by them.
            base = base + np.array([len(a) for a in accepted])
            caches[1].lengths = list(base + n)
    # The cache now holds, for every text, what appending the accepted tokens one after the other would have left.
    i = 2
    k = caches[1].dense(i)[0][base[i] - len(accepted[i]):base[i]]
    assert k.shape[0] == len(accepted[i])
    new_k = new[starts[i] + accepted[i], heads:heads + kv].astype(np.float64)
    place = base[i] - len(accepted[i]) + np.arange(len(accepted[i]))
    want, bound = turned(new_k, place, D.rotary_frequencies(d), False), turned_bound(new_k, d // 2, False, None)
    assert (np.abs(k - want) <= bound + (2.0 ** -8 * np.abs(want) if elem == "bf16" else 0)).all()
