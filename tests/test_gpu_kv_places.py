"""The operators around a paged cache where its memory lies otherwise than in their own tests: pages more than 2^33 bytes apart, pages that sequences share, two calls on
two streams at once.  Each against the same call on a cache of its own, bit for bit."""
import math

import numpy as np
import pytest
import torch

from altius_amd import device as D
from test_gpu_kv_cache import Paged, attend, gpu, held_to_definition, here  # noqa: F401 (a fixture)
from test_gpu_kv_mass import Mass, held_to_masses
from test_gpu_kv_sparse import Sparse, held_to_choice, page_means
from test_gpu_kv_tree import attend_tree, held_to_tree, random_tree

pytestmark = pytest.mark.gpu

APART = (1 << 31) + 192  # elements from a page to the next


def spread(whole, x):
    """x, [pages, ...], with its pages that far apart."""
    inner = [math.prod(x.shape[i + 1:]) for i in range(1, x.dim())]
    far = whole.as_strided(x.shape, (APART, *inner))
    far.copy_(x)
    return far


@pytest.fixture(scope="module")
def far_memory():
    """Room for three pages of keys, of values, of masses, of positions and of means."""
    memory = [torch.empty(2 * APART + 4096, device="cuda") for _ in range(4)] + [torch.empty(2 * APART + 4096, device="cuda", dtype=torch.int32)]
    yield memory
    memory.clear()
    torch.cuda.empty_cache()


def near_and_far(rng, far_memory, n, length, d=64, slots=16):
    near = Paged(rng, n, [length], 1, d, slots, spare_pages=0)
    assert near.pages == 3
    far = Paged(rng, n, [length], 1, d, slots, spare_pages=0)
    far.table, far.table_on = near.table, near.table_on
    far.on = [spread(whole, x) for whole, x in zip(far_memory, near.on)]
    return near, far


@pytest.mark.parametrize("n", [1, 20])
def test_trees_of_a_cache_past_32_bits(here, case, far_memory, n):  # noqa: F811
    case(f"tree far {n}")
    rng = np.random.default_rng(50 + n)
    near, far = near_and_far(rng, far_memory, [n], 45)
    q, parents = gpu(rng.standard_normal((n, 4, 64)).astype(np.float32)), random_tree(rng, n)
    a, b = (attend_tree(here, paged, q, parents) for paged in (near, far))
    here.sync()
    assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 20])
def test_masses_of_a_cache_past_32_bits(here, case, far_memory, n):  # noqa: F811
    case(f"mass far {n}")
    rng = np.random.default_rng(60 + n)
    near, far = near_and_far(rng, far_memory, [n], 45)
    q = gpu(rng.standard_normal((n, 4, 64)).astype(np.float32))
    a, b = (Mass(here, paged, q, np.random.default_rng(1)) for paged in (near, far))
    b.mass, b.positions = spread(far_memory[2], a.mass), spread(far_memory[4], a.positions)
    b.history = D.KvHistory(mass=b.mass.data_ptr(), positions=b.positions.data_ptr(), page_stride=APART, head_stride=16)
    a.run(here), b.run(here)
    here.sync()
    assert torch.equal(a.out, b.out) and torch.equal(a.mass, b.mass) and torch.equal(a.positions, b.positions)


@pytest.mark.parametrize("n", [1, 20])
def test_chosen_pages_of_a_cache_past_32_bits(here, case, far_memory, n):  # noqa: F811
    case(f"sparse far {n}")
    rng = np.random.default_rng(70 + n)
    near, far = near_and_far(rng, far_memory, [n], 48)
    q = gpu(rng.standard_normal((n, 4, 64)).astype(np.float32))
    a, b = (Sparse(here, paged, q, 2) for paged in (near, far))
    b.means = spread(far_memory[3], a.means)
    b.sparse.means, b.sparse.page_stride = b.means.data_ptr(), APART
    a.run(here), b.run(here)
    here.sync()
    assert torch.equal(a.out, b.out) and torch.equal(a.chosen, b.chosen) and torch.equal(a.means, b.means) and not torch.isnan(a.means).any()


@pytest.mark.parametrize("slots", [16, 700])
def test_evictions_and_moves_of_a_cache_past_32_bits(here, case, far_memory, slots):  # noqa: F811
    case(f"evict and move far {slots}")
    rng = np.random.default_rng(80)
    length = 3 * slots - 3
    budget = length // 2
    near, far = near_and_far(rng, far_memory, [1], length, 4, slots)
    mass, positions = gpu(rng.random((3, 1, slots)).astype(np.float32)), gpu(rng.permutation(3 * slots).reshape(3, 1, slots).astype(np.int32))
    histories = [(mass, positions, slots), (spread(far_memory[2], mass), spread(far_memory[4], positions), APART)]
    lists = []
    for paged, (m, p, stride) in zip((near, far), histories):
        sources, targets = (torch.full((budget + 1,), -9, device="cuda", dtype=torch.int32) for _ in range(2))
        counts, kept = (torch.full((1,), -9, device="cuda", dtype=torch.int32) for _ in range(2))
        history = D.KvHistory(mass=m.data_ptr(), positions=p.data_ptr(), page_stride=stride, head_stride=slots)
        torch.cuda.synchronize()
        here.kv_evict_raw(paged.cache(), paged.batch(), history, D.KvEviction(budget=budget, recent=7, first=2, most=budget + 1, max_keys=length, sources=sources.data_ptr(),
                                                                               targets=targets.data_ptr(), counts=counts.data_ptr(), lengths=kept.data_ptr()))
        here.kv_move_raw(paged.cache(), paged.batch(), D.KvMoves(sources=sources.data_ptr(), targets=targets.data_ptr(), counts=counts.data_ptr(), strides=(budget + 1, 0),
                                                                count_strides=(1, 0), most=budget + 1, apart=1), history)
        here.sync()
        lists.append((sources, targets, counts, kept))
    assert int(lists[0][2]) > 0 and all(torch.equal(x, y) for x, y in zip(*lists))
    assert all(torch.equal(x, y) for x, y in zip(near.on, far.on)) and torch.equal(*(h[0] for h in histories)) and torch.equal(*(h[1] for h in histories))


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_sequences_that_share_a_prefix(here, case, elem):  # noqa: F811
    """The first five pages of three sequences are the same: trees of drafted tokens and chosen pages read them, whoever else does."""
    case(f"shared prefix {elem}")
    rng = np.random.default_rng(90)
    n, lengths = [6, 1, 30], [100, 90, 120]
    paged = Paged(rng, n, lengths, 2, 64, 16, elem)
    paged.table[1:, :5] = paged.table[0, :5]
    paged.table_on = gpu(paged.table)
    q, parents = rng.standard_normal((sum(n), 8, 64)).astype(np.float32), np.concatenate([random_tree(rng, m) for m in n])
    on = gpu(q)
    held_to_tree(attend_tree(here, paged, on, parents).cpu().numpy(), paged, q, parents)
    got = Sparse(here, paged, on, 4, 1, 1)
    full = page_means(paged)
    for s, (m, l) in enumerate(zip(n, lengths)):
        before = torch.from_numpy(paged.table[s, :(l - m) // 16].astype(np.int64)).cuda()
        got.means[before] = full[before]
    held_to_choice(got.run(here), q)
    here.sync()


def test_two_calls_at_once(here, case):  # noqa: F811
    """Two contexts with streams and workspaces of their own, without a wait between their calls."""
    case("two calls at once")
    rng = np.random.default_rng(91)
    calls = []
    for elem, n, lengths in (("f32", [1, 40], [3000, 900]), ("bf16", [70, 1], [400, 5000])):
        paged = Paged(rng, n, lengths, 2, 128, 16, elem)
        q = rng.standard_normal((sum(n), 8, 128)).astype(np.float32)
        on = gpu(q)
        calls.append((Mass(here, paged, on, rng), Sparse(here, paged, on, 9, 1, 2), q, on))
    streams = [torch.cuda.Stream() for _ in calls]
    contexts = [D.Context(0, stream=s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, (mass, *_) in zip(contexts, calls):
            c.kv_attention_mass_raw(mass.paged.cache(), mass.paged.batch(), mass.call, mass.history, 0.0, mass.rows.data_ptr())
        for c, (_, sparse, *_) in zip(contexts, calls):
            c.kv_attention_sparse_raw(sparse.paged.cache(), sparse.paged.batch(), sparse.call, sparse.sparse)
    for c in contexts:
        c.sync()
        c.close()
    for mass, sparse, q, _ in calls:
        mass.decay = 0.0
        held_to_masses(mass, q)
        held_to_choice(sparse, q)


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_means_of_pages_that_moved_slots_fill(here, case, elem):  # noqa: F811
    """Accepted tokens of a tree go to the front and fill a page: its mean is made with them as the newest rows, and the next token chooses by it."""
    case(f"means behind moves {elem}")
    rng = np.random.default_rng(92)
    paged = Paged(rng, [12], [62], 2, 64, 8, elem)
    sources, targets, count = (gpu(np.array(x, np.int32)) for x in ([50, 52, 55, 56, 58, 61], range(50, 56), [6]))
    torch.cuda.synchronize()
    here.kv_move_raw(paged.cache(), paged.batch(), D.KvMoves(sources=sources.data_ptr(), targets=targets.data_ptr(), counts=count.data_ptr(), strides=(6, 0), count_strides=(1, 0), most=6))
    here.sync()
    q = rng.standard_normal((1, 8, 64)).astype(np.float32)
    paged.n, paged.lengths = [1], [57]
    got = Sparse(here, paged, gpu(q), 4, 1, 1)
    got.means[int(paged.table[0, 6])] = math.nan
    for n, length in ((6, 56), (1, 57)):
        paged.starts_on, paged.lengths_on = gpu(np.array([0, n], np.int32)), gpu(np.array([length], np.int32))
        torch.cuda.synchronize()
        if n == 6:
            here.kv_page_means_raw(paged.cache(), paged.batch(), got.sparse, 6)
            here.sync()
        else:
            got.run(here)
    here.sync()
    held_to_choice(got, q)


@pytest.mark.parametrize("d", [68, 72, 76, 80, 84, 88, 92, 96])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("n,lengths", [([1, 1], [300, 33]), ([3, 50], [90, 120])])
def test_few_rows_of_heads_of_65_to_96_channels(here, case, d, page, n, lengths):  # noqa: F811
    """Channels behind the 64th go to the lanes one or two a lane."""
    case(f"few rows, {d} channels, pages of {page}, {n}")
    rng = np.random.default_rng(d + page)
    paged = Paged(rng, n, lengths, 2, d, page)
    q = rng.standard_normal((sum(n), 6, d)).astype(np.float32)
    on = gpu(q)
    held_to_definition(attend(here, paged, on).cpu().numpy(), paged, q)
    held_to_masses(Mass(here, paged, on, rng).run(here), q)
    held_to_choice(Sparse(here, paged, on, 3, 1, 1).run(here), q)
    here.sync()
