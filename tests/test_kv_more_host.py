"""The host side of the operators around a paged cache, no GPU needed: the workspaces that they want, what they refuse, and their structures as the header has them."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest

from altius_amd import _lib
from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_SHAPE, ERR_UNSUPPORTED, AltiusHipError

CACHE = dict(elem=D.KV_F32, kv_heads=8, head_size=128, page_size=16, pages=100, page_stride=8 * 16 * 128, head_stride=16 * 128, slot_stride=128)
BATCH = dict(sequences=4, table_pages=50, table_stride=50)
ATTEND = dict(tokens=4, q_heads=32, q_strides=(32 * 128, 128), out_strides=(32 * 128, 128), scale=0.1, max_tokens=1, causal=1)
SPARSE = dict(means=16, page_stride=8 * 128, head_stride=128, chosen=16, most=10, first=1, last=2)
KINDS = {"cache": (CACHE, D.KvCache), "batch": (BATCH, D.KvBatch), "attend": (ATTEND, D.KvAttend), "sparse": (SPARSE, D.KvSparse)}


def described(names, changed):
    """The structures of these names; changed: {"attend.scale": ..}."""
    return [kind(**{**base, **{k.split(".")[1]: v for k, v in changed.items() if k.split(".")[0] == name}}) for name, (base, kind) in ((n, KINDS[n]) for n in names)]


def mass_workspace(**changed):
    return D.kv_attention_mass_workspace(None, *described(("cache", "batch", "attend"), changed))


def sparse_workspace(**changed):
    return D.kv_attention_sparse_workspace(None, *described(("cache", "batch", "attend", "sparse"), changed))


def plain_workspace(**changed):
    return D.kv_attention_workspace(None, *described(("cache", "batch", "attend"), changed))


def test_masses_want_statistics_and_scores_beside_attention():
    # 4 tokens of up to 800 keys, 4 query heads for each of 8: attention's own, two numbers a row and head, 4 rows of 800 scores for each of 32 pairs.
    assert mass_workspace() == plain_workspace() + 4 * 32 * 2 * 4 + 32 * 4 * 800 * 4
    # A prompt of 1000 tokens: scores are kept for as many rows as a short sequence beside it can have,
    # 32, and sums of up to 16 parts of its rows.
    prompt = {"batch.sequences": 1, "attend.tokens": 1000, "attend.max_tokens": 1000}
    most = plain_workspace(**prompt) + 1000 * 32 * 2 * 4 + 8 * 32 * 800 * 4 + 16 * 8 * 800 * 4
    assert most - 16 * 8 * 800 * 4 < mass_workspace(**prompt) <= most + 64


def test_the_workspace_of_masses_has_an_end():
    """Scores are kept up to 2^30 bytes; with more the weights are computed again."""
    long = {"batch.sequences": 64, "batch.table_pages": 1 << 16, "batch.table_stride": 1 << 16, "attend.tokens": 64}
    assert mass_workspace(**long) < plain_workspace(**long) + (1 << 30)
    assert mass_workspace(**{**long, "attend.max_keys": 4096}) <= plain_workspace(**{**long, "attend.max_keys": 4096}) + 64 * 32 * 2 * 4 + 64 * 8 * 4 * 4096 * 4


def test_chosen_pages_want_a_table_a_row():
    """Each row is a sequence of its own: what attention wants for those, their starts and lengths, and a table of 10 pages for each row and head of keys."""
    of_rows = {"batch.sequences": 4, "batch.table_pages": 10, "batch.table_stride": 80}
    up16 = lambda n: -(-n // 16) * 16  # noqa: E731
    attention = up16(plain_workspace(**of_rows))
    assert sparse_workspace() == attention + up16(5 * 4) + up16(4 * 4) + 4 * 8 * 10 * 4
    # One token of 65536 keys: scores of its 4096 pages, in 64 bits, made by blocks of their own.
    one = {"batch.sequences": 1, "batch.table_pages": 4096, "batch.table_stride": 4096, "attend.tokens": 1}
    assert sparse_workspace(**one) == up16(plain_workspace(**{**of_rows, "batch.sequences": 1, "attend.tokens": 1})) + 16 + 16 + 8 * 10 * 4 + 8 * 4096 * 8


REFUSED = [(ERR_ARG, {"cache.elem": 2}), (ERR_ARG, {"cache.page_size": 0}), (ERR_ARG, {"cache.page_stride": -4}), (ERR_ARG, {"batch.sequences": -1}), (ERR_SHAPE, {"attend.q_heads": 31}),
           (ERR_ARG, {"attend.scale": math.nan}), (ERR_UNSUPPORTED, {"cache.head_size": 260}), (ERR_UNSUPPORTED, {"cache.slot_stride": 130}), (ERR_UNSUPPORTED, {"attend.workspace": 8}),
           (ERR_UNSUPPORTED, {"attend.q": 8}), (ERR_UNSUPPORTED, {"batch.sequences": 1 << 21})]


@pytest.mark.parametrize("code,changed", REFUSED)
@pytest.mark.parametrize("workspace", [mass_workspace, sparse_workspace])
def test_what_attention_refuses_they_refuse(workspace, code, changed):
    with pytest.raises(AltiusHipError) as e:
        workspace(**changed)
    assert e.value.code == code and str(e.value)


@pytest.mark.parametrize("code,changed", [
    (ERR_UNSUPPORTED, {"attend.causal": 0}), (ERR_UNSUPPORTED, {"attend.window": 3}), (ERR_UNSUPPORTED, {"attend.slopes": 16}), (ERR_UNSUPPORTED, {"attend.prefix": 16}),
    (ERR_UNSUPPORTED, {"attend.first_keys": 16}), (ERR_ARG, {"sparse.first": -1}), (ERR_ARG, {"sparse.last": 0}), (ERR_ARG, {"sparse.last": 10}), (ERR_ARG, {"sparse.most": 2}),
    (ERR_ARG, {"sparse.first": (1 << 31) - 1, "sparse.last": (1 << 31) - 1}), (ERR_ARG, {"sparse.page_stride": -4}), (ERR_ARG, {"sparse.head_stride": 1 << 50}),
    (ERR_UNSUPPORTED, {"sparse.means": 8}), (ERR_UNSUPPORTED, {"sparse.page_stride": 1026}), (ERR_UNSUPPORTED, {"sparse.head_stride": 126}), (ERR_UNSUPPORTED, {"sparse.most": 1 << 28}),
    (ERR_UNSUPPORTED, {"sparse.most": 16385, "batch.table_pages": 16386, "batch.table_stride": 16386}), (ERR_UNSUPPORTED, {"attend.tokens": 1 << 20})])
def test_chosen_pages_refuse(code, changed):
    with pytest.raises(AltiusHipError) as e:
        sparse_workspace(**changed)
    assert e.value.code == code and str(e.value)


def test_all_pages_may_be_chosen_whatever_their_number():
    many = {"batch.table_pages": 16385, "batch.table_stride": 16385}
    sparse_workspace(**many, **{"sparse.most": 16384})
    sparse_workspace(**many, **{"sparse.most": 16385})
    sparse_workspace(**many, **{"sparse.most": 50000, "attend.max_keys": 400})


def test_null_arguments_are_refused():
    L = _lib.lib()
    n = ctypes.c_size_t()
    cache, batch, attend, sparse = described(("cache", "batch", "attend", "sparse"), {})
    assert L.ahip_kv_attention_mass_workspace(None, None, None, None, ctypes.byref(n)) == ERR_ARG
    assert L.ahip_kv_attention_mass_workspace(None, cache, batch, None, ctypes.byref(n)) == ERR_ARG
    assert L.ahip_kv_attention_mass_workspace(None, cache, batch, attend, None) == ERR_ARG
    assert L.ahip_kv_attention_sparse_workspace(None, None, batch, attend, sparse, ctypes.byref(n)) == ERR_ARG
    assert L.ahip_kv_attention_sparse_workspace(None, cache, batch, attend, None, ctypes.byref(n)) == ERR_ARG
    assert L.ahip_kv_attention_sparse_workspace(None, cache, batch, attend, sparse, None) == ERR_ARG
    assert L.ahip_kv_attention_tree(None, None, None, None, None) == ERR_ARG and L.ahip_kv_attention_mass(None, None, None, None, None, 1.0, None) == ERR_ARG
    assert L.ahip_kv_evict(None, None, None, None, None) == ERR_ARG and L.ahip_kv_move(None, None, None, None, None) == ERR_ARG
    assert L.ahip_kv_attention_sparse(None, None, None, None, None) == ERR_ARG and L.ahip_kv_page_means(None, None, None, None, 0, 0) == ERR_ARG


def test_the_workspace_of_attention_is_enough_for_trees():
    """Whose keys are cut where a piece's are not: 16 of up to 48 tokens behind up to 7952."""
    trees = {"cache.elem": D.KV_BF16, "batch.sequences": 16, "batch.table_pages": 500, "batch.table_stride": 500, "attend.tokens": 16 * 48, "attend.max_tokens": 48}
    assert plain_workspace(**trees) > plain_workspace(**{**trees, "attend.causal": 0})


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_structures_are_the_headers(tmp_path):
    kinds = {"ahip_kv_history": D.KvHistory, "ahip_kv_eviction": D.KvEviction, "ahip_kv_moves": D.KvMoves, "ahip_kv_sparse": D.KvSparse}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f' printf("%zu\\n", offsetof({c}, {f[0]}));' for f in kind._fields_) for c, kind in kinds.items()]
    source = tmp_path / "sizes.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"altius_hip.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-I", include, str(source), "-o", str(tmp_path / "sizes")], check=True)
    told = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert told == [x for kind in kinds.values() for x in [ctypes.sizeof(kind)] + [getattr(kind, f[0]).offset for f in kind._fields_]]
