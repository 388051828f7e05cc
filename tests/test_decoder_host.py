"""The host side of the decoder's operators, no GPU needed: frequencies of rotary positions, the workspace that attention
over a paged cache wants, and what it refuses."""
import ctypes
import math

import numpy as np
import pytest

from altius_amd import _lib
from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_SHAPE, ERR_UNSUPPORTED, AltiusHipError


def test_frequencies_by_their_formulas():
    plain = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    np.testing.assert_allclose(D.rotary_frequencies(64), plain, rtol=1e-14)
    np.testing.assert_allclose(D.rotary_frequencies(64, base=5e5), 5e5 ** (-np.arange(0, 64, 2) / 64), rtol=1e-14)
    np.testing.assert_allclose(D.rotary_frequencies(64, scaling=D.ROTARY_LINEAR, factor=4), plain / 4, rtol=1e-14)
    stretched = D.rotary_frequencies(64, scaling=D.ROTARY_BASE, factor=8)
    assert stretched[0] == 1.0 and math.isclose(stretched[-1], plain[-1] / 8, rel_tol=1e-12) and (np.diff(stretched / plain) < 0).all()
    by_turns = D.rotary_frequencies(64, scaling=D.ROTARY_TURNS, factor=8, length=1024, slow_turns=1, fast_turns=4)
    turns = 1024 * plain / (2 * math.pi)
    keep = np.clip((turns - 1) / 3, 0, 1)
    np.testing.assert_allclose(by_turns, plain * (keep + (1 - keep) / 8), rtol=1e-13)
    assert (by_turns[turns >= 4] == D.rotary_frequencies(64)[turns >= 4]).all() and D.rotary_frequencies(0).size == 0


@pytest.mark.parametrize("arguments", [dict(dim=7), dict(dim=-2), dict(dim=8, base=0.0), dict(dim=8, base=math.inf), dict(dim=8, scaling=4), dict(dim=8, scaling=-1),
                                       dict(dim=8, scaling=D.ROTARY_LINEAR, factor=0.0), dict(dim=8, scaling=D.ROTARY_LINEAR, factor=math.nan),
                                       dict(dim=2, scaling=D.ROTARY_BASE, factor=2.0), dict(dim=8, scaling=D.ROTARY_TURNS, factor=2.0),
                                       dict(dim=8, scaling=D.ROTARY_TURNS, factor=2.0, length=64.0, slow_turns=4.0, fast_turns=4.0)])
def test_frequencies_refused(arguments):
    with pytest.raises(AltiusHipError) as e:
        D.rotary_frequencies(**arguments)
    assert e.value.code == ERR_ARG


CACHE = dict(elem=D.KV_F32, kv_heads=8, head_size=128, page_size=16, pages=100, page_stride=8 * 16 * 128, head_stride=16 * 128, slot_stride=128)
BATCH = dict(sequences=4, table_pages=50, table_stride=50)
ATTEND = dict(tokens=4, q_heads=32, q_strides=(32 * 128, 128), out_strides=(32 * 128, 128), scale=0.1, max_tokens=1)


def workspace(**changed):
    one = lambda base, kind: kind(**{**base, **{k: v for k, v in changed.items() if k in base or (k in dict(kind._fields_) and k not in {**CACHE, **BATCH, **ATTEND})}})  # noqa: E731
    return D.kv_attention_workspace(None, one(CACHE, D.KvCache), one(BATCH, D.KvBatch), one(ATTEND, D.KvAttend))


def test_the_workspace_goes_by_the_sizes():
    few = workspace()
    assert few >= 0 and few % 4 == 0
    long = workspace(sequences=1, tokens=1, table_pages=4096, table_stride=4096)
    row = (128 + 2) * 4
    assert long > 0 and long % row == 0 and long // row % 32 == 0  # whole splits of 32 rows
    assert workspace(sequences=1, tokens=1, table_pages=4096, table_stride=4096, max_keys=64) == 0  # short sequences are not split
    # Many rows of a sequence have blocks enough: what is kept does not grow with the prompt.
    assert workspace(sequences=1, tokens=100000, max_tokens=100000, table_pages=8000) <= 64 * 8 * 8000 * 16 // 64 * row


@pytest.mark.parametrize("code,changed", [
    (ERR_ARG, dict(elem=2)), (ERR_ARG, dict(kv_heads=0)), (ERR_ARG, dict(kv_heads=-1)), (ERR_ARG, dict(kv_heads=40000, q_heads=40000)), (ERR_ARG, dict(page_size=0)),
    (ERR_ARG, dict(head_size=0)), (ERR_ARG, dict(pages=-1)), (ERR_ARG, dict(pages=1 << 31)), (ERR_ARG, dict(page_stride=-4)), (ERR_ARG, dict(slot_stride=1 << 31)),
    (ERR_ARG, dict(sequences=-1)), (ERR_ARG, dict(table_pages=-1)), (ERR_ARG, dict(table_stride=-1)), (ERR_UNSUPPORTED, dict(table_pages=1 << 30)),
    (ERR_SHAPE, dict(q_heads=31)), (ERR_SHAPE, dict(q_heads=0)), (ERR_SHAPE, dict(q_heads=-8)), (ERR_ARG, dict(scale=math.inf)), (ERR_ARG, dict(scale=math.nan)),
    (ERR_ARG, dict(softcap=-1.0)), (ERR_ARG, dict(softcap=math.nan)), (ERR_ARG, dict(window=-1)), (ERR_UNSUPPORTED, dict(head_size=260)),
    (ERR_UNSUPPORTED, dict(head_size=130)), (ERR_UNSUPPORTED, dict(elem=D.KV_BF16, head_size=100)), (ERR_UNSUPPORTED, dict(slot_stride=130)),
    (ERR_UNSUPPORTED, dict(elem=D.KV_BF16, page_stride=4)), (ERR_UNSUPPORTED, dict(q=8)), (ERR_UNSUPPORTED, dict(out=4)), (ERR_UNSUPPORTED, dict(keys=2)),
    (ERR_UNSUPPORTED, dict(workspace=8)), (ERR_UNSUPPORTED, dict(q_strides=(4096, 126))), (ERR_UNSUPPORTED, dict(out_strides=(4098, 128))),
    (ERR_UNSUPPORTED, dict(tokens=1 << 23))])
def test_attention_refuses(code, changed):
    with pytest.raises(AltiusHipError) as e:
        workspace(**changed)
    assert e.value.code == code and str(e.value)


@pytest.mark.parametrize("changed", [dict(tokens=(1 << 23) - 1, max_tokens=0, q_heads=8 * 129), dict(sequences=1 << 21), dict(table_pages=(1 << 27) - 1, table_stride=1 << 27), dict(sequences=(1 << 31) - 1, kv_heads=32767, q_heads=32767)])
def test_attention_refuses_what_its_row_numbers_do_not_hold(changed):
    with pytest.raises(AltiusHipError) as e:
        workspace(**changed)
    assert e.value.code == ERR_UNSUPPORTED


@pytest.mark.parametrize("elem", [D.KV_F32, D.KV_BF16])
@pytest.mark.parametrize("head_size", [64, 96, 128, 256])
def test_the_workspace_has_an_end(elem, head_size):
    """However long the sequences and however many, no more parts are kept than blocks at work at once and one a row tile."""
    cache = dict(elem=elem, head_size=head_size, page_stride=8 * 16 * head_size, head_stride=16 * head_size, slot_stride=head_size)
    for sequences in (1, 3, 64, 500):
        for max_tokens in (1, 4, 33, 400):
            for table_pages in (1, 30, 5000, 1 << 26):
                bytes_ = workspace(sequences=sequences, tokens=sequences * max_tokens, max_tokens=max_tokens, table_pages=table_pages, table_stride=table_pages, **cache)
                rows = max_tokens * 4
                few, many = 8 * sequences * -(-min(rows, 32) // 16), 8 * sequences * -(-rows // 128)
                assert bytes_ <= ((1024 + few) * 16 + (1024 + many) * 128) * (head_size + 2) * 4


def test_null_arguments_are_refused():
    L = _lib.lib()
    n = ctypes.c_size_t()
    assert L.ahip_kv_attention_workspace(None, None, None, None, ctypes.byref(n)) == ERR_ARG
    assert L.ahip_kv_attention_workspace(None, D.KvCache(**CACHE), D.KvBatch(**BATCH), D.KvAttend(**ATTEND), None) == ERR_ARG
    assert L.ahip_rotary_heads(None, None, None) == ERR_ARG and L.ahip_kv_append(None, None, None, None, None) == ERR_ARG
    assert L.ahip_kv_attention(None, None, None, None) == ERR_ARG
    assert L.ahip_rotary_frequencies(None, 8, 10000.0, 0, 1.0, 0.0, 0.0, 0.0) == ERR_ARG


@pytest.mark.parametrize("changed", [dict(softcap=1e-40), dict(softcap=1e-30), dict(softcap=1e30), dict(softcap=2e38), dict(softcap=3e38, scale=0.0), dict(softcap=3e38, scale=1e20),
                                     dict(softcap=1.0, scale=1e-20), dict(softcap=1.0, scale=-1e20), dict(scale=3e38)])
def test_caps_that_fp32_does_not_hold_beside_the_scale_are_refused(changed):
    with pytest.raises(AltiusHipError) as e:
        workspace(**changed)
    assert e.value.code == ERR_ARG
    for fine in (dict(softcap=1e-18), dict(softcap=1e18), dict(softcap=50.0, scale=-0.1), dict(softcap=1e-30, scale=0.0), dict(softcap=2e38, scale=1e20)):
        workspace(**fine)


def parts_bytes(units, tile, at_once, least, tiles, head_size=128):
    """Parts of at least `least` units of 64 keys, as many as blocks at work at once and one more a row tile and kv head; rows of a maximum, a
    sum and head_size channels."""
    return (min(at_once, units * tiles // least) + tiles) * tile * (2 + head_size) * 4


def test_the_workspace_is_what_the_parts_hold():
    """256 CUs: 512 blocks of 16 rows at work at once (fp32, 128 channels), 256 of 128 rows; parts of 128 keys at least."""
    # 4 tokens of up to 800 keys: 13 units of 64 keys for each of 32 (sequence, kv head).
    assert workspace() == parts_bytes(13, 16, 512, 2, 32)
    # One token of up to 65536 keys: more units than blocks at work at once.
    one = dict(sequences=1, tokens=1, table_pages=4096, table_stride=4096)
    assert workspace(**one) == parts_bytes(1024, 16, 512, 2, 8)
    # 200 tokens: two blocks a place and more, nothing is cut.
    assert workspace(sequences=200, tokens=200) == 0
    # A piece of 300 tokens (10 row tiles of 128 rows) behind 65536 keys at most, whose keys are cut, and 16 rows of it if it is shorter.
    assert workspace(sequences=1, tokens=300, max_tokens=300, table_pages=4096, table_stride=4096) == parts_bytes(1024, 128, 256, 2, 80) + parts_bytes(1024, 16, 512, 2, 8)
    # Prompts of so many row tiles that none is cut: what remains is for 32 rows of a shorter piece, and does not grow with the prompt.
    long = [workspace(sequences=1, tokens=t, max_tokens=t, table_pages=8000, table_stride=8000) for t in (1000, 10000, 100000)]
    assert long == [parts_bytes(2000, 16, 512, 2, 16)] * 3


@pytest.mark.parametrize("arguments", [dict(dim=4, factor=1e200), dict(dim=4, factor=1e-200), dict(dim=8, base=1e300, factor=1e10)])
def test_a_stretched_base_that_64_bits_do_not_hold_is_refused(arguments):
    with pytest.raises(AltiusHipError) as e:
        D.rotary_frequencies(scaling=D.ROTARY_BASE, **arguments)
    assert e.value.code == ERR_ARG
