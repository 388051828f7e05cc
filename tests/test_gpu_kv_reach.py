"""The operators around a paged cache at sizes that choose among their kernels or that a sum feels: sums of many weights."""
import numpy as np
import pytest
import torch

from decoder_oracle import STEP
from test_gpu_kv_cache import Paged, here  # noqa: F401 (a fixture)
from test_gpu_kv_mass import Mass

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
