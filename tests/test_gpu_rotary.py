"""Rotary positions and norms of heads (ahip_rotary_heads) against their definition in float64."""
import numpy as np
import pytest
import torch

from altius_amd import device as D
from altius_amd._lib import ERR_ARG, ERR_SHAPE, ERR_UNSUPPORTED, AltiusHipError
from decoder_oracle import normed, turned, turned_bound

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture
def here():
    with D.Context(0, stream=torch.cuda.current_stream().cuda_stream) as c:
        yield c


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rotate(ctx, x, positions, frequencies, interleaved, gamma=None, magnitude=1.0, out=None, x_strides=None, out_strides=None, **more):
    """x [b, t, h, d] on the GPU in whatever order its strides say."""
    b, t, h, d = x.shape
    out = torch.full_like(x, 7.0) if out is None else out
    f = gpu(np.asarray(frequencies, np.float64)) if len(frequencies) else None
    rows = D.HeadRows(out=out.data_ptr(), x=x.data_ptr(), batch=b, tokens=t, heads=h, head_size=d, x_strides=x.stride()[:3], out_strides=out.stride()[:3],
                      gamma=gamma.data_ptr() if gamma is not None else None, epsilon=EPS, **more)
    if positions is not None:
        rows.positions, rows.position_size = positions.data_ptr(), positions.element_size()
    ctx.rotary_raw(rows, D.Rotary(f.data_ptr() if f is not None else None, 2 * len(frequencies), int(interleaved), magnitude))
    torch.cuda.synchronize()
    ctx.sync()
    return out


def held(got, x, positions, frequencies, interleaved, gamma=None, magnitude=1.0):
    n = normed(x, gamma, EPS)
    want = turned(n, positions, frequencies, interleaved, magnitude)
    bound = turned_bound(n, len(frequencies), interleaved, gamma, magnitude) + 1e-37
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= bound).all(), f"{(off / bound).max()} times the bound at {np.unravel_index((off / bound).argmax(), off.shape)}"


SIZES = [(64, 64), (64, 32), (128, 128), (80, 40), (96, 96), (256, 64), (512, 512), (512, 8), (20, 12), (7, 6), (13, 4), (600, 600), (130, 66), (8, 2), (1, 0), (68, 64)]


@pytest.mark.parametrize("d,dim", SIZES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_heads_turn(here, case, d, dim, interleaved, norm):
    case(f"rotary d {d} dim {dim} interleaved {interleaved} norm {norm}")
    rng = np.random.default_rng(d * 31 + dim)
    x = rng.standard_normal((2, 5, 3, d)).astype(np.float32)
    positions = rng.integers(-50, 200000, (2, 5)).astype(np.int32)
    frequencies = D.rotary_frequencies(dim) if dim else np.empty(0)
    gamma = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32) if norm else None
    got = rotate(here, gpu(x), gpu(positions), frequencies, interleaved, gpu(gamma) if norm else None, position_stride=5, magnitude=1.25)
    held(got.cpu().numpy(), x, positions, frequencies, interleaved, gamma, 1.25)


@pytest.mark.parametrize("b,t,h", [(1, 1, 1), (1, 1, 12), (3, 17, 9), (1, 1000, 1), (2, 3, 100), (1, 300, 33)])
@pytest.mark.parametrize("order", ["token", "head"])
def test_numbers_of_tokens_and_heads(here, case, b, t, h, order):
    case(f"rotary [{b}, {t}, {h}, 64] {order}")
    rng = np.random.default_rng(t + h)
    x = rng.standard_normal((b, t, h, 64)).astype(np.float32)
    on = gpu(x) if order == "token" else gpu(x.transpose(0, 2, 1, 3)).transpose(1, 2)
    f = D.rotary_frequencies(64)
    got = rotate(here, on, None, f, False, first_position=41)
    held(got.cpu().numpy(), x, np.broadcast_to(41 + np.arange(t), (b, t)), f, False)


def test_positions_of_either_type_shared_or_not(here, case):
    case("rotary positions")
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 6, 2, 32)).astype(np.float32)
    f = D.rotary_frequencies(32)
    p = rng.integers(0, 1 << 40, (3, 6))
    held(rotate(here, gpu(x), gpu(p), f * 1e-7, True, position_stride=6).cpu().numpy(), x, p, f * 1e-7, True)
    held(rotate(here, gpu(x), gpu(p[0].astype(np.int32) & 0xFFFFF), f, True).cpu().numpy(), x, np.broadcast_to(p[0].astype(np.int32) & 0xFFFFF, (3, 6)), f, True)


def test_in_place_and_beside_other_columns(here, case):
    """Queries and keys as column blocks of one packed product, turned where they are: the values' columns stay."""
    case("rotary in place")
    rng = np.random.default_rng(6)
    packed = rng.standard_normal((1, 11, 9, 64)).astype(np.float32)
    f, on = D.rotary_frequencies(64), gpu(packed)
    rotate(here, on[:, :, :6], None, f, False, out=on[:, :, :6])
    got = on.cpu().numpy()
    held(got[:, :, :6], packed[:, :, :6], np.arange(11)[None], f, False)
    assert (got[:, :, 6:] == packed[:, :, 6:]).all()


def test_unaligned_rows_take_the_other_kernel(here, case):
    case("rotary unaligned")
    rng = np.random.default_rng(7)
    x = rng.standard_normal((1, 4, 3, 67)).astype(np.float32)
    on, f = gpu(x), D.rotary_frequencies(64)
    got = rotate(here, on[..., 1:65], None, f, False, first_position=3, out=on[..., 1:65])
    held(got.cpu().numpy(), x[..., 1:65], 3 + np.arange(4)[None], f, False)
    assert (on.cpu().numpy()[..., 65:] == x[..., 65:]).all() and (on.cpu().numpy()[..., 0] == x[..., 0]).all()


def test_channels_that_stay_keep_their_bits(here, case):
    """Infinities, NaN and negative zeros behind the part that turns come through as they are."""
    case("rotary, what stays")
    x = np.zeros((1, 2, 1, 24), np.float32)
    x[..., 12:] = np.array([np.inf, -np.inf, -0.0, 3.5, np.nan, 1e38, -1e-40, 0, 1, 2, 3, 4], np.float32)
    for interleaved in (False, True):
        got = rotate(here, gpu(x), None, D.rotary_frequencies(12), interleaved).cpu().numpy()
        np.testing.assert_array_equal(got[..., 12:].view(np.uint32), x[..., 12:].view(np.uint32))
        assert (got[..., :12] == 0).all()


def test_a_row_of_zeros_and_a_large_one_are_normed(here, case):
    case("norm of zeros")
    x = np.zeros((1, 2, 1, 64), np.float32)
    x[0, 1] = 1e15
    gamma = np.full(64, 2.0, np.float32)
    got = rotate(here, gpu(x), None, np.empty(0), False, gpu(gamma)).cpu().numpy()
    assert (got[0, 0] == 0).all()
    np.testing.assert_allclose(got[0, 1], 2.0, rtol=16 * 2.0 ** -24)


def test_recorded_and_replayed(here, case):
    """A recorded call reads the positions anew on every replay."""
    case("rotary replay")
    rng = np.random.default_rng(8)
    x, f = rng.standard_normal((1, 5, 4, 64)).astype(np.float32), D.rotary_frequencies(64)
    on, positions, freq = gpu(x), torch.zeros(5, dtype=torch.int32, device="cuda"), gpu(f)
    out = torch.zeros_like(on)
    stream = torch.cuda.Stream()
    with D.Context(0, stream=stream.cuda_stream) as c:
        rows = D.HeadRows(out=out.data_ptr(), x=on.data_ptr(), batch=1, tokens=5, heads=4, head_size=64, x_strides=on.stride()[:3], out_strides=on.stride()[:3],
                          positions=positions.data_ptr())
        rotary = D.Rotary(freq.data_ptr(), 64)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.rotary_raw(rows, rotary)
        for first in (0, 7, 100000):
            positions.copy_(torch.arange(first, first + 5, dtype=torch.int32))
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            held(out.cpu().numpy(), x, np.arange(first, first + 5)[None], f, False)


def test_refusals(here, case):
    case("rotary refusals")
    x = torch.zeros((1, 2, 2, 8), device="cuda")
    f = gpu(D.rotary_frequencies(8))

    def code(rotary, **more):
        fields = dict(out=x.data_ptr(), x=x.data_ptr(), batch=1, tokens=2, heads=2, head_size=8, x_strides=x.stride()[:3], out_strides=x.stride()[:3])
        try:
            here.rotary_raw(D.HeadRows(**{**fields, **more}), rotary)
        except AltiusHipError as e:
            return e.code
        return 0

    turns = D.Rotary(f.data_ptr(), 8)
    assert code(turns) == 0
    assert code(None) == ERR_ARG                                     # nothing to do
    assert code(D.Rotary(f.data_ptr(), 7)) == ERR_SHAPE and code(D.Rotary(f.data_ptr(), 10)) == ERR_SHAPE and code(D.Rotary(f.data_ptr(), -2)) == ERR_SHAPE
    assert code(D.Rotary(f.data_ptr(), 8, 2)) == ERR_ARG and code(D.Rotary(None, 8)) == ERR_ARG
    assert code(turns, x=None) == ERR_ARG and code(turns, out=None) == ERR_ARG
    assert code(turns, positions=x.data_ptr(), position_size=2) == ERR_ARG
    assert code(turns, positions=x.data_ptr() + 4, position_size=8) == ERR_ARG
    assert code(turns, out_strides=(32, 8, 16)) == ERR_ARG           # in place with other strides
    assert code(turns, tokens=1 << 24) == ERR_UNSUPPORTED and code(turns, heads=1 << 16) == ERR_UNSUPPORTED
    assert code(turns, tokens=0, x=None) == 0 and code(turns, heads=0) == 0 and code(turns, batch=0) == 0
    here.sync()
