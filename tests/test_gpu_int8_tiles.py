"""GPU: every tile form of the 8-bit product, on each side of the numbers of tiles that choose
it, with rows, columns and channels that end inside a tile, both grids, all types, output rows
that are and are not whole 16-byte pieces."""
import pytest
import torch

from oracle import serving
from tests.test_gpu_int8_linear import DTYPES, _check, _tokens, _weights

pytestmark = pytest.mark.gpu


def tiles(T, N, size):
    return -(-T // size) * -(-N // size)


# form (tile, groups that share K) and (tokens, channels, columns)
FORMS = [
    (256, 1, 3329, 3585, 130), (256, 1, 2823, 4096, 700), (256, 1, 257, 24577, 257),
    (128, 1, 1793, 2001, 272), (128, 1, 1792, 2048, 1025), (128, 1, 65, 28672, 64),
    (64, 1, 1473, 1473, 96), (64, 1, 1472, 1536, 515), (64, 1, 70, 16500, 33),
    (64, 2, 1100, 1100, 1), (64, 2, 1088, 1152, 300), (64, 2, 100, 8300, 1300),
    (64, 4, 1000, 1000, 40), (64, 4, 1024, 1024, 768), (64, 4, 100, 8190, 2050),
]


@pytest.mark.parametrize("size,groups,T,N,K", FORMS)
def test_every_tile_form(dev, size, groups, T, N, K):
    from g2ptq_amd import Int8Linear
    form = (256, 1) if tiles(T, N, 256) >= 192 else (128, 1) if tiles(T, N, 128) >= 224 else \
        (64, 1 if tiles(T, N, 64) > 512 else 2 if tiles(T, N, 64) > 256 else 4)
    assert form == (size, groups) and T > 64
    w, wscale, bias = _weights(N, K, T + N)
    for sym in (True, False):
        b = None if sym else bias
        lin = Int8Linear(w.to(dev), wscale.to(dev), bias=None if b is None else b.to(dev), sym=sym)
        for dtype in DTYPES:
            x = _tokens(T, K, dtype, T + K)
            rc, rs, rz = serving.quantize(x, 8, sym)
            _check(lin(x.to(dev)), rc, rs, rz, w, wscale, b, dtype)


@pytest.mark.parametrize("size,below,above", [
    (256, (2900, 3800), (2900, 3900)), (128, (1700, 1900), (1700, 2000)),
    (64, (1472, 1400), (1472, 1472)), (64, (1000, 1024), (1000, 1025))])
def test_each_side_of_the_numbers_of_tiles(dev, size, below, above):
    """One more tile chooses the next form: both give the product."""
    from g2ptq_amd import Int8Linear
    K = 200
    for T, N in (below, above):
        w, wscale, bias = _weights(N, K, N)
        x = _tokens(T, K, torch.float16, T)
        rc, rs, rz = serving.quantize(x, 8, False)
        lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=False)
        _check(lin(x.to(dev)), rc, rs, rz, w, wscale, bias, torch.float16)
