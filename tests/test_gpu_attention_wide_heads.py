"""GPU: attention with heads of 160 to 256 channels over long contexts: shares of one row joined
by a whole wave, rings of scales and pages that wrap, chunks of more rows than one tile."""
import pytest
import torch

from tests._util import assert_bitexact
from tests.test_gpu_paged_attention import Batch

pytestmark = pytest.mark.gpu

WIDE = [(8, True), (8, False), (4, True), (4, False)]


@pytest.mark.parametrize("dim", [160, 256])
@pytest.mark.parametrize("bits,sym", WIDE)
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [5001]), ([1, 2, 1], [4100, 1, 2700]),
                                            ([4], [3300])], ids=str)
def test_few_rows_over_many_keys(dev, q_lens, kv_lens, bits, sym, dim):
    b = Batch(dev, q_lens, kv_lens, 4, 2, dim, 64, bits, sym, torch.float16)
    b.check(b.run(), "unsized")
    b.check(b.run(max_q=max(q_lens), max_kv=max(kv_lens)), "sized")
    b.check(b.run(max_q=1, max_kv=1), "unshared")


@pytest.mark.parametrize("dim", [160, 256])
@pytest.mark.parametrize("bits,sym", WIDE)
@pytest.mark.parametrize("q_lens,kv_lens", [([50], [1500]), ([20, 150], [1100, 2000])], ids=str)
def test_chunks_over_many_keys(dev, q_lens, kv_lens, bits, sym, dim):
    b = Batch(dev, q_lens, kv_lens, 4, 2, dim, 16, bits, sym, torch.bfloat16)
    b.check(b.run(max_q=max(q_lens), max_kv=max(kv_lens)), "shared")
    b.check(b.run(max_q=20, max_kv=1), "unshared")
    assert_bitexact(b.run(), b.run(), "again")
