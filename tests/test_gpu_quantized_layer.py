"""GPU: the example layer end to end: 8-bit linears from GPTQ exports, the paged cache
and attention over it, in chunks and single tokens, against the layer in fp32."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "quantized_layer.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("quantized_layer", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits,tokens,steps,limit", [(8, 200, 8, 0.05), (8, 3, 3, 0.05),
                                                     (4, 150, 4, 0.25)])
def test_layer_follows_its_fp32_form(dev, example, bits, tokens, steps, limit):
    """A group of 8 bits has noise of about range/255/√12, under 1 % of its values'
    size for normal data, in each of six roundings (tokens, weights, keys, values,
    attended tokens, output weights): 5 % in all is ample.  With 4 bits, keys' and values'
    noise is about 2·3/15/√12 = 12 % of their size each."""
    outs, refs = example.serve(bits=bits, tokens=tokens, steps=steps, device="cuda:0")
    for y, ref in zip(outs, refs):
        assert y.shape == ref.shape and y.dtype is torch.bfloat16
        assert bool(torch.isfinite(y).all())
        err = float((y.float() - ref).norm() / ref.norm())
        print(f"{bits} bits, {len(y)} tokens: relative error {err:.4f}")
        assert err < limit
