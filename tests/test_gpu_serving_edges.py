"""GPU: the operators of a quantized layer at the edges that a user's program reaches."""
import pytest
import torch

from oracle import serving
from tests._util import assert_bitexact, gen
from tests.test_gpu_int8_linear import _check, _tokens, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sym", [True, False])
def test_casts_of_a_model_leave_its_int8_linears_right(dev, sym):
    from g2ptq_amd import Int8Linear, int8_matmul, quantize_tokens
    w, wscale, bias = _weights(70, 130, 3)
    for T in (1, 40):
        x = _tokens(T, 130, torch.float16, T)
        rc, rs, rz = serving.quantize(x, 8, sym)
        for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                     lambda m: m.cpu().half().to(dev)):
            lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=sym)
            cast(torch.nn.Sequential(torch.nn.Linear(8, 8, device=dev), lin))
            y = lin(x.to(dev))
            _check(y, rc, rs, rz, w, wscale, bias, torch.float16)
            c, s, z = quantize_tokens(x.to(dev), sym=sym)
            assert_bitexact(int8_matmul(c, s, lin, zero=z, dtype=torch.float16), y, "apart")
    lin.load_state_dict({k: v.half() if v.is_floating_point() else v
                         for k, v in lin.state_dict().items()}, assign=True)
    for call in (lambda: lin(x.to(dev)), lambda: int8_matmul(c, s, lin, zero=z)):
        with pytest.raises(ValueError, match="weight_scale is torch.float16"):
            call()
    lin.load_state_dict(Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev),
                                   sym=sym).state_dict(), assign=True)
    lin.weight_scale = lin.weight_scale.cpu()
    with pytest.raises(ValueError, match="weight_scale is .* on cpu"):
        lin(x.to(dev))
