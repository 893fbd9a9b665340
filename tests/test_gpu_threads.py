"""The operators called from host threads of their own: threads that have called
nothing else yet, and layers of unlike size in several of them."""

from __future__ import annotations

import threading

import pytest
import torch

from oracle import goap

pytestmark = pytest.mark.gpu


def in_thread(f):
    out = []

    def work():
        try:
            out.append(f())
        except Exception as e:
            out.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(out[0], Exception):
        raise out[0]
    return out[0]


def quant_linear(rows, cols):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as ts
    w = torch.from_numpy(goap.student_t_weights((rows, cols), seed=rows)).cuda()
    return ts.QuantLinear.from_device_quant(ts.quantize_device(w, bits=4, group_size=128, outlier_frac=0.002))


def test_a_layer_is_the_first_call_of_a_thread():
    layer, x = quant_linear(2048, 4096), torch.randn(300, 4096, device="cuda").to(torch.float16)
    want = layer(x)
    assert torch.allclose(in_thread(lambda: layer(x)), want, rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_an_fp4_product_is_the_first_call_of_a_thread(m):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as ts
    x, w = torch.randn(m, 512, device="cuda").to(torch.bfloat16), ts.fp4_quantize(torch.randn(640, 512, device="cuda"))
    a = ts.fp4_quantize(x)
    for f in (lambda: ts.fp4_matmul(a, w), lambda: ts.fp4_linear(x, w), lambda: ts.fp4_quantize(x).codes,
              lambda: ts.fp4_dequantize(w)):
        want = f()
        assert torch.equal(in_thread(f), want)
