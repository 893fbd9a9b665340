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


def test_layers_of_any_size_run_after_any_other_threads():
    """How much shared memory a kernel's launches may have is one setting for the
    whole process: a small layer of one thread leaves room for a larger one of another."""
    calls = []
    for rows, cols in ((128, 128), (256, 1024), (1000, 2048), (2048, 4096), (640, 8192)):
        layer = quant_linear(rows, cols)
        for m in (1, 8, 70, 300):
            x = torch.randn(m, cols, device="cuda").to(torch.float16)
            calls.append(lambda layer=layer, x=x: layer(x))
    want = [f() for f in calls]
    for small in calls:
        in_thread(small)
        for f, y in zip(calls, want):
            assert torch.allclose(f(), y, rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("small,large", [(1, 16), (4, 12)])
def test_decode_attention_of_any_group(small, large):
    """The dense cache's attention: its shared memory grows with the query heads of a kv head."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tensorshrink_b200 import kernels

    def attend(group):
        g = torch.Generator(device="cuda").manual_seed(group)
        qkv = torch.randn(2, (group + 2) * 128, generator=g, device="cuda").to(torch.bfloat16)
        k, v = (torch.randn(2, 1, 64, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        pos = torch.full((1,), 40, dtype=torch.int64, device="cuda")
        cos, sin = torch.ones(64, 64, device="cuda"), torch.zeros(64, 64, device="cuda")
        return kernels.decode_attention(qkv, group, 1, 128, pos, cos, sin, k, v, 64)
    want = attend(large)
    in_thread(lambda: attend(small))
    assert torch.equal(attend(large), want)
