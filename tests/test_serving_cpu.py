"""Host side of the fp4 and paged operators, without a GPU: struct layouts,
sizes, and refusals that come before any CUDA call."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

import tensorshrink_b200 as ts
from tensorshrink_b200 import _C, fp4


def test_struct_layouts_match_header():
    assert C.sizeof(_C.TsPagedCache) == 8 * 2 + 8 * 3 + 8 + 8 + 8 * 3 + 4 * 8
    assert C.sizeof(_C.TsFp4Tensor) == 8 * 3 + 8 * 2 + 4 * 2


@pytest.mark.parametrize("rows,cols", [(0, 1), (1, 1), (1, 64), (128, 65), (129, 128), (300, 4099)])
def test_scale_sizes(rows, cols):
    for name, code in fp4.FORMATS.items():
        tiles = -(-rows // 128) * -(-(-(-cols // 64) * 64 // fp4.BLOCK[name]) // 4)
        assert fp4.scales_nbytes(rows, cols, name) == tiles * 512
        assert _C.load().ts_fp4_scales_bytes(rows, cols, code) == tiles * 512


def tensor(**kw):
    t = _C.TsFp4Tensor()
    t.codes, t.scales, t.rows, t.cols, t.format = 4096, 4096, 4, 64, 0
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def cache(**kw):
    c = _C.TsPagedCache()
    for name in ("k_pages", "v_pages", "page_table", "seq_lens"):
        setattr(c, name, 4096)
    c.page_stride, c.head_stride, c.token_stride = 1024, 1024, 64
    c.dtype, c.batch, c.n_kv, c.head_dim, c.page_size, c.num_pages, c.max_pages = _C.TS_BF16, 2, 1, 64, 16, 4, 2
    for k, v in kw.items():
        setattr(c, k, v)
    return c


INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4


@pytest.mark.parametrize("kw,rc", [(dict(cols=0), INVALID), (dict(format=7), UNSUPPORTED), (dict(codes=None), INVALID),
                                   (dict(codes=4100), INVALID), (dict(rows=-1), INVALID)])
def test_fp4_tensors_are_checked(kw, rc):
    lib = _C.load()
    t = tensor(**kw)
    assert lib.ts_fp4_dequantize(t, 4096, _C.TS_F32, 64, None) == rc
    assert lib.ts_fp4_matmul(t, tensor(), None, 0, 4096, _C.TS_F32, 64, None, 0, None) == rc
    assert lib.ts_fp4_quantize(4096, _C.TS_BF16, 64, t, 0, None, 0, None) == rc
    assert lib.ts_last_error()


def test_fp4_calls_are_checked():
    lib = _C.load()
    t = tensor()
    assert lib.ts_fp4_quantize(4096, 9, 64, t, 0, None, 0, None) == UNSUPPORTED
    assert lib.ts_fp4_quantize(4096, _C.TS_BF16, 64, t, 1, None, 0, None) == INVALID          # nowhere to put the scale
    assert lib.ts_fp4_quantize(4096, _C.TS_BF16, 64, tensor(global_scale=4096), 1, None, 0, None) == WORKSPACE
    assert lib.ts_fp4_quantize(None, _C.TS_BF16, 64, t, 0, None, 0, None) == INVALID
    assert lib.ts_fp4_matmul(t, tensor(format=1), None, 0, 4096, _C.TS_F32, 64, None, 0, None) == INVALID
    assert lib.ts_fp4_matmul(t, tensor(cols=128), None, 0, 4096, _C.TS_F32, 64, None, 0, None) == INVALID
    assert lib.ts_fp4_matmul(t, t, None, 0, 4096, 5, 64, None, 0, None) == UNSUPPORTED
    # nothing to do is no error
    assert lib.ts_fp4_matmul(tensor(rows=0), t, None, 0, None, _C.TS_F32, 64, None, 0, None) == 0
    assert lib.ts_fp4_dequantize(tensor(rows=0, codes=None, scales=None), None, _C.TS_F32, 64, None) == 0


@pytest.mark.parametrize("kw,rc", [(dict(k_pages=None), INVALID), (dict(dtype=_C.TS_F32), UNSUPPORTED),
                                   (dict(head_dim=40), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED),
                                   (dict(page_size=0), INVALID), (dict(token_stride=60), INVALID),
                                   (dict(v_pages=4104), INVALID), (dict(max_pages=1 << 30), INVALID)])
def test_caches_are_checked(kw, rc):
    lib = _C.load()
    c = cache(**kw)
    three = (C.c_int64 * 3)(64, 64, 64)
    assert lib.ts_paged_append(4096, three, 4096, three, 1, None, c, None, None, None, 0, None, None, None) == rc
    assert lib.ts_paged_decode_attention(4096, 192, 1, c, 4096, None, None, 0, 0.1, 0, 4096, 64, None, 0, None) == rc
    assert lib.ts_paged_evict(c, 4, 0, None, 0, None) == rc


def test_paged_calls_are_checked():
    lib = _C.load()

    def attend(c=None, n_q=1, pos=4096, cos=None, sin=None, scale=0.1, acc=0, out=4096, stride=64):
        return lib.ts_paged_decode_attention(4096, 192, n_q, c or cache(), pos, cos, sin, 0, scale, acc, out, stride, None,
                                             0, None)
    assert attend(n_q=0) == INVALID and attend(cache(n_kv=2), n_q=3) == INVALID
    assert attend(cos=4096) == INVALID and attend(out=None) == INVALID
    assert attend(pos=None, cos=4096, sin=4096) == INVALID
    assert attend(scale=0.0) == INVALID and attend(scale=float("nan")) == INVALID and attend(scale=float("inf")) == INVALID
    assert attend(acc=1) == INVALID and attend(stride=63) == INVALID
    assert attend(cache(batch=0)) == 0
    three, odd = (C.c_int64 * 3)(64, 64, 64), (C.c_int64 * 3)(64, 60, 64)
    assert lib.ts_paged_append(4096, odd, 4096, three, 1, None, cache(), None, None, None, 0, None, None, None) == INVALID
    assert lib.ts_paged_append(4096, three, 4096, three, 1, None, cache(), None, None, None, 0, 4096, three, None) == INVALID
    assert lib.ts_paged_append(4096, three, 4096, three, 0, None, cache(), None, None, None, 0, None, None, None) == 0
    full = cache(scores=4096, slot_pos=4096)
    assert lib.ts_paged_evict(cache(), 4, 0, None, 0, None) == INVALID
    for budget, recent in ((0, 0), (4, 5), (4, -1)):
        assert lib.ts_paged_evict(full, budget, recent, None, 0, None) == INVALID
    assert lib.ts_paged_evict(full, 4, 0, None, 0, None) == WORKSPACE
    assert lib.ts_paged_evict(full, 32, 0, None, 0, None) == 0           # no sequence can be longer


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    with pytest.raises(RuntimeError):
        ts.fp4_quantize(x)
    with pytest.raises(RuntimeError):
        ts.Fp4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), None, 4, 64, "nvfp4")
    with pytest.raises(NotImplementedError):
        ts.fp4_quantize(x, "e2m1")
    with pytest.raises(RuntimeError):
        ts.PagedKVCache.allocate(2, 2, 64, 32, device="cpu")
