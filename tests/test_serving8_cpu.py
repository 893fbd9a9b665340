"""The host side of the 8-bit serving operators, without a GPU: what the library
refuses before a launch, what tracing says of shapes and writes, and CPU tensors."""

from __future__ import annotations

import ctypes as C
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode, UnsupportedOperatorException

import tensorshrink_b200 as ts
from tensorshrink_b200 import _C

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4
P = 4096                                             # an aligned address that nothing reads


def matrix(**kw):
    t = _C.TsInt8Tensor()
    t.codes, t.row_stride, t.scales, t.rows, t.cols = P, 64, P, 8, 64
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def cache(**kw):
    c = _C.TsPagedCache8()
    c.k_pages = c.v_pages = c.k_scales = c.v_scales = c.page_table = c.seq_lens = P
    c.page_stride, c.head_stride, c.token_stride = 2048, 1024, 64
    c.code, c.batch, c.n_kv, c.head_dim, c.page_size, c.num_pages, c.max_pages, c.block = 0, 2, 2, 64, 32, 4, 2, 16
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw,rc", [(dict(cols=0), INVALID), (dict(rows=-1), INVALID), (dict(codes=None), INVALID),
                                   (dict(scales=None), INVALID), (dict(codes=4100), INVALID), (dict(row_stride=72), INVALID),
                                   (dict(row_stride=48), INVALID), (dict(cols=131073, row_stride=131088), UNSUPPORTED)])
def test_int8_tensors_are_checked(kw, rc):
    lib = _C.load()
    t = matrix(**kw)
    assert lib.ts_int8_quantize(P, _C.TS_BF16, 64, t, None) == rc
    assert lib.ts_int8_dequantize(t, P, _C.TS_F32, 64, None) == rc
    assert lib.ts_int8_matmul(t, matrix(), None, 0, P, _C.TS_F32, 64, None, 0, None) == rc
    assert lib.ts_int8_matmul(matrix(), t, None, 0, P, _C.TS_F32, 64, None, 0, None) == rc
    assert lib.ts_last_error()


def test_int8_calls_are_checked():
    lib = _C.load()
    t = matrix()
    assert lib.ts_int8_quantize(P, 9, 64, t, None) == UNSUPPORTED
    assert lib.ts_int8_quantize(None, _C.TS_BF16, 64, t, None) == INVALID
    assert lib.ts_int8_quantize(4097, _C.TS_BF16, 64, t, None) == INVALID
    assert lib.ts_int8_dequantize(t, None, _C.TS_F32, 64, None) == INVALID
    assert lib.ts_int8_matmul(t, matrix(cols=48), None, 0, P, _C.TS_F32, 64, None, 0, None) == INVALID
    assert lib.ts_int8_matmul(t, t, None, 0, P, 7, 64, None, 0, None) == UNSUPPORTED
    assert lib.ts_int8_matmul(t, t, P, 9, P, _C.TS_F32, 64, None, 0, None) == UNSUPPORTED
    assert lib.ts_int8_matmul(t, t, None, 0, None, _C.TS_F32, 64, None, 0, None) == INVALID
    assert lib.ts_int8_matmul(t, t, None, 0, P, _C.TS_F32, 64, None, 0, None) == WORKSPACE
    assert lib.ts_int8_linear(P, _C.TS_BF16, 4, 64, t, None, 0, P, _C.TS_F32, 64, None, 0, None) == WORKSPACE
    assert lib.ts_int8_linear(P, _C.TS_BF16, -1, 64, t, None, 0, P, _C.TS_F32, 64, None, 0, None) == INVALID
    # nothing to do is no error
    none = matrix(rows=0, codes=None, scales=None)
    assert lib.ts_int8_quantize(None, _C.TS_BF16, 64, none, None) == 0
    assert lib.ts_int8_matmul(none, t, None, 0, None, _C.TS_F32, 64, None, 0, None) == 0
    assert lib.ts_int8_linear(None, _C.TS_BF16, 0, 64, t, None, 0, None, _C.TS_F32, 64, None, 0, None) == 0


@pytest.mark.parametrize("kw,rc", [(dict(k_pages=None), INVALID), (dict(v_scales=None), INVALID), (dict(code=2), UNSUPPORTED),
                                   (dict(head_dim=40), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED),
                                   (dict(block=8), UNSUPPORTED), (dict(block=48), UNSUPPORTED), (dict(block=0), INVALID),
                                   (dict(page_size=0), INVALID), (dict(token_stride=72), INVALID), (dict(v_pages=4104), INVALID),
                                   (dict(max_pages=1 << 30), INVALID), (dict(num_pages=0), INVALID), (dict(batch=-1), INVALID)])
def test_caches_are_checked(kw, rc):
    lib = _C.load()
    c = cache(**kw)
    three = (C.c_int64 * 3)(128, 128, 64)
    assert lib.ts_paged8_append(P, three, P, three, _C.TS_BF16, 1, None, None, c, None, None, None, 0, None) == rc
    assert lib.ts_paged8_attention(P, _C.TS_BF16, 128, 2, c, None, None, None, 0, 0.1, P, 128, None, 0, None) == rc
    assert lib.ts_paged8_decode_attention(P, _C.TS_BF16, 384, 2, c, P, None, None, 0, 0.1, P, 128, None, 0, None) == rc
    assert lib.ts_paged8_dequantize(c, P, P, _C.TS_F32, None) == rc


def test_paged8_calls_are_checked():
    lib = _C.load()

    def attend(c=None, q=P, dtype=_C.TS_BF16, n_q=2, pos=None, cos=None, sin=None, scale=0.1, out=P, stride=128, ws=None):
        return lib.ts_paged8_attention(q, dtype, 128, n_q, c or cache(), pos, cos, sin, 0, scale, out, stride, ws, 0, None)
    assert attend(dtype=_C.TS_F32) == UNSUPPORTED
    assert attend(n_q=0) == INVALID and attend(n_q=3) == INVALID
    assert attend(cos=P) == INVALID and attend(cos=P, sin=P) == INVALID
    assert attend(scale=0.0) == INVALID and attend(scale=float("nan")) == INVALID and attend(scale=float("inf")) == INVALID
    assert attend(out=None) == INVALID and attend(stride=127) == INVALID
    assert attend() == WORKSPACE
    assert attend(cache(batch=0)) == 0
    three, odd = (C.c_int64 * 3)(128, 128, 64), (C.c_int64 * 3)(128, 124, 64)

    def put(k=P, ks=three, dtype=_C.TS_BF16, tokens=1, cos=None, sin=None, c=None):
        return lib.ts_paged8_append(k, ks, P, three, dtype, tokens, None, None, c or cache(), None, cos, sin, 0, None)
    assert put(dtype=_C.TS_F32) == UNSUPPORTED and put(k=None) == INVALID and put(k=4104) == INVALID
    assert put(ks=odd) == INVALID and put(tokens=-1) == INVALID and put(cos=P) == INVALID
    assert put(tokens=0) == 0 and put(c=cache(batch=0)) == 0
    assert lib.ts_paged8_dequantize(cache(), P, None, _C.TS_F32, None) == INVALID
    assert lib.ts_paged8_dequantize(cache(), P, P, 9, None) == UNSUPPORTED


def test_norm_calls_are_checked():
    lib = _C.load()

    def norm(x=P, dtype=_C.TS_BF16, stride=256, tokens=1, n_q=2, n_kv=1, d=64, qw=P, kw=P, wdt=_C.TS_F32, eps=1e-6, pos=None,
             cos=None, sin=None, out=P, ostride=256, c=None, slots=None):
        return lib.ts_qk_norm_rope(x, dtype, stride, tokens, n_q, n_kv, d, qw, kw, wdt, eps, pos, cos, sin, 0, out, ostride, c,
                                   slots, None)
    assert norm(dtype=_C.TS_F32) == UNSUPPORTED and norm(d=40) == UNSUPPORTED and norm(d=272) == UNSUPPORTED
    assert norm(wdt=_C.TS_F16) == UNSUPPORTED
    assert norm(n_q=-1) == INVALID and norm(n_q=0, n_kv=0) == INVALID and norm(tokens=-1) == INVALID
    assert norm(eps=-1.0) == INVALID and norm(eps=float("nan")) == INVALID
    assert norm(cos=P) == INVALID and norm(cos=P, sin=P) == INVALID
    assert norm(x=None) == INVALID and norm(x=4104) == INVALID and norm(stride=252) == INVALID and norm(out=4104) == INVALID
    assert norm(qw=4100) == INVALID and norm(slots=P) == INVALID
    c = _C.TsPagedCache()
    c.k_pages = c.v_pages = c.page_table = c.seq_lens = P
    c.page_stride, c.head_stride, c.token_stride = 1024, 1024, 64
    c.dtype, c.batch, c.n_kv, c.head_dim, c.page_size, c.num_pages, c.max_pages = _C.TS_BF16, 2, 2, 64, 16, 4, 2
    assert norm(c=c) == INVALID and norm(c=c, slots=P) == INVALID          # two kv heads
    assert norm(tokens=0, x=None, out=None) == 0


def test_table_calls_are_checked():
    lib = _C.load()

    def views(**kw):
        p, t = _C.TsPagePool(), _C.TsPageTable()
        p.free_pages, p.n_free, p.capacity = P, P, 8
        t.table, t.table_stride, t.seq_lens, t.batch, t.max_pages, t.page_size, t.num_pages = P, 4, P, 2, 4, 16, 8
        for k, v in kw.items():
            setattr(p if hasattr(p, k) else t, k, v)
        return p, t

    def reserve(n_new=P, tokens=4, slots=P, **kw):
        p, t = views(**kw)
        return lib.ts_paged_reserve(p, t, n_new, None, tokens, P, P, slots, P, P, None)
    assert reserve(n_new=None) == INVALID and reserve(tokens=-1) == INVALID and reserve(slots=None) == INVALID
    assert reserve(page_size=0) == INVALID and reserve(max_pages=1 << 28) == INVALID and reserve(seq_lens=None) == INVALID
    assert reserve(batch=0) == INVALID and reserve(batch=8193) == UNSUPPORTED and reserve(free_pages=None) == INVALID
    p, t = views(batch=0)
    assert lib.ts_paged_release(p, t, None, None) == 0
    p, t = views()
    assert lib.ts_paged_release(p, t, None, None) == INVALID


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    for f in (lambda: ts.int8_quantize(x), lambda: ts.qk_norm_rope(x.half(), 2, 1),
              lambda: ts.Int8Tensor(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)),
              lambda: ts.PagedKVCache8.allocate(2, 2, 64, 32, device="cpu"), lambda: ts.PagePool.allocate(4, "cpu")):
        with pytest.raises(RuntimeError):
            f()


@pytest.fixture
def fake():
    """Fake CUDA tensors; a kernel that touches their memory warns, which is an error here."""
    with warnings.catch_warnings(), FakeTensorMode() as mode:
        warnings.simplefilter("error")
        yield mode


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_shapes_of_products_and_norms(fake):
    t = ts.int8_quantize(empty(5, 200))
    assert t.codes.shape == (5, 208) and t.codes.dtype == torch.int8 and t.scales.shape == (5,)
    assert ts.int8_dequantize(t, torch.float16).shape == (5, 200)
    w = ts.int8_quantize(empty(30, 200))
    assert ts.int8_matmul(t, w, out_dtype=torch.float32).shape == (5, 30)
    y = ts.int8_linear(empty(2, 3, 200), w)
    assert y.shape == (2, 3, 30) and y.dtype == torch.bfloat16
    with pytest.raises(ValueError):
        ts.int8_linear(empty(2, 3, 199), w)
    x = empty(7, 6 * 64)
    assert ts.qk_norm_rope(x, 2, 2, empty(64), empty(64)).shape == x.shape
    assert ts.qk_norm_rope(x, 2, 2, out=x) is x
    with pytest.raises(UnsupportedOperatorException):            # what tracing makes of a NotImplementedError
        ts.qk_norm_rope(empty(7, 6 * 64, dtype=torch.float32), 2, 2)


@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
def test_shapes_of_the_cache(fake, held):
    i = lambda *s: empty(*s, dtype=torch.int32)  # noqa: E731
    c = ts.PagedKVCache8(empty(9, 2, 32, 64, dtype=held), empty(9, 2, 32, 64, dtype=held), empty(9, 2, 2, dtype=torch.float32),
                         empty(9, 2, 2, dtype=torch.float32), i(3, 4), i(3))
    assert c.block == 16 and c.capacity == 128 and c.batch == 3
    assert ts.paged_attention(empty(3, 8 * 64), c).shape == (3, 512)
    assert ts.paged_decode_attention(empty(3, 12 * 64), 8, c).shape == (3, 512)
    ts.paged_append(empty(3, 5, 2, 64), empty(3, 5, 2, 64), c)
    ts.paged_append(empty(5, 2, 64), empty(5, 2, 64), c, offsets=i(4))
    k, v = ts.paged_dequantize(c, torch.float16)
    assert k.shape == v.shape == (9, 2, 32, 64) and k.dtype == torch.float16
    with pytest.raises(UnsupportedOperatorException):
        ts.paged_attention(empty(3, 512, dtype=torch.float32), c)
    pool = ts.PagePool(i(9), i(1))
    got = ts.paged_reserve(pool, c, i(3), 40)
    assert [t.shape[0] for t in got] == [3, 4, 40, 40, 40] and got.slots.dtype == torch.int64
    ts.paged_release(pool, c, i(3))


def test_schemas_say_what_is_written():
    ops = _C.serving_ops()

    def written(name, overload="default"):
        s = getattr(getattr(ops, name), overload)._schema
        return {a.name for a in s.arguments if a.alias_info is not None and a.alias_info.is_write}
    pages = {"k_pages", "v_pages", "k_scales", "v_scales"}
    assert written("paged8_append") == written("paged8_decode_attention") == pages
    assert written("paged8_attention") == written("paged8_dequantize") == set()
    assert written("paged_reserve") == {"n_free", "page_table"}
    assert written("paged_release") == {"free", "n_free", "page_table", "seq_lens"}
    assert written("qk_norm_rope_store") == {"k_pages", "v_pages", "scores", "slot_pos"}
    assert written("qk_norm_rope") == written("int8_linear") == set()
    assert written("qk_norm_rope", "out") == {"out"}
