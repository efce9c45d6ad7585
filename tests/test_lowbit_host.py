"""The refusals of the 8-bit linears and the 4-bit cache that need no device: the C entry points without a context, the
parameter structures against the header, and the Python front ends' checks (before anything is issued)."""
import ctypes
import re

import pytest
import torch

from llmr_amd import capi, int8, serve

F16, I8, U8 = torch.float16, torch.int8, torch.uint8


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_entry_points_refuse_a_null_context():
    L = capi.lib()
    c = capi.Mx4Cache(16, 16)
    for name, args in (("llmr_qkv_tokens_mx4", [None] * 9 + [c, c, None]),
                       ("llmr_paged_attention_mx4", [None, 16, c, c, 1, 16, 16, 16, 16, 16, 0, None]),
                       ("llmr_mx4_rows", [None, c, c, 16, 16, 16, None]),
                       ("llmr_quantize_rows_i8", [None, 16, 16, 16, 16, None]),
                       ("llmr_matmul_i8", [None, 16, 16, 16, 16, 16, None])):
        assert getattr(L, name)(*args) == capi.LLMR_ERR_INVALID_ARG
        assert "context" in capi.last_error()
    assert L.llmr_paged_attention_mx4_scratch_bytes(None, None) == 0


def test_params_have_the_headers_fields():
    text = open(capi.HEADER_PATH).read()
    types = {"uint32_t": ctypes.c_uint32, "float": ctypes.c_float, "void*": ctypes.c_void_p}
    for cls, name in ((capi.Mx4Cache, "mx4_cache"), (capi.Mx4RowsParams, "mx4_rows_params"),
                      (capi.QuantizeRowsParams, "quantize_rows_params"), (capi.MatmulI8Params, "matmul_i8_params")):
        body = re.search(r"typedef struct llmr_%s \{(.*?)\} llmr_%s;" % (name, name), text, re.S).group(1)
        fields = re.findall(r"(uint32_t|float|void\*)\s+(\w+);", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
        assert [(n, types[t]) for t, n in fields] == cls._fields_


def test_an_empty_cache_has_its_shapes():
    c = serve.Mx4Cache.empty(3, 2, 16, 128, "cpu")
    assert c.data.shape == (3, 2, 16, 64) and c.scales.shape == (3, 2, 16, 4)
    assert c.data.dtype is U8 and int(c.data.sum()) + int(c.scales.sum()) == 0


def test_shapes_and_types_of_caches_are_checked():
    c, q, i = serve.Mx4Cache.empty(3, 1, 16, 64, "cpu"), torch.zeros(4, 2, 64, dtype=F16), _i32
    C = serve.Mx4Cache
    bad = [C(c.data, c.scales[:, :, :, :1]), C(c.data.char(), c.scales), C(c.data[0], c.scales[0]),
           C(c.data[:2], c.scales[:2]), C(c.data.transpose(1, 2), c.scales), C(c.data, c.scales.float()),
           C(torch.zeros(3, 1, 16, 40, dtype=U8), c.scales)]
    for b in bad:
        for k, v in ((c, b), (b, c)):
            with pytest.raises(ValueError, match="cache"):
                serve.paged_attention_mx4(q, k, v, i(3), i(2), i(2, 2), 1)
            with pytest.raises(ValueError, match="cache"):
                serve.qkv_tokens_mx4(torch.zeros(4, 4 * 64), q, k, v, i(4))
            with pytest.raises(ValueError, match="cache"):
                serve.mx4_rows(k, v, i(4), q[:, :1], q[:, 1:])
    with pytest.raises(ValueError, match="one per request"):
        serve.paged_attention_mx4(q, c, c, i(4), i(2), i(2, 2), 1)
    with pytest.raises(ValueError, match="max_new"):
        serve.paged_attention_mx4(q, c, c, i(3), i(2), i(2, 2), -1)
    with pytest.raises(ValueError, match="max_new"):
        serve.paged_attention_mx4_scratch(q, c, i(2, 2), -1)
    with pytest.raises(ValueError, match="float16"):
        serve.paged_attention_mx4(q.float(), c, c, i(3), i(2), i(2, 2), 1)
    with pytest.raises(ValueError, match="float16"):
        serve.qkv_tokens_mx4(torch.zeros(4, 4 * 64), q.float(), c, c, i(4))
    with pytest.raises(ValueError, match="head_dim"):
        serve.qkv_tokens_mx4(torch.zeros(4, 4 * 64), q[:, :, :32].contiguous(), c, c, i(4))
    with pytest.raises(ValueError, match="slots"):
        serve.qkv_tokens_mx4(torch.zeros(4, 4 * 64), q, c, c, i(3))
    for tabs in (tuple(torch.zeros(0, 32) for _ in range(2)), (torch.zeros(9, 16),) * 2):
        with pytest.raises(ValueError, match="rope"):
            serve.qkv_tokens_mx4(torch.zeros(4, 4 * 64), q, c, c, i(4), rope=tabs)
    with pytest.raises(ValueError, match="alike"):
        serve.mx4_rows(c, c, i(4), q[:, :1], q)
    with pytest.raises(ValueError, match="heads side by side"):
        serve.mx4_rows(c, c, i(4), q, q.clone())


def test_shapes_and_types_of_linears_are_checked():
    x, w, s = torch.zeros(4, 64, dtype=I8), torch.zeros(6, 64, dtype=I8), torch.ones(6)
    for args, kw, what in (((x.float(), s[:4], w, s), {}, "int8"), ((x, s[:4], w[:, :32], s), {}, "in_dim"),
                           ((x, s[:3], w, s), {}, "x_scales"), ((x, s[:4], w, s[:5]), {}, "w_scales"),
                           ((x, s[:4].double(), w, s), {}, "x_scales"), ((x[0], s[:4], w, s), {}, "2-D"),
                           ((x, s[:4], w, s), dict(out=torch.zeros(4, 5)), "out"),
                           ((x, s[:4], w, s), dict(out=torch.zeros(6, 4).t()), "contiguous rows"),
                           ((x, s[:4], w, s), dict(dtype=torch.float64), "out")):
        with pytest.raises(ValueError, match=what):
            int8.matmul(*args, **kw)
    f = torch.zeros(4, 64)
    for args, kw, what in (((f.double(),), {}, "float32"), ((f,), dict(norm=s), "norm"), ((f[0],), {}, "2-D"),
                           ((f,), dict(q=x[:, :32]), "q"), ((f,), dict(q=f), "int8"), ((f,), dict(scales=s), "scales")):
        with pytest.raises(ValueError, match=what):
            int8.quantize_rows(*args, **kw)


def test_strides_past_32_bits_are_refused():
    far = torch.empty_strided((4, 64), (1 << 32, 1), dtype=I8, device="meta")
    x, s = torch.zeros(4, 64, dtype=I8), torch.ones(4)
    with pytest.raises(ValueError, match="2\\^32"):
        int8.matmul(far, s, x, s)
    with pytest.raises(ValueError, match="2\\^32"):
        int8.matmul(x, s, far, s)
    with pytest.raises(ValueError, match="2\\^32"):
        int8.quantize_rows(torch.empty_strided((4, 64), (1 << 32, 1), device="meta"))


class _Recorder:
    """A graph on no device whose context keeps what a call would be issued with."""
    device = -1  # a host tensor's get_device()

    def __init__(self):
        self.ctx, self.calls = self, []

    def set_stream(self, stream):
        pass

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args))


def test_one_rows_stride_does_not_matter(monkeypatch):
    """One row: its stride is nothing, whatever it is; the call has one that the library takes."""
    monkeypatch.setattr(serve, "_raw_stream", lambda dev: 0)
    g = _Recorder()
    x = torch.zeros(64, dtype=I8).as_strided((1, 64), (1 << 33, 1))
    w, s = torch.zeros(6, 64, dtype=I8), torch.ones(6)
    int8.matmul(x, s[:1], w, s, out=torch.zeros(6).as_strided((1, 6), (3, 1)), g=g)
    int8.quantize_rows(torch.zeros(64).as_strided((1, 64), (1 << 33, 1)), g=g)
    (name, a), (name2, b) = g.calls
    assert (name, a[-1].x_stride, a[-1].w_stride, a[-1].out_stride) == ("matmul_i8", 64, 64, 16)
    assert (name2, b[-1].x_stride, b[-1].q_stride) == ("quantize_rows_i8", 64, 64)
