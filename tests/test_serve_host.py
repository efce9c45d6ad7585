"""The batch operators' refusals that need no device: the C entry points without a context, and the Python front
end's checks of shapes and types (before anything is issued)."""
import ctypes

import pytest
import torch

from llmr_amd import capi, serve

F16 = torch.float16


def test_entry_points_refuse_a_null_context():
    L = capi.lib()
    for name, n in (("llmr_prompt_attention", 7), ("llmr_paged_plan", 11), ("llmr_qkv_tokens", 11),
                    ("llmr_paged_attention", 10)):
        args = [None] * n
        if name == "llmr_prompt_attention":
            args = [None, 16, 16, 16, 1, 16, 16]
        elif name == "llmr_paged_attention":
            args = [None, 16, 16, 16, 1, 16, 16, 16, 16, 16, 0]
        assert getattr(L, name)(*args, None) == capi.LLMR_ERR_INVALID_ARG
        assert "context" in capi.last_error()
    assert L.llmr_paged_attention_scratch_bytes(None, None) == 0


def test_params_have_the_headers_fields():
    """Every params structure has the header's fields in the header's order."""
    import re
    text = open(capi.HEADER_PATH).read()
    for cls, name in ((capi.PromptAttentionParams, "prompt_attention"), (capi.PagedPlanParams, "paged_plan"),
                      (capi.QkvTokensParams, "qkv_tokens"), (capi.PagedAttentionParams, "paged_attention")):
        body = re.search(r"typedef struct llmr_%s_params \{(.*?)\} llmr_%s_params;" % (name, name), text, re.S).group(1)
        fields = re.findall(r"(uint32_t|float)\s+(\w+);", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
        types = {"uint32_t": ctypes.c_uint32, "float": ctypes.c_float}
        assert [(n, types[t]) for t, n in fields] == cls._fields_
    assert "LLMR_MAX_SEQS %du" % capi.MAX_SEQS in text


def test_tensors_have_to_be_on_the_device():
    q, k = torch.zeros(4, 2, 64, dtype=F16), torch.zeros(4, 1, 64, dtype=F16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(k=k[:3]), dict(seq_offsets=off.long()),
                dict(out=torch.zeros(4, 64, dtype=F16))):
        with pytest.raises(ValueError):
            serve.prompt_attention(**{**dict(q=q, k=k, v=k.clone(), seq_offsets=off), **bad})


def test_shapes_are_checked():
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    b = serve.PagedBatch.empty(2, 5, "cpu")
    with pytest.raises(ValueError, match="one per request"):
        serve.paged_plan(i32(2), i32(3), i32(4), i32(1), i32(4).view(2, 2), 16, b)
    with pytest.raises(ValueError, match="PagedBatch"):
        serve.paged_plan(i32(3), i32(3), i32(4), i32(1), i32(6).view(3, 2), 16, b)
    with pytest.raises(ValueError, match="int32"):
        serve.paged_plan(i32(2), i32(2).long(), i32(4), i32(1), i32(4).view(2, 2), 16, b)
    cache = torch.zeros(3, 1, 16, 64, dtype=F16)
    q = torch.zeros(4, 2, 64, dtype=F16)
    with pytest.raises(ValueError, match="one per request"):
        serve.paged_attention(q, cache, cache.clone(), i32(4), i32(2), i32(4).view(2, 2), 1)
    with pytest.raises(ValueError, match="dtype"):
        serve.paged_attention(q, cache, cache.float(), i32(3), i32(2), i32(4).view(2, 2), 1)
    with pytest.raises(ValueError, match="qkv"):
        serve.qkv_tokens(torch.zeros(4, 3 * 64), q, q[:, :1], q[:, :1])


def test_max_new_is_not_negative():
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    cache, q = torch.zeros(3, 1, 16, 64, dtype=F16), torch.zeros(4, 2, 64, dtype=F16)
    with pytest.raises(ValueError, match="max_new"):
        serve.paged_attention(q, cache, cache.clone(), i32(3), i32(2), i32(4).view(2, 2), -1)
    with pytest.raises(ValueError, match="max_new"):
        serve.paged_attention_scratch(q, cache, i32(4).view(2, 2), -1)


def test_strides_past_32_bits_are_refused():
    """(They would be cut to the parameters' 32 bits.)"""
    far = lambda n, h: torch.empty_strided((n, h, 64), (64, 1 << 32, 1), dtype=F16, device="meta")  # noqa: E731
    off = torch.tensor([0, 4], dtype=torch.int32)
    q = torch.zeros(4, 2, 64, dtype=F16)
    with pytest.raises(ValueError, match="2\\^32"):
        serve.prompt_attention(q, far(4, 2), far(4, 2), off)
    with pytest.raises(ValueError, match="2\\^32"):
        serve.prompt_attention(far(4, 2), q, q.clone(), off)
    with pytest.raises(ValueError, match="2\\^32"):
        serve.qkv_tokens(torch.empty_strided((4, 256), (1 << 32, 1), device="meta"), q, q[:, :1], q[:, :1])


def test_empty_rotation_tables_are_refused():
    """(An empty tensor's address is null, which stands for no rotation.)"""
    q = torch.zeros(4, 2, 64, dtype=F16)
    tabs = tuple(torch.zeros(0, 32) for _ in range(2))
    for positions in (None, torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError, match="rope"):
            serve.qkv_tokens(torch.zeros(4, 4 * 64), q, q[:, :1], q[:, 1:], positions=positions, rope=tabs)


class _Recorder:
    """A graph on no device whose context keeps what a call would be issued with."""
    device = -1  # a host tensor's get_device()

    def __init__(self):
        self.ctx, self.calls = self, []

    def set_stream(self, stream):
        pass

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args))


def test_strides_of_dimensions_of_one_do_not_matter(monkeypatch):
    """One token, or one key/value head: its stride in that dimension is nothing, also where k's and v's differ."""
    monkeypatch.setattr(serve, "_raw_stream", lambda dev: 0)
    off = torch.tensor([0, 1], dtype=torch.int32)
    wide = torch.zeros(5, 8, 64, dtype=F16)
    for T, Hk in ((1, 2), (1, 1), (5, 1)):
        q = torch.zeros(T, 2, 64, dtype=F16)
        k = torch.zeros(T, Hk, 64, dtype=F16)
        v = torch.zeros(5, Hk, 64, dtype=F16)[:T].as_strided((T, Hk, 64), (64 * Hk if T > 1 else 512, 64 if Hk > 1 else 640, 1))
        if Hk == 1:  # past the parameters' 32 bits, were it one that counts
            k = k.as_strided(k.shape, (64, 1 << 33, 1))
        g = _Recorder()
        serve.prompt_attention(q, k, v, off, g=g)
        serve.qkv_tokens(torch.zeros(T, (2 + 2 * Hk) * 64), q, k, v, g=g)
        (name, a), (name2, b) = g.calls
        p, r = a[-1], b[-1]
        assert (name, p.kv_stride, p.kv_head_stride) == ("prompt_attention", Hk * 64, 64)
        assert (name2, r.kv_stride) == ("qkv_tokens", Hk * 64)
    for k, v in ((wide[:, :2], torch.zeros(5, 2, 64, dtype=F16)), (wide[:, :1], torch.zeros(5, 1, 64, dtype=F16))):
        q = torch.zeros(5, 2, 64, dtype=F16)
        with pytest.raises(ValueError, match="alike"):  # strides that count do have to be the same
            serve.prompt_attention(q, k, v, off, g=_Recorder())
        with pytest.raises(ValueError, match="alike"):
            serve.qkv_tokens(torch.zeros(5, 8 * 64), q, k, v, g=_Recorder())
