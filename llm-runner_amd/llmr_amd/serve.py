"""Batches of requests of the text path: causal attention of packed prompts and
the paged key/value cache, on torch device tensors.

The requests' tokens lie one after the other in packed rows; request s has the
rows seq_offsets[s] .. seq_offsets[s + 1]. A step of a batch:

    batch = serve.paged_plan(past_len, new_len, free_pages, free_count, block_table, page_size, batch)
    ops.dispatch_batch_matmul(...)                      # the QKV projection of the packed rows
    serve.qkv_tokens(qkv, q, k_cache, v_cache, slots=batch.slots, positions=batch.positions, rope=tables)
    serve.paged_attention(q, k_cache, v_cache, batch.seq_offsets, batch.kv_len, block_table, max_new)

A prompt that needs no cache (the text encoder's) goes through qkv_tokens
without slots and prompt_attention. Each function issues one C-ABI call on the
current torch stream of the graph's device; lengths, offsets, tables and slots
are int32 device tensors that nothing here reads back.
"""
from __future__ import annotations

import dataclasses

import torch

from . import capi
from .gguf import GGML_BF16, GGML_F16
from .ops import RenderGraph, default_graph

_TYPES = {torch.float16: GGML_F16, torch.bfloat16: GGML_BF16}
_I32, _F32 = torch.int32, torch.float32
_U32 = 0xffffffff  # the parameters' integers
# the stream's handle alone, without the Stream object that torch.cuda.current_stream makes
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


# The checks below are written out flat: a call's host time is what single-token steps wait for.


def _graph(g: RenderGraph | None, *tensors) -> RenderGraph:
    """The graph, on its device's current stream; every tensor has to be on that device."""
    if g is None:
        g = default_graph()
    dev = g.ctx.device
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError(f"all tensors must be on the graph's device (cuda:{dev})")
    g.ctx.set_stream(_raw_stream(dev))
    return g


def _ints(t: torch.Tensor, what: str, n: int) -> int:
    if t.dtype is not _I32 or t.numel() < n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 device tensor of >= {n} elements")
    return t.data_ptr()


def _vec(t, what: str, n: int):
    if t is None:
        return None
    if t.dtype is not _F32 or t.numel() < n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous f32 device tensor of >= {n} elements")
    return t.data_ptr()


def _heads(t: torch.Tensor, what: str):
    """(tokens, heads, dim) and the strides of tokens and heads of a 3-D view with contiguous heads; a
    dimension of one has no stride of its own and gets one that the library takes."""
    if t.dim() != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim] with contiguous heads")
    T, H, D = t.shape
    ts, hs, ds = t.stride()
    if ds != 1:
        raise ValueError(f"{what} must be [tokens, heads, head_dim] with contiguous heads")
    ts, hs = ts if T > 1 else H * D, hs if H > 1 else D
    if ts > _U32 or hs > _U32:
        raise ValueError(f"{what}'s strides must be under 2^32 elements")
    return T, H, D, ts, hs


def _alike(k: torch.Tensor, v: torch.Tensor) -> bool:
    """Whether v has k's shape and strides, but for those of a dimension of one."""
    return v.shape == k.shape and (v.stride() == k.stride() or _heads(v, "v")[3:] == _heads(k, "k")[3:])


def _out_stride(out: torch.Tensor, T: int, width: int, like: torch.Tensor) -> int:
    if out.dtype is not like.dtype or out.shape != (T, width) or out.stride(1) != 1 or out.stride(0) > _U32:
        raise ValueError(f"out must be a [{T}, {width}] view of q's dtype with contiguous rows, under 2^32 apart")
    return out.stride(0) if T > 1 else width


def _cache(k: torch.Tensor, v: torch.Tensor):
    if k.dim() != 4 or k.shape != v.shape or not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("k and v caches must be contiguous [n_pages, n_kv_heads, page_size, head_dim] alike")
    return k.shape


def _type(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> int:
    d = q.dtype
    t = _TYPES.get(d)
    if t is None or k.dtype is not d or v.dtype is not d:
        raise ValueError(f"{what} must share one dtype, float16 or bfloat16")
    return t


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seq_offsets: torch.Tensor,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     g: RenderGraph | None = None) -> torch.Tensor:
    """Causal attention of packed prompts (llmr_prompt_attention). q [T, n_heads, D], k and v [T, n_kv_heads,
    D] f16 or bf16, any strides of tokens and heads (column slices of one QKV buffer, head-major buffers
    transposed); seq_offsets int32 [n_seqs + 1]; scale 1/sqrt(D) by default. out [T, n_heads * D], q's dtype;
    its rows that belong to no request keep what they hold (a new `out`: undefined). out may be q's own rows
    and overlaps nothing else."""
    T, H, D, qs, qh = _heads(q, "q")
    Tk, Hk, Dk, ks, kh = _heads(k, "k")
    if Tk != T or Dk != D or not _alike(k, v):
        raise ValueError("k and v must be [tokens, n_kv_heads, head_dim] alike, with q's tokens and head_dim")
    t = _type("q, k and v", q, k, v)
    if out is None:
        out = torch.empty(T, H * D, dtype=q.dtype, device=q.device)
    os_ = _out_stride(out, T, H * D, q)
    n = seq_offsets.numel() - 1
    if n < 0:
        raise ValueError("seq_offsets must have n_seqs + 1 elements")
    off = _ints(seq_offsets, "seq_offsets", 1)
    _graph(g, q, k, v, seq_offsets, out).ctx.prompt_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), t, out.data_ptr(), off,
        capi.PromptAttentionParams(D, H, Hk, T, n, qs, qh, ks, kh, os_, D ** -0.5 if scale is None else scale))
    return out


@dataclasses.dataclass
class PagedBatch:
    """What paged_plan writes: seq_offsets [n_seqs + 1], kv_len [n_seqs], slots and positions [n_tokens]
    (-1 and 0 for the rows behind the last request), pages [2] (left in the free list, lacking); int32."""
    seq_offsets: torch.Tensor
    kv_len: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    pages: torch.Tensor

    @staticmethod
    def empty(n_seqs: int, n_tokens: int, device="cuda") -> "PagedBatch":
        return PagedBatch(*(torch.empty(n, dtype=torch.int32, device=device)
                            for n in (n_seqs + 1, n_seqs, n_tokens, n_tokens, 2)))


def paged_plan(past_len: torch.Tensor, new_len: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
               block_table: torch.Tensor, page_size: int, batch: PagedBatch, g: RenderGraph | None = None) -> PagedBatch:
    """Pages and slots of one step from the requests' lengths (llmr_paged_plan): past_len, new_len int32
    [n_seqs]; free_pages [capacity] with free_count [1] of them free, taken from the end; block_table
    [n_seqs, max_pages], whose new entries are filled in; batch receives the rest. The new tokens' sum is
    at most batch.slots' length."""
    n, T = past_len.numel(), batch.slots.numel()
    if block_table.dim() != 2 or block_table.shape[0] != n or new_len.numel() != n:
        raise ValueError("past_len, new_len and block_table's rows must be one per request")
    if batch.seq_offsets.numel() != n + 1 or batch.positions.numel() != T:
        raise ValueError("batch must be PagedBatch.empty(n_seqs, n_tokens)")
    off, kvl, slots, pos, pages = batch.seq_offsets, batch.kv_len, batch.slots, batch.positions, batch.pages
    args = (_ints(past_len, "past_len", n), _ints(new_len, "new_len", n), _ints(free_pages, "free_pages", 0),
            _ints(free_count, "free_count", 1), _ints(block_table, "block_table", 0), _ints(off, "seq_offsets", 0),
            _ints(kvl, "kv_len", n), _ints(slots, "slots", 0), _ints(pos, "positions", 0), _ints(pages, "pages", 2))
    _graph(g, past_len, new_len, free_pages, free_count, block_table, off, kvl, slots, pos, pages).ctx.paged_plan(
        *args, capi.PagedPlanParams(n, T, page_size, block_table.shape[1], free_pages.numel()))
    return batch


def qkv_tokens(qkv: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               slots: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
               rope: tuple | None = None, halves: bool = True, g: RenderGraph | None = None) -> None:
    """Rows of a QKV projection (f32 [T, >= (n_heads + 2 n_kv_heads) D], Q | K | V from column 0) -> head
    norm, rotation and rows of q [T, n_heads, D] and of k and v (llmr_qkv_tokens): with slots (int32 [T]) the
    caches [n_pages, n_kv_heads, page_size, D], a row with slot -1 nowhere; without, rows [T, n_kv_heads, D].
    rope: (cos, sin) f32 [n_positions, D / 2], taken at positions (int32 [T]; None: the row), rotating the
    pairs (j, j + D/2), or (2j, 2j + 1) where halves is False."""
    if qkv.dim() != 2 or qkv.dtype is not _F32 or (qkv.shape[1] > 1 and qkv.stride(1) != 1) or qkv.stride(0) > _U32:
        raise ValueError("qkv must be a 2-D f32 view with contiguous rows, under 2^32 apart")
    T, H, D, qs, qh = _heads(q, "q")
    if qkv.shape[0] != T or qh != D:
        raise ValueError("q must be [tokens, n_heads, head_dim] with qkv's tokens and heads side by side")
    t = _type("q, k and v", q, k, v)
    ks = n_pages = page = 0
    if slots is not None:
        n_pages, Hk, page, Dk = _cache(k, v)
        sp = _ints(slots, "slots", T)
    else:
        Tk, Hk, Dk, ks, kh = _heads(k, "k")
        sp = None
        if not _alike(k, v) or Tk != T or kh != D:
            raise ValueError("k and v must be [tokens, n_kv_heads, head_dim] alike, heads side by side")
    if Dk != D or qkv.shape[1] < (H + 2 * Hk) * D:
        raise ValueError("k and v must have q's head_dim, and qkv (n_heads + 2 n_kv_heads) * head_dim columns")
    cos = sin = None
    n_pos = 0
    if rope is not None:
        cos, sin = rope
        if cos.dim() != 2 or cos.shape[1] != D // 2 or sin.shape != cos.shape or cos.shape[0] == 0:
            raise ValueError("rope must be (cos, sin) of [n_positions, head_dim / 2], n_positions >= 1")
        n_pos = cos.shape[0]
    pp = _ints(positions, "positions", T) if positions is not None else None
    args = (_vec(q_norm, "q_norm", D), _vec(k_norm, "k_norm", D), _vec(cos, "rope_cos", 0), _vec(sin, "rope_sin", 0))
    p = capi.QkvTokensParams(D, H, Hk, T, qkv.stride(0) if T > 1 else qkv.shape[1] + -qkv.shape[1] % 4, qs, t, ks, page,
                             n_pages, n_pos, halves, eps)
    on = [x for x in (qkv, q, k, v, slots, positions, q_norm, k_norm, cos, sin) if x is not None]
    _graph(g, *on).ctx.qkv_tokens(qkv.data_ptr(), *args, pp, sp, q.data_ptr(), k.data_ptr(), v.data_ptr(), p)


def paged_attention_scratch(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, max_new: int,
                            g: RenderGraph | None = None) -> torch.Tensor:
    """A scratch tensor for paged_attention calls of these shapes (llmr_paged_attention_scratch_bytes)."""
    T, H, D = q.shape
    n_pages, Hk, page, _ = k_cache.shape
    if max_new < 0:
        raise ValueError("max_new must be >= 0")
    p = capi.PagedAttentionParams(D, H, Hk, T, block_table.shape[0], min(max_new, T), page, n_pages,
                                  block_table.shape[1], H * D, H * D, 1.0)
    g = _graph(g, q)
    return torch.empty(g.ctx.paged_attention_scratch_bytes(p), dtype=torch.uint8, device=q.device)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seq_offsets: torch.Tensor,
                    kv_len: torch.Tensor, block_table: torch.Tensor, max_new: int, scale: float | None = None,
                    out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                    g: RenderGraph | None = None) -> torch.Tensor:
    """Attention of the requests' new tokens over the paged cache (llmr_paged_attention): q [T, n_heads, D],
    caches [n_pages, n_kv_heads, page_size, D], seq_offsets [n_seqs + 1], kv_len [n_seqs] (the new tokens
    counted), block_table [n_seqs, max_pages]; max_new: the most new tokens of a request (1 while every request
    decodes). out [T, n_heads * D] of q's dtype (rows of no request keep what they hold; a new `out`:
    undefined), which may be q's own rows and overlaps nothing else. scratch: paged_attention_scratch's, one per
    call that may overlap another; None: a new one."""
    T, H, D, qs, qh = _heads(q, "q")
    n_pages, Hk, page, Dk = _cache(k_cache, v_cache)
    n = kv_len.numel()
    if Dk != D or qh != D:
        raise ValueError("q must be [tokens, n_heads, head_dim], heads side by side, with the caches' head_dim")
    if seq_offsets.numel() != n + 1 or block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError("kv_len, block_table's rows and seq_offsets (one more) must be one per request")
    if max_new < 0:
        raise ValueError("max_new must be >= 0")
    t = _type("q and the caches", q, k_cache, v_cache)
    if out is None:
        out = torch.empty(T, H * D, dtype=q.dtype, device=q.device)
    p = capi.PagedAttentionParams(D, H, Hk, T, n, min(max_new, T), page, n_pages, block_table.shape[1], qs,
                                  _out_stride(out, T, H * D, q), D ** -0.5 if scale is None else scale)
    off, kvl, tab = _ints(seq_offsets, "seq_offsets", 0), _ints(kv_len, "kv_len", 0), _ints(block_table, "block_table", 0)
    g = _graph(g, q, k_cache, v_cache, seq_offsets, kv_len, block_table, out)
    if scratch is None:
        scratch = torch.empty(g.ctx.paged_attention_scratch_bytes(p), dtype=torch.uint8, device=q.device)
    elif scratch.get_device() != q.get_device() or not scratch.is_contiguous():
        raise ValueError("scratch must be a contiguous tensor on q's device")
    g.ctx.paged_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), t, out.data_ptr(), off, kvl, tab,
                          scratch.data_ptr(), scratch.numel() * scratch.element_size(), p)
    return out
