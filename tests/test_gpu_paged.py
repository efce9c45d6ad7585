"""GPU plan of a batch's pages and slots (llmr_paged_plan, whole numbers: equal), the projection's rows into the
cache (llmr_qkv_tokens, against its formula in 64 bits), and a run of them with the attention that reads it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _plan_oracle(past, new, free, count, table, page, n_tokens):
    """llmr_paged_plan from its definition, request by request."""
    table = [list(r) for r in table]
    cols = len(table[0]) if table else 0
    offs, kv, slots, pos, lacking = [0], [], [-1] * n_tokens, [0] * n_tokens, 0
    left = min(max(count, 0), len(free))
    for s, (p, n) in enumerate(zip(past, new)):
        p, n = max(p, 0), max(n, 0)
        for c in range(min(-(-p // page), cols), min(-(-(p + n) // page), cols)):
            if left:
                left -= 1
                table[s][c] = free[left]
            else:
                lacking += 1
                table[s][c] = -1
        for i in range(n):
            t = offs[-1] + i
            if t < n_tokens:
                c = (p + i) // page
                at = table[s][c] if c < cols else -1
                pos[t] = p + i
                slots[t] = at * page + (p + i) % page if at >= 0 and at * page + (p + i) % page < 2 ** 31 else -1
        offs.append(offs[-1] + n)
        kv.append(p + n)
    return offs, kv, slots, pos, [left, lacking], table


def _plan(dev, past, new, free, count, table, page, n_tokens, cols):
    from llmr_amd import serve
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t = i32(table).reshape(len(past), cols)
    guard = torch.full((n_tokens + 64,), 77, dtype=torch.int32, device=dev)
    b = serve.PagedBatch.empty(len(past), n_tokens, dev)
    b.slots = guard[:n_tokens]
    serve.paged_plan(i32(past), i32(new), i32(free), i32([count]), t, page, b)
    torch.cuda.synchronize()
    assert bool((guard[n_tokens:] == 77).all())
    return [x.tolist() for x in (b.seq_offsets, b.kv_len, b.slots, b.positions, b.pages)] + [t.tolist()]


def _held(past, page, cols, order):
    rows, used = [], 0
    for p in past:
        h = min(-(-max(p, 0) // page), cols)
        rows.append(order[used:used + h] + [-9] * (cols - h))
        used += h
    return rows, order[used:]


# (past, new, page, cols, spare free pages, rows behind the last token)
PLANS = [([0], [1], 16, 1, 0, 0), ([5], [1], 16, 4, 2, 0), ([16], [1], 16, 4, 2, 0), ([15], [1], 16, 4, 2, 3),
         ([0, 0, 0], [0, 0, 0], 16, 3, 4, 5), ([0, 31, 32, 33, 7], [40, 1, 1, 0, 200], 32, 20, 5, 0),
         ([100] * 70, [1] * 70, 16, 9, 100, 10), (list(range(300)), [(7 * i) % 50 for i in range(300)], 64, 8, 300, 99),
         ([0] * 1000, [1 + i % 3 for i in range(1000)], 256, 2, 1000, 0), ([4000, 0], [1, 3000], 128, 60, 30, 0)]


@pytest.mark.parametrize("past,new,page,cols,spare,pad", PLANS, ids=lambda x: str(x).replace(" ", "")[:24])
def test_paged_plan(dev, past, new, page, cols, spare, pad):
    g = torch.Generator().manual_seed(len(past) + page)
    need = sum(-(-(p + n) // page) for p, n in zip(past, new))
    order = torch.randperm(need + spare, generator=g).tolist()
    table, free = _held(past, page, cols, order)
    T = sum(new) + pad
    args = (past, new, free + [123456] * 3, len(free), table, page, T)
    assert _plan(dev, *args, cols) == list(_plan_oracle(*args))


@pytest.mark.parametrize("seed", range(6))
def test_paged_plan_random(dev, seed):
    import random
    r = random.Random(seed)
    n = r.choice([1, 3, 64, 257, 513, 1100])
    page, cols = r.choice([16, 32, 256]), r.randint(1, 40)
    past = [r.choice([0, r.randint(0, 600)]) for _ in range(n)]
    new = [r.choice([0, 1, 1, r.randint(0, 300)]) for _ in range(n)]
    order = list(range(40 * n + 7))
    r.shuffle(order)
    table, free = _held(past, page, cols, order)
    count = r.choice([len(free), 0, 1, min(len(free), 5), len(free) + 100])  # too few, and more than there is room for
    T = max(0, sum(new) + r.choice([0, 50, -20]))  # and fewer rows than new tokens
    args = (past, new, free, count, table, page, T)
    assert _plan(dev, *args, cols) == list(_plan_oracle(*args))


def test_paged_plan_bad_values(dev):
    """Negative lengths count as 0, a missing page gives slot -1, past the table's columns too, a negative count is
    no free page, a slot past 2^31 is none."""
    for past, new, free, count, table, page, T, cols in [
            ([-5, 20, 3], [2, -7, 1], [4, 5, 6], 3, [-9] * 6, 16, 8, 2),
            ([0, 10], [40, 40], [8, 9], 2, [-9] * 4, 16, 80, 2),
            ([0], [20], [8, 9], -4, [-9] * 4, 16, 20, 4),
            ([17], [3], [8], 1, [-1, -1, -9], 16, 3, 3),
            ([17, 1], [3, 2], [8], 1, [3, 2 ** 31 - 1, 2 ** 27, -9], 16, 5, 2),
            ([2 ** 31 - 1, 0], [2 ** 31 - 1, 1], [8], 1, [-9] * 4, 16, 40, 2)]:
        rows = [table[i * cols:(i + 1) * cols] for i in range(len(past))]
        got = _plan(dev, past, new, free, count, table, page, T, cols)
        if max(past) < 2 ** 31 - 1:
            assert got == list(_plan_oracle(past, new, free, count, rows, page, T))
        else:  # past the table from the start; the next request takes its page, its token is past the rows
            assert got[5] == [[-9, -9], [8, -9]] and got[2] == [-1] * T


def test_paged_plan_captured(dev):
    """A captured plan replays with other lengths and another free list."""
    from llmr_amd import serve
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    past, new, free, count = i32([0, 0, 0]), i32([3, 3, 3]), i32(list(range(50))), i32([50])
    table, b = torch.full((3, 8), -9, dtype=torch.int32, device=dev), serve.PagedBatch.empty(3, 64, dev)

    def step():
        serve.paged_plan(past, new, free, count, table, 16, b)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for p, n, c in (([0, 5, 16], [1, 20, 1], 50), ([31, 0, 32], [2, 0, 30], 4), ([0, 0, 0], [0, 0, 0], 0)):
        past.copy_(i32(p)), new.copy_(i32(n)), count.fill_(c)
        rows = [[40 + i if i < -(-x // 16) else -9 for i in range(8)] for x in p]
        table.copy_(i32(rows))
        graph.replay()
        torch.cuda.synchronize()
        want = _plan_oracle(p, n, list(range(50)), c, rows, 16, 64)
        assert [x.tolist() for x in (b.seq_offsets, b.kv_len, b.slots, b.positions, b.pages, table)] == list(want)


def test_paged_plan_refuses(dev):
    from llmr_amd import capi, serve
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
    past, new, free, count, table, b = i32(3), i32(3), i32(9), i32(1), i32(12).view(3, 4), serve.PagedBatch.empty(3, 20, dev)
    serve.paged_plan(past, new, free, count, table, 16, b)
    for args in ((past[:2], new, free, count, table, 16, b), (past.long(), new, free, count, table, 16, b),
                 (past, new, free, count, table.t(), 16, b), (past, new, free.cpu(), count, table, 16, b),
                 (past, new, free, count, table, 16, serve.PagedBatch.empty(2, 20, dev))):
        with pytest.raises(ValueError):
            serve.paged_plan(*args)
    for page in (0, 8, 24, 512):
        with pytest.raises(capi.LlmrError, match="page_size"):
            serve.paged_plan(past, new, free, count, table, page, b)
    shared = serve.PagedBatch.empty(3, 20, dev)
    shared.kv_len = past
    with pytest.raises(capi.LlmrError, match="kv_len overlaps past_len"):
        serve.paged_plan(past, new, free, count, table, 16, shared)
    buf = i32(60)
    shared = serve.PagedBatch.empty(3, 20, dev)
    shared.slots, shared.positions = buf[:20], buf[19:39]
    with pytest.raises(capi.LlmrError, match="positions overlaps slots"):
        serve.paged_plan(past, new, free, count, table, 16, shared)
    n = capi.MAX_SEQS + 1
    with pytest.raises(capi.LlmrError, match="n_seqs"):
        serve.paged_plan(i32(n), i32(n), free, count, i32(n).view(n, 1), 16, serve.PagedBatch.empty(n, 1, dev))


# ---- the projection's rows ----------------------------------------------------------


def _tables(dev, n, D):
    a = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
        -torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
    return a.cos().float(), a.sin().float()


def _rows_oracle(x, w, eps, rope, pos, halves):
    """x [T, heads, D] f32 -> (value, size) in 64 bits; size bounds what the f32 roundings scale with."""
    x = x.double()
    D = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if rope is None:
        return x, x.abs()
    c, s = (t.double()[pos][:, None] for t in rope)
    if halves:
        a, b = x[..., :D // 2], x[..., D // 2:]
        return (torch.cat([a * c - b * s, a * s + b * c], -1),
                torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1))
    a, b = x[..., ::2], x[..., 1::2]
    return (torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2),
            torch.stack([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1).flatten(-2))


def _close(got, want, size, dtype, what):
    """One rounding to the type (u |x|, fp16 under 2^-14: 2^-25) on a f32 result that is off by at most 2^-17 of its
    terms' sizes: the mean of D squares D 2^-24, halved by the root, then root, division, two products, two of the
    rotation and its sum, each 2^-24: (64 + 8) 2^-24 < 2^-17."""
    u = torch.finfo(dtype).eps / 2
    err = (got.double() - want).abs()
    bound = u * want.abs() + 2.0 ** -17 * size * (1 + u) + 2.0 ** -25
    assert bool((err <= bound).all()), (what, float((err / bound).max()))


# (D, H, Hk, T, page, norm, rope, halves)
ROWS = [(128, 4, 2, 1, 16, True, True, True), (64, 3, 1, 7, 32, True, True, False), (128, 32, 8, 64, 16, True, True, True),
        (64, 14, 2, 33, 64, False, True, True), (128, 5, 5, 100, 256, True, False, True), (64, 1, 1, 3, 16, False, False, False),
        (128, 30, 6, 21, 16, False, True, False), (64, 16, 4, 1030, 16, True, True, True), (128, 2, 1, 517, 128, True, True, False)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,H,Hk,T,page,norm,rope,halves", ROWS)
def test_qkv_tokens(dev, dtype, D, H, Hk, T, page, norm, rope, halves):
    from llmr_amd import serve
    g = torch.Generator(device=dev).manual_seed(T + H)
    width = (H + 2 * Hk) * D
    qkv = torch.randn(T, width + 12, generator=g, device=dev)[:, :width + 4] * 2
    qn, kn = (torch.rand(D, generator=g, device=dev) + 0.5 if norm else None for _ in range(2))
    tabs = _tables(dev, 900, D) if rope else None
    pos = torch.randint(0, 900, (T,), generator=g, device=dev)
    n_pages = -(-T // page) + 2
    slots = torch.randperm(n_pages * page, generator=g, device=dev)[:T].int()
    drop = torch.rand(T, generator=g, device=dev) < 0.2
    slots[drop] = torch.where(torch.rand(int(drop.sum()), generator=g, device=dev) < 0.5, -1, n_pages * page + 3).int()
    caches = [torch.full((n_pages, Hk, page, D), 7.0, dtype=dtype, device=dev) for _ in range(2)]
    q = torch.full((T, H + 1, D), 7.0, dtype=dtype, device=dev)
    serve.qkv_tokens(qkv, q[:, :H], caches[0], caches[1], slots=slots, positions=pos.int(), q_norm=qn, k_norm=kn,
                     eps=1e-5, rope=tabs, halves=halves)
    rows = [torch.empty(T, Hk, D, dtype=dtype, device=dev) for _ in range(2)]
    q2 = torch.empty(T, H, D, dtype=dtype, device=dev)
    serve.qkv_tokens(qkv, q2, rows[0], rows[1], positions=pos.int(), q_norm=qn, k_norm=kn, eps=1e-5, rope=tabs,
                     halves=halves)
    torch.cuda.synchronize()
    x = qkv[:, :width].reshape(T, H + 2 * Hk, D)
    _close(q[:, :H], *_rows_oracle(x[:, :H], qn, 1e-5, tabs, pos, halves), dtype, "q")
    _close(rows[0], *_rows_oracle(x[:, H:H + Hk], kn, 1e-5, tabs, pos, halves), dtype, "k")
    assert torch.equal(rows[1], x[:, H + Hk:].to(dtype))
    assert bool((q[:, H] == 7).all()) and torch.equal(q2, q[:, :H])
    live = ~drop
    at = slots[live].long()
    for c, r in zip(caches, rows):
        want = torch.full_like(c, 7.0).transpose(1, 2).reshape(-1, Hk, D)
        want[at] = r[live]
        assert torch.equal(c.transpose(1, 2).reshape(-1, Hk, D), want)


def test_qkv_tokens_positions(dev):
    """No positions: the row; positions outside the tables are taken at their ends."""
    from llmr_amd import serve
    D, T = 64, 40
    qkv = torch.randn(T, 3 * D, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    tabs = _tables(dev, T, D)

    def rows(pos):
        out = [torch.empty(T, 1, D, dtype=BF16, device=dev) for _ in range(3)]
        serve.qkv_tokens(qkv, *out, positions=pos, rope=tabs)
        return out

    i = torch.arange(T, device=dev, dtype=torch.int32)
    assert all(torch.equal(a, b) for a, b in zip(rows(None), rows(i)))
    far = i.clone()
    far[3], far[4], far[5] = -7, 2 ** 31 - 1, T
    near = i.clone()
    near[3], near[4], near[5] = 0, T - 1, T - 1
    assert all(torch.equal(a, b) for a, b in zip(rows(far), rows(near)))


def test_qkv_tokens_special_values(dev):
    """Infinities and NaN stay in their own head; a row of zeros with eps 0 is NaN as the formula says."""
    from llmr_amd import serve
    D, T, H, Hk = 128, 6, 2, 1
    qkv = torch.randn(T, 4 * D, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    w = torch.ones(D, device=dev)

    def rows(x, eps=1e-6):
        out = [torch.empty(T, h, D, dtype=F16, device=dev) for h in (H, Hk, Hk)]
        serve.qkv_tokens(x, *out, q_norm=w, k_norm=w, eps=eps)
        return out

    ref, bad = rows(qkv), qkv.clone()
    bad[2, 5] = math.nan          # q head 0
    bad[3, 3 * D + 1] = 1e9       # v: past fp16
    bad[4, 2 * D] = math.inf      # k
    got = rows(bad)
    keep = torch.ones(T, dtype=torch.bool, device=dev)
    keep[2] = False
    assert torch.equal(got[0][keep], ref[0][keep]) and torch.equal(got[0][2, 1], ref[0][2, 1])
    assert bool(got[0][2, 0].isnan().all())
    assert bool(got[2][3, 0, 1].isinf()) and int(got[2].isinf().sum()) == 1
    assert bool(got[1][4].isnan().any()) and bool(torch.isfinite(got[1][[0, 1, 2, 3, 5]]).all())
    zero = qkv.clone()
    zero[1, :D] = 0
    assert bool(rows(zero, 0.0)[0][1, 0].isnan().all()) and bool((rows(zero)[0][1, 0] == 0).all())


def test_qkv_tokens_refuses(dev):
    from llmr_amd import capi, serve
    D, T = 64, 5
    qkv = torch.zeros(T, 8 * D, device=dev)
    q, k, v = (torch.empty(T, h, D, dtype=F16, device=dev) for h in (4, 2, 2))
    cache = [torch.empty(3, 2, 16, D, dtype=F16, device=dev) for _ in range(2)]
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    tabs = _tables(dev, 4, D)
    serve.qkv_tokens(qkv, q, k, v)
    serve.qkv_tokens(qkv, q, *cache, slots=slots)
    for args, kw in (((qkv.half(), q, k, v), {}), ((qkv[:4], q, k, v), {}), ((qkv[:, :7 * D], q, k, v), {}),
                     ((qkv, q, k, v[:, :1]), {}), ((qkv, q, k, v.bfloat16()), {}), ((qkv, q, *cache), {}),
                     ((qkv, q, k, v), dict(slots=slots)), ((qkv, q, *cache), dict(slots=slots.long())),
                     ((qkv, q, *cache), dict(slots=slots[:4])), ((qkv, q, k, v), dict(q_norm=torch.ones(D, device=dev).half())),
                     ((qkv, q, k, v), dict(rope=(tabs[0], tabs[1][:, :8]))), ((qkv, q, k, v), dict(rope=tabs)),
                     ((qkv, q.float(), k.float(), v.float()), {}), ((qkv, q, k, v), dict(eps=-1.0)),
                     ((qkv, q, k, v), dict(eps=math.nan)), ((qkv.cpu(), q, k, v), {}),
                     ((qkv, q.transpose(0, 1).contiguous().transpose(0, 1), k, v), {})):
        with pytest.raises((ValueError, capi.LlmrError)):
            serve.qkv_tokens(*args, **kw)
    serve.qkv_tokens(qkv[:0], q[:0], k[:0], v[:0])


# ---- a run of them ------------------------------------------------------------------


def _softmax_rows(q, k, v):
    """Causal attention of the last rows q [n, H, D] over k, v [m, Hk, D] in f64."""
    n, H, D = q.shape
    m, Hk = k.shape[:2]
    out = torch.empty(n, H, D, dtype=torch.float64, device=q.device)
    hidden = torch.arange(m, device=q.device)[None] > torch.arange(m - n, m, device=q.device)[:, None]
    for h in range(H):
        s = (q[:, h].double() @ k[:, h // (H // Hk)].double().t() / math.sqrt(D)).masked_fill(hidden, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, h // (H // Hk)].double()
    return out


@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_steps(dev, captured):
    """Requests that come, grow by chunks and by single tokens and leave, over Q8_0 projections: plan, QKV GEMM,
    qkv_tokens, paged_attention on one padded batch, four steps; each request's rows equal the attention over all its
    rows so far, kept contiguously beside. The first step's chunk equals prompt_attention's rows."""
    import numpy as np

    from llmr_amd import gguf, ops, serve, synth
    D, H, Hk, hidden, page, rows = 64, 4, 2, 256, 16, 160
    width = (H + 2 * Hk) * D
    w = torch.from_numpy(gguf.quantize(synth.normal(3, 2, width * hidden, 0.06), gguf.GGML_Q8_0)).to(dev)
    W = ops.Tensor.quantized(w, gguf.GGML_Q8_0, width, hidden)
    qn, kn = (torch.from_numpy(synth.normal(3, 10 + i, D, 0.1) + 1).float().to(dev) for i in range(2))
    tabs = _tables(dev, 512, D)
    n = 3
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    past, new = i32([0] * n), i32([0] * n)
    free, count = torch.arange(40, dtype=torch.int32, device=dev), i32([40])
    table = torch.full((n, 16), -1, dtype=torch.int32, device=dev)
    caches = [torch.full((40, Hk, page, D), math.nan, dtype=BF16, device=dev) for _ in range(2)]
    x = torch.zeros(rows, hidden, dtype=BF16, device=dev)
    qkv = torch.zeros(rows, width, device=dev)
    q = torch.zeros(rows, H, D, dtype=BF16, device=dev)
    out = torch.zeros(rows, H * D, dtype=BF16, device=dev)
    b = serve.PagedBatch.empty(n, rows, dev)
    scratch = serve.paged_attention_scratch(q, caches[0], table, rows)
    g = ops.default_graph()

    def step():
        serve.paged_plan(past, new, free, count, table, page, b)
        ops.dispatch_batch_matmul(g, W, ops.Tensor.from_torch(x), ops.Tensor.from_torch(qkv), width, hidden, rows, 0)
        serve.qkv_tokens(qkv, q, *caches, slots=b.slots, positions=b.positions, q_norm=qn, k_norm=kn, rope=tabs)
        serve.paged_attention(q, *caches, b.seq_offsets, b.kv_len, table, rows, out=out, scratch=scratch)

    graph = None
    if captured:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    seen = [[None, None] for _ in range(n)]
    lens = [0] * n
    rng = np.random.default_rng(0)
    for i, (ns, ends) in enumerate([([90, 30, 0], []), ([1, 1, 47], []), ([1, 33, 1], [0]), ([150, 1, 1], [])]):
        past.copy_(i32(lens)), new.copy_(i32(ns))
        x.copy_(torch.from_numpy(rng.standard_normal((rows, hidden)).astype(np.float32)))
        out.fill_(7.0)
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        T = sum(ns)
        kr, vr = (torch.empty(rows, Hk, D, dtype=BF16, device=dev) for _ in range(2))
        q2 = torch.empty_like(q)
        serve.qkv_tokens(qkv, q2, kr, vr, positions=b.positions, q_norm=qn, k_norm=kn, rope=tabs)
        assert torch.equal(q, q2) and bool((out[T:] == 7).all())
        if i == 0:
            first = serve.prompt_attention(q, kr, vr, b.seq_offsets)
            assert float((first[:T].double() - out[:T].double()).abs().max()) <= 4 * 2.0 ** -8 * 4
        at = 0
        for s, m in enumerate(ns):
            for j, r in enumerate((kr, vr)):
                part = r[at:at + m].clone()
                seen[s][j] = part if seen[s][j] is None else torch.cat([seen[s][j], part])
            lens[s] += m
            if m:
                ref = _softmax_rows(q[at:at + m], *seen[s])
                err = (out[at:at + m].unflatten(1, (H, D)).double() - ref).abs().max()
                # weights rounded (2 u A), result rounded (u A), A <= max |v|
                assert float(err) <= 3.2 * 2.0 ** -8 * float(seen[s][1].double().abs().max()), (i, s)
            at += m
        count.copy_(b.pages[:1])
        assert int(b.pages[1]) == 0
        for s in ends:  # its pages go back; the request in its place starts anew
            held = -(-lens[s] // page)
            c = int(count)
            free[c:c + held] = table[s, :held]
            count += held
            lens[s], seen[s] = 0, [None, None]
            table[s] = -1


def test_qkv_tokens_more_rows_than_one_grid_dimension(dev):
    """2^24 rows and more (workgroups of 256 threads: more than 2^32 threads along one dimension of a grid)."""
    from llmr_amd import serve
    D, T = 64, 2 ** 24 + 37
    g = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn(T, 3 * D, generator=g, device=dev)
    w = torch.rand(D, generator=g, device=dev) + 0.5
    pos = torch.randint(0, 900, (T,), generator=g, device=dev, dtype=torch.int32)
    tabs = _tables(dev, 900, D)
    q, k, v = (torch.zeros(T, 1, D, dtype=BF16, device=dev) for _ in range(3))
    serve.qkv_tokens(qkv, q, k, v, positions=pos, q_norm=w, k_norm=w, rope=tabs)
    torch.cuda.synchronize()
    assert torch.equal(v[:, 0], qkv[:, 2 * D:].bfloat16())
    n = 1 << 22
    for a in range(0, T, n):  # the same rows, fewer at a time
        b = min(T, a + n)
        parts = [torch.zeros(b - a, 1, D, dtype=BF16, device=dev) for _ in range(3)]
        serve.qkv_tokens(qkv[a:b], *parts, positions=pos[a:b], q_norm=w, k_norm=w, rope=tabs)
        assert torch.equal(parts[0], q[a:b]) and torch.equal(parts[1], k[a:b]), a
    page = 256
    caches = [torch.zeros(-(-T // page), 1, page, D, dtype=BF16, device=dev) for _ in range(2)]
    slots = torch.arange(T - 1, -1, -1, dtype=torch.int32, device=dev)
    serve.qkv_tokens(qkv, q, *caches, slots=slots, positions=pos, q_norm=w, k_norm=w, rope=tabs)
    torch.cuda.synchronize()
    assert torch.equal(caches[0].view(-1, D)[:T].flip(0), k[:, 0]) and torch.equal(caches[1].view(-1, D)[:T].flip(0), v[:, 0])
