"""GPU attention of batches of requests (llmr_prompt_attention, llmr_paged_attention) against its definition in
64 bits, element by element.

Where a tolerance is compared, it is this bound. With u = eps / 2 of the type (half a step):
  - a softmax weight is rounded to the type once, for its product with v: weights p_j (1 + d_j), |d_j| <= u. The
    sum that divides is of the weights before that: the result is off by at most u A, A = sum_j p_j |v_j|; by
    at most 2 u A / (1 - u), which is what is allowed here, were it of the rounded ones;
  - a score is a f32 sum of D products: off by at most (D + 4) 2^-24 sum_d |q_d k_jd| scale (the four: the scale,
    its product with log2(e), the running maximum's subtraction), its exponential relatively as much, and 2^-22
    for exp2 itself and the sums' own f32 additions (their terms are non-negative: a tree over 64 lanes or fewer
    and a running sum, n 2^-24 at the worst, taken in full): together e, again 2 e A;
  - fp16 weights under 2^-14 of their scale lose bits: at most 2^-25 each before the division by the sum, whose
    largest term is at least 2^-8 of the scale (the kernels let a maximum lag by 2^8), so n 2^-17 max|v| is a
    bound for any n keys; none for bf16, which has f32's exponents;
  - the result is rounded once: u |out| (fp16 results under 2^-14: 2^-25).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _definition(q, k, v, scale, first):
    """q [n, H, D], k, v [m, Hk, D] (as given, any type) -> out [n, H, D], A, e in 64 bits; query i sees the keys
    j <= first + i. What a row does not see is left out of its sums whatever it holds."""
    n, H, D = q.shape
    m, Hk = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    out, A = (torch.zeros(n, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    e = torch.zeros(n, H, 1, dtype=torch.float64, device=q.device)
    pos = torch.arange(n, device=q.device) + first
    for h in range(H):
        kh, vh = k[:, h // (H // Hk)], v[:, h // (H // Hk)]
        hidden = torch.arange(m, device=q.device)[None] > pos[:, None]
        s = torch.where(hidden, -math.inf, q[:, h] @ kh.t() * scale) if not kh.isnan().any() else torch.where(
            hidden, -math.inf, (q[:, h][:, None] * kh[None]).sum(-1) * scale)
        size = torch.where(hidden, 0.0, q[:, h].abs() @ kh.abs().nan_to_num(0, 0, 0).t() * scale)
        p = torch.softmax(s, dim=-1).nan_to_num(0.0) if not bool((pos >= 0).all()) else torch.softmax(s, dim=-1)
        fine = vh.isfinite().all()
        if bool(fine):
            out[:, h], A[:, h] = p @ vh, p @ vh.abs()
        else:
            x = torch.where(hidden[:, :, None], 0.0, p[:, :, None] * vh[None])
            out[:, h], A[:, h] = x.sum(1), x.abs().sum(1)
        e[:, h, 0] = size.amax(-1) * (D + 4) * 2.0 ** -24 + 2.0 ** -22 + m * 2.0 ** -24
    return out, A, e


def _check(got, out, A, e, vmax, keys, dtype, what):
    u = torch.finfo(dtype).eps / 2
    lost = keys * 2.0 ** -17 * vmax if dtype == F16 else 0.0
    bound = 2 * (u / (1 - u) + e) * A + u * out.abs() + lost + 2.0 ** -25
    got = got.double()
    nan = out.isnan()
    assert torch.equal(got.isnan(), nan), (what, "NaN in other places", int((got.isnan() != nan).sum()))
    off = torch.where(nan, 0.0, (got - out).abs() / bound)
    worst = float(off.max()) if off.numel() else 0.0
    print(f"{what}: worst error {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)


def _near(a, b, v, what):
    """Two results of one definition, each within 2 u A + u |out| of it (A, |out| <= max|v|), f32's part aside."""
    assert bool(torch.isfinite(a).all()) and bool(torch.isfinite(b).all()), what
    u, vmax = torch.finfo(v.dtype).eps / 2, float(v.double().nan_to_num(0, 0, 0).abs().max())
    worst = float((a.double() - b.double()).abs().max()) if a.numel() else 0.0
    assert worst <= 6.2 * u * vmax, (what, worst)


def _say(*a):
    print(*a, flush=True)


def _prompt_case(dev, dtype, D, H, Hk, lens, pad=0, seed=0, layout="tokens", qstd=1.5, shift=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lens) + pad

    def rnd(heads, std=1.0):
        return torch.randn(T, heads, D, generator=g, device=dev) * std

    q, k, v = rnd(H, qstd) + shift, rnd(Hk) + shift, rnd(Hk)
    if layout == "columns":  # slices of one wider QKV row
        buf = torch.zeros(T, (H + 2 * Hk) * D + 24, dtype=dtype, device=dev)
        x = buf[:, 8:8 + (H + 2 * Hk) * D].unflatten(1, (H + 2 * Hk, D))
        x.copy_(torch.cat([q, k, v], dim=1))
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    elif layout == "heads":  # head-major, as llmr_qkv_heads writes them
        q, k, v = (t.to(dtype).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    else:
        q, k, v = (t.to(dtype) for t in (q, k, v))
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return q, k, v, at, torch.tensor(at, dtype=torch.int32, device=dev)


def _prompt_check(q, k, v, at, out, scale, what, fill=None):
    H, D = q.shape[1:]
    for i, (a, b) in enumerate(zip(at, at[1:])):
        if b > a:
            o, A, e = _definition(q[a:b], k[a:b], v[a:b], scale, 0)
            vm = float(v[a:b].double().nan_to_num(0, 0, 0).abs().max())
            _check(out[a:b].unflatten(1, (H, D)), o, A, e, vm, b - a, q.dtype, f"{what} request {i} ({b - a} rows)")
    if fill is not None:
        assert bool((out[at[-1]:] == fill).all()) and bool((out[:at[0]] == fill).all())


# (D, H, Hk, lens, pad): one token; around the tiles of 16, 32, 64, 128 and 256 rows or keys; empty requests first,
# last and between; groups of 1 to 16 heads that divide a tile and that do not; many short requests in one tile
PROMPTS = [(128, 4, 2, [1], 0), (64, 3, 1, [1, 0, 1], 5), (128, 8, 2, [77], 0), (128, 2, 2, [63, 64, 65], 3),
           (64, 6, 2, [0, 255, 1, 0, 256, 0], 0), (128, 5, 1, [257, 31], 9), (64, 7, 1, [129, 128, 127], 0),
           (128, 16, 1, [33, 15, 17, 300], 1), (128, 3, 3, [513], 0), (64, 8, 8, [700, 3], 64),
           (128, 4, 1, [1] * 70 + [2, 3, 5, 200], 7), (64, 14, 2, [1000], 0), (128, 32, 8, [1500, 41], 0),
           (128, 12, 2, [2100], 11)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,H,Hk,lens,pad", PROMPTS, ids=lambda x: str(x).replace(" ", "")[:30])
def test_prompt_attention(dev, dtype, D, H, Hk, lens, pad):
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, dtype, D, H, Hk, lens, pad, seed=sum(lens) + H)
    if pad:  # what lies behind the last request is nobody's
        for t in (q, k, v):
            t[at[-1]:] = math.nan
    out = torch.full((q.shape[0], H * D), 7.0, dtype=dtype, device=dev)
    assert serve.prompt_attention(q, k, v, off, out=out) is out
    torch.cuda.synchronize()
    _prompt_check(q, k, v, at, out, 1 / math.sqrt(D), f"{dtype} D={D} H={H}/{Hk}", 7.0)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,H,Hk,lens", [(64, 24, 8, [2800, 150]), (64, 18, 6, [13, 40, 200, 1, 370, 90] * 6),
                                         (128, 20, 5, [5, 130, 64, 300] * 5)], ids=["long", "ragged", "ragged128"])
def test_prompt_attention_more_rows_than_the_card_holds(dev, dtype, D, H, Hk, lens):
    """256 rows a workgroup: waves whose rows begin or end tiles away from their neighbours'."""
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, dtype, D, H, Hk, lens, seed=len(lens))
    out = serve.prompt_attention(q, k, v, off)
    torch.cuda.synchronize()
    _prompt_check(q, k, v, at, out, 1 / math.sqrt(D), f"{dtype} D={D} H={H}/{Hk}")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_prompt_attention_unseen_values_across_requests(dev, bad):
    """Keys and values of one packed request that are not finite reach no row of its neighbours, whichever tile of a
    shared workgroup they lie in."""
    from llmr_amd import serve
    lens = [30, 100, 200, 7, 64, 64, 90, 1, 150]
    q, k, v, at, off = _prompt_case(dev, BF16, 128, 8, 2, lens, seed=17)
    ref = serve.prompt_attention(q, k, v, off)
    for i in (1, 3, 5, 8):
        for t in (k, v):
            t[at[i]:at[i + 1]] = bad
    out = serve.prompt_attention(q, k, v, off)
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(at, at[1:])):
        if i in (1, 3, 5, 8):
            assert not bool(out[a:b].isfinite().any()), i
        else:
            assert torch.equal(out[a:b], ref[a:b]), i


@pytest.mark.parametrize("layout", ["columns", "heads"])
@pytest.mark.parametrize("D,H,Hk,lens", [(128, 6, 2, [70, 0, 200]), (64, 4, 4, [300, 1]), (128, 1, 1, [90])])
def test_prompt_attention_strides(dev, layout, D, H, Hk, lens):
    """Column slices of a wider row, head-major buffers, and out in the columns of a wider row."""
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, F16, D, H, Hk, lens, seed=3, layout=layout)
    wide = torch.full((q.shape[0], H * D + 40), 7.0, dtype=F16, device=dev)
    serve.prompt_attention(q, k, v, off, 0.11, out=wide[:, 16:16 + H * D])
    torch.cuda.synchronize()
    _prompt_check(q, k, v, at, wide[:, 16:16 + H * D], 0.11, layout)
    assert bool((wide[:, :16] == 7).all()) and bool((wide[:, 16 + H * D:] == 7).all())
    same = serve.prompt_attention(*(t.contiguous() for t in (q, k, v)), off, 0.11)
    assert torch.equal(same, wide[:, 16:16 + H * D])


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("qstd,shift", [(30.0, 0.0), (0.01, 0.0), (1.0, 1.5), (1.0, -3.0)])
def test_prompt_attention_score_ranges(dev, dtype, qstd, shift):
    """Scores of hundreds (the maximum rises many times), next to zero, and far from zero on one side."""
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, dtype, 128, 4, 2, [400, 90], seed=9, qstd=qstd, shift=abs(shift))
    if shift < 0:  # all scores far below zero
        q = -q
    out = serve.prompt_attention(q, k, v, off)
    torch.cuda.synchronize()
    _prompt_check(q, k, v, at, out, 1 / math.sqrt(128), f"qstd {qstd} shift {shift}")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_prompt_attention_rising_and_falling_scores(dev, dtype):
    """Keys in order of their scores, up and down: every key raises the maximum, or every later weight is tiny."""
    from llmr_amd import serve
    T, D = 600, 64
    v = torch.randn(T, 1, D, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(dtype)
    for sign in (1.0, -1.0):
        ramp = torch.linspace(0, 40, T, device=dev)[:, None, None] * sign
        k = torch.zeros(T, 1, D, device=dev)
        k[..., :1] = ramp
        q = torch.zeros(T, 2, D, device=dev)
        q[..., :1] = torch.tensor([1.0, 4.0], device=dev)[None, :, None]
        q, k = q.to(dtype), k.to(dtype)
        out = serve.prompt_attention(q, k, v, torch.tensor([0, T], dtype=torch.int32, device=dev), 1.0)
        torch.cuda.synchronize()
        _prompt_check(q, k, v, [0, T], out, 1.0, f"ramp {sign}")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_attention_unseen_values_do_not_matter(dev, dtype, bad):
    """An infinity or NaN in a key or a value reaches the rows that see it and no other: earlier rows of its own
    request (whose tiles hold it) and other requests beside it are as if it were not there."""
    from llmr_amd import serve
    lens = [40, 150, 70]
    for where in ("k", "v"):
        for row in (0, 39, 45, 189, 190, 200, 259):
            _say(f"{bad} in {where} row {row}")
            q, k, v, at, off = _prompt_case(dev, dtype, 128, 4, 2, lens, seed=12)
            clean = serve.prompt_attention(q, k, v, off).clone()
            (k if where == "k" else v)[row, 1, 5] = bad
            out = serve.prompt_attention(q, k, v, off)
            torch.cuda.synchronize()
            s = next(i for i in range(3) if at[i] <= row < at[i + 1])
            sees = torch.zeros(sum(lens), dtype=torch.bool, device=dev)
            sees[row:at[s + 1]] = True
            o, c = (t.unflatten(1, (4, 128)) for t in (out, clean))
            _near(o[~sees], c[~sees], v, (where, row))
            _near(o[:, :2], c[:, :2], v, (where, row))  # the other key/value head
            ref = _definition(q[at[s]:at[s + 1]], k[at[s]:at[s + 1]], v[at[s]:at[s + 1]], 1 / math.sqrt(128), 0)[0]
            got = o[at[s]:at[s + 1]].double()
            if where == "v":
                assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isinf(), ref.isinf()), (row, bad)
            else:
                assert torch.equal(got.isnan(), ref.isnan()), (row, bad)


def test_prompt_attention_lowest_values(dev):
    """Keys of the type's lowest and largest values (a mask written into the data): finite scores in f32."""
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, BF16, 64, 2, 1, [130], seed=4)
    q = torch.zeros_like(q)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[5::7, :, 0] = torch.finfo(BF16).min
    out = serve.prompt_attention(q, k, v, off, 1.0)
    torch.cuda.synchronize()
    o = _definition(q, k, v, 1.0, 0)[0]
    assert bool(torch.isfinite(out).all())
    u = torch.finfo(BF16).eps / 2
    err = (out.unflatten(1, (2, 64)).double() - o).abs()
    assert bool((err <= 3.1 * u * 5).all())  # weights are 0 or equal: means of values within +-5
    k[:, :, 0] = torch.finfo(BF16).min  # every score the lowest: a plain mean
    out = serve.prompt_attention(q, k, v, off, 1.0)
    err = (out.unflatten(1, (2, 64)).double() - _definition(q, k, v, 1.0, 0)[0]).abs()
    assert bool((err <= 3.1 * u * 5).all())


def test_prompt_attention_matches_one_request_at_a_time(dev):
    """Packing changes no bit: a request's rows are the same alone and between others."""
    from llmr_amd import serve
    lens = [256, 300, 0, 64, 512]
    q, k, v, at, off = _prompt_case(dev, BF16, 128, 8, 2, lens, seed=21)
    out = serve.prompt_attention(q, k, v, off)
    again = serve.prompt_attention(q, k, v, off)
    assert torch.equal(out, again)
    for a, b in zip(at, at[1:]):
        if b > a:
            one = serve.prompt_attention(q[a:b], k[a:b], v[a:b], torch.tensor([0, b - a], dtype=torch.int32, device=dev))
            err = (one.double() - out[a:b].double()).abs().max()
            assert float(err) <= 4 * 2.0 ** -8 * 5


def test_prompt_attention_offsets_outside_the_rows(dev):
    """Offsets past n_tokens, negative or not starting at 0 read and write nothing outside the rows."""
    from llmr_amd import serve
    q, k, v, _, _ = _prompt_case(dev, F16, 64, 2, 2, [100], seed=5)
    guard = torch.full((164, 128), 7.0, dtype=F16, device=dev)
    for offs, rows in (([10, 60], (10, 60)), ([40, 1000], (40, 100)), ([100, 200], (100, 100)), ([0, 0, 0], (0, 0))):
        guard.fill_(7.0)
        serve.prompt_attention(q, k, v, torch.tensor(offs, dtype=torch.int32, device=dev), out=guard[:100])
        torch.cuda.synchronize()
        assert bool((guard[:rows[0]] == 7).all()) and bool((guard[rows[1]:] == 7).all()), offs
        if rows[1] > rows[0]:
            a, b = rows
            one = serve.prompt_attention(q[a:b], k[a:b], v[a:b], torch.tensor([0, b - a], dtype=torch.int32, device=dev))
            assert float((one.double() - guard[a:b].double()).abs().max()) <= 4 * 2.0 ** -11 * 5


def _capture(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fn()
    return g


def test_prompt_attention_captured(dev):
    """A captured call replays with other lengths and inputs, beside eager calls of its own."""
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, BF16, 128, 6, 2, [100, 0, 211], 30, seed=6)
    out = torch.full((q.shape[0], 768), 7.0, dtype=BF16, device=dev)
    graph = _capture(lambda: serve.prompt_attention(q, k, v, off, out=out))
    for offs in ([0, 100, 100, 311], [0, 5, 300, 341], [0, 0, 0, 1], [0, 341, 341, 341]):
        off.copy_(torch.tensor(offs, dtype=torch.int32, device=dev))
        v.mul_(-1)
        out.fill_(7.0)
        graph.replay()
        eager = torch.full_like(out, 7.0)
        serve.prompt_attention(q, k, v, off, out=eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), offs
        _prompt_check(q, k, v, offs, out, 1 / math.sqrt(128), str(offs), 7.0)


def test_prompt_attention_streams(dev):
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, F16, 64, 8, 2, [500, 40], seed=8)
    ref = serve.prompt_attention(q, k, v, off)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(serve.prompt_attention(q, k, v, off))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


# ---- paged ------------------------------------------------------------------------


def _paged_case(dev, dtype, D, H, Hk, page, past, new, pad=0, seed=0, spare=3, poison=True, qstd=1.5):
    """Contiguous rows of every request (the oracle's), the same in shuffled pages; what no request holds is NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    kv = [p + n for p, n in zip(past, new)]
    need = [-(-n // page) for n in kv]
    n_pages = sum(need) + spare
    caches = [torch.full((n_pages, Hk, page, D), math.nan if poison else 0.0, dtype=dtype, device=dev) for _ in range(2)]
    order = torch.randperm(n_pages, generator=g, device=dev)
    table = torch.full((len(kv), max(max(need), 1) + 1), -1, dtype=torch.int32, device=dev)
    rows, used = [], 0
    for i, n in enumerate(kv):
        k, v = (torch.randn(n, Hk, D, generator=g, device=dev).to(dtype) for _ in range(2))
        rows.append((k, v))
        pages = order[used:used + need[i]]
        used += need[i]
        table[i, :need[i]] = pages.int()
        j = torch.arange(n, device=dev)
        for c, x in zip(caches, (k, v)):
            c[pages[j // page], :, j % page] = x
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    q = (torch.randn(at[-1] + pad, H, D, generator=g, device=dev) * qstd).to(dtype)
    if pad:
        q[at[-1]:] = math.nan
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    return q, caches[0], caches[1], rows, at, i32(at), i32(kv), table, kv


def _paged_check(q, rows, at, kv, out, scale, what):
    H, D = q.shape[1:]
    for i, (a, b) in enumerate(zip(at, at[1:])):
        if b > a:
            k, v = rows[i]
            o, A, e = _definition(q[a:b], k, v, scale, kv[i] - (b - a))
            _check(out[a:b].unflatten(1, (H, D)), o, A, e, float(v.double().abs().max()), kv[i], q.dtype,
                   f"{what} request {i} ({b - a} of {kv[i]})")


# (D, H, Hk, page, past, new, pad): single tokens from one cached key to long contexts; pages that end inside a tile;
# requests with nothing new; small chunks of one tile with their group; chunks over several tiles; all at once
PAGED = [(128, 4, 2, 16, [0], [1], 0), (128, 32, 8, 16, [1100], [1], 0), (64, 8, 2, 32, [15, 16, 17, 0, 300], [1] * 5, 3),
         (128, 30, 6, 16, [5, 1000, 63, 64, 127, 128, 2047], [1] * 7, 0), (128, 8, 8, 64, [64, 63, 700], [1, 1, 1], 0),
         (64, 16, 1, 256, [3000, 1, 255, 256], [1] * 4, 0), (128, 4, 4, 128, [20000], [1], 0),
         (128, 8, 2, 16, [50, 0, 200, 7], [4, 4, 2, 0], 0), (64, 14, 2, 16, [33, 900], [2, 5], 1),
         (128, 32, 8, 32, [500], [64], 0), (128, 12, 2, 64, [0], [130], 0), (64, 5, 1, 16, [77, 0], [300, 1], 5),
         (128, 8, 2, 16, [40, 3000, 0, 1000, 9], [1, 129, 257, 0, 33], 6), (64, 3, 3, 128, [100, 600], [200, 100], 0),
         (128, 16, 1, 16, [1500], [17], 0), (128, 24, 8, 16, [0] * 12 + [400] * 12, [1, 20] * 12, 0),
         (128, 8, 1, 16, [70, 70], [9, 40], 0), (128, 2, 2, 16, [300, 2], [31, 65], 0)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,H,Hk,page,past,new,pad", PAGED, ids=lambda x: str(x).replace(" ", "")[:24])
def test_paged_attention(dev, dtype, D, H, Hk, page, past, new, pad):
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, H, Hk, page, past, new, pad, seed=sum(past) + H)
    out = torch.full((q.shape[0], H * D), 7.0, dtype=dtype, device=dev)
    assert serve.paged_attention(q, kc, vc, off, kvl, table, max(new), out=out) is out
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(D), f"D={D} H={H}/{Hk} page={page}")
    assert bool((out[at[-1]:] == 7).all())
    # a larger bound on the new tokens, another scratch and a wider table change the split at most
    wide = torch.full((table.shape[0], table.shape[1] + 700), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    out2 = serve.paged_attention(q, kc, vc, off, kvl, wide, q.shape[0])
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out2, 1 / math.sqrt(D), "wide")


# more requests than a wave's lanes, some of them with nothing new, at the ends too
MANY = [(128, 8, 2, [0, 1, 1, 0, 1] * 40), (64, 8, 2, [0, 5, 1, 8] * 30 + [0] * 70 + [3]), (128, 8, 2, [16, 0, 9, 1] * 20),
        (64, 4, 1, [0] * 65 + [70, 1, 0, 300, 2] * 14 + [0] * 3)]


@pytest.mark.parametrize("D,H,Hk,new", MANY, ids=["1", "8", "16", "300"])
def test_paged_attention_many_requests(dev, D, H, Hk, new):
    from llmr_amd import serve
    past = [(37 * i * i) % 211 for i in range(len(new))]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, D, H, Hk, 16, past, new, 2, seed=len(new))
    out = torch.full((q.shape[0], H * D), 7.0, dtype=BF16, device=dev)
    serve.paged_attention(q, kc, vc, off, kvl, table, max(new), out=out)
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(D), f"{len(new)} requests")
    assert bool((out[at[-1]:] == 7).all())


@pytest.mark.parametrize("hole", [None, 1000, 68000], ids=["whole", "hole-early", "hole-late"])
def test_paged_attention_table_longer_than_is_staged_at_once(dev, hole):
    """2048 new tokens behind 70000 keys: a workgroup's share is more tiles than it keeps pages of. Keys on no page
    are nobody's; the first and last rows of the chunk are looked at."""
    from llmr_amd import serve
    D, H, Hk, page, past, new = 64, 32, 8, 16, 70000, 2048
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, D, H, Hk, page, [past], [new], seed=5)
    k, v = rows[0]
    if hole is not None:
        table[0, hole // page] = -1
        lo = hole // page * page
        k, v = (torch.cat([t[:lo], t[lo + page:]]) for t in (k, v))
        past -= page
    out = serve.paged_attention(q, kc, vc, off, kvl, table, new)
    torch.cuda.synchronize()
    vm = float(v.double().abs().max())
    for a, b in ((0, 20), (new - 20, new)):
        o, A, e = _definition(q[a:b], k, v, 1 / math.sqrt(D), past + a)
        _check(out[a:b].unflatten(1, (H, D)), o, A, e, vm, past + b, F16, f"rows {a} .. {b}")


@pytest.mark.parametrize("qstd", [30.0, 0.01])
@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_paged_attention_score_ranges(dev, qstd, new):
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 128, 8, 2, 16, [900, 333], new, seed=2, qstd=qstd)
    out = serve.paged_attention(q, kc, vc, off, kvl, table, max(new))
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(128), f"qstd {qstd}")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,row", [(3, 98), (3, 99), (100, 150), (100, 190), (40, 101), (40, 120)])
def test_paged_attention_unseen_values_do_not_matter(dev, dtype, new, row):
    """A NaN or infinity in the key or value of a new token reaches the rows that see it and no other."""
    from llmr_amd import serve
    past = 97 if new == 3 else 96
    for where in (0, 1):
        for bad in (math.nan, math.inf):
            _say(f"{bad} in {'kv'[where]}, {new} new")
            q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, 128, 8, 2, 16, [past, 60], [new, 1], seed=5)
            clean = serve.paged_attention(q, kc, vc, off, kvl, table, new).clone()
            page = int(table[0, row // 16])
            (kc, vc)[where][page, 1, row % 16, 70] = bad
            rows[0][where][row, 1, 70] = bad
            out = serve.paged_attention(q, kc, vc, off, kvl, table, new)
            torch.cuda.synchronize()
            o, c = (t.unflatten(1, (8, 128)) for t in (out, clean))
            first = row - past  # the new token it belongs to
            keep = torch.ones(new + 1, dtype=torch.bool, device=dev)
            keep[first:new] = False
            _near(o[keep], c[keep], rows[0][1], (where, bad))
            _near(o[:, :4], c[:, :4], rows[0][1], (where, bad))
            ref = _definition(q[:new], *rows[0], 1 / math.sqrt(128), past)[0]
            got = o[:new].double()
            assert torch.equal(got.isnan(), ref.isnan()), (where, bad)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [20, 1, 70, 2]])
def test_paged_attention_bad_tables_and_lengths(dev, new):
    """Pages outside the cache are seen by nobody, lengths past the table end with it, a row that sees no key is
    0, and requests beside them keep their results."""
    from llmr_amd import serve
    past = [200, 100, 90, 50]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, 128, 4, 2, 16, past, new, seed=7)
    ref = serve.paged_attention(q, kc, vc, off, kvl, table, max(new)).clone()
    cols = table.shape[1]
    n_pages = kc.shape[0]
    bad = table.clone()
    bad[0, 3], bad[0, 5], bad[0, 6] = -1, n_pages, 2 ** 31 - 1
    out = serve.paged_attention(q, kc, vc, off, kvl, bad, max(new))
    torch.cuda.synchronize()
    assert torch.equal(out[at[1]:], ref[at[1]:])
    seen = torch.ones(kv[0], dtype=torch.bool, device=dev)
    for c in (3, 5, 6):
        seen[16 * c:16 * c + 16] = False
    k, v = (x[seen] for x in rows[0])
    n = at[1]
    o, A, e = _definition(q[:n], k, v, 1 / math.sqrt(128), int(seen.sum()) - n)
    _check(out[:n].unflatten(1, (4, 128)), o, A, e, float(v.double().abs().max()), kv[0], BF16, "holes")
    bad = torch.full_like(table, -1)
    out = serve.paged_attention(q, kc, vc, off, kvl, bad, max(new))
    torch.cuda.synchronize()
    assert bool((out[:at[-1]] == 0).all())
    for lens in ([0, 0, 0, 0], [-5, -1, -2 ** 31, -100]):  # shorter than the new tokens: no key for the first ones
        out = serve.paged_attention(q, kc, vc, off, torch.tensor(lens, dtype=torch.int32, device=dev), table, max(new))
        torch.cuda.synchronize()
        assert bool((out[:at[-1]] == 0).all()), lens
    big = kvl.clone()
    big[1], big[2] = 2 ** 31 - 1, 16 * cols + 1000  # the table ends first; what is past it nobody sees
    filled = table.clone()
    filled[filled < 0] = int(table[0, 0])
    out = serve.paged_attention(q, kc.nan_to_num(0.0), vc.nan_to_num(0.0), off, big, filled, max(new))
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out[:at[-1]]).all())
    for i in (0, 3):
        _near(out[at[i]:at[i + 1]], ref[at[i]:at[i + 1]], rows[i][1], i)


def test_paged_attention_more_new_than_cached(dev):
    """kv_len under the request's rows: the first rows see nothing and are 0, the last see the cached keys."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 64, 4, 1, 16, [0], [100], seed=3)
    kvl.fill_(70)
    out = serve.paged_attention(q, kc, vc, off, kvl, table, 100)
    torch.cuda.synchronize()
    assert bool((out[:30] == 0).all())
    k, v = (x[:70] for x in rows[0])
    o, A, e = _definition(q[30:], k, v, 1 / 8, 0)
    _check(out[30:].unflatten(1, (4, 64)), o, A, e, float(v.double().abs().max()), 70, F16, "short")


def test_paged_attention_rows_past_max_new_are_left(dev):
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 128, 4, 2, 16, [100, 20], [60, 1], seed=3)
    ref = serve.paged_attention(q, kc, vc, off, kvl, table, 60).clone()
    for most in (1, 2, 33):
        out = torch.full_like(ref, 7.0)
        serve.paged_attention(q, kc, vc, off, kvl, table, most, out=out)
        torch.cuda.synchronize()
        assert bool((out[most:60] == 7).all())
        err = (out[[*range(most), 60]].double() - ref[[*range(most), 60]].double()).abs().max()
        assert float(err) <= 4 * 2.0 ** -11 * 5


@pytest.mark.parametrize("new", [[1] * 6, [30, 1, 1, 200, 0, 2]])
def test_paged_attention_captured(dev, new):
    """A captured call replays with other lengths, tables and inputs; the scratch is the caller's, one per graph."""
    from llmr_amd import serve
    past = [100, 7, 900, 333, 64, 15]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, 128, 8, 2, 16, past, new, 4, seed=4)
    outs = [torch.full((q.shape[0], 1024), 7.0, dtype=BF16, device=dev) for _ in range(2)]
    scr = [serve.paged_attention_scratch(q, kc, table, max(new)) for _ in range(2)]
    graphs = [_capture(lambda o=o, s=s: serve.paged_attention(q, kc, vc, off, kvl, table, max(new), out=o, scratch=s))
              for o, s in zip(outs, scr)]
    short = torch.tensor([n for n in new], dtype=torch.int32, device=dev)
    full = kvl.clone()
    for lens in (full, short, full, torch.maximum(full - 50, short)):
        kvl.copy_(lens)
        for s in scr:
            s.fill_(255)
        for g in graphs:
            g.replay()
        eager = torch.full_like(outs[0], 7.0)
        serve.paged_attention(q, kc, vc, off, kvl, table, max(new), out=eager)
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, eager)
    kvl.copy_(full)
    graphs[0].replay()
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, outs[0], 1 / math.sqrt(128), "captured")


def test_paged_attention_two_at_once(dev):
    """Two calls on two streams, each with its own scratch, and repeated calls give the same bits."""
    from llmr_amd import serve
    cases = [_paged_case(dev, F16, 128, 8, 2, 16, [3000, 100], new, seed=i) for i, new in enumerate(([1, 1], [50, 3]))]
    refs = [serve.paged_attention(c[0], c[1], c[2], c[5], c[6], c[7], 50) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        outs = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                outs.append(serve.paged_attention(c[0], c[1], c[2], c[5], c[6], c[7], 50))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, refs))


def test_paged_attention_equals_prompt_attention(dev):
    """A whole prompt as one chunk over an empty cache is the prompt's own attention."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, 128, 8, 2, 32, [0, 0], [333, 90], seed=14)
    out = serve.paged_attention(q, kc, vc, off, kvl, table, 333)
    k, v = (torch.cat([r[i] for r in rows]) for i in range(2))
    ref = serve.prompt_attention(q, k, v, off)
    torch.cuda.synchronize()
    assert float((out.double() - ref.double()).abs().max()) <= 4 * 2.0 ** -8 * 5


def test_cache_past_32_bit_offsets(dev):
    """Pages whose byte and element offsets pass 2^32: a request whose pages lie at the end of a 9 GiB cache."""
    from llmr_amd import serve
    Hk, page, D = 8, 64, 128
    n_pages = (9 << 30) // (Hk * page * D * 2)
    kc = torch.zeros(n_pages, Hk, page, D, dtype=F16, device=dev)
    vc = torch.zeros_like(kc)
    g = torch.Generator(device=dev).manual_seed(1)
    for new in ([1], [70]):
        n = 300
        pages = torch.tensor([n_pages - 1, 0, n_pages - 2, n_pages // 2, n_pages - 7], device=dev)
        k, v = (torch.randn(n, Hk, D, generator=g, device=dev).half() for _ in range(2))
        j = torch.arange(n, device=dev)
        for c, x in ((kc, k), (vc, v)):
            c[pages[j // page], :, j % page] = x
        q = torch.randn(new[0], 16, D, generator=g, device=dev).half()
        out = serve.paged_attention(q, kc, vc, torch.tensor([0, new[0]], dtype=torch.int32, device=dev),
                                    torch.tensor([n], dtype=torch.int32, device=dev), pages.int()[None].contiguous(), new[0])
        torch.cuda.synchronize()
        _paged_check(q, [(k, v)], [0, new[0]], [n], out, 1 / math.sqrt(D), f"far pages, {new[0]} new")


# ---- refusals ---------------------------------------------------------------------


def test_prompt_attention_refuses(dev):
    from llmr_amd import capi, serve
    q, k, v, at, off = _prompt_case(dev, F16, 64, 4, 2, [50])
    ok = lambda **kw: serve.prompt_attention(**{**dict(q=q, k=k, v=v, seq_offsets=off), **kw})  # noqa: E731
    ok()
    for kw in (dict(q=q.float()), dict(k=k.bfloat16()), dict(v=v[:49]), dict(seq_offsets=off.long()),
               dict(q=q[:, :, :32]), dict(out=torch.empty(50, 255, dtype=F16, device=dev)),
               dict(out=torch.empty(50, 256, dtype=BF16, device=dev)), dict(seq_offsets=off.cpu()),
               dict(q=q[..., ::2]), dict(seq_offsets=off[:0])):
        with pytest.raises((ValueError, capi.LlmrError)):
            ok(**kw)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
               dict(k=torch.cat([k, k[:, :1]], 1), v=torch.cat([v, v[:, :1]], 1)),  # 4 heads over 3
               dict(q=torch.zeros(50, 4, 96, dtype=F16, device=dev), k=torch.zeros(50, 2, 96, dtype=F16, device=dev),
                    v=torch.zeros(50, 2, 96, dtype=F16, device=dev)),
               dict(q=torch.zeros(50 * 256 + 8, dtype=F16, device=dev)[4:4 + 50 * 256].view(50, 4, 64)),  # 8-byte aligned
               dict(out=torch.empty(50, 260, dtype=F16, device=dev)[:, :256])):  # rows 260 apart
        with pytest.raises(capi.LlmrError) as err:
            ok(**kw)
        assert err.value.code == capi.LLMR_ERR_INVALID_ARG
    assert ok(q=q[:0], k=k[:0], v=v[:0]).shape == (0, 256)
    assert serve.prompt_attention(q, k, v, off[:1], out=torch.zeros(50, 256, dtype=F16, device=dev)).abs().sum() == 0


def test_paged_attention_refuses(dev):
    from llmr_amd import capi, serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 64, 4, 2, 16, [50, 9], [3, 1], seed=1)
    base = dict(q=q, k_cache=kc, v_cache=vc, seq_offsets=off, kv_len=kvl, block_table=table, max_new=3)
    serve.paged_attention(**base)
    for kw in (dict(q=q.bfloat16()), dict(v_cache=vc[:-1]), dict(k_cache=kc.transpose(1, 2)), dict(seq_offsets=off[:2]),
               dict(kv_len=kvl.float()), dict(block_table=table.t()), dict(block_table=table.long()),
               dict(block_table=table[:1]), dict(q=q[:, :, :32])):
        with pytest.raises((ValueError, capi.LlmrError)):
            serve.paged_attention(**{**base, **kw})
    for kw in (dict(scale=0.0), dict(k_cache=torch.zeros(9, 2, 24, 64, dtype=F16, device=dev),
                                     v_cache=torch.zeros(9, 2, 24, 64, dtype=F16, device=dev)),
               dict(k_cache=torch.zeros(9, 3, 16, 64, dtype=F16, device=dev),
                    v_cache=torch.zeros(9, 3, 16, 64, dtype=F16, device=dev))):
        with pytest.raises(capi.LlmrError) as err:
            serve.paged_attention(**{**base, **kw})
        assert err.value.code == capi.LLMR_ERR_INVALID_ARG
    need = serve.paged_attention_scratch(q, kc, table, 3).numel()
    if need:
        with pytest.raises(capi.LlmrError, match="scratch"):
            serve.paged_attention(**base, scratch=torch.empty(need - 16, dtype=torch.uint8, device=dev))
        with pytest.raises(capi.LlmrError, match="scratch"):
            serve.paged_attention(**base, scratch=torch.empty(need + 4, dtype=torch.uint8, device=dev)[4:])
    assert serve.paged_attention(**{**base, "q": q[:0]}).shape == (0, 256)
    big = capi.MAX_SEQS + 1
    with pytest.raises(capi.LlmrError, match="n_seqs"):
        serve.paged_attention(q, kc, vc, torch.zeros(big + 1, dtype=torch.int32, device=dev),
                              torch.zeros(big, dtype=torch.int32, device=dev),
                              torch.zeros(big, 1, dtype=torch.int32, device=dev), 1)


# ---- what the chunk form counts -----------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,cols", [(128, 1), (64, 2), (128, 3), (64, 4), (64, 5), (128, 15)])
@pytest.mark.parametrize("new", [1, 12, 70])
def test_paged_attention_lengths_past_the_table(dev, dtype, D, cols, new):
    """Requests that outgrew their table (paged_plan's kv_len goes on): the keys are those of its pages and no other,
    at every remainder of a tile that the table may end at, in the form for few rows and in the one for chunks."""
    from llmr_amd import serve
    cap = 16 * cols
    q, kc, vc, rows, at, off, _, table, _ = _paged_case(dev, dtype, D, 4, 2, 16, [cap, cap, cap], [new] * 3, seed=cols)
    lens = [cap + 1000, cap + 20, 2 ** 31 - 1]
    out = serve.paged_attention(q, kc, vc, off, torch.tensor(lens, dtype=torch.int32, device=dev),
                                table[:, :cols].contiguous(), new)
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(at, at[1:])):
        k, v = (x[:cap] for x in rows[i])
        o, A, e = _definition(q[a:b], k, v, 1 / math.sqrt(D), lens[i] - new)
        _check(out[a:b].unflatten(1, (4, D)), o, A, e, float(v.double().abs().max()), cap, dtype,
               f"{cols} pages, length {lens[i]}, {new} new")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,new,hole", [(128, 64, 3), (64, 64, 0), (128, 64, 1), (64, 20, 0), (128, 150, 0), (64, 150, 4),
                                        (128, 150, 9), (64, 5, 0)])
def test_paged_attention_rows_of_a_chunk_around_a_missing_page(dev, dtype, D, new, hole):
    """A chunk over an empty cache with one page lacking (as paged_plan enters it): rows that see only the first few
    keys of a page are whole, before the hole and behind it."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, 4, 2, 16, [0], [new], seed=hole + new)
    table[0, hole] = -1
    out = torch.full((new, 4 * D), 7.0, dtype=dtype, device=dev)
    serve.paged_attention(q, kc, vc, off, kvl, table, new, out=out)
    torch.cuda.synchronize()
    k, v = rows[0]
    lo, hi = min(16 * hole, new), min(16 * hole + 16, new)
    seen = [torch.cat([x[:lo], x[hi:]]) for x in (k, v)]
    for a, b, kk, vv, first in ((0, lo, k[:lo], v[:lo], 0), (lo, hi, k[:lo], v[:lo], lo), (hi, new, *seen, lo)):
        if b > a and len(kk):
            o, A, e = _definition(q[a:b], kk, vv, 1 / math.sqrt(D), first)
            _check(out[a:b].unflatten(1, (4, D)), o, A, e, float(vv.double().abs().max()), new, dtype, f"rows {a} .. {b}")
        else:  # keys of the missing page alone
            assert bool((out[a:b] == 0).all()), (a, b)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[200], [90, 60, 150]], ids=["one", "packed"])
def test_prompt_attention_unseen_keys_change_no_bit(dev, dtype, D, lens):
    """A key far above the others raises the maximum of the rows that see it: the rows before it and other requests'
    in the same wave keep their bits."""
    from llmr_amd import serve
    q, k, v, at, off = _prompt_case(dev, dtype, D, 4, 2, lens, seed=31)
    clean = serve.prompt_attention(q, k, v, off)
    for row in (100, 137, at[-1] - 3):
        far = k.clone()
        far[row] *= 60
        out = serve.prompt_attention(q, far, v, off)
        torch.cuda.synchronize()
        end = next(e for e in at if e > row)
        assert not torch.equal(out[row:end], clean[row:end]), row
        assert torch.equal(out[:row], clean[:row]) and torch.equal(out[end:], clean[end:]), row


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [8, 24, 100])
def test_paged_attention_unseen_keys_change_no_bit(dev, dtype, D, new):
    """The same over a cache long enough that every wave takes several tiles."""
    from llmr_amd import serve
    past = 30000
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, 16, 8, 16, [past], [new], seed=32)
    clean = serve.paged_attention(q, kc, vc, off, kvl, table, new)
    for first in (new // 2, new - 2):
        page, at_page = int(table[0, (past + first) // 16]), (past + first) % 16
        far = kc.clone()
        far[page, :, at_page] *= 60
        out = serve.paged_attention(q, far, vc, off, kvl, table, new)
        torch.cuda.synchronize()
        assert not torch.equal(out[first:], clean[first:]), first
        assert torch.equal(out[:first], clean[:first]), first


@pytest.mark.parametrize("D,H,Hk", [(128, 8, 2), (64, 5, 1)])
def test_out_may_be_q(dev, D, H, Hk):
    """The queries' own rows as the output's, in every form: prompts, few rows, chunks, parts of several workgroups."""
    from llmr_amd import serve
    for lens in ([70, 0, 200], [900, 1100, 2000]):
        q, k, v, at, off = _prompt_case(dev, BF16, D, H, Hk, lens, 5, seed=41)
        ref = serve.prompt_attention(q, k, v, off, out=q.clone().flatten(1))
        serve.prompt_attention(q, k, v, off, out=q.flatten(1))
        torch.cuda.synchronize()
        assert torch.equal(q.flatten(1), ref)
    for past, new in (([9000, 3, 70], [1, 1, 1]), ([4000, 0], [6, 4]), ([5000, 100, 0], [300, 1, 70])):
        q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, D, H, Hk, 16, past, new, seed=42)
        ref = serve.paged_attention(q, kc, vc, off, kvl, table, max(new))
        serve.paged_attention(q, kc, vc, off, kvl, table, max(new), out=q.flatten(1))
        torch.cuda.synchronize()
        assert torch.equal(q.flatten(1), ref), new
