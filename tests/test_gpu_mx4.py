"""GPU key/value cache in 4 bits: the projection's rows into it (llmr_qkv_tokens_mx4) and back (llmr_mx4_rows), whole
numbers and exact values, compared for equality; attention over it (llmr_paged_attention_mx4) against its definition in
64 bits, element by element, with the bound that the attention over 16-bit caches has: a block's values are numbers of
either type, so nothing but the weights' and the result's rounding and f32 sums is between them; a run of them with the
8-bit linears around them."""
import math

import pytest
import torch
from test_gpu_paged import _rows_oracle, _tables
from test_gpu_seq_attn import _capture, _check, _definition, _near

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _pow2(e):
    """2^e in 64 bits for whole e (torch's own powers are not all exact on a device)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x):
    """f64 or f32 [.., D] -> codes [.., D / 2] and scales [.., D / 32] from the definition, block by block."""
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], 0.0, b)
    top = b.abs().amax(-1)
    # two significant bits: 1, 1.5, 2 times a power of two, ties up (a tie rounds 1.25 -> 1.5, 1.75 -> 2)
    e = torch.frexp(torch.where(top > 0, top, 2.0 ** -60))[1] - 1
    e = e + (top * _pow2(-e) >= 1.75).int() - 2
    e = e.clamp(-23, 13)
    a = (b.abs() * _pow2(-e)[..., None]).clamp(max=6.0)
    n = torch.tensor(NUMBERS, dtype=torch.float64, device=x.device)
    far = (a[..., None] - n).abs()
    near = far.amin(-1, keepdim=True)
    even = torch.tensor([0, 1, 0, 1, 0, 1, 0, 1], device=x.device)
    code = torch.where(far == near, even * 8, 100).add(torch.arange(8, device=x.device)).argmin(-1)  # nearest, ties to even
    code = (code + 8 * torch.signbit(b)).flatten(-2).to(torch.uint8)
    return code[..., ::2] | code[..., 1::2] << 4, torch.where(bad, 255, e + 127).to(torch.uint8)


def _decode(data, scales, dtype=torch.float64):
    n = torch.tensor(NUMBERS + [-x for x in NUMBERS], dtype=torch.float64, device=data.device)
    code = torch.stack([data & 15, data >> 4], -1).flatten(-2).long()
    s = torch.where(scales == 255, math.nan, _pow2(scales.int() - 127))
    return (n[code].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2).to(dtype)


def _caches(n_pages, Hk, page, D, dev, fill=0):
    from llmr_amd import serve
    c = [serve.Mx4Cache.empty(n_pages, Hk, page, D, dev) for _ in range(2)]
    for x in c:
        x.data.fill_(fill)
        x.scales.fill_(fill)
    return c


def _at(t, slots):
    """Rows [n, Hk, ..] of a cache's tensor [pages, Hk, page, ..]."""
    page = t.shape[2]
    return t[slots // page, :, slots % page]


# ---- rows into the cache ----------------------------------------------------------

ROWS = [(128, 4, 2, 1, 16, True, True, True), (64, 3, 1, 7, 32, True, True, False), (128, 32, 8, 64, 16, True, True, True),
        (64, 14, 2, 33, 64, False, True, True), (128, 5, 5, 100, 256, True, False, True), (64, 1, 1, 3, 16, False, False, False),
        (128, 30, 6, 21, 16, False, True, False), (64, 16, 4, 1030, 16, True, True, True), (128, 2, 1, 517, 128, True, True, False),
        (128, 4, 4, 2000, 16, True, True, True)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,H,Hk,T,page,norm,rope,halves", ROWS)
def test_qkv_tokens_mx4(dev, dtype, D, H, Hk, T, page, norm, rope, halves):
    """Queries as qkv_tokens' bit for bit, codes and scales as the definition's, nothing else touched."""
    from llmr_amd import serve
    g = torch.Generator(device=dev).manual_seed(T + H)
    width = (H + 2 * Hk) * D
    qkv = torch.randn(T, width + 12, generator=g, device=dev)[:, :width + 4] * 2
    qkv[:, ::7] *= torch.exp(3 * torch.randn(T, 1, generator=g, device=dev))
    qn, kn = (torch.rand(D, generator=g, device=dev) + 0.5 if norm else None for _ in range(2))
    tabs = _tables(dev, 900, D) if rope else None
    pos = torch.randint(0, 900, (T,), generator=g, device=dev)
    n_pages = -(-T // page) + 2
    slots = torch.randperm(n_pages * page, generator=g, device=dev)[:T].int()
    drop = torch.rand(T, generator=g, device=dev) < 0.2
    slots[drop] = torch.where(torch.rand(int(drop.sum()), generator=g, device=dev) < 0.5, -1, n_pages * page + 3).int()
    kc, vc = _caches(n_pages, Hk, page, D, dev, 77)
    q = torch.full((T, H + 1, D), 7.0, dtype=dtype, device=dev)
    kw = dict(positions=pos.int(), q_norm=qn, k_norm=kn, eps=1e-5, rope=tabs, halves=halves)
    serve.qkv_tokens_mx4(qkv, q[:, :H], kc, vc, slots, **kw)
    rows = [torch.empty(T, h, D, dtype=dtype, device=dev) for h in (H, Hk, Hk)]
    serve.qkv_tokens(qkv, *rows, **kw)
    torch.cuda.synchronize()
    assert torch.equal(q[:, :H], rows[0]) and bool((q[:, H] == 7).all())
    x = qkv[:, :width].reshape(T, H + 2 * Hk, D)
    live = ~drop
    at = slots[live].long()
    other = torch.ones(n_pages * page, dtype=torch.bool, device=dev)
    other[at] = False
    for c, y in ((kc, _rows_oracle(x[:, H:H + Hk], kn, 1e-5, tabs, pos, halves)[0]), (vc, x[:, H + Hk:].double())):
        for got, want in zip((c.data, c.scales), _encode(y)):
            if got.shape[-1] == D // 2:  # (the sign of a zero is not looked at)
                assert torch.equal(_decode(_at(got, at), _at(c.scales, at)), _decode(want[live], _encode(y)[1][live]))
            else:
                assert torch.equal(_at(got, at), want[live])
            assert bool((got.transpose(1, 2).flatten(0, 1)[other] == 77).all())


def test_blocks_at_the_borders(dev):
    """Values (no norm, no rotation) at, just under and just over every border between two numbers, for powers of two
    from the smallest to the largest and past both; blocks whose largest value is at a border between two powers."""
    from llmr_amd import serve
    D, Hk = 64, 3
    rows = []
    for e in (-140, -30, -24, -23, -22, -3, 0, 5, 12, 13, 14, 40, 120):
        for top in (6.0, 4.0, 3.5, 3.4999998, 3.5000005, 5.0, 6.9999995):
            m = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 3.0], dtype=torch.float32)
            m = torch.cat([m, torch.nextafter(m, torch.zeros(())), torch.nextafter(m, torch.full((), 9.0))])
            m = torch.minimum(m, torch.tensor(top))
            v = torch.zeros(32)
            v[:30], v[30], v[31] = m * (1 - 2 * (torch.arange(30) % 2)), top, -0.0
            rows.append(torch.ldexp(v.double(), torch.tensor(e)).float())
    x = torch.stack(rows)
    n = -(-len(x) // 6)
    x = torch.cat([x, torch.zeros(6 * n - len(x), 32)]).view(n, 3 * D).to(dev)
    qkv = torch.cat([torch.zeros(n, Hk * D, device=dev), x, x.flip(0)], 1).contiguous()
    kc, vc = _caches(-(-n // 16), Hk, 16, D, dev)
    q = torch.empty(n, Hk, D, dtype=F16, device=dev)
    slots = torch.arange(n, dtype=torch.int32, device=dev)
    for halves in (True, False):
        serve.qkv_tokens_mx4(qkv, q, kc, vc, slots, halves=halves)
        torch.cuda.synchronize()
        for c, y in ((kc, x), (vc, x.flip(0))):
            data, scales = _encode(y.view(n, Hk, D))
            assert torch.equal(_at(c.scales, slots.long()), scales)
            got = _decode(_at(c.data, slots.long()), scales)
            assert torch.equal(got, _decode(data, scales)), halves


def test_blocks_next_to_a_border_after_the_norm(dev):
    """Rows of one direction and many sizes: normed, all are next to the same borders, on either side by as little as
    64-bit rounding of the row; 32-bit norms would scatter them."""
    from llmr_amd import serve
    D, T = 128, 4096
    g = torch.Generator(device=dev).manual_seed(2)
    w = torch.ones(D, device=dev)
    base = torch.tensor(NUMBERS[1:], device=dev)[torch.randint(0, 7, (T, 3, D), generator=g, device=dev)]
    base = base + 0.25 * torch.randint(-1, 2, base.shape, generator=g, device=dev)  # numbers and halfway between some
    x = base * torch.exp(torch.randn(T, 3, 1, generator=g, device=dev))
    qkv = x.reshape(T, 3 * D).contiguous()
    kc, vc = _caches(T // 16, 1, 16, D, dev)
    q = torch.empty(T, 1, D, dtype=BF16, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    serve.qkv_tokens_mx4(qkv, q, kc, vc, slots, k_norm=w, eps=0.0)
    torch.cuda.synchronize()
    want = _rows_oracle(qkv.view(T, 3, D)[:, 1:2], w, 0.0, None, None, True)[0]
    data, scales = _encode(want)
    got = _decode(_at(kc.data, slots.long()), _at(kc.scales, slots.long()))
    # (a value that 64 bits put on a border has no side; there are next to none)
    assert torch.equal(_at(kc.scales, slots.long()), scales)
    assert int((got != _decode(data, scales)).sum()) <= 2


def test_blocks_of_no_number(dev):
    """An infinity or NaN makes its block NaN and no other; with a norm, its row."""
    from llmr_amd import serve
    D, T = 128, 8
    g = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn(T, 3 * D, generator=g, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)

    def caches(x, **kw):
        kc, vc = _caches(1, 1, 16, D, dev)
        q = torch.empty(T, 1, D, dtype=F16, device=dev)
        serve.qkv_tokens_mx4(x, q, kc, vc, slots, **kw)
        torch.cuda.synchronize()
        return [(_at(c.data, slots.long())[:, 0], _at(c.scales, slots.long())[:, 0]) for c in (kc, vc)]

    ref = caches(qkv)
    bad = qkv.clone()
    bad[1, D + 40], bad[2, 2 * D + 5], bad[3, 2 * D + 127], bad[4, D + 64] = math.nan, math.inf, -math.inf, -math.nan
    got = caches(bad)
    for (data, scales), (rd, rs), marks in zip(got, ref, ([(1, 1), (4, 2)], [(2, 0), (3, 3)])):
        keep = torch.ones(T, 4, dtype=torch.bool, device=dev)
        for r, b in marks:
            assert int(scales[r, b]) == 255 and bool((data[r, 16 * b:16 * b + 16] == 0).all())
            keep[r, b] = False
        assert torch.equal(scales[keep], rs[keep]) and torch.equal(data.view(T, 4, 16)[keep], rd.view(T, 4, 16)[keep])
    data, scales = caches(bad, k_norm=torch.ones(D, device=dev))[0]
    assert bool((scales[1] == 255).all())  # a NaN in the sum of squares
    zero = torch.zeros_like(qkv)
    for data, scales in caches(zero, k_norm=torch.ones(D, device=dev)):
        assert bool((data & 0x77 == 0).all()) and bool((scales == 104).all())


def test_positions_and_rows_of_no_slot(dev):
    """No positions: the row; positions outside the tables are taken at their ends, as qkv_tokens does."""
    from llmr_amd import serve
    D, T = 64, 40
    qkv = torch.randn(T, 3 * D, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    tabs = _tables(dev, T, D)

    def rows(pos):
        kc, vc = _caches(3, 1, 16, D, dev)
        q = torch.empty(T, 1, D, dtype=BF16, device=dev)
        serve.qkv_tokens_mx4(qkv, q, kc, vc, torch.arange(T, dtype=torch.int32, device=dev), positions=pos, rope=tabs)
        return q, kc.data, kc.scales, vc.data

    i = torch.arange(T, device=dev, dtype=torch.int32)
    assert all(torch.equal(a, b) for a, b in zip(rows(None), rows(i)))
    far = i.clone()
    far[3], far[4], far[5] = -7, 2 ** 31 - 1, T
    near = i.clone()
    near[3], near[4], near[5] = 0, T - 1, T - 1
    assert all(torch.equal(a, b) for a, b in zip(rows(far), rows(near)))


# ---- rows back --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,Hk,page,n", [(128, 8, 16, 300), (64, 3, 256, 77), (128, 1, 64, 1), (64, 12, 32, 2000)])
def test_mx4_rows(dev, dtype, D, Hk, page, n):
    """Every byte with every scale that the cache has, in any order and the same one twice; rows of no slot stay."""
    from llmr_amd import serve
    g = torch.Generator(device=dev).manual_seed(n)
    n_pages = 40 if page < 64 else 5
    kc, vc = _caches(n_pages, Hk, page, D, dev)
    for c in (kc, vc):
        c.data.copy_(torch.randint(0, 256, c.data.shape, generator=g, device=dev))
        c.scales.copy_(torch.randint(104, 141, c.scales.shape, generator=g, device=dev))
        c.scales[torch.rand(c.scales.shape, generator=g, device=dev) < 0.02] = 255
    slots = torch.randint(0, n_pages * page, (n,), generator=g, device=dev, dtype=torch.int32)
    if n > 1:
        slots[1], slots[n // 2], slots[n - 1] = -1, n_pages * page, slots[0]
    wide = [torch.full((n, Hk + 1, D), 7.0, dtype=dtype, device=dev) for _ in range(2)]
    ko, vo = (x[:, :Hk] for x in wide)
    serve.mx4_rows(kc, vc, slots, ko, vo)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < n_pages * page)
    for c, o, x in ((kc, ko, wide[0]), (vc, vo, wide[1])):
        at = slots[live].long()
        want = _decode(_at(c.data, at), _at(c.scales, at), dtype)
        assert torch.equal(o[live].isnan(), want.isnan()) and torch.equal(o[live].nan_to_num(0.0), want.nan_to_num(0.0))
        assert bool((o[~live] == 7).all()) and bool((x[:, Hk] == 7).all())


def test_more_rows_than_a_launch_has_along_x(dev):
    """2^23 + 37 rows into a cache and back: the first, those around the border and the last as a call of their own."""
    from llmr_amd import serve
    T, D, page = (1 << 23) + 37, 64, 256
    g = torch.Generator(device=dev).manual_seed(9)
    n_pages = -(-T // page)
    qkv = torch.empty(T, 3 * D, device=dev).normal_(generator=g)
    q = torch.zeros(T, 1, D, dtype=F16, device=dev)
    kc, vc = _caches(n_pages, 1, page, D, dev, 77)
    slots = torch.arange(T, dtype=torch.int32, device=dev).flip(0)
    slots[5::1000] = -1
    serve.qkv_tokens_mx4(qkv, q, kc, vc, slots)
    ko, vo = (torch.full((T, 1, D), 7.0, dtype=F16, device=dev) for _ in range(2))
    serve.mx4_rows(kc, vc, slots, ko, vo)
    torch.cuda.synchronize()
    for a, b in ((0, 2000), ((1 << 23) - 1000, T)):
        live = slots[a:b] >= 0
        x = qkv[a:b].view(-1, 3, D)
        assert torch.equal(q[a:b, 0], x[:, 0].half())
        for got, y in ((ko, x[:, 1:2]), (vo, x[:, 2:])):
            want = _decode(*_encode(y))
            assert torch.equal(got[a:b][live].double(), want[live]) and bool((got[a:b][~live] == 7).all())
    unused = torch.ones(n_pages * page, dtype=torch.bool, device=dev)
    unused[slots[slots >= 0].long()] = False
    assert bool((kc.data.view(-1, D // 2)[unused] == 77).all()) and bool((vc.scales.view(-1, 2)[unused] == 77).all())


# ---- attention over the pages -------------------------------------------------------


def _paged_case(dev, dtype, D, H, Hk, page, past, new, pad=0, seed=0, spare=3, poison=True, qstd=1.5):
    """Contiguous 64-bit rows of every request (the oracle's), the same as blocks in shuffled pages; what no request
    holds is NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    kv = [p + n for p, n in zip(past, new)]
    need = [-(-n // page) for n in kv]
    n_pages = sum(need) + spare
    caches = _caches(n_pages, Hk, page, D, dev, 255 if poison else 0)
    order = torch.randperm(n_pages, generator=g, device=dev)
    table = torch.full((len(kv), max(max(need), 1) + 1), -1, dtype=torch.int32, device=dev)
    rows, used = [], 0
    for i, n in enumerate(kv):
        blocks = [_encode(torch.randn(n, Hk, D, generator=g, device=dev)) for _ in range(2)]
        rows.append([_decode(*b) for b in blocks])
        pages = order[used:used + need[i]]
        used += need[i]
        table[i, :need[i]] = pages.int()
        j = torch.arange(n, device=dev)
        for c, (data, scales) in zip(caches, blocks):
            c.data[pages[j // page], :, j % page] = data
            c.scales[pages[j // page], :, j % page] = scales
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
            _check(out[a:b].unflatten(1, (H, D)), o, A, e, float(v.abs().max()), kv[i], q.dtype,
                   f"{what} request {i} ({b - a} of {kv[i]})")


def _beside(out, ref, v, what):
    """Two results of one definition in out's type (_near's bound)."""
    _near(out, ref, v.to(out.dtype), what)


# (D, H, Hk, page, past, new, pad): single tokens from one cached key to long contexts; pages that end inside a tile;
# requests with nothing new; small chunks of one tile with their group; chunks over several tiles; all at once
PAGED = [(128, 4, 2, 16, [0], [1], 0), (128, 32, 8, 16, [1100], [1], 0), (64, 8, 2, 32, [15, 16, 17, 0, 300], [1] * 5, 3),
         (128, 30, 6, 16, [5, 1000, 63, 64, 127, 128, 2047], [1] * 7, 0), (128, 8, 8, 64, [64, 63, 700], [1, 1, 1], 0),
         (64, 16, 1, 256, [3000, 1, 255, 256], [1] * 4, 0), (128, 4, 4, 128, [20000], [1], 0),
         (128, 8, 2, 16, [50, 0, 200, 7], [4, 4, 2, 0], 0), (64, 14, 2, 16, [33, 900], [2, 5], 1),
         (128, 32, 8, 32, [500], [64], 0), (128, 12, 2, 64, [0], [130], 0), (64, 5, 1, 16, [77, 0], [300, 1], 5),
         (128, 8, 2, 16, [40, 3000, 0, 1000, 9], [1, 129, 257, 0, 33], 6), (64, 3, 3, 128, [100, 600], [200, 100], 0),
         (128, 16, 1, 16, [1500], [17], 0), (128, 24, 8, 16, [0] * 12 + [400] * 12, [1, 20] * 12, 0),
         (128, 8, 1, 16, [70, 70], [9, 40], 0), (128, 2, 2, 16, [300, 2], [31, 65], 0), (64, 28, 4, 32, [9000, 40], [4, 2], 0),
         (64, 48, 1, 16, [5000, 3], [1, 1], 0), (128, 64, 1, 16, [5000, 3, 130], [1, 1, 1], 2), (128, 40, 1, 16, [700], [2], 0)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,H,Hk,page,past,new,pad", PAGED, ids=lambda x: str(x).replace(" ", "")[:24])
def test_paged_attention_mx4(dev, dtype, D, H, Hk, page, past, new, pad):
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, H, Hk, page, past, new, pad, seed=sum(past) + H)
    out = torch.full((q.shape[0], H * D), 7.0, dtype=dtype, device=dev)
    assert serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new), out=out) is out
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(D), f"D={D} H={H}/{Hk} page={page}")
    assert bool((out[at[-1]:] == 7).all())
    # a larger bound on the new tokens, another scratch and a wider table change the split at most
    wide = torch.full((table.shape[0], table.shape[1] + 700), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    out2 = serve.paged_attention_mx4(q, kc, vc, off, kvl, wide, q.shape[0])
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out2, 1 / math.sqrt(D), "wide")


# more requests than a wave's lanes, some of them with nothing new, at the ends too
MANY = [(128, 8, 2, [0, 1, 1, 0, 1] * 40), (64, 8, 2, [0, 5, 1, 8] * 30 + [0] * 70 + [3]), (128, 8, 2, [16, 0, 9, 1] * 20),
        (64, 4, 1, [0] * 65 + [70, 1, 0, 300, 2] * 14 + [0] * 3)]


@pytest.mark.parametrize("D,H,Hk,new", MANY, ids=["1", "8", "16", "300"])
def test_many_requests(dev, D, H, Hk, new):
    from llmr_amd import serve
    past = [(37 * i * i) % 211 for i in range(len(new))]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, D, H, Hk, 16, past, new, 2, seed=len(new))
    out = torch.full((q.shape[0], H * D), 7.0, dtype=BF16, device=dev)
    serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new), out=out)
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(D), f"{len(new)} requests")
    assert bool((out[at[-1]:] == 7).all())


@pytest.mark.parametrize("hole", [None, 1000, 68000], ids=["whole", "hole-early", "hole-late"])
@pytest.mark.parametrize("new", [2, 2048])
def test_long_tables(dev, new, hole):
    """New tokens behind 70000 keys: a workgroup's share is more tiles than it keeps pages of, a wave's more units than
    it keeps pages of. Keys on no page are nobody's; the first and last rows of the chunk are looked at."""
    from llmr_amd import serve
    D, H, Hk, page, past = 64, 32, 8, 16, 70000
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, D, H, Hk, page, [past], [new], seed=5)
    k, v = rows[0]
    if hole is not None:
        table[0, hole // page] = -1
        lo = hole // page * page
        k, v = (torch.cat([t[:lo], t[lo + page:]]) for t in (k, v))
        past -= page
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
    torch.cuda.synchronize()
    vm = float(v.abs().max())
    for a, b in ((0, min(20, new)), (max(0, new - 20), new)):
        o, A, e = _definition(q[a:b], k, v, 1 / math.sqrt(D), past + a)
        _check(out[a:b].unflatten(1, (H, D)), o, A, e, vm, past + b, F16, f"rows {a} .. {b}")


@pytest.mark.parametrize("qstd", [30.0, 0.01])
@pytest.mark.parametrize("new", [[1, 1], [5, 3], [40, 3]])
def test_score_ranges(dev, qstd, new):
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 128, 8, 2, 16, [900, 333], new, seed=2, qstd=qstd)
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new))
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(128), f"qstd {qstd}")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("e", [-23, -20, 10, 13])
@pytest.mark.parametrize("new", [1, 3, 50])
def test_powers_of_two_at_the_ends(dev, dtype, e, new):
    """Blocks with the smallest and largest powers: fp16's subnormals and its largest values, in keys or in values."""
    from llmr_amd import serve
    for where in (0, 1):
        q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, 64, 4, 2, 16, [200], [new], seed=e + 30, poison=False)
        c = (kc, vc)[where]
        c.scales.fill_(e + 127)
        j = torch.arange(kv[0], device=dev)
        pages = table[0].long()
        k, v = (_decode(x.data[pages[j // 16], :, j % 16], x.scales[pages[j // 16], :, j % 16]) for x in (kc, vc))
        scale = 2.0 ** -(e + 3) if where == 0 else 0.125
        out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new, scale=scale)
        torch.cuda.synchronize()
        o, A, err = _definition(q[:new], k, v, scale, 200)
        _check(out[:new].unflatten(1, (4, 64)), o, A, err, float(v.abs().max()), kv[0], dtype, f"2^{e} in {'kv'[where]}")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,row", [(3, 98), (3, 99), (100, 150), (100, 190), (40, 101), (40, 120)])
def test_unseen_values_do_not_matter(dev, dtype, new, row):
    """A NaN block in the key or value of a new token reaches the rows that see it and no other."""
    from llmr_amd import serve
    past = 97 if new == 3 else 96
    for where in (0, 1):
        print(f"NaN in {'kv'[where]}, {new} new", flush=True)
        q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, 128, 8, 2, 16, [past, 60], [new, 1], seed=5)
        clean = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new).clone()
        page = int(table[0, row // 16])
        (kc, vc)[where].scales[page, 1, row % 16, 2] = 255
        rows[0][where][row, 1, 64:96] = math.nan
        out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
        torch.cuda.synchronize()
        o, c = (t.unflatten(1, (8, 128)) for t in (out, clean))
        first = row - past  # the new token it belongs to
        keep = torch.ones(new + 1, dtype=torch.bool, device=dev)
        keep[first:new] = False
        assert torch.equal(o[keep], c[keep]) and torch.equal(o[:, :4], c[:, :4])
        ref = _definition(q[:new], *rows[0], 1 / math.sqrt(128), past)[0]
        assert torch.equal(o[:new].double().isnan(), ref.isnan()), where


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 5, 20, 90])
def test_what_unused_slots_hold_does_not_matter(dev, dtype, D, new):
    """Slots behind a request's last key, and pages that nobody holds, with any bytes: no bit of the result changes."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, 8, 2, 64, [70, 3, 500], [new, 1, 1], seed=9, poison=False)
    ref = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
    used = torch.zeros(kc.data.shape[0], 64, dtype=torch.bool, device=dev)
    for i, n in enumerate(kv):
        j = torch.arange(n, device=dev)
        used[table[i].long()[j // 64], j % 64] = True
    free = ~used[:, None, :, None]
    for power, code in ((255, 0xff), (254, 0x77), (200, 0xf7), (0, 0x11)):
        c = [serve.Mx4Cache(torch.where(free, code, x.data).to(torch.uint8), torch.where(free, power, x.scales).to(torch.uint8))
             for x in (kc, vc)]
        out = serve.paged_attention_mx4(q, *c, off, kvl, table, new)
        torch.cuda.synchronize()
        assert torch.equal(out, ref), power


def test_a_cache_of_no_pages(dev):
    """Every key is on a page that there is not: rows are 0."""
    from llmr_amd import serve
    for D, new in ((128, 1), (64, 3), (128, 40)):
        kc, vc = _caches(0, 2, 16, D, dev)
        q = torch.randn(new, 8, D, device=dev).half()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        for table in (torch.zeros(1, 9, dtype=torch.int32, device=dev), torch.zeros(1, 0, dtype=torch.int32, device=dev)):
            out = serve.paged_attention_mx4(q, kc, vc, i32([0, new]), i32([100]), table, new)
            torch.cuda.synchronize()
            assert bool((out == 0).all())
    serve.qkv_tokens_mx4(torch.randn(3, 6 * 64, device=dev), torch.empty(3, 2, 64, dtype=F16, device=dev),
                         *(serve.Mx4Cache(torch.empty(1, 2, 16, 32, dtype=torch.uint8, device=dev)[:0],
                                          torch.empty(1, 2, 16, 2, dtype=torch.uint8, device=dev)[:0]) for _ in range(2)),
                         torch.tensor([0, -1, 5], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 8, 24, 100])
def test_nan_values_that_rows_see(dev, D, new):
    """NaN blocks deep in the context, which every row sees, and next to the last keys, in pages of their own."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, D, 8, 2, 16, [3000], [new], seed=6)
    for row, head, block in ((17, 0, 0), (2999, 1, D // 32 - 1), (3000 + new - 1, 0, 1)):
        vc.scales[int(table[0, row // 16]), head, row % 16, block] = 255
        rows[0][1][row, head, 32 * block:32 * block + 32] = math.nan
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
    torch.cuda.synchronize()
    k, v = rows[0]
    want = _definition(q, k, v, 1 / math.sqrt(D), 3000)[0]
    assert torch.equal(out.unflatten(1, (8, D)).isnan(), want.isnan())
    o, A, e = _definition(q, k, v.nan_to_num(0.0), 1 / math.sqrt(D), 3000)
    got = torch.where(want.isnan(), o, out.unflatten(1, (8, D)).double())
    _check(got, o, A, e, float(v.nan_to_num(0.0).abs().max()), kv[0], BF16, "beside NaN")


# Powers above those that qkv_tokens_mx4 writes (a cache filled by other means): finite in bf16; in fp16 2^14 times 4
# and 6, and 2^16 times anything but 0, are infinite.
FAR_POWERS = [141, 143, 160, 200, 230, 255]


def _check_infinite(got, out, A, e, v, keys, dtype, what):
    """_check where values are infinite: those sums are infinite or NaN in the same places."""
    got = got.double()
    inf = out.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], out[inf]), (what, "infinities in other places")
    zero = torch.zeros_like(out)
    _check(torch.where(inf, zero, got), torch.where(inf, zero, out), torch.where(A.isfinite(), A, zero), e,
           float(v.nan_to_num(0, 0, 0).abs().max()), keys, dtype, what)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 5, 20, 100])
@pytest.mark.parametrize("power", FAR_POWERS)
def test_values_of_powers_past_the_writers(dev, dtype, D, new, power):
    """A value block of such a power is the same numbers wherever it lies: deep in the context, next to the last keys, in
    a new token that some rows see and others do not, and by itself in a context of few keys."""
    from llmr_amd import serve
    for past, places in ((3000, (17, 2999, 3000 + new - 1)), (3000, (1234,)), (3000, (3000 + new // 2,)), (4, (2,))):
        q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, 8, 2, 16, [past], [new], seed=power + new)
        clean = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new).clone()
        v = rows[0][1]
        for i, row in enumerate(places):
            head, block = i % 2, (i + 1) % (D // 32)
            page = int(table[0, row // 16])
            vc.scales[page, head, row % 16, block] = power
            v[row, head] = _decode(vc.data[page, head, row % 16], vc.scales[page, head, row % 16])
        v = v.to(dtype).double()  # the values that mx4_rows reads
        out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
        torch.cuda.synchronize()
        o, A, e = _definition(q, rows[0][0], v, 1 / math.sqrt(D), past)
        _check_infinite(out.unflatten(1, (8, D)), o, A, e, v, kv[0], dtype, f"2^{power - 127} at {places} of {kv[0]}")
        unseen = max(0, min(places) - past)  # rows before the first of them
        assert torch.equal(out[:unseen], clean[:unseen])


@pytest.mark.parametrize("e", [14, 40, 90])
@pytest.mark.parametrize("new", [1, 3, 50])
def test_keys_of_powers_past_the_writers(dev, e, new):
    """Keys of larger powers in bf16, against a scale that leaves their scores as they are."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, 64, 4, 2, 16, [200], [new], seed=e, poison=False)
    kc.scales.fill_(e + 127)
    j = torch.arange(kv[0], device=dev)
    pages = table[0].long()
    k = _decode(kc.data[pages[j // 16], :, j % 16], kc.scales[pages[j // 16], :, j % 16])
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new, scale=2.0 ** -(e + 3))
    torch.cuda.synchronize()
    v = rows[0][1]
    o, A, err = _definition(q[:new], k, v, 2.0 ** -(e + 3), 200)
    _check(out[:new].unflatten(1, (4, 64)), o, A, err, float(v.abs().max()), kv[0], BF16, f"2^{e}")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_mx4_rows_of_every_power(dev, dtype):
    """Each code under each of the 256 powers: its value, rounded to the type (infinite past it)."""
    from llmr_amd import serve
    kc, vc = _caches(16, 1, 16, 64, dev)
    code = torch.arange(64, device=dev) % 16
    for c in (kc, vc):
        c.data[:] = (code[::2] | code[1::2] << 4).to(torch.uint8)
        c.scales[:] = torch.arange(256, device=dev).view(16, 1, 16, 1).to(torch.uint8)
    ko, vo = (torch.empty(256, 1, 64, dtype=dtype, device=dev) for _ in range(2))
    serve.mx4_rows(kc, vc, torch.arange(256, dtype=torch.int32, device=dev), ko, vo)
    torch.cuda.synchronize()
    n = torch.tensor(NUMBERS + [-x for x in NUMBERS], dtype=torch.float64)
    s = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], dtype=torch.float64)
    want = (s[:, None] * n).to(dtype)[:, code.cpu()]
    for got in (ko[:, 0].cpu(), vo[:, 0].cpu()):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0, math.inf, -math.inf), want.nan_to_num(0.0, math.inf, -math.inf))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [20, 1, 70, 2]])
def test_bad_tables_and_lengths(dev, new):
    """Pages outside the cache are seen by nobody, lengths past the table end with it, a row that sees no key is
    0, and requests beside them keep their results."""
    from llmr_amd import serve
    past = [200, 100, 90, 50]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, 128, 4, 2, 16, past, new, seed=7)
    ref = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new)).clone()
    cols = table.shape[1]
    n_pages = kc.data.shape[0]
    bad = table.clone()
    bad[0, 3], bad[0, 5], bad[0, 6] = -1, n_pages, 2 ** 31 - 1
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, bad, max(new))
    torch.cuda.synchronize()
    assert torch.equal(out[at[1]:], ref[at[1]:])
    seen = torch.ones(kv[0], dtype=torch.bool, device=dev)
    for c in (3, 5, 6):
        seen[16 * c:16 * c + 16] = False
    k, v = (x[seen] for x in rows[0])
    n = at[1]
    o, A, e = _definition(q[:n], k, v, 1 / math.sqrt(128), int(seen.sum()) - n)
    _check(out[:n].unflatten(1, (4, 128)), o, A, e, float(v.abs().max()), kv[0], BF16, "holes")
    bad = torch.full_like(table, -1)
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, bad, max(new))
    torch.cuda.synchronize()
    assert bool((out[:at[-1]] == 0).all())
    for lens in ([0, 0, 0, 0], [-5, -1, -2 ** 31, -100]):  # shorter than the new tokens: no key for the first ones
        out = serve.paged_attention_mx4(q, kc, vc, off, torch.tensor(lens, dtype=torch.int32, device=dev), table, max(new))
        torch.cuda.synchronize()
        assert bool((out[:at[-1]] == 0).all()), lens
    big = kvl.clone()
    big[1], big[2] = 2 ** 31 - 1, 16 * cols + 1000  # the table ends first; what is past it nobody sees
    filled = table.clone()
    filled[filled < 0] = int(table[0, 0])
    for c in (kc, vc):
        c.scales[c.scales == 255] = 104
    out = serve.paged_attention_mx4(q, kc, vc, off, big, filled, max(new))
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out[:at[-1]]).all())
    for i in (0, 3):
        _beside(out[at[i]:at[i + 1]], ref[at[i]:at[i + 1]], rows[i][1], i)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,cols", [(128, 1), (64, 2), (128, 3), (64, 5), (128, 15)])
@pytest.mark.parametrize("new", [1, 12, 70])
def test_lengths_past_the_table(dev, dtype, D, cols, new):
    """Requests that outgrew their table: the keys are those of its pages and no other, at every remainder of a tile
    that the table may end at, in the form for few rows and in the one for chunks."""
    from llmr_amd import serve
    cap = 16 * cols
    q, kc, vc, rows, at, off, _, table, _ = _paged_case(dev, dtype, D, 4, 2, 16, [cap, cap, cap], [new] * 3, seed=cols)
    lens = [cap + 1000, cap + 20, 2 ** 31 - 1]
    out = serve.paged_attention_mx4(q, kc, vc, off, torch.tensor(lens, dtype=torch.int32, device=dev),
                                    table[:, :cols].contiguous(), new)
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(at, at[1:])):
        k, v = (x[:cap] for x in rows[i])
        o, A, e = _definition(q[a:b], k, v, 1 / math.sqrt(D), lens[i] - new)
        _check(out[a:b].unflatten(1, (4, D)), o, A, e, float(v.abs().max()), cap, dtype,
               f"{cols} pages, length {lens[i]}, {new} new")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,new,hole", [(128, 64, 3), (64, 64, 0), (128, 64, 1), (64, 20, 0), (128, 150, 0), (64, 150, 4),
                                        (128, 150, 9), (64, 5, 0)])
def test_rows_of_a_chunk_around_a_missing_page(dev, dtype, D, new, hole):
    """A chunk over an empty cache with one page lacking: rows that see only the first few keys of a page are whole,
    before the hole and behind it."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, 4, 2, 16, [0], [new], seed=hole + new)
    table[0, hole] = -1
    out = torch.full((new, 4 * D), 7.0, dtype=dtype, device=dev)
    serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new, out=out)
    torch.cuda.synchronize()
    k, v = rows[0]
    lo, hi = min(16 * hole, new), min(16 * hole + 16, new)
    seen = [torch.cat([x[:lo], x[hi:]]) for x in (k, v)]
    for a, b, kk, vv, first in ((0, lo, k[:lo], v[:lo], 0), (lo, hi, k[:lo], v[:lo], lo), (hi, new, *seen, lo)):
        if b > a and len(kk):
            o, A, e = _definition(q[a:b], kk, vv, 1 / math.sqrt(D), first)
            _check(out[a:b].unflatten(1, (4, D)), o, A, e, float(vv.abs().max()), new, dtype, f"rows {a} .. {b}")
        else:  # keys of the missing page alone
            assert bool((out[a:b] == 0).all()), (a, b)


def test_more_new_than_cached_and_rows_past_max_new(dev):
    """kv_len under the request's rows: the first rows see nothing and are 0, the last see the cached keys. Rows past
    max_new are left."""
    from llmr_amd import serve
    for n, have in ((100, 70), (9, 6)):
        q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 64, 4, 1, 16, [0], [n], seed=3)
        kvl.fill_(have)
        out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, n)
        torch.cuda.synchronize()
        assert bool((out[:n - have] == 0).all())
        k, v = (x[:have] for x in rows[0])
        o, A, e = _definition(q[n - have:], k, v, 1 / 8, 0)
        _check(out[n - have:].unflatten(1, (4, 64)), o, A, e, float(v.abs().max()), have, F16, "short")
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 128, 4, 2, 16, [100, 20], [60, 1], seed=3)
    for most in (1, 2, 33):
        out = torch.full((61, 512), 7.0, dtype=F16, device=dev)
        serve.paged_attention_mx4(q, kc, vc, off, kvl, table, most, out=out)
        torch.cuda.synchronize()
        assert bool((out[most:60] == 7).all())
        o, A, e = _definition(q[:most], *rows[0], 1 / math.sqrt(128), 100)
        _check(out[:most].unflatten(1, (4, 128)), o, A, e, float(rows[0][1].abs().max()), 160, F16, f"first {most}")


@pytest.mark.parametrize("new", [[1] * 6, [30, 1, 1, 200, 0, 2], [4, 1, 0, 2, 3, 4]])
def test_captured(dev, new):
    """A captured call replays with other lengths, tables and inputs; the scratch is the caller's, one per graph."""
    from llmr_amd import serve
    past = [100, 7, 900, 333, 64, 15]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, 128, 8, 2, 16, past, new, 4, seed=4)
    outs = [torch.full((q.shape[0], 1024), 7.0, dtype=BF16, device=dev) for _ in range(2)]
    scr = [serve.paged_attention_mx4_scratch(q, kc, table, max(new)) for _ in range(2)]
    graphs = [_capture(lambda o=o, s=s: serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new), out=o, scratch=s))
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
        serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new), out=eager)
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, eager)
    kvl.copy_(full)
    graphs[0].replay()
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, outs[0], 1 / math.sqrt(128), "captured")


def test_two_at_once(dev):
    """Calls on several streams, each with its own scratch, and repeated calls give the same bits."""
    from llmr_amd import serve
    cases = [_paged_case(dev, F16, 128, 8, 2, 16, [3000, 100], new, seed=i)
             for i, new in enumerate(([1, 1], [50, 3], [4, 8]))]
    call = lambda c, n: serve.paged_attention_mx4(c[0], c[1], c[2], c[5], c[6], c[7], n)  # noqa: E731
    refs = [call(c, n) for c, n in zip(cases, (1, 50, 8))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        outs = []
        for s, c, n in zip(streams, cases, (1, 50, 8)):
            with torch.cuda.stream(s):
                outs.append(call(c, n))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, refs))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 1, 7], [60, 1, 300]])
def test_equals_attention_over_a_16_bit_cache(dev, dtype, new):
    """The same values in a 16-bit cache: both are within the same bound of one definition."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, 128, 8, 2, 32, [2000, 77, 0], new, seed=14, poison=False)
    wide = [_decode(c.data, c.scales, dtype) for c in (kc, vc)]
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new))
    ref = serve.paged_attention(q, *wide, off, kvl, table, max(new))
    torch.cuda.synchronize()
    _beside(out, ref, wide[1], new)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [8, 24, 100])
def test_unseen_keys_change_no_bit(dev, dtype, D, new):
    """A key far above the others raises the maximum of the rows that see it: the rows before it keep their bits."""
    from llmr_amd import serve
    past = 30000
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, D, 16, 8, 16, [past], [new], seed=32)
    clean = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
    for first in (new // 2, new - 2):
        page, at_page = int(table[0, (past + first) // 16]), (past + first) % 16
        far = serve.Mx4Cache(kc.data, kc.scales.clone())
        far.scales[page, :, at_page] += 6
        out = serve.paged_attention_mx4(q, far, vc, off, kvl, table, new)
        torch.cuda.synchronize()
        assert not torch.equal(out[first:], clean[first:]), first
        assert torch.equal(out[:first], clean[:first]), first


@pytest.mark.parametrize("D,H,Hk", [(128, 8, 2), (64, 6, 3)])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 1, 2], [70, 1, 33]])
def test_strided_rows_and_shared_pages(dev, D, H, Hk, new):
    """Queries among other columns and a result into columns of a wider buffer; requests with the same first pages."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, D, H, Hk, 16, [900, 900, 333], new, 3, seed=21)
    table[1, :40] = table[0, :40]
    for i in (0, 1):
        rows[1][i][:640] = rows[0][i][:640]
    wide = torch.full((q.shape[0], H + 3, D), math.nan, dtype=F16, device=dev)
    wide[:, 1:H + 1] = q
    buf = torch.full((q.shape[0], H * D + 24), 7.0, dtype=F16, device=dev)
    out = buf[:, 8:8 + H * D]
    assert serve.paged_attention_mx4(wide[:, 1:H + 1], kc, vc, off, kvl, table, max(new), out=out) is out
    ref = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new))
    torch.cuda.synchronize()
    _paged_check(q, rows, at, kv, out, 1 / math.sqrt(D), "strided")
    assert torch.equal(out[:at[-1]], ref[:at[-1]])
    out[:at[-1]] = 7.0
    assert bool((buf == 7).all())


@pytest.mark.parametrize("new", [1, 3])
def test_as_many_requests_as_a_call_takes(dev, new):
    from llmr_amd import capi, serve
    n, D, H, Hk = capi.MAX_SEQS, 64, 4, 1
    past = [(31 * i) % 90 for i in range(n)]
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, D, H, Hk, 16, past, [new] * n, seed=n)
    out = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, new)
    torch.cuda.synchronize()
    for i in list(range(0, n, 257)) + [n - 1]:
        o, A, e = _definition(q[at[i]:at[i + 1]], *rows[i], 1 / math.sqrt(D), past[i])
        _check(out[at[i]:at[i + 1]].unflatten(1, (H, D)), o, A, e, float(rows[i][1].abs().max()), kv[i], BF16, f"request {i}")
    # the same rows a request at a time lie within the bound of one definition
    for i in (0, 1000, n - 1):
        one = serve.paged_attention_mx4(q[at[i]:at[i + 1]].contiguous(), kc, vc, off[:2].contiguous(), kvl[i:i + 1].contiguous(),
                                        table[i:i + 1].contiguous(), new)
        torch.cuda.synchronize()
        _beside(out[at[i]:at[i + 1]], one, rows[i][1], i)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new", [[1, 1], [5, 2], [60, 30]])
def test_a_query_of_no_number(dev, dtype, new):
    """An infinity or NaN in one head of one row makes that row NaN and changes no bit of the others."""
    from llmr_amd import serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, dtype, 128, 8, 2, 16, [3000, 40], new, seed=3)
    ref = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new)).view(-1, 8, 128)
    row = at[1] - 1
    for bad in (math.nan, math.inf, -math.inf):
        other = q.clone()
        other[row, 3, 5] = bad
        out = serve.paged_attention_mx4(other, kc, vc, off, kvl, table, max(new)).view(-1, 8, 128)
        torch.cuda.synchronize()
        assert bool(out[row, 3].isnan().all())
        out[row, 3] = ref[row, 3]
        assert torch.equal(out, ref), bad


@pytest.mark.parametrize("D,H,Hk", [(128, 8, 2), (64, 5, 1)])
def test_out_may_be_q(dev, D, H, Hk):
    from llmr_amd import serve
    for past, new in (([9000, 3, 70], [1, 1, 1]), ([4000, 0], [6, 4]), ([5000, 100, 0], [300, 1, 70])):
        q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, BF16, D, H, Hk, 16, past, new, seed=42)
        ref = serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new))
        serve.paged_attention_mx4(q, kc, vc, off, kvl, table, max(new), out=q.flatten(1))
        torch.cuda.synchronize()
        assert torch.equal(q.flatten(1), ref), new


def test_cache_past_32_bit_offsets(dev):
    """Pages whose byte offsets pass 2^32: rows stored to, read back from and attended to at the end of a 5 GiB cache."""
    from llmr_amd import serve
    Hk, page, D = 8, 64, 128
    n_pages = (5 << 30) // (Hk * page * D // 2)
    kc, vc = _caches(n_pages, Hk, page, D, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    n, H = 300, 16
    pages = torch.tensor([n_pages - 1, 0, n_pages - 2, n_pages // 2, n_pages - 7], device=dev)
    j = torch.arange(n, device=dev)
    slots = (pages[j // page] * page + j % page).int()
    qkv = torch.randn(n, (H + 2 * Hk) * D, generator=g, device=dev)
    q = torch.empty(n, H, D, dtype=F16, device=dev)
    serve.qkv_tokens_mx4(qkv, q, kc, vc, slots)
    ko, vo = (torch.empty(n, Hk, D, dtype=F16, device=dev) for _ in range(2))
    serve.mx4_rows(kc, vc, slots, ko, vo)
    torch.cuda.synchronize()
    x = qkv.view(n, H + 2 * Hk, D)
    assert torch.equal(ko.double(), _decode(*_encode(x[:, H:H + Hk]))) and torch.equal(vo.double(), _decode(*_encode(x[:, H + Hk:])))
    for new in (1, 6, 70):
        qs = q[n - new:].contiguous()
        out = serve.paged_attention_mx4(qs, kc, vc, torch.tensor([0, new], dtype=torch.int32, device=dev),
                                        torch.tensor([n], dtype=torch.int32, device=dev), pages.int()[None].contiguous(), new)
        torch.cuda.synchronize()
        _paged_check(qs, [(ko.double(), vo.double())], [0, new], [n], out, 1 / math.sqrt(D), f"far pages, {new} new")


# ---- refusals ---------------------------------------------------------------------


def test_refusals(dev):
    from llmr_amd import capi, serve
    q, kc, vc, rows, at, off, kvl, table, kv = _paged_case(dev, F16, 64, 4, 2, 16, [50, 9], [3, 1], seed=1)
    base = dict(q=q, k=kc, v=vc, seq_offsets=off, kv_len=kvl, block_table=table, max_new=3)
    serve.paged_attention_mx4(**base)
    C = serve.Mx4Cache
    empty = lambda *s: C.empty(*s, dev)  # noqa: E731
    for kw in (dict(q=q.float()), dict(v=C(vc.data[:-1], vc.scales[:-1])), dict(k=C(kc.data.transpose(1, 2), kc.scales)),
               dict(k=C(kc.data, kc.scales[:, :, :, :1])), dict(k=C(kc.data.char(), kc.scales)), dict(seq_offsets=off[:2]),
               dict(kv_len=kvl.float()), dict(block_table=table.t()), dict(block_table=table.long()),
               dict(block_table=table[:1]), dict(q=q[:, :, :32]), dict(v=C(vc.data.cpu(), vc.scales)), dict(max_new=-1)):
        with pytest.raises((ValueError, capi.LlmrError)):
            serve.paged_attention_mx4(**{**base, **kw})
    for kw in (dict(scale=0.0), dict(scale=math.nan), dict(k=empty(9, 2, 24, 64), v=empty(9, 2, 24, 64)),
               dict(k=empty(9, 3, 16, 64), v=empty(9, 3, 16, 64)),
               dict(q=torch.zeros(4, 4, 96, dtype=F16, device=dev), k=empty(9, 2, 16, 96), v=empty(9, 2, 16, 96)),
               dict(out=torch.empty(4, 260, dtype=F16, device=dev)[:, :256])):
        with pytest.raises(capi.LlmrError) as err:
            serve.paged_attention_mx4(**{**base, **kw})
        assert err.value.code == capi.LLMR_ERR_INVALID_ARG
    need = serve.paged_attention_mx4_scratch(q, kc, table, 3).numel()
    if need:
        with pytest.raises(capi.LlmrError, match="scratch"):
            serve.paged_attention_mx4(**base, scratch=torch.empty(need - 16, dtype=torch.uint8, device=dev))
        with pytest.raises(capi.LlmrError, match="scratch"):
            serve.paged_attention_mx4(**base, scratch=torch.empty(need + 4, dtype=torch.uint8, device=dev)[4:])
    assert serve.paged_attention_mx4(**{**base, "q": q[:0]}).shape == (0, 256)
    D, T = 64, 5
    qkv = torch.zeros(T, 8 * D, device=dev)
    q = torch.empty(T, 4, D, dtype=F16, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    tabs = _tables(dev, 4, D)
    kc, vc = empty(3, 2, 16, D), empty(3, 2, 16, D)
    serve.qkv_tokens_mx4(qkv, q, kc, vc, slots)
    for args, kw in (((qkv.half(), q, kc, vc, slots), {}), ((qkv[:4], q, kc, vc, slots), {}),
                     ((qkv[:, :7 * D], q, kc, vc, slots), {}), ((qkv, q.float(), kc, vc, slots), {}),
                     ((qkv, q, kc, vc, slots.long()), {}), ((qkv, q, kc, vc, slots[:4]), {}),
                     ((qkv, q, kc, vc, slots), dict(rope=tabs)), ((qkv, q, kc, vc, slots), dict(eps=-1.0)),
                     ((qkv, q, kc, kc, slots), {}), ((qkv, q, empty(3, 2, 16, 128), empty(3, 2, 16, 128), slots), {}),
                     ((qkv, q, empty(3, 2, 24, D), empty(3, 2, 24, D), slots), {}),
                     ((qkv, q, kc, C(vc.data, kc.scales), slots), {})):
        with pytest.raises((ValueError, capi.LlmrError)):
            serve.qkv_tokens_mx4(*args, **kw)
    serve.qkv_tokens_mx4(qkv[:0], q[:0], kc, vc, slots)
    ko, vo = (torch.empty(T, 2, D, dtype=F16, device=dev) for _ in range(2))
    serve.mx4_rows(kc, vc, slots, ko, vo)
    for args in ((kc, vc, slots, ko, vo.bfloat16()), (kc, vc, slots, ko.float(), vo.float()), (kc, vc, slots[:4], ko, vo),
                 (kc, vc, slots.long(), ko, vo), (kc, vc, slots, ko[:, :1], vo[:, :1]), (kc, vc, slots, ko, ko),
                 (kc, vc, slots, ko, vo[:4]), (kc, empty(4, 2, 16, D), slots, ko, vo)):
        with pytest.raises((ValueError, capi.LlmrError)):
            serve.mx4_rows(*args)
    with pytest.raises(capi.LlmrError, match="overlap"):
        serve.mx4_rows(kc, vc, slots, ko, kc.data.view(-1)[:T * 2 * D * 2].view(F16).view(T, 2, D))
    serve.mx4_rows(kc, vc, slots, ko[:0], vo[:0])


# ---- a run of them ------------------------------------------------------------------


@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_steps(dev, captured):
    """Requests that come, grow by chunks and single tokens and leave, over 8-bit linears and a 4-bit cache, one padded
    batch, four steps: plan, rows to integers with the norm, QKV product, rows into the cache, attention, rows to
    integers, output product. Each step's pieces are compared with their definitions on what the step left."""
    import numpy as np

    from llmr_amd import int8, serve
    D, H, Hk, hidden, page, rows, n = 64, 4, 2, 256, 16, 160, 3
    width = (H + 2 * Hk) * D
    g = torch.Generator(device=dev).manual_seed(8)
    w, ws = int8.quantize_rows(torch.randn(width, hidden, generator=g, device=dev) * 0.06)
    wo, wos = int8.quantize_rows(torch.randn(hidden, H * D, generator=g, device=dev) * 0.06)
    qn, kn, xn = (torch.rand(m, generator=g, device=dev) + 0.5 for m in (D, D, hidden))
    tabs = _tables(dev, 512, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    past, new = i32([0] * n), i32([0] * n)
    free, count = torch.arange(40, dtype=torch.int32, device=dev), i32([40])
    table = torch.full((n, 16), -1, dtype=torch.int32, device=dev)
    kc, vc = _caches(40, Hk, page, D, dev, 255)
    x = torch.zeros(rows, hidden, device=dev)
    xq, xs = torch.empty(rows, hidden, dtype=torch.int8, device=dev), torch.empty(rows, device=dev)
    aq, as_ = torch.empty(rows, H * D, dtype=torch.int8, device=dev), torch.empty(rows, device=dev)
    qkv = torch.zeros(rows, width, device=dev)
    q = torch.zeros(rows, H, D, dtype=BF16, device=dev)
    att = torch.zeros(rows, H * D, dtype=BF16, device=dev)
    y = torch.zeros(rows, hidden, device=dev)
    b = serve.PagedBatch.empty(n, rows, dev)
    scratch = serve.paged_attention_mx4_scratch(q, kc, table, rows)

    def step():
        serve.paged_plan(past, new, free, count, table, page, b)
        int8.quantize_rows(x, norm=xn, q=xq, scales=xs)
        int8.matmul(xq, xs, w, ws, out=qkv)
        serve.qkv_tokens_mx4(qkv, q, kc, vc, b.slots, positions=b.positions, q_norm=qn, k_norm=kn, rope=tabs)
        serve.paged_attention_mx4(q, kc, vc, b.seq_offsets, b.kv_len, table, rows, out=att, scratch=scratch)
        int8.quantize_rows(att, q=aq, scales=as_)
        int8.matmul(aq, as_, wo, wos, out=y)

    graph = _capture(step) if captured else None
    table.fill_(-1)
    lens = [0] * n
    rng = np.random.default_rng(0)
    for i, (ns, ends) in enumerate([([90, 30, 0], []), ([1, 1, 47], []), ([1, 33, 1], [0]), ([150, 1, 1], [])]):
        past.copy_(i32(lens)), new.copy_(i32(ns))
        x.copy_(torch.from_numpy(rng.standard_normal((rows, hidden)).astype(np.float32)))
        att.fill_(7.0)
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        T = sum(ns)
        assert bool((att[T:] == 7).all())
        z = x.double() * xn.double()
        top = z.abs().amax(1, keepdim=True)
        assert torch.equal(xq, torch.round(127 * z / top).to(torch.int8))
        assert torch.equal(qkv, ((xq.double() @ w.double().t().contiguous()).float() * xs[:, None]) * ws)
        live = b.slots[:T].long()
        k64 = _rows_oracle(qkv.view(rows, H + 2 * Hk, D)[:T, H:H + Hk], kn, 1e-6, tabs, b.positions[:T].long(), True)[0]
        for c, want in ((kc, k64), (vc, qkv.view(rows, H + 2 * Hk, D)[:T, H + Hk:].double())):
            assert torch.equal(_decode(_at(c.data, live), _at(c.scales, live)), _decode(*_encode(want)))
        at = 0
        for s, m in enumerate(ns):
            lens[s] += m
            if m:
                place = torch.arange(lens[s], device=dev)
                have = table[s].long()[place // page] * page + place % page
                k, v = (_decode(_at(c.data, have), _at(c.scales, have)) for c in (kc, vc))
                o, A, e = _definition(q[at:at + m], k, v, 1 / math.sqrt(D), lens[s] - m)
                _check(att[at:at + m].unflatten(1, (H, D)), o, A, e, float(v.abs().max()), lens[s], BF16, f"step {i}")
            at += m
        assert torch.equal(y, ((aq.double() @ wo.double().t().contiguous()).float() * as_[:, None]) * wos)
        top = att.double().abs().amax(1, keepdim=True)
        assert torch.equal(aq, torch.round(127 * att.double() / torch.where(top > 0, top, 1.0)).to(torch.int8))
        count.copy_(b.pages[:1])
        assert int(b.pages[1]) == 0
        for s in ends:  # its pages go back; the request in its place starts anew
            held = -(-lens[s] // page)
            c = int(count)
            free[c:c + held] = table[s, :held]
            count += held
            lens[s] = 0
            table[s] = -1
