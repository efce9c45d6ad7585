"""GPU linears in 8-bit integers (llmr_quantize_rows_i8, llmr_matmul_i8). The integers and the products' sums are whole
numbers, and each rounding of the results is a step of the definition: everything is compared for equality, but the
scales, whose 64-bit terms may be added in any order (one f32 rounding, 2^-24, and 2^-40 for those)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rows_oracle(x, norm, eps):
    """q, scales in 64 bits, from the definition."""
    x = x.double()
    y = x if norm is None else x * norm.double()
    bad = ~torch.isfinite(y).all(dim=1)
    y = torch.where(bad[:, None], 0.0, y)
    a = y.abs().amax(dim=1) if y.shape[0] else y.new_zeros(0)
    # 127 y / a next to a half: the quotient is one rounding of the exact one, and a half itself is exact
    q = torch.round(127.0 * y / torch.where(a > 0, a, 1.0)[:, None]).to(torch.int8)
    s = a / 127
    if norm is not None:
        s = torch.where(a > 0, s / torch.sqrt((x * x).mean(dim=1) + eps), 0.0)
    return q, torch.where(bad, math.nan, s)


def _check_rows(x, norm=None, eps=1e-6, **kw):
    from llmr_amd import int8
    q, s = int8.quantize_rows(x, norm=norm, eps=eps, **kw)
    torch.cuda.synchronize()
    wq, ws = _rows_oracle(x, norm, eps)
    assert torch.equal(q, wq), int((q != wq).sum())
    assert torch.equal(s.isnan(), ws.isnan())
    off = torch.where(ws.isnan(), 0.0, (s.double() - ws).abs())
    assert bool((off <= ws.nan_to_num(0.0) * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -150).all())
    return q, s


# one piece of 16; rows shorter than the workgroup, around its 2048 elements, several times it, the longest
ROWS = [(1, 16), (3, 48), (5, 4096), (2, 2064), (7, 2048), (4, 2032), (300, 272), (64, 3840), (9, 10240), (2, 131056),
        (2500, 64), (5, 512), (6, 528), (7, 1024), (3, 1040), (5, 8192), (2, 8208), (3, 16384), (3, 16400), (11, 5008)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,K", ROWS)
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_quantize_rows(dev, dtype, T, K, norm):
    g = torch.Generator(device=dev).manual_seed(T + K)
    x = (torch.randn(T, K, generator=g, device=dev) * torch.exp(2 * torch.randn(T, 1, generator=g, device=dev))).to(dtype)
    w = torch.randn(K, generator=g, device=dev) if norm else None
    _check_rows(x, w)
    # columns of a wider buffer, into columns of one whose other bytes stay
    wide = torch.zeros(T, K + 48, dtype=dtype, device=dev)
    wide[:, 16:16 + K] = x
    q = torch.full((T, K + 32), 77, dtype=torch.int8, device=dev)
    _check_rows(wide[:, 16:16 + K], w, q=q[:, 16:16 + K])
    assert bool((q[:, :16] == 77).all()) and bool((q[:, 16 + K:] == 77).all())


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_quantize_rows_ties(dev, dtype):
    """Rows whose largest element is a multiple of 127 steps: 127 y / a is a half for many of a type's numbers."""
    steps = [1, 2] if dtype == BF16 else list(range(1, 17))
    x = torch.zeros(len(steps), 528, dtype=F32, device=dev)
    for i, m in enumerate(steps):
        half = torch.arange(0, 127, device=dev) + 0.5
        v = (half * m).to(dtype).float()
        x[i, :127], x[i, 127:254] = v, -v
        x[i, 254:381] = torch.nextafter(v.to(dtype), torch.zeros_like(v, dtype=dtype)).float()
        x[i, 400] = 127.0 * m
        assert float((v == half * m).float().mean()) > 0.4  # halves that the type has
    _check_rows(x.to(dtype))
    _check_rows(x)
    _check_rows(x, torch.ones(528, device=dev))
    _check_rows(torch.ldexp(x, torch.tensor(-130, device=dev)))  # among the subnormals


def _exact_rows(x, norm):
    """q from the definition in whole fractions: 127 y / a to nearest, ties to even, for rows on the host."""
    from fractions import Fraction
    out = []
    for row in x.tolist():
        y = [Fraction(a) * Fraction(b) for a, b in zip(row, norm.tolist())]
        a = max(map(abs, y))
        out.append([round(127 * v / a) if a else 0 for v in y])
    return torch.tensor(out, dtype=torch.int8)


@pytest.mark.parametrize("K", [528, 16400])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_quantize_rows_ties_under_a_norm(dev, dtype, K):
    """Halves of rows with a norm whose weights have all of f32's bits: (2 k + 1) m against 254 m, m as long as the type
    allows, their neighbours, and halves that two weights make. y and a are products of 48 bits, 127 y has 55."""
    g = torch.Generator().manual_seed(17)
    bits = {F32: 16, BF16: 1, F16: 4}[dtype]
    x = torch.zeros(8, K, dtype=F32)
    norm = torch.rand(K, generator=g) + 0.5
    k = torch.arange(127, dtype=F32)
    for i in range(8):
        m = float(torch.randint(2 ** (bits - 1), 2 ** bits, (), generator=g)) if bits > 1 else 1.0
        v = ((2 * k + 1) * m).to(dtype).float()
        x[i, :127], x[i, 127:254] = v, -v
        x[i, 254:381] = torch.nextafter(v.to(dtype), torch.zeros_like(v, dtype=dtype)).float()
        x[i, 400] = 254 * m
        # half the largest by the weight: the element is the largest one's
        x[i, 401], x[i, K - 1] = 254 * m, -254 * m
    w = float(norm[0])
    norm[:401] = w
    norm[401], norm[K - 1] = w / 2, w / 2
    x = x.to(dtype)
    from llmr_amd import int8
    q, _ = int8.quantize_rows(x.to(dev), norm=norm.to(dev))
    torch.cuda.synchronize()
    want = _exact_rows(x.double()[:, :528], norm[:528].double())
    if K > 528:
        want[:, 401:] = 0
        want[:, 401] = 64
    got = q.cpu()[:, :528]
    assert torch.equal(got, want), int((got != want).sum())
    assert bool((want[:, 401] == 64).all()) and bool((q.cpu()[:, K - 1] == -64).all())


@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_quantize_rows_special_values(dev, norm):
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(12, 160, generator=g, device=dev)
    x[1] = 0
    x[2, 70], x[3, 0], x[4, 159] = math.inf, -math.inf, math.nan
    x[5] *= 3e38 / x[5].abs().max()
    x[6] *= 1e-38
    x[7] *= 1e-44
    x[8, 1:] = 0
    x[9] = torch.finfo(F32).min
    x[10] = 2.0 ** -149
    w = torch.randn(160, generator=g, device=dev) if norm else None
    q, s = _check_rows(x, w)
    assert bool((q[[1, 2, 3, 4]] == 0).all()) and bool(s[[2, 3, 4]].isnan().all()) and float(s[1]) == 0.0
    if norm:
        _check_rows(x, torch.full((160,), 1e38, device=dev))
        _check_rows(x, torch.zeros(160, device=dev))
        w[3] = math.nan
        assert bool(_check_rows(x, w)[1].isnan().all())


def _product_oracle(x, xs, w, ws, dtype):
    # whole numbers below 2^31: exact in 64 bits whatever the order
    acc = x.double() @ w.double().t().contiguous()
    return ((acc.float() * xs[:, None]) * ws[None]).to(dtype)


def _ints(g, dev, *shape):
    return torch.randint(-128, 128, shape, generator=g, device=dev, dtype=torch.int32).to(torch.int8)


def _check_product(dev, M, N, K, dtype, seed=0, stride=0):
    """The product into the middle of a buffer whose other elements stay."""
    from llmr_amd import int8
    g = torch.Generator(device=dev).manual_seed(seed + M + N + K)
    x, w = _ints(g, dev, M, K + stride)[:, :K], _ints(g, dev, N, K + 2 * stride)[:, :K]
    xs, ws = (torch.rand(n, generator=g, device=dev) * 0.01 + 0.001 for n in (M, N))
    buf = torch.full((M + 2, N + 7), 7.0, dtype=dtype, device=dev)
    out = buf[1:M + 1, 3:N + 3]
    assert int8.matmul(x, xs, w, ws, out=out) is out
    new = int8.matmul(x, xs, w, ws, dtype=dtype)
    torch.cuda.synchronize()
    want = _product_oracle(x, xs, w, ws, dtype)
    assert torch.equal(out, want), (M, N, K, int((out != want).sum()))
    assert torch.equal(new, want)
    buf[1:M + 1, 3:N + 3] = 7.0
    assert bool((buf == 7).all())


# (M, N, K): one of each; around the tiles of 16, 32, 64, 128 and 256; K of one piece, of odd numbers of them, around the
# K tiles; few rows of long sums; more tiles than the card takes at once
PRODUCTS = [(1, 1, 16), (1, 60, 64), (2, 17, 48), (15, 33, 80), (16, 16, 64), (17, 129, 112), (1, 6144, 4096), (5, 4096, 14336),
            (31, 255, 128), (32, 256, 256), (33, 257, 272), (64, 4096, 4096), (63, 1000, 1040), (65, 513, 2064), (100, 126, 656),
            (127, 128, 144), (128, 128, 4096), (129, 384, 400), (200, 3425, 416), (255, 512, 512), (256, 256, 1024),
            (257, 2049, 784), (300, 96, 14400), (511, 777, 3856), (777, 1021, 3840), (1024, 2560, 2560), (2049, 1537, 528),
            (4100, 300, 1600), (300, 600, 16000), (130, 1000, 14336), (1000, 40, 5008), (65, 16, 2064), (30, 10240, 2064),
            (60, 12000, 1040), (3, 20480, 96), (16, 16400, 1104), (1, 16, 131056), (40, 24, 131056), (300, 290, 131056)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_matmul(dev, dtype, M, N, K):
    _check_product(dev, M, N, K, dtype)


@pytest.mark.parametrize("M,N,K", [(1, 100, 64), (20, 65, 96), (70, 300, 208), (300, 520, 336), (600, 1030, 144)])
def test_matmul_strides(dev, M, N, K):
    _check_product(dev, M, N, K, BF16, stride=16)
    _check_product(dev, M, N, K, F32, stride=4096)


@pytest.mark.parametrize("M,N", [(1, 20), (33, 300), (300, 300), (700, 600)])
def test_matmul_extreme_sums(dev, M, N):
    """The longest rows of -128 on both sides: 131056 * 2^14, just within an int32; and of alternating signs."""
    from llmr_amd import int8
    K = 131056
    x, w = torch.full((M, K), -128, dtype=torch.int8, device=dev), torch.full((N, K), -128, dtype=torch.int8, device=dev)
    w[1::2] = 127
    out = int8.matmul(x, torch.ones(M, device=dev), w, torch.ones(N, device=dev), dtype=F32)
    torch.cuda.synchronize()
    assert bool((out[:, ::2] == float(K * 2 ** 14)).all())
    assert bool((out[:, 1::2] == torch.tensor(-128.0 * 127 * K, dtype=F32, device=dev)).all())


def test_matmul_scales_of_no_number(dev):
    """A row's NaN stays in its row, a channel's in its channel; scales of 0, infinite and tiny ones as multiplied."""
    from llmr_amd import int8
    g = torch.Generator(device=dev).manual_seed(3)
    for M, N, K in ((5, 40, 64), (300, 280, 128)):
        x, w = _ints(g, dev, M, K), _ints(g, dev, N, K)
        xs, ws = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
        xs[1], xs[2], xs[3], ws[7], ws[8] = math.nan, 0.0, 1e-40, math.nan, 2e-39
        x[4] = 0
        for dtype in (F32, F16):
            out = int8.matmul(x, xs, w, ws, dtype=dtype)
            torch.cuda.synchronize()
            want = _product_oracle(x, xs, w, ws, dtype)
            assert torch.equal(out.isnan(), want.isnan())
            assert torch.equal(out.nan_to_num(0.0), want.nan_to_num(0.0))
            assert int(out.isnan().sum()) == M + N - 1


def test_offsets_past_32_bits(dev):
    """Outputs and rows whose byte offsets pass 2^32."""
    from llmr_amd import int8
    g = torch.Generator(device=dev).manual_seed(4)
    M, N, K = 70000, 20011, 16
    x, w = _ints(g, dev, M, K), _ints(g, dev, N, K)
    xs, ws = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
    out = int8.matmul(x, xs, w, ws, dtype=F32)
    torch.cuda.synchronize()
    for a in (0, 30000, M - 300):
        assert torch.equal(out[a:a + 300], _product_oracle(x[a:a + 300], xs[a:a + 300], w, ws, F32)), a
    del out
    far = torch.empty(600, 1 << 23, dtype=torch.int8, device=dev)
    far[:, :64] = _ints(g, dev, 600, 64)
    x, w = far[:, :64], far.flip(0)[:, :64].contiguous()
    for a, b in ((x, w), (w, x), (x[:3], w), (w[:3], x)):
        M, N = a.shape[0], b.shape[0]
        xs, ws = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
        out = int8.matmul(a, xs, b, ws, dtype=F32)
        torch.cuda.synchronize()
        assert torch.equal(out, _product_oracle(a, xs, b, ws, F32)), (M, N)
    rows = torch.randn(3, 1 << 30, dtype=F16, device=dev)[:, :64]  # 2 GiB apart
    _check_rows(rows)


@pytest.mark.parametrize("M,N", [(1, 1 << 28), (20, (1 << 27) + 5), ((1 << 22) + 100, 17), (5000000, 3)])
def test_very_wide_and_very_tall(dev, M, N):
    """More workgroups than one dimension of a launch takes."""
    from llmr_amd import int8
    g = torch.Generator(device=dev).manual_seed(6)
    x, w = _ints(g, dev, M, 16), _ints(g, dev, N, 16)
    xs, ws = torch.rand(M, generator=g, device=dev), torch.rand(N, generator=g, device=dev)
    out = int8.matmul(x, xs, w, ws, dtype=BF16)
    torch.cuda.synchronize()
    m, n = min(M, 300), min(N, 300)
    for a in (0, (M - m) // 2, M - m):
        for b in (0, (N - n) // 2, N - n):
            want = _product_oracle(x[a:a + m], xs[a:a + m], w[b:b + n], ws[b:b + n], BF16)
            assert torch.equal(out[a:a + m, b:b + n], want), (a, b)


def _capture(fn):
    fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fn()
    return graph


@pytest.mark.parametrize("M,N,K", [(1, 6144, 4096), (40, 1000, 4096), (300, 2000, 4000), (700, 1024, 512)])
def test_captured_and_on_streams(dev, M, N, K):
    """Rows to integers and their product, captured: replays with other rows, between eager calls; and at once on
    several streams with outputs of their own."""
    from llmr_amd import int8
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(M, K, generator=g, device=dev)
    norm = torch.rand(K, generator=g, device=dev) + 0.5
    w, ws = int8.quantize_rows(torch.randn(N, K, generator=g, device=dev) * 0.02)
    bufs = [(torch.empty(M, K, dtype=torch.int8, device=dev), torch.empty(M, device=dev),
             torch.empty(M, N, dtype=BF16, device=dev)) for _ in range(3)]

    def linear(x, b):
        int8.quantize_rows(x, norm=norm, q=b[0], scales=b[1])
        return int8.matmul(b[0], b[1], w, ws, out=b[2])

    graph = _capture(lambda: linear(x, bufs[0]))
    for i in range(4):
        x.copy_(torch.randn(M, K, generator=g, device=dev) * (i + 1))
        bufs[0][2].fill_(7.0)
        graph.replay()
        eager = linear(x, bufs[1])
        torch.cuda.synchronize()
        assert torch.equal(bufs[0][2], eager)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        for s, b in zip(streams, bufs):
            b[2].fill_(7.0)
        torch.cuda.synchronize()
        for s, b in zip(streams, bufs):
            with torch.cuda.stream(s):
                linear(x, b)
        torch.cuda.synchronize()
        assert all(torch.equal(b[2], eager) for b in bufs)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_a_linear_is_near_its_weights(dev, dtype):
    """RMS norm, integers and product against the f64 linear of the unrounded weights. Both factors of each term are off
    by at most half a step of their row: |y - s q| <= s / 2 (s = a / 127), the weights' alike, so a sum is off by at
    most sum_k (s_x |w| + s_w |y| + s_x s_w / 2) / 2, its roundings to f32 and to the type aside."""
    from llmr_amd import int8
    g = torch.Generator(device=dev).manual_seed(6)
    M, N, K = 37, 250, 1024
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    norm = torch.rand(K, generator=g, device=dev) + 0.5
    w = torch.randn(N, K, generator=g, device=dev) * 0.03
    wq, ws = int8.quantize_rows(w)
    q, s = int8.quantize_rows(x, norm=norm)
    out = int8.matmul(q, s, wq, ws, dtype=dtype)
    torch.cuda.synchronize()
    x = x.double()
    y = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * norm.double()
    want = y @ w.double().t().contiguous()
    sx, sw = s.double()[:, None], ws.double()[None]
    off = 0.5 * (sx * w.double().abs().sum(1)[None] + sw * y.abs().sum(1)[:, None] + 0.5 * K * sx * sw)
    # scales are off by 2^-24, results by three f32 roundings and the type's one
    bound = off * (1 + 2.0 ** -20) + (want.abs() + off) * (2.0 ** -20 + torch.finfo(dtype).eps / 2)
    assert bool(((out.double() - want).abs() <= bound).all())


def test_refusals(dev):
    from llmr_amd import capi, int8
    x, w = torch.zeros(4, 64, dtype=torch.int8, device=dev), torch.zeros(6, 64, dtype=torch.int8, device=dev)
    xs, ws, f = torch.ones(4, device=dev), torch.ones(6, device=dev), torch.zeros(4, 64, device=dev)
    int8.matmul(x, xs, w, ws)
    out = torch.zeros(4, 6, device=dev)
    for args, kw in (((x.float(), xs, w, ws), {}), ((x, xs, w[:, :48], ws), {}), ((x, xs[:3], w, ws), {}),
                     ((x, xs, w, ws[:5]), {}), ((x, xs.double(), w, ws), {}), ((x, xs, w.cpu(), ws), {}),
                     ((x, xs, w, ws), dict(out=out[:3])), ((x, xs, w, ws), dict(out=out.double())),
                     ((x, xs, w, ws), dict(out=out.t().contiguous().t())), ((x[0], xs, w, ws), {}),
                     ((x.t().contiguous().t(), xs, w, ws), {}), ((x, xs, w, ws), dict(dtype=torch.int32))):
        with pytest.raises((ValueError, capi.LlmrError)):
            int8.matmul(*args, **kw)
    odd = torch.zeros(4 * 64 + 8, dtype=torch.int8, device=dev)[8:].view(4, 64)
    for args, kw in (((x[:, :24], xs, w[:, :24], ws), {}), ((odd, xs, w, ws), {}), ((x[:, :0], xs, w[:, :0], ws), {}),
                     ((torch.zeros(4, 72, dtype=torch.int8, device=dev)[:, :64], xs, w, ws), {}),
                     ((x.expand(4, 64), xs, w[:1].expand(6, 64), ws), {}),
                     ((x, xs, w, ws), dict(out=out.view(-1)[:6].expand(4, 6)))):
        with pytest.raises(capi.LlmrError) as err:
            int8.matmul(*args, **kw)
        assert err.value.code == capi.LLMR_ERR_INVALID_ARG
    far = 131072
    with pytest.raises(capi.LlmrError, match="in_dim"):
        int8.matmul(torch.zeros(1, far, dtype=torch.int8, device=dev), xs[:1], torch.zeros(1, far, dtype=torch.int8, device=dev),
                    ws[:1])
    both = torch.zeros(2048, dtype=torch.int8, device=dev)
    with pytest.raises(capi.LlmrError, match="overlap"):
        int8.matmul(both[:256].view(4, 64), xs, w, ws, out=both[240:336].view(F32).view(4, 6))
    buf = torch.ones(40, device=dev)
    with pytest.raises(capi.LlmrError, match="overlap"):
        int8.matmul(x, xs, w, buf[20:26], out=buf[:24].view(4, 6))
    assert int8.matmul(x[:0], xs[:0], w, ws).shape == (0, 6) and int8.matmul(x, xs, w[:0], ws[:0]).shape == (4, 0)
    int8.quantize_rows(f)
    for args, kw in (((f.double(),), {}), ((f,), dict(norm=xs)), ((f,), dict(norm=torch.ones(64, device=dev).half())),
                     ((f,), dict(q=torch.zeros(4, 48, dtype=torch.int8, device=dev))), ((f,), dict(scales=xs[:3])),
                     ((f.cpu(),), dict(q=x, scales=xs)), ((f[0],), {}), ((f,), dict(q=f))):
        with pytest.raises((ValueError, capi.LlmrError)):
            int8.quantize_rows(*args, **kw)
    one = torch.ones(64, device=dev)
    for args, kw in (((f[:, :24],), {}), ((f[:, :0],), {}), ((torch.zeros(4, 66, device=dev)[:, :64],), {}),
                     ((torch.zeros(4, 65, device=dev)[:, 1:],), {}), ((f,), dict(norm=one, eps=-1.0)),
                     ((f,), dict(norm=one, eps=math.nan)), ((torch.zeros(1, far, device=dev),), {}),
                     ((f,), dict(q=f.view(torch.int8).view(-1)[:256].view(4, 64))),
                     ((f,), dict(scales=f.view(-1)[:4]))):
        with pytest.raises(capi.LlmrError) as err:
            int8.quantize_rows(*args, **kw)
        assert err.value.code == capi.LLMR_ERR_INVALID_ARG
    assert int8.quantize_rows(f[:0])[0].shape == (0, 64)
