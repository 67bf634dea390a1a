"""Products over int8 weights with a scale a channel, the activations quantized to int8 with a scale a token,
against the definition: codes and scales by IEEE F32 steps in numpy, exact integer sums in 64 bits, then
the F32 steps of an output bit for bit, and the real value in 64 bits within what its roundings can do."""
import numpy as np
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of F32
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def I():
    require_gpu()
    import syntropy_amd.int8 as I
    return I


def quantized(x):
    """(codes, scales) of rows by the definition, in numpy F32."""
    x = x.float().cpu().numpy()
    with np.errstate(all="ignore"):
        a = np.abs(x).max(1)
        s = (a / np.float32(127)).astype(np.float32)
        inv = (np.float32(1) / s).astype(np.float32)
        inv = np.where(np.isfinite(inv) & np.isfinite(a), inv, np.float32(0))
        q = np.rint(np.where(np.isfinite(x), x, np.float32(0)) * inv[:, None])
    assert np.abs(q).max(initial=0) <= 127
    bad = ~np.isfinite(x).all(1)
    q[bad] = 0
    return q.astype(np.int64), np.where(bad, np.float32(np.nan), s).astype(np.float32)


def sums(q, codes):
    """Exact: whole numbers below 2^53 in 64-bit floats."""
    return np.rint((torch.from_numpy(q).double() @ codes.cpu().double().t()).numpy()).astype(np.int64)


def value(S, sx, sw, bias):
    """An output's F32 steps, and its value in 64 bits with the most that those steps move it."""
    with np.errstate(all="ignore"):
        v = (S.astype(np.float32) * sx[:, None]) * sw[None, :]
        r = S.astype(np.float64) * sx[:, None].astype(np.float64) * sw[None, :].astype(np.float64)
        err = np.abs(r) * (3.01 * U) + 2.0 ** -148  # a conversion and two products
        if bias is not None:
            v = v + bias[None, :]
            r = r + bias[None, :].astype(np.float64)
            err = err + np.abs(r) * U * 1.01 + err * U
    return v, r, err


def make(n, k, seed, bias=False, pad=0, codes=None):
    g = torch.Generator().manual_seed(seed)
    ld = -(-k // 16) * 16 + 16 * pad
    held = torch.randint(-127, 128, (n, ld), generator=g, dtype=torch.int8)  # behind a row's codes: anything
    if codes is not None:
        held[:, :k] = codes
    s = torch.rand(n, generator=g) * 1e-3 + 1e-5
    b = torch.randn(n, generator=g) if bias else None
    return held.cuda()[:, :k], s.cuda(), None if b is None else b.cuda()


def rows_of(rows, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.logspace(-2, 2, rows)[:, None]
    x[:, ::37] *= 8
    return x.to(dtype)


def same(got, want, what=""):
    got, want = got.cpu(), torch.as_tensor(want)
    assert got.shape == want.shape and got.dtype == want.dtype, what
    ok = (got == want) | (got.isnan() & want.isnan())
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} differ, first {got[~ok][:3]} for {want[~ok][:3]}"


def check(I, w, x, rows, what, gated=False, y=None, ws=None, stream=None):
    codes, s, b = w
    W = I.Weights(codes, s, b)
    got = (I.gate_up_act if gated else I.gemv)(W, x, rows, y=y, ws=ws, stream=stream)
    torch.cuda.synchronize()
    q, sx = quantized(x[:rows])
    v, r, err = value(sums(q, codes), sx, s.cpu().numpy(), None if b is None else b.cpu().numpy())
    dt = got.dtype
    if not gated:
        assert ((np.abs(v - r) <= err) | ~np.isfinite(r)).all(), "the oracle's own steps"
        same(got[:rows], torch.from_numpy(v).to(dt), what)
        return got
    n = codes.shape[0] // 2
    g, u, eg, eu = r[:, :n], r[:, n:], err[:, :n], err[:, n:]
    with np.errstate(all="ignore"):
        sig = 1 / (1 + np.exp(-g))
        want = g * sig * u
        # |silu'| <= 1.1; exp within 2 steps (4 U), the sum, the quotient, the product: U each; where exp(-g)
        # passes F32's range the quotient is 0 for a value below 2^-126 * |g|
        tol = (1.1 * eg + np.abs(g * sig) * 8 * U + 2.0 ** -118) * np.abs(u) + np.abs(g * sig) * eu
        tol = tol * 1.01 + np.abs(want) * (U + HALF[dt]) * 1.01 + (2.0 ** -25 if dt is torch.float16 else 2.0 ** -133)
    d = got[:rows].double().cpu().numpy()
    ok = (np.abs(d - want) <= tol) | (np.isnan(d) & np.isnan(want)) | (d == want)
    if dt is torch.float16:  # past its range
        ok |= (np.abs(want) + tol >= 65504) & (np.abs(d) >= 65472) & (np.sign(d) == np.sign(want))
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.size} out of tolerance: {d[~ok][:3]} for {want[~ok][:3]}"
    return got


SHAPES = [(1, 1, 1), (1, 16, 1), (17, 100, 1), (300, 4096, 1), (4100, 2011, 1), (64, 14336, 1), (33, 15, 2),
          (48, 129, 3), (1000, 1024, 4), (130, 5000, 6), (257, 128, 8), (16, 127, 9), (512, 2048, 15), (95, 640, 16),
          (31, 4097, 17), (256, 256, 24), (700, 1408, 31), (129, 2048, 32), (128, 64, 33), (640, 4096, 47),
          (255, 512, 63), (256, 2000, 64), (1025, 1000, 65), (384, 3000, 100), (511, 768, 127), (256, 8192, 128),
          (130, 130, 129), (1280, 1100, 200), (513, 333, 255), (768, 2560, 256), (257, 2011, 257), (2048, 512, 333),
          (4096, 384, 513), (5, 700, 1000), (300, 160, 2049)]


@pytest.mark.parametrize("n,k,rows", SHAPES)
def test_gemv_is_its_definition(I, n, k, rows):
    for j, dt in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        announce(f"int8 gemv {n}x{k} rows {rows} {dt}")
        check(I, make(n, k, n + k + rows, bias=j == 1, pad=j), rows_of(rows, k, dt, rows + j).cuda(), rows, f"{n}x{k} {rows}")


@pytest.mark.parametrize("n,k,rows", SHAPES)
def test_gate_up_is_its_definition(I, n, k, rows):
    for j, dt in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        announce(f"int8 gate_up {n}x{k} rows {rows} {dt}")
        w = make(2 * n, k, n + k + rows, bias=j == 1, pad=j)
        w[1].mul_(3.0 / (k ** 0.5))
        x = rows_of(rows, k, dt, rows + j)
        x = (x / torch.logspace(-2, 2, rows)[:, None].to(dt)).cuda()  # gates of the size at which silu bends
        check(I, w, x, rows, f"{n}x{k} {rows}", gated=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4096), (3, 127), (5, 129), (2, 14336), (200, 2011), (1, 131072)])
def test_quantize_rows(I, dtype, rows, k):
    x = rows_of(rows, k, dtype, k)
    announce(f"quantize_rows {rows}x{k} {dtype}")
    codes, scales = I.quantize_rows(x.cuda())
    q, s = quantized(x)
    same(codes, torch.from_numpy(q).to(torch.int8))
    same(scales, torch.from_numpy(s))
    held = codes.as_strided((rows, codes.stride(0)), (codes.stride(0), 1))
    assert codes.stride(0) % 128 == 0 and not held[:, k:].any()


def edge_rows(k, dtype):
    x = rows_of(12, k, torch.float32, 5)
    tiny = {torch.float16: 2.0 ** -24}.get(dtype, 2.0 ** -133)  # the type's least value, or near it
    x[0] = 0
    x[1, k // 2] = float("nan")
    x[2, 0] = float("inf")
    x[3, k - 1] = float("-inf")
    x[4] = tiny
    x[5] = torch.where(torch.arange(k) % 2 == 0, tiny, -3 * tiny)
    x[6] = -x[7]
    x[8] = 60000.0
    x[9] = 0
    x[9, k - 1] = -2.5
    x[10] = torch.arange(k) % 255 - 127.0  # every code, the halves between them
    x[11] = (torch.arange(k) % 509 - 254.0) / 2
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [520, 2011])
def test_rows_of_zeros_nans_infinities_and_least_values(I, dtype, k):
    x = edge_rows(k, dtype).cuda()
    codes, scales = I.quantize_rows(x)
    q, s = quantized(x)
    same(codes, torch.from_numpy(q).to(torch.int8), "codes")
    same(scales, torch.from_numpy(s), "scales")
    w = make(70, k, 3)
    for rows in (1, 2, 4, 12):  # on each kernel; a NaN stays in its row
        announce(f"edge rows {rows} k {k} {dtype}")
        check(I, w, x, rows, f"{rows} rows")
        for r in range(0, 12, 4):
            check(I, w, x[r:], min(rows, 12 - r), f"{rows} rows from {r}")
    many = x.repeat(9, 1)
    announce("edge rows, many")
    check(I, w, many, 108, "many rows")


@pytest.mark.parametrize("rows", [1, 7, 40, 200])
def test_extreme_codes_and_the_longest_rows(I, rows):
    """The largest sum that fits: every product 127 * -128 over 131072 values; a scale of 0, a NaN scale."""
    k = 131072
    codes = torch.full((34, k), -128, dtype=torch.int8)
    codes[1::2] = 127
    codes[5, ::2] = 127
    w = make(34, k, 4, codes=codes)
    w[1][3] = 0.0
    w[1][4] = float("nan")
    w[1][6] = -1e-3
    x = torch.ones(rows, k)
    x[rows // 2, 1::2] = -1
    announce(f"longest rows, {rows}")
    check(I, w, x.cuda(), rows, "longest rows")


@pytest.mark.parametrize("rows", [1, 5, 20, 150])
@pytest.mark.parametrize("k", [256, 261])
def test_strided_and_unaligned_operands(I, rows, k):
    """Rows of x and y at any value's address with other values between them, which stay as they were."""
    for dt, ydt in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)):
        n = 75
        big = rows_of(rows + 2, 3 * k, dt, 9).cuda()
        x = big[1:, k - 1:2 * k - 1]
        out = torch.full((rows + 3, 2 * n + 3), 7.0, dtype=ydt, device="cuda")
        y = out[1:rows + 2, 3:n + 3]
        announce(f"strided {rows} rows k {k} {dt} -> {ydt}")
        for gated, w in ((False, make(n, k, 6)), (True, make(2 * n, k, 7))):
            out.fill_(7.0)
            got = check(I, w, x, rows, "strided", gated=gated, y=y)
            assert got.data_ptr() == y.data_ptr()
            mask = torch.ones_like(out, dtype=torch.bool)
            mask[1:rows + 1, 3:n + 3] = False
            assert (out[mask] == 7.0).all(), "values around y changed"


def test_offsets_past_32_bits(I):
    """Weight rows, x rows and y rows more than 2^32 bytes from the first."""
    n, k, rows = 40, 512, 36
    far = 1 << 27
    held = torch.empty(n * far, dtype=torch.int8, device="cuda")  # 5 GiB
    codes = held.as_strided((n, k), (far, 1))
    w = make(n, k, 8)
    codes.copy_(w[0])
    x = torch.empty(rows * far, dtype=torch.bfloat16, device="cuda").as_strided((rows, k), (far, 1))
    x.copy_(rows_of(rows, k, torch.bfloat16, 3).cuda())
    y = torch.empty(rows * far, dtype=torch.float16, device="cuda").as_strided((rows, n), (far, 1))
    for r in (1, 2, 20, rows):
        announce(f"far rows {r}")
        y.fill_(0)
        check(I, (codes, w[1], None), x, r, "far weights")
        check(I, w, x[rows - r:], r, "far x and y", y=y[rows - r:])
        check(I, (codes, w[1], None), x[rows - r:], r, "gated", gated=True, y=y[rows - r:, :n // 2])


@pytest.mark.parametrize("far", [False, True])
def test_the_most_rows(I, far):
    """2,097,120 rows, over weights side by side and over weight rows too far apart for a tile."""
    rows, n, k = 2097120, 8, 16
    w = make(n, k, 5)
    codes = torch.empty(n << 28, dtype=torch.int8, device="cuda").as_strided((n, k), (1 << 28, 1)) if far else w[0]
    codes.copy_(w[0].clone())
    x = torch.randn(rows, k, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    announce(f"most rows, far {far}")
    y = I.gemv(I.Weights(codes, w[1]), x, rows)
    q, sx = I.quantize_rows(x)
    S = (q.double() @ w[0].double().t()).float()
    assert torch.equal(y, S * sx[:, None] * w[1])
    with pytest.raises(I.SynError):
        I.gemv(I.Weights(codes, w[1]), torch.empty(rows + 1, k, device="cuda"), rows + 1)


@pytest.mark.parametrize("rows", [1, 6, 33, 256])
def test_codes_held_on_odd_bytes_are_laid_out_once(I, rows):
    k, n = 77, 50
    odd = make(n, k, 2)[0].contiguous()
    for codes in (odd, make(n, k + 3, 2)[0][:, 3:], odd.t().contiguous().t()):
        W = I.Weights(codes, torch.ones(n, device="cuda"))
        assert W.codes.stride(0) % 16 == 0 and W.codes.data_ptr() % 16 == 0 and (W.codes == codes).all()
    check(I, (odd, torch.ones(n, device="cuda"), None), rows_of(rows, k, torch.float32, 1).cuda(), rows, "odd codes")


@pytest.mark.parametrize("rows", [1, 9, 130])
def test_rows_quantized_once_for_several_matrices(I, rows):
    k = 1000
    x = rows_of(rows, k, torch.bfloat16, 4).cuda()
    ws = [make(n, k, n, bias=n == 96) for n in (512, 96, 1)]
    r = I.Rows(rows, k, 512, 96, 1)
    announce(f"quantize_into {rows}")
    I.quantize_into(x, r)
    for w in ws:
        W = I.Weights(*w)
        y = I.gemv_quantized(W, r, torch.empty(rows, W.n_out, device="cuda"))
        same(y, I.gemv(W, x, rows, dtype=torch.float32).cpu())


def test_a_row_does_not_depend_on_the_others(I):
    """One row alone, among few and among many: the same bits."""
    w = make(400, 1111, 1)
    W, x = I.Weights(*w), rows_of(300, 1111, torch.float32, 2).cuda()
    whole = I.gemv(W, x, 300)
    for rows in (1, 2, 3, 8, 16, 17, 32, 40, 64, 90, 128, 200):
        announce(f"alone and among {rows}")
        same(I.gemv(W, x[100:], rows), whole[100:100 + rows].cpu(), f"{rows}")


def test_refusals_on_the_device(I):
    """What is wrong with operands that are on the device; nothing is written."""
    W = I.Weights(*make(8, 64, 1))
    x, y = torch.ones(4, 64, device="cuda"), torch.full((4, 8), 7.0, device="cuda")
    for bad in (dict(x=x[:, :63]), dict(x=x.double()), dict(x=x.cpu()), dict(rows=5), dict(y=y[:3]), dict(y=y.int()),
                dict(y=y.bfloat16(), dtype=torch.float32), dict(dtype=torch.float64), dict(y=y[:, ::2]),
                dict(x=x[:1].expand(4, 64)), dict(y=y.cpu()), dict(ws=torch.empty(1 << 20, device="cuda"), rows=2),
                dict(ws=torch.empty(1 << 20, dtype=torch.uint8), rows=2), dict(rows=-1)):
        with pytest.raises(I.GemvError):
            I.gemv(W, **{**dict(x=x, rows=4, y=y if "dtype" not in bad else None), **bad})
    with pytest.raises(I.SynError):
        I.gemv(W, torch.ones(20, 64, device="cuda"), 20, y=torch.empty(20, 8, device="cuda"),
               ws=torch.empty(256, dtype=torch.uint8, device="cuda"))
    with pytest.raises(I.GemvError):
        I.gate_up_act(I.Weights(*make(9, 64, 1)), x, 4)
    for codes, scales in ((W.codes, W.scales[:7]), (W.codes, W.scales.double()), (W.codes.float(), W.scales),
                          (W.codes, W.scales.cpu()), (W.codes[0], W.scales)):
        with pytest.raises(I.GemvError):
            I.Weights(codes, scales)
    with pytest.raises(I.GemvError):
        I.Weights(torch.empty(1, 131073, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(AttributeError):
        W.codes = W.codes[:4]
    torch.cuda.synchronize()
    assert (y == 7.0).all()


def test_no_rows_and_no_outputs(I):
    W = I.Weights(*make(8, 64, 1))
    assert I.gemv(W, torch.empty(0, 64, device="cuda"), 0).shape == (0, 8)
    none = I.Weights(torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"))
    assert I.gemv(none, torch.ones(3, 64, device="cuda"), 3).shape == (3, 0)
    c, s = I.quantize_rows(torch.empty(0, 64, device="cuda"))
    assert c.shape == (0, 64) and s.shape == (0,)


def test_logits_over_an_int8_head(I):
    import syntropy_amd.gemv as S
    vocab, hidden, rows = 3001, 1024, 5
    g = (torch.rand(hidden) + 0.5).cuda()
    x = rows_of(rows, hidden, torch.float32, 1).cuda()
    head = I.Weights(*make(vocab, hidden, 9))
    announce("int8 logits")
    got = I.logits(head, g, 1e-5, x, rows)
    same(got, I.gemv(head, S.rms_norm(x, g, 1e-5, rows), rows).cpu())


@pytest.mark.parametrize("rows", [1, 6, 30, 100, 520])
def test_captured_and_replayed(I, rows):
    """A captured call follows its inputs at every replay, with eager calls of the same shape between."""
    n, k = 600, 2100
    w = make(2 * n, k, 3)
    W, G = I.Weights(w[0][:n], w[1][:n]), I.Weights(w[0], w[1])
    x = rows_of(rows, k, torch.float32, 1).cuda()
    y, h = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    I.gemv(W, x, rows, y=y), I.gate_up_act(G, x, rows, y=h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    announce(f"capture {rows} rows")
    with torch.cuda.graph(graph):
        I.gemv(W, x, rows, y=y)
        I.gate_up_act(G, x, rows, y=h)
    for i in range(3):
        x.copy_(rows_of(rows, k, torch.float32, 10 + i))
        want_y, want_h = I.gemv(W, x, rows), I.gate_up_act(G, x, rows)
        y.fill_(float("nan")), h.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        same(y, want_y.cpu()), same(h, want_h.cpu())


def test_on_other_streams_at_once(I):
    """Two streams at once, each with its own operands and workspace, by a stream object and by its handle."""
    n, k, rows = 2000, 4096, 150
    w = [make(n, k, i) for i in range(2)]
    W = [I.Weights(*v) for v in w]
    xs = [rows_of(rows, k, torch.bfloat16, 7 + i).cuda() for i in range(2)]
    want = [I.gemv(W[i], xs[i], rows).cpu() for i in range(2)]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    announce("two streams")
    got = [[], []]
    for _ in range(5):
        got[0].append(I.gemv(W[0], xs[0], rows, stream=st[0]))
        got[1].append(I.gemv(W[1], xs[1], rows, stream=st[1].cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            same(y, want[i])
