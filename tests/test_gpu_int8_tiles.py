"""Every form of the int8 products' kernels: CASES holds odd sizes for which the package chooses each tile, with K
in one part and in several, and each kernel of few rows, gated or not (test_int8_launches.py holds that they do).
Whole outputs against the definition, computed on the device: the codes of quantize_rows (held elsewhere against numpy),
sums in 64-bit floats, whole numbers below 2^53 and so exact, then the F32 steps; gated outputs against 64 bits within
2^-21 of silu, the product's step and the type's."""
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # a second rounding, to the type
LEAST = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}

# gated, outputs, values of K, rows
CASES = [
    # few rows: quantized in the product's workgroups, a piece a lane and several; before it; in groups of 16
    (0, 301, 500, 1), (0, 701, 9001, 1), (0, 37, 20003, 1), (0, 301, 900, 3), (0, 701, 3901, 3), (0, 301, 5001, 7),
    (0, 101, 701, 13), (1, 301, 500, 1), (1, 351, 9001, 1), (1, 151, 5001, 7), (1, 101, 701, 13),
    # 64 x 32, K over four wavefronts
    (0, 67, 103, 21), (0, 61, 3753, 21), (1, 67, 103, 21), (1, 61, 3753, 21),
    # 64 x 64, K over four
    (0, 8279, 102, 37), (0, 1237, 6507, 33), (1, 5713, 116, 33), (1, 613, 7606, 33), (0, 1001, 8201, 101),
    # 64 x 128, K over two
    (0, 6187, 104, 79), (0, 1391, 8412, 69), (1, 3425, 101, 75), (1, 685, 8137, 85), (0, 4101, 8195, 101),
    # 128 x 128, K over two
    (0, 5519, 5247, 329), (0, 1833, 13806, 525), (1, 5443, 5355, 137), (1, 1773, 13063, 273),
    # 128 x 128
    (0, 8211, 298, 195), (0, 8203, 11364, 67), (1, 8367, 365, 71), (1, 4821, 11756, 73),
    # 128 x 256
    (0, 8677, 532, 695), (0, 8561, 10232, 147), (1, 1941, 537, 1575), (1, 2977, 12878, 139), (0, 5003, 2051, 1001),
    # 256 x 128
    (0, 3623, 823, 2155), (0, 3689, 12330, 513), (1, 6323, 785, 517), (1, 8203, 11364, 67),
    # 256 x 256
    (0, 8469, 259, 1455), (0, 8391, 10539, 497), (1, 7365, 267, 771), (1, 8943, 8378, 137), (0, 2501, 1027, 4097),
]


@pytest.fixture(scope="module")
def I():
    require_gpu()
    import syntropy_amd.int8 as I
    return I


def operands(n, k, rows, dtype, bias, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(-128, 128, (n, -(-k // 16) * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    scales = (0.5 + torch.rand(n, generator=g, device="cuda")) * (3.0 / (74 * k ** 0.5))  # outputs of a few units
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    x = torch.randn(rows, k, generator=g, device="cuda")
    return codes, scales, b, x.to(dtype)


def definition(I, codes, scales, bias, x):
    q, s = I.quantize_rows(x)
    v = (q.double() @ codes.double().t().contiguous()).float() * s[:, None] * scales
    return v if bias is None else v + bias


def hold(got, v, gated, what):
    t = got.dtype
    if not gated:
        wrong = (got != v.to(t)).nonzero()
        assert len(wrong) == 0, f"{what}: {len(wrong)} of {got.numel()} differ, first at {wrong[0].tolist()}"
        return
    n = got.shape[1]
    g, u = v[:, :n].double(), v[:, n:].double()
    s = g / (1 + torch.exp(-g))
    want = s * u
    tol = (8 * U * s.abs() + 2.0 ** -150) * u.abs() * (1 + 2 * U) + U * want.abs() + 2.0 ** -150
    tol = tol * (1 + HALF[t]) + HALF[t] * want.abs() + LEAST[t]
    wrong = (~((got.double() - want).abs() <= tol)).nonzero()
    assert len(wrong) == 0, f"{what}: {len(wrong)} of {got.numel()} out of tolerance, first at {wrong[0].tolist()}"


@pytest.mark.parametrize("gated,n,k,rows", CASES)
def test_each_form_is_its_definition(I, gated, n, k, rows):
    for j, t in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        what = f"int8 {'gate_up' if gated else 'gemv'} {n}x{k} rows {rows} {t}"
        announce(what)
        codes, scales, b, x = operands((1 + gated) * n, k, rows, t, j == 1, n + k + rows + j)
        out = torch.full((rows + 2, n + 5), 7.0, dtype=t, device="cuda")  # rows at odd addresses, others around them
        y = out[1:rows + 1, 3:n + 3]
        (I.gate_up_act if gated else I.gemv)(I.Weights(codes, scales, b), x, rows, y=y)
        hold(y, definition(I, codes, scales, b, x), gated, what)
        y.fill_(7.0)
        assert (out == 7.0).all(), f"{what}: values around y changed"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(257, 5001), (301, 9001), (270, 20003)])
def test_quantize_many_long_rows(I, dtype, rows, k):
    """Rows on 256 threads in four and eight pieces a lane, and longer than the registers hold."""
    x = operands(1, k, rows, dtype, False, k)[3]
    x[5, k - 1], x[7, k - 2], x[9] = float("nan"), 60000.0, 0
    announce(f"quantize_rows {rows}x{k} {dtype}")
    codes, scales = I.quantize_rows(x)
    v = x.float()
    most = v.abs().amax(1)
    s = most / torch.full_like(most, 127.0)  # (a division by a number would be a product with its inverse)
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    want = torch.round(v * inv[:, None])
    want[5] = 0
    assert torch.equal(codes.float(), want)
    assert torch.equal(scales.nan_to_num(-1.0), s.nan_to_num(-1.0)) and scales[5].isnan()


@pytest.mark.parametrize("n,k,rows", [(1237, 6507, 33), (61, 3753, 21)])
def test_rows_quantized_for_smaller_matrices(I, n, k, rows):
    """A workspace without room for the parts of K, and with room for some of them: the same values."""
    codes, scales, b, x = operands(n, k, rows, torch.bfloat16, True, 4)
    W, want = I.Weights(codes, scales, b), None
    for others in ((1,), (n // 3,), (n,)):
        r = I.Rows(rows, k, *others)
        announce(f"rows quantized for {others}, product of {n}")
        I.quantize_into(x, r)
        y = I.gemv_quantized(W, r, torch.empty(rows, n, device="cuda"))
        want = definition(I, codes, scales, b, x) if want is None else want
        hold(y, want, False, f"rows for {others}")
