"""mxfa_rmsnorm_quantize on the GPU: h bit for bit, codes and scales against rule R1 applied to y in 64 bits, with
what fp32 arithmetic can move (kv4ref.norm_delta) and no more."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4ref as R  # noqa: E402
import mxfa  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(codes, scales, y, delta, gemm):
    """Each code lies between those of y (1 - delta) and y (1 + delta) under the block's scale, which is one of those
    of the block's largest |y| moved alike."""
    rows, cols = y.shape
    sc = scales.cpu().numpy().astype(int)
    sc = (sc.T if gemm else sc.reshape(rows, -1)) - 127
    got = codes.view(torch.float8_e4m3fn).float().cpu().numpy().astype(np.float64).reshape(rows, -1, 32)
    b = y.reshape(rows, -1, 32)
    amax = np.abs(b).max(-1)
    # (rule R1 takes floor(log2) from a float logarithm: within 44 ulps below a power of two it is the next)
    lo, hi = R.r1_scale(amax * (1 - delta)), R.r1_scale(amax * (1 + delta + 44 * 2.0 ** -23))
    assert np.all((sc >= lo) & (sc <= hi))
    z = np.ldexp(np.abs(b), -sc[..., None])
    a, c = R.r1_round(z * (1 - delta)), R.r1_round(z * (1 + delta + 2.0 ** -22))
    g = np.abs(got)
    assert np.all((g >= a) & (g <= c)), (g[(g < a) | (g > c)][:4], a[(g < a) | (g > c)][:4])
    assert np.all((got == 0) | (np.sign(got) == np.sign(b)))
    # where nothing is near a boundary, which is nearly everywhere, that pins the code
    assert (a != c).mean() < 0.01 + 40 * delta


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,residual,offset,gemm", [
    (1, 32, False, 0.0, False), (1, 64, True, 0.0, True), (3, 4096, True, 0.0, True), (17, 2048, True, 1.0, False),
    (5, 8192, False, 1.0, True), (2, 8224, True, 0.0, False), (3, 20000 // 32 * 32, True, 0.0, True), (130, 160, True, 0.0, True),
    (64, 512, False, 0.0, True),
])
def test_norm(rows, cols, residual, offset, gemm, dtype):
    print(f"norm {rows} x {cols} residual {residual} offset {offset} gemm {gemm} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn((rows, cols), generator=g) * torch.exp(torch.randn((rows, 1), generator=g) * 3)
    x[:, ::97] *= 30.0
    x, r = x.to(dtype), torch.randn((rows, cols), generator=g).to(dtype)
    w = (1 - offset + 0.3 * torch.randn((cols,), generator=g)).to(dtype)
    if rows > 2:
        x[1], r[1] = 0.0, 0.0                                     # a row of zeros
    codes, scales, h = mxfa.rmsnorm_quantize(x.to(DEV), w.to(DEV), eps=1e-5, residual=r.to(DEV) if residual else None,
                                             weight_offset=offset, gemm_scales=gemm)
    y, want_h = R.norm(x, w, 1e-5, residual=r if residual else None, offset=offset)
    if dtype is torch.float32 and residual:
        want_h = x + r                                            # one fp32 rounding of the sum
    assert torch.equal(h.cpu(), want_h)
    assert codes.shape == x.shape and scales.shape == ((cols // 32, rows) if gemm else (rows, cols // 32))
    _check(codes, scales, y, R.norm_delta(cols), gemm)


def test_norm_of_extreme_rows():
    """Rows near both ends of fp32 whose squares stay inside it, and rows with NaN or infinities: those give the
    codes that mxfa_quantize_rows gives NaN (0), and leave the others alone."""
    cols = 256
    g = torch.Generator().manual_seed(9)
    x = torch.randn((6, cols), generator=g)
    x[0] *= 1e17
    x[1] *= 1e-17
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    w = torch.ones(cols)
    codes, scales, _ = mxfa.rmsnorm_quantize(x.to(DEV), w.to(DEV), eps=0.0)
    y, _ = R.norm(x, w, 0.0)
    for i in (0, 1, 2, 5):
        _check(codes[i:i + 1], scales[i:i + 1], y[i:i + 1], R.norm_delta(cols), False)
    assert not bool(codes[3].any()) and not bool(scales[3].any())
    assert not bool((codes[4] & 0x7f).any()) and not bool(scales[4].any())


@pytest.mark.parametrize("cols", [512, 9600])
def test_norm_in_place_and_shapes(cols):
    """h in the residual's or x's place, leading axes, and codes that mxfa_gemm takes."""
    g = torch.Generator(device=DEV).manual_seed(11)
    x, r = (torch.randn((2, 8, cols), generator=g, device=DEV).bfloat16() for _ in range(2))
    w = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
    codes, scales, h = mxfa.rmsnorm_quantize(x, w, residual=r)
    assert scales.shape == (2, 8, cols // 32)
    for where in ("residual", "x"):
        x1, r1 = x.clone(), r.clone()
        t = r1 if where == "residual" else x1
        c1, s1, h1 = mxfa.rmsnorm_quantize(x1, w, residual=r1, h=t)
        assert h1 is t and torch.equal(t, h) and torch.equal(c1, codes) and torch.equal(s1, scales)
    c2, s2, h2 = mxfa.rmsnorm_quantize(x.view(16, cols), w, residual=r.view(16, cols), gemm_scales=True)
    assert torch.equal(c2.view_as(codes), codes) and torch.equal(s2.t().contiguous().view_as(scales), scales)
    c3, s3, h3 = mxfa.rmsnorm_quantize(h, w)
    assert h3 is h and torch.equal(c3, codes) and torch.equal(s3, scales)
    copy = torch.empty_like(h)
    mxfa.rmsnorm_quantize(h, w, h=copy)
    assert torch.equal(copy, h)


def test_norm_codes_are_those_of_quantize_rows():
    """With a weight and rows that make y a power-of-two multiple of x, the codes are quantize_rows' of x."""
    x = torch.randn((8, 256), device=DEV)
    x = x / x.square().mean(-1, keepdim=True).sqrt()
    codes, scales, _ = mxfa.rmsnorm_quantize(x, torch.ones(256, device=DEV), eps=0.0)
    want_c, want_s = mxfa.quantize_rows(x)
    assert (codes != want_c).float().mean() < 2e-3 and torch.equal(scales, want_s)


def test_norm_scale_stride_leaves_other_columns():
    """scale_stride beyond the rows (a GEMM whose m is padded): only the rows' own scales are written."""
    x = torch.randn((5, 64), device=DEV)
    w = torch.ones(64, device=DEV)
    codes = torch.full((16, 64), 9, dtype=torch.uint8, device=DEV)
    scales = torch.full((2, 16), 9, dtype=torch.uint8, device=DEV)
    p = mxfa.NormParams(5, 64, mxfa.C_F32, 1e-6, 0.0, 16)
    assert mxfa.lib().mxfa_rmsnorm_quantize(p, x.data_ptr(), None, w.data_ptr(), None, codes.data_ptr(), scales.data_ptr(),
                                            torch.cuda.current_stream().cuda_stream) == 0
    want_c, want_s, _ = mxfa.rmsnorm_quantize(x, w, gemm_scales=True)
    assert torch.equal(codes[:5], want_c) and torch.equal(scales[:, :5], want_s)
    assert bool((codes[5:] == 9).all()) and bool((scales[:, 5:] == 9).all())


def test_norm_refusals():
    x = torch.zeros((4, 64), device=DEV)
    w = torch.ones(64, device=DEV)
    for f in (lambda: mxfa.rmsnorm_quantize(x.cpu(), w), lambda: mxfa.rmsnorm_quantize(x.half(), w.half()),
              lambda: mxfa.rmsnorm_quantize(x, w.bfloat16()), lambda: mxfa.rmsnorm_quantize(x, w[:32]),
              lambda: mxfa.rmsnorm_quantize(x[:, :48], w), lambda: mxfa.rmsnorm_quantize(x[:, :32], w[:32]),
              lambda: mxfa.rmsnorm_quantize(x, w, residual=x[:2]), lambda: mxfa.rmsnorm_quantize(x, w, residual=x.bfloat16()),
              lambda: mxfa.rmsnorm_quantize(x, w, residual=x, h=torch.zeros((4, 32), device=DEV)),
              lambda: mxfa.rmsnorm_quantize(x, w, eps=-1.0), lambda: mxfa.rmsnorm_quantize(x, w, weight_offset=float("nan"))):
        with pytest.raises(mxfa.MxfaError):
            f()
    codes, scales, h = mxfa.rmsnorm_quantize(x[:0], w, gemm_scales=True)
    assert codes.shape == (0, 64) and scales.shape == (2, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_just_below_a_power_of_two(dtype):
    """y = 4 (1 - 5e-9) lies below 4, though nearest to it in 32 bits: the block's scale is that of the values from 2 on,
    2^(1 - 8), under which y saturates at 448.  And y = 17/16 (1 - 5e-9), just below a tie of two codes, takes the
    lower one."""
    w = torch.full((128,), 4.0, dtype=dtype, device=DEV)
    w[64:] = 17 / 16
    codes, scales, _ = mxfa.rmsnorm_quantize(torch.ones((3, 128), dtype=dtype, device=DEV), w, eps=1e-8)
    assert scales.cpu().tolist() == [[120, 120, 119, 119]] * 3
    got = codes.view(torch.float8_e4m3fn).float().cpu()
    assert bool((got[:, :64] == 448).all()) and bool((got[:, 64:] == 256).all())
