"""Rows to E4M3 codes (quantize_rows_fp8, rms_norm_fp8, add_rms_norm_fp8) and their products (linear_w8a8) against
float64.

Codes. quantize_rows_fp8 divides as a division rounds, so its codes and scales are those of quantize_fp8. A norm's
values carry a float32 sum of n squares, its root and four products, below d = (n + 32) * 2^-24 relative, and its scale
two more products: a code is off the quotient by at most half of E4M3's step there (2^-4 of its power of two, 2^-10
below 2^-6) and 2 d of the quotient, a scale by d.

Products. Of codes that are small integers, with scales that are powers of two, every sum is exact in float32 in any
order, and so is what a product without an activation returns. Of any codes, K float32 additions are off by at most
K * 2^-23 of the sum of magnitudes s (2^-23 covers an addition that truncates), scales, bias and row_add by 2^-23 each
of their partial results, below (K + 8) * 2^-23 * (s + |bias| + |row_add|) before the output's rounding (half a step:
2^-11 relative for float16, 2^-8 for bfloat16). The activations here have slopes of at most 1.2 (SwiGLU, silu(g) u: 1.2
|u| and |g|), and their own float32 evaluation is off by at most 64 steps of 2^-24 of their argument and result."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
E4M3 = torch.float8_e4m3fn


def rnd(*shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


# ------------------------------------------------------------------ rows


def rows64(y):
    """Scale and quotients of float64 rows."""
    top = y.abs().amax(-1)
    scale = torch.where(top > 0, (top / 448).clamp_min(2.0**-126), 1.0)
    return y / scale[..., None], scale


def check_codes(codes, scale, y, n):
    q, s = rows64(y)
    d = (n + 32) * 2.0**-24
    assert codes.dtype == E4M3 and codes.is_contiguous() and scale.dtype == torch.float32
    assert codes.shape == y.shape and scale.shape == y.shape[:-1]
    assert bool(((scale.double() - s).abs() <= d * s).all())
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0**-6))) - 3)
    assert bool(((codes.double() - q).abs() <= step / 2 + 2 * d * q.abs() + 1e-30).all())


def check_same_codes(codes, scale, x):
    """The codes and scales that quantize_fp8 gives the rows on the CPU, bit for bit."""
    import fused_decode as fd

    want, s = fd.quantize_fp8(x.float().cpu().reshape(-1, x.shape[-1]))
    assert torch.equal(codes.cpu().view(torch.uint8).reshape(want.shape), want.view(torch.uint8))
    assert torch.equal(scale.cpu().reshape(s.shape), s)


def norm64(t, w, eps):
    return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w.double()


# lanes of a row change after 64, 128, 256 and 512 elements, vectors of a lane after 1024, 2048, 4096, 8192, 16384
LENGTHS = [8, 9, 15, 64, 65, 100, 128, 129, 256, 257, 512, 513, 1025, 2049, 4096, 4097, 8191, 8193, 16384, 16385, 32767]
ODD = [1, 2, 7, 32769, 40001]  # the kernel for any strides


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", LENGTHS + ODD)
def test_rows_of_any_length_and_alignment(dtype, n):
    import fused_decode as fd

    eps, rows = 1e-5, 5
    for offset in (0, 1):
        buf = rnd(rows * (n + 3) + 1, seed=n, dtype=dtype, scale=3.0)
        x = buf[offset : offset + rows * (n + 3)].view(rows, n + 3)[:, :n]
        check_same_codes(*fd.quantize_rows_fp8(x), x)
        r = rnd(rows, n, seed=n + 1, dtype=dtype)
        for wdtype in (torch.float16, torch.bfloat16, torch.float32):
            w = rnd(n + 1, seed=n + 2, dtype=wdtype)[offset : offset + n]
            check_codes(*fd.rms_norm_fp8(x, w, eps), norm64(x.double(), w, eps), n)
            codes, scale, ro = fd.add_rms_norm_fp8(x, r, w, eps)
            total = x.double() + r.double()
            check_codes(codes, scale, norm64(total, w, eps), n)
            assert ro.dtype == dtype and torch.equal(ro, (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("rows", [1, 3, 1023, 1024, 1025, 4099])
@pytest.mark.parametrize("n", [40, 520, 1032, 2056, 4096])
def test_many_rows(rows, n):
    import fused_decode as fd

    x, r, w = (rnd(rows, n, seed=1, dtype=torch.bfloat16), rnd(rows, n, seed=2, dtype=torch.bfloat16),
               rnd(n, seed=3, dtype=torch.float32))
    check_same_codes(*fd.quantize_rows_fp8(x), x)
    check_codes(*fd.rms_norm_fp8(x, w), norm64(x.double(), w, 1e-6), n)
    before = r.clone()
    total = x.double() + r.double()
    codes, scale, ro = fd.add_rms_norm_fp8(x, r, w, residual_out=r)
    assert ro is r and torch.equal(r, (x.float() + before.float()).to(r.dtype))
    check_codes(codes, scale, norm64(total, w, 1e-6), n)
    codes2, scale2, _ = fd.add_rms_norm_fp8(x, before, w)
    assert torch.equal(codes2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scale2, scale)


def test_strides_and_leading_dims():
    """Views of a wider buffer, a column stride, a broadcast row, dims that do not merge, one dimension."""
    import fused_decode as fd

    base = rnd(3, 4, 5, 6, 80, seed=7, dtype=torch.float16)
    w = rnd(80, seed=8, dtype=torch.float16)
    views = [base, base.transpose(0, 1), base.permute(3, 1, 0, 2, 4), base[:, ::2, :, 1:, 3:67], base[..., ::2],
             base.transpose(-1, -2), base[0, 0, 0, 0], base[:1, :1, :1, :1].expand(3, 4, 5, 6, 80)]
    for x in views:
        n = x.shape[-1]
        check_same_codes(*fd.quantize_rows_fp8(x), x)
        wn = w[: n] if n <= 80 else w
        check_codes(*fd.rms_norm_fp8(x, wn, 1e-5), norm64(x.double(), wn, 1e-5), n)
        r = rnd(*x.shape, seed=9, dtype=torch.float16)
        out = torch.empty(x.shape, dtype=E4M3, device=DEV)
        so = torch.empty(x.shape[:-1], device=DEV)
        wide = torch.full((*x.shape[:-1], n + 2), 7.0, dtype=torch.float16, device=DEV)
        ro = wide[..., 1:-1]
        c, s, got = fd.add_rms_norm_fp8(x, r, wn, 1e-5, out=out, scale_out=so, residual_out=ro)
        assert c is out and s is so and got is ro
        check_codes(c, s, norm64(x.double() + r.double(), wn, 1e-5), n)
        assert torch.equal(ro, (x.float() + r.float()).half()) and bool((wide[..., [0, -1]] == 7).all())
    stepped = torch.ones(160, device=DEV)[::2]
    check_codes(*fd.rms_norm_fp8(base, stepped, 1e-5), norm64(base.double(), stepped, 1e-5), 80)


@pytest.mark.parametrize("n", [16, 600, 4096, 40000])
def test_rows_of_extreme_values(n):
    """Zeros, one value, the type's ends, infinities, NaN: each row by itself."""
    import fused_decode as fd

    for dtype in (torch.float16, torch.bfloat16):
        top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        x = rnd(9, n, seed=n, dtype=dtype)
        x[0], x[1], x[2], x[3], x[4] = 0, tiny, top, 0, -0.0
        x[3, n - 1] = -tiny
        x[5, n - 1], x[6, 0], x[7, n // 2] = math.inf, -math.inf, math.nan
        codes, scale = fd.quantize_rows_fp8(x)
        assert bool((codes[:1].float() == 0).all()) and float(scale[0]) == 1 and float(scale[4]) == 1
        assert bool(codes[5:8].float().isnan().all()) and bool(scale[5:8].isnan().all())
        assert bool((scale[:5] >= 2.0**-126).all()) and bool(scale[:5].isfinite().all())
        for i in (1, 2, 3, 8):  # a scale of 2^-126 keeps what 448 of it covers
            q, s = rows64(x[i].double())
            assert abs(float(scale[i].double() / s) - 1) <= 2.0**-23
            step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0**-6))) - 3)
            assert bool(((codes[i].double() - q).abs() <= step / 2 + 2.0**-22 * q.abs()).all())
        w = torch.ones(n, device=DEV)
        for c, s in (fd.rms_norm_fp8(x, w, 1e-5), fd.add_rms_norm_fp8(x, torch.zeros_like(x), w, 1e-5)[:2]):
            assert bool((c[0].float() == 0).all()) and float(s[0]) == 1
            assert bool(c[5:8].float().isnan().all()) and bool(s[5:8].isnan().all())
            check_codes(c[8:], s[8:], norm64(x[8:].double(), w, 1e-5), n)


def test_signs_of_zeros():
    """A negative zero, and what rounds to one, keep their sign."""
    import fused_decode as fd

    for n in (64, 40000):
        x = rnd(2, n, seed=n, dtype=torch.float16)
        x[:, ::3], x[:, 1::3] = -0.0, -torch.finfo(torch.float16).smallest_normal / 1024
        check_same_codes(*fd.quantize_rows_fp8(x), x)


def test_rows_of_no_element():
    import fused_decode as fd

    for shape in ((0, 16), (3, 0), (0,), (2, 0, 8)):
        x = torch.empty(shape, dtype=torch.float16, device=DEV)
        w = torch.ones(shape[-1], device=DEV)
        for c, s, *ro in (fd.quantize_rows_fp8(x), fd.rms_norm_fp8(x, w), fd.add_rms_norm_fp8(x, x.clone(), w)):
            assert c.shape == shape and s.shape == shape[:-1] and bool((s == 1).all())
            assert all(r.shape == shape and r.dtype == x.dtype for r in ro)


# ------------------------------------------------------------------ products


def small_codes(*shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g).float().to(E4M3).to(DEV)


def powers(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.exp2(torch.randint(-3, 4, (n,), generator=g).float()).to(DEV)


def exact_case(m, n, k, seed, dtype):
    """Codes, scales, a bias and an addend whose every partial result is exact in float32."""
    x, w = small_codes(m, k, seed=seed), small_codes(n, k, seed=seed + 1)
    xs, ws = powers(m, seed + 2), powers(n, seed + 3)
    g = torch.Generator().manual_seed(seed + 4)
    bias = torch.randint(-8, 9, (n,), generator=g).float().to(DEV)
    add = torch.randint(-8, 9, (m, n), generator=g).to(dtype).to(DEV)
    v = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    return x, xs, w, ws, bias, add, v


SIZES = [(1, 1, 1), (1, 16, 128), (1, 33, 4096), (2, 130, 272), (3, 4, 16), (7, 257, 1008), (13, 96, 2064), (16, 640, 512),
         (17, 128, 640), (31, 200, 144), (32, 1000, 1024), (33, 48, 96), (64, 127, 256), (65, 129, 128), (100, 384, 400),
         (128, 128, 8192), (129, 260, 160), (257, 255, 384), (300, 515, 48), (513, 769, 272)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SIZES + [(5, 40, 131), (70, 140, 1023), (130, 300, 257), (9, 24, 15), (1, 520, 4097),
                                           (20, 100, 2051), (3, 70, 8191), (40, 33, 8200), (12, 9, 17), (2, 300, 13)])
def test_products_of_small_integers_are_exact(m, n, k, dtype):
    import fused_decode as fd

    x, xs, w, ws, bias, add, v = exact_case(m, n, k, 11 * m + n + k, dtype)
    assert torch.equal(fd.linear_w8a8(x, xs, w, ws, dtype=dtype), v.to(dtype))
    full = v + bias.double()
    assert torch.equal(fd.linear_w8a8(x, xs, w, ws, bias, row_add=add, dtype=dtype), (full + add.double()).to(dtype))
    assert torch.equal(fd.linear_w8a8(x, xs, w, ws, bias.half(), activation="relu", dtype=dtype), full.clamp_min(0).to(dtype))
    # each row alone, and the rows in another order, are the same rows
    assert torch.equal(fd.linear_w8a8(x[m // 2], xs[m // 2], w, ws, dtype=dtype), v[m // 2].to(dtype))
    assert torch.equal(fd.linear_w8a8(x.flip(0), xs.flip(0), w, ws, dtype=dtype), v.flip(0).to(dtype))


@pytest.mark.parametrize("m,n,k,name", [(4000, 8200, 400, None), (4091, 16390, 272, "swiglu"), (4100, 8195, 129, "relu")])
def test_products_of_large_tiles(m, n, k, name):
    """Many rows and columns, neither a multiple of a tile, K no multiple of a step."""
    import fused_decode as fd

    x, xs, w, ws, bias, _, v = exact_case(m, n, k, m, torch.bfloat16)
    v = v + bias.double()
    if name == "swiglu":
        v, xs, bias = v * 2.0**-6, xs * 2.0**-6, bias * 2.0**-6  # sigmoids that are neither 0 nor 1
        ref = v[:, : n // 2] * torch.sigmoid(v[:, : n // 2]) * v[:, n // 2:]
        y = fd.linear_w8a8(x, xs, w, ws, bias, activation=name)
        # exact arguments: the sigmoid's own float32 evaluation (64 steps of 2^-24) and the output's rounding
        assert bool(((y.double() - ref).abs() <= (2.0**-18 + 2.0**-8) * ref.abs() + 1e-30).all())
    else:
        want = v.clamp_min(0) if name == "relu" else v
        assert torch.equal(fd.linear_w8a8(x, xs, w, ws, bias, activation=name), want.bfloat16())


def act64(v, name):
    if name == "relu":
        return v.clamp_min(0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))
    return v


def check_product(y, x, xs, w, ws, bias, name, add, dtype):
    k = x.shape[-1]
    a = x.double() * xs.double()[:, None]
    b = w.double() * ws.double()[:, None]
    v, s = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        v, s = v + bias.double(), s + bias.double().abs()
    tol = (k + 8) * 2.0**-23 * s
    if name == "swiglu":
        half = v.shape[1] // 2
        g, u, tg, tu = v[:, :half], v[:, half:], tol[:, :half], tol[:, half:]
        ref = g * torch.sigmoid(g) * u
        tol = 1.2 * tg * (u.abs() + tu) + (g.abs() + tg) * tu + 2.0**-18 * ((g.abs() + 1) * u.abs())
    else:
        ref = act64(v, name)
        tol = 1.2 * tol + (2.0**-18 * (ref.abs() + v.abs()) if name else 0)
    if add is not None:
        ref = ref + add.double()
        tol = tol + 2.0**-23 * ref.abs()
    assert y.dtype == dtype and y.shape == ref.shape
    floor = 2.0**-25 if dtype == torch.float16 else 0  # half of float16's smallest step
    if dtype == torch.float16:
        # float16 ends at 65504 in steps of 32: 65504 + 16 and more is infinite, and what may lie on either side of it
        # within the tolerance may be either
        over, under = ref.abs() - tol >= 65520, ref.abs() + tol < 65520
        assert bool((y[over].double() == ref[over].sign() * float("inf")).all())
        keep = under | ~y.isinf()
        y, ref, tol = y[keep & ~over], ref[keep & ~over], tol[keep & ~over]
    off = (y.double() - ref).abs() - (tol + HALF_STEP[dtype] * (ref.abs() + tol) + floor)
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("name", [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (5, 30, 1040), (16, 1026, 512), (33, 264, 384), (150, 402, 640),
                                   (300, 130, 77), (4, 62, 201)])
def test_activations(name, m, n, k):
    import fused_decode as fd

    for dtype, bdt, rdt in ((torch.float16, torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16, torch.float32)):
        x, xs = fd.quantize_rows_fp8(rnd(m, k, seed=m, dtype=dtype))
        w, ws = fd.quantize_fp8(rnd(n, k, seed=n, scale=2 * k**-0.5))
        bias, nout = rnd(n, seed=3, dtype=bdt), n // 2 if name == "swiglu" else n
        add = rnd(m, nout, seed=4, dtype=rdt)
        for b, r in ((None, None), (bias, None), (bias, add), (None, add)):
            y = fd.linear_w8a8(x, xs, w, ws, b, activation=name, row_add=r, dtype=dtype)
            check_product(y, x, xs, w, ws, b, name, r, dtype)


def test_activations_of_large_values():
    """Arguments far out on either side: no overflow on the way, and the limits."""
    import fused_decode as fd

    x, xs = torch.ones(3, 16, device=DEV).to(E4M3), torch.tensor([1.0, 1e3, 1e30], device=DEV)
    w, ws = torch.tensor([1.0, -1.0], device=DEV)[:, None].expand(2, 16).contiguous().to(E4M3), torch.ones(2, device=DEV)
    for name in ("relu", "silu", "gelu", "gelu_tanh"):
        y = fd.linear_w8a8(x, xs, w, ws, activation=name).float()
        assert bool((y[:, 0] > 0).all()) and bool((y[1:, 1] == 0).all()) and bool(y.isfinite().all())
        assert float(y[1, 0]) == float(torch.tensor(16e3).bfloat16())


def test_any_codes_and_nan():
    """Every code at every place of a step; a NaN code spoils its row or column and no other."""
    import fused_decode as fd

    k = 528
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    codes = codes[(codes & 0x7F) != 0x7F]
    w = codes.repeat(9)[: 4 * k].view(4, k).to(DEV).view(E4M3)
    for m in (3, 40):
        x, xs = fd.quantize_rows_fp8(rnd(m, k, seed=m, dtype=torch.float16))
        ws = torch.ones(4, device=DEV)
        check_product(fd.linear_w8a8(x, xs, w, ws), x, xs, w, ws, None, None, None, torch.bfloat16)
        bad = w.clone().view(torch.uint8)
        bad[2, k - 1] = 0x7F
        y = fd.linear_w8a8(x, xs, bad.view(E4M3), ws)
        assert bool(y[:, 2].isnan().all()) and not bool(y[:, [0, 1, 3]].isnan().any())
        xb = x.clone().view(torch.uint8)
        xb[1, 0] = 0xFF
        y = fd.linear_w8a8(xb.view(E4M3), xs, w, ws)
        assert bool(y[1].isnan().all()) and not bool(y[0].isnan().any()) and not bool(y[2:].isnan().any())


@pytest.mark.parametrize("m,n,k", [(6, 48, 160), (40, 200, 272), (150, 64, 1024)])
def test_strides_alignments_and_broadcasts(m, n, k):
    import fused_decode as fd

    x, xs, w, ws, bias, add, v = exact_case(m, n, k, m, torch.float16)
    want = (v + bias.double()).half()

    def placed(t, pitch, offset):
        buf = torch.zeros(t.shape[0] * pitch + offset + 64, dtype=torch.uint8, device=DEV)
        view = buf[offset:].as_strided(t.shape, (pitch, 1))
        view.copy_(t.view(torch.uint8))
        return view.view(E4M3)

    for pitch, offset in ((k + 16, 0), (k + 16, 16), (k + 1, 0), (k, 3), (k + 8, 8), (k + 5, 1)):
        xp, wp = placed(x, pitch, offset), placed(w, pitch, offset)
        assert torch.equal(fd.linear_w8a8(xp, xs, w, ws, bias, dtype=torch.float16), want)
        assert torch.equal(fd.linear_w8a8(x, xs, wp, ws, bias, dtype=torch.float16), want)
        assert torch.equal(fd.linear_w8a8(xp, xs, wp, ws, bias, dtype=torch.float16), want)
    xt = x.view(torch.uint8).t().contiguous().view(E4M3).t()
    wt = w.view(torch.uint8).t().contiguous().view(E4M3).t()
    b2, s2 = torch.stack((bias, bias), 1)[:, 0], torch.stack((ws, ws), 1)[:, 1]
    assert torch.equal(fd.linear_w8a8(xt, xs, wt, s2, b2, dtype=torch.float16), want)
    x3, xs3 = x.view(2, m // 2, k), xs.view(2, m // 2)
    flipped = fd.linear_w8a8(x3.transpose(0, 1), xs3.transpose(0, 1), w, ws, bias, dtype=torch.float16)
    assert torch.equal(flipped, want.view(2, m // 2, n).transpose(0, 1))
    for r in (add[:1], add[:, :1], add[0], add[:1, :1], add.float(), add.t().contiguous().t(), add[:, :1].bfloat16()):
        got = fd.linear_w8a8(x, xs, w, ws, bias, row_add=r, dtype=torch.float16)
        assert torch.equal(got, (v + bias.double() + r.double()).half())
    got = fd.linear_w8a8(x3, xs3, w, ws, row_add=add.view(2, m // 2, n)[:, :1], dtype=torch.float16)
    assert torch.equal(got, (v.view(2, m // 2, n) + add.double().view(2, m // 2, n)[:, :1]).half())


def test_output_given_or_over_an_operand():
    import fused_decode as fd

    for m, n, k in ((8, 64, 128), (200, 128, 256)):
        x, xs, w, ws, bias, add, v = exact_case(m, n, k, 5, torch.bfloat16)
        want = (v + add.double()).bfloat16()
        guard = torch.full((m + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
        out = guard[1:-1]
        assert fd.linear_w8a8(x, xs, w, ws, row_add=add, out=out) is out
        assert torch.equal(out, want) and bool((guard[[0, -1]] == 7).all())
        stream = add.clone()
        fd.linear_w8a8(x, xs, w, ws, row_add=stream, out=stream)  # the residual stream in place
        assert torch.equal(stream, want)
        half = torch.zeros(m * n, dtype=torch.bfloat16, device=DEV)
        half[:n] = bias.bfloat16()
        fd.linear_w8a8(x, xs, w, ws, half[:n], out=half.view(m, n))  # over its own bias
        assert torch.equal(half.view(m, n), (v + bias.double()).bfloat16())
        half.view(m, n).copy_(add)
        fd.linear_w8a8(x, xs, w, ws, row_add=half.view(m, n)[:1], out=half.view(m, n))  # over a broadcast addend
        assert torch.equal(half.view(m, n), (v + add[:1].double()).bfloat16())


def test_sizes_of_zero():
    import fused_decode as fd

    e = lambda *s: torch.empty(s, device=DEV).to(E4M3)
    f = lambda *s: torch.ones(s, device=DEV)
    assert fd.linear_w8a8(e(0, 32), f(0), e(8, 32), f(8)).shape == (0, 8)
    assert fd.linear_w8a8(e(3, 32), f(3), e(0, 32), f(0)).shape == (3, 0)
    assert fd.linear_w8a8(e(2, 0, 32), f(2, 0), e(8, 32), f(8), activation="swiglu").shape == (2, 0, 4)
    bias, add = rnd(8, seed=1), rnd(3, 8, seed=2)
    y = fd.linear_w8a8(e(3, 0), f(3), e(8, 0), f(8), bias, activation="relu", row_add=add)
    assert torch.equal(y, (bias.clamp_min(0) + add).bfloat16())
    assert bool((fd.linear_w8a8(e(3, 0), f(3), e(8, 0), f(8)) == 0).all())


# ------------------------------------------------------------------ together


def plain_mlp(h, nw, gu, sg, wd, sd, eps, dtype):
    """The MLP block in float64, quantised where the operators quantise."""
    def codes(y):
        q, s = rows64(y.double())
        return q.float().to(E4M3).double() * s[..., None]

    v = codes(norm64(h.double(), nw, eps)) @ (gu.double() * sg.double()[:, None]).t()
    g, u = v.chunk(2, -1)
    mid = (g * torch.sigmoid(g) * u).to(dtype)
    return codes(mid) @ (wd.double() * sd.double()[:, None]).t() + h.double()


def block(h, nw, gu, sg, wd, sd, eps):
    import fused_decode as fd

    c, s = fd.rms_norm_fp8(h, nw, eps)
    c, s = fd.quantize_rows_fp8(fd.linear_w8a8(c, s, gu, sg, activation="swiglu", dtype=h.dtype))
    return fd.linear_w8a8(c, s, wd, sd, row_add=h, dtype=h.dtype)


def block_inputs(m, h, i, seed, dtype):
    import fused_decode as fd

    gu, sg = fd.quantize_fp8(rnd(2 * i, h, seed=seed, scale=h**-0.5))
    wd, sd = fd.quantize_fp8(rnd(h, i, seed=seed + 1, scale=i**-0.5))
    return rnd(m, h, seed=seed + 2, dtype=dtype), 1 + rnd(h, seed=seed + 3, dtype=dtype, scale=0.1), gu, sg, wd, sd, 1e-5


@pytest.mark.parametrize("m", [1, 13, 47, 200])
def test_an_mlp_block(m):
    """Each operator within its own bound on what the one before it returned, and the block against float64. mid is
    rounded to float16 on both sides, and float32 sums next to a border fall on either side of it: mid, and with it its
    row's scale, may be one step (2^-10) off, so a quotient of the second quantisation q up to e = 2 * 2^-10 relative.
    Such a shift crosses a border between codes, a step apart, in e q / step of the cases, each worth step^2 <= 2^-3 q
    step: 2^-3 e q^2 = 2^-12 q^2 in the mean, 2^-6 of the norm of the down product, which is less than the result's
    (the residual is independent of it), besides the result's own rounding, 2^-11."""
    import fused_decode as fd

    h, nw, gu, sg, wd, sd, eps = args = block_inputs(m, 512, 1024, m, torch.float16)
    c, s = fd.rms_norm_fp8(h, nw, eps)
    check_codes(c, s, norm64(h.double(), nw, eps), 512)
    mid = fd.linear_w8a8(c, s, gu, sg, activation="swiglu", dtype=torch.float16)
    check_product(mid, c, s, gu, sg, None, "swiglu", None, torch.float16)
    c, s = fd.quantize_rows_fp8(mid)
    check_same_codes(c, s, mid)
    y = fd.linear_w8a8(c, s, wd, sd, row_add=h, dtype=torch.float16)
    check_product(y, c, s, wd, sd, None, None, h, torch.float16)
    assert torch.equal(block(*args), y)
    ref = plain_mlp(*args, torch.float16)
    assert float((y.double() - ref).norm() / ref.norm()) <= 2.0**-6 + 2.0**-11


@pytest.mark.parametrize("m", [1, 24, 150])
def test_captured_and_replayed(m):
    """A graph's replays, with new inputs and eager work between them, give what eager calls give, bit for bit; two graphs
    captured one after another do not share workspaces."""
    args = block_inputs(m, 768, 1536, m, torch.bfloat16)
    other = block_inputs(m, 768, 1536, m + 50, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(*args), block(*other)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in (args, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(*a))
        graphs.append(g)
    for seed in range(3):
        args[0].copy_(rnd(m, 768, seed=seed, dtype=torch.bfloat16))
        graphs[0].replay()
        graphs[1].replay()
        want, want2 = block(*args), block(*other)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_on_another_stream():
    """Calls follow torch's current stream; two streams at once have workspaces of their own."""
    args, other = block_inputs(120, 512, 4096, 1, torch.bfloat16), block_inputs(120, 512, 4096, 9, torch.bfloat16)
    want, want2 = block(*args), block(*other)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = block(*args)
        with torch.cuda.stream(s2):
            b = block(*other)
        s1.synchronize(), s2.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want2)


def test_custom_ops_and_gradients():
    """torch.ops.fused_decode.* compile whole; a wanted gradient is refused when it is asked for."""
    import fused_decode as fd

    x, w, r = (rnd(6, 256, seed=1, dtype=torch.float16), rnd(256, seed=2, dtype=torch.float16),
               rnd(6, 256, seed=3, dtype=torch.float16))
    q, qs = fd.quantize_fp8(rnd(64, 256, seed=4))

    def f(x, w, r, q, qs):
        c, s, ro = torch.ops.fused_decode.add_rms_norm_fp8(x, r, w, 1e-5)
        c2, s2 = torch.ops.fused_decode.quantize_rows_fp8(ro)
        c3, s3 = torch.ops.fused_decode.rms_norm_fp8(ro, w, 1e-5)
        lin = torch.ops.fused_decode.linear_w8a8
        return (lin(c, s, q, qs, None, "swiglu", None, torch.float16), lin(c2, s2, q, qs), lin(c3, s3, q, qs, None, "gelu"))

    want = f(x, w, r, q, qs)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(x, w, r, q, qs)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    eager = fd.linear_w8a8(*fd.add_rms_norm_fp8(x, r, w, 1e-5)[:2], q, qs, activation="swiglu", dtype=torch.float16)
    assert torch.equal(eager, want[0])
    bias = torch.zeros(64, device=DEV, requires_grad=True)
    c, s = fd.quantize_rows_fp8(x)
    y = fd.linear_w8a8(c, s, q, qs, bias)
    assert torch.equal(y.detach(), fd.linear_w8a8(c, s, q, qs))
    with pytest.raises(RuntimeError):
        y.float().sum().backward()
    out = torch.empty(6, 64, dtype=torch.float16, device=DEV)
    with torch.no_grad():
        assert fd.linear_w8a8(c, s, q, qs, bias, out=out) is out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ["relu", "silu", "gelu", "gelu_tanh", "swiglu"])
def test_activations_of_infinities(name, dtype):
    """A NaN stays one, an infinity gives the activation's limit: itself above, and below nothing but 0 or NaN."""
    import fused_decode as fd

    k, top = 32, 3e38
    bias = torch.tensor([top, -top, float("nan"), 0.0], device=DEV)
    x = torch.ones(2, k, device=DEV).to(E4M3)
    w = torch.tensor([1.0, -1.0, 0.0, 0.0], device=DEV)[:, None].expand(4, k).contiguous().to(E4M3)
    xs, ws = torch.full((2,), 2.0**60, device=DEV), torch.full((4,), 2.0**67, device=DEV)  # 2^132: past float32
    y = fd.linear_w8a8(x, xs, w, ws, bias, activation=None if name == "swiglu" else name, dtype=dtype)
    if name != "swiglu":
        assert bool((y[:, 0] == float("inf")).all()) and bool(y[:, 2].isnan().all()) and bool((y[:, 3] == 0).all())
        assert bool(((y[:, 1] == 0) | y[:, 1].isnan()).all())
    half = torch.tensor([0.0, 0.0, 2.0, 1.0], device=DEV)
    gate_up = fd.linear_w8a8(x, xs, w, ws, half, activation="swiglu", dtype=dtype)
    assert bool((gate_up[:, 0] == float("inf")).all())


def test_more_rows_than_one_launch_takes():
    """Rows past the 2^32 threads of a launch, at a workgroup a row: the last ones are computed like any others."""
    import fused_decode as fd

    rows, n = 2**24 + 1000, 4
    x = torch.ones(rows, n, dtype=torch.float16, device=DEV)
    x[-2000:] = rnd(2000, n, seed=1, dtype=torch.float16)
    codes, scale = fd.quantize_rows_fp8(x)
    check_same_codes(codes[-2000:], scale[-2000:], x[-2000:])
    assert bool((codes[:-2000].view(torch.uint8) == 0x7E).all())  # 448
    assert torch.equal(scale[:-2000], scale[:1].expand(rows - 2000))


def test_a_negation_still_to_be_made():
    import fused_decode as fd

    x, w = rnd(5, 64, seed=1, dtype=torch.float16), rnd(64, seed=2)
    for got, want in ((fd.quantize_rows_fp8(torch._neg_view(x)), fd.quantize_rows_fp8(-x)),
                      (fd.rms_norm_fp8(x, torch._neg_view(w)), fd.rms_norm_fp8(x, -w)),
                      (fd.add_rms_norm_fp8(x, torch._neg_view(x), w), fd.add_rms_norm_fp8(x, -x, w))):
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    c, s = fd.quantize_rows_fp8(x)
    assert torch.equal(fd.linear_w8a8(c, s, c, s, torch._neg_view(s)), fd.linear_w8a8(c, s, c, s, -s))


@pytest.mark.parametrize("n,k", [(1, 16), (2, 17), (3, 1024), (9, 1040), (130, 4096), (257, 4100), (40, 8191), (33, 8192),
                                 (6145, 4097), (20, 33000), (4, 140001), (28, 9 * 1024)])
def test_one_row(n, k):
    """One row's own kernel: rows of any pitch and address, chunks of K that end anywhere, an odd number of outputs,
    with and without its epilogue. Integer codes and powers of two: exact in any order."""
    import fused_decode as fd

    f16, bf16 = torch.float16, torch.bfloat16
    for dtype, bdt, rdt in ((f16, f16, bf16), (bf16, bf16, torch.float32)):
        for offset, pitch in ((0, (k + 15) // 16 * 16), (1, k), (16, k + 7)):
            x, w = small_codes(1, k, seed=n), small_codes(2 * n, k, seed=k)
            buf = torch.zeros(offset + 2 * n * pitch + 16, dtype=torch.uint8, device=DEV).view(E4M3)
            wp = buf[offset : offset + 2 * n * pitch].view(2 * n, pitch)[:, :k]
            wp.copy_(w)
            xp = torch.zeros(offset + k, dtype=torch.uint8, device=DEV).view(E4M3)[offset:].view(1, k)
            xp.copy_(x)
            xs, ws = powers(1, seed=3), powers(2 * n, seed=4)
            bias, row = small_codes(2 * n, seed=5).to(bdt), small_codes(1, n, seed=6).to(rdt)
            sums = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
            assert torch.equal(fd.linear_w8a8(xp, xs, wp, ws, dtype=dtype), sums.to(dtype))
            v = sums + bias.double()
            y = fd.linear_w8a8(xp[:1], xs, wp[:n], ws[:n], bias[:n], row_add=row, activation="relu", dtype=dtype)
            assert torch.equal(y, (v[:, :n].clamp_min(0) + row.double()).float().to(dtype))
            y = fd.linear_w8a8(xp, xs, wp, ws, bias, activation="swiglu", row_add=row, dtype=dtype)
            check_product(y, x, xs, w, ws, bias, "swiglu", row, dtype)


def test_captured_as_the_first_call():
    """A capture that also makes the launch plans: nothing of them belongs to the graph, whose replays and the eager
    calls after it agree, before and after the graph is gone."""
    import fused_decode as fd
    from fused_decode import ops

    ops.clear_plans()
    x, w = rnd(90, 2048, seed=1, dtype=torch.bfloat16), rnd(2048, seed=2)
    q, qs = fd.quantize_fp8(rnd(600, 2048, seed=3))
    odd, odds = fd.quantize_fp8(rnd(70, 2047, seed=4))

    def run():
        c, s, h = fd.add_rms_norm_fp8(x, x, w)
        d, t = fd.quantize_rows_fp8(h[:, 1:])
        return (fd.linear_w8a8(c, s, q, qs, activation="silu"), fd.linear_w8a8(c[:1], s[:1], q, qs),
                fd.linear_w8a8(c[:9], s[:9], q, qs), fd.linear_w8a8(d, t, odd, odds))

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    kept = [t.clone() for t in got]
    del got, graph
    assert all(torch.equal(a, b) for a, b in zip(kept, run()))
