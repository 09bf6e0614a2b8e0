"""Products of E4M3 codes in every kernel and form that linear_w8a8 takes, chosen by size and checked against its query.

Codes are small integers, scales powers of two: sums are exact in float32 in any order, so outputs without an activation
are compared bit for bit. Where there is one its argument is exact, and it is off by at most 64 steps of 2^-24 of argument
and result (SwiGLU: of (|g| + 1) |u|) besides the output's rounding, half a step."""

from __future__ import annotations

import ctypes

import pytest
import torch

DEV = "cuda"
E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
ACT = 2.0**-18


def form(m, n, k):
    from fused_decode import _lib as L

    out = (ctypes.c_int * 4)()
    assert L.lib().fd_linear_w8a8_form(m, n, k, out) == L.FD_OK
    return tuple(out)


# rows, weight rows (even; products without SwiGLU take one less too), K, tile, K splits: more stages than a ring holds
# and fewer, a last stage that is short, halves that are odd or whole vectors, more row blocks than a group of them
TILES = [
    (133, 66, 2064, (64, 64), 1), (301, 2602, 1600, (64, 64), 1), (401, 130, 8208, (64, 64), 10),
    (501, 4002, 1040, (64, 128), 1), (257, 4098, 272, (64, 128), 1), (401, 66, 40016, (64, 128), 32),
    (91, 66, 1040, (128, 32), 1), (91, 66, 272, (128, 32), 1), (601, 1502, 144, (128, 32), 1), (91, 66, 6032, (128, 32), 8),
    (91, 128, 6032, (128, 32), 8), (257, 6002, 2064, (128, 128), 1), (133, 8202, 272, (128, 128), 1),
    (257, 2002, 8208, (128, 128), 5), (257, 2000, 8208, (128, 128), 5), (779, 5006, 2064, (256, 128), 1),
    (401, 8202, 48, (256, 128), 1), (779, 5006, 16, (256, 128), 1), (401, 4098, 6032, (256, 128), 3),
    (1003, 8202, 1040, (256, 256), 1), (779, 10006, 272, (256, 256), 1), (779, 5006, 14352, (256, 256), 3),
]

# 2 to 32 rows: both sides of where the kept steps change, one tile a workgroup and several with a short last one, a K
# that not every wave has a step of, and more outputs than the workgroups of one round hold
FEW = [(m, 9002, k) for m in (2, 16) for k in (4096, 4112, 8192, 8208, 16384)]
FEW += [(m, 9002, k) for m in (17, 32) for k in (4096, 4112, 8192)]
FEW += [(13, 28672, 4096), (16, 16396, 512), (16, 4096, 14336), (31, 9002, 272), (3, 70002, 256), (24, 70002, 144), (5, 300, 16),
        (32, 514, 8192)]


class Case:
    """Operands, and the exact float64 values before an activation."""

    def __init__(self, m, n, k, seed, dtype):
        g = torch.Generator(device=DEV).manual_seed(seed)
        ints = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, device=DEV)
        self.x, self.w = ints(-2, 3, m, k).to(torch.float16).to(E4M3), ints(-2, 3, n, k).to(torch.float16).to(E4M3)
        self.xs, self.ws = ints(-3, 4, m).float().exp2(), ints(-3, 4, n).float().exp2()
        self.bias, self.add = ints(-8, 9, n).float(), ints(-8, 9, m, n).to(dtype)
        self.v = torch.empty(m, n, dtype=torch.float64, device=DEV)
        for i in range(0, n, 4096):  # (a strip of the weights in float64 at a time)
            self.v[:, i : i + 4096] = self.x.double() @ self.w[i : i + 4096].double().t().contiguous()
        self.v *= self.xs.double()[:, None] * self.ws.double()


def check_exact(c, n, dtype):
    """The first n weight rows: alone, with everything exact in the epilogue, and into a buffer with rows around it."""
    import fused_decode as fd

    m = c.x.shape[0]
    w, ws, bias, add, v = c.w[:n], c.ws[:n], c.bias[:n], c.add[:, :n], c.v[:, :n]
    assert torch.equal(fd.linear_w8a8(c.x, c.xs, w, ws, dtype=dtype), v.to(dtype))
    full = v + bias.double()
    guard = torch.full((m + 2, n), 7.0, dtype=dtype, device=DEV)
    y = fd.linear_w8a8(c.x, c.xs, w, ws, bias, row_add=add, out=guard[1:-1])
    assert torch.equal(y, (full + add.double()).to(dtype)) and bool((guard[[0, -1]] == 7).all())
    for row in (add.float(), add[:, :1], add[:1].float()):
        y = fd.linear_w8a8(c.x, c.xs, w, ws, bias.to(dtype), activation="relu", row_add=row, dtype=dtype)
        assert torch.equal(y, (full.clamp_min(0) + row.double()).to(dtype))
    y = add.clone(memory_format=torch.contiguous_format)
    assert torch.equal(fd.linear_w8a8(c.x, c.xs, w, ws, row_add=y, out=y), (v + add.double()).to(dtype))


def check_activations(c, n, dtype):
    """Arguments times 2^-6, at which the activations are neither 0 nor the identity; SwiGLU over all rows."""
    import fused_decode as fd

    xs, bias, add = c.xs * 2.0**-6, c.bias * 2.0**-6, c.add

    def near(y, ref, tol):
        tol = tol + 2.0**-24 * ref.abs()  # the addition
        ref, y = ref.clamp(-65472, 65472), y.double().clamp(-65472, 65472)  # below float16's end
        floor = 2.0**-25 if dtype == torch.float16 else 0.0  # half its smallest step
        off = (y - ref).abs() - (tol + HALF_STEP[dtype] * (ref.abs() + tol) + floor)
        assert bool((off <= 0).all()), float(off.max())

    v = (c.v * 2.0**-6 + bias.double())[:, :n]
    for name, want in (("silu", v * torch.sigmoid(v)),
                       ("gelu", 0.5 * v * torch.special.erfc(-v * 0.5**0.5)),
                       ("gelu_tanh", v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v**3)))):
        y = fd.linear_w8a8(c.x, xs, c.w[:n], c.ws[:n], bias[:n], activation=name, row_add=add[:, :n], dtype=dtype)
        near(y, want + add[:, :n].double(), ACT * (want.abs() + v.abs()))
    half = c.w.shape[0] // 2
    full = c.v * 2.0**-6 + bias.double()
    gate, up = full[:, :half], full[:, half:]
    want = gate * torch.sigmoid(gate) * up
    tol = ACT * (gate.abs() + 1) * up.abs()
    near(fd.linear_w8a8(c.x, xs, c.w, c.ws, bias, activation="swiglu", dtype=dtype), want, tol)
    row = add[:, half:].float()
    near(fd.linear_w8a8(c.x, xs, c.w, c.ws, bias, activation="swiglu", row_add=row, dtype=dtype), want + row.double(), tol)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,tile,splits", TILES)
def test_tiles(m, n, k, tile, splits):
    assert form(m, n, k) == form(m, n - 1, k) == (4, *tile, splits)
    dtype = torch.float16 if (m + k // 16) % 2 else torch.bfloat16
    c = Case(m, n, k, m + n + k, dtype)
    check_exact(c, n, dtype)
    check_exact(c, n - 1, dtype)
    check_activations(c, n - 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", FEW)
def test_few_rows(m, n, k):
    assert form(m, n, k)[0] == 3
    dtype = torch.float16 if (m + k // 16) % 2 else torch.bfloat16
    c = Case(m, n, k, m + n + k, dtype)
    check_exact(c, n, dtype)
    check_exact(c, n - 1, dtype)
    check_activations(c, n - 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(401, 8202, 2051), (91, 66, 6031), (257, 2002, 8193), (24, 9002, 1001), (9, 9002, 8195)])
def test_rows_that_are_copied_first(m, n, k):
    """K of no whole pieces, at forms whose scratch holds the copies and the splits' sums one after the other."""
    c = Case(m, n, k, m + n + k, torch.bfloat16)
    check_exact(c, n - 1, torch.bfloat16)
    check_activations(c, n - 1, torch.bfloat16)
