"""Every tile of the linears for many rows, against the 64-bit definition: with 4- and 8-bit activations, one weight and two,
K whole and split, ending inside an instruction and with it, rows and columns past the last full tile.

Operands are any codes; what lies between their rows is NaN, or the largest element.  The launch's name tells the tile.
"""

from __future__ import annotations

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd import _lib
from qpu_xla_amd.kernels import mxfp4_gated_gemm, mxfp4_gemm

pytestmark = pytest.mark.gpu

# (format of the activations, weights, tile, K is split, [(rows, columns, K)])
CASES = [
    ("mxfp4", 1, "256x256", False, [(649, 16816, 672), (386, 24899, 1056), (388, 25349, 1152), (385, 24665, 3200)]),
    ("mxfp4", 1, "256x256", True, [(387, 9480, 20000)]),
    ("mxfp4", 1, "128x128", False, [(194, 12335, 672), (193, 12555, 640)]),
    ("mxfp4", 1, "128x128", True, [(2185, 261, 12320), (2209, 264, 12416)]),
    ("mxfp4", 1, "128x64", False, [(134, 16819, 1056), (131, 17073, 1152)]),
    ("mxfp4", 1, "128x64", True, [(65, 8279, 8224), (1835, 321, 12416)]),
    ("mxfp4", 1, "64x64", False, [(17, 33, 672), (17, 32, 640)]),
    ("mxfp4", 1, "64x64", True, [(17, 33, 1696), (20, 32, 3200)]),
    ("mxfp4", 1, "128x32", False, [(65, 17173, 3104), (68, 16713, 3200)]),
    ("mxfp4", 1, "128x32", True, [(22, 5558, 8224), (17, 5669, 8320)]),
    ("mxfp4", 2, "256x256", False, [(516, 10592, 672), (132, 25760, 1056), (134, 24736, 1152), (130, 25504, 3200)]),
    ("mxfp4", 2, "256x256", True, [(194, 8864, 20000)]),
    ("mxfp4", 2, "128x128", False, [(65, 12320, 672), (68, 12320, 640)]),
    ("mxfp4", 2, "128x128", True, [(73, 4320, 8224), (65, 4192, 8320)]),
    ("mxfp4", 2, "128x64", False, [(129, 9056, 1056), (136, 8352, 1152)]),
    ("mxfp4", 2, "128x64", True, [(70, 4128, 8224), (71, 2784, 12416)]),
    ("mxfp4", 2, "64x64", False, [(17, 32, 672), (17, 32, 640)]),
    ("mxfp4", 2, "64x64", True, [(17, 32, 1696), (17, 32, 3200)]),
    ("mxfp4", 2, "128x32", False, [(21, 16480, 1056), (20, 17248, 1152)]),
    ("mxfp4", 2, "128x32", True, [(20, 2784, 8224), (19, 2784, 8320)]),
    ("mxfp8", 1, "256x256", False, [(2311, 5258, 672), (466, 28783, 1056), (452, 29478, 1152), (1427, 31342, 3200)]),
    ("mxfp8", 1, "256x256", True, [(132, 13193, 20000)]),
    ("mxfp8", 1, "128x128", False, [(194, 26636, 288), (2040, 10153, 640)]),
    ("mxfp8", 1, "128x128", True, [(2143, 1029, 12320), (2372, 907, 12416)]),
    ("mxfp8", 1, "128x64", False, [(135, 16778, 672), (133, 16523, 640)]),
    ("mxfp8", 1, "128x64", True, [(1835, 323, 8224), (1795, 322, 8320)]),
    ("mxfp8", 1, "64x64", False, [(17, 35, 672), (18, 32, 640)]),
    ("mxfp8", 1, "64x64", True, [(18, 34, 1056), (19, 33, 1152)]),
    ("mxfp8", 1, "128x32", False, [(17, 16650, 672), (17, 16540, 640)]),
    ("mxfp8", 1, "128x32", True, [(17, 4195, 1696), (65, 2052, 1664)]),
    ("mxfp8", 2, "256x256", False, [(2370, 2592, 672), (207, 29216, 1056), (193, 28768, 1152), (708, 30816, 3200)]),
    ("mxfp8", 2, "256x256", True, [(136, 6560, 20000)]),
    ("mxfp8", 2, "128x128", False, [(65, 27680, 288)]),
    ("mxfp8", 2, "128x128", True, [(199, 4896, 12320), (194, 4832, 12416)]),
    ("mxfp8", 2, "128x64", False, [(132, 8544, 672), (131, 8608, 640)]),
    ("mxfp8", 2, "128x64", True, [(33, 4448, 8224), (37, 4320, 8320)]),
    ("mxfp8", 2, "64x64", False, [(17, 32, 672), (17, 32, 640)]),
    ("mxfp8", 2, "64x64", True, [(17, 32, 1056), (17, 32, 1152)]),
    ("mxfp8", 2, "128x32", False, [(18, 8928, 672), (18, 9120, 640)]),
    ("mxfp8", 2, "128x32", True, [(69, 1056, 1696), (17, 2144, 1664)]),
]


def _rows(gen, rows, k, fmt, power):
    """(values and scales between other bytes, what they stand for): any codes but NaN, powers of two about 2^power."""
    columns = k if fmt == "mxfp8" else k // 2
    store = torch.full((rows, columns + 32), 0x7F if fmt == "mxfp8" else 0x77, dtype=torch.uint8, device="cuda")
    scale_store = torch.full((rows, k // 32 + 8), 0xFF, dtype=torch.uint8, device="cuda")
    values, scales = store[:, 16:16 + columns], scale_store[:, 4:4 + k // 32]
    codes = torch.randint(0, 256, (rows, columns), generator=gen, device="cuda", dtype=torch.uint8)
    if fmt == "mxfp8":
        codes = torch.where(codes % 128 == 127, codes - 1, codes)
    values.copy_(codes)
    scales.copy_(torch.randint(126 + power, 129 + power, scales.shape, generator=gen, device="cuda", dtype=torch.uint8))
    if fmt == "mxfp8":
        numbers = codes.view(torch.float8_e4m3fn).double()
    else:
        grid = torch.cat([reference.FP4, -reference.FP4]).cuda()
        numbers = grid[torch.stack((codes & 15, codes >> 4), -1).flatten(1).int()]
    return (values.view(torch.float8_e4m3fn) if fmt == "mxfp8" else values, scales), numbers * (
        2.0 ** (scales.double() - 127)).repeat_interleave(32, 1)


def _launched(call):
    with _lib.launch_timing() as timing:
        result = call()
    torch.cuda.synchronize()
    return result, [name for name, _ in timing.records]


@pytest.mark.parametrize("fmt,weights,tile,split,shapes", CASES, ids=[f"{c[0]}-{c[1]}-{c[2]}-{'split' if c[3] else 'whole'}" for c in CASES])
def test_tile(fmt, weights, tile, split, shapes) -> None:
    for m, n, k in shapes:
        gen = torch.Generator(device="cuda").manual_seed(m + n + k)
        a, a_numbers = _rows(gen, m, k, fmt, -12 if fmt == "mxfp8" else -6)
        w, w_numbers = _rows(gen, n, k, "mxfp4", -2)
        store = torch.full((m, n + 16), 7.0, device="cuda")
        out = store[:, 8:8 + n]
        if weights == 1:
            want, size = reference.product(a_numbers, w_numbers)
            error = reference.sum_error(size, k, fmt, True)
            call = lambda **options: mxfp4_gemm(*a, *w, **options)  # noqa: B023, E731
            other = {"dtype": torch.float16}
        else:
            u, u_numbers = _rows(gen, n, k, "mxfp4", -2)
            want, error = reference.gated(a_numbers, w_numbers, u_numbers, "silu", fmt, True)
            call = lambda **options: mxfp4_gated_gemm(*a, *w, *u, **options)  # noqa: B023, E731
            other = {"output": torch.float16}
        want, error = want.cpu(), error.cpu()
        _, names = _launched(lambda: call(out=out))
        assert f"mxfp4_tile_kernel {tile}" in names and ("mxfp4_join_kernel" in names) == split, (m, n, k, names)
        reference.check(out, want, reference.rounded(want, error, torch.float32))
        assert bool((store[:, :8] == 7).all()) and bool((store[:, 8 + n:] == 7).all())
        first = out.clone()
        for _ in range(3):  # the same bits at every call
            out.zero_()
            assert torch.equal(call(out=out), first)
        assert torch.equal(call(**other), first.half())  # one sum, whatever the result's type
        if weights == 2:
            for kind in ("mxfp8", "mxfp4"):
                values, scales = call(output=kind)
                codes, want_scales = reference.quantize(first.cpu(), kind)
                assert torch.equal(scales.cpu(), want_scales) and torch.equal(reference.unpack(values, kind), codes)
