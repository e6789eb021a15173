"""Norms, blocks, linears and gated products used together: feed-forward blocks, captured graphs, several streams, other tensors."""

from __future__ import annotations

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd import quantization
from qpu_xla_amd.kernels import (
    add_rms_norm,
    add_rms_norm_int8,
    add_rms_norm_mxfp4,
    add_rms_norm_mxfp8,
    add_rms_norm_q8_0,
    dequantize_mxfp4,
    mxfp4_gated_gemm,
    mxfp4_gated_linear,
    mxfp4_gemm,
    mxfp4_linear,
    quantize_mxfp4,
    quantize_mxfp8,
    quantize_q4_0,
    quantize_q8_0,
)
from qpu_xla_amd.kernels.gemm_int8 import w8a8_gemm_dequantize
from qpu_xla_amd.kernels.ggml_q4_0 import ggml_q4_0_q8_0_linear
from qpu_xla_amd.kernels.ggml_q8_0 import ggml_q8_0_q8_0_linear

pytestmark = pytest.mark.gpu

QUANTIZE = {"mxfp4": quantize_mxfp4, "mxfp8": quantize_mxfp8}
NORM = {"mxfp4": add_rms_norm_mxfp4, "mxfp8": add_rms_norm_mxfp8}


def _layer(d, hidden, seed=0):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda n, k: quantization.quantize_matrix_mxfp4((torch.randn((n, k), generator=gen) * k**-0.5).cuda())  # noqa: E731
    return (1 + 0.1 * torch.randn(d, generator=gen)).cuda(), draw(hidden, d), draw(hidden, d), draw(d, hidden)


def _rows(m, d, dtype, seed=0):
    gen = torch.Generator().manual_seed(100 + seed)
    return torch.randn((m, d), generator=gen).to(dtype).cuda(), torch.randn((m, d), generator=gen).to(dtype).cuda()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,d,hidden", [(1, 2048, 5632), (3, 96, 160), (29, 512, 1024), (150, 256, 704)])
def test_feed_forward(m, d, hidden, dtype, fmt) -> None:
    """Each operator against its definition, from the blocks that the one before it wrote."""
    weight, gate, up, down = _layer(d, hidden)
    x, residual = _rows(m, d, dtype)
    y, total = quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down, activations=fmt)
    values, scales, again = NORM[fmt](x, weight, residual)
    _, rounded, want_total = reference.norm(x, weight, residual, 1e-6)
    codes, want_scales = reference.quantize(rounded, fmt)
    assert torch.equal(total.cpu(), want_total) and torch.equal(again.cpu(), want_total)
    assert torch.equal(reference.unpack(values, fmt), codes) and torch.equal(scales.cpu(), want_scales)
    inner = mxfp4_gated_gemm(values, scales, gate.values, gate.scales, up.values, up.scales, output=fmt)
    operands = [reference.read(*t, f) for t, f in (((values, scales), fmt), ((gate.values, gate.scales), "mxfp4"), ((up.values, up.scales), "mxfp4"))]
    want, error = reference.gated(*operands, "silu", fmt, False)
    reference.check_blocks(*inner, fmt, want, error)
    want, size = reference.product(reference.read(*inner, fmt), reference.read(down.values, down.scales, "mxfp4"))
    assert y.dtype is dtype
    reference.check(y, want, reference.rounded(want, reference.sum_error(size, hidden, fmt, dtype is torch.float32), dtype))


def test_feed_forward_outputs_and_refusals() -> None:
    weight, gate, up, down = _layer(64, 96)
    x, residual = _rows(4, 64, torch.bfloat16)
    out, total = torch.empty((4, 64), device="cuda"), torch.empty_like(residual)
    y, got_total = quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down, function="gelu", residual_out=total, out=out)
    assert y is out and got_total is total
    plain = quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down, function="gelu", dtype=torch.float32)
    assert torch.equal(plain[0], out)
    assert quantization.mxfp4_feed_forward(x, None, weight, gate, up, down)[1] is None
    with pytest.raises(ValueError, match="block format"):
        quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down, activations="int8")
    with pytest.raises(ValueError, match="gate function"):
        quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down, function="relu")
    with pytest.raises(ValueError, match="differ in K"):
        quantization.mxfp4_feed_forward(x, residual, weight, gate, up, gate)


def test_matrix() -> None:
    w = torch.randn((70, 96), generator=torch.Generator().manual_seed(3))
    matrix = quantization.quantize_matrix_mxfp4(w.cuda())
    assert matrix.shape == (70, 96)
    assert torch.equal(matrix.dequantize().cpu().double(), reference.read(*reference.stored(w, "mxfp4"), "mxfp4"))
    assert matrix.dequantize(torch.bfloat16).dtype is torch.bfloat16
    x = torch.randn((5, 96), device="cuda")
    assert torch.equal(quantization.mxfp4_linear(x, matrix), mxfp4_linear(x, matrix.values, matrix.scales))


@pytest.mark.parametrize("m", [1, 12, 40, 300])
def test_captured_and_replayed(m) -> None:
    """A graph of a feed-forward block and float linears, replayed with new rows and eager work of the same shapes between."""
    weight, gate, up, down = _layer(1024, 2048)
    x, residual = _rows(m, 1024, torch.bfloat16)

    def step():
        y, total = quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down)
        z = mxfp4_linear(y, gate.values, gate.scales, activations="mxfp4")
        h = mxfp4_gated_linear(total, gate.values, gate.scales, up.values, up.scales)
        return y, total, z, h, add_rms_norm(y, weight, total)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for turn in range(4):
        rows = _rows(m, 1024, torch.bfloat16, seed=turn)
        x.copy_(rows[0])
        residual.copy_(rows[1])
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for t in captured:
            t.fill_(7)
        graph.replay()
        if turn % 2:
            torch.cuda.synchronize()
        for got, expected in zip(captured, want):
            assert torch.equal(got, expected)


@pytest.mark.parametrize("m", [1, 40, 260])
def test_two_graphs_replayed_in_turn(m) -> None:
    weight, gate, up, down = _layer(512, 1024)
    steps, graphs, outputs = [], [], []
    for seed in range(2):
        x, residual = _rows(m, 512, torch.bfloat16, seed=seed)
        steps.append(lambda x=x, residual=residual: quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down)[0])
    want = [step().clone() for step in steps]
    torch.cuda.synchronize()
    for step in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outputs.append(step())
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for out in outputs:
            out.zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):  # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(outputs, want):
            assert torch.equal(got, expected)


@pytest.mark.parametrize("m", [1, 24, 200])
def test_calls_on_two_streams_at_once(m) -> None:
    weight, gate, up, down = _layer(1024, 2048)
    inputs = [_rows(m, 1024, torch.bfloat16, seed=s) for s in range(2)]
    run = lambda rows, stream: quantization.mxfp4_feed_forward(*rows, weight, gate, up, down, stream=stream)[0]  # noqa: E731
    want = [run(rows, None).clone() for rows in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(5):
        got = []
        for rows, stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                got.append(run(rows, stream))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


@pytest.mark.parametrize("m", [1, 24, 200])
def test_stream_argument_that_is_not_the_current_one(m) -> None:
    """Work goes to ``stream``, with temporaries allocated on the current one: they must live until the work is done."""
    weight, gate, up, down = _layer(1024, 2048)
    x, residual = _rows(m, 1024, torch.bfloat16)
    want = quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down)[0]
    part = x[:, 1:993]  # not aligned: quantised to a workspace first
    linear = mxfp4_linear(part, gate.values[:, :496], gate.scales[:, :31])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for _ in range(3):
        got = quantization.mxfp4_feed_forward(x, residual, weight, gate, up, down, stream=stream)[0]
        other = mxfp4_linear(part, gate.values[:, :496], gate.scales[:, :31], stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert torch.equal(other, linear)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m", [1, 3, 16, 70])
def test_not_finite_activations(m, fmt) -> None:
    """A block with a NaN or an infinity makes its row NaN, and no other row."""
    gen = torch.Generator().manual_seed(m)
    x = torch.randn((m, 512), generator=gen).cuda()
    w = quantize_mxfp4(torch.randn((96, 512), generator=gen).cuda())
    clean = mxfp4_linear(x, *w, activations=fmt)
    clean_gated = mxfp4_gated_linear(x, *w, *w, activations=fmt)
    for value in (float("inf"), float("-inf"), float("nan")):
        bad = x.clone()
        bad[m // 2, 77] = value
        for got, want in ((mxfp4_linear(bad, *w, activations=fmt), clean), (mxfp4_gated_linear(bad, *w, *w, activations=fmt), clean_gated)):
            others = torch.arange(m) != m // 2
            assert bool(torch.isnan(got[m // 2]).all())
            assert torch.equal(got[others.cuda()], want[others.cuda()])
        values, scales = mxfp4_gated_linear(bad, *w, *w, activations=fmt, output="mxfp8")
        assert bool((scales[m // 2] == 255).all()) and not bool((scales[others.cuda()] == 255).any())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 1056, 96), (6, 512, 40), (16, 2048, 100), (40, 352, 64)])
def test_float_rows_of_any_alignment_and_stride(m, k, n, dtype, fmt) -> None:
    gen = torch.Generator().manual_seed(k)
    x = torch.randn((m, k), generator=gen).to(dtype).cuda()
    w = quantize_mxfp4(torch.randn((n, k), generator=gen).cuda())
    want, want_gated = mxfp4_linear(x, *w, activations=fmt), mxfp4_gated_linear(x, *w, *w, activations=fmt)
    for at, pad in ((0, 8), (1, 3), (8, 16), (0, 1)):
        store = torch.full((m, k + at + pad), float("nan"), dtype=dtype, device="cuda")
        view = store[:, at:at + k]
        view.copy_(x)
        assert torch.equal(mxfp4_linear(view, *w, activations=fmt), want)
        assert torch.equal(mxfp4_gated_linear(view, *w, *w, activations=fmt), want_gated)


@pytest.mark.parametrize("m", [2, 40])
def test_rows_of_one_tensor_used_twice(m) -> None:
    """Activations as weights of the same call, one matrix as gate and up, a sum written over its residual."""
    x = torch.randn((m, 256), generator=torch.Generator().manual_seed(m)).cuda()
    a = quantize_mxfp4(x)
    want, _ = reference.product(reference.read(*a, "mxfp4"), reference.read(*a, "mxfp4"))
    size = reference.product(reference.read(*a, "mxfp4").abs(), reference.read(*a, "mxfp4").abs())[0]
    reference.check(mxfp4_gemm(*a, *a), want, reference.rounded(want, reference.sum_error(size, 256, "mxfp4", True), torch.float32))
    residual = torch.randn_like(x)
    y, total = add_rms_norm(x, torch.ones(256, device="cuda"), residual)
    kept = residual.clone()
    again, written = add_rms_norm(x, torch.ones(256, device="cuda"), residual, residual_out=residual)
    assert written is residual and torch.equal(residual, total) and torch.equal(again, y) and torch.equal(total, x + kept)


@pytest.mark.parametrize("m", [1, 40])
def test_scales_at_the_ends_of_their_range(m) -> None:
    """Blocks at the smallest and the largest powers of two: products past the range of float32 become infinities, or zero."""
    a_values, w_values = torch.full((m, 16), 0x22, dtype=torch.uint8, device="cuda"), torch.full((33, 16), 0x22, dtype=torch.uint8, device="cuda")
    byte = lambda rows, v: torch.full((rows, 1), v, dtype=torch.uint8, device="cuda")  # noqa: E731
    for a, w, want in ((254, 0, 32.0), (0, 254, 32.0), (127, 127, 32.0), (254, 254, float("inf")), (0, 0, 0.0), (67, 67, 32 * 2.0**-120)):
        got = mxfp4_gemm(a_values, byte(m, a), w_values, byte(33, w))
        expected = torch.full((m, 33), want, device="cuda")
        assert torch.equal(got, expected), (a, w, float(got[0, 0]), want)


def test_other_device_is_refused() -> None:
    x, w = torch.zeros((2, 64), device="cuda"), quantize_mxfp4(torch.ones((32, 64), device="cuda"))
    with pytest.raises(ValueError, match="HIP device"):
        mxfp4_linear(x.cpu(), *w)
    with pytest.raises(ValueError, match="HIP device"):
        mxfp4_linear(x, w[0].cpu(), w[1])
    with pytest.raises(ValueError, match="HIP device"):
        add_rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="HIP device"):
        quantize_mxfp4(x, w[0][:2].cpu())
    with pytest.raises(ValueError, match="HIP device"):
        dequantize_mxfp4(w[0], w[1].cpu())


@pytest.mark.parametrize("m", [2, 40])
def test_types_of_blocks_that_torch_names(m) -> None:
    """Packed pairs as float4_e2m1fn_x2 and scales as float8_e8m0fnu are the same bytes."""
    gen = torch.Generator().manual_seed(m)
    x, w = torch.randn((m, 128), generator=gen).cuda(), quantize_mxfp4(torch.randn((64, 128), generator=gen).cuda())
    named = (w[0].view(torch.float4_e2m1fn_x2), w[1].view(torch.float8_e8m0fnu))
    a = quantize_mxfp4(x)
    named_a = (a[0].view(torch.float4_e2m1fn_x2), a[1].view(torch.float8_e8m0fnu))
    assert torch.equal(mxfp4_linear(x, *named), mxfp4_linear(x, *w))
    assert torch.equal(mxfp4_gemm(*named_a, *named), mxfp4_gemm(*a, *w))
    assert torch.equal(mxfp4_gated_gemm(*named_a, *named, *named), mxfp4_gated_gemm(*a, *w, *w))
    assert torch.equal(dequantize_mxfp4(*named), dequantize_mxfp4(*w))
    values, scales = quantize_mxfp4(x, torch.empty_like(a[0]).view(torch.float4_e2m1fn_x2), torch.empty_like(a[1]).view(torch.float8_e8m0fnu))
    assert torch.equal(values.view(torch.uint8), a[0]) and torch.equal(scales.view(torch.uint8), a[1])


def test_outputs_in_given_tensors() -> None:
    a, w = quantize_mxfp8(torch.randn((3, 128), device="cuda")), quantize_mxfp4(torch.randn((64, 128), device="cuda"))
    out = torch.empty((3, 64), dtype=torch.float16, device="cuda")
    assert mxfp4_gated_gemm(*a, *w, *w, out) is out
    assert torch.equal(out, mxfp4_gated_gemm(*a, *w, *w, output=torch.float16))
    pair = (torch.empty((3, 64), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((3, 2), dtype=torch.uint8, device="cuda"))
    got = mxfp4_gated_gemm(*a, *w, *w, pair, output="mxfp8")
    assert got[0] is pair[0] and got[1] is pair[1]
    x = torch.randn((64, 64), device="cuda")
    with pytest.raises(Exception, match="shares memory"):
        mxfp4_linear(x, *quantize_mxfp4(x), out=x)
    wide = torch.randn((5, 256), device="cuda")
    left, right = wide[:, :128], wide[:, 128:192]
    want = mxfp4_linear(left, *w)
    mxfp4_linear(left, *w, out=right)  # columns of one tensor share none
    assert torch.equal(right, want)


@pytest.mark.parametrize("m", [1, 5, 40])
def test_norms_before_the_other_linears(m) -> None:
    """Rows that the norm quantised give what the W8A8, Q4_0 and Q8_0 linears make of the norm in floats."""
    gen = torch.Generator().manual_seed(m)
    weight, w = (1 + 0.1 * torch.randn(256, generator=gen)).cuda(), (torch.randn((64, 256), generator=gen) / 16).cuda()
    x, residual = torch.randn((m, 256), generator=gen).cuda(), torch.randn((m, 256), generator=gen).cuda()
    y, total = add_rms_norm(x, weight, residual)
    matrix = quantization.quantize_per_output_channel_int8(w)
    codes, scales, again = add_rms_norm_int8(x, weight, residual)
    assert torch.equal(again, total)
    assert torch.equal(w8a8_gemm_dequantize(codes, matrix.values, scales, matrix.scales), quantization.w8a8_linear(y, matrix))
    blocks, again = add_rms_norm_q8_0(x, weight, residual)
    assert torch.equal(again, total)
    q4, q8 = quantize_q4_0(w), quantize_q8_0(w)
    assert torch.equal(ggml_q4_0_q8_0_linear(blocks, q4), ggml_q4_0_q8_0_linear(quantize_q8_0(y), q4))
    assert torch.equal(ggml_q8_0_q8_0_linear(blocks, q8), ggml_q8_0_q8_0_linear(quantize_q8_0(y), q8))
