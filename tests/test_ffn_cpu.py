"""Dense feed-forward operators without a device: what the library exports, what it refuses before it launches anything, and the
reference formulas the GPU tests go by."""
import ctypes
import os
import re

import pytest
import torch

from tests import mx4_reference as ref
from zerocool_b200 import ffn
from zerocool_b200.moe import ZC_EEXEC, ZC_EINVAL, ZC_OK
from zerocool_b200.records import BF16, F16, F32

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20        # an address nothing is read from: 16-byte aligned, far from the others below
BIG = 1 << 40


def at(i):
    return P + i * BIG


def test_every_declared_symbol_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "zc_ffn.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(zc_[a-z0-9_]+)\s*\(", text)))
    lib = ffn.load_library()
    assert names == sorted(ffn.EXPORTS)
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("rows,cols,want", [(1, 32, 512), (128, 128, 512), (129, 128, 1024), (128, 160, 1024), (0, 64, 0), (8192, 4096, 64 * 32 * 512)])
def test_scale_bytes(rows, cols, want):
    n = ctypes.c_uint64()
    assert ffn.load_library().zc_mx4_scale_bytes(rows, cols, ctypes.byref(n)) == ZC_OK and n.value == want


def quantize(x=at(0), dtype=BF16, rows=4, cols=64, ld=64, codes=at(1), scales=at(2)):
    return ffn.load_library().zc_mx4_quantize(x, dtype, rows, cols, ld, codes, scales, None)


def linear(x=None, x_dtype=F32, x_ld=0, xc=at(0), xs=at(1), tokens=4, cols=64, wc=at(2), ws=at(3), rows=8, out=at(4), out_dtype=BF16, out_ld=8):
    return ffn.load_library().zc_mx4_linear(x, x_dtype, x_ld, xc, xs, tokens, cols, wc, ws, rows, out, out_dtype, out_ld, None)


def gated4(x=None, xc=at(0), xs=at(1), tokens=4, cols=64, gc=at(2), gs=at(3), uc=at(5), us=at(6), ffn_=8, out=at(4), out_dtype=BF16, out_ld=8):
    return ffn.load_library().zc_mx4_gated(x, F32, cols, xc, xs, tokens, cols, gc, gs, uc, us, ffn_, out, out_dtype, out_ld, None)


def forward(x=at(0), x_ld=16, gate=at(1), up=at(2), dtype=BF16, tokens=4, hidden=16, ffn_=8, h=at(3), g=at(4), u=at(5), saved=F32):
    return ffn.load_library().zc_gated_forward(x, x_ld, gate, up, dtype, tokens, hidden, ffn_, h, g, u, saved, None)


def backward(dh=at(0), dh_ld=8, x=at(1), x_ld=16, gate=at(2), up=at(3), g=at(4), u=at(5), dtype=BF16, tokens=4, hidden=16, ffn_=8, dg=at(6), du=at(7), dx=at(8), dgate=at(9), dup=at(10), saved=F32):
    return ffn.load_library().zc_gated_backward(dh, dh_ld, x, x_ld, gate, up, g, u, saved, dtype, tokens, hidden, ffn_, dg, du, dx, dgate, dup, None)


@pytest.mark.parametrize("call,why", [
    (lambda: quantize(x=None), b"missing buffer"), (lambda: quantize(codes=None), b"missing buffer"), (lambda: quantize(scales=None), b"missing buffer"),
    (lambda: quantize(cols=48, ld=48), b"multiple of 32"), (lambda: quantize(cols=0, ld=0), b"multiple of 32"), (lambda: quantize(cols=(1 << 20) + 32, ld=1 << 21), b"multiple of 32"),
    (lambda: quantize(ld=63), b"row stride"), (lambda: quantize(ld=(1 << 30) + 1), b"row stride"), (lambda: quantize(dtype=7), b"dtype"), (lambda: quantize(dtype=3), b"dtype"), (lambda: quantize(rows=1 << 31), b"rows"),
    (lambda: quantize(codes=at(1) + 8), b"16-byte aligned"), (lambda: quantize(scales=at(2) + 4), b"16-byte aligned"), (lambda: quantize(x=at(0) + 1), b"aligned to its elements"),
    (lambda: quantize(codes=at(0) + 64), b"overlapping"), (lambda: quantize(scales=at(1) + 64), b"overlapping"),
    (lambda: linear(xc=None), b"missing buffer"), (lambda: linear(ws=None), b"missing buffer"), (lambda: linear(out=None), b"missing buffer"),
    (lambda: linear(cols=72), b"multiple of 32"), (lambda: linear(rows=0), b"no rows"), (lambda: linear(out_ld=7), b"row stride"), (lambda: linear(out_dtype=3), b"dtype"),
    (lambda: linear(wc=at(2) + 8), b"16-byte aligned"), (lambda: linear(out=at(0) + 32), b"overlapping"), (lambda: linear(out=at(3) + 16), b"overlapping"),
    (lambda: linear(x=at(7), x_dtype=5, x_ld=64), b"dtype"), (lambda: linear(x=at(7), x_ld=63), b"row stride"), (lambda: linear(x=at(0) + 64, x_ld=64), b"overlapping"),
    (lambda: linear(x=at(7), x_ld=64, xc=at(2) + 32), b"overlapping"), (lambda: linear(x=at(7) + 2, x_ld=64), b"aligned to its elements"),
    (lambda: gated4(uc=None), b"missing buffer"), (lambda: gated4(us=at(6) + 1), b"16-byte aligned"), (lambda: gated4(out=at(5)), b"overlapping"), (lambda: gated4(ffn_=0), b"no rows"),
    (lambda: forward(dtype=F32), b"dtype"), (lambda: forward(hidden=20, x_ld=24), b"multiples of 8"), (lambda: forward(ffn_=12), b"multiples of 8"), (lambda: forward(x_ld=20), b"multiple of 16 bytes"),
    (lambda: forward(x_ld=8), b"row stride"), (lambda: forward(u=None), b"go together"), (lambda: forward(g=None), b"go together"), (lambda: forward(x=at(0) + 2), b"16-byte aligned"),
    (lambda: forward(gate=None), b"missing buffer"), (lambda: forward(h=at(1)), b"overlapping"), (lambda: forward(g=at(3) + 16), b"overlapping"),
    (lambda: forward(saved=F16), b"g and u must be"), (lambda: forward(saved=7), b"g and u must be"), (lambda: forward(u=at(4) + 64), b"overlapping"), (lambda: forward(g=at(4) + 4), b"16-byte aligned"),
    (lambda: backward(saved=F16), b"g and u must be"), (lambda: backward(dx=at(4) + 96), b"overlapping"),
    (lambda: backward(dtype=F32), b"dtype"), (lambda: backward(dh_ld=12), b"multiple of 16 bytes"), (lambda: backward(dup=None), b"go together"), (lambda: backward(dg=None), b"missing buffer"),
    (lambda: backward(du=at(6)), b"overlapping"), (lambda: backward(dx=at(1)), b"overlapping"), (lambda: backward(dgate=at(2)), b"overlapping"), (lambda: backward(tokens=1 << 31), b"shape"),
])
def test_refusals(call, why):
    assert call() == ZC_EINVAL
    assert why in ffn.load_library().zc_last_error()


def test_no_rows_is_a_valid_call():
    assert quantize(rows=0, x=None, codes=None, scales=None) == ZC_OK
    assert linear(tokens=0, xc=None, xs=None, out=None) == ZC_OK
    assert forward(tokens=0, x=None, h=None, g=None, u=None) == ZC_OK
    assert backward(tokens=0, dh=None, x=None, g=None, u=None, dg=None, du=None, dx=None, dgate=None, dup=None) == ZC_OK


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ffn.mx4_quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        ffn.Mx4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        ffn.gated_forward(x.half(), x.half(), x.half())
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        ffn.gated_forward(x, x, x)


def test_reference_rounding():
    """The e2m1 grid: ties to the even code, saturation at 6, the scale from the largest magnitude."""
    x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.99, -0.25, -0.26, -7.0] + [0.0] * 20).view(1, 32)
    codes, scales = ref.quantise(x)
    assert scales.item() == 127
    assert ref.values(codes, scales)[0, :12].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -0.5, -6]


def test_reference_gradient_against_differences():
    torch.manual_seed(3)
    x, gate, up, dh = (torch.randn(s, dtype=torch.float64) for s in ((5, 7), (6, 7), (6, 7), (5, 6)))
    loss = lambda x, gate, up: (dh * ref.silu(x @ gate.T) * (x @ up.T)).sum()  # noqa: E731
    _, _, dx, dgate, dup = ref.gated_gradient(dh, x, gate, up, x @ gate.T, x @ up.T)
    for t, want in ((x, dx), (gate, dgate), (up, dup)):
        for i in range(0, t.numel(), 3):
            step = torch.zeros_like(t)
            step.view(-1)[i] = 1e-6
            args = [v + step if v is t else v for v in (x, gate, up)]
            back = [v - step if v is t else v for v in (x, gate, up)]
            assert abs((loss(*args) - loss(*back)).item() / 2e-6 - want.reshape(-1)[i].item()) < 1e-6 * (1 + want.abs().max().item())


@pytest.mark.parametrize("wrong", [None, 3, torch.zeros(()), torch.zeros(4)])
def test_arguments_of_the_wrong_kind_are_value_errors(wrong):
    from zerocool_b200 import ffn
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    for call in (lambda: ffn.mx4_dequantize(wrong), lambda: ffn.Mx4(wrong, torch.zeros(512, dtype=torch.uint8)),
                 lambda: ffn.Mx4(torch.zeros(1, 16, dtype=torch.uint8), wrong), lambda: ffn.mx4_from_rows(wrong, torch.zeros(1, 1, dtype=torch.uint8)),
                 lambda: ffn.mx4_from_rows(torch.zeros(1, 16, dtype=torch.uint8), wrong), lambda: ffn.mx4_quantize(x, out=3),
                 lambda: ffn.gated_forward(x, wrong, x), lambda: ffn.gated_backward(x, x, wrong, x, x, x)):
        with pytest.raises(ValueError):
            call()


def test_wait_limit():
    assert ffn.wait_limit(5) == ffn.WAIT_POLLS == 1 << 20 and ffn.wait_limit() == 5
    for wrong in (-1, (1 << 27) + 1, 2.0, None, True):
        with pytest.raises(ValueError, match="2\\^27"):
            ffn.wait_limit(wrong)
    assert ffn.load_library().zc_ffn_wait_limit((1 << 27) + 1, None) == ZC_EINVAL and ffn.wait_limit() == ffn.WAIT_POLLS


@pytest.mark.parametrize("rows,cols,device", [(4, 64, "cpu"), (4, 64, "meta"), (0, 32, "cpu"), (-1, 64, "cuda"), (4, 48, "cuda"), (4, 0, "cuda"), (4.0, 64, "cuda"), (4, None, "cuda")])
def test_matrices_yet_to_be_written_are_on_a_cuda_device(rows, cols, device):
    with pytest.raises(ValueError):
        ffn.Mx4.empty(rows, cols, device)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused ends for want of a device")
@pytest.mark.parametrize("x,x_dtype,out,out_dtype,ld,apart", [
    (0, F32, 64, F32, 72, True), (8, F32, 0, F32, 72, True), (0, F32, 64, F32, 73, True), (0, F32, 63, F32, 72, False), (7, F32, 0, F32, 72, False),
    (0, F32, 64, F32, 71, False), (72, F32, 64, F32, 72, True), (72, F32, 63, F32, 72, False), (0, F32, 64 + 3 * 72, F32, 72, True), (0, F32, 62 + 3 * 72, F32, 72, False),
])
def test_columns_of_one_buffer_side_by_side(x, x_dtype, out, out_dtype, ld, apart):
    """x (64 columns) and out (8) of four rows in one buffer, their first elements at these places: refused only where they share an element."""
    rc = linear(x=at(7) + 4 * x, x_dtype=x_dtype, x_ld=ld, out=at(7) + 4 * out, out_dtype=out_dtype, out_ld=ld)
    rows = lambda first, n: {first + r * ld + c for r in range(4) for c in range(n)}  # noqa: E731
    assert apart == (not rows(x, 64) & rows(out, 8))
    assert rc == (ZC_EEXEC if apart else ZC_EINVAL) and (b"overlapping" in ffn.load_library().zc_last_error()) != apart


@pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused ends for want of a device")
@pytest.mark.parametrize("ld", [0, 8, 20, 1 << 40])
def test_the_stride_of_a_single_row_is_not_looked_at(ld):
    for call in (lambda: forward(tokens=1, x_ld=ld), lambda: backward(tokens=1, dh_ld=ld, x_ld=ld), lambda: linear(x=at(7), x_ld=ld, tokens=1, out_ld=ld), lambda: quantize(rows=1, ld=ld)):
        assert call() == ZC_EEXEC


def test_strides_of_several_rows_are():
    for ld in (0, 8, 20, 1 << 40):
        assert forward(tokens=2, x_ld=ld) == ZC_EINVAL and backward(tokens=2, x_ld=ld) == ZC_EINVAL and quantize(rows=2, ld=ld) == ZC_EINVAL
