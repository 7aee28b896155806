"""Dense feed-forward operators on the GPU where their arithmetic, their plans and their arguments end (definitions: tests/mx4_reference.py;
the tolerances are those of tests/test_ffn_gpu.py, and what a test adds to them stands beside it)."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from tests import mx4_reference as ref
from tests.test_ffn_gpu import close, ffn, randn, sums, view_of  # noqa: F401

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAR = (0.0, 4.0, 16.0, 21.0, 24.0, 28.0, 32.0, 36.0, 48.0, 96.0)


@pytest.mark.parametrize("tokens", [1, 5, 60, 300])
def test_far_gates_keep_their_values(ffn, tokens):
    """Gates from -64 to -160, where e^-g passes FP32's range, with an `up` of 2^100: h is -1e3 to -1e-38, not 0. silu(g) may itself be rounded to
    a multiple of 2^-149 (half of one, times |u|), and 2^-20 of the value as for every gate."""
    x, gate, up = (torch.zeros(r, 64, device="cuda") for r in (tokens, len(FAR), len(FAR)))
    x[:, 0], x[:, 32] = 4.0, 1.0
    gate[:, 0], gate[:, 32], up[:, 0] = -16.0, -torch.tensor(FAR, device="cuda"), 2.0 ** 98
    gate, up = ffn.mx4_quantize(gate), ffn.mx4_quantize(up)
    g, u = ref.of(ffn.mx4_quantize(x)) @ ref.of(gate).T, ref.of(ffn.mx4_quantize(x)) @ ref.of(up).T
    want = ref.silu(g) * u
    for dtype in (torch.float32, torch.bfloat16):
        close(ffn.mx4_gated(x, gate, up, dtype), want, 2.0 ** -20 * want.abs() + 2.0 ** -150 * u.abs())
    x, gate, up = (torch.zeros(r, 64, dtype=torch.bfloat16, device="cuda") for r in (tokens, 16, 16))
    x[:, 0], up[:, 0] = 1.0, 2.0 ** 100
    gate[:, 0] = -torch.linspace(60, 120, 16, device="cuda")
    h, g, u = ffn.gated_forward(x, gate, up, save=True)
    want = ref.silu(g.double()) * u.double()
    close(h, want, 2.0 ** -20 * want.abs() + 2.0 ** -150 * u.double().abs())


def gradient(ffn, dh, x, gate, up, g, u, want_x=True, want_w=True):
    """zc_gated_backward with dg and du in the test's own hands -> dg, du, dx, dgate, dup."""
    (tokens, width), hidden, new = dh.shape, x.shape[1], x.new_empty
    dg, du = new((tokens, width)), new((tokens, width))
    dx, dgate, dup = new((tokens, hidden)) if want_x else None, new((width, hidden)) if want_w else None, new((width, hidden)) if want_w else None
    at = lambda t: ctypes.c_void_p(None if t is None else t.data_ptr())  # noqa: E731
    rc = ffn.load_library().zc_gated_backward(at(dh), dh.stride(0), at(x), x.stride(0), at(gate), at(up), at(g), at(u), ffn.CODES[g.dtype], ffn.CODES[x.dtype], tokens, hidden, width,
                                              at(dg), at(du), at(dx), at(dgate), at(dup), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, ffn.load_library().zc_last_error()
    return dg, du, dx, dgate, dup


def elementwise_slack(dh, g, u):
    """dg and du are computed in FP32: 2^-18 of the terms before they cancel in 1 + g (1 - s) (fast exponential and reciprocal; the exponential's
    error grows with its argument, 2 + |1.18 g| units of 2^-23), and a sigmoid, or a product on the way to it, that may be subnormal."""
    s, each = torch.sigmoid(g), 2.0 ** -18 + (2 + 1.18 * g.abs()) * 2.0 ** -23
    under = 2.0 ** -149 * (1 + g.abs())
    return each * (dh * u * s).abs() * (1 + g.abs() * (1 - s)) + under, each * (dh * g * s).abs() + under


@pytest.mark.parametrize("saved", [torch.float32, torch.bfloat16])
def test_far_gates_keep_their_gradients(ffn, saved):
    """Gates of -60 to -160 whose dh and u are large enough for a gradient that is far above the smallest number."""
    g = -torch.linspace(60, 160, 64, device="cuda").repeat(3, 1).to(saved)
    u = torch.full_like(g, 2.0 ** 60)
    dh = torch.full((3, 64), 2.0 ** 40, dtype=torch.bfloat16, device="cuda")
    x, gate, up = (torch.zeros(r, 8, dtype=torch.bfloat16, device="cuda") for r in (3, 64, 64))
    dg, du, *_ = gradient(ffn, dh, x, gate, up, g, u)
    d = [t.double() for t in (dh, g, u)]
    want = ref.gated_gradient(d[0], x.double(), gate.double(), up.double(), d[1], d[2])[:2]
    for got, right, slack in zip((dg, du), want, elementwise_slack(*d)):
        close(got, right, slack)
    assert bool((dg[:, :40] < 0).all()) and bool((du[:, :40] < 0).all())


# -- waits that run out --------------------------------------------------------------------------------------------------------

@pytest.fixture
def short_waits(ffn):
    """A limit of the kernels' waits that a test makes run out: they give up, drain what they have started and return."""
    yield ffn.wait_limit
    ffn.wait_limit()
    torch.cuda.synchronize()
    ffn.status()


def every_plan(ffn):
    """Calls of every kernel: few tokens alone and in clusters, quantised inside or not, with ring wraps; tiles of either width, alone, many a pair, K shared."""
    x16 = {(t, k): randn((t, k), 1, dtype=torch.bfloat16) for t, k in ((1, 4128), (19, 2080), (60, 2048), (200, 8224), (300, 992), (700, 4104), (129, 2056))}
    w4 = {(n, k): ffn.mx4_quantize(randn((n, k), 2, 0.1)) for n, k in ((300, 4128), (14300, 2080), (300, 8224), (1000, 992), (9000, 992))}
    w16 = {(n, k): randn((n, k), 3, 0.1, torch.bfloat16) for n, k in ((520, 4104), (136, 2056), (2600, 2056), (520, 2048), (4104, 992))}
    calls = [lambda: ffn.mx4_linear(x16[1, 4128], w4[300, 4128]), lambda: ffn.mx4_gated(x16[19, 2080], w4[14300, 2080], w4[14300, 2080]),
             lambda: ffn.mx4_linear(x16[19, 2080], w4[14300, 2080]), lambda: ffn.mx4_linear(x16[200, 8224], w4[300, 8224]), lambda: ffn.mx4_gated(x16[200, 8224], w4[300, 8224], w4[300, 8224]),
             lambda: ffn.mx4_linear(x16[300, 992], w4[1000, 992]), lambda: ffn.mx4_linear(x16[300, 992], w4[9000, 992]), lambda: ffn.mx4_gated(x16[300, 992], w4[9000, 992], w4[9000, 992])]
    for (t, k), (n, _) in (((60, 2048), (520, 2048)), ((700, 4104), (520, 4104)), ((129, 2056), (136, 2056)), ((129, 2056), (2600, 2056)), ((300, 992), (4104, 992))):
        g, u, dh = (randn((t, n), s) for s in (4, 5, 6))
        calls.append(lambda x=x16[t, k], w=w16[n, k]: ffn.gated_forward(x, w, w))
        calls.append(lambda x=x16[t, k], w=w16[n, k], g=g, u=u, dh=dh.bfloat16(): torch.cat([v.reshape(-1) for v in ffn.gated_backward(dh, x, w, w, g, u)]))
    return calls


def test_waits_that_run_out_are_reported_and_leave_the_device_usable(ffn, short_waits):
    """No wait is granted a poll: every product gives up with its copies in flight, says so, and the next call is right."""
    calls = every_plan(ffn)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    assert ffn.status() == 0
    for i, call in enumerate(calls):
        assert short_waits(0) == ffn.WAIT_POLLS
        call()
        assert ffn.status() == 2 and ffn.status() == 0, i       # ZC_STATUS_TIMEOUT, taken by the call that returns it
        assert short_waits() == 0
        assert torch.equal(call(), want[i]) and ffn.status() == 0, i


@pytest.mark.parametrize("polls", [1, 2, 3, 4, 6, 8, 12, 20])
def test_waits_that_run_out_somewhere(ffn, short_waits, polls):
    """Limits at which some waits run out and others do not: a call says that it gave up, or its result is right."""
    for i, call in enumerate(every_plan(ffn)):
        want = call()
        for _ in range(3):
            short_waits(polls)
            got = call()
            gave_up = ffn.status()
            short_waits()
            assert gave_up in (0, 2) and (gave_up or torch.equal(got, want)), i
        assert torch.equal(call(), want) and ffn.status() == 0, i


def test_no_time_out_is_cleared_unseen(ffn, short_waits):
    """Time-outs raised on one stream at every moment of a status call on another: the call returns it, or the next one does."""
    x, w = randn((1, 256), 1, dtype=torch.bfloat16), ffn.mx4_quantize(randn((128, 256), 2))
    ffn.mx4_linear(x, w)
    raising, asking = torch.cuda.Stream(), torch.cuda.Stream()
    late = torch.zeros(600 << 17, device="cuda")
    torch.cuda.synchronize()
    lost = 0
    for i in range(600):
        with torch.cuda.stream(raising):
            late[:i << 17].add_(1.0)             # up to 100 us and more: the call below meets the time-out at another moment each time
            short_waits(0)
            ffn.mx4_linear(x, w)
            short_waits()
        with torch.cuda.stream(asking):
            seen = ffn.status()
        raising.synchronize()
        seen |= ffn.status()
        lost += seen != 2
    assert lost == 0


# -- clusters that add their sums ----------------------------------------------------------------------------------------------

def test_sums_of_ragged_tiles_while_clusters_come_and_go(ffn):
    """Tiles of which most rows lie past the matrix, their K split over clusters of up to eight CTAs, on three streams at once: clusters start and end
    beside one another all the time, and every result is that of the call alone."""
    jobs = []
    for rows in (1, 5, 130, 200, 259):
        w = [ffn.mx4_quantize(randn((rows, 2080), 10 + i, 0.1)) for i in range(2)]
        for tokens in (1, 3, 33, 130, 260):
            x = randn((tokens, 2080), tokens, dtype=torch.bfloat16)
            jobs += [lambda x=x, w=w: ffn.mx4_linear(x, w[0]), lambda x=x, w=w: ffn.mx4_gated(x, *w)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for round_ in range(6):
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[(i + round_) % 3]):
                got.append((i, job()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


@pytest.mark.parametrize("tokens", [1, 20, 60, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_x_and_result_side_by_side_in_one_buffer(ffn, tokens, dtype):
    """x and the results of two products as columns of one buffer, of aligned and of odd row strides: every column keeps what belongs to it."""
    w, v = ffn.mx4_quantize(randn((200, 320), 1, 0.1)), ffn.mx4_quantize(randn((200, 320), 2, 0.1))
    x = randn((tokens, 320), 3, dtype=dtype)
    for gap in (0, 1, 8):
        buffer = torch.full((tokens, 720 + 2 * gap), 7.0, dtype=dtype, device="cuda")
        left, mid, right = buffer[:, :200], buffer[:, 200 + gap:520 + gap], buffer[:, 520 + 2 * gap:]
        mid.copy_(x)
        ffn.mx4_linear(mid, w, out=left)
        ffn.mx4_gated(mid, w, v, out=right)
        assert torch.equal(left, ffn.mx4_linear(x, w, dtype)) and torch.equal(right, ffn.mx4_gated(x, w, v, dtype)) and torch.equal(mid, x)
        with pytest.raises(ValueError, match="overlapping"):
            ffn.mx4_linear(mid, w, out=buffer[:, 1 + gap:201 + gap])


def test_operands_that_require_gradients(ffn):
    """Where gradients are recorded a result without one is refused; without recording the call is as ever, and gated_backward gives the gradients."""
    x, gate, up = (randn((r, 64), s, dtype=torch.bfloat16) for s, r in ((1, 5), (2, 16), (3, 16)))
    w = ffn.mx4_quantize(gate.requires_grad_())                     # codes have no gradient: nothing is lost
    want = ffn.gated_forward(x, gate.detach(), up)
    for call in (lambda: ffn.gated_forward(x, gate, up), lambda: ffn.gated_forward(x.clone().requires_grad_(), gate.detach(), up, save=True),
                 lambda: ffn.gated_forward(x, gate.detach(), up.clone().requires_grad_()), lambda: ffn.mx4_linear(x.clone().requires_grad_(), w),
                 lambda: ffn.mx4_gated(x.clone().requires_grad_(), w, w)):
        with pytest.raises(ValueError, match="autograd"):
            call()
    with torch.no_grad():
        h, g, u = ffn.gated_forward(x, gate, up, save=True)
        assert torch.equal(h, want)
    dx, dgate, dup = ffn.gated_backward(torch.ones_like(h), x, gate, up, g, u)
    assert not (dx.requires_grad or dgate.requires_grad or dup.requires_grad)
    with torch.inference_mode():
        assert torch.equal(ffn.mx4_linear(x, w), ffn.mx4_linear(x.detach(), w))


@pytest.mark.parametrize("ld", [0, 8, 20, 1 << 40])
def test_a_single_row_of_any_stride(ffn, ld):
    x, gate, up = (randn((r, 64), s, dtype=torch.bfloat16) for s, r in ((1, 1), (2, 16), (3, 16)))
    h, g, u = torch.empty(1, 16, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 16, device="cuda"), torch.empty(1, 16, device="cuda")
    code, stream = ffn.CODES[torch.bfloat16], torch.cuda.current_stream().cuda_stream
    assert ffn.load_library().zc_gated_forward(x.data_ptr(), ld, gate.data_ptr(), up.data_ptr(), code, 1, 64, 16, h.data_ptr(), g.data_ptr(), u.data_ptr(), ffn.CODES[torch.float32], stream) == 0
    assert all(torch.equal(a, b) for a, b in zip((h, g, u), ffn.gated_forward(x, gate, up, save=True)))
    got, want = torch.empty_like(up), ffn.gated_backward(h, x, gate, up, g, u)
    dg, du, dx, dgate = torch.empty_like(h), torch.empty_like(h), torch.empty_like(x), torch.empty_like(gate)
    assert ffn.load_library().zc_gated_backward(h.data_ptr(), ld, x.data_ptr(), ld, gate.data_ptr(), up.data_ptr(), g.data_ptr(), u.data_ptr(), ffn.CODES[torch.float32], code, 1, 64, 16,
                                                dg.data_ptr(), du.data_ptr(), dx.data_ptr(), dgate.data_ptr(), got.data_ptr(), stream) == 0
    assert torch.equal(dx, want[0]) and torch.equal(dgate, want[1]) and torch.equal(got, want[2])


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (37, 288), (130, 1056)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_plain_matrices_of_any_alignment(ffn, rows, cols, dtype):
    """Every call that takes or gives a plain matrix of the microscaled forms, at an element's alignment: dequantisation into it, products from and into it."""
    q, w = ffn.mx4_quantize(randn((rows, cols), 1)), ffn.mx4_quantize(randn((72, cols), 2, 0.1))
    for left, right in ((1, 0), (3, 2), (0, 1), (8, 8), (5, 3)):
        big = torch.full((rows + 2, cols + left + right), 7.0, dtype=dtype, device="cuda")
        out = big[1:rows + 1, left:left + cols]
        assert ffn.mx4_dequantize(q, out=out) is out
        assert torch.equal(out.double(), ref.of(q).to(dtype).double())
        product, gated = ffn.mx4_linear(out.contiguous(), w, dtype), ffn.mx4_gated(out.contiguous(), w, w, dtype)
        into = torch.empty(rows * 72 + 3, dtype=dtype, device="cuda")[left % 4:][:rows * 72].view(rows, 72)
        assert torch.equal(ffn.mx4_linear(out, w, out=into), product) and torch.equal(ffn.mx4_gated(out, w, w, out=into), gated)
        out.fill_(7.0)
        assert bool((big == 7.0).all())
    scales = torch.empty(rows * (cols // 32) + 3, dtype=torch.uint8, device="cuda")[3:].view(rows, cols // 32)
    scales.copy_(ref.row_scales(q))
    assert torch.equal(ffn.mx4_from_rows(q.codes, scales).scales, q.scales)


def test_the_gated_block_writes_where_it_is_told(ffn):
    x, gate, up = (randn((r, 64), s, dtype=torch.float16) for s, r in ((1, 70), (2, 48), (3, 48)))
    for tokens in (1, 40, 70):
        big = torch.full((tokens + 2, 48), 7.0, dtype=torch.float16, device="cuda")
        out = big[1:-1]
        h, g, u = ffn.gated_forward(x[:tokens], gate, up, save=True, out=out)
        assert h is out and torch.equal(h, ffn.gated_forward(x[:tokens], gate, up))
        assert bool((big[0] == 7.0).all()) and bool((big[-1] == 7.0).all())
        for wrong in (big, big[:, :40], big.float()[1:-1], out.t(), 3, out.cpu()):
            with pytest.raises(ValueError):
                ffn.gated_forward(x[:tokens], gate, up, out=wrong)


# -- plans that the sizes of test_ffn_gpu.py do not reach ----------------------------------------------------------------------

@pytest.mark.parametrize("tokens,rows,cols", [(19, 14300, 2080), (40, 18900, 4128), (3, 19100, 2080), (17, 14210, 8224), (32, 15000, 288), (48, 19000, 800)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_few_tokens_over_many_rows(ffn, tokens, rows, cols, dtype):
    """As many tiles of rows as SMs: no cluster, the whole of K in one CTA, more of its blocks than the ring has stages."""
    x, gate, up = randn((tokens, cols), 1, dtype=dtype), *(ffn.mx4_quantize(randn((rows, cols), s, 0.05)) for s in (2, 3))
    q = ffn.mx4_quantize(x)
    xd, gd, ud = ref.of(q), ref.of(gate), ref.of(up)
    g, u, gs, us = xd @ gd.T, xd @ ud.T, sums(xd, gd, 64), sums(xd, ud, 64)
    h, slack = ref.silu(g) * u, 1.1 * gs * u.abs() + ref.silu(g).abs() * us + 1.1 * gs * us + 2.0 ** -20 * (ref.silu(g) * u).abs()
    for a in (x, q):
        close(ffn.mx4_linear(a, gate, dtype), g, gs)
        close(ffn.mx4_gated(a, gate, up, dtype), h, slack)


@pytest.mark.parametrize("tokens,hidden,width", [(33, 2056, 16392), (5, 1032, 20008), (64, 4104, 14216), (48, 520, 19000)])
def test_few_tokens_over_many_rows_in_16_bits(ffn, tokens, hidden, width):
    for dtype in (torch.bfloat16, torch.float16):
        x, gate, up = randn((tokens, hidden), 1, dtype=dtype), randn((width, hidden), 2, 0.1, dtype), randn((width, hidden), 3, 0.1, dtype)
        h, g, u = ffn.gated_forward(x, gate, up, save=True)
        xd, gd, ud = x.double(), gate.double(), up.double()
        gw, uw, gs, us = xd @ gd.T, xd @ ud.T, sums(xd, gd, 16), sums(xd, ud, 16)
        close(g, gw, gs)
        close(u, uw, us)
        close(h, ref.silu(gw) * uw, 1.1 * gs * uw.abs() + ref.silu(gw).abs() * us + 1.1 * gs * us + 2.0 ** -20 * (ref.silu(gw) * uw).abs())


@pytest.mark.parametrize("tokens,hidden,width", [(60, 16392, 264), (5, 20008, 136), (40, 19000, 1032), (65, 520, 4104), (513, 320, 264), (2, 40, 20008), (64, 2056, 4104), (33, 264, 200),
                                                 (129, 264, 72), (1500, 2056, 136), (200, 2056, 136), (900, 520, 1200), (1100, 264, 2600), (300, 16, 8), (1, 64, 128), (4100, 136, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_are_the_products_of_dg_and_du(ffn, tokens, hidden, width, dtype):
    """dg and du element by element against the formula, then dx, dgate and dup against the 64-bit products of the very dg and du that the call left: with
    nothing but the sums and one rounding to allow for, a token, a column of K or a segment that is missing anywhere shows."""
    x, gate, up = randn((tokens, hidden), 1, dtype=dtype), randn((width, hidden), 2, 0.2, dtype), randn((width, hidden), 3, 0.2, dtype)
    g, u, dh = randn((tokens, width), 4, 2.0), randn((tokens, width), 5, 2.0), randn((tokens, width), 6, 0.5, dtype)
    dg, du, dx, dgate, dup = gradient(ffn, dh, x, gate, up, g, u)
    d = [t.double() for t in (dh, x, gate, up, g, u)]
    for got, want, slack in zip((dg, du), ref.gated_gradient(*d)[:2], elementwise_slack(d[0], d[4], d[5])):
        close(got, want, slack)
    gd, ud, xd, wg, wu = dg.double(), du.double(), d[1], d[2], d[3]
    close(dx, gd @ wg + ud @ wu, 2 * -(-width // 16) * 2.0 ** -22 * (gd.abs() @ wg.abs() + ud.abs() @ wu.abs()), "dx")
    close(dgate, gd.T @ xd, sums(gd.T, xd.T, 16), "dgate")
    close(dup, ud.T @ xd, sums(ud.T, xd.T, 16), "dup")
    only_x, only_w = gradient(ffn, dh, x, gate, up, g, u, want_w=False), gradient(ffn, dh, x, gate, up, g, u, want_x=False)
    assert torch.equal(only_x[2], dx) and torch.equal(only_w[3], dgate) and torch.equal(only_w[4], dup)
    assert torch.equal(only_x[0], dg) and torch.equal(only_w[1], du)


def test_beside_products_of_other_libraries(ffn):
    """Kernels of few and of many tokens beside torch's own products of several sizes on another stream, which use tensor memory and clusters as well."""
    w4, w16 = [ffn.mx4_quantize(randn((1024, 2048), 2 + i, 0.05)) for i in range(2)], [randn((1024, 2048), 4 + i, 0.05, torch.bfloat16) for i in range(2)]
    jobs = []
    for tokens in (1, 7, 40, 64, 300):
        x = randn((tokens, 2048), tokens, dtype=torch.bfloat16)
        g, u, dh = randn((tokens, 1024), 6), randn((tokens, 1024), 7), randn((tokens, 1024), 8, dtype=torch.bfloat16)
        jobs += [lambda x=x: ffn.mx4_linear(x, w4[0]), lambda x=x: ffn.mx4_gated(x, *w4), lambda x=x: ffn.gated_forward(x, *w16),
                 lambda x=x, g=g, u=u, dh=dh: ffn.gated_backward(dh, x, *w16, g, u, weight_grads=False)[0]]
    others = [(randn((n, k), 9, dtype=torch.bfloat16), randn((k, m), 10, dtype=torch.bfloat16)) for n, k, m in ((64, 512, 512), (128, 4096, 256), (256, 1024, 1024), (512, 512, 2048), (2048, 2048, 2048))]
    want, theirs = [job() for job in jobs], [a @ b for a, b in others]
    torch.cuda.synchronize()
    streams, got, kept = [torch.cuda.Stream() for _ in range(3)], [], []
    for round_ in range(8):
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[0]):
                got.append((i, job()))
            for s in streams[1:]:
                with torch.cuda.stream(s):
                    j = (i + round_) % len(others)
                    kept.append((j, others[j][0] @ others[j][1]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    assert all(torch.allclose(y.float(), theirs[j].float(), rtol=2e-2, atol=1.0) for j, y in kept)


# -- the largest sizes, the same matrix twice, threads ---------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [1, 12, 70, 300])
def test_the_longest_rows(ffn, tokens):
    """K, then the rows of the weights, of 2^20."""
    x, gate, up = randn((tokens, 1 << 20), 1), *(ffn.mx4_quantize(randn((72, 1 << 20), s, 0.01)) for s in (2, 3))
    q = ffn.mx4_quantize(x)
    xd, gd, ud = ref.of(q), ref.of(gate), ref.of(up)
    g, u, gs, us = xd @ gd.T, xd @ ud.T, sums(xd, gd, 64), sums(xd, ud, 64)
    slack = 1.1 * gs * u.abs() + ref.silu(g).abs() * us + 1.1 * gs * us + 2.0 ** -20 * (ref.silu(g) * u).abs()
    for a in (x, q):
        close(ffn.mx4_linear(a, gate, torch.float32), g, gs)
        close(ffn.mx4_gated(a, gate, up, torch.float32), ref.silu(g) * u, slack)
    x, gate = randn((tokens, 8), 1, dtype=torch.bfloat16), randn((1 << 20, 8), 2, dtype=torch.bfloat16)
    h, g, u = ffn.gated_forward(x, gate, gate, save=True)
    gw, gs = x.double() @ gate.double().T, sums(x.double(), gate.double(), 16)
    close(g, gw, gs)
    close(h, ref.silu(gw) * gw, 2.1 * gs * gw.abs() + 1.1 * gs * gs + 2.0 ** -20 * (ref.silu(gw) * gw).abs())
    dg, du, dx, dgate, dup = gradient(ffn, h, x, gate, gate, g, u)
    gd, ud, xd, wd = dg.double(), du.double(), x.double(), gate.double()
    close(dx, gd @ wd + ud @ wd, 2 * (1 << 16) * 2.0 ** -22 * (gd.abs() + ud.abs()) @ wd.abs(), "dx")
    close(dgate, gd.T @ xd, sums(gd.T, xd.T, 16), "dgate")
    close(dup, ud.T @ xd, sums(ud.T, xd.T, 16), "dup")


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_a_matrix_with_itself(ffn, rows):
    """x, gate and up may be one and the same."""
    q = ffn.mx4_quantize(randn((rows, 544), 1, 0.3))
    v = ref.of(q)
    g, s = v @ v.T, sums(v, v, 64)
    close(ffn.mx4_linear(q, q, torch.float32), g, s)
    close(ffn.mx4_gated(q, q, q, torch.float32), ref.silu(g) * g, 2.1 * s * g.abs() + 1.1 * s * s + 2.0 ** -20 * (ref.silu(g) * g).abs())


THREADS = """
import threading, torch
from zerocool_b200 import ffn
torch.manual_seed(0)
w, v = torch.randn(304, 512, device="cuda").bfloat16(), torch.randn(304, 512, device="cuda").bfloat16()
scales = torch.randint(100, 130, (3 * 4 * 512,), device="cuda").to(torch.uint8)
q = ffn.Mx4(torch.randint(0, 256, (304, 256), device="cuda").to(torch.uint8), scales)
xs = [torch.randn(n, 512, device="cuda").bfloat16() for n in (1, 40, 300, 700)]
torch.cuda.synchronize()
start, results = threading.Barrier(len(xs)), {}

def work(i, x):
    out = []
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):
            h, g, u = ffn.gated_forward(x, w, v, save=True)
            out.append([ffn.mx4_linear(x, q), ffn.mx4_gated(x, q, q), ffn.mx4_quantize(x).codes, h, *ffn.gated_backward(h, x, w, v, g, u)])
            try:
                ffn.mx4_linear(x[:, :32 + 32 * i], q)
            except ValueError as e:
                assert f"{32 + 32 * i} columns" in str(e)
        torch.cuda.current_stream().synchronize()
    results[i] = out

threads = [threading.Thread(target=work, args=a) for a in enumerate(xs)]
[t.start() for t in threads], [t.join() for t in threads]
for i, x in enumerate(xs):
    h, g, u = ffn.gated_forward(x, w, v, save=True)
    want = [ffn.mx4_linear(x, q), ffn.mx4_gated(x, q, q), ffn.mx4_quantize(x).codes, h, *ffn.gated_backward(h, x, w, v, g, u)]
    for got in results[i]:
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
assert ffn.status() == 0
print("done")
"""


def test_threads_that_call_first_at_the_same_time(ffn):
    """Four threads of a fresh process, each on a stream of its own: their first calls of every kernel meet."""
    done = subprocess.run([sys.executable, "-c", THREADS], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0 and done.stdout.endswith("done\n"), done.stderr[-2000:]


# -- captures ------------------------------------------------------------------------------------------------------------------

CAPTURES = """
import sys, torch
from zerocool_b200 import ffn
first, tokens = sys.argv[1] == "first", int(sys.argv[2])
torch.manual_seed(0)
x, dh = torch.randn(tokens, 512, device="cuda").bfloat16(), torch.randn(tokens, 296, device="cuda").bfloat16()
w, g, u = torch.randn(296, 512, device="cuda").bfloat16(), torch.randn(tokens, 296, device="cuda"), torch.randn(tokens, 296, device="cuda")
codes, rows = torch.randint(0, 256, (296, 256), device="cuda").to(torch.uint8), torch.randint(100, 130, (296, 16), device="cuda").to(torch.uint8)
scales = torch.randint(100, 130, (3 * 4 * 512,), device="cuda").to(torch.uint8)
q = ffn.Mx4(codes, scales)

def calls(n):
    a = slice(0, n)
    return [lambda: ffn.mx4_quantize(x[a].float() if n > 1 else x[a]).codes, lambda: ffn.mx4_dequantize(q, torch.float16 if n > 1 else torch.bfloat16), lambda: ffn.mx4_from_rows(codes, rows).scales,
            lambda: ffn.mx4_linear(x[a], q), lambda: ffn.mx4_gated(x[a], q, q, torch.float16), lambda: ffn.gated_forward(x[a], w, w),
            lambda: torch.cat([v.flatten() for v in ffn.gated_backward(dh[a], x[a], w, w, g[a], u[a])])]

torch.cat([v.flatten() for v in (x[:1].float().half(), w)])       # torch's own kernels
if not first:
    for call in calls(1):
        call()
torch.cuda.synchronize()
for i, call in enumerate(calls(tokens)):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    graph.replay()
    torch.cuda.synchronize()
    got = got.clone()
    assert torch.equal(got, call()), i
assert ffn.status() == 0
print("captured")
"""


@pytest.mark.parametrize("before", ["first", "another size"])
@pytest.mark.parametrize("tokens", [1, 50, 300])
def test_captures_of_kernels_that_have_not_run(before, tokens):
    """Processes whose first call of every entry point is a captured one, or that have called it with one token before (which takes other kernels)."""
    done = subprocess.run([sys.executable, "-c", CAPTURES, before, str(tokens)], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0 and done.stdout.endswith("captured\n"), done.stderr[-2000:]
