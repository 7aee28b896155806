"""Dense feed-forward operators on the GPU against their definitions in 64 bits (tests/mx4_reference.py).

Tolerances. Products of e2m1 values and power-of-two scales are exact in FP32, and so are those of BF16 or FP16 values; what a tensor-core
product loses is in its sums: a step adds the products of 64 (MX4) or 16 (16-bit) k to an FP32 accumulator, aligned to the largest term,
so at most 2^-22 of the magnitudes summed so far. Over the steps: steps x 2^-22 x sum |x||w| (`sums`). A result is then rounded once:
half a step of its type, 2^-8 (BF16), 2^-11 (FP16), 2^-24 (FP32) of the value, and half the smallest subnormal.
"""
import pytest
import torch

from tests import mx4_reference as ref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ffn():
    from zerocool_b200 import ffn
    yield ffn
    assert ffn.status() == 0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(shape, seed, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * scale).to(dtype)


def sums(x, w, step):
    """Bound of what the FP32 sums of x w^T lose."""
    return -(-x.shape[1] // step) * 2.0 ** -22 * (x.abs() @ w.abs().T)


def close(got, want, slack, name=""):
    want = want.double()
    bound = slack + HALF[got.dtype] * (want.abs() + slack) + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), name
    worst = (off / bound).max().item() if got.numel() else 0.0
    assert worst <= 1.0, (name, worst, off.max().item())


def view_of(t, extra):
    """The same values as a view whose rows are `extra` elements further apart, starting `extra` elements in."""
    big = torch.full((t.shape[0], t.shape[1] + 2 * extra), float("nan"), dtype=t.dtype, device=t.device)
    big[:, extra:extra + t.shape[1]] = t
    return big[:, extra:extra + t.shape[1]]


# -- quantisation --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,extra", [(1, 32, 0), (3, 64, 0), (128, 128, 0), (129, 160, 0), (37, 288, 8), (5, 96, 3), (130, 1056, 1), (300, 256, 0)])
def test_quantisation_is_the_definition_bit_for_bit(ffn, dtype, rows, cols, extra):
    x = randn((rows, cols), rows + cols)
    x = x * torch.exp2(torch.randint(-6, 7, (rows, cols // 32), device="cuda", generator=gen(1)).float()).repeat_interleave(32, 1)
    x = (torch.round(x * 4) / 4).to(dtype) if rows % 2 else x.to(dtype)        # odd row counts: values on the borders of the grid
    q = ffn.mx4_quantize(view_of(x, extra) if extra else x)
    codes, scales = ref.quantise(x)
    assert torch.equal(ref.unpack(q.codes), codes)
    assert torch.equal(ref.row_scales(q), scales)
    used = torch.zeros(q.scales.numel(), dtype=torch.bool, device="cuda")
    used[ref.scale_index(rows, cols, "cuda").reshape(-1)] = True
    assert not q.scales[~used].any()                                           # what lies past the matrix is 0
    for out in TYPES:
        want = ref.values(codes, scales)
        got = ffn.mx4_dequantize(q, out)
        assert torch.equal(got.double(), want.to(out).double())


def test_quantisation_of_zeros_extremes_and_what_is_not_finite(ffn):
    x = torch.zeros(12, 96, device="cuda")
    x[1] = -0.0
    x[2, 3], x[3, 40], x[4, 95] = float("nan"), float("inf"), float("-inf")
    x[5] = 2.0 ** -149
    x[6] = torch.finfo(torch.float32).max
    x[7] = -2.0 ** -126
    x[8, 0] = 2.0 ** -125
    x[9] = 2.0 ** 127
    x[10, 31], x[10, 32] = 1.0, 64.0
    q = ffn.mx4_quantize(x)
    codes, scales = ref.quantise(x)
    assert torch.equal(ref.unpack(q.codes), codes) and torch.equal(ref.row_scales(q), scales)
    assert scales[2].tolist() == [255, 0, 0] and scales[3].tolist() == [0, 255, 0] and scales[4].tolist() == [0, 0, 255]
    back = ffn.mx4_dequantize(q, torch.float32)
    assert bool(torch.isnan(back[2, :32]).all()) and not back[2, 32:].any()
    y = ffn.mx4_linear(q, ffn.mx4_quantize(torch.ones(8, 96, device="cuda")), torch.float32)
    assert torch.isnan(y).any(1).tolist() == [False, False, True, True, True] + [False] * 7


def test_every_code_and_scale_comes_back(ffn):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(16, 16).repeat(16, 1).contiguous()      # [256, 16]: 32 values a row
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").view(256, 1).contiguous()
    q = ffn.mx4_from_rows(codes, scales)
    want = ref.values(ref.unpack(codes), scales.long())
    for dtype in (torch.bfloat16, torch.float32):
        got = ffn.mx4_dequantize(q, dtype)
        # scale bytes 253 and 254 reach 2^128 and beyond, which is infinity in every type here
        assert torch.equal(got[:255].double(), want[:255].to(dtype).double()) and bool(torch.isnan(got[255]).all())


def test_row_major_scales_take_their_tiles(ffn):
    for rows, cols in ((1, 32), (127, 160), (257, 384)):
        q = ffn.mx4_quantize(randn((rows, cols), 5))
        again = ffn.mx4_from_rows(q.codes, ref.row_scales(q).to(torch.uint8).contiguous())
        assert torch.equal(again.scales, q.scales)


def test_quantise_into_buffers_of_the_caller(ffn):
    x = randn((9, 64), 2)
    q = ffn.Mx4.empty(9, 64, "cuda")
    assert ffn.mx4_quantize(x, out=q) is q and torch.equal(q.codes, ffn.mx4_quantize(x).codes)
    with pytest.raises(ValueError, match="out must be"):
        ffn.mx4_quantize(x, out=ffn.Mx4.empty(8, 64, "cuda"))


# -- microscaled products ------------------------------------------------------------------------------------------------------

SIZES = [(1, 1, 32), (2, 128, 64), (7, 129, 96), (16, 64, 128), (17, 300, 160), (64, 257, 256), (100, 100, 288), (127, 128, 512), (128, 256, 544), (129, 511, 1024),
         (255, 33, 2048), (257, 513, 320), (300, 1000, 992),
         (1, 260, 4128), (5, 300, 8192), (33, 200, 8224), (128, 140, 2080), (3, 20000, 96), (31, 2400, 1056),
         (1300, 2600, 160), (700, 4100, 416), (129, 9000, 2080),
         (200, 300, 8224), (260, 141, 3104), (1000, 520, 6400), (129, 1, 32), (300, 7, 96), (1, 7, 32), (64, 64, 64), (65, 64, 64), (400, 600, 4000), (1000, 520, 9312), (40, 300, 512), (40, 300, 544), (60, 300, 2048), (50, 300, 2080)]


@pytest.mark.parametrize("tokens,rows,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear(ffn, tokens, rows, cols, dtype):
    x, w = randn((tokens, cols), 1, dtype=dtype), ffn.mx4_quantize(randn((rows, cols), 2, 0.05))
    q = ffn.mx4_quantize(x)
    xd, wd = ref.of(q), ref.of(w)
    want, slack = xd @ wd.T, sums(xd, wd, 64)
    got = ffn.mx4_linear(q, w, dtype)
    close(got, want, slack)
    close(ffn.mx4_linear(x, w, dtype), want, slack, "plain")
    assert torch.equal(got, ffn.mx4_linear(q, w, dtype))


@pytest.mark.parametrize("tokens,ffn_,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_gated4(ffn, tokens, ffn_, cols, dtype):
    x = randn((tokens, cols), 3, dtype=dtype)
    gate, up = (ffn.mx4_quantize(randn((ffn_, cols), s, 0.1)) for s in (4, 5))
    q = ffn.mx4_quantize(x)
    xd, gd, ud = ref.of(q), ref.of(gate), ref.of(up)
    g, u = xd @ gd.T, xd @ ud.T
    # |silu'| <= 1.1; the activation itself: an exponential, a sum and a quotient in FP32, and the product (2^-20 in all)
    slack = 1.1 * sums(xd, gd, 64) * u.abs() + ref.silu(g).abs() * sums(xd, ud, 64) + 1.1 * sums(xd, gd, 64) * sums(xd, ud, 64) + 2.0 ** -20 * (ref.silu(g) * u).abs()
    close(ffn.mx4_gated(q, gate, up, dtype), ref.silu(g) * u, slack)
    close(ffn.mx4_gated(x, gate, up, dtype), ref.silu(g) * u, slack, "plain")


@pytest.mark.parametrize("tokens", [5, 60, 200])
def test_what_is_not_finite_stays_in_its_row(ffn, tokens):
    """A NaN or an infinity in one row of x, or of the weights, makes that row (column) of the result NaN and no other."""
    x, w = randn((tokens, 320), 1), randn((150, 320), 2)
    x[2, 5], x[4, 319], w[149, 100] = float("nan"), float("inf"), float("-inf")
    qw = ffn.mx4_quantize(w)
    for y in (ffn.mx4_linear(x, qw), ffn.mx4_linear(ffn.mx4_quantize(x), qw, torch.float32), ffn.mx4_gated(x, qw, qw)):
        want = torch.zeros(tokens, 150, dtype=torch.bool, device="cuda")
        want[2], want[4], want[:, 149] = True, True, True
        assert torch.equal(torch.isnan(y), want)
    x = randn((tokens, 64), 3, dtype=torch.bfloat16)
    x[2, 5] = float("nan")
    gate, up, dh = randn((72, 64), 4, dtype=torch.bfloat16), randn((72, 64), 5, dtype=torch.bfloat16), randn((tokens, 72), 6, dtype=torch.bfloat16)
    h, g, u = ffn.gated_forward(x, gate, up, save=True)
    dx, dgate, dup = ffn.gated_backward(dh, x, gate, up, g, u)
    for y in (h, g, u, dx):
        assert torch.isnan(y).any(1).nonzero().view(-1).tolist() == [2] and bool(torch.isnan(y[2]).all())
    assert bool(torch.isnan(dgate).all()) and bool(torch.isnan(dup).all())


def test_matrices_beyond_two_gigabytes_of_offsets(ffn):
    """Offsets of x, codes and results that pass 32 bits: the last rows are those of the same rows alone."""
    rows, cols = 1100000, 4096                    # 4.5e9 values
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-300:] = randn((300, cols), 1, dtype=torch.bfloat16)
    q = ffn.mx4_quantize(x)
    tail = ffn.mx4_quantize(x[-300:])
    assert torch.equal(q.codes[-300:], tail.codes) and not q.codes[:1000].any()
    w = ffn.mx4_quantize(randn((4096, cols), 2, 0.05))
    want = ffn.mx4_linear(tail, w)
    out = torch.full((rows, 4096), 3.0, dtype=torch.bfloat16, device="cuda")
    ffn.mx4_linear(q, w, out=out)
    assert torch.equal(out[-300:], want) and not out[1000000].any()
    out.fill_(3.0)
    ffn.mx4_dequantize(q, out=out)
    assert torch.equal(out[-300:], ffn.mx4_dequantize(tail)) and not out[1000000].any()


@pytest.mark.parametrize("tokens", [3, 40, 200])
def test_linear_scales_of_every_size(ffn, tokens):
    """Blocks whose scales differ by 2^40: every block's own pair of scales is used, in every position of a tile."""
    rows, cols = 200, 640
    x, w = randn((tokens, cols), 1), randn((rows, cols), 2)
    x = x * torch.exp2(torch.randint(-20, 21, (tokens, cols // 32), device="cuda", generator=gen(7)).float()).repeat_interleave(32, 1)
    w = w * torch.exp2(torch.randint(-20, 21, (rows, cols // 32), device="cuda", generator=gen(8)).float()).repeat_interleave(32, 1)
    qx, qw = ffn.mx4_quantize(x), ffn.mx4_quantize(w)
    close(ffn.mx4_linear(qx, qw, torch.float32), ref.of(qx) @ ref.of(qw).T, sums(ref.of(qx), ref.of(qw), 64))


@pytest.mark.parametrize("tokens,rows", [(1, 90), (35, 90), (70, 90), (70, 96), (300, 700), (35, 2000)])
def test_outputs_of_the_caller_keep_what_lies_around_them(ffn, tokens, rows):
    """Views as output: row strides of every alignment, the rows and columns around the result untouched."""
    x, w, v = ffn.mx4_quantize(randn((tokens, 1056), 1)), ffn.mx4_quantize(randn((rows, 1056), 2)), ffn.mx4_quantize(randn((rows, 1056), 3))
    want, gated = ffn.mx4_linear(x, w, torch.float32), ffn.mx4_gated(x, w, v, torch.float32)
    for dtype in TYPES:
        for left, right in ((0, 1), (1, 2), (8, 6), (16, 22), (8, 0), (0, 8)):
            big = torch.full((tokens + 4, rows + left + right), 7.0, dtype=dtype, device="cuda")
            out = big[2:tokens + 2, left:left + rows]
            assert ffn.mx4_linear(x, w, out=out) is out
            assert torch.equal(out, want.to(dtype))
            assert torch.equal(ffn.mx4_gated(x, w, v, out=out), gated.to(dtype))
            out.fill_(7.0)
            assert bool((big == 7.0).all())


def test_no_tokens(ffn):
    w = ffn.mx4_quantize(randn((64, 64), 1))
    assert ffn.mx4_linear(torch.empty(0, 64, device="cuda"), w).shape == (0, 64)
    assert ffn.mx4_gated(ffn.mx4_quantize(torch.empty(0, 64, device="cuda")), w, w).shape == (0, 64)
    assert ffn.mx4_dequantize(ffn.mx4_quantize(torch.empty(0, 64, device="cuda"))).shape == (0, 64)
    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    gate = randn((8, 64), 1, dtype=torch.bfloat16)
    h, g, u = ffn.gated_forward(e, gate, gate, save=True)
    dx, dgate, dup = ffn.gated_backward(h, e, gate, gate, g, u)
    assert h.shape == (0, 8) and dx.shape == (0, 64) and not dgate.any() and not dup.any()


# -- the gated block in 16 bits ------------------------------------------------------------------------------------------------

BLOCKS = [(1, 8, 8), (1, 64, 128), (5, 72, 136), (16, 128, 64), (33, 64, 200), (127, 136, 128), (128, 64, 256), (129, 264, 72), (200, 520, 392), (256, 128, 512), (513, 320, 264),
          (1, 2056, 1160), (9, 4096, 136), (65, 520, 4104), (128, 1032, 1032), (2, 40, 20008), (1100, 264, 2600), (1500, 2056, 136),
          (200, 2056, 136), (130, 40, 4104), (1500, 136, 136), (900, 1032, 520), (130, 8, 8), (300, 16, 8), (64, 8, 264), (70, 264, 8), (900, 2312, 520), (900, 520, 1200), (2400, 520, 520), (40, 512, 136), (40, 520, 264), (60, 2048, 72), (50, 2056, 1032)]


@pytest.mark.parametrize("tokens,hidden,width", BLOCKS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gated_forward(ffn, tokens, hidden, width, dtype):
    x, gate, up = randn((tokens, hidden), 1, dtype=dtype), randn((width, hidden), 2, 0.2, dtype), randn((width, hidden), 3, 0.2, dtype)
    h, g, u = ffn.gated_forward(x, gate, up, save=True)
    xd, gd, ud = x.double(), gate.double(), up.double()
    gw, uw, gs, us = xd @ gd.T, xd @ ud.T, sums(xd, gd, 16), sums(xd, ud, 16)
    close(g, gw, gs)
    close(u, uw, us)
    close(h, ref.silu(gw) * uw, 1.1 * gs * uw.abs() + ref.silu(gw).abs() * us + 1.1 * gs * us + 2.0 ** -20 * (ref.silu(gw) * uw).abs())
    assert g.dtype == u.dtype == torch.float32
    assert torch.equal(h, ffn.gated_forward(view_of(x, 8), gate, up))
    small = ffn.gated_forward(x, gate, up, save=True, save_dtype=dtype)
    assert torch.equal(small[0], h) and torch.equal(small[1], g.to(dtype)) and torch.equal(small[2], u.to(dtype))


def gradient_slack(dtype, dh, x, gate, up, g, u):
    """What dx, dgate and dup may be off: dg and du are rounded to 16 bits (and computed in FP32: 2^-18 with the fast exponential and
    reciprocal, of the terms before they cancel in 1 + g (1 - s)), then summed."""
    s = torch.sigmoid(g)
    each = HALF[dtype] + 2.0 ** -18
    ag = each * (dh * u * s).abs() * (1 + g.abs() * (1 - s)) + TINY[dtype]
    au = each * (dh * g * s).abs() + TINY[dtype]
    dg, du, _, _, _ = ref.gated_gradient(dh, x, gate, up, g, u)
    mg, mu, steps = dg.abs() + ag, du.abs() + au, -(-x.shape[0] // 16)
    dx = ag @ gate.abs() + au @ up.abs() + 2 * -(-g.shape[1] // 16) * 2.0 ** -22 * (mg @ gate.abs() + mu @ up.abs())
    return dx, ag.T @ x.abs() + steps * 2.0 ** -22 * (mg.T @ x.abs()), au.T @ x.abs() + steps * 2.0 ** -22 * (mu.T @ x.abs())


@pytest.mark.parametrize("tokens,hidden,width", BLOCKS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gated_backward(ffn, tokens, hidden, width, dtype):
    x, gate, up = randn((tokens, hidden), 1, dtype=dtype), randn((width, hidden), 2, 0.2, dtype), randn((width, hidden), 3, 0.2, dtype)
    dh = randn((tokens, width), 4, 0.5, dtype)
    for saved in (dtype, torch.float32):
        _, g, u = ffn.gated_forward(x, gate, up, save=True, save_dtype=saved)
        d = [t.double() for t in (dh, x, gate, up, g, u)]
        got = ffn.gated_backward(dh, x, gate, up, g, u)
        for name, a, b, slack in zip(("dx", "dgate", "dup"), got, ref.gated_gradient(*d)[2:], gradient_slack(dtype, *d)):
            close(a, b, slack, name)
    again = ffn.gated_backward(view_of(dh, 8), view_of(x, 8), gate, up, g, u)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    only_x = ffn.gated_backward(dh, x, gate, up, g, u, weight_grads=False)
    only_w = ffn.gated_backward(dh, x, gate, up, g, u, input_grad=False)
    assert torch.equal(only_x[0], got[0]) and only_x[1] is None and only_x[2] is None
    assert only_w[0] is None and torch.equal(only_w[1], got[1]) and torch.equal(only_w[2], got[2])


def test_large_gates_saturate(ffn):
    """Gates far into either side of the sigmoid: silu is 0 or the gate itself, the gradient finite."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.tensor([-300.0, 300.0, -20.0, 20.0])
    gate, up = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    gate[:, 0], up[:, 0] = 1.0, 0.5
    h, g, u = ffn.gated_forward(x, gate, up, save=True)
    want = ref.silu(g.double()) * u.double()
    close(h, want, 2.0 ** -20 * want.abs())
    got = ffn.gated_backward(torch.ones_like(h), x, gate, up, g, u)
    d = [t.double() for t in (torch.ones_like(h), x, gate, up, g, u)]
    for a, b, slack in zip(got, ref.gated_gradient(*d)[2:], gradient_slack(torch.bfloat16, *d)):
        close(a, b, slack)


# -- how calls go together -----------------------------------------------------------------------------------------------------

def test_block_is_trained_quantised_and_served(ffn):
    """The operators in a row: a step of the 16-bit block, its weights quantised, the block and its output projection from 4 bits."""
    tokens, hidden, width = 130, 256, 384
    x, gate, up, down = randn((tokens, hidden), 1, dtype=torch.bfloat16), *(randn(s, i, 0.06, torch.bfloat16) for i, s in ((2, (width, hidden)), (3, (width, hidden)), (4, (hidden, width))))
    h, g, u = ffn.gated_forward(x, gate, up, save=True)
    dh = (h.float() @ down.float().T @ down.float()).bfloat16()
    _, dgate, dup = ffn.gated_backward(dh, x, gate, up, g, u)
    gate, up = (gate.float() - 1e-3 * dgate.float()).bfloat16(), (up.float() - 1e-3 * dup.float()).bfloat16()
    qg, qu, qd = ffn.mx4_quantize(gate), ffn.mx4_quantize(up), ffn.mx4_quantize(down)
    h4 = ffn.mx4_gated(x, qg, qu)
    y = ffn.mx4_linear(h4, qd, torch.float32)
    hq = ref.of(ffn.mx4_quantize(h4))
    close(y, hq @ ref.of(qd).T, sums(hq, ref.of(qd), 64))
    xq = ref.values(*ref.quantise(x))
    gw, uw = xq @ ref.of(qg).T, xq @ ref.of(qu).T
    gs, us = sums(xq, ref.of(qg), 64), sums(xq, ref.of(qu), 64)
    close(h4, ref.silu(gw) * uw, 1.1 * gs * uw.abs() + ref.silu(gw).abs() * us + 1.1 * gs * us + 2.0 ** -20 * (ref.silu(gw) * uw).abs())


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_captured_calls_replay_on_new_inputs(ffn, tokens):
    x, dh = randn((tokens, 256), 1, dtype=torch.bfloat16), randn((tokens, 128), 4, dtype=torch.bfloat16)
    gate, up = randn((128, 256), 2, 0.1, torch.bfloat16), randn((128, 256), 3, 0.1, torch.bfloat16)
    qg, qu = ffn.mx4_quantize(gate), ffn.mx4_quantize(up)

    def calls():
        h, g, u = ffn.gated_forward(x, gate, up, save=True)
        return [ffn.mx4_linear(x, qg), ffn.mx4_gated(x, qg, qu), h, g, u, *ffn.gated_backward(dh, x, gate, up, g, u)]

    calls()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                        # two graphs of the same calls: they share no scratch
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = calls()
        graphs.append((graph, outs))
    x.copy_(randn((tokens, 256), 11))
    dh.copy_(randn((tokens, 128), 14))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for (graph, _), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    want = calls()
    for _, outs in graphs:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_on_two_streams_at_once(ffn):
    x = randn((200, 512), 1, dtype=torch.bfloat16)
    ws = [ffn.mx4_quantize(randn((300, 512), 2 + i, 0.1)) for i in range(2)]
    want = [ffn.mx4_linear(x, w) for w in ws]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ffn.mx4_linear(x, ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_every_kernel_beside_every_other_and_the_expert_layer(ffn):
    """Kernels of one and of many tokens, in 4 and in 16 bits, on four streams at once, beside the routed layer's tensor-core kernels: the
    results are those of the calls alone."""
    from tests import util
    from zerocool_b200.moe import Moe
    cfg = util.cfg2(experts=32, max_tokens=512)
    layer = Moe(cfg, 0)
    layer.synth_fill_layer(0, 7)
    tokens = randn((512, cfg.hidden), 9, dtype=torch.bfloat16)
    w = [ffn.mx4_quantize(randn((1024, 2048), 20 + i, 0.05)) for i in range(2)]
    v = [randn((1024, 2048), 30 + i, 0.05, torch.bfloat16) for i in range(2)]
    jobs = []
    for n in (1, 60, 64, 300, 900):
        x = randn((n, 2048), 40 + n, dtype=torch.bfloat16)
        jobs += [lambda x=x: ffn.mx4_linear(x, w[0]), lambda x=x: ffn.mx4_gated(x, *w), lambda x=x: ffn.gated_forward(x, *v)]
    jobs.append(lambda: layer.prefill(0, tokens))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for round_ in range(6):
        for i, job in enumerate(jobs[:-1]):
            with torch.cuda.stream(streams[(i + round_) % 3]):
                got.append((i, job()))
        got.append((len(jobs) - 1, jobs[-1]()))            # a handle is driven by one stream
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    assert layer.status() == 0


def test_python_refusals(ffn):
    x, w = randn((4, 64), 1), ffn.mx4_quantize(randn((8, 64), 2))
    for call, why in ((lambda: ffn.mx4_quantize(x.double()), "dtype"), (lambda: ffn.mx4_quantize(x[:, :40]), "multiple of 32"), (lambda: ffn.mx4_quantize(x.t()), "columns"),
                      (lambda: ffn.mx4_quantize(x[0]), "matrix"), (lambda: ffn.mx4_linear(x[:, :32].contiguous(), w), "columns"), (lambda: ffn.mx4_linear(x, w, torch.int8), "dtype"),
                      (lambda: ffn.mx4_linear(x, w, out=torch.empty(4, 9, device="cuda")), "out must be"),
                      (lambda: ffn.mx4_gated(x, w, ffn.mx4_quantize(randn((9, 64), 2))), "differ in shape"), (lambda: ffn.mx4_linear(x, x), "must be Mx4"),
                      (lambda: ffn.mx4_from_rows(w.codes[0], torch.zeros(8, 2, dtype=torch.uint8, device="cuda")), "codes must be"),
                      (lambda: ffn.mx4_linear(x.cpu(), w), "CUDA"), (lambda: ffn.mx4_linear(x, w, out=torch.empty(4, 8)), "CUDA"),
                      (lambda: ffn.Mx4(w.codes[:, :8], w.scales), "codes"), (lambda: ffn.Mx4(w.codes, w.scales[:256]), "scales"),
                      (lambda: ffn.mx4_from_rows(w.codes, torch.zeros(8, 3, dtype=torch.uint8, device="cuda")), "scales"),
                      (lambda: ffn.gated_forward(x.bfloat16(), x.half(), x.half()), "gate must be"), (lambda: ffn.gated_forward(x.half(), x.half()[:, :32], x.half()), "gate must be"),
                      (lambda: ffn.gated_forward(x.half(), x.half(), x.half(), save=True, save_dtype=torch.bfloat16), "save_dtype"),
                      (lambda: ffn.gated_forward(x.half()[:, :20], x.half()[:, :20].contiguous(), x.half()[:, :20].contiguous()), "multiples of 8")):
        with pytest.raises(ValueError, match=why):
            call()
