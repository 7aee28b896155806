"""Dense feed-forward operators on the GPU where their arithmetic, their plans and their arguments end (definitions: tests/mx4_reference.py;
the tolerances are those of tests/test_ffn_gpu.py, and what a test adds to them stands beside it)."""
import pytest
import torch

from tests import mx4_reference as ref
from tests.test_ffn_gpu import HALF, TINY, close, ffn, gen, randn, sums, view_of  # noqa: F401

pytestmark = pytest.mark.gpu

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
