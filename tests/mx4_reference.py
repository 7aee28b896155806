"""Microscaled 4-bit matrices and the gated block in 64 bits, value by value from their definitions (CPU tensors or any device)."""
import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x):
    """-> (codes [rows, cols] 0..15, scale bytes [rows, cols / 32]) as int64."""
    rows, cols = x.shape
    b = x.double().reshape(rows, cols // 32, 32)
    finite = torch.isfinite(b).all(2)
    top = torch.where(finite, b.abs().amax(2), torch.ones((), dtype=torch.float64, device=x.device))
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -1000, dtype=torch.int32)).clamp(-127, 125)
    v = b / torch.exp2(e.double()).unsqueeze(2)
    mag, code = v.abs(), torch.zeros_like(v, dtype=torch.int64)
    for c in range(7):                       # beyond the middle of two neighbours: the upper one; in the middle: the even code
        middle = (GRID[c] + GRID[c + 1]) / 2
        code += (mag > middle) | ((mag == middle) & (c % 2 == 1))
    code += 8 * torch.signbit(b)
    code = torch.where(finite.unsqueeze(2), code, torch.zeros_like(code))
    return code.reshape(rows, cols), torch.where(finite, e.long() + 127, torch.full_like(e, 255).long())


def values(codes, scales):
    grid = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    v = torch.where(codes >= 8, -grid[codes & 7], grid[codes & 7])
    f = torch.exp2(scales.double() - 127)
    f = torch.where(scales == 255, torch.full_like(f, float("nan")), f)
    return v * f.repeat_interleave(32, dim=1)


def unpack(packed):
    """uint8 [rows, cols / 2] -> codes [rows, cols]."""
    p = packed.long()
    return torch.stack((p & 15, p >> 4), 2).reshape(p.shape[0], -1)


def scale_index(rows, cols, device):
    """Where the tile layout keeps the scale of (row, block)."""
    r, b = torch.arange(rows, device=device)[:, None], torch.arange(cols // 32, device=device)[None, :]
    return (r // 128 * -(-cols // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def row_scales(q):
    return q.scales.long()[scale_index(q.rows, q.cols, q.device)]


def of(q):
    """The values of a zerocool_b200.ffn.Mx4."""
    return values(unpack(q.codes), row_scales(q))


def silu(g):
    return g * torch.sigmoid(g)


def gated_gradient(dh, x, gate, up, g, u):
    s = torch.sigmoid(g)
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    return dg, du, dg @ gate + du @ up, dg.T @ x, du.T @ x
