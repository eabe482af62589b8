"""Plain restatement of the AdamW step and its 8-bit moments (torch, any device).

``step`` works in the dtype it is given (FP64 in most tests); the 8-bit helpers work on
FP32 values bit by bit, as the states are defined.
"""
import math

import torch

BLOCK = 256
U = 2.0 ** -24     # half a step of FP32, relative


def step(w, g, m, v, t, *, lr, betas, eps, weight_decay, clip=1.0):
    """One update with step number ``t`` (1, 2, ...): new (w, m, v)."""
    b1, b2 = betas
    g = g * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return w * (1 - lr * weight_decay) - update, m, v


def step_bounds(w, g, m, v, t, *, lr, betas, eps, weight_decay, clip=1.0, clipped=False,
                approximate=False):
    """Largest rounding errors of an FP32 evaluation of ``step`` (elementwise, first order).

    Units of U.  g' = clip g: 1 for the product; clip itself 4 (norm, + 1e-6, reciprocal,
    product) when it is computed.  m: each product has 1 for its constant and 1 for itself,
    the sum 1: 3 |b1 m| + (3 + e) |(1-b1) g'|, e = error of g'.  v: g'^2 has 1 + 2e, then as
    m.  sqrt halves v's error; + 1 for itself, 1 for the constant 1/sqrt(1-b2^t), 1 for the
    product, 1 for + eps, 1 for eps itself.  The quotient 1, lr/(1-b1^t) 1, the product 1.
    ``approximate``: root and quotient by hardware approximations, each within 2 units in the last
    place = 4 half steps instead of 1.
    Weights: constant 1, product 1, difference 1."""
    b1, b2 = betas
    e = 5.0 if clipped else 0.0
    gp = (g * clip).abs()
    _, m1, v1 = step(w, g, m, v, t, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, clip=clip)
    dm = U * (3 * b1 * m.abs() + (3 + e) * (1 - b1) * gp)
    dv = U * (3 * b2 * v + (4 + 2 * e) * (1 - b2) * gp * gp)
    size, root = lr / (1 - b1 ** t), v1.sqrt() / math.sqrt(1 - b2 ** t)
    den = root + eps
    more = 3 if approximate else 0
    dden = 0.5 * dv / v1.clamp_min(1e-300) * root + U * (5 + more) * den
    update = size * m1.abs() / den
    dupdate = size * dm / den + update * (dden / den + (3 + more) * U)
    dw = dupdate + U * 3 * (w.abs() + update)
    return 1.01 * dw, 1.01 * dm, 1.01 * dv


def philox(quads, t, seed):
    """Philox4x32-7 words [len(quads), 4] of counters (quad, t) and key ``seed`` (published algorithm:
    Salmon et al. 2011), in Python integers."""
    mask, out = 0xFFFFFFFF, []
    for q in quads:
        c = [q & mask, q >> 32, t & mask, t >> 32]
        k0, k1 = seed & mask, seed >> 32
        for _ in range(7):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k0, b & mask, (a >> 32) ^ c[3] ^ k1, a & mask]
            k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
        out.append(c)
    return torch.tensor(out, dtype=torch.int64)


def random_bits(first, count, t, seed):
    """(r16 of the first, r16 of the second moment) of ``count`` values whose state starts at ``first``
    (a multiple of 256)."""
    words = philox(range(first // 4, first // 4 + -(-count // 4)), t, seed).reshape(-1)[:count]
    return words & 0xFFFF, words >> 16


def _blocks(x):
    pad = -x.numel() % BLOCK
    return torch.cat([x.reshape(-1), x.new_zeros(pad)]).view(-1, BLOCK)


def table(signed):
    """Values of all 256 codes at scale 1."""
    exponents, low = (15, 16) if signed else (31, 32)
    out = []
    for code in range(256):
        c = code & 127 if signed else code
        value = 0.0 if c == 0 else (8 + c % 8) / 8 * 2.0 ** (c // 8 - exponents)
        out.append(-value if signed and code > 127 else value)
    return torch.tensor(out, dtype=torch.float64)


def decode(codes, scale_bytes, signed):
    """FP64 values of uint8 codes (any shape) with one scale byte per 256."""
    x = _blocks(table(signed)[codes.long().cpu()].reshape(-1))
    x = x * torch.exp2(scale_bytes.double().cpu() - 127).unsqueeze(1)
    return x.reshape(-1)[:codes.numel()].view(codes.shape)


def encode(x, r16, signed):
    """(codes, scale bytes) of FP32 values ``x``: of the two codes next to |x| / scale the upper one when
    the fraction between them plus r16 / 65536 reaches one."""
    x = x.float().reshape(-1).cpu()
    blocks = _blocks(x.abs())
    _, e = torch.frexp(blocks.amax(1))          # largest in [2^(e-1), 2^e)
    byte = torch.where(blocks.amax(1) < 2.0 ** -126, torch.ones_like(e), (e + 127).clamp(1, 253))
    a = (blocks.double() * torch.exp2(127.0 - byte.double()).unsqueeze(1)).reshape(-1)[:x.numel()]
    grid = table(signed)[:128 if signed else 256]
    below = torch.searchsorted(grid, a, right=True) - 1
    below = below.clamp(max=grid.numel() - 1)
    above = (below + 1).clamp(max=grid.numel() - 1)
    gap = (grid[above] - grid[below]).clamp_min(1e-300)
    fraction = (a - grid[below]) / gap
    r = r16.double()
    # above the least value the pattern adds r16 / 65536 of a step; below it r16 / 65536 < share
    up = torch.where(below > 0, fraction + r / 65536 >= 1, r < (a / grid[1]) * 65536)
    if not signed:
        up = torch.where(below == 0, a > 0, up)
    code = torch.where(up, above, below)
    if signed:
        code = code + 128 * ((x < 0) & (code > 0)).long()
    return code.to(torch.uint8), byte.to(torch.uint8)
