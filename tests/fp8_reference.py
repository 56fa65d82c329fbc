"""The 8-bit row format and the operators on it, from their definitions in float64 on the
CPU, for the tests: blocks of 128 columns, the least power of two s >= 2^-126 with
max|x| <= 448 s over finite values (1 for a block of zeros), x / s rounded to e4m3."""

import math

import torch

BLOCK = 128


def e4m3_round(u: torch.Tensor) -> torch.Tensor:
    """float64 u, |u| <= 448, to the nearest e4m3 number, ties to even: 3 bits behind the
    leading one down to 2^-6, steps of 2^-9 below that."""
    _, e = torch.frexp(u.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(u), e - 4)
    return torch.round(u / step) * step


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The values that the 8-bit form of rows x stands for (float64, NaN where x is not
    finite), and the scales (rows, blocks)."""
    x = x.detach().double().cpu()
    out = torch.empty_like(x)
    scales = []
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK]
        fin = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        top = fin.abs().amax(1)
        s = []
        for t in top.tolist():  # the least e with t <= 448 * 2^e, searched from its definition
            if t == 0:
                s.append(1.0)
                continue
            e = math.frexp(t)[1] - 12
            while t > 448 * 2.0 ** e:
                e += 1
            s.append(2.0 ** max(e, -126))
        s = torch.tensor(s, dtype=torch.float64)[:, None]
        q = e4m3_round(fin / s) * s
        out[:, c:c + BLOCK] = torch.where(torch.isfinite(v), q, torch.full_like(q, math.nan))
        scales.append(s)
    return out, torch.cat(scales, 1)


def norm_modulate(x, scale, shift, kind, eps):
    """float64 norm(x) * (1 + scale) + shift of x (B, T, D); vectors (B, D) or (B, T, D)."""
    x = x.detach().double().cpu()
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x if kind == "none" else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)

    def vec(v):
        v = v.detach().double().cpu()
        return v if v.dim() == 3 else v[:, None]

    if scale is not None:
        y = y * (1 + vec(scale))
    return y + vec(shift) if shift is not None else y


def gelu_tanh(v):
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))


def attention(q, k, v, heads, left_out, bias, gate, scale):
    """float64 attention of q (B, Tq, H*d) to k, v (B, Tk, H*d) over the keys that are not
    left out (B, Tk); bias (B, Tk) or None, gate logits (B, Tq, H) or None."""
    b, tq, width = q.shape
    d = width // heads
    out = torch.zeros(b, tq, width, dtype=torch.float64)
    for i in range(b):
        keep = torch.nonzero(~left_out[i]).flatten()
        if keep.numel() == 0:
            continue
        for h in range(heads):
            c = slice(h * d, (h + 1) * d)
            s = q[i, :, c].double() @ k[i, keep, c].double().t() * scale
            if bias is not None:
                s = s + bias[i, keep].double()
            o = torch.softmax(s, -1) @ v[i, keep, c].double()
            if gate is not None:
                o = o * 2 * torch.sigmoid(gate[i, :, h].double())[:, None]
            out[i, :, c] = o
    return out
