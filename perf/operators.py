"""Operators of the DiT block on 8-bit rows and padded text contexts: what is measured.

Three kinds of case:

  "linear"  a projection of bf16 activations with a weight held as e4m3 values and one
            power-of-two scale per row and block of 128 columns; the activations are
            quantised the same way inside the call. Optional bias, GELU (tanh form), or
            residual + gate * (..), or (norm = True) an RMS norm with adaLN scale and
            shift in front of the quantisation.
  "norm"    an RMS or LayerNorm with adaLN scale and shift whose result is held as e4m3
            rows with a power-of-two scale per block of 128 columns; the values that the
            rows stand for come back.
  "cross"   attention of Tq queries to Tk encoder states of another length under a
            per-sample key mask (boolean, or additive), with the optional per-(token,
            head) output gate 2 * sigmoid(logit). A sample without any key gives zeros.

The 8-bit form of a row x: for every 128 columns, s is the smallest power of two with
max|x| <= 448 s (at least 2^-126; 1 for a block of zeros), and each value is x / s rounded
to the nearest e4m3 number.
"""

import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = Path(__file__).resolve().parents[1] / "ltx-nv_b200"
EPS = 1e-6
BLOCK = 128


def _nn():
    """The framework's module of building blocks (flat modules, as its users import them)."""
    if str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    import ltx_nn

    return ltx_nn


# ------------------------------------------------------------------------------- cases


def _linear(name, b, t, k, n, epilogue="none", bias=False, norm=False):
    return {"name": name, "kind": "linear", "B": b, "T": t, "K": k, "N": n, "epilogue": epilogue, "bias": bias,
            "norm": norm}


def _norm(name, b, t, d, norm="rms", dtype="bf16", per_token=False):
    return {"name": name, "kind": "norm", "B": b, "T": t, "D": d, "norm": norm, "dtype": dtype,
            "per_token": per_token}


def _cross(name, b, tq, tk, h, d, mask, gate=True, dtype="bf16"):
    return {"name": name, "kind": "cross", "B": b, "Tq": tq, "Tk": tk, "H": h, "d": d, "mask": mask, "gate": gate,
            "dtype": dtype}


def listed():
    return [
        # The feed-forward of a 2048-wide video block on one CFG pair of 6144 latent tokens:
        # norm + adaLN in front of the first product, gated residual after the second.
        _linear("ffn in, video", 2, 6144, 2048, 8192, epilogue="gelu", bias=True, norm=True),
        _linear("ffn out, video", 2, 6144, 8192, 2048, epilogue="residual", bias=True),
        # q, k, v and gate logits of the 126-token audio stream in one packed projection.
        _linear("packed qkv, audio", 2, 126, 2048, 6176, bias=True),
        # adaLN-single: one row per sample of the CFG pair, where the weight's bytes count.
        _linear("adaln, one row a sample", 2, 1, 2048, 12288, bias=True),
        # Odd sizes: a last block of 13 columns, a last output tile of a few columns.
        _linear("odd sizes", 1, 1001, 1037, 1371, bias=True),
        # The normalised operand of one block's projections, and the audio stream's with a
        # modulation of its own for every token, in the accuracy mode's type.
        _norm("norm to 8 bits, video", 2, 6144, 2048),
        _norm("norm to 8 bits, audio", 2, 126, 2048, norm="layer", dtype="f32", per_token=True),
        # Video tokens to a 1024-token text context: prompts padded on the left.
        _cross("text context, video", 2, 6144, 1024, 32, 64, "left"),
        # The guidance batch of four at 128 columns a head, an additive mask.
        _cross("text context, wide heads", 4, 1536, 1024, 32, 128, "additive"),
        # Audio tokens to a short prompt with tokens dropped anywhere; one sample is empty.
        _cross("text context, audio", 4, 126, 250, 32, 64, "holes"),
        # One query token against a long context.
        _cross("one query token", 2, 1, 4099, 32, 128, "right", gate=False),
        # The accuracy mode.
        _cross("text context, fp32", 1, 480, 200, 8, 64, "left", dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "cross", "cross"])
    if kind == "linear":
        while True:
            b = rng.choice([1, 2, 4])
            t, k, n = _log(rng, 1, 6144), _log(rng, 16, 8192), _log(rng, 8, 12288)
            norm = rng.random() < 0.3
            if norm:
                k = 8 * max(1, k // 8)
            if 1e4 < 2.0 * b * t * k * n <= 4.0e11:
                break
        c = _linear("", b, t, k, n, epilogue=rng.choice(["none", "gelu", "residual"]), bias=rng.random() < 0.5,
                    norm=norm)
    elif kind == "norm":
        while True:
            b, t, d = rng.choice([1, 2, 4]), _log(rng, 1, 6144), 8 * _log(rng, 4, 1024)
            if b * t * d <= 2.5e7:
                break
        c = _norm("", b, t, d, norm=rng.choice(["rms", "layer"]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                  per_token=rng.random() < 0.3)
    else:
        while True:
            b, h, d = rng.choice([1, 2, 3, 4]), rng.choice([4, 8, 16, 32]), rng.choice([64, 128])
            tq, tk = _log(rng, 1, 6144), _log(rng, 1, 4096)
            dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
            if b * h * tq * tk * d <= (1.5e9 if dtype == "f32" else 2.5e10):
                break
        c = _cross("", b, tq, tk, h, d, rng.choice(["left", "right", "holes", "additive"]), gate=rng.random() < 0.5,
                   dtype=dtype)
    del c["name"]
    return c


# ------------------------------------------------------------------------------ inputs


def _dtype(case):
    return torch.float32 if case.get("dtype") == "f32" else torch.bfloat16


def _to_blocks(x):
    """(..., K) -> (..., blocks, 128), the last block filled up with zeros."""
    pad = -x.shape[-1] % BLOCK
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], dim=-1)
    return x.reshape(*x.shape[:-1], -1, BLOCK)


def _quantize(x):
    """e4m3 values and power-of-two scales (..., blocks) of float32 rows."""
    blocks = _to_blocks(x)
    m, e = torch.frexp(blocks.abs().amax(dim=-1))  # 448 = 0.875 * 2^9, m in [0.5, 1)
    e = torch.where(m == 0, 0, (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126))
    s = ((e.to(torch.int32) + 127) << 23).view(torch.float32)  # 2^e by its bits: exact
    q = (blocks / s[..., None]).to(torch.float8_e4m3fn)
    return q.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]], s


def _values(q, s):
    """The float32 values that e4m3 numbers q (..., K) with scales s (..., blocks) stand for."""
    return (_to_blocks(q.to(torch.float32)) * s[..., None]).reshape(*q.shape[:-1], -1)[..., :q.shape[-1]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype or _dtype(case))

    s = {"case": dict(case)}
    if case["kind"] == "linear":
        b, t, k, n = case["B"], case["T"], case["K"], case["N"]
        # a residual stream's channels differ in size; a few are far larger than the rest
        channel = 1.0 + 15.0 * (torch.rand(k, generator=g, device=dev) < 0.01)
        s["x"] = (torch.randn(b, t, k, generator=g, device=dev) * channel).to(torch.bfloat16)
        s["w"], s["w_scale"] = _quantize(torch.randn(n, k, generator=g, device=dev) * k ** -0.5)
        s["bias"] = randn(n, std=0.1) if case["bias"] else None
        if case["epilogue"] == "residual":
            s["residual"] = randn(b, t, n)
            s["gate"] = randn(b, n, std=0.5)
        if case["norm"]:
            s["scale"], s["shift"] = randn(b, k, std=0.2), randn(b, k, std=0.2)
    elif case["kind"] == "norm":
        b, t, d = case["B"], case["T"], case["D"]
        s["x"] = randn(b, t, d, std=2.0) + 0.25
        shape = (b, t, d) if case["per_token"] else (b, d)
        s["scale"], s["shift"] = randn(*shape, std=0.2), randn(*shape, std=0.2)
    else:
        b, tq, tk, h, d = (case[f] for f in ("B", "Tq", "Tk", "H", "d"))
        inner = h * d
        # q and the gate logits are columns of one packed projection, k and v of another
        qg = randn(b, tq, inner + -(-h // 8) * 8)
        kv = randn(b, tk, 2 * inner)
        s["q"], s["k"], s["v"] = qg[..., :inner], kv[..., :inner], kv[..., inner:]
        s["gate"] = qg[..., inner:inner + h] if case["gate"] else None
        length = torch.randint(1, tk + 1, (b, 1), generator=g, device=dev)
        at = torch.arange(tk, device=dev)[None, :]
        if case["mask"] == "left":
            mask = at >= tk - length
        elif case["mask"] == "right":
            mask = at < length
        else:
            mask = torch.rand(b, tk, generator=g, device=dev) < 0.7
            if case["mask"] == "holes" and b > 1:
                mask[b - 1] = False  # a sample whose prompt is empty
        if case["mask"] == "additive":
            bias = 0.5 * torch.randn(b, tk, generator=g, device=dev)
            lowest = torch.finfo(_dtype(case)).min
            mask = torch.where(mask, bias.to(_dtype(case)), torch.full_like(bias, lowest).to(_dtype(case)))
        s["mask"] = mask
    return s


# --------------------------------------------------------------------------- plain form


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


def _modulated_norm(x, scale, shift, kind):
    """float32 norm(x) * (1 + scale) + shift; scale and shift (B, D) or (B, T, D)."""
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    scale, shift = ((v if v.dim() == 3 else v[:, None]).to(x.dtype) for v in (scale, shift))
    return y * (1 + scale) + shift


def _left_out(mask):
    """(B, Tk) truth values: keys that no query attends to."""
    if mask.dtype == torch.bool:
        return ~mask
    return mask <= torch.finfo(mask.dtype).min / 2


def _plain_linear(s):
    case = s["case"]
    x = s["x"].to(torch.float32)
    if case["norm"]:
        x = _modulated_norm(x, s["scale"], s["shift"], "rms")
    y = torch.matmul(_values(*_quantize(x)), _values(s["w"], s["w_scale"]).t())
    if s["bias"] is not None:
        y = y + s["bias"].to(torch.float32)
    if case["epilogue"] == "gelu":
        y = _gelu(y)
    elif case["epilogue"] == "residual":
        y = s["residual"].to(torch.float32) + s["gate"].to(torch.float32)[:, None] * y
    return y.to(torch.bfloat16)


def _plain_norm(s):
    y = _modulated_norm(s["x"].to(torch.float32), s["scale"], s["shift"], s["case"]["norm"])
    return _values(*_quantize(y)).to(torch.bfloat16)


def _heads(x, h):
    b, t, w = x.shape
    return x.to(torch.float32).reshape(b, t, h, w // h).transpose(1, 2)


def _plain_cross(s):
    case = s["case"]
    h, d = case["H"], case["d"]
    q, k, v = (_heads(s[n], h) for n in ("q", "k", "v"))
    logits = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    out = _left_out(s["mask"])[:, None, None, :]
    if s["mask"].dtype != torch.bool:
        logits = logits + s["mask"].to(torch.float32)[:, None, None, :]
    logits = logits.masked_fill(out, -torch.inf)
    top = logits.amax(dim=-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    if s["gate"] is not None:
        o = o * (2 / (1 + torch.exp(-s["gate"].to(torch.float32)))).transpose(1, 2)[..., None]
    return o.transpose(1, 2).reshape(s["q"].shape).to(_dtype(case))


# ------------------------------------------------------------------------------ the pass


def _own_linear(s):
    nn, case = _nn(), s["case"]
    if "weight" not in s:  # the handle that a program builds once when it loads its weights
        s["weight"] = nn.Fp8Rows.from_parts(s["w"], s["w_scale"])
    x = s["x"]
    if case["norm"]:
        x = nn.norm_modulate_fp8(x, scale=s["scale"], shift=s["shift"], kind="rms", eps=EPS)
    return nn.linear_fp8(x, s["weight"], s["bias"], activation="gelu_tanh" if case["epilogue"] == "gelu" else None,
                         residual=s.get("residual"), gate=s.get("gate"))


def _own_norm(s):
    rows = _nn().norm_modulate_fp8(s["x"], scale=s["scale"], shift=s["shift"], kind=s["case"]["norm"], eps=EPS)
    return rows.dequantize(torch.bfloat16)


def _own_cross(s):
    return _nn().cross_attention(s["q"], s["k"], s["v"], s["case"]["H"], mask=s["mask"], gate_logits=s["gate"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "cross": _own_cross}[kind](state)
    return {"linear": _plain_linear, "norm": _plain_norm, "cross": _plain_cross}[kind](state)


# --------------------------------------------------------------------------------- work


def work(case):
    if case["kind"] == "linear":
        m, k, n = case["B"] * case["T"], case["K"], case["N"]
        size = 2 * m * k + n * k + n * -(-k // BLOCK) + 2 * m * n + (2 * n if case["bias"] else 0)
        if case["epilogue"] == "residual":
            size += 2 * m * n + 2 * case["B"] * n
        if case["norm"]:
            size += 4 * case["B"] * k
        return {"bytes": size, "flops": 2 * m * n * k}
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "norm":
        m, d = case["B"] * case["T"], case["D"]
        mod = 2 * e * d * (m if case["per_token"] else case["B"])
        return {"bytes": e * m * d + mod + 2 * m * d, "flops": 8 * m * d}
    b, tq, tk, h, d = (case[f] for f in ("B", "Tq", "Tk", "H", "d"))
    # lengths are uniform in 1..Tk, so about half of the keys take part; 0.7 where dropped singly
    keep = 0.5 if case["mask"] in ("left", "right") else 0.7
    size = e * (2 * b * tq * h * d + 2 * b * int(keep * tk + 0.5) * h * d + (b * tq * h if case["gate"] else 0))
    size += b * tk * (e if case["mask"] == "additive" else 1)
    return {"bytes": size, "flops": int(4 * b * h * tq * keep * tk * d) + 1}


# -------------------------------------------------------------------- definition, 64 bits


def _pow2(e):
    """2^e in float64 for whole numbers e, by its bits: exact."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rows(y):
    """The values of the 8-bit form of float64 rows, block by block from its definition."""
    out = torch.empty_like(y)
    for c in range(0, y.shape[-1], BLOCK):
        v = y[..., c:c + BLOCK]
        top = v.abs().amax(dim=-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448))
        e = torch.where(top > 448 * _pow2(e), e + 1, torch.where(top <= 448 * _pow2(e - 1), e - 1, e))
        s = _pow2(torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-126))
        u = v / s
        # e4m3: 3 bits after the leading one down to 2^-6, steps of 2^-9 below
        step = _pow2(torch.frexp(u.abs().clamp(min=2.0 ** -6)).exponent - 4)
        out[..., c:c + BLOCK] = torch.round(u / step) * step * s
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("linear", "norm"):
        x = s["x"].double()
        if case["kind"] == "norm" or case["norm"]:
            if case.get("norm") == "layer":
                y = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, keepdim=True, correction=0) + EPS)
            else:
                y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
            sc, sh = s["scale"].double(), s["shift"].double()
            x = torch.addcmul(sh if sh.dim() == 3 else sh[:, None], y, 1 + (sc if sc.dim() == 3 else sc[:, None]))
        x = _exact_rows(x)
        if case["kind"] == "norm":
            return x
        w = s["w"].double() * s["w_scale"].double().repeat_interleave(BLOCK, dim=1)[:, :case["K"]]
        y = torch.einsum("btk,nk->btn", x, w)
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["epilogue"] == "gelu":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        elif case["epilogue"] == "residual":
            y = torch.addcmul(s["residual"].double(), s["gate"].double()[:, None], y)
        return y
    h, d = case["H"], case["d"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i in range(case["B"]):
        keys = torch.nonzero(~_left_out(s["mask"][i])).flatten()
        if keys.numel() == 0:
            continue
        for j in range(h):
            c = slice(j * d, (j + 1) * d)
            a = s["q"][i, :, c].double() @ s["k"][i, keys, c].double().t() / math.sqrt(d)
            if s["mask"].dtype != torch.bool:
                a = a + s["mask"][i, keys].double()
            o[i, :, c] = torch.softmax(a, dim=-1) @ s["v"][i, keys, c].double()
            if s["gate"] is not None:
                o[i, :, c] *= 2 * torch.sigmoid(s["gate"][i, :, j].double())[:, None]
    return o
