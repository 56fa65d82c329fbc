"""B200-native neural building blocks of the LTX DiT (drop-in for lipaul/ltx-nv
standalone/ltx_nn.py).

Same module / function names, constructor arguments, parameter names and call
signatures as the reference; every forward runs libltxb200's sm_100a kernels through
_native (the reference runs cuBLAS + cuDNN SDPA + torch element-wise ops). Activations
are (B, T, D) CUDA tensors in float32 (the accuracy mode) or bfloat16.

Layout choices that differ inside (not at the API):
  * RoPE tables are kept token-major, (T, H*d/2), shared by all samples whose positions
    agree; precompute_freqs_cis returns them as (B, H, T, d/2) views of that storage so
    callers see the reference's shapes.
  * Attention and FeedForward modules may hold their weights in 8 bits as well
    (quantize_fp8): their products then run on 8-bit rows (linear_fp8).
  * q, k, v and the gate logits of a self-attention are one packed (3D+H, D) weight:
    the module's own to_q / to_k / to_v / to_gate_logits parameters become views into
    it, so state_dict() is unchanged and nothing is stored twice.
"""

from __future__ import annotations

import functools
import math

import numpy
import torch

import _native as nat
from _native import Fp8Rows


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x.reshape(-1, x.shape[-1])


def rms_norm(x: torch.Tensor, eps: float = 1e-6, weight: torch.Tensor | None = None) -> torch.Tensor:
    """ltx_nn.py:18-19. weight=None only (the learned-weight form is Attention's q/k norm)."""
    if weight is not None:
        raise NotImplementedError("rms_norm with a weight runs fused inside Attention (ltx_qk_norm_rope)")
    xr = _rows(x.contiguous())
    y = torch.empty_like(xr)
    nat.norm_modulate(xr, y, xr.shape[0], nat.LTX_NORM_RMS, eps, None)
    return y.view_as(x)


def sdpa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor | None = None) -> torch.Tensor:
    """ltx_nn.py:22-26: q, k, v (B, H, T, d) -> (B, H, T, d), non-causal. mask: one that does
    not depend on the query or the head, (B or 1, 1, 1, Tk), (B or 1, Tk) or (Tk,), bool
    (True: the key takes part) or additive; see cross_attention."""
    b, h, tq, d = q.shape
    tk = k.shape[2]

    def rows(x, t):
        return x.transpose(1, 2).reshape(b, t, h * d)

    if mask is not None:
        o = cross_attention(rows(q, tq), rows(k, tk), rows(v, tk), h, mask=mask)
        return o.view(b, tq, h, d).transpose(1, 2)
    qt, kt, vt = (rows(x, t).reshape(b * t, h * d).contiguous() for x, t in ((q, tq), (k, tk), (v, tk)))
    o = torch.empty_like(qt)
    nat.attention(qt, kt, vt, o, b, tq, tk, h, d, d ** -0.5, None)
    return o.view(b, tq, h, d).transpose(1, 2)


# ---------------------------------------------------------------------------------------
# Attention to another sequence under a key mask
# ---------------------------------------------------------------------------------------


def key_mask(mask: torch.Tensor, batch: int, tk: int) -> torch.Tensor:
    """A mask over the keys as the (B or 1, Tk) row-major view that nat.attention_masked
    takes, from (Tk,), (B or 1, Tk) or (B or 1, 1, 1, Tk)."""
    if mask.dim() == 4:
        if mask.shape[1] != 1 or mask.shape[2] != 1:
            raise NotImplementedError(f"masks that depend on the query or the head, got {tuple(mask.shape)}")
        mask = mask[:, 0, 0]
    elif mask.dim() == 1:
        mask = mask[None]
    if mask.dim() != 2 or mask.shape[1] != tk or mask.shape[0] not in (1, batch):
        raise ValueError(f"a key mask is ({batch} or 1, 1, 1, {tk}), ({batch} or 1, {tk}) or ({tk},), got "
                         f"{tuple(mask.shape)}")
    return mask if tk == 1 or mask.stride(1) == 1 else mask.contiguous()


def _row_major(x: torch.Tensor) -> torch.Tensor:
    """x (..., W) as a (rows, W) row-major view; a copy only where there is no such view, or
    where its rows overlap (expanded tensors)."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(1) == 1 and x2.stride(0) >= x2.shape[1]:
        return x2
    return x2.clone(memory_format=torch.contiguous_format)  # contiguous() keeps a single row's odd strides


def _token_rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x (B, T, W) as a tensor and its row stride: x itself where its B * T rows are evenly
    spaced, without the cost of a view; else _row_major's."""
    b, t, w = x.shape
    sb, st, sw = x.stride()
    if sw == 1 and t > 1 and st >= w and (b == 1 or sb == t * st):
        return x, st
    x2 = _row_major(x)
    return x2, x2.stride(0)


def _spans_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the addresses from the first to the last element of a and of b overlap."""
    if not a.numel() or not b.numel():
        return False
    pa, pb = a.data_ptr(), b.data_ptr()
    na, nb = (1 + sum([(n - 1) * st for n, st in zip(t.shape, t.stride())]) for t in (a, b))
    return pa < pb + nb * b.element_size() and pb < pa + na * a.element_size()


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, heads: int,
                    mask: torch.Tensor | None = None, gate_logits: torch.Tensor | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * scale + mask) v per sample and head: q (B, Tq, H*d), k and v (B, Tk,
    H*d) token-major (column views of packed projections are taken as they are), out (B, Tq,
    H*d), optionally times 2 * sigmoid(gate_logits), gate_logits (B, Tq, H) (ltx_nn.py:22-26,
    231-235).

    mask (key_mask's shapes): bool, True where a key takes part; or float32 / bfloat16, added
    to the scores, a key being left out where it is at or below half of the type's lowest
    finite value. What k and v hold at a key that is left out does not matter. A sample
    without any key gives zeros (torch's softmax would give NaN, or a mean over the padding
    for masks of the lowest value). out may be q, but not overlap k or v. Without a mask this
    is the framework's attention."""
    b, tq, width = q.shape
    tk = k.shape[1]
    if heads <= 0 or width % heads:
        raise ValueError(f"the width {width} is not a multiple of {heads} heads")
    if k.shape != (b, tk, width) or v.shape != (b, tk, width):
        raise ValueError(f"k and v must be ({b}, Tk, {width}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if gate_logits is not None and gate_logits.shape != (b, tq, heads):
        raise ValueError(f"gate_logits must be ({b}, {tq}, {heads}), got {tuple(gate_logits.shape)}")
    if out is None:
        out = torch.empty(b, tq, width, device=q.device, dtype=q.dtype)
    elif tuple(out.shape) != (b, tq, width) or not out.is_contiguous() or out.dtype != q.dtype:
        raise ValueError(f"out must be a contiguous {q.dtype} ({b}, {tq}, {width}) tensor")
    elif _spans_overlap(out, k) or _spans_overlap(out, v):
        raise ValueError("out must not overlap k or v, which other queries still read")
    if mask is not None:
        mask = key_mask(mask, b, tk)
    if out.numel() == 0:
        return out
    if tk == 0:
        return out.zero_()
    d = width // heads
    scale = d ** -0.5 if scale is None else float(scale)
    if mask is None:
        nat.attention(_row_major(q), _row_major(k), _row_major(v), out.view(b * tq, width), b, tq, tk, heads, d, scale,
                      _row_major(gate_logits) if gate_logits is not None else None)
    else:
        nat.attention_masked_rows(*_token_rows(q), *_token_rows(k), *_token_rows(v), out, width, b, tq, tk, heads, d,
                                  scale, mask, *(_token_rows(gate_logits) if gate_logits is not None else (None, 0)))
    return out


# ---------------------------------------------------------------------------------------
# 8-bit rows: linear layers and the norm in front of them
# ---------------------------------------------------------------------------------------


def quantize_fp8(x: torch.Tensor, out: Fp8Rows | None = None) -> Fp8Rows:
    """x (..., K) float32 or bfloat16 -> its 8-bit rows: e4m3 values with a power-of-two scale
    per 128 columns. Weights (N, K) are quantised with it once. out: rows of x's shape to
    write to instead of new ones."""
    if x.shape[-1] == 0:
        raise ValueError("x has no columns")
    if out is not None and out.shape != tuple(x.shape):
        raise ValueError(f"out is {out.shape}, x is {tuple(x.shape)}")
    return nat.quantize_fp8(_row_major(x), x.shape, out)


def _modulation(x: torch.Tensor, shift: torch.Tensor | None, scale: torch.Tensor | None):
    """nat.Modulation of shift / scale vectors given per sample (B, D) or per token (B, T, D),
    and the tensors that it points to. One descriptor addresses both vectors from the lower
    of their addresses, with one stride; vectors that do not share it are copied."""
    b, t, d = x.shape
    vecs = [v for v in (shift, scale) if v is not None]
    if not vecs:
        return None, vecs
    first = vecs[0]
    for vec in vecs:
        if vec.shape != first.shape or vec.shape not in ((b, d), (b, t, d)):
            raise ValueError(f"shift and scale must be ({b}, {d}) or ({b}, {t}, {d}), one like the other, got "
                             f"{tuple(vec.shape)}")
        if vec.dtype != x.dtype or vec.get_device() != x.get_device():
            raise ValueError(f"shift and scale must be {x.dtype} on {x.device}")
    st = first.stride()
    if any([v.stride() != st or v.data_ptr() % 32 for v in vecs]) or st[-1] != 1 or any([i % 8 for i in st[:-1]]):
        vecs = [torch.empty(v.shape, dtype=v.dtype, device=v.device).copy_(v) for v in vecs]
        st = vecs[0].stride()
    ptrs = [v.data_ptr() for v in vecs]
    m = nat.Modulation()
    m.mod = base = min(ptrs)
    m.mod_ld_batch, m.mod_ld_tok = st[0], (st[1] if len(st) == 3 else 0)
    size = x.element_size()
    if shift is not None:
        m.has_shift, m.shift_mod_off = 1, (ptrs[0] - base) // size
    if scale is not None:
        m.has_scale, m.scale_mod_off = 1, (ptrs[-1] - base) // size
    return m, vecs


_NORM_KINDS = {"rms": nat.LTX_NORM_RMS, "layer": nat.LTX_NORM_LAYER, "none": nat.LTX_NORM_NONE}


def norm_modulate_fp8(x: torch.Tensor, scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
                      kind: str = "rms", eps: float = 1e-6) -> Fp8Rows:
    """norm(x) * (1 + scale) + shift of x (B, T, D) as 8-bit rows, the operand of linear_fp8:
    fp32 arithmetic and one rounding. scale and shift (B, D) or (B, T, D) in x's type; kind
    "rms", "layer" or "none"; D a multiple of 8."""
    if kind not in _NORM_KINDS:
        raise ValueError(f"kind must be one of {sorted(_NORM_KINDS)}, got {kind!r}")
    if x.dim() != 3:
        raise ValueError(f"expected (batch, tokens, width), got {tuple(x.shape)}")
    x2 = _row_major(x)
    mod, held = _modulation(x, shift, scale)
    out = nat.norm_modulate_fp8(x2, max(x.shape[1], 1), _NORM_KINDS[kind], eps, mod, x.shape)
    del held  # the vectors live until the launch; the allocator keeps stream order after it
    return out


_ACTIVATIONS = {None: nat.EPI_NONE, "gelu_tanh": nat.EPI_GELU_TANH, "silu": nat.EPI_SILU}


def linear_fp8(x, weight: Fp8Rows, bias: torch.Tensor | None = None, *, activation: str | None = None,
               residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """activation(x W^T + bias), or residual + gate * (x W^T + bias), with both operands in
    8-bit rows and fp32 sums, rounded once to `dtype`.

    x: (..., K) float32 or bfloat16, quantised here (quantize_fp8), or 8-bit rows already
    (norm_modulate_fp8). weight: (N, K) Fp8Rows. The result is (..., N) in `dtype` (default:
    x's type; for 8-bit rows the residual's, or bfloat16). gate: (B, N) per sample or (B, T,
    N) per token of a (B, T, N) result; bias, residual and gate are in `dtype`. out may be the
    residual itself, and x too."""
    if not isinstance(weight, Fp8Rows):
        raise TypeError("weight must be Fp8Rows (quantize_fp8 or Fp8Rows.from_parts)")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_ACTIVATIONS)}, got {activation!r}")
    if gate is not None and residual is None:
        raise ValueError("a gate needs a residual")
    if activation is not None and residual is not None:
        raise ValueError("an activation and a residual exclude each other")
    n = weight.rows
    if dtype is None:
        dtype = x.dtype if isinstance(x, torch.Tensor) else residual.dtype if residual is not None else torch.bfloat16
    if x.shape[-1] != weight.cols or len(weight.shape) != 2:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight is {weight.shape}")
    if weight.cols == 0:
        raise ValueError("the weight has no columns")
    lead = x.shape[:-1]
    shape = (*lead, n)
    dev = x.device
    for name, t, want in (("bias", bias, (n,)), ("residual", residual, shape), ("out", out, shape)):
        if t is not None and (t.shape != want or t.dtype != dtype or t.device != dev):
            raise ValueError(f"{name} must be {dtype} {want} on {dev}, got {t.dtype} {tuple(t.shape)}")
    kind, rpb, mod = _ACTIVATIONS[activation], 1, None
    if residual is not None:
        kind = nat.EPI_GATE_RESIDUAL
        residual2 = _row_major(residual)
        if gate is not None:
            if residual.dim() != 3 or tuple(gate.shape) not in ((lead[0], n), shape):
                raise ValueError(f"gate must be (B, N) or (B, T, N) of a (B, T, N) residual, got {tuple(gate.shape)}")
            if gate.dtype != dtype or gate.device != dev:
                raise ValueError(f"gate must be {dtype} on {dev}")
            gate = gate.contiguous()
            rpb = max(lead[1], 1)
            per_tok = gate.dim() == 3
            mod = nat.modulation(None, gate, shift=None, scale=(0, 0), mod_ld_batch=rpb * n if per_tok else n,
                                 mod_ld_tok=n if per_tok else 0)
    if out is None:
        out = torch.empty(shape, device=dev, dtype=dtype)
    elif not out.is_contiguous():
        raise ValueError("out must be contiguous")
    epi = nat.epilogue(kind, bias=bias.contiguous() if bias is not None else None,
                       residual=residual2 if residual is not None else None, gate=mod, rows_per_batch=rpb)
    if isinstance(x, Fp8Rows):
        nat.linear_fp8(x, weight, out, epi)
    else:
        nat.quantize_linear_fp8(_row_major(x), weight, out, epi)
    return out


def project(x, weight: torch.Tensor, weight8: Fp8Rows | None, out: torch.Tensor, epi: nat.Epilogue) -> None:
    """out = epilogue(x W^T) of a module's projection: on 8-bit rows when the weight has an
    8-bit form (x may then be 8-bit rows already), else in x's type."""
    if weight8 is None:
        nat.linear(x, weight, out, epi)
    elif isinstance(x, Fp8Rows):
        nat.linear_fp8(x, weight8, out, epi)
    else:
        nat.quantize_linear_fp8(x, weight8, out, epi)


def norm_into(x: torch.Tensor, h: torch.Tensor, rows_per_batch: int, kind: int, eps: float,
              mod: nat.Modulation | None, fp8: bool):
    """norm_modulate of x (rows, D) as the operand of project: written to h, or as 8-bit rows."""
    if fp8:
        return nat.norm_modulate_fp8(x, rows_per_batch, kind, eps, mod)
    nat.norm_modulate(x, h, rows_per_batch, kind, eps, mod)
    return h


# ---------------------------------------------------------------------------------------
# RoPE (split type)
# ---------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=8)
def generate_freq_grid_np(theta: float, n_axes: int, inner_dim: int) -> torch.Tensor:
    """ltx_nn.py:34-46: float64 frequency grid theta^linspace(0,1) * pi/2, as float32."""
    n_elem = 2 * n_axes
    pw = numpy.power(theta, numpy.linspace(0.0, 1.0, inner_dim // n_elem, dtype=numpy.float64))
    return torch.as_tensor(pw * math.pi / 2, dtype=torch.float32)


@functools.lru_cache(maxsize=8)
def generate_freq_grid_pytorch(theta: float, n_axes: int, inner_dim: int) -> torch.Tensor:
    """ltx_nn.py:49-60 (float32 grid)."""
    n_elem = 2 * n_axes
    idx = theta ** torch.linspace(math.log(1.0, theta), math.log(theta, theta), inner_dim // n_elem,
                                  dtype=torch.float32)
    return idx.to(torch.float32) * math.pi / 2


class RopeTables:
    """cos/sin tables (T, dim/2) per distinct sample, token-major, in the activation dtype.

    `ld_batch` is the element stride between samples (0 when every sample shares the
    same positions, the CFG case). `heads` is the head count the reference splits the
    table with (it fixes which RoPE pairs (j, j + d/2) belong together)."""

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, ld_batch: int, heads: int):
        self.cos, self.sin, self.ld_batch, self.heads = cos, sin, ld_batch, heads

    def reference_layout(self, batch: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(B, H, T, d/2) views matching precompute_freqs_cis's return value."""
        t, half = self.cos.shape[-2], self.cos.shape[-1]
        h = self.heads

        def view(x):
            x = x.view(-1, t, h, half // h)
            if x.shape[0] == 1:
                x = x.expand(batch, -1, -1, -1)
            return x.permute(0, 2, 1, 3)

        return view(self.cos), view(self.sin)


def rope_tables(positions: torch.Tensor, dim: int, out_dtype: torch.dtype, theta: float, max_pos: list,
                heads: int, double_precision: bool = True) -> RopeTables:
    """Native RoPE tables for positions (B, n_axes, T, 2) (ltx_nn.py:63-96)."""
    b, n_axes, t, _ = positions.shape
    gen = generate_freq_grid_np if double_precision else generate_freq_grid_pytorch
    dev = positions.device
    freqs = gen(float(theta), n_axes, dim).to(dev)
    mp = torch.tensor([float(m) for m in max_pos[:n_axes]], dtype=torch.float32, device=dev)
    pos = positions.to(torch.float32)
    shared = b == 1 or bool((pos == pos[:1]).all())
    nb = 1 if shared else b
    cos = torch.empty(nb, t, dim // 2, device=dev, dtype=out_dtype)
    sin = torch.empty_like(cos)
    for i in range(nb):
        nat.rope_tables(pos[i].contiguous(), freqs, mp, dim, cos[i], sin[i])
    return RopeTables(cos, sin, 0 if shared else t * (dim // 2), heads)


def precompute_freqs_cis(indices_grid: torch.Tensor, dim: int, out_dtype: torch.dtype, theta: float = 10000.0,
                         max_pos: list[int] | None = None, use_middle_indices_grid: bool = True,
                         num_attention_heads: int = 32,
                         double_precision: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """ltx_nn.py:63-96 -> (cos, sin) of shape (B, H, T, dim/2/H) (views of token-major tables)."""
    if not use_middle_indices_grid or indices_grid.ndim != 4:
        raise NotImplementedError("only the mid-point (B, n_axes, T, 2) position grid is used by LTX")
    tabs = rope_tables(indices_grid, dim, out_dtype, theta, max_pos or [20, 2048, 2048], num_attention_heads,
                       double_precision)
    return tabs.reference_layout(indices_grid.shape[0])


def _tables_from_reference_layout(freqs_cis) -> RopeTables:
    cos, sin = freqs_cis
    if isinstance(freqs_cis, RopeTables):
        return freqs_cis
    b, h, t, q = cos.shape
    base_c = cos.permute(0, 2, 1, 3)
    base_s = sin.permute(0, 2, 1, 3)
    if base_c.stride(0) == 0 or b == 1:
        c = base_c[:1].reshape(1, t, h * q).contiguous()
        s = base_s[:1].reshape(1, t, h * q).contiguous()
        return RopeTables(c, s, 0, h)
    c = base_c.reshape(b, t, h * q).contiguous()
    s = base_s.reshape(b, t, h * q).contiguous()
    return RopeTables(c, s, t * h * q, h)


def apply_split_rotary_emb(x: torch.Tensor, freqs_cis) -> torch.Tensor:
    """ltx_nn.py:99-115 (no norm): rotates pairs (j, j + d/2) of each head."""
    tabs = _tables_from_reference_layout(freqs_cis)
    if x.ndim == 4:
        b, h, t, d = x.shape
        xt = x.transpose(1, 2).reshape(b * t, h * d).contiguous()
    else:
        b, t, dd = x.shape
        xt = x.reshape(b * t, dd).contiguous()
    heads = tabs.heads
    hd = xt.shape[1] // heads
    # weight=None: rotation only (no q/k RMSNorm).
    nat.qk_norm_rope(xt, t, heads, hd, None, 0.0, tabs.cos.reshape(-1, xt.shape[1] // 2),
                     tabs.sin.reshape(-1, xt.shape[1] // 2), rope_ld_batch=tabs.ld_batch)
    if x.ndim == 4:
        return xt.view(b, t, h, d).transpose(1, 2)
    return xt.view_as(x)


# ---------------------------------------------------------------------------------------
# Timestep embedding / adaLN-single
# ---------------------------------------------------------------------------------------


class TimestepEmbedder(torch.nn.Module):
    """ltx_nn.py:123-130: linear_2(silu(linear_1(x)))."""

    def __init__(self, in_channels: int, time_embed_dim: int):
        super().__init__()
        self.linear_1 = torch.nn.Linear(in_channels, time_embed_dim)
        self.linear_2 = torch.nn.Linear(time_embed_dim, time_embed_dim)

    def forward(self, x: torch.Tensor, silu_out: torch.Tensor | None = None) -> torch.Tensor:
        h = torch.empty(x.shape[0], self.linear_1.out_features, device=x.device, dtype=x.dtype)
        nat.linear(x, self.linear_1.weight, h, nat.epilogue(nat.EPI_SILU, bias=self.linear_1.bias))
        out = torch.empty(x.shape[0], self.linear_2.out_features, device=x.device, dtype=x.dtype)
        nat.linear(h, self.linear_2.weight, out, nat.epilogue(bias=self.linear_2.bias))
        if silu_out is not None:
            nat.linear(h, self.linear_2.weight, silu_out, nat.epilogue(nat.EPI_SILU, bias=self.linear_2.bias))
        return out


class CombinedTimestepEmbeddings(torch.nn.Module):
    """ltx_nn.py:133-145: 256-dim [cos, sin] sinusoid -> TimestepEmbedder."""

    def __init__(self, embedding_dim: int):
        super().__init__()
        self.timestep_embedder = TimestepEmbedder(256, embedding_dim)

    def forward(self, timestep: torch.Tensor, hidden_dtype: torch.dtype, scale: float = 1.0,
                silu_out: torch.Tensor | None = None) -> torch.Tensor:
        t = timestep.reshape(-1).to(torch.float32).contiguous()
        proj = torch.empty(t.numel(), 256, device=t.device, dtype=hidden_dtype)
        nat.timestep_embedding(t, scale, 256, 10000.0, proj)
        return self.timestep_embedder(proj, silu_out)


class AdaLayerNormSingle(torch.nn.Module):
    """ltx_nn.py:148-158: (Linear(silu(emb)) , emb)."""

    def __init__(self, embedding_dim: int, embedding_coefficient: int = 6):
        super().__init__()
        self.emb = CombinedTimestepEmbeddings(embedding_dim)
        self.linear = torch.nn.Linear(embedding_dim, embedding_coefficient * embedding_dim, bias=True)

    def forward(self, timestep: torch.Tensor, hidden_dtype: torch.dtype,
                scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
        """timestep (N,) -> (modulation (N, n*D), embedded (N, D)). `scale` multiplies
        the timestep inside the kernel (the reference's *timestep_scale_multiplier)."""
        n = timestep.numel()
        d = self.linear.in_features
        dev = timestep.device
        if n < 32:
            emb = self.emb(timestep, hidden_dtype, scale)
            mod = torch.empty(n, self.linear.out_features, device=dev, dtype=hidden_dtype)
            nat.linear(emb, self.linear.weight, mod, nat.epilogue(bias=self.linear.bias, silu_input=True))
        else:
            silu = torch.empty(n, d, device=dev, dtype=hidden_dtype)
            emb = self.emb(timestep, hidden_dtype, scale, silu_out=silu)
            mod = torch.empty(n, self.linear.out_features, device=dev, dtype=hidden_dtype)
            nat.linear(silu, self.linear.weight, mod, nat.epilogue(bias=self.linear.bias))
        return mod, emb


# ---------------------------------------------------------------------------------------
# Attention + FFN
# ---------------------------------------------------------------------------------------


def _pack(mod: torch.nn.Module, names: list[str], attr: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Pack the listed Linear sub-modules' weights (and biases) into one contiguous
    buffer and re-point their parameters at views of it. Idempotent."""
    key = "_packed_" + attr
    subs = [getattr(mod, n) for n in names]
    cached = getattr(mod, key, None)
    if cached is not None:
        w, b, ptrs = cached
        if ptrs == [s.weight.data_ptr() for s in subs] and w.device == subs[0].weight.device \
                and w.dtype == subs[0].weight.dtype:
            return w, b
    rows = sum(s.weight.shape[0] for s in subs)
    pad = (-rows) % 8  # keep the packed output's row stride a multiple of 8 elements
    ref = subs[0].weight
    with torch.inference_mode(False):  # the parameters stay ordinary tensors, whose writes torch counts
        w = torch.zeros(rows + pad, ref.shape[1], device=ref.device, dtype=ref.dtype)
        b = torch.zeros(rows + pad, device=ref.device, dtype=ref.dtype)
        torch.cat([s.weight.detach() for s in subs], dim=0, out=w[:rows])
        torch.cat([s.bias.detach() for s in subs], dim=0, out=b[:rows])
        row = 0
        for s in subs:
            n = s.weight.shape[0]
            s.weight.data = w[row:row + n]
            s.bias.data = b[row:row + n]
            row += n
    setattr(mod, key, (w, b, [s.weight.data_ptr() for s in subs]))
    return w, b


def _version(t: torch.Tensor) -> int:
    """torch's count of in-place writes; -1 for inference tensors, which have none."""
    return -1 if t.is_inference() else t._version


def _requantize_fp8(module: "Fp8Module", _incompatible_keys) -> None:
    for name in [n for n in module.fp8 if n in module._fp8_stamps]:
        module.weight8(name, module._fp8_weight(name), loaded=True)


class Fp8Module(torch.nn.Module):
    """A module that may hold 8-bit forms of its weights beside the parameters: fp8, name ->
    Fp8Rows, which weight8 gives to the products. They follow the parameters: load_state_dict
    quantises the new ones, and weight8 those that have been moved, replaced or written by an
    in-place operation since (not what torch does not count: writes through .data, or to
    inference tensors; quantise again after those). The same rows are written, so captured
    graphs that read them follow too."""

    FP8_PARTS: dict[str, tuple[str, ...]] = {}  # name -> the Linear sub-modules it packs

    def __init__(self):
        super().__init__()
        self.fp8: dict[str, Fp8Rows] = {}
        self._fp8_stamps: dict[str, tuple] = {}
        self.register_load_state_dict_post_hook(_requantize_fp8)

    def _fp8_weight(self, name: str) -> torch.Tensor:
        """The parameter or packed weight that fp8[name] is the 8-bit form of."""
        return getattr(self, self.FP8_PARTS[name][0]).weight

    def _fp8_stamp(self, name: str, weight: torch.Tensor) -> tuple:
        parts = [self._modules.get(n) for n in self.FP8_PARTS[name]]
        return (weight.data_ptr(), _version(weight), *[_version(m.weight) for m in parts if m is not None])

    def _quantize_weight(self, name: str, weight: torch.Tensor) -> None:
        rows = self.fp8.get(name)
        if rows is not None and (name not in self._fp8_stamps or rows.shape != tuple(weight.shape)
                                 or rows.device != weight.device):
            rows = None  # the caller's, or of another weight
        stamp = self._fp8_stamp(name, weight)
        self.fp8[name] = quantize_fp8(weight.detach(), rows)
        self._fp8_stamps[name] = stamp

    def _quantize_weights(self, names: tuple[str, ...]) -> None:
        """8-bit forms of these weights, and of no others, as they are now."""
        for name in set(self.fp8) - set(names):
            del self.fp8[name]
            self._fp8_stamps.pop(name, None)
        for name in names:
            self._quantize_weight(name, self._fp8_weight(name))

    def weight8(self, name: str, weight: torch.Tensor, loaded: bool = False) -> Fp8Rows | None:
        """The 8-bit form of `weight`, in step with it; None if it has none. Rows that a caller
        put into fp8 are taken as they are. loaded: the weight has just been written."""
        rows = self.fp8.get(name)
        if rows is None or name not in self._fp8_stamps:
            return rows
        if loaded and not weight.is_cuda:
            self._fp8_stamps[name] = ()  # quantised when it is back on the GPU and used
        elif loaded or self._fp8_stamps[name] != self._fp8_stamp(name, weight):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the weights have changed since they were quantised: quantise them, or run the "
                                   "module once, before the capture")
            self._quantize_weight(name, weight)
        return self.fp8[name]


class Attention(Fp8Module):
    """ltx_nn.py:166-236: gated multi-head attention with q/k RMSNorm over the inner
    dim and split RoPE. Same parameters and forward signature as the reference."""

    FP8_PARTS = {"self": ("to_q", "to_k", "to_v", "to_gate_logits"), "q": ("to_q", "to_gate_logits"),
                 "kv": ("to_k", "to_v"), "out": ("to_out",)}

    def __init__(self, query_dim: int, context_dim: int | None = None, heads: int = 8, dim_head: int = 64,
                 norm_eps: float = 1e-6, apply_gated_attention: bool = False):
        super().__init__()
        self.heads = heads
        self.dim_head = dim_head
        self.norm_eps = norm_eps
        inner = heads * dim_head
        context_dim = query_dim if context_dim is None else context_dim
        self.q_norm = torch.nn.RMSNorm(inner, eps=norm_eps)
        self.k_norm = torch.nn.RMSNorm(inner, eps=norm_eps)
        self.to_q = torch.nn.Linear(query_dim, inner, bias=True)
        self.to_k = torch.nn.Linear(context_dim, inner, bias=True)
        self.to_v = torch.nn.Linear(context_dim, inner, bias=True)
        self.to_gate_logits = torch.nn.Linear(query_dim, heads, bias=True) if apply_gated_attention else None
        self.to_out = torch.nn.Linear(inner, query_dim, bias=True)

    def quantize_fp8(self, packings: tuple[str, ...]) -> None:
        """8-bit forms of the named packed weights ("self", or "q" and "kv") and of to_out,
        used from now on; the parameters stay as they are."""
        self._quantize_weights((*packings, "out"))

    def _fp8_weight(self, name: str) -> torch.Tensor:
        packed = {"self": self.packed_self, "q": self.packed_q, "kv": self.packed_kv}
        return packed[name]()[0] if name in packed else self.to_out.weight

    # packed weights -----------------------------------------------------------------
    def packed_self(self):
        names = ["to_q", "to_k", "to_v"] + (["to_gate_logits"] if self.to_gate_logits is not None else [])
        return _pack(self, names, "self")

    def packed_q(self):
        names = ["to_q"] + (["to_gate_logits"] if self.to_gate_logits is not None else [])
        return _pack(self, names, "q")

    def packed_kv(self):
        return _pack(self, ["to_k", "to_v"], "kv")

    # native core ----------------------------------------------------------------------
    def project_qkv(self, x2, rows_per_batch: int, pe: RopeTables | None,
                    k_pe: RopeTables | None = None, normalize: bool = True) -> torch.Tensor:
        """Self-attention projections of x2 (B*T, D), or its 8-bit rows, -> packed (B*T,
        3I(+H)) buffer with q and k normalised and rotated in place (normalize=False: left as
        projected, for a caller that fuses the normalisation into its exchange)."""
        inner = self.heads * self.dim_head
        w, b = self.packed_self()
        qkv = torch.empty(x2.shape[0], w.shape[0], device=w.device, dtype=w.dtype)
        project(x2, w, self.weight8("self", w), qkv, nat.epilogue(bias=b))
        if not normalize:
            return qkv
        if k_pe is None:
            # q and k share the tables: one pass over both blocks
            if pe is None:
                nat.qk_norm_rope_pair(qkv, inner, rows_per_batch, self.heads, self.dim_head, self.q_norm.weight,
                                      self.k_norm.weight, self.norm_eps, None, None)
            else:
                rh = pe.heads
                nat.qk_norm_rope_pair(qkv, inner, rows_per_batch, rh, inner // rh, self.q_norm.weight,
                                      self.k_norm.weight, self.norm_eps,
                                      pe.cos.view(-1, inner // 2) if pe.cos.dim() == 3 else pe.cos,
                                      pe.sin.view(-1, inner // 2) if pe.sin.dim() == 3 else pe.sin,
                                      rope_ld_batch=pe.ld_batch)
            return qkv
        self._norm_rope(qkv[:, :inner], rows_per_batch, self.q_norm.weight, pe)
        self._norm_rope(qkv[:, inner:2 * inner], rows_per_batch, self.k_norm.weight, k_pe)
        return qkv

    def _norm_rope(self, view: torch.Tensor, rows_per_batch: int, weight: torch.Tensor, pe: RopeTables | None):
        inner = self.heads * self.dim_head
        if pe is None:
            nat.qk_norm_rope(view, rows_per_batch, self.heads, self.dim_head, weight, self.norm_eps, None, None)
        else:
            rh = pe.heads
            nat.qk_norm_rope(view, rows_per_batch, rh, inner // rh, weight, self.norm_eps, pe.cos.view(-1, inner // 2)
                             if pe.cos.dim() == 3 else pe.cos, pe.sin.view(-1, inner // 2) if pe.sin.dim() == 3
                             else pe.sin, rope_ld_batch=pe.ld_batch)

    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor | None, batch: int,
               tq: int, tk: int, mask: torch.Tensor | None = None) -> torch.Tensor:
        """mask: a key mask as nat.attention_masked takes it (key_mask)."""
        o = torch.empty(q.shape[0], self.heads * self.dim_head, device=q.device, dtype=q.dtype)
        args = (q, k, v, o, batch, tq, tk, self.heads, self.dim_head, self.dim_head ** -0.5)
        if mask is None:
            nat.attention(*args, gate)
        else:
            nat.attention_masked(*args, mask, gate)
        return o

    def project_out(self, o: torch.Tensor, out: torch.Tensor, epi: nat.Epilogue) -> None:
        weight = self.to_out.weight
        project(o, weight, self.weight8("out", weight), out, epi)

    def forward(self, x: torch.Tensor, context: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                pe=None, k_pe=None, perturbation_mask: torch.Tensor | None = None,
                all_perturbed: bool = False) -> torch.Tensor:
        """mask: over the keys (the context's tokens, or x's own), as sdpa takes it."""
        if perturbation_mask is not None or all_perturbed:
            raise NotImplementedError("STG perturbation is not supported yet")
        b, t, _ = x.shape
        if mask is not None:
            mask = key_mask(mask, b, t if context is None else context.shape[1])
        inner = self.heads * self.dim_head
        x2 = x.reshape(b * t, -1)
        pe_t = _tables_from_reference_layout(pe) if pe is not None else None
        kpe_t = _tables_from_reference_layout(k_pe) if k_pe is not None else None
        gated = self.to_gate_logits is not None
        if context is None:
            qkv = self.project_qkv(x2, t, pe_t, kpe_t)
            o = self.attend(qkv[:, :inner], qkv[:, inner:2 * inner], qkv[:, 2 * inner:3 * inner],
                            qkv[:, 3 * inner:] if gated else None, b, t, t, mask)
        else:
            s = context.shape[1]
            c2 = context.reshape(b * s, -1)
            wq, bq = self.packed_q()
            qg = torch.empty(b * t, wq.shape[0], device=x.device, dtype=x.dtype)
            project(x2, wq, self.weight8("q", wq), qg, nat.epilogue(bias=bq))
            wkv, bkv = self.packed_kv()
            kv = torch.empty(b * s, 2 * inner, device=x.device, dtype=x.dtype)
            project(c2, wkv, self.weight8("kv", wkv), kv, nat.epilogue(bias=bkv))
            self._norm_rope(qg[:, :inner], t, self.q_norm.weight, pe_t)
            self._norm_rope(kv[:, :inner], s, self.k_norm.weight, kpe_t if kpe_t is not None else pe_t)
            o = self.attend(qg[:, :inner], kv[:, :inner], kv[:, inner:], qg[:, inner:] if gated else None, b, t, s, mask)
        out = torch.empty(b * t, self.to_out.out_features, device=x.device, dtype=x.dtype)
        self.project_out(o, out, nat.epilogue(bias=self.to_out.bias))
        return out.view(b, t, -1)


class FeedForward(Fp8Module):
    """ltx_nn.py:239-248: proj_out(gelu_tanh(proj_in(x)))."""

    FP8_PARTS = {"in": ("proj_in",), "out": ("proj_out",)}

    def __init__(self, dim: int, dim_out: int | None = None, mult: int = 4, bias: bool = True):
        super().__init__()
        dim_out = dim if dim_out is None else dim_out
        inner = int(dim * mult)
        self.proj_in = torch.nn.Linear(dim, inner, bias=bias)
        self.proj_out = torch.nn.Linear(inner, dim_out, bias=bias)

    def quantize_fp8(self) -> None:
        """8-bit forms of both weights, used from now on; the parameters stay as they are."""
        self._quantize_weights(("in", "out"))

    def run(self, x2, out: torch.Tensor, epi: nat.Epilogue) -> None:
        """out = epilogue(proj_out(gelu_tanh(proj_in(x2)))), x2 (rows, dim) or its 8-bit rows."""
        h = torch.empty(out.shape[0], self.proj_in.out_features, device=out.device, dtype=out.dtype)
        w_in, w_out = self.proj_in.weight, self.proj_out.weight
        project(x2, w_in, self.weight8("in", w_in), h, nat.epilogue(nat.EPI_GELU_TANH, bias=self.proj_in.bias))
        project(h, w_out, self.weight8("out", w_out), out, epi)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        b, t, d = x.shape
        out = torch.empty(b * t, self.proj_out.out_features, device=x.device, dtype=x.dtype)
        self.run(x.reshape(b * t, d), out, nat.epilogue(bias=self.proj_out.bias))
        return out.view(b, t, -1)
