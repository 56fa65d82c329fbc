"""Attention under a key mask on the B200 against its definition in float64."""

import math

import pytest
import torch

import _native as nat
import fp8_reference as ref
import ltx_nn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def inputs(seed, b, tq, tk, h, d, dtype):
    """q and gate logits as columns of one packed buffer, k and v of another."""
    g = gen(seed)
    inner = h * d
    qg = torch.randn(b, tq, inner + -(-h // 8) * 8, generator=g, device=DEV).to(dtype)
    kv = torch.randn(b, tk, 2 * inner, generator=g, device=DEV).to(dtype)
    return g, qg[..., :inner], kv[..., :inner], kv[..., inner:], qg[..., inner:inner + h]


def mask_of(kind, g, b, tk):
    at = torch.arange(tk, device=DEV)[None]
    n = torch.randint(1, tk + 1, (b, 1), generator=g, device=DEV)
    if kind == "left":
        return at >= tk - n
    if kind == "right":
        return at < n
    if kind == "all":
        return torch.ones(b, tk, dtype=torch.bool, device=DEV)
    if kind == "one":
        return at == n - 1
    m = torch.rand(b, tk, generator=g, device=DEV) < (0.05 if kind == "sparse" else 0.7)
    m[b - 1] = False  # a sample without keys
    return m


def check(got, q, k, v, heads, left_out, bias, gate, scale):
    """fp32: scores are sums of d products (off by d 2^-23 of sum|q k| scale, called e below),
    weights exp of them (off by e + 2^-22 relative), sums of Tk weights and products.
    bf16 adds the rounding of the weights to bf16 (2^-8 relative each, in the numerator only: the
    denominator is summed in fp32) and of the result (2^-8); the weights' own exponential may
    be a cubic with relative error 2^-13. All bounds are relative to A = sum of weights * |v| / sum."""
    cpu = [t.double().cpu() for t in (q, k, v)]
    gd = gate.double().cpu() if gate is not None else None
    lo = left_out.cpu()
    bd = bias.double().cpu() if bias is not None else None
    want = ref.attention(*cpu, heads, lo, bd, gd, scale)
    size = ref.attention(cpu[0], cpu[1], cpu[2].abs(), heads, lo, bd, gd, scale)
    d = q.shape[-1] // heads
    tk = k.shape[1]
    top = (cpu[0].abs().amax() * cpu[1].abs().amax()).item() * d * scale  # bounds sum|q k| scale
    big = 0.0 if bd is None else torch.where(lo, torch.zeros_like(bd), bd).abs().amax().item()
    e = d * 2.0 ** -23 * top + (top + big) * 2.0 ** -22 + (tk + 8) * 2.0 ** -23
    if q.dtype == torch.bfloat16:
        tol = size * (2 * e + 2.0 ** -8 + 2.0 ** -12) + want.abs() * 2.0 ** -8 * 3
    else:
        tol = size * 2 * e
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - want).abs() / (tol + 1e-30)).max():.2f}"
    if q.dtype == torch.bfloat16 and want.norm() > 0:
        # rounding errors of independent weights and results: their root mean square is
        # 2^-8 / sqrt(3) each at the most, and the gate's adds another
        assert (got - want).norm() / want.norm() <= 2.0 ** -8 * 1.25
    empty = lo.all(1)
    assert (got[empty] == 0).all()


SHAPES = [(1, 1, 1, 1, 64), (2, 1, 7, 2, 128), (1, 3, 128, 4, 64), (2, 5, 129, 3, 64), (3, 126, 250, 4, 64),
          (2, 128, 127, 2, 128), (1, 129, 256, 2, 64), (2, 255, 384, 2, 128), (1, 256, 640, 4, 64), (1, 300, 1024, 2, 64),
          (4, 257, 1000, 2, 128), (2, 1, 4099, 4, 128), (3, 2, 2048, 5, 64), (2, 16, 513, 8, 64), (1, 17, 1300, 3, 128),
          (2, 700, 77, 5, 64), (1, 513, 130, 20, 128), (1, 64, 5000, 2, 64),
          # more units than SMs, every second one with rows in one of its two query tiles only
          (4, 300, 200, 40, 64), (4, 270, 140, 40, 128), (40, 30, 260, 5, 64)]


@pytest.mark.parametrize("kind", ["left", "right", "holes", "sparse", "all", "one"])
@pytest.mark.parametrize("b,tq,tk,h,d", SHAPES)
def test_boolean_masks_bf16(b, tq, tk, h, d, kind):
    g, q, k, v, gate = inputs(b * tq + tk + h, b, tq, tk, h, d, torch.bfloat16)
    m = mask_of(kind, g, b, tk)
    got = ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate)
    check(got, q, k, v, h, ~m, None, gate, d ** -0.5)
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,tq,tk,h,d", [(2, 9, 70, 2, 64), (1, 130, 300, 2, 128), (3, 1, 600, 2, 64), (2, 300, 129, 3, 64)])
def test_additive_masks(b, tq, tk, h, d, dtype):
    """Finite values are added to the scores; -inf, the type's lowest value and everything down
    to half of it leave a key out; -1e9 (a common padding value) is just a large number."""
    g, q, k, v, _ = inputs(tk, b, tq, tk, h, d, dtype)
    for mdt in (torch.float32, torch.bfloat16):
        lowest = torch.finfo(mdt).min
        bias = torch.randn(b, tk, generator=g, device=DEV).to(mdt)
        for pad in (-math.inf, lowest, lowest / 2):
            keep = mask_of("holes", g, b, tk)
            m = torch.where(keep, bias, torch.full_like(bias, pad))
            got = ltx_nn.cross_attention(q, k, v, h, mask=m, scale=0.1)
            check(got, q, k, v, h, ~keep, m, None, 0.1)
        keep = mask_of("left", g, b, tk)
        keep[0, tk // 2] = True
        m = torch.where(keep, bias, torch.full_like(bias, -1e9))
        got = ltx_nn.cross_attention(q, k, v, h, mask=m[:, None, None], scale=0.1)
        check(got[:1], q[:1], k[:1], v[:1], h, ~keep[:1], m[:1], None, 0.1)
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("tq", [1, 40, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_left_out_keys_may_hold_anything(tq, dtype):
    """NaN and infinities in k and v of left-out keys, and in the next sample's rows, change
    no bit of the result."""
    b, tk, h, d = 3, 333, 2, 64
    g, q, k, v, gate = inputs(3, b, tq, tk, h, d, dtype)
    for kind in ("left", "right", "holes"):
        m = mask_of(kind, g, b, tk)
        m[1] = False  # a sample without keys between two others
        clean = ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate)
        k2, v2 = k.clone(), v.clone()
        for t, bad in ((k2, math.nan), (v2, math.nan), (k2, math.inf), (v2, -math.inf)):
            t[~m] = bad
            got = ltx_nn.cross_attention(q, k2, v2, h, mask=m, gate_logits=gate)
            assert torch.equal(got, clean)


@pytest.mark.parametrize("tq", [1, 300])
def test_scores_of_any_size(tq):
    """Scores up to thousands, all -inf rows among them, and NaN where a kept key has it."""
    b, tk, h, d = 2, 200, 2, 64
    g, q, k, v, _ = inputs(4, b, tq, tk, h, d, torch.bfloat16)
    m = mask_of("right", g, b, tk)
    m[:, 0] = True
    big = (q * 60).contiguous()
    got = ltx_nn.cross_attention(big, k, v, h, mask=m)
    assert torch.isfinite(got).all()
    want = ref.attention(big.cpu(), k.cpu(), v.cpu(), h, (~m).cpu(), None, None, d ** -0.5)
    assert (got.double().cpu() - want).norm() / want.norm() < 0.02  # a score's fp32 step is 2^-12 at 4000
    k2 = k.clone()
    k2[0, 0, 5] = math.nan
    got = ltx_nn.cross_attention(q, k2, v, h, mask=m)
    assert torch.isnan(got[0, :, :d]).all() and torch.isfinite(got[0, :, d:]).all() and torch.isfinite(got[1]).all()


def test_shared_masks_strides_and_sdpa():
    b, tq, tk, h, d = 3, 70, 190, 4, 64
    g, q, k, v, gate = inputs(5, b, tq, tk, h, d, torch.bfloat16)
    one = mask_of("left", g, 1, tk)
    want = ltx_nn.cross_attention(q, k, v, h, mask=one.expand(b, tk).contiguous(), gate_logits=gate)
    for m in (one, one[0], one[:, None, None], one.expand(b, tk), torch.stack([one, one], -1)[..., 0]):
        assert torch.equal(ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate), want)
    # keys shared by all samples (an expanded batch), and (B, H, T, d) operands
    ks, vs = k[:1].expand(b, tk, h * d), v[:1].expand(b, tk, h * d)
    a = ltx_nn.cross_attention(q, ks, vs, h, mask=one)
    assert torch.equal(a, ltx_nn.cross_attention(q, ks.contiguous(), vs.contiguous(), h, mask=one))

    def heads(x):
        return x.reshape(b, -1, h, d).transpose(1, 2)

    o = ltx_nn.sdpa(heads(q), heads(k), heads(v), mask=one[:, None, None])
    assert torch.equal(o.transpose(1, 2).reshape(b, tq, h * d), ltx_nn.cross_attention(q, k, v, h, mask=one))
    out = torch.empty(b, tq, h * d, dtype=q.dtype, device=DEV)
    assert ltx_nn.cross_attention(q, k, v, h, mask=one, out=out) is out


def test_lengths_of_zero():
    q = torch.randn(2, 3, 128, device=DEV, dtype=torch.bfloat16)
    none = q[:, :0]
    mask = torch.ones(2, 0, dtype=torch.bool, device=DEV)
    assert (ltx_nn.cross_attention(q, none, none, 2, mask=mask) == 0).all()
    assert ltx_nn.cross_attention(none, q, q, 2, mask=torch.ones(2, 3, dtype=torch.bool, device=DEV)).shape == (2, 0, 128)


@pytest.mark.parametrize("b,tq,tk,h,d", [(2, 1, 2000, 4, 128), (2, 40, 700, 3, 64), (1, 600, 1100, 2, 64), (2, 300, 100, 2, 64)])
def test_repeats_and_captured_replays_are_equal(b, tq, tk, h, d):
    g, q, k, v, gate = inputs(6, b, tq, tk, h, d, torch.bfloat16)
    m = mask_of("left", g, b, tk)
    want = ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate)
    graphs = []
    for _ in range(2):  # two captured calls, replayed in turn and on two streams at once
        out = torch.empty(b, tq, h * d, dtype=q.dtype, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate, out=out)
        graphs.append((graph, out))
    for graph, out in graphs * 2:
        graph.replay()
    streams = [torch.cuda.Stream() for _ in graphs]
    for s, (graph, _) in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out, want)
    # the mask is read at replay
    m.copy_(mask_of("right", g, b, tk))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate))


def test_a_sample_does_not_depend_on_its_batch():
    b, tq, tk, h, d = 4, 200, 500, 2, 64
    g, q, k, v, _ = inputs(7, b, tq, tk, h, d, torch.bfloat16)
    m = mask_of("holes", g, b, tk)
    whole = ltx_nn.cross_attention(q, k, v, h, mask=m)
    for i in range(b):
        one = ltx_nn.cross_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], h, mask=m[i:i + 1])
        err = (one.double() - whole[i:i + 1].double()).abs()
        assert (err <= whole[i:i + 1].double().abs() * 2.0 ** -7 + 2.0 ** -9).all()


# Few queries: one, or groups of four with a last one that is not full; keys that end inside
# a chunk of 32, contexts of one chunk up to many for every warp of a cluster's eight CTAs,
# and more units than a wave of CTAs.
FEW = [(1, 1, 1, 1), (2, 1, 31, 3), (1, 4, 33, 2), (3, 3, 129, 4), (2, 2, 255, 5), (1, 1, 1030, 2), (2, 4, 2049, 1),
       (1, 1, 9001, 1), (70, 1, 70, 9), (40, 3, 260, 16)]


@pytest.mark.parametrize("kind", ["right", "holes", "all", "one"])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 32),
                                     (torch.float32, 64), (torch.float32, 128)])
@pytest.mark.parametrize("b,tq,tk,h", FEW)
def test_few_queries(b, tq, tk, h, dtype, d, kind):
    g, q, k, v, gate = inputs(b + 3 * tq + tk + h, b, tq, tk, h, d, dtype)
    m = mask_of(kind, g, b, tk)
    out = torch.full((b, tq, h * d), 5.0, device=DEV, dtype=dtype)
    got = ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate, out=out)
    assert got is out
    check(got, q, k, v, h, ~m, None, gate, d ** -0.5)


@pytest.mark.parametrize("b,tq,tk,h,d", [(10, 129, 70, 8, 64), (19, 5, 33, 8, 32), (20, 129, 40, 15, 128), (2, 600, 129, 2, 64),
                                         (1, 300, 70, 3, 32)])
def test_fp32_with_many_and_few_blocks(b, tq, tk, h, d):
    g, q, k, v, gate = inputs(17, b, tq, tk, h, d, torch.float32)
    m = mask_of("holes", g, b, tk)
    check(ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate), q, k, v, h, ~m, None, gate, d ** -0.5)


@pytest.mark.parametrize("kind", ["left", "holes", "sparse", "one"])
@pytest.mark.parametrize("b,tq,h,d", [(1, 5, 1, 64), (2, 130, 2, 128), (1, 257, 80, 64)])
def test_contexts_of_many_tiles(b, tq, h, d, kind):
    """More key tiles than one pass over the list of a sample's tiles takes at a time, also
    when a cluster's CTAs share them, and with most of them empty."""
    tk = 9000
    g, q, k, v, gate = inputs(tq, b, tq, tk, h, d, torch.bfloat16)
    m = mask_of(kind, g, b, tk)
    check(ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate), q, k, v, h, ~m, None, gate, d ** -0.5)


def test_layouts_that_are_no_row_major_view():
    """Expanded (shared) keys, a single row with odd strides, batch-first slices: all taken."""
    b, tq, tk, h, d = 3, 5, 40, 2, 64
    g, q, k, v, _ = inputs(5, b, tq, tk, h, d, torch.bfloat16)
    m = mask_of("right", g, b, tk)
    shared = k[:1].expand(b, tk, h * d)
    row = v[:1, :1].expand(1, tk, h * d).expand(b, tk, h * d)
    want = ltx_nn.cross_attention(q.contiguous(), shared.contiguous(), row.contiguous(), h, mask=m)
    assert torch.equal(ltx_nn.cross_attention(q, shared, row, h, mask=m), want)
    qt = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(ltx_nn.cross_attention(qt, shared, row, h, mask=m), want)
    one = torch.randn(h * d, 1, device=DEV, dtype=torch.bfloat16).T[None]  # (1, 1, W) of strides (., 1, 1)
    a = ltx_nn.cross_attention(one, k[:1], v[:1], h, mask=m[:1])
    assert torch.equal(a, ltx_nn.cross_attention(one.clone(memory_format=torch.contiguous_format), k[:1], v[:1], h,
                                                 mask=m[:1]))


# -------------------------------------------- NaN and -inf scores of keys that take part


@pytest.mark.parametrize("masked", ["none", "first", "last"])
@pytest.mark.parametrize("tq,tk", [(40, 256), (300, 200), (20, 640)])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_at_every_kept_key_reaches_its_head(d, tq, tk, masked):
    """Wherever in a tile of 128 keys the NaN lies, and whether the tile holds a left-out key
    (`masked`) or not, every query of that head gets NaN, and the other head keeps its bits."""
    b, h = 1, 2
    g, q, k, v, _ = inputs(11, b, tq, tk, h, d, torch.bfloat16)
    m = torch.ones(b, tk, dtype=torch.bool, device=DEV)
    if masked != "none":
        m[0, 0 if masked == "first" else tk - 1] = False
    clean = ltx_nn.cross_attention(q, k, v, h, mask=m)
    keys = [i for i in (*range(128), *range(128, tk, 37)) if m[0, i]]
    for c0 in (0, d):  # the NaN's head
        lost = []
        for key in keys:
            k2 = k.clone()
            k2[0, key, c0 + key % d] = math.nan
            got = ltx_nn.cross_attention(q, k2, v, h, mask=m)
            other = slice(d - c0, 2 * d - c0)
            if not (torch.isnan(got[..., c0:c0 + d]).all() and torch.equal(got[..., other], clean[..., other])):
                lost.append(key)
        assert not lost, lost
    q2 = q.clone()
    q2[0, 7, 3] = math.nan
    got = ltx_nn.cross_attention(q2, k, v, h, mask=m)
    assert torch.isnan(got[0, 7, :d]).all()
    got[0, 7, :d] = clean[0, 7, :d]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("tq,tk", [(1, 256), (40, 128), (300, 384), (20, 640)])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_rows_of_minus_infinite_scores_are_zero(dtype, d, tq, tk, masked):
    b, h = 2, 2
    g, q, k, v, gate = inputs(12, b, tq, tk, h, d, dtype)
    m = torch.ones(b, tk, dtype=torch.bool, device=DEV)
    if masked:
        m[:, 5] = False
    want = ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate)
    q2, k2 = q.clone(), k.clone()
    q2[1, :, 0] = q[1, :, 0].abs() + 1
    k2[1, :, 0] = -math.inf  # sample 1, head 0: every score is -inf
    got = ltx_nn.cross_attention(q2, k2, v, h, mask=m, gate_logits=gate)
    assert (got[1, :, :d] == 0).all(), got[1, :, :d].abs().max()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :, d:], want[1, :, d:])


@pytest.mark.parametrize("low", [-math.inf, -4e4, -2000.0])
@pytest.mark.parametrize("tq,tk", [(40, 256), (300, 128), (20, 640)])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_far_below_the_maximum_weigh_nothing(d, tq, tk, low):
    """Kept keys whose scores are -inf, or hundreds below the row's largest, have weights below
    exp(-200) = 2^-288: with values of 2^120 they add less than 2^-160, so the result is that
    of the other keys."""
    b, h = 1, 2
    g, q, k, v, _ = inputs(13, b, tq, tk, h, d, torch.bfloat16)
    q, k, v = q.clone(), k.clone(), v.clone()
    q[..., ::d] = 2.0
    k[..., ::d] = 0.0
    m = torch.ones(b, tk, dtype=torch.bool, device=DEV)
    low_keys = torch.arange(tk, device=DEV) % 3 == 1
    left_out = low_keys[None].expand(b, tk)
    k2, v2 = k.clone(), v.clone()
    k2[:, low_keys] = 0.0
    k2[:, low_keys, ::d] = low
    v2[:, low_keys] = 2.0 ** 120
    got = ltx_nn.cross_attention(q, k2, v2, h, mask=m, scale=0.1)
    k[:, low_keys], v[:, low_keys] = 0.0, 0.0
    check(got, q, k, v, h, left_out, None, None, 0.1)


@pytest.mark.parametrize("b,tq,tk,h,d,dtype", [(2, 1, 900, 4, 128, torch.bfloat16), (3, 4, 200, 3, 64, torch.bfloat16),
                                               (1, 40, 3000, 2, 64, torch.bfloat16), (2, 600, 300, 5, 128, torch.bfloat16),
                                               (1, 9, 300, 2, 64, torch.float32), (8, 300, 70, 9, 64, torch.float32)])
def test_the_result_may_be_written_over_the_queries(b, tq, tk, h, d, dtype):
    g, q, k, v, gate = inputs(15, b, tq, tk, h, d, dtype)
    m = mask_of("holes", g, b, tk)
    want = ltx_nn.cross_attention(q, k, v, h, mask=m, gate_logits=gate)
    for _ in range(5):
        buf = q.contiguous().clone()
        assert ltx_nn.cross_attention(buf, k, v, h, mask=m, gate_logits=gate, out=buf) is buf
        assert torch.equal(buf, want)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("b,tq,tk,h,d", [(1, 300, 128, 2, 64), (1, 300, 128, 2, 128), (2, 200, 640, 2, 64),
                                         (1, 700, 1000, 2, 128)])
def test_rows_whose_scores_are_all_far_below_zero(b, tq, tk, h, d, masked):
    """The row maximum is that of the row's own scores: anything else that entered it, a zero
    say, would leave these rows (scores around -80) without any weight."""
    g, q, k, v, _ = inputs(16, b, tq, tk, h, d, torch.bfloat16)
    q, k = q.abs() + 0.5, (k * 0.5 - 80 / (1.3 * d * d ** -0.5)).contiguous()
    m = torch.ones(b, tk, dtype=torch.bool, device=DEV)
    got = ltx_nn.cross_attention(q, k, v, h, mask=m if masked else None)
    check(got, q, k, v, h, ~m, None, None, d ** -0.5)


@pytest.mark.parametrize("parts", [0, 3])
@pytest.mark.parametrize("tq,tk", [(40, 128), (300, 256), (300, 500)])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_at_every_key_reaches_its_head_without_a_mask(d, tq, tk, parts):
    """The same without a mask, in whole units and in parts of a unit's keys."""
    b, h = 1, 2
    g, q, k, v, _ = inputs(14, b, tq, tk, h, d, torch.bfloat16)
    nat.attention_force_split(parts)
    try:
        clean = ltx_nn.cross_attention(q, k, v, h)
        lost = []
        for key in (*range(128), *range(128, tk, 37)):
            k2 = k.clone()
            k2[0, key, key % d] = math.nan
            got = ltx_nn.cross_attention(q, k2, v, h)
            if not (torch.isnan(got[..., :d]).all() and torch.equal(got[..., d:], clean[..., d:])):
                lost.append(key)
        assert not lost, lost
    finally:
        nat.attention_force_split(0)
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_large_equal_scores_average_the_values(d):
    """Keys that are all alike weigh the same, whatever their score: up to 1.2e9 in log2 units
    the rounding of the maximum is below 2^-24 of it, a factor of 2^72 that cancels."""
    b, tq, tk, h = 1, 300, 256, 2
    g, q, k, v, _ = inputs(18, b, tq, tk, h, d, torch.bfloat16)
    k = k[:, :1].expand(b, tk, h * d)
    m = torch.ones(b, tk, dtype=torch.bool, device=DEV)
    mean = v.double().mean(1, keepdim=True)
    size = v.double().abs().mean(1, keepdim=True)
    for scale in (1.0, 3e2, 3e4, 1e6, 3e6):
        top = (q.double().abs() @ k[0, 0].double().abs()).max().item() * 200.0 * scale * d ** -0.5 * 1.4427
        if top > 1.2e9:
            continue
        got = ltx_nn.cross_attention((q * 200.0).contiguous(), k, v, h, mask=m, scale=scale * d ** -0.5).double()
        assert ((got - mean).abs() <= size * (2.0 ** -8 + 2.0 ** -12) + mean.abs() * 2.0 ** -8).all(), scale
