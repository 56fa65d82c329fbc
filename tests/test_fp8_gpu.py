"""8-bit rows on the B200 against their definition in float64: the quantiser and the norm in
front of it, the format's layout, and the linear layers."""

import math

import pytest
import torch

import _native as nat
import fp8_reference as ref
import ltx_nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def codes(rows: nat.Fp8Rows) -> torch.Tensor:
    """The scales (rows, blocks) in float64, read by the documented word layout."""
    p = (rows.rows + 255) // 256 * 256
    words = rows.scales.cpu()
    blocks = (rows.cols + 127) // 128
    r = torch.arange(rows.rows)[:, None]
    b = torch.arange(blocks)[None, :]
    w = words[(b // 4) * p + (r // 128) * 128 + (r % 32) * 4 + (r % 128) // 32]
    code = (w >> (8 * (b % 4))) & 255
    return torch.ldexp(torch.ones(code.shape, dtype=torch.float64), code - 127)


# ------------------------------------------------------------------------------ format


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (33, 511), (130, 512), (7, 513),
                                       (257, 640), (64, 2048), (9, 4104)])
def test_quantize_is_the_definition(rows, cols, dtype):
    """Every value and scale equal to the definition's: bf16 and fp32 inputs divide by a
    power of two exactly, so one rounding is all there is."""
    g = gen(rows * 10007 + cols)
    # magnitudes over many blocks' exponents, ties among them (bf16 has 5 bits to spare)
    x = randn(g, rows, cols, dtype=torch.float32) * torch.exp2(
        torch.randint(-30, 30, (rows, 1), generator=g, device=DEV).float())
    x = x.to(dtype)
    q = nat.quantize_fp8(x)
    want, scales = ref.quantize(x)
    assert q.data.stride(0) % 16 == 0 and q.shape == (rows, cols)
    assert torch.equal(codes(q), scales)
    assert torch.equal(q.dequantize(torch.float32).double().cpu(), want)
    assert torch.equal(q.dequantize(torch.bfloat16).double().cpu(), want)  # 4 bits fit in bf16's 8
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("top", [448.0, 447.9999, 448.00003, 1.75, 1.7500001, 3.0e38, 1.2e-38, 1e-44, 2.0 ** -126])
def test_quantize_borders_of_the_scale(top):
    x = torch.linspace(-1, 1, 128, dtype=torch.float64).mul(top).float()[None].to(DEV)
    x[0, 5] = top
    q = nat.quantize_fp8(x)
    want, scales = ref.quantize(x)
    assert torch.equal(codes(q), scales)
    # values below the normal range of fp32 come back as zero or themselves
    got = q.dequantize(torch.float32).double().cpu()
    assert ((got == want) | (want.abs() < 2.0 ** -126)).all()


def test_quantize_zeros_nan_and_infinities():
    x = torch.randn(6, 300, device=DEV)
    x[0] = 0
    x[1, 3], x[1, 140], x[1, 299] = math.nan, math.inf, -math.inf
    x[2] = math.nan
    x[3, :128] = -0.0
    q = nat.quantize_fp8(x)
    want, scales = ref.quantize(x)
    assert torch.equal(codes(q), scales)
    got = q.dequantize(torch.float32).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_quantize_strided_unaligned_and_rows_around_the_output():
    """Column views of a wider buffer, an odd offset (scalar loads), and output rows inside a
    larger buffer whose other bytes stay as they were."""
    g = gen(5)
    base = randn(g, 40, 1001)
    for view in (base[:, 8:520], base[:, 3:500], base[::2, 1:2], base[:, :1]):
        assert torch.equal(nat.quantize_fp8(view).dequantize(torch.float32).double().cpu(), ref.quantize(view)[0])
    x = base[:, :200]
    buf = torch.full((40, 256), 0x55, dtype=torch.uint8, device=DEV)
    scales = torch.full((nat.load_library().ltx_fp8_scale_bytes(40, 200) // 4,), -1, dtype=torch.int32, device=DEV)
    nat._on(x, "ltx_quantize_fp8", x.data_ptr(), x.stride(0), 40, 200, buf.data_ptr(), 256, scales.data_ptr(),
            nat.LTX_BF16)
    assert torch.equal(buf[:, :200].view(torch.float8_e4m3fn).float(), nat.quantize_fp8(x).data.float())
    assert (buf[:, 200:208] == 0).all() and (buf[:, 208:] == 0x55).all()
    written = scales != -1
    assert int(written.sum()) == 40  # one word per row: the padded rows are not touched


def test_from_parts_round_trip_and_refusals():
    g = gen(6)
    x = randn(g, 77, 1000)
    want, scales = ref.quantize(x)
    s = scales.float().to(DEV)
    data = (want / scales.repeat_interleave(128, 1)[:, :1000]).float().to(DEV).to(torch.float8_e4m3fn)
    rows = nat.Fp8Rows.from_parts(data, s)
    assert torch.equal(rows.dequantize(torch.float32).double().cpu(), want)
    q = nat.quantize_fp8(x)
    assert torch.equal(codes(rows), codes(q))
    for bad in (0.0, 3.0, -2.0, math.inf, math.nan, 2.0 ** -127):
        s2 = s.clone()
        s2[3, 2] = bad
        with pytest.raises(ValueError, match="powers of two"):
            nat.Fp8Rows.from_parts(data, s2)


# -------------------------------------------------------------------------------- norm


@pytest.mark.parametrize("kind", ["rms", "layer", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,d,per_token", [(1, 1, 8, False), (2, 3, 120, True), (2, 130, 512, False),
                                             (3, 7, 1064, False), (1, 50, 2048, True), (2, 9, 4096, False),
                                             (1, 3, 16384, False)])
def test_norm_modulate_fp8(b, t, d, per_token, dtype, kind):
    """Against the float64 definition. The kernel's fp32 value y' is within
    d * 2^-24 + 8 * 2^-24 (sum of d squares, root, quotient, two products, sums) of y before it is
    rounded to 8 bits, relative to |x rstd (1 + scale)| + |shift|. Two values that close
    round to the same e4m3 number or, next to a tie, to neighbours: the results differ by at
    most one step of the larger (2^-3 of its magnitude, or 2^-9 s below 2^-6 s) and only
    where y lies that close to a tie or the scales differ."""
    g = gen(d + t)
    x = randn(g, b, t, d, dtype=dtype, std=2.0) + 0.25
    shape = (b, t, d) if per_token else (b, d)
    sc, sh = randn(g, *shape, dtype=dtype, std=0.3), randn(g, *shape, dtype=dtype, std=0.3)
    for scale, shift in ((sc, sh), (sc, None), (None, sh), (None, None)):
        got = ltx_nn.norm_modulate_fp8(x, scale=scale, shift=shift, kind=kind, eps=1e-6)
        y = ref.norm_modulate(x, scale, shift, kind, 1e-6).reshape(b * t, d)
        want, s = ref.quantize(y)
        assert got.shape == (b, t, d)
        v = got.dequantize(torch.float32).double().cpu().view(b * t, d)
        step = torch.maximum(want.abs() * 2.0 ** -3, s.repeat_interleave(128, 1)[:, :d] * 2.0 ** -9)
        assert ((v - want).abs() <= 2 * step).all()
        # a tie within eps of y: probability about 2 eps / step-to-magnitude 2^-4, times 4 for
        # the spread of the count
        eps = (d + 8) * 2.0 ** -24
        differ = (v != want).double().mean().item()
        assert differ <= max(8 * eps * 2 ** 4, 2.0 / v.numel()), differ
    assert nat.device_error_flags() == 0


def test_norm_modulate_fp8_takes_slices_of_an_adaln_output():
    """Vectors with a stride (columns of the (B, 6 D) modulation) and a table row."""
    g = gen(9)
    b, t, d = 2, 33, 1024
    x, mod, table = randn(g, b, t, d), randn(g, b, 6 * d, std=0.3), randn(g, 6, d, std=0.3)
    a = ltx_nn.norm_modulate_fp8(x, scale=mod[:, d:2 * d], shift=mod[:, :d])
    b_ = ltx_nn.norm_modulate_fp8(x, scale=mod[:, d:2 * d].clone(), shift=mod[:, :d].clone())
    assert torch.equal(a.data.float(), b_.data.float()) and torch.equal(codes(a), codes(b_))
    m = nat.modulation(table, mod, shift=(0, 0), scale=(d, d), mod_ld_batch=6 * d)
    got = nat.norm_modulate_fp8(x.view(-1, d), t, nat.LTX_NORM_RMS, 1e-6, m)
    y = ref.norm_modulate(x, mod[:, d:2 * d].double() + table[1].double(), mod[:, :d].double() + table[0].double(),
                          "rms", 1e-6)
    want, _ = ref.quantize(y.reshape(-1, d))
    assert torch.equal(got.data.float(), nat.norm_modulate_fp8(x.view(-1, d), t, 0, 1e-6, m, (b, t, d)).data.float())
    v = got.dequantize(torch.float32).double().cpu()
    assert (v != want).double().mean() <= 8 * (d + 8) * 2.0 ** -24 * 2 ** 4


# ------------------------------------------------------------------------------ linear


def linear_case(seed, m, n, k, dtype=torch.bfloat16):
    g = gen(seed)
    x = randn(g, m, k, dtype=dtype)
    w = randn(g, n, k, std=k ** -0.5)
    return g, x, w


def check(got, want, slack, dtype):
    """|got - want| <= half a step of the result + slack, and no drift in the norm."""
    got = got.double().cpu()
    tol = want.abs() * HALF[dtype] * (1 + 2.0 ** -6) + slack
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - want).abs() / tol).max():.2f} of the bound"
    rel = (got - want).norm() / want.norm().clamp(min=1e-30)
    assert rel <= HALF[dtype] + 2e-6, rel


SHAPES = [(1, 1, 1), (1, 8, 16), (2, 12288, 2048), (3, 5, 100), (4, 33, 1200), (5, 5000, 999), (7, 17, 8200),
          (8, 2000, 4097), (6, 24, 20000), (9, 40, 600), (31, 256, 128), (32, 128, 129), (33, 300, 512),
          (100, 72, 4096), (127, 129, 130), (128, 128, 1024), (129, 257, 640), (252, 6176, 2048), (256, 512, 513),
          (257, 1371, 1037), (300, 2048, 8192), (1000, 96, 64), (1025, 776, 1536), (2048, 2304, 256),
          (3000, 4100, 384), (2560, 5120, 1040)]  # more than one tile per SM pair


@pytest.fixture(params=[-1, 0, 1], ids=["auto", "tile", "pair"])
def kernel(request):
    nat.fp8_force_pair(request.param)
    yield request.param
    nat.fp8_force_pair(-1)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_fp8_bf16(m, n, k, kernel):
    """The operands are exact in float64, so only the sums' and the result's rounding is
    allowed: a sum of k terms in fp32 is off by at most k 2^-23 of sum|a w| whatever the
    order and whether an addition rounds or truncates."""
    g, x, w = linear_case(m + n + k, m, n, k)
    xq, wq = nat.quantize_fp8(x), nat.quantize_fp8(w)
    a, b = xq.dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    want, slack = (a @ b.t()).cpu(), (a.abs() @ b.abs().t()).cpu() * k * 2.0 ** -23
    bias = randn(g, n)
    check(ltx_nn.linear_fp8(x, wq), want, slack, torch.bfloat16)
    got = ltx_nn.linear_fp8(xq, wq, bias)
    want = want + bias.double().cpu()
    check(got, want, slack, torch.bfloat16)
    # the same rows give the same bits: alone, in another batch, and again
    assert torch.equal(ltx_nn.linear_fp8(xq, wq, bias), got)
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (2, 2048, 1024), (70, 100, 520), (300, 515, 1037), (512, 768, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_fp8_epilogues(m, n, k, dtype, kernel):
    """Every epilogue, in both result types; the activations' own arithmetic (an exponential
    of 2 units, a quotient of 2) adds 8 * 2^-23 of the value."""
    g, x, w = linear_case(m * 3 + n, m, n, k, dtype)
    wq = nat.quantize_fp8(w)
    a = nat.quantize_fp8(x).dequantize(torch.float32).double()
    b = wq.dequantize(torch.float32).double()
    bias, res = randn(g, n, dtype=dtype), randn(g, 1, m, n, dtype=dtype)
    lin = (a @ b.t()).cpu() + bias.double().cpu()
    slack = (a.abs() @ b.abs().t()).cpu() * k * 2.0 ** -23 + bias.double().cpu().abs() * 2.0 ** -23
    for act, f in (("gelu_tanh", ref.gelu_tanh), ("silu", lambda v: v * torch.sigmoid(v))):
        got = ltx_nn.linear_fp8(x, wq, bias, activation=act)
        # both have slopes within [-0.13, 1.13]
        check(got, f(lin), 1.13 * slack + (f(lin).abs() + lin.abs() * 2.0 ** -20) * 8 * 2.0 ** -23, dtype)
    r = res.double().cpu()
    for gate in (None, randn(g, 1, n, dtype=dtype), randn(g, 1, m, n, dtype=dtype)):
        gd = torch.ones(1, m, n, dtype=torch.float64) if gate is None else \
            (gate if gate.dim() == 3 else gate[:, None]).double().cpu()
        want = r + gd * lin
        s = slack * gd.abs() + (gd * lin).abs() * 2.0 ** -23
        got = ltx_nn.linear_fp8(x[None], wq, bias, residual=res, gate=gate)
        check(got, want, s, dtype)
        buf = res.clone()  # in place, as the block's residual stream is updated
        assert ltx_nn.linear_fp8(x[None], wq, bias, residual=buf, gate=gate, out=buf) is buf
        assert torch.equal(buf, got)
    mask = (torch.arange(m, device=DEV) % 3 == 0).float()
    vec = randn(g, n, dtype=dtype)
    out = torch.empty(m, n, dtype=dtype, device=DEV)
    nat.linear_fp8(nat.quantize_fp8(x), wq, out,
                   nat.epilogue(nat.EPI_ROW_MASK_ADD, bias=bias, row_mask=mask, row_vec=vec))
    check(out, lin + mask.double().cpu()[:, None] * vec.double().cpu(), slack + lin.abs() * 2.0 ** -23, dtype)


def test_linear_fp8_gate_per_sample_and_per_token(kernel):
    g = gen(17)
    b, t, k, n = 3, 150, 256, 320
    x, w, res = randn(g, b, t, k), nat.quantize_fp8(randn(g, n, k, std=0.06)), randn(g, b, t, n)
    gate = randn(g, b, n)
    per_sample = ltx_nn.linear_fp8(x, w, residual=res, gate=gate)
    assert torch.equal(per_sample, ltx_nn.linear_fp8(x, w, residual=res, gate=gate[:, None].expand(b, t, n)))
    for i in range(b):  # a batch is its samples
        assert torch.equal(per_sample[i:i + 1], ltx_nn.linear_fp8(x[i:i + 1], w, residual=res[i:i + 1],
                                                                  gate=gate[i:i + 1]))


def test_linear_fp8_writes_its_rows_and_columns_only(kernel):
    g = gen(18)
    for m, n, k in ((5, 100, 64), (130, 264, 200), (300, 300, 512)):
        x, w = nat.quantize_fp8(randn(g, m, k)), nat.quantize_fp8(randn(g, n, k))
        for ld in (n + 8 - n % 8 + 8, n + 3):
            buf = torch.full((m + 4, ld), 7.0, dtype=torch.bfloat16, device=DEV)
            nat.linear_fp8(x, w, buf[:m, :n])
            assert (buf[m:] == 7).all() and (buf[:, n:] == 7).all()
            dense = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
            nat.linear_fp8(x, w, dense)
            assert torch.equal(dense, buf[:m, :n])


def test_linear_fp8_nan_rows_stay_in_their_rows(kernel):
    """NaN and infinite activations make their own rows NaN, a NaN weight its column; what
    lies behind the last row or column of an operand reaches nothing."""
    g = gen(19)
    x, w = randn(g, 70, 200), randn(g, 90, 200)
    clean = ltx_nn.linear_fp8(x, nat.quantize_fp8(w))
    x2, w2 = x.clone(), w.clone()
    x2[3, 7], x2[69, 199], w2[11, 0] = math.nan, math.inf, math.nan
    got = ltx_nn.linear_fp8(x2, nat.quantize_fp8(w2))
    bad = torch.zeros(70, 90, dtype=torch.bool, device=DEV)
    bad[3] = bad[69] = True
    bad[:, 11] = True
    assert torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], clean[~bad])


def test_linear_fp8_wide_range_of_scales(kernel):
    """Blocks whose scales differ by 2^60 within a row: each product is scaled exactly."""
    g = gen(20)
    k = 128 * 9
    x, w = randn(g, 140, k, dtype=torch.float32), randn(g, 260, k, dtype=torch.float32)
    ex = torch.randint(-30, 30, (140, 9), generator=g, device=DEV).float().repeat_interleave(128, 1)
    ew = torch.randint(-30, 30, (260, 9), generator=g, device=DEV).float().repeat_interleave(128, 1)
    xq, wq = nat.quantize_fp8(x * torch.exp2(ex)), nat.quantize_fp8(w * torch.exp2(ew))
    a, b = xq.dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    got = ltx_nn.linear_fp8(xq, wq, dtype=torch.float32).double()
    slack = (a.abs() @ b.abs().t()) * k * 2.0 ** -23
    assert ((got - a @ b.t()).abs() <= slack).all()


def test_linear_fp8_on_another_stream_and_captured():
    """A captured norm -> product pair replayed on new inputs equals the eager calls."""
    g = gen(21)
    x = randn(g, 2, 200, 512)
    mod = randn(g, 2, 512, std=0.3)
    w = nat.quantize_fp8(randn(g, 640, 512, std=0.05))

    def step(inp):
        return ltx_nn.linear_fp8(ltx_nn.norm_modulate_fp8(inp, scale=mod, shift=mod), w, activation="gelu_tanh")

    buf = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = step(buf)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(eager, step(buf))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for seed in (1, 2):
        new = randn(gen(seed), 2, 200, 512)
        buf.copy_(new)
        graph.replay()
        assert torch.equal(out, step(new))


@pytest.mark.parametrize("m", [2, 9, 252])
def test_linear_fp8_takes_a_bias_of_any_stride(m):
    g = gen(m)
    n, k = 640, 512
    x, w = randn(g, m, k), nat.quantize_fp8(randn(g, n, k, std=0.05))
    buf = randn(g, n, 3)
    for bias in (buf[:, 0], buf[:1, 1].expand(n)):
        want = ltx_nn.linear_fp8(x, w, bias.clone(memory_format=torch.contiguous_format).contiguous())
        for _ in range(3):
            assert torch.equal(ltx_nn.linear_fp8(x, w, bias), want)
            assert torch.equal(ltx_nn.linear_fp8(nat.quantize_fp8(x), w, bias), ltx_nn.linear_fp8(
                nat.quantize_fp8(x), w, bias.contiguous()))


@pytest.mark.parametrize("m", [1, 2, 8, 9, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_fp8_in_place(m, dtype):
    """x, residual and out may be one tensor: the result is that of the rows quantised first."""
    g = gen(m)
    n = 2048
    x, w, bias = randn(g, 1, m, n, dtype=dtype), nat.quantize_fp8(randn(g, n, n, std=0.02)), randn(g, n, dtype=dtype)
    want = ltx_nn.linear_fp8(ltx_nn.quantize_fp8(x), w, bias, residual=x)
    plain = ltx_nn.linear_fp8(ltx_nn.quantize_fp8(x), w, bias, dtype=dtype)
    for _ in range(5):
        buf = x.clone()
        assert ltx_nn.linear_fp8(buf, w, bias, residual=buf, out=buf) is buf
        assert torch.equal(buf, want)
        buf = x.clone()
        ltx_nn.linear_fp8(buf, w, bias, out=buf)
        assert torch.equal(buf, plain)
    # rows of one buffer that interleave without sharing a byte
    wide = torch.zeros(m, 2 * n, dtype=dtype, device=DEV)
    wide[:, :n] = x[0]
    nat.quantize_linear_fp8(wide[:, :n], w, wide[:, n:], nat.epilogue(bias=bias))
    assert torch.equal(wide[:, :n], x[0])
    assert torch.equal(wide[:, n:], ltx_nn.linear_fp8(x, w, bias)[0])


@pytest.mark.parametrize("m", [1, 3, 8, 9])
@pytest.mark.parametrize("ex,ew", [(100, -95), (-110, 100), (118, -118), (-118, 118), (58, 60), (-58, -60),
                                   (-63, -62)])
def test_linear_fp8_of_huge_and_tiny_operands(m, ex, ew):
    """Scales whose product is in range: partial products of a block that carry one operand's
    scale alone would leave fp32."""
    g = gen(m + ex)
    k, n = 1000, 260
    x = randn(g, m, k, dtype=torch.float32) * 2.0 ** ex
    w = randn(g, n, k, dtype=torch.float32) * 2.0 ** ew
    wq = nat.quantize_fp8(w)
    a, b = nat.quantize_fp8(x).dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    got = ltx_nn.linear_fp8(x, wq).double()
    assert ((got - a @ b.t()).abs() <= (a.abs() @ b.abs().t()) * k * 2.0 ** -23).all()


def test_linear_fp8_of_nearly_2_to_the_31_weight_rows():
    """Row indices up to the documented limit: the step behind a CTA's last rows passes 2^31."""
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 48 GB of device memory")
    n = 2 ** 31 - 257
    w = nat.Fp8Rows(n, 1, device=DEV)
    w.buf[:w.scale_bytes].fill_(127)  # every scale 1
    w.buf[w.scale_bytes:].fill_(0x38)  # every value 1
    marked = torch.tensor([0, 15, 4735, 4736, 2 ** 30 + 1, n - 4737, n - 4736, n - 17, n - 1], device=DEV)
    w.buf[w.scale_bytes + marked * w.ld] = 0x40  # 2
    x = torch.full((1, 1), 3.0, device=DEV, dtype=torch.bfloat16)
    out = ltx_nn.linear_fp8(x, w)[0]
    assert (out[marked] == 6).all()
    out[marked] = 3.0
    assert int(out.min()) == 3 and int(out.max()) == 3
    assert nat.device_error_flags() == 0
    del w, out
    torch.cuda.empty_cache()
