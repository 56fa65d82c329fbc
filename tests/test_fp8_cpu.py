"""Refusals of the 8-bit row and masked-attention entry points, and their host arithmetic:
no GPU is touched (every check comes before the first CUDA call)."""

import ctypes
import weakref

import pytest
import torch

import _native as nat
import fp8_reference as ref
import ltx_dit
import ltx_nn

INVALID, UNSUPPORTED = 1, 3
P = 4096  # a 16-byte aligned address that no call gets to use


@pytest.fixture(scope="module")
def lib():
    return nat.load_library()


def test_reference_rounding_matches_torch():
    x = torch.randn(64, 300).to(torch.bfloat16)
    want, s = ref.quantize(x)
    s = s.repeat_interleave(128, 1)[:, :300]
    assert torch.equal((x.float() / s.float()).to(torch.float8_e4m3fn).double() * s, want)


def test_scale_bytes(lib):
    assert lib.ltx_fp8_scale_bytes(1, 1) == 256 * 4
    assert lib.ltx_fp8_scale_bytes(256, 512) == 256 * 4
    assert lib.ltx_fp8_scale_bytes(257, 513) == 512 * 2 * 4
    assert lib.ltx_fp8_scale_bytes(0, 5) == 0 and lib.ltx_fp8_scale_bytes(5, -1) == 0
    r = nat.Fp8Rows(257, 513, device="cpu")
    assert r.scales.numel() * 4 == lib.ltx_fp8_scale_bytes(257, 513)
    assert r.data.shape == (257, 513) and r.data.stride(0) == 528


@pytest.mark.parametrize("change,msg", [
    ({"x": None}, b"x must be"), ({"q": None}, b"non-NULL"), ({"scales": None}, b"non-NULL"),
    ({"rows": 0}, b"positive"), ({"cols": 0}, b"positive"), ({"rows": 1 << 31}, b"out of range"),
    ({"ldq": 511}, b"multiple of 16"), ({"ldq": 496}, b"multiple of 16"), ({"ldx": 511}, b"ldx"),
    ({"q": P + 8}, b"16-byte"), ({"scales": P + 4}, b"16-byte"), ({"x": P + 1}, b"aligned"), ({"dtype": 2}, b"dtype")])
def test_quantize_refusals(lib, change, msg):
    a = {"x": P, "ldx": 512, "rows": 4, "cols": 512, "q": P, "ldq": 512, "scales": P, "dtype": 1, "stream": None} | change
    assert lib.ltx_quantize_fp8(*a.values()) == INVALID
    assert msg in lib.ltx_last_error()
    a = {"q": a["q"], "ldq": a["ldq"], "scales": a["scales"], "rows": a["rows"], "cols": a["cols"], "x": a["x"],
         "ldx": a["ldx"], "dtype": a["dtype"], "stream": None}
    assert lib.ltx_dequantize_fp8(*a.values()) == INVALID


@pytest.mark.parametrize("change,status", [
    ({"x": None}, INVALID), ({"D": 100}, INVALID), ({"D": 16392, "ldx": 16392, "ldq": 16400}, UNSUPPORTED),
    ({"ldx": 500}, INVALID), ({"x": P + 2}, INVALID), ({"rpb": 0}, INVALID), ({"kind": 3}, INVALID),
    ({"q": P + 1}, INVALID), ({"rows": 0}, INVALID), ({"dtype": 5}, INVALID)])
def test_norm_refusals(lib, change, status):
    a = {"x": P, "ldx": 512, "q": P, "ldq": 512, "scales": P, "rows": 4, "rpb": 2, "D": 512, "kind": 0, "eps": 1e-6,
         "mod": None, "dtype": 1, "stream": None} | change
    assert lib.ltx_norm_modulate_fp8(*a.values()) == status, lib.ltx_last_error()


@pytest.mark.parametrize("change,msg", [
    ({"A": None}, b"A:"), ({"Ws": None}, b"W:"), ({"C": None}, b"C must"), ({"M": 0}, b"positive"),
    ({"lda": 250}, b"multiple of 16"), ({"ldw": 240}, b"hold the columns"), ({"ldc": 63}, b"ldc"), ({"C": P + 1}, b"aligned"),
    ({"dtype": 7}, b"dtype"), ({"N": 1 << 31, "ldc": 1 << 31}, b"out of range")])
def test_linear_refusals(lib, change, msg):
    a = {"A": P, "lda": 256, "As": P, "W": P, "ldw": 256, "Ws": P, "C": P, "ldc": 64, "M": 4, "N": 64, "K": 256,
         "epi": None, "dtype": 1, "stream": None} | change
    assert lib.ltx_linear_fp8(*a.values()) == INVALID
    assert msg in lib.ltx_last_error(), lib.ltx_last_error()


@pytest.mark.parametrize("fields,msg", [
    ({"kind": 9}, b"kind"), ({"silu_input": 1}, b"silu_input"), ({"kind": nat.EPI_GATE_RESIDUAL}, b"residual"),
    ({"kind": nat.EPI_GATE_RESIDUAL, "residual": P, "ld_residual": 63}, b"ld_residual"),
    ({"kind": nat.EPI_ROW_MASK_ADD}, b"row_mask"), ({"bias": P + 1}, b"aligned")])
def test_linear_epilogue_refusals(lib, fields, msg):
    e = nat.Epilogue()
    for k, v in fields.items():
        setattr(e, k, v)
    st = lib.ltx_linear_fp8(P, 256, P, P, 256, P, P, 64, 4, 64, 256, ctypes.byref(e), 1, None)
    assert st == INVALID and msg in lib.ltx_last_error(), lib.ltx_last_error()


@pytest.mark.parametrize("change,msg", [
    ({"x": None}, b"non-NULL"), ({"C": None}, b"non-NULL"), ({"xdt": 2}, b"x_dtype"), ({"dtype": 2}, b"dtype must"),
    ({"K": 0}, b"positive"), ({"ldx": 255}, b"ldx"), ({"ldc": 63}, b"ldc"), ({"x": P + 1}, b"aligned"),
    ({"C": P + 1}, b"aligned"), ({"ldw": 250}, b"multiple of 16"), ({"W": P + 8}, b"16-byte"), ({"M": 1 << 31}, b"out of range"),
    ({"M": 9, "ws": None}, b"workspace"), ({"M": 9, "ws": P + 4}, b"workspace"), ({"M": 9, "bytes": 9 * 256}, b"workspace")])
def test_quantize_linear_refusals(lib, change, msg):
    a = {"x": P, "ldx": 256, "xdt": 1, "W": P, "ldw": 256, "Ws": P, "C": P, "ldc": 64, "M": 4, "N": 64, "K": 256,
         "epi": None, "ws": P, "bytes": 1 << 20, "dtype": 1, "stream": None} | change
    assert lib.ltx_quantize_linear_fp8(*a.values()) == INVALID
    assert msg in lib.ltx_last_error(), lib.ltx_last_error()


def test_quantize_linear_workspace(lib):
    """Nothing for up to eight rows, else the 8-bit rows of x."""
    f = lib.ltx_quantize_linear_fp8_workspace_bytes
    assert f(0, 256) == f(8, 256) == f(-1, 5) == 0
    assert f(9, 1037) == 9 * 1040 + lib.ltx_fp8_scale_bytes(9, 1037)
    assert f(8, 1 << 20) == (8 << 20) + lib.ltx_fp8_scale_bytes(8, 1 << 20)  # too wide for shared memory


def test_rows_are_views_of_one_buffer():
    r = nat.Fp8Rows(3, 100, 1037, device="cpu")
    assert r.shape == (3, 100, 1037) and (r.rows, r.cols, r.ld) == (300, 1037, 1040)
    assert tuple(r.data.shape) == (300, 1037) and r.data.stride() == (1040, 1) and r.data.dtype == torch.float8_e4m3fn
    data, ld, scales = r.operand()
    assert (data, ld, scales) == (r.data.data_ptr(), 1040, r.scales.data_ptr()) and (data - scales) % 16 == 0
    assert r.scales.numel() == 512 * 3 and r.buf.numel() == 300 * 1040 + 512 * 3 * 4
    assert nat.Fp8Rows(0, 64, device="cpu").data.shape == (0, 64) and nat.Fp8Rows(5, 0, device="cpu").data.shape == (5, 0)


def test_masks_of_a_guidance_batch():
    cat = ltx_dit._cat_masks
    a = torch.arange(6)[None] < 4
    assert cat([None, None], 6) is None
    assert torch.equal(cat([a, None], 6), torch.stack([a[0], torch.ones(6, dtype=torch.bool)]))
    add = torch.where(a[0], 0.0, -1e4)
    assert torch.equal(cat([None, add, add.reshape(1, 1, 1, 6)], 6), torch.stack([torch.zeros(6), add, add]))
    with pytest.raises(TypeError, match="one type"):
        cat([a, add], 6)
    with pytest.raises(RuntimeError):
        cat([a, None], 7)


@pytest.mark.parametrize("change,status", [
    ({"mask": None}, INVALID), ({"q": None}, INVALID), ({"B": 0}, INVALID), ({"Tk": 0}, INVALID),
    ({"heads": 0}, INVALID), ({"d": 96, "ldq": 400}, UNSUPPORTED), ({"d": 32}, UNSUPPORTED), ({"ldk": 120}, INVALID),
    ({"ldo": 132}, INVALID), ({"v": P + 8}, INVALID), ({"ld_mask": 99}, INVALID), ({"kind": 3}, INVALID),
    ({"kind": 1, "mask": P + 2}, INVALID), ({"scale": 0.0}, INVALID), ({"scale": float("inf")}, INVALID),
    ({"scale": float("nan")}, INVALID), ({"gate": P, "ld_gate": 1}, INVALID), ({"B": 1 << 20}, INVALID),
    ({"Tq": 1 << 31}, INVALID), ({"dtype": 2}, INVALID)])
def test_masked_attention_refusals(lib, change, status):
    a = {"q": P, "ldq": 128, "k": P, "ldk": 128, "v": P, "ldv": 128, "o": P, "ldo": 128, "B": 2, "Tq": 5, "Tk": 100,
         "heads": 2, "d": 64, "scale": 0.125, "mask": P, "ld_mask": 100, "kind": 0, "gate": None, "ld_gate": 0,
         "dtype": 1, "stream": None} | change
    assert lib.ltx_attention_masked(*a.values()) == status, lib.ltx_last_error()


def test_python_entry_points_refuse_bad_arguments():
    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    w = nat.Fp8Rows(64, 256, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ltx_nn.quantize_fp8(x)
    with pytest.raises(TypeError):
        ltx_nn.quantize_fp8(x.half())
    with pytest.raises(ValueError, match="columns"):
        ltx_nn.linear_fp8(x[..., :128], w)
    with pytest.raises(TypeError, match="Fp8Rows"):
        ltx_nn.linear_fp8(x, x)
    with pytest.raises(ValueError, match="activation"):
        ltx_nn.linear_fp8(x, w, activation="relu")
    res = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="exclude"):
        ltx_nn.linear_fp8(x, w, activation="silu", residual=res)
    with pytest.raises(ValueError, match="gate needs"):
        ltx_nn.linear_fp8(x, w, gate=res)
    with pytest.raises(ValueError, match="residual must"):
        ltx_nn.linear_fp8(x, w, residual=res.float())
    with pytest.raises(ValueError, match="gate must"):
        ltx_nn.linear_fp8(x, w, residual=res, gate=torch.zeros(3, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="bias must"):
        ltx_nn.linear_fp8(x, w, bias=torch.zeros(63, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        ltx_nn.linear_fp8(x, w, out=torch.zeros(2, 64, 3, dtype=torch.bfloat16).transpose(1, 2))
    with pytest.raises(ValueError, match="residual must"):
        ltx_nn.linear_fp8(nat.Fp8Rows(7, 256, device="cpu"), w, residual=res)
    with pytest.raises(ValueError, match="kind"):
        ltx_nn.norm_modulate_fp8(x, kind="batch")
    with pytest.raises(ValueError, match="scale must"):
        ltx_nn.norm_modulate_fp8(x, scale=torch.zeros(2, 255, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="like the other"):
        ltx_nn.norm_modulate_fp8(x, scale=torch.zeros(2, 256, dtype=torch.bfloat16), shift=x)
    with pytest.raises(ValueError, match="float8"):
        nat.Fp8Rows.from_parts(x[0], torch.ones(3, 2))
    with pytest.raises(ValueError, match="one per 128"):
        nat.Fp8Rows.from_parts(torch.zeros(3, 256).to(torch.float8_e4m3fn), torch.ones(3, 3))


def test_masks_refused():
    q, k = torch.zeros(2, 5, 128, dtype=torch.bfloat16), torch.zeros(2, 9, 128, dtype=torch.bfloat16)
    ones = torch.ones(2, 9, dtype=torch.bool)

    def call(mask, **kw):
        return ltx_nn.cross_attention(q, k, k, 2, mask=mask, **kw)

    with pytest.raises(NotImplementedError, match="depend on the query"):
        call(torch.ones(2, 1, 5, 9, dtype=torch.bool))
    with pytest.raises(NotImplementedError):
        ltx_nn.sdpa(*(x.view(2, -1, 2, 64).transpose(1, 2) for x in (q, k, k)), mask=torch.ones(2, 2, 1, 9))
    for bad in (ones[:, :8], torch.ones(3, 9, dtype=torch.bool), torch.ones(2, 1, 9, dtype=torch.bool)):
        with pytest.raises(ValueError, match="key mask"):
            call(bad)
    with pytest.raises(TypeError, match="mask dtype"):
        call(ones.to(torch.int32))
    with pytest.raises(TypeError, match="mask dtype"):
        call(ones.half())
    with pytest.raises(ValueError, match="CUDA"):
        call(ones)
    with pytest.raises(ValueError, match="gate_logits"):
        call(ones, gate_logits=q[..., :3])
    with pytest.raises(ValueError, match="heads"):
        ltx_nn.cross_attention(q, k, k, 3, mask=ones)
    with pytest.raises(ValueError, match="k and v"):
        ltx_nn.cross_attention(q, k, k[:, :8], 2, mask=ones)
    with pytest.raises(TypeError):
        ltx_nn.cross_attention(q, k.float(), k, 2, mask=ones)
    with pytest.raises(ValueError, match="out must"):
        call(ones, out=torch.zeros(2, 5, 128))


@pytest.mark.parametrize("bias", ["strided", "expanded"])
@pytest.mark.parametrize("quantised", [False, True])
def test_copies_made_for_an_epilogue_live_until_the_launch(monkeypatch, bias, quantised):
    """The epilogue holds addresses: a vector that had to be copied must still exist when the
    launch reads it (its memory could be given to the call's own workspace otherwise)."""
    copies, calls = [], []
    contiguous = torch.Tensor.contiguous

    def copying(t, *a, **kw):
        r = contiguous(t, *a, **kw)
        if r is not t:
            copies.append((r.data_ptr(), weakref.ref(r)))
        return r

    def launch(x, w, c, epi):
        alive = {p for p, ref_ in copies if ref_() is not None}
        calls.append(epi.bias in alive and epi.gate.mod in alive)

    monkeypatch.setattr(torch.Tensor, "contiguous", copying)
    monkeypatch.setattr(nat, "quantize_linear_fp8", launch)
    monkeypatch.setattr(nat, "linear_fp8", launch)
    monkeypatch.setattr(nat, "_ptr", lambda t: t.data_ptr() if t is not None else None)
    x = torch.zeros(2, 5, 256, dtype=torch.bfloat16)
    if quantised:
        x = nat.Fp8Rows(2, 5, 256, device="cpu")
    wide = torch.zeros(64, 2, dtype=torch.bfloat16)
    b = wide[:, 0] if bias == "strided" else wide[:1, 0].expand(64)
    gate = torch.zeros(2, 128, dtype=torch.bfloat16)[:, ::2]
    ltx_nn.linear_fp8(x, nat.Fp8Rows(64, 256, device="cpu"), b, residual=torch.zeros(2, 5, 64, dtype=torch.bfloat16),
                      gate=gate)
    assert len(copies) == 2 and calls == [True]


def test_quantize_linear_in_place_needs_the_workspace(lib):
    """Where C shares a byte with x, the rows are quantised before anything is stored."""
    a = {"x": P, "ldx": 256, "xdt": 1, "W": P, "ldw": 256, "Ws": P, "C": P, "ldc": 256, "M": 4, "N": 256, "K": 256,
         "epi": None, "ws": None, "bytes": 0, "dtype": 1, "stream": None}
    need = 4 * 256 + lib.ltx_fp8_scale_bytes(4, 256)
    for change in ({}, {"C": P + 2 * (3 * 256 + 255)}, {"C": P + 2 * 255, "ldx": 512, "ldc": 512}, {"M": 1},
                   {"x": P + 2 * (3 * 256 + 255)}, {"ws": P, "bytes": need - 1}, {"ws": P + 4, "bytes": need},
                   {"xdt": 0, "dtype": 0, "C": P + 1020}):
        assert lib.ltx_quantize_linear_fp8(*(a | change).values()) == INVALID
        assert b"overlaps x" in lib.ltx_last_error(), change


def test_quantize_linear_passes_a_workspace_when_in_place(monkeypatch):
    sizes = []
    monkeypatch.setattr(nat, "_same_device", lambda *a: None)
    monkeypatch.setattr(nat, "_on", lambda t, name, *args, **kw: sizes.append(args[13]))
    w = nat.Fp8Rows(256, 256, device="cpu")
    buf = torch.zeros(8, 512, dtype=torch.bfloat16)
    nat.quantize_linear_fp8(buf[:4, :256], w, torch.zeros(4, 256, dtype=torch.bfloat16))
    nat.quantize_linear_fp8(buf[:4, :256], w, buf[4:, :256])
    assert sizes == [0, 0]
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    nat.quantize_linear_fp8(x, w, x)
    ltx_nn.linear_fp8(x, w, out=x)
    nat.quantize_linear_fp8(buf[:4, :256], w, buf[3:7, :256])
    need = 4 * 256 + nat.load_library().ltx_fp8_scale_bytes(4, 256)
    assert sizes[2:] == [need] * 3


def test_weights_without_columns_are_refused():
    """An empty reduction has no blocks and no 8-bit form: refused for both kinds of x, before
    a result is allocated."""
    w = nat.Fp8Rows(5, 0, device="cpu")
    for x in (torch.zeros(3, 0), nat.Fp8Rows(3, 0, device="cpu")):
        with pytest.raises(ValueError, match="no columns"):
            ltx_nn.linear_fp8(x, w)
        with pytest.raises(ValueError, match="no columns"):
            ltx_nn.linear_fp8(x, w, residual=torch.zeros(3, 5), dtype=torch.float32)
    with pytest.raises(ValueError, match="no columns"):
        ltx_nn.quantize_fp8(torch.zeros(3, 0))


class _FakeQuantiser:
    """Stands in for the quantiser: rows on the CPU that remember the weight's values."""

    def __init__(self, monkeypatch):
        self.seen = {}
        monkeypatch.setattr(ltx_nn, "quantize_fp8", self)

    def __call__(self, x, out=None):
        rows = out if out is not None else nat.Fp8Rows(*x.shape, device="cpu")
        self.seen[id(rows)] = (rows, x.clone())
        return rows

    def holds(self, module, name):
        rows = module.weight8(name, module._fp8_weight(name))
        return torch.equal(self.seen[id(rows)][1], module._fp8_weight(name))


@pytest.mark.parametrize("inference", [False, True])
def test_quantised_weights_follow_the_parameters(monkeypatch, inference):
    fake = _FakeQuantiser(monkeypatch)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    attn = ltx_nn.Attention(64, 128, heads=1, dim_head=64, apply_gated_attention=True)
    ff = ltx_nn.FeedForward(64)
    with torch.inference_mode(inference):
        attn.quantize_fp8(("q", "kv"))
        ff.quantize_fp8()
    kept = {(id(m), n): m.fp8[n] for m in (attn, ff) for n in m.fp8}

    def step(change):
        for m in (attn, ff):
            change(m)
        for m in (attn, ff):
            for n in m.fp8:
                assert fake.holds(m, n), (type(m).__name__, n)
                assert m.fp8[n] is kept[id(m), n]  # the same rows: captured graphs read them

    step(lambda m: m.load_state_dict({k: torch.randn_like(v) for k, v in m.state_dict().items()}))
    step(lambda m: m.load_state_dict({k: torch.randn_like(v) for k, v in m.state_dict().items()}, assign=True))

    def merge(m):
        with torch.no_grad():
            for p in m.parameters():
                p.add_(0.5)

    step(merge)
    with torch.inference_mode():
        step(merge)
    step(lambda m: m.to(torch.bfloat16))
    def uncounted(m):
        for p in m.parameters():
            p.data.mul_(2)
        m.quantize_fp8(("q", "kv")) if m is attn else m.quantize_fp8()

    step(uncounted)
    count = len(fake.seen)
    assert all(m.weight8(n, m._fp8_weight(n)) is m.fp8[n] for m in (attn, ff) for n in m.fp8) and len(fake.seen) == count
    assert attn.weight8("self", attn.to_q.weight) is None
    # rows that a caller put there are the caller's
    own = nat.Fp8Rows(64, 64, device="cpu")
    attn.fp8["own"] = own
    assert attn.weight8("own", attn.to_q.weight) is own
    ff.fp8["own"] = own
    for m in (attn, ff):
        m.load_state_dict(m.state_dict())
    assert attn.fp8["own"] is own and ff.fp8["own"] is own
    del attn.fp8["own"], ff.fp8["own"]
    # not in the middle of a capture, which would quantise at every replay
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    merge(ff)
    with pytest.raises(RuntimeError, match="before the capture"):
        ff.weight8("in", ff.proj_in.weight)


def test_quantise_into_rows(monkeypatch):
    with pytest.raises(ValueError, match="out is"):
        ltx_nn.quantize_fp8(torch.zeros(3, 64), nat.Fp8Rows(4, 64, device="cpu"))
    monkeypatch.setattr(nat, "_same_device", lambda *a: None)
    with pytest.raises(ValueError, match="out holds"):
        nat.quantize_fp8(torch.zeros(3, 64), out=nat.Fp8Rows(4, 64, device="cpu"))
    calls = []
    monkeypatch.setattr(nat, "_on", lambda t, name, *args, **kw: calls.append(args))
    rows = nat.Fp8Rows(3, 64, device="cpu")
    assert ltx_nn.quantize_fp8(torch.zeros(3, 64), rows) is rows
    assert calls[0][4:7] == rows.operand()


def test_rows_on_the_host_are_not_given_to_a_kernel():
    """Rows moved to the host (a pickled model, say) have addresses no kernel may read."""
    for dtype in (torch.bfloat16, torch.float32):
        with pytest.raises(ValueError, match="CUDA"):
            nat.Fp8Rows(3, 64, device="cpu").dequantize(dtype)


def test_operands_that_are_not_aligned_to_their_type_are_refused(lib):
    """Every remaining pointer that a kernel reads by element: scales, row masks, gate logits."""
    assert lib.ltx_fp8_pack_scales(P + 2, 2, 4, 256, P, None) == INVALID
    assert b"aligned" in lib.ltx_last_error()
    e = nat.Epilogue()
    e.kind, e.row_mask, e.row_vec = nat.EPI_ROW_MASK_ADD, P + 2, P
    assert lib.ltx_linear_fp8(P, 256, P, P, 256, P, P, 64, 4, 64, 256, ctypes.byref(e), 1, None) == INVALID
    assert b"row_mask" in lib.ltx_last_error()
    for dtype, gate in ((0, P + 2), (1, P + 1)):
        assert lib.ltx_attention_masked(P, 128, P, 128, P, 128, P, 128, 2, 5, 100, 2, 64, 0.125, P, 100, 0, gate, 2, dtype,
                                        None) == INVALID
        assert b"gate_logits" in lib.ltx_last_error()


def test_masked_attention_refuses_to_write_over_its_keys():
    """Blocks of queries read every key of their head, each at its own time: a result over k or
    v would be read as keys. Over q it is fine: a query's row is read before it is written."""
    buf = torch.zeros(3, 2, 9, 128, dtype=torch.bfloat16)
    q, k, v = buf
    ones = torch.ones(2, 9, dtype=torch.bool)
    across = buf.view(-1)[200:200 + k.numel()].view(2, 9, 128)  # starts inside q, ends inside k
    for out in (k, v, across):
        with pytest.raises(ValueError, match="overlap"):
            ltx_nn.cross_attention(q, k, v, 2, mask=ones, out=out)
    with pytest.raises(ValueError, match="CUDA"):
        ltx_nn.cross_attention(q, k, v, 2, mask=ones, out=q)
    with pytest.raises(ValueError, match="CUDA"):
        ltx_nn.cross_attention(q, k, v, 2, mask=ones, out=torch.empty_like(q))
