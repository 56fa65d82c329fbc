"""The 8-bit products and the masked text context inside the models: LTXModel.quantize_fp8,
Modality.context_mask, guided and CFG steps, Attention.forward(mask) and the connector
without registers."""

import pytest
import torch

import _native as nat
import ltx_dit
import ltx_nn
import ltx_te
from model_fixtures import philox_model
from oracle import ltx_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def rel_l2(a, b):
    a, b = a.detach().float().cpu(), b.detach().float().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def video_inputs(cfg, dtype, frames=(3, 8, 8), s=40, b=2, seed=5):
    f, h, w = frames
    t = f * h * w
    g = torch.Generator(device=DEV).manual_seed(seed)
    lat = torch.randn(b, t, cfg.video_in, generator=g, device=DEV).to(dtype)
    ctx = torch.randn(b, s, cfg.video_cross_dim, generator=g, device=DEV).to(dtype)
    pos = ltx_dit.video_positions(b, f, h, w, 24.0, DEV)
    sig = torch.full((b,), 0.7, device=DEV)
    return ltx_dit.Modality(latent=lat, sigma=sig, timesteps=torch.full((b, t, 1), 0.7, device=DEV), positions=pos,
                            context=ctx)


def small_cfg(dtype=torch.bfloat16, cross_adaln=False):
    cfg = ltx_dit.DiTConfig.video_only(num_layers=2, heads=4, head_dim=64, cross_dim=384)
    if cross_adaln:
        import dataclasses

        cfg = dataclasses.replace(cfg, cross_attention_adaln=True, video_cross_dim=256)
    return cfg


# ------------------------------------------------------------------------------- fp8


@pytest.mark.parametrize("cross_adaln", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantized_model_follows_the_model(dtype, cross_adaln):
    """Every product's operands are off by at most half an e4m3 step, 2^-4 of a value, 2^-4 /
    sqrt(3) = 3.6 % in the root mean square, so a product by at most 5.1 % of its size; a
    branch of the block chains two of them (7.2 %) before its gated residual update, and
    attention weights move by the relative change of scores of about 1 (another 5.1 %).
    The stream they are added to is exact at first and carries at most the sum of the
    branches' errors: below 15 % of the velocity for two blocks."""
    cfg = small_cfg(cross_adaln=cross_adaln)
    model, _ = philox_model(cfg, 11, host_copy=False, dtype=dtype)
    video = video_inputs(cfg, dtype)
    want, _ = model(video, None)
    assert model.quantize_fp8() is model
    with nat.profile() as prof:
        got, _ = model(video, None)
    calls = prof.summary()
    n8 = sum(v["launches"] for k, v in calls.items() if "linear_fp8" in k)
    n16 = sum(v["launches"] for k, v in calls.items() if k.startswith("linear "))
    blocks = cfg.num_layers
    # per block: qkv, out, text q, text out, feed-forward in and out (and the text k, v)
    assert n8 == blocks * (7 if cross_adaln else 6), calls.keys()
    assert n16 > 0  # the projections around the blocks and the gates' logits keep their type
    assert got.dtype == dtype and torch.isfinite(got).all()
    assert 1e-4 < rel_l2(got, want) < 0.15, rel_l2(got, want)
    assert torch.equal(model(video, None)[0], got)
    assert nat.device_error_flags() == 0


def test_quantized_block_against_the_dequantized_weights():
    """The same model with every block weight replaced by the values of its 8-bit form, in
    bf16 (exact: 4 bits): what is left is the activations' quantisation alone, half the
    variance of the above."""
    cfg = small_cfg()
    model, host = philox_model(cfg, 12)
    video = video_inputs(cfg, torch.bfloat16)
    model.quantize_fp8()
    got, _ = model(video, None)
    plain, _ = philox_model(cfg, 12, host_copy=False)
    for blk, ref in zip(plain.blocks, model.blocks):
        for name in ("attn1", "attn2"):
            a, r = getattr(blk, name), getattr(ref, name)
            w, _ = a.packed_self() if name == "attn1" else a.packed_q()
            w.copy_(r.fp8["self" if name == "attn1" else "q"].dequantize())
            a.to_out.weight.data.copy_(r.fp8["out"].dequantize())
        blk.ff.proj_in.weight.data.copy_(ref.ff.fp8["in"].dequantize())
        blk.ff.proj_out.weight.data.copy_(ref.ff.fp8["out"].dequantize())
    want, _ = plain(video, None)
    both, _ = philox_model(cfg, 12, host_copy=False)[0](video, None)
    assert rel_l2(got, want) < 0.15 / 2 ** 0.5
    assert rel_l2(got, want) < rel_l2(got, both)


def test_quantized_audio_video_model_and_guided_step():
    cfg = ltx_dit.DiTConfig(num_layers=2, video_heads=4, video_head_dim=64, video_cross_dim=256, audio_heads=4,
                            audio_head_dim=64, audio_cross_dim=256, audio_ff_bias=True)
    model, _ = philox_model(cfg, 13, host_copy=False)
    vs, as_ = ltx_dit.create_noised_states(1, 17, 128, 128, 24.0, 3, DEV, torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(2)
    ctx = {k: torch.randn(1, 32, 256, generator=g, device=DEV).to(torch.bfloat16)
           for k in ("v_pos", "v_neg", "a_pos", "a_neg")}
    p = ltx_dit.GuiderParams(cfg_scale=3.0, stg_scale=1.0, rescale_scale=0.7, modality_scale=3.0, stg_blocks=[1])
    args = (vs, as_, ctx, torch.tensor(0.6), 0, p, p, cfg)
    _, _, want = ltx_dit.guided_denoise_step(model, *args)
    model.quantize_fp8()
    dv, da, got = ltx_dit.guided_denoise_step(model, *args)
    assert torch.isfinite(dv.float()).all() and torch.isfinite(da.float()).all()
    for name in want:  # the passes' x0 = latent - 0.6 velocity, before the guidance amplifies differences
        for i in range(2):
            assert rel_l2(got[name][i], want[name][i]) < 0.15
    # masks of padded prompts: the padding's content does not matter, to the last bit
    ctx["v_neg_mask"] = torch.arange(32, device=DEV)[None] >= 11
    ctx["a_pos_mask"] = torch.arange(32, device=DEV)[None] < 20
    dv, da, _ = ltx_dit.guided_denoise_step(model, *args)
    noisy = dict(ctx)
    noisy["v_neg"], noisy["a_pos"] = ctx["v_neg"].clone(), ctx["a_pos"].clone()
    noisy["v_neg"][:, :11] = 7.0
    noisy["a_pos"][:, 20:] = -3.0
    dv2, da2, _ = ltx_dit.guided_denoise_step(model, vs, as_, noisy, *args[3:])
    assert torch.equal(dv, dv2) and torch.equal(da, da2)


def test_quantized_cfg_step_captured_in_a_graph():
    cfg = small_cfg()
    model, _ = philox_model(cfg, 14, host_copy=False)
    model.quantize_fp8()
    m = video_inputs(cfg, torch.bfloat16, b=1)
    ctx = torch.randn(2, 24, 384, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.bfloat16)
    mask = torch.arange(24, device=DEV)[None] < 9
    sigmas = torch.linspace(1.0, 0.0, 9)
    lat = m.latent.clone()

    cp, cn = ctx[:1].contiguous(), ctx[1:].contiguous()

    def step():
        return ltx_dit.cfg_denoise_step(model, lat, m.positions, cp, cn, sigmas, 2, 3.0, context_mask_neg=mask)

    eager = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    for a, b in zip(out, eager):
        assert torch.equal(a, b)
    lat.copy_(torch.randn_like(lat))
    graph.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------ masks


@pytest.mark.parametrize("cross_adaln", [False, True])
@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_context_equals_the_short_context(dtype, side, cross_adaln):
    """The text keys carry no position, so a padded and masked context gives what the context
    without its padding gives, within the two attention kernels' rounding (the model's bar:
    1e-2 in bf16, 1e-4 in fp32); what the padding holds changes no bit."""
    cfg = small_cfg(cross_adaln=cross_adaln)
    model, _ = philox_model(cfg, 15, host_copy=False, dtype=dtype)
    video = video_inputs(cfg, dtype, s=40)
    keep = 23
    sl = slice(40 - keep, 40) if side == "left" else slice(0, keep)
    import dataclasses

    want, _ = model(dataclasses.replace(video, context=video.context[:, sl].contiguous()), None)
    mask = torch.zeros(1, 40, dtype=torch.bool, device=DEV)
    mask[:, sl] = True
    masked = dataclasses.replace(video, context_mask=mask)
    got, _ = model(masked, None)
    assert rel_l2(got, want) < (1e-2 if dtype == torch.bfloat16 else 1e-4)
    assert rel_l2(got, model(video, None)[0]) > 1e-4  # the mask does something
    ctx = video.context.clone()
    ctx[:, ~mask[0]] = 100.0
    assert torch.equal(model(dataclasses.replace(masked, context=ctx), None)[0], got)
    additive = torch.where(mask, 0.0, torch.finfo(dtype).min).to(dtype)
    assert torch.equal(model(dataclasses.replace(masked, context_mask=additive), None)[0], got)


def test_attention_module_masks():
    torch.manual_seed(3)
    attn = ltx_nn.Attention(256, 192, heads=4, dim_head=64, apply_gated_attention=True).to(DEV, torch.bfloat16)
    own = ltx_nn.Attention(256, None, heads=4, dim_head=64).to(DEV, torch.bfloat16)
    x = torch.randn(2, 70, 256, device=DEV, dtype=torch.bfloat16)
    ctx = torch.randn(2, 50, 192, device=DEV, dtype=torch.bfloat16)
    mask = torch.arange(50, device=DEV)[None] < 31
    with torch.inference_mode():
        assert rel_l2(attn(x, ctx, mask=mask), attn(x, ctx[:, :31])) < 1e-2
        assert rel_l2(attn(x, ctx, mask=mask[:, None, None]), attn(x, ctx[:, :31])) < 1e-2
        # a self-attention over its first 40 tokens gives those tokens what they give alone
        m2 = torch.arange(70, device=DEV)[None] < 40
        assert rel_l2(own(x, mask=m2)[:, :40], own(x[:, :40])) < 1e-2
        with pytest.raises(ValueError, match="key mask"):
            attn(x, ctx, mask=m2)
        with pytest.raises(NotImplementedError):
            attn(x, ctx, mask=torch.ones(2, 1, 70, 50, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_connector_without_registers_against_the_oracle(dtype):
    """The additive mask of a connector without learnable registers (it raised before)."""
    conn = ltx_te.Embeddings1DConnector(heads=4, dim_head=64, num_layers=2, max_pos=[64], registers=0, gated=True,
                                        ff_bias=True)
    sd = ltx_oracle.synthetic_state_dict([(k, tuple(v.shape)) for k, v in conn.named_parameters()], 4)
    conn.load_state_dict(sd)
    conn = conn.to(DEV, dtype)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 48, 256, generator=g).to(dtype)
    mask = torch.zeros(2, 1, 1, 48, dtype=dtype)
    mask[0, ..., 30:] = -10000.0  # a common padding value: large, not the lowest
    mask[1, ..., :13] = torch.finfo(dtype).min
    want, _ = ltx_oracle.connector_forward({k: v.to(dtype) for k, v in sd.items()}, "", 4, 64, 2, [64], 0, True, x, mask)
    got, out_mask = conn(x.to(DEV), mask.to(DEV))
    assert rel_l2(got, want) < (1e-2 if dtype == torch.bfloat16 else 1e-4)
    assert torch.equal(out_mask.cpu(), mask)


# ----------------------------------------------------------------- weights that change


def _modules():
    torch.manual_seed(21)
    attn = ltx_nn.Attention(256, 192, heads=4, dim_head=64, apply_gated_attention=True).to(DEV, torch.bfloat16)
    ff = ltx_nn.FeedForward(256).to(DEV, torch.bfloat16)
    attn.quantize_fp8(("q", "kv"))
    ff.quantize_fp8()
    return attn, ff


def test_quantised_modules_follow_their_weights():
    """After load_state_dict, in-place updates and moves the products use what the parameters
    hold now: the bits of a module that was quantised with them."""
    attn, ff = _modules()
    x = torch.randn(2, 70, 256, device=DEV, dtype=torch.bfloat16)
    ctx = torch.randn(2, 50, 192, device=DEV, dtype=torch.bfloat16)

    def outputs(a, f):
        with torch.inference_mode():
            return a(x, ctx), f(x)

    def fresh():
        a = ltx_nn.Attention(256, 192, heads=4, dim_head=64, apply_gated_attention=True).to(DEV, torch.bfloat16)
        f = ltx_nn.FeedForward(256).to(DEV, torch.bfloat16)
        a.load_state_dict(attn.state_dict())
        f.load_state_dict(ff.state_dict())
        a.quantize_fp8(("q", "kv"))
        f.quantize_fp8()
        return outputs(a, f)

    def merge():
        with torch.no_grad():
            for m in (attn, ff):
                for name, p in m.named_parameters():
                    if name.startswith(("to_", "proj_")):
                        p.add_(torch.randn_like(p) * 0.02)

    def load():
        for m in (attn, ff):
            m.load_state_dict({k: v + torch.randn_like(v) * 0.02 for k, v in m.state_dict().items()})

    def move():
        for m in (attn, ff):
            m.to(torch.float32)
            merge()
            m.to(torch.bfloat16)

    old = outputs(attn, ff)
    for change in (load, merge, move):
        change()
        new = outputs(attn, ff)
        for a, b, c in zip(new, fresh(), old):
            assert torch.equal(a, b) and not torch.equal(a, c), change.__name__
        old = new


def test_captured_products_follow_loaded_weights():
    """A graph reads the 8-bit rows by address: loading weights, and quantising again, write the
    same rows."""
    attn, ff = _modules()
    x = torch.randn(2, 70, 256, device=DEV, dtype=torch.bfloat16)
    ctx = torch.randn(2, 50, 192, device=DEV, dtype=torch.bfloat16)

    def step():
        return ff(attn(x, ctx))

    with torch.inference_mode():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for again in (False, True):
            for m in (attn, ff):
                if again:
                    for p in m.parameters():
                        p.data.mul_(0.9)
                else:
                    m.load_state_dict({k: v + torch.randn_like(v) * 0.02 for k, v in m.state_dict().items()})
            if again:
                attn.quantize_fp8(("q", "kv"))
                ff.quantize_fp8()
            graph.replay()
            assert torch.equal(out, step())


def test_quantised_model_with_other_weights_loaded():
    cfg = small_cfg()
    model, _ = philox_model(cfg, 31, host_copy=False)
    other, _ = philox_model(cfg, 32, host_copy=False)
    model.quantize_fp8()
    video = video_inputs(cfg, torch.bfloat16)
    first, _ = model(video, None)
    model.load_state_dict(other.state_dict())
    video.context = video.context.clone()  # the projection of a context is cached with it
    got, _ = model(video, None)
    other.quantize_fp8()
    assert torch.equal(got, other(video, None)[0]) and not torch.equal(got, first)


def test_connector_block_runs_its_quantised_weights():
    """Modules that were quantised are used so wherever they stand: four 8-bit products a block."""
    conn = ltx_te.Embeddings1DConnector(heads=4, dim_head=64, num_layers=1, max_pos=[64], registers=0, gated=False,
                                        ff_bias=True)
    sd = ltx_oracle.synthetic_state_dict([(k, tuple(v.shape)) for k, v in conn.named_parameters()], 5)
    conn.load_state_dict(sd)
    conn = conn.to(DEV, torch.bfloat16)
    x = torch.randn(2, 48, 256, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    want = conn.blocks[0](x)
    conn.blocks[0].attn1.quantize_fp8(("self",))
    conn.blocks[0].ff.quantize_fp8()
    with nat.profile() as prof:
        got = conn.blocks[0](x)
    calls = prof.summary()
    assert sum(v["launches"] for k, v in calls.items() if "linear_fp8" in k) == 4
    assert not any(k.startswith("linear ") for k in calls)
    assert 1e-4 < rel_l2(got, want) < 0.15


@pytest.mark.parametrize("quantised", [False, True])
def test_a_cached_context_projection_follows_the_weights(quantised):
    """The keys and values of a text context are kept over the denoise steps, not over a change
    of the weights that made them."""
    cfg = small_cfg()
    model, _ = philox_model(cfg, 33, host_copy=False)
    other, _ = philox_model(cfg, 34, host_copy=False)
    if quantised:
        model.quantize_fp8()
        other.quantize_fp8()
    video = video_inputs(cfg, torch.bfloat16)
    model(video, None)
    model.load_state_dict(other.state_dict())
    assert torch.equal(model(video, None)[0], other(video, None)[0])
    with torch.no_grad():
        for m in (model, other):
            for name, p in m.named_parameters():
                if name.endswith(("attn2.to_k.bias", "attn2.to_v.weight", "attn2.k_norm.weight")):
                    p.mul_(1.5)
    other._kv_cache.clear()
    assert torch.equal(model(video, None)[0], other(video, None)[0])
