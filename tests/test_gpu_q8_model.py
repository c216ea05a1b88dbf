"""The 8-bit K/V cache and key spans on the model's own paths: streaming pipeline, step graphs, whole clips, prompt
lengths."""
import pytest
import torch

import cases
import q8_reference as ref
from oracle import causal_attention_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Attn:
    num_heads, head_dim, sink_size, adapt_sink_thr, evict_idx = 2, 128, 1, -1, None


def _kv(rows, tokens, heads, q8):
    from streamdiffusionv2_b200 import ops
    t = ops.q8_cache(rows, tokens, heads, DEV) if q8 else {
        n: torch.zeros(rows, tokens, heads, 128, dtype=torch.bfloat16, device=DEV) for n in ("k", "v")}
    return {**t, "global_end_index": torch.zeros(rows, dtype=torch.long, device=DEV),
            "local_end_index": torch.zeros(rows, dtype=torch.long, device=DEV), "total_steps": 1, "current_step": 1}


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("with_norm", [False, True])
def test_cached_attention_over_an_8_bit_cache(with_norm):
    """A wrapping stream: index tensors and evict queue as with a bf16 cache, the cache what the format makes of the bf16
    cache path's K and V, the output attention over the values it holds."""
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    H, gh, gw, frames = 2, 4, 5, 2
    n, S = frames * gh * gw, 7 * gh * gw
    table, grid = orc.rope_table(128), torch.tensor([[frames, gh, gw]])
    mods, kvs = (_Attn(), _Attn()), (_kv(1, S, H, True), _kv(1, S, H, False))
    norm = (_randn(7, H * 128), _randn(8, H * 128), 1e-6) if with_norm else None
    for step in range(7):
        q, k, v = (_randn(10 * step + i, 1, n, H, 128) for i in range(3))
        outs = [ca.cached_attention(m, q, k, v, grid, table, kv, [step * n], norm=norm) for m, kv in zip(mods, kvs)]
        q8, plain = kvs
        for name in ("global_end_index", "local_end_index"):
            assert q8[name].tolist() == plain[name].tolist()
        assert mods[0].evict_idx == mods[1].evict_idx
        filled = int(q8["local_end_index"][0])
        # V is stored from the same bf16 values; K from the unrounded rope, at most a rounding step apart
        held, exps = ref.quantise(plain["v"][:, :filled].double().cpu())
        assert torch.equal(q8["v"][:, :filled].cpu(), held) and torch.equal(q8["v_exp"][:, :filled].cpu(), exps)
        kk, vv = ops.kv_read_q8(q8["k"], q8["v"], q8["k_exp"], q8["v_exp"], [0], filled, dtype=torch.float32)
        top = plain["k"][:, :filled].float().abs().amax(-1, keepdim=True)
        # half a step of 2^-6 of the exponent (<= 2^-6 of the maximum; a whole one above 127.5 steps) and the bf16 cache's own 2^-8
        assert bool(((kk - plain["k"][:, :filled].float()).abs() <= top * (2.0 ** -6 + 2.0 ** -8)).all())
        qn = q if norm is None else ops.rmsnorm(q.flatten(2), norm[0], norm[2]).view_as(q)
        rq = ops.rope_kv_append(qn, torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q),
                                ops.rope_table_device(table, q.device), (frames, gh, gw), [step * frames], [0])
        end = torch.full((1, n), filled)
        want, weight = ref.span_attention(rq, kk, vv, torch.zeros_like(end), end)
        ref.check_attention(outs[0], want, weight, filled, step)
    ops.read_status(torch.device(DEV))


def _stream(q8, graphs, adapt=-1, case_name="m_stream_1f"):
    from streamdiffusionv2_b200.ring_state import RingState
    from streamdiffusionv2_b200.stream_pipeline import DiffusionWrapper, StreamPipeline
    from streamdiffusionv2_b200.wan_model import CausalWanModel
    case = cases.MODEL_CASES[case_name]
    model = CausalWanModel(**cases.MODEL_KW)
    cases.seed_parameters(model)
    model = model.to(device=DEV, dtype=torch.bfloat16).eval()
    prompt, first, chunks = (cases.model_inputs(case))
    h, w = case["latent_hw"]
    pipe = StreamPipeline(DiffusionWrapper(model), lambda text_prompts: {"prompt_embeds": prompt.to(DEV, torch.bfloat16)},
                          case["levels"], cases.MODEL_KW["num_layers"], cases.MODEL_KW["num_heads"], (h // 2) * (w // 2),
                          case["cache_frames"], case["sink"], adapt, case["frames"], device=DEV, kv_cache_q8=q8)
    fs, sched = cases.model_schedule(case)
    outs = []
    with torch.no_grad():
        torch.manual_seed(11)
        pipe.prepare(text_prompts=["p"], device=torch.device(DEV), dtype=torch.bfloat16, noise=first.to(DEV, torch.bfloat16),
                     current_start=0, current_end=fs * (1 + case["frames"]))
        if graphs:
            pipe.enable_step_graphs()
        for (start, end), chunk in zip(sched, chunks):
            outs.append(pipe.inference_stream(chunk.to(DEV, torch.bfloat16), start, end).clone())
    for blk in model.blocks:
        RingState.sync_queue(blk.self_attn)
    state = [(kv["global_end_index"].tolist(), kv["local_end_index"].tolist(), blk.self_attn.evict_idx)
             for kv, blk in zip(pipe.kv_cache1, model.blocks)]
    return outs, pipe, state


@pytest.mark.parametrize("adapt", [-1, 0.2])
def test_streaming_with_an_8_bit_cache(adapt):
    """Same index state as with the bf16 cache (without the data-dependent sink test), finite latents near the bf16
    cache's, half the cache memory; steps replayed from a graph leave what eager steps leave, bit for bit."""
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    eager, pipe, state = _stream(True, False, adapt)
    replayed, gpipe, gstate = _stream(True, True, adapt)
    assert gpipe.step_graphs.replays > 0
    for a, b in zip(eager, replayed):
        assert torch.equal(a, b)
    assert state == gstate
    for x, y in zip(pipe.kv_cache1, gpipe.kv_cache1):
        assert all(torch.equal(x[n], y[n]) for n in ca.cache_tensors(x))
    plain, ppipe, pstate = _stream(False, False, adapt)
    if adapt < 0:
        assert state == pstate
    size = lambda p: sum(kv[n].numel() * kv[n].element_size() for kv in p.kv_cache1 for n in ca.cache_tensors(kv))  # noqa: E731
    assert size(pipe) * 256 == size(ppipe) * 129
    assert all(bool(torch.isfinite(t).all()) for t in eager)
    ops.read_status(torch.device(DEV))


def test_clip_attention_is_what_streaming_through_a_cache_computes():
    """Blocks of a clip in one pass against 64-bit attention over the keys that streaming block by block would hold."""
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    H, frames, gh, gw, per = 2, 6, 6, 9, 2
    n = frames * gh * gw
    q, k, v = (_randn(i, 2, n, H, 128) for i in range(3))
    table = orc.rope_table(128)
    for window in (-1, 3):
        spans = ca.block_causal_spans(frames, gh * gw, per, DEV, rows=2, window_frames=window)
        out = ca.clip_attention(q, k, v, torch.tensor([[frames, gh, gw]] * 2), table, spans)
        rq, rk = (orc.rope_apply(t.cpu(), (frames, gh, gw), table, [0, 0]).to(torch.bfloat16) for t in (q, k))
        begin = torch.zeros_like(spans.end) if spans.begin is None else spans.begin
        want, weight = ref.span_attention(rq.to(DEV), rk.to(DEV), v, begin, spans.end)
        ref.check_attention(out, want, weight, n, window)
    ops.read_status(torch.device(DEV))


def test_clip_forward_is_causal_over_blocks_and_heeds_prompt_lengths():
    """Later blocks change nothing in earlier ones, text behind a prompt's length changes nothing at all."""
    from streamdiffusionv2_b200.wan_model import CausalWanModel
    model = CausalWanModel(**cases.MODEL_KW)
    cases.seed_parameters(model)
    model = model.to(device=DEV, dtype=torch.bfloat16).eval()
    x, t = _randn(1, 2, 16, 4, 12, 10), torch.full((2, 4), 500, device=DEV)
    ctx = _randn(2, 2, 512, cases.MODEL_KW["text_dim"])
    lens = torch.tensor([512, 60], device=DEV)
    out = model.forward_clip(x, t, ctx, frames_per_block=2, context_lens=lens)
    assert out.shape == x.shape and bool(torch.isfinite(out).all())
    x2, ctx2 = x.clone(), ctx.clone()
    x2[:, :, 2:] = _randn(3, 2, 16, 2, 12, 10)
    ctx2[1, 60:] = 50.0
    again = model.forward_clip(x2, t, ctx2, frames_per_block=2, context_lens=lens)
    assert torch.equal(out[:, :, :2], again[:, :, :2]) and not torch.equal(out[:, :, 2:], again[:, :, 2:])
    whole = model.forward_clip(x, t, ctx2, frames_per_block=2)
    assert not torch.equal(whole[1], out[1])


def test_cross_attention_context_lengths():
    """Rows with lengths 512, 77, 1 and 0 against the same module on each row's own text; a gradient is refused."""
    from streamdiffusionv2_b200.wan_model import TextCrossAttention
    torch.manual_seed(0)
    m = TextCrossAttention(256, 2).to(DEV, torch.bfloat16)
    x, ctx = _randn(1, 4, 150, 256), _randn(2, 4, 512, 256)
    lens = [512, 77, 1, 0]
    with torch.no_grad():
        out = m(x, ctx, torch.tensor(lens, device=DEV))
        for b, n in enumerate(lens[:3]):
            alone = m(x[b:b + 1], ctx[b:b + 1, :n].contiguous(), None)
            # o-projection of attention outputs that are a rounding step (2^-8) apart at most: 256 terms of it
            assert (out[b] - alone[0]).abs().max().item() <= 2.0 ** -7 * 2 * alone.abs().max().item()
        assert torch.equal(out[3], m.o(torch.zeros_like(x[3])))
    with pytest.raises(RuntimeError):
        m(x.requires_grad_(), ctx, torch.tensor(lens, device=DEV))
