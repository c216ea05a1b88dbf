"""The 8-bit cache and key spans on the model's paths: what a wrong wiring would change."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("wants", ["x", "context", "q", "k", "v"])
def test_context_lengths_drop_no_gradient(wants):
    """Whichever of the inputs and weights wants one: the norms in front run outside of autograd on CUDA."""
    from streamdiffusionv2_b200.wan_model import TextCrossAttention
    m = TextCrossAttention(256, 2).to(DEV, torch.bfloat16).requires_grad_(False)
    x, ctx = _randn(1, 1, 4, 256), _randn(2, 1, 5, 256)
    {"x": x, "context": ctx}[wants].requires_grad_() if wants in ("x", "context") else getattr(m, wants).requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        m(x, ctx, [3])


def _stream(q8, adapt=-1, case_name="m_stream_1f"):
    """The latents of a stream and the pipeline behind it, eager."""
    import cases
    from streamdiffusionv2_b200.stream_pipeline import DiffusionWrapper, StreamPipeline
    from streamdiffusionv2_b200.wan_model import CausalWanModel
    case = cases.MODEL_CASES[case_name]
    model = CausalWanModel(**cases.MODEL_KW)
    cases.seed_parameters(model)
    model = model.to(device=DEV, dtype=torch.bfloat16).eval()
    prompt, first, chunks = cases.model_inputs(case)
    h, w = case["latent_hw"]
    pipe = StreamPipeline(DiffusionWrapper(model), lambda text_prompts: {"prompt_embeds": prompt.to(DEV, torch.bfloat16)},
                          case["levels"], cases.MODEL_KW["num_layers"], cases.MODEL_KW["num_heads"], (h // 2) * (w // 2),
                          case["cache_frames"], case["sink"], adapt, case["frames"], device=DEV, kv_cache_q8=q8)
    fs, sched = cases.model_schedule(case)
    outs = []
    with torch.no_grad():
        torch.manual_seed(11)
        outs.append(pipe.prepare(text_prompts=["p"], device=torch.device(DEV), dtype=torch.bfloat16,
                                 noise=first.to(DEV, torch.bfloat16), current_start=0, current_end=fs * (1 + case["frames"])))
        for (start, end), chunk in zip(sched, chunks):
            outs.append(pipe.inference_stream(chunk.to(DEV, torch.bfloat16), start, end).clone())
    return outs, pipe


@pytest.mark.parametrize("case_name", ["m_stream_1f", "m_stream"])
def test_a_stream_with_an_8_bit_cache_stays_near_the_bf16_one(monkeypatch, case_name):
    """Chunk by chunk.  The yardstick is a stream through a bf16 cache whose K and V are each put off by one whole step of the
    8-bit format, up or down at random: the format itself is off by a uniform half step at most, whose root mean square
    is sqrt(12) = 3.5 times smaller, so to first order the 8-bit stream's difference is that much smaller too.  It has
    to stay within the yardstick's, whereas a wrong slot, length or exponent moves the latents by their own size."""
    from streamdiffusionv2_b200 import ops
    q8, _ = _stream(True, case_name=case_name)
    plain, _ = _stream(False, case_name=case_name)
    true_append, gen = ops.rope_kv_append, torch.Generator(DEV).manual_seed(1)

    def off_by_a_step(q, k, v, k_cache, v_cache, table, grid, start_frames, dst_begin, **kw):
        out = true_append(q, k, v, k_cache, v_cache, table, grid, start_frames, dst_begin, **kw)
        for c in (k_cache, v_cache):
            for b, d in enumerate(dst_begin):
                x = c[b, d:d + q.shape[1]].float()
                step = torch.exp2(torch.floor(torch.log2(x.abs().amax(-1, keepdim=True).clamp_min(1e-30))) - 6)
                sign = torch.randint(0, 2, x.shape, generator=gen, device=DEV) * 2 - 1
                c[b, d:d + q.shape[1]] = (x + sign * step).to(c.dtype)
        return out

    monkeypatch.setattr(ops, "rope_kv_append", off_by_a_step)
    off, _ = _stream(False, case_name=case_name)
    rms = lambda x: x.float().square().mean().sqrt().item()  # noqa: E731
    for i, (a, p, o) in enumerate(zip(q8, plain, off)):
        assert 0 < rms(a - p) <= rms(o - p) < 0.5 * rms(p), (i, rms(a - p), rms(o - p), rms(p))
    ops.read_status(torch.device(DEV))


@pytest.mark.parametrize("adapt", [-1, 0.2])
def test_every_layer_of_a_stream_holds_and_attends_what_it_should(monkeypatch, adapt):
    """Call by call inside a whole stream, with and without the adaptive sink test: the bytes and exponents of the slot are
    the format of this call's K and V and nothing else changes; the attention is over the same cache up to the layer's
    end index, right against 64 bits; the sink similarities are those of what the cache holds."""
    import q8_reference as ref
    from oracle import causal_attention_oracle as orc
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    append, attend, similar = ops.rope_kv_append_q8, ops.attn_kvcache_q8, ca.adaptive_similarities
    table = torch.view_as_real(orc.rope_table(128)).contiguous()
    seen = {"append": 0, "attend": 0, "similar": 0}
    last = {}

    def checked_append(q, k, v, kc, vc, ke, ve, tab, grid, start_frames, dst_begin, **kw):
        before = [t.clone().cpu() for t in (kc, vc, ke, ve)]
        out = append(q, k, v, kc, vc, ke, ve, tab, grid, start_frames, dst_begin, **kw)
        if kw.get("step_params") is not None:
            start_frames, dst_begin = kw["step_params"][0].tolist(), kw["step_params"][1].tolist()
        held = (*ref.quantise(ref.rope64(k.cpu(), table, grid, start_frames)), *ref.quantise(v.cpu().double()))
        for want, new in zip(before, (held[0], held[2], held[1], held[3])):
            for b, d in enumerate(dst_begin):
                want[b, d:d + q.shape[1]] = new[b]
        for want, t in zip(before, (kc, vc, ke, ve)):
            assert torch.equal(t.cpu(), want)
        last.update(cache=(kc, vc, ke, ve), ends=kw["index_tensors"][1].tolist(), q=out)
        seen["append"] += 1
        return out

    def checked_attend(q, kc, vc, ke, ve, lens, **kw):
        out = attend(q, kc, vc, ke, ve, lens, **kw)
        assert q is last["q"] and all(a.data_ptr() == b.data_ptr() for a, b in zip((kc, vc, ke, ve), last["cache"]))
        assert list(lens) == last["ends"][:q.shape[0]]
        k, v = ref.values(kc.cpu(), ke.cpu()), ref.values(vc.cpu(), ve.cpu())
        end = torch.tensor(lens)[:, None].expand(-1, q.shape[1])
        want, weight = ref.span_attention(q.cpu(), k, v, torch.zeros_like(end), end)
        ref.check_attention(out, want, weight, k.shape[1])
        seen["attend"] += 1
        return out

    def checked_similar(kv, roped_k, v, sink, frame_tokens):
        got = similar(kv, roped_k, v, sink, frame_tokens)
        rows = roped_k.shape[0]
        sims = []
        for c, e, new in ((kv["k"], kv["k_exp"], roped_k), (kv["v"], kv["v_exp"], v)):
            old = ref.values(c[:rows, :sink * frame_tokens].cpu(), e[:rows, :sink * frame_tokens].cpu())
            old = old.reshape(rows, sink, frame_tokens, -1).mean(2)
            sims.append(torch.cosine_similarity(old, new.cpu().double().reshape(rows, 1, frame_tokens, -1).mean(2), dim=-1))
        # means rounded to bf16 (2^-8 of each value on either side) and a cosine in bf16: a few 2^-8
        assert ((sims[0] + sims[1]) / 2 - got.cpu().double()).abs().max().item() <= 2.0 ** -5
        seen["similar"] += 1
        return got

    monkeypatch.setattr(ops, "rope_kv_append_q8", checked_append)
    monkeypatch.setattr(ops, "attn_kvcache_q8", checked_attend)
    monkeypatch.setattr(ca, "adaptive_similarities", checked_similar)
    outs, pipe = _stream(True, adapt)
    assert seen["append"] == seen["attend"] > 0 and (seen["similar"] > 0) == (adapt >= 0)
    assert all(bool(torch.isfinite(t).all()) for t in outs)
    ops.read_status(torch.device(DEV))


def test_the_adaptive_sink_test_on_an_8_bit_cache_picks_the_oracles_slots():
    """Two rows of frames that keep or change their look: slots, index tensors and evict queues of a wrapping stream are
    those of the oracle on the values that the cache holds.  The decisions are far from the threshold."""
    import q8_reference as ref
    from oracle import causal_attention_oracle as orc
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    from streamdiffusionv2_b200.ring_state import RingState
    H, gh, gw, sink, frames, thr = 2, 3, 4, 2, 5, 0.25
    n, S = gh * gw, frames * gh * gw
    table, g = orc.rope_table(128), torch.Generator().manual_seed(21)

    class Attn:
        num_heads, head_dim, sink_size, adapt_sink_thr, evict_idx = H, 128, sink, thr, None

    module = Attn()
    kv = dict(ops.q8_cache(2, S, H, DEV), global_end_index=torch.zeros(2, dtype=torch.long, device=DEV),
              local_end_index=torch.zeros(2, dtype=torch.long, device=DEV), total_steps=1, current_step=1)
    st = orc.RingLayerState(S, 2)
    looks = {c: torch.randn(2, n, H, 128, generator=g) for c in "ab"}      # of K and V
    shows = ("aaaaabaabbab", "aaaaaaabaaaa")
    refreshed = [0, 0]
    for step in range(len(shows[0])):
        noise = lambda: 0.3 * torch.randn(2, n, H, 128, generator=g)  # noqa: E731
        v = (torch.stack([looks[s[step]][1] for s in shows]) + noise()).to(torch.bfloat16)
        k = (torch.stack([looks[s[step]][0] for s in shows]) + noise()).to(torch.bfloat16)
        q = torch.randn(2, n, H, 128, generator=g).to(torch.bfloat16)
        hk, hv = ref.values(kv["k"].cpu(), kv["k_exp"].cpu()), ref.values(kv["v"].cpu(), kv["v_exp"].cpu())
        rk = ref.rope64(k, torch.view_as_real(table).contiguous(), (1, gh, gw), [step, step])
        orc._ensure_queues(st)
        before = [t.cpu() for t in (kv["k"], kv["v"], kv["k_exp"], kv["v_exp"])]
        dst, lens = [], []
        for b in range(2):
            front = orc.adaptive_sink_front(hk, hv, rk, v.double(), b, sink, n, thr)
            if step >= sink:                                # before, the sink frames are empty: similarity 0
                margins = [orc.adaptive_sink_front(hk, hv, rk, v.double(), b, sink, n, thr + d) for d in (-0.05, 0.05)]
                assert margins[0] == margins[1] == front, (step, b)
            refreshed[b] += front is not None and step >= frames
            d, le = orc.ring_plan_row(st, b, step * n, n, n, sink, front)
            dst.append(d)
            lens.append(le)
        out = ca.cached_attention(module, *(t.to(DEV) for t in (q, k, v)), torch.tensor([[1, gh, gw]] * 2), table, kv,
                                  [step * n] * 2)
        held = (*ref.quantise(rk), *ref.quantise(v.double()))
        for want, new, name in zip(before, (held[0], held[2], held[1], held[3]), ("k", "v", "k_exp", "v_exp")):
            for b, d in enumerate(dst):
                want[b, d:d + n] = new[b]
            assert torch.equal(kv[name].cpu(), want), (step, name)
        RingState.sync_queue(module)
        assert [list(x) for x in module.evict_idx] == st.evict_idx, step
        assert kv["global_end_index"].tolist() == st.global_end and kv["local_end_index"].tolist() == st.local_end
        rq = ref.rope64(q, torch.view_as_real(table).contiguous(), (1, gh, gw), [step, step]).to(torch.bfloat16)
        end = torch.tensor(lens)[:, None].expand(-1, n)
        hk, hv = ref.values(kv["k"].cpu(), kv["k_exp"].cpu()), ref.values(kv["v"].cpu(), kv["v_exp"].cpu())
        want, weight = ref.span_attention(rq, hk, hv, torch.zeros_like(end), end)
        ref.check_attention(out, want, weight, S, step)
    assert refreshed[0] > 1 and refreshed[1] >= 1
    ops.read_status(torch.device(DEV))


@pytest.mark.parametrize("window", [-1, 3])
def test_a_clip_in_one_pass_is_streaming_block_by_block(window):
    """The same q, k, v as a whole clip and block by block through a bf16 cache that keeps every frame: both against 64-bit
    attention with a mask written out from frame and block numbers.  (With a window: the clip alone.)"""
    import q8_reference as ref
    from oracle import causal_attention_oracle as orc
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    H, frames, gh, gw, per = 2, 6, 6, 9, 2
    n, m = frames * gh * gw, per * gh * gw
    q, k, v = (_randn(i, 2, n, H, 128) for i in range(3))
    table = orc.rope_table(128)
    spans = ca.block_causal_spans(frames, gh * gw, per, DEV, rows=2, window_frames=window)
    clip = ca.clip_attention(q, k, v, torch.tensor([[frames, gh, gw]] * 2), table, spans)
    rq, rk = (ref.rope64(t.cpu(), torch.view_as_real(table).contiguous(), (frames, gh, gw), [0, 0]).to(torch.bfloat16).to(DEV)
              for t in (q, k))
    frame = torch.arange(n) // (gh * gw)
    end_frame = (frame // per + 1) * per
    begin = torch.zeros_like(frame) if window < 0 else (end_frame - window).clamp_min(0)
    want, weight = ref.span_attention(rq, rk, v, (begin * gh * gw).expand(2, -1), (end_frame * gh * gw).expand(2, -1))
    ref.check_attention(clip, want, weight, n, window)
    if window > 0:
        return

    class Attn:
        num_heads, head_dim, sink_size, adapt_sink_thr, evict_idx = H, 128, 0, -1, None

    kv = {name: torch.zeros(2, n, H, 128, dtype=torch.bfloat16, device=DEV) for name in ("k", "v")}
    kv.update(global_end_index=torch.zeros(2, dtype=torch.long, device=DEV),
              local_end_index=torch.zeros(2, dtype=torch.long, device=DEV), total_steps=1, current_step=1)
    module = Attn()
    streamed = torch.cat([ca.cached_attention(module, *(t[:, s:s + m] for t in (q, k, v)), torch.tensor([[per, gh, gw]] * 2),
                                              table, kv, [s] * 2) for s in range(0, n, m)], 1)
    ref.check_attention(streamed, want, weight, n)
    ops.read_status(torch.device(DEV))


def test_a_clip_forward_is_the_streamed_forward(monkeypatch):
    """forward_clip against the cached model block by block at the same timestep, text K/V shared.  The two differ by
    the roundings of their attention kernels (about 2^-9 of the output each, root mean square); the yardstick is the
    streamed forward with every self-attention output put off by 2^-7 of itself, up or down at random."""
    import cases
    from streamdiffusionv2_b200 import causal_attention as ca, ops
    from streamdiffusionv2_b200.wan_model import CausalWanModel
    model = CausalWanModel(**cases.MODEL_KW)
    cases.seed_parameters(model)
    model = model.to(device=DEV, dtype=torch.bfloat16).eval()
    heads, per, frames, gh, gw = cases.MODEL_KW["num_heads"], 2, 6, 6, 5
    for blk in model.blocks:
        blk.self_attn.sink_size, blk.self_attn.adapt_sink_thr = 0, -1
    x, t = _randn(1, 2, 16, frames, 2 * gh, 2 * gw), torch.full((2, frames), 500, device=DEV)
    ctx = _randn(2, 2, 512, cases.MODEL_KW["text_dim"])
    clip = model.forward_clip(x, t, ctx, frames_per_block=per)

    def streamed():
        n, m = frames * gh * gw, per * gh * gw
        kvs = [{"k": torch.zeros(2, n, heads, 128, dtype=torch.bfloat16, device=DEV),
                "v": torch.zeros(2, n, heads, 128, dtype=torch.bfloat16, device=DEV),
                "global_end_index": torch.zeros(2, dtype=torch.long, device=DEV),
                "local_end_index": torch.zeros(2, dtype=torch.long, device=DEV), "total_steps": 1, "current_step": 1}
               for _ in model.blocks]
        cross = [{"k": None, "v": None, "is_init": False} for _ in model.blocks]
        for blk in model.blocks:
            blk.self_attn.evict_idx = None
        with torch.no_grad():
            parts = [model(x[:, :, f:f + per], t[:, f:f + per], ctx, 10 ** 6, kv_cache=kvs, crossattn_cache=cross,
                           current_start=torch.full((2,), f * gh * gw, dtype=torch.long, device=DEV),
                           current_end=f * gh * gw + m) for f in range(0, frames, per)]
        return torch.cat(parts, 2)

    by_block = streamed()
    attend, gen = ops.attn_kvcache, torch.Generator(DEV).manual_seed(1)

    def put_off(*args, **kw):
        out = attend(*args, **kw)
        sign = torch.randint(0, 2, out.shape, generator=gen, device=DEV) * 2 - 1
        return (out.float() * (1 + sign * 2.0 ** -7)).to(out.dtype)

    monkeypatch.setattr(ops, "attn_kvcache", put_off)
    off = streamed()
    rms = lambda y: y.float().square().mean().sqrt().item()  # noqa: E731
    assert rms(clip - by_block) <= rms(off - by_block) < 0.1 * rms(by_block), (rms(clip - by_block), rms(off - by_block), rms(by_block))
    ops.read_status(torch.device(DEV))
