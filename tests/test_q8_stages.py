"""The 8-bit cache of a pipeline-parallel stream on CPU ranks (gloo): its four tensors are shared by prepare, replicated,
released or kept for blocks that a rank does not own, and move between stages with their block.  The kernels are stood
in for by plain statements of them."""
import traceback

import pytest
import torch
import torch.distributed as dist

import cases
import test_stage_transport as stages

NAMES = ("k", "v", "k_exp", "v_exp")


def _fakes(monkeypatch):
    """The oracle's stand-ins, and for the 8-bit cache the tests' statements of its format."""
    import fake_ops
    import q8_reference as ref
    from oracle import causal_attention_oracle as orc
    from streamdiffusionv2_b200 import ops
    fake_ops.install(monkeypatch)

    def append(q, k, v, kc, vc, ke, ve, table, grid, start_frames, dst_begin, *, index_tensors=None, index_values=None):
        rk = orc.rope_apply(k, grid, table, start_frames)
        for c, e, x in ((kc, ke, rk), (vc, ve, v)):
            m, exps = ref.quantise(x.double())
            for b, d in enumerate(dst_begin):
                c[b, d:d + q.shape[1]], e[b, d:d + q.shape[1]] = m[b], exps[b]
        for t, values in zip(index_tensors, index_values):
            t.data[:len(values)] = torch.tensor(values[:t.numel()], dtype=torch.long)
        return orc.rope_apply(q, grid, table, start_frames).type_as(v)

    def attend(q, kc, vc, ke, ve, lens):
        return orc.attend_cache(q, ref.values(kc, ke).to(q.dtype), ref.values(vc, ve).to(q.dtype), lens)

    monkeypatch.setattr(ops, "rope_kv_append_q8", append)
    monkeypatch.setattr(ops, "attn_kvcache_q8", attend)


def _pipeline(case):
    from streamdiffusionv2_b200.stream_pipeline import DiffusionWrapper, StreamPipeline
    from streamdiffusionv2_b200.wan_model import CausalWanModel
    model = CausalWanModel(**cases.MODEL_KW)
    cases.seed_parameters(model)
    model = model.to(torch.bfloat16).eval()
    prompt, first, chunks = cases.model_inputs(case)
    h, w = case["latent_hw"]
    pipe = StreamPipeline(DiffusionWrapper(model), lambda text_prompts: {"prompt_embeds": prompt.to(torch.bfloat16)}, case["levels"],
                          cases.MODEL_KW["num_layers"], cases.MODEL_KW["num_heads"], (h // 2) * (w // 2), case["cache_frames"],
                          case["sink"], -1, case["frames"], device="cpu", kv_cache_q8=True)
    return pipe, first.to(torch.bfloat16), [c.to(torch.bfloat16) for c in chunks]


def _held(pipe):
    return {i: {n: kv[n].numpy().copy() for n in NAMES} for i, kv in enumerate(pipe.kv_cache1) if kv["k"].shape[1] > 0}


def _worker(rank, world, port, ranges, new_ranges, unowned, q):
    """4 chunks, blocks moved where new_ranges says so, 4 more chunks; rank 1 prepares from other noise."""
    try:
        stages._init(rank, world, port)
        from streamdiffusionv2_b200.pipeline_runner import PipelineStageRunner
        from streamdiffusionv2_b200.stage_transport import StageLink
        _fakes(stages._Patch())
        case = cases.MODEL_CASES["m_stages"]
        fs, sched = cases.model_schedule(case)
        pipe, first, chunks = _pipeline(case)
        outs = []
        with torch.no_grad():
            torch.manual_seed(case["seed"] + 1)
            pipe.prepare(text_prompts=["p"], device=torch.device("cpu"), dtype=torch.bfloat16, noise=first + rank, current_start=0,
                         current_end=fs * (1 + case["frames"]), block_mode="input" if rank == 0 else "output",
                         owned_blocks=range(*ranges[rank]), unowned=unowned)
            prepared = _held(pipe)
            shapes = {i: [tuple(kv[n].shape) for n in NAMES] for i, kv in enumerate(pipe.kv_cache1)}
            torch.manual_seed(case["seed"] + 2)
            link = StageLink(rank, world, torch.device("cpu"), (len(case["levels"]), fs * case["frames"], cases.MODEL_KW["dim"]),
                             tuple(pipe.hidden_states.shape), dtype=torch.bfloat16, timeout_s=60)
            runner = PipelineStageRunner(pipe, link, rank, world, ranges)
            for i, (noise, (cs, ce)) in enumerate(zip(chunks, sched)):
                if i == 4 and new_ranges is not None:
                    runner.rebalance(new_ranges)
                o = runner.step(i, noise, cs, ce, None, last=(i == 3))
                if o is not None:
                    outs.append(o.float().numpy().copy())
                if i == 3:
                    runner.quiesce()
            runner.finish()
            own = range(*runner.block_range)
            ends = {i: (pipe.kv_cache1[i]["global_end_index"].tolist(), pipe.kv_cache1[i]["local_end_index"].tolist(),
                        pipe.generator.model.blocks[i].self_attn.evict_idx) for i in own}
            q.put((rank, "ok", outs, (prepared, shapes, {i: h for i, h in _held(pipe).items() if i in own}, ends)))
    except Exception:
        q.put((rank, "error", traceback.format_exc(), None))
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


def _run(*args):
    res = stages._run(_worker, 2, *args)
    for r, v in res.items():
        assert v[0] == "ok", v[1]
    return res


def _same(a, b):
    assert a.keys() == b.keys()
    for n in NAMES:
        assert a[n].dtype == b[n].dtype and a[n].shape == b[n].shape and (a[n] == b[n]).all(), n


@pytest.fixture(scope="module")
def unmoved():
    return {unowned: _run([[0, 2], [2, 3]], None, unowned) for unowned in ("cpu", "free")}


def test_prepare_shares_the_four_tensors_and_keeps_or_releases_what_a_rank_does_not_own(unmoved):
    """Rank 0's cache arrives on rank 1, which had another; one row per level; "free" leaves no tokens of blocks owned
    elsewhere, "cpu" all of them."""
    tokens = cases.MODEL_CASES["m_stages"]["cache_frames"] * 6
    for unowned, res in unmoved.items():
        for rank, own in ((0, {0, 1}), (1, {2})):
            prepared, shapes = res[rank][2][0], res[rank][2][1]
            for i, four in shapes.items():
                t = tokens if unowned == "cpu" or i in own else 0
                assert four == [(2, t, 2, 128)] * 2 + [(2, t, 2)] * 2, (unowned, rank, i)
            assert set(prepared) == (own if unowned == "free" else {0, 1, 2})
    both = [unmoved["cpu"][r][2][0] for r in (0, 1)]
    for i in range(3):
        _same(both[0][i], both[1][i])
        assert all((both[0][i][n][0] == both[0][i][n][1]).all() for n in NAMES)
        distinct = [both[0][i][n][:, :12].tobytes() for n in NAMES]      # the first chunk's two frames
        assert len(set(distinct)) == 4
    for r, own in ((0, (0, 1)), (1, (2,))):
        for i in own:
            _same(unmoved["free"][r][2][0][i], both[r][i])


@pytest.mark.parametrize("unowned", ["cpu", "free"])
@pytest.mark.parametrize("a,b", [([[0, 2], [2, 3]], [[0, 1], [1, 3]]), ([[0, 1], [1, 3]], [[0, 2], [2, 3]])])
def test_a_moved_block_takes_its_four_tensors_along(unmoved, a, b, unowned):
    """Outputs, caches, index tensors and queues are those of a stream whose blocks stay where they are, bit for bit."""
    res, want = _run(a, b, unowned), unmoved[unowned]
    assert len(res[1][1]) == len(want[1][1]) == cases.MODEL_CASES["m_stages"]["chunks"]
    for x, y in zip(res[1][1], want[1][1]):
        assert (x == y).all()
    held = {**want[0][2][2], **want[1][2][2]}
    ends = {**want[0][2][3], **want[1][2][3]}
    for r in (0, 1):
        assert set(res[r][2][2]) == set(range(*b[r]))
        for i in range(*b[r]):
            _same(res[r][2][2][i], held[i])
            assert res[r][2][3][i] == ends[i]
