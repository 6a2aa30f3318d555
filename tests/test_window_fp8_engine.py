"""Windowed models and the 8-bit KV cache in the model and the rollout engine (CPU paths; the GPU ones at the end)."""

from dataclasses import replace

import pytest
import torch

from psrl_b200.models import PRESETS, build_model, packed_positions
from psrl_b200.rollout import EngineWeights, GenRequest, RolloutEngine, SamplingParams


def _logits(m, toks, dev="cpu"):
    pos, cu, mx = packed_positions([len(toks)], dev)
    with torch.no_grad():
        return m.logits(torch.tensor(toks, device=dev), pos, cu, mx)


def _generate(eng, prompts, n=12, temperature=0.0):
    for i, p in enumerate(prompts):
        eng.add_request(GenRequest(i, list(p), SamplingParams(temperature=temperature, max_tokens=n, ignore_eos=True,
                                                              seed=i)))
    outs = {}
    while eng.has_unfinished():
        for o in eng.step():
            outs[o.request_id] = o
    return [outs[i] for i in range(len(prompts))]


def _prompts(a, lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(3, a.vocab_size, (n,), generator=g).tolist() for n in lens]


def _agreement(m, eng, prompts, n=12, dev="cpu"):
    """Share of greedy tokens that are the model's argmax, and how far log-probs of sampled tokens (temperature 1;
    a greedy token's is reported as 0) are from the model's."""
    hit = total = 0
    worst = 0.0
    for p, o in zip(prompts, _generate(eng, prompts, n)):
        lp = _logits(m, (list(p) + o.output_ids)[:-1], dev)[len(p) - 1:]
        hit += int((lp.argmax(-1).cpu() == torch.tensor(o.output_ids)).sum())
        total += len(o.output_ids)
    for p, o in zip(prompts, _generate(eng, prompts, n, temperature=1.0)):
        toks = list(p) + o.output_ids
        lp = _logits(m, toks[:-1], dev).float().log_softmax(-1)[len(p) - 1:]
        own = lp.gather(-1, torch.tensor(o.output_ids, device=dev)[:, None])[:, 0].cpu()
        worst = max(worst, float((own - torch.tensor(o.logprobs)).abs().max()))
    return hit / total, worst


# ------------------------------------------------------------------ families
@pytest.mark.parametrize("name", ["mistral", "qwen2"])
def test_windowed_family_matches_hf(tmp_path, name):
    transformers = pytest.importorskip("transformers")
    import json

    from psrl_b200.models.config import ModelArgs
    from psrl_b200.models.families import hf_config_from_args
    from psrl_b200.models.hf_io import load_hf_into
    small = dict(vocab_size=160, hidden_size=64, intermediate_size=96, num_hidden_layers=3, num_attention_heads=4,
                 num_key_value_heads=2, max_position_embeddings=512)
    cfg = (transformers.MistralConfig(**small, head_dim=16, sliding_window=8) if name == "mistral" else
           transformers.Qwen2Config(**small, use_sliding_window=True, sliding_window=8, max_window_layers=1))
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    hf = transformers.AutoModelForCausalLM.from_config(cfg).float().eval()
    hf.save_pretrained(tmp_path)
    with open(tmp_path / "config.json") as fh:
        a = ModelArgs.from_hf_config(json.load(fh))
    assert a.sliding_window == 8 and a.window_from_layer == (0 if name == "mistral" else 1)
    assert ModelArgs.from_hf_config(hf_config_from_args(a)).window_from_layer == a.window_from_layer
    m = build_model(a, "cpu", torch.float32)
    load_hf_into(m, str(tmp_path))
    ids = torch.randint(3, 160, (1, 40))
    with torch.no_grad():
        want = hf(ids).logits[0]
    assert torch.allclose(_logits(m, ids[0].tolist()), want, atol=1e-4, rtol=1e-4)
    full = build_model(replace(a, sliding_window=None), "cpu", torch.float32)
    load_hf_into(full, str(tmp_path))
    assert not torch.allclose(_logits(full, ids[0].tolist()), want, atol=1e-3)       # the window matters here


def test_mixed_layer_kinds_are_refused():
    from psrl_b200.models.config import ModelArgs
    cfg = dict(model_type="qwen2", vocab_size=64, hidden_size=64, num_hidden_layers=2, num_attention_heads=4,
               num_key_value_heads=2, intermediate_size=96, use_sliding_window=True, sliding_window=8,
               max_position_embeddings=64, rms_norm_eps=1e-6, layer_types=["sliding_attention", "full_attention"])
    with pytest.raises(NotImplementedError, match="full attention above"):
        ModelArgs.from_hf_config(cfg)


# -------------------------------------------------------------------- engine
@pytest.mark.parametrize("window,sinks,first", [(9, 0, 0), (9, 2, 1), (16, 4, 0)])
def test_windowed_engine_matches_model(window, sinks, first):
    a = replace(PRESETS["tiny"], sliding_window=window, attention_sinks=sinks, window_from_layer=first)
    m = build_model(a, "cpu", torch.float32, seed=1)
    eng = RolloutEngine(a, EngineWeights.from_model(m, dtype=torch.float32), max_num_seqs=4, max_model_len=128,
                        block_size=16, num_blocks=40, max_num_batched_tokens=20)
    prompts = _prompts(a, (5, 40, 17))
    share, worst = _agreement(m, eng, prompts)
    assert share == 1.0 and worst < 1e-3


def test_fp8_engine_cpu():
    a = PRESETS["tiny"]
    m = build_model(a, "cpu", torch.float32, seed=1)
    make = lambda kind, **k: RolloutEngine(a, EngineWeights.from_model(m, dtype=torch.float32), max_num_seqs=4,  # noqa: E731
                                           max_model_len=128, block_size=16, max_num_batched_tokens=20,
                                           kv_cache_dtype=kind, **k)
    eng = make("fp8", num_blocks=40)
    prompts = _prompts(a, (5, 40, 17))
    _, worst = _agreement(m, eng, prompts)
    # keys and values off by at most 2^-4 of themselves: small next to the entropy of a random model's tokens
    assert worst < 0.1
    assert make("fp8", kv_cache_gb=0.01).num_blocks > 3 * make("auto", kv_cache_gb=0.01).num_blocks    # fp32 weights here
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        make("int4")


def test_fp8_migration_and_offload_cpu():
    a = PRESETS["tiny"]
    m = build_model(a, "cpu", torch.float32, seed=1)
    make = lambda kind, **k: RolloutEngine(a, EngineWeights.from_model(m, dtype=torch.float32), max_num_seqs=4,  # noqa: E731
                                           max_model_len=128, block_size=16, kv_cache_dtype=kind, **k)
    prompt = _prompts(a, (40,))
    whole = _generate(make("fp8", num_blocks=40), prompt)[0]
    for dst_kind in ("fp8", "auto"):
        src, dst = make("fp8", num_blocks=40), make(dst_kind, num_blocks=40)
        src.add_request(GenRequest(0, list(prompt[0]), SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)))
        for _ in range(5):
            src.step()
        blocks = list(src.by_id[0].blocks)
        n = src.by_id[0].num_computed
        assert src.migrate_request(0, dst)
        new = dst.by_id[0].blocks
        for l in range(a.num_layers):
            if dst_kind == "fp8":
                for s, d in zip((src.k_scale, src.v_scale), (dst.k_scale, dst.v_scale)):
                    assert torch.equal(s[l][blocks[0]], d[l][new[0]])
            else:
                from psrl_b200.ops import read_kv_cache
                for c, e, d in ((src.k_cache, src.k_scale, dst.k_cache), (src.v_cache, src.v_scale, dst.v_cache)):
                    want = read_kv_cache(c[l], e[l], torch.tensor(blocks[:-(-n // 16)]))
                    assert torch.equal(d[l][torch.tensor(new[: want.shape[0]])].float(), want.float())
        outs = []
        while dst.has_unfinished():
            outs += dst.step()
        if dst_kind == "fp8":
            assert outs[0].output_ids == whole.output_ids
        else:
            assert len(outs[0].output_ids) == 12
    src, dst = make("auto", num_blocks=40), make("fp8", num_blocks=40)
    src.add_request(GenRequest(0, list(prompt[0]), SamplingParams(max_tokens=4)))
    src.step()
    assert not src.migrate_request(0, dst) and 0 in src.by_id                        # refused, request kept
    # a cache too small for two requests: preempted blocks go to the host and come back
    eng = make("fp8", num_blocks=7, kv_offload_blocks=16, enable_prefix_caching=False)
    two = _prompts(a, (40, 40), seed=3)
    got = _generate(eng, two, n=30)
    ref = _generate(make("fp8", num_blocks=40), two, n=30)
    assert eng.stats["offloaded_blocks"] > 0 and eng.stats["onloaded_blocks"] > 0
    assert [o.output_ids for o in got] == [o.output_ids for o in ref]


# ----------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["auto", "fp8"])
@pytest.mark.parametrize("how", [dict(), dict(sliding_window=100, attention_sinks=4)])
@pytest.mark.parametrize("graph", [True, False])
def test_engine_gpu(kind, how, graph):
    dev = torch.device("cuda", 0)
    a = replace(PRESETS["tiny128"], **how)
    m = build_model(a, dev, torch.bfloat16, seed=1)
    eng = RolloutEngine(a, EngineWeights.from_model(m), max_num_seqs=8, max_model_len=1024, block_size=64,
                        max_num_batched_tokens=300, num_blocks=96, use_cuda_graph=graph, kv_cache_dtype=kind)
    prompts = _prompts(a, (5, 70, 330, 9, 500))
    share, worst = _agreement(m, eng, prompts, 20, dev)
    # bf16 paths differ slightly; with an 8-bit cache near-ties flip more often
    assert share > (0.9 if kind == "auto" else 0.7) and worst < (0.1 if kind == "auto" else 0.3), (share, worst)
    from psrl_b200.ops.gemm import check_errors
    check_errors()


@pytest.mark.gpu
def test_train_step_of_a_windowed_model_gpu():
    """Log-probs and gradients of the windowed decoder on the GPU against the fp32 CPU model."""
    a = replace(PRESETS["tiny128"], sliding_window=50, attention_sinks=3)
    cpu = build_model(a, "cpu", torch.float32, seed=2)
    gpu = build_model(a, torch.device("cuda", 0), torch.bfloat16, seed=2)
    with torch.no_grad():
        for p, q in zip(cpu.parameters(), gpu.parameters()):
            p.copy_(q.float().cpu())
    lens = [130, 7, 300]
    g = torch.Generator().manual_seed(0)
    ids, labels = (torch.randint(3, a.vocab_size, (sum(lens),), generator=g) for _ in range(2))
    res = []
    for m, dev in ((cpu, "cpu"), (gpu, "cuda")):
        pos, cu, mx = packed_positions(lens, dev)
        lp, _ = m.logprobs(ids.to(dev), pos, cu, mx, labels.to(dev))
        (-lp.mean()).backward()
        res.append((lp.detach().float().cpu(), [p.grad.float().cpu() for p in m.parameters()]))
    assert (res[0][0] - res[1][0]).abs().max() < 0.05
    for (n, _), x, y in zip(cpu.named_parameters(), res[0][1], res[1][1]):
        assert (x - y).norm() <= 0.05 * x.norm() + 1e-6, n


@pytest.mark.gpu
def test_fp8_migration_gpu():
    dev = torch.device("cuda", 0)
    a = PRESETS["tiny128"]
    m = build_model(a, dev, torch.bfloat16, seed=1)
    make = lambda kind: RolloutEngine(a, EngineWeights.from_model(m), max_num_seqs=4, max_model_len=512,  # noqa: E731
                                      block_size=64, num_blocks=32, kv_cache_dtype=kind)
    prompt = _prompts(a, (150,))
    whole = _generate(make("fp8"), prompt)[0]
    for kind in ("fp8", "auto"):
        src, dst = make("fp8"), make(kind)
        src.add_request(GenRequest(0, list(prompt[0]), SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)))
        for _ in range(5):
            src.step()
        assert src.migrate_request(0, dst)
        outs = []
        while dst.has_unfinished():
            outs += dst.step()
        assert len(outs[0].output_ids) == 12
        if kind == "fp8":
            # the tokens decoded before the move are recomputed by nobody: the continuation is the unmoved run's
            assert outs[0].output_ids == whole.output_ids


@pytest.mark.gpu
def test_fp8_engine_refusals_gpu():
    dev = torch.device("cuda", 0)
    a = PRESETS["tiny128"]
    w = EngineWeights.from_model(build_model(a, dev, torch.bfloat16, seed=1))
    with pytest.raises(ValueError, match="power of two"):
        RolloutEngine(a, w, max_model_len=256, block_size=24, num_blocks=16, kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="65536"):
        RolloutEngine(a, w, max_model_len=70000, block_size=64, num_blocks=2200, kv_cache_dtype="fp8")
