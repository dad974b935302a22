"""The engine with its cache in 8 bits where its layers are not plain Llama's: a window whose pages are given back, a cache that another layer
reads, a layer without positions.  Every call of the cache's kernels is held against plain operations, what is stored to the bit."""
import pytest
import torch

import q8_plain as plain
from helpers import prompts_for
from test_gpu_q8_engine import Watch

pytestmark = pytest.mark.gpu

CFG = {"architectures": ["LlamaForCausalLM"], "model_type": "llama", "num_hidden_layers": 4, "hidden_size": 128,
       "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 192, "vocab_size": 300,
       "rope_theta": 10000.0, "rms_norm_eps": 1e-5, "max_position_embeddings": 256, "tie_word_embeddings": False}


class ExactWatch(Watch):
    """... and equality of every number that is stored, keys too."""

    def on_append(self, q_out, q, k, v, cos_sin, positions, token_req, q_start, table, kc, vc, ks, vs, H, G, hd):
        n, rows = q.shape[0], q_start.tolist()
        lens = [b - a for a, b in zip(rows, rows[1:])]
        starts = [int(positions[a]) for a in rows[:-1]]
        kr, vr, before = plain.turned(k, cos_sin, positions, G, hd), v.cpu().double().view(n, G, hd), (kc.clone(), ks.clone())
        super().on_append(q_out, q, k, v, cos_sin, positions, token_req, q_start, table, kc, vc, ks, vs, H, G, hd)
        want, _, _ = plain.append(*before, kr, vr, True, table.tolist(), starts, lens)
        assert torch.equal(kc.cpu().float().double(), want)


def with_layers(monkeypatch):
    """Layer 0 without positions, layer 1 reading its cache (and turning its queries), layer 2 with a window, layer 3 as it is."""
    from kllm_b200.engine import engine
    from kllm_b200.parts.spec import LayerCall
    build = engine.build_model_spec

    def changed(cfg):
        spec = build(cfg)
        spec.blocks[0].mixer.params["position"] = None
        spec.blocks[2].mixer.params["window"] = 24
        spec.schedule = [LayerCall(0, 0), LayerCall(1, 0, writes_cache=False), LayerCall(2, 1), LayerCall(3, 2)]
        return spec
    monkeypatch.setattr(engine, "build_model_spec", changed)


def engine(dtype, **kw):
    from kllm_b200 import Engine, Options
    kw = dict(dict(max_seq=256, block_size=16, num_blocks=48, max_batch=3, max_step_tokens=40, cache_dtype="float8_e4m3fn"), **kw)
    return Engine(None, Options(dtype=dtype, **kw), config=CFG, random_seed=3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("block", [16, 5])
def test_every_call_of_a_run(dtype, block, monkeypatch):
    from kllm_b200 import Scheduler
    with_layers(monkeypatch)
    eng = engine(dtype, cuda_graphs=False, block_size=block, num_blocks=26 * 16 // block)
    assert [g.need.window for g in eng.cache.groups] == [None, 24] and len(eng.model.cache_needs()) == 3
    watch = ExactWatch(monkeypatch)
    sched = Scheduler(eng)
    reqs = [sched.submit(p, 6) for p in prompts_for(CFG, [33, 7, 90, 16, 1], seed=2)]
    sched.run()
    assert all(r.error is None and len(r.generated) == 6 for r in reqs)
    assert min(watch.calls.values()) >= 2 and watch.calls["decode"] + watch.calls["prefill"] > watch.calls["append"]
    eng.cache.audit()
    eng.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replayed_steps_are_the_eager_ones(dtype, monkeypatch):
    with_layers(monkeypatch)
    outs = []
    for graphs in (True, False):
        eng = engine(dtype, cuda_graphs=graphs)
        outs.append(eng.generate(prompts_for(CFG, [20, 65, 3], seed=4), max_new_tokens=60))
        eng.close()
    assert outs[0] == outs[1]
