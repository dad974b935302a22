"""The engine with its cache in 8 bits: every call that a step makes of the cache's kernels against plain operations in 64
bits on what the call was given, in the steps that the engine forms itself, and what a user sees of it."""
import numpy as np
import pytest
import torch

import q8_plain as plain
from helpers import make_weights, plain_logits, prompts_for, write_model_dir

pytestmark = pytest.mark.gpu

CFG = {"architectures": ["LlamaForCausalLM"], "model_type": "llama", "num_hidden_layers": 2, "hidden_size": 128,
       "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 192, "vocab_size": 300,
       "rope_theta": 10000.0, "rms_norm_eps": 1e-5, "max_position_embeddings": 256, "tie_word_embeddings": False}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from plain import llama_plain
    out = {}
    for dtype in ("float32", "bfloat16"):
        d = str(tmp_path_factory.mktemp("q8" + dtype))
        w = llama_plain.random_weights(CFG, 3, gain_std=0.05, std=0.05)
        for k in list(w):
            if k.endswith("q_proj.weight") or k.endswith("k_proj.weight"):
                w[k] = (w[k] * 2.0).astype(np.float32)
        out[dtype] = (write_model_dir(d, CFG, w, bf16=dtype == "bfloat16"), w)
    return out


def engine(folder, dtype, **kw):
    from kllm_b200 import Engine, Options
    kw = dict(dict(max_seq=256, block_size=16, num_blocks=48, max_batch=6, max_step_tokens=96, cache_dtype="float8_e4m3fn"), **kw)
    return Engine(folder, Options(dtype=dtype, **kw))


class Watch:
    """Stands between the parts and the faces of the kernels and holds every call against the plain operations."""

    def __init__(self, monkeypatch):
        from kllm_b200 import kernels
        self.calls = {"append": 0, "decode": 0, "prefill": 0}
        self.append, self.decode, self.prefill = kernels.rope_append_q8, kernels.attention_decode_q8, kernels.attention_prefill_q8
        monkeypatch.setattr(kernels, "rope_append_q8", self.on_append)
        monkeypatch.setattr(kernels, "attention_decode_q8", self.on_decode)
        monkeypatch.setattr(kernels, "attention_prefill_q8", self.on_prefill)

    def on_append(self, q_out, q, k, v, cos_sin, positions, token_req, q_start, table, kc, vc, ks, vs, H, G, hd):
        self.calls["append"] += 1
        n, rows = q.shape[0], q_start.tolist()
        lens = [b - a for a, b in zip(rows, rows[1:])]
        starts = [int(positions[a]) for a in rows[:-1]]
        kr, vr = plain.turned(k, cos_sin, positions, G, hd), v.cpu().double().view(n, G, hd)
        before = [t.clone() for t in (kc, ks, vc, vs)]
        self.append(q_out, q, k, v, cos_sin, positions, token_req, q_start, table, kc, vc, ks, vs, H, G, hd)
        for key, (store, scale), (s0, c0) in ((True, (kc, ks), before[:2]), (False, (vc, vs), before[2:])):
            want, sc, _ = plain.append(s0, c0, kr, vr, key, table.tolist(), starts, lens)
            assert torch.equal(scale.cpu().double(), sc)
            differ = store.cpu().float().double() != want
            assert int(differ.sum()) <= (2 if key else 0)       # a rotated key beside a border of e4m3

    def _check(self, out, q, kc, vc, ks, vs, table, starts, lens, H, G, hd, window, scale):
        want, err = plain.attention(q, kc, vc, ks, vs, table.tolist(), starts, lens, H, G, hd, window, scale)
        assert bool(((out.cpu().double() - want).abs() <= err).all())

    def on_decode(self, out, q, kc, vc, ks, vs, positions, token_req, table, H, G, hd, window, scale, bound):
        self.calls["decode"] += 1
        self.decode(out, q, kc, vc, ks, vs, positions, token_req, table, H, G, hd, window, scale, bound)
        n = q.shape[0]
        req = list(range(n)) if token_req is None else token_req.tolist()
        assert int(positions.max()) < bound
        self._check(out, q, kc, vc, ks, vs, table[req], positions.tolist(), [1] * n, H, G, hd, window, scale)

    def on_prefill(self, out, q, kc, vc, ks, vs, q_start, start_pos, table, R, H, G, hd, window, scale, bound):
        self.calls["prefill"] += 1
        before = out.clone()
        self.prefill(out, q, kc, vc, ks, vs, q_start, start_pos, table, R, H, G, hd, window, scale, bound)
        rows = q_start.tolist()[:R + 1]
        lens = [b - a for a, b in zip(rows, rows[1:])]
        at = slice(rows[0], rows[-1])
        assert torch.equal(out[:rows[0]], before[:rows[0]])
        self._check(out[at], q[at], kc, vc, ks, vs, table, start_pos.tolist()[:R], lens, H, G, hd, window, scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_every_call_of_a_run(folders, dtype, monkeypatch):
    """Prompts cut by the step's budget beside tokens of other requests, more requests than slots, pages used again."""
    from kllm_b200 import Scheduler
    eng = engine(folders[dtype][0], dtype, cuda_graphs=False, num_blocks=26, max_batch=3, max_step_tokens=40)
    watch = Watch(monkeypatch)
    sched = Scheduler(eng)
    reqs = [sched.submit(p, 6) for p in prompts_for(CFG, [33, 7, 90, 16, 1], seed=2)]
    sched.run()
    assert all(r.error is None and len(r.generated) == 6 for r in reqs)
    assert min(watch.calls.values()) >= 2 and watch.calls["append"] >= 20
    eng.cache.audit()
    eng.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replayed_steps_are_the_eager_ones(folders, dtype):
    outs = []
    for graphs in (True, False):
        eng = engine(folders[dtype][0], dtype, cuda_graphs=graphs)
        outs.append(eng.generate(prompts_for(CFG, [20, 65, 3], seed=4), max_new_tokens=30))
        eng.close()
    assert outs[0] == outs[1]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_stay_near_those_of_the_wide_cache(folders, dtype):
    """Keys and values are off by at most 2^-4 of themselves; what that does to the logits of two layers is below a tenth of the
    largest, and well above the wide cache's own error."""
    folder, w = folders[dtype]
    ids = prompts_for(CFG, [120], seed=7)[0]
    want = plain_logits(w, CFG, ids, dtype)
    eng = engine(folder, dtype, max_step_tokens=128)
    from kllm_b200 import StepEntry
    r = eng.cache.open()
    parts, at = [], 0
    for n in (50, 1, 30, 39):
        parts.append(eng.step([StepEntry(r, ids[at:at + n], list(range(n)))]).cpu().numpy())
        at += n
    got = np.concatenate(parts)
    err = np.abs(got - want).max() / np.abs(want).max()
    assert 1e-4 < err < 0.1
    eng.close()


def test_half_the_bytes_and_the_command_line(folders, capsys):
    from kllm_b200 import cli
    folder = folders["bfloat16"][0]
    wide, narrow = engine(folder, "bfloat16", cache_dtype="", num_blocks=0, cache_bytes=10 ** 7), \
        engine(folder, "bfloat16", num_blocks=0, cache_bytes=10 ** 7)
    assert 1.9 < narrow.cache.num_pages / wide.cache.num_pages <= 2.0
    want = narrow.generate([1, 17, 42, 100, 7], max_new_tokens=5)
    wide.close(), narrow.close()
    assert cli.main(["--model", folder, "--ids", "1 17 42 100 7", "--steps", "5", "--cache-dtype", "float8_e4m3fn"]) == 0
    assert "generated: [" + " ".join(map(str, want)) + "]" in capsys.readouterr().out


def test_architectures_without_it_say_so(tmp_path):
    from helpers import TINY
    from kllm_b200 import Engine, Options
    cfg, w = make_weights("A")
    assert TINY["A"][0]["head_dim"] == 16
    d = write_model_dir(str(tmp_path), cfg, w)
    with pytest.raises(ValueError, match="does not take a cache in 8 bits"):
        Engine(d, Options(cache_dtype="float8_e4m3fn"))
