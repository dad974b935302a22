"""What the faces of the cache in 8 bits refuse, and how contexts are cut: no GPU needed."""
import pytest
import torch

from kllm_b200 import kernels
from kllm_b200.kernels import KernelError

H, G, HD, PS, R, N = 8, 2, 64, 16, 3, 5


def operands():
    f8 = lambda *s: torch.zeros(*s, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros(N, H * HD), out=torch.zeros(N, H * HD), k=torch.zeros(N, G * HD), v=torch.zeros(N, G * HD),
                cos_sin=torch.zeros(40, HD), positions=i(0, 1, 2, 3, 4), token_req=i(0, 0, 1, 2, 2), q_start=i(0, 2, 3, 5),
                start_pos=i(0, 2, 3), table=torch.zeros(R, 3, dtype=torch.int32), kcache=f8(7, G, PS, HD),
                vcache=f8(7, G, PS, HD), kscale=torch.ones(7, G), vscale=torch.ones(7, G), n_heads=H, n_kv=G, head_dim=HD)


def append(o):
    kernels.rope_append_q8(o["out"], o["q"], o["k"], o["v"], o["cos_sin"], o["positions"], o["token_req"], o["q_start"], o["table"],
                           o["kcache"], o["vcache"], o["kscale"], o["vscale"], o["n_heads"], o["n_kv"], o["head_dim"])


def decode(o):
    kernels.attention_decode_q8(o["out"], o["q"], o["kcache"], o["vcache"], o["kscale"], o["vscale"], o["positions"], o["token_req"],
                                o["table"], o["n_heads"], o["n_kv"], o["head_dim"], 0, 0.125, 40)


def prefill(o):
    kernels.attention_prefill_q8(o["out"], o["q"], o["kcache"], o["vcache"], o["kscale"], o["vscale"], o["q_start"], o["start_pos"],
                                 o["table"], R, o["n_heads"], o["n_kv"], o["head_dim"], 0, 0.125, 40)


CALLS = {"append": append, "decode": decode, "prefill": prefill}


@pytest.mark.parametrize("call", CALLS)
def test_a_sound_call_gets_as_far_as_the_device(call):
    with pytest.raises(KernelError, match="not on a CUDA device"):
        CALLS[call](operands())


def strided(t, dim=-1):
    return torch.cat([t, t], dim=dim).narrow(dim, 0, t.shape[dim]) if dim != -1 else torch.stack([t, t], dim=-1)[..., 0]


BAD = {
    "key store of another type": lambda o: o.update(kcache=o["kcache"].to(torch.bfloat16)),
    "value store of bytes": lambda o: o.update(vcache=o["vcache"].view(torch.uint8)),
    "stores of two shapes": lambda o: o.update(vcache=o["vcache"][:6]),
    "another head count": lambda o: o.update(n_kv=4),
    "heads no multiple of kv heads": lambda o: o.update(n_heads=7),
    "no kv heads": lambda o: o.update(n_kv=0),
    "another head size": lambda o: o.update(head_dim=32),
    "scales in bfloat16": lambda o: o.update(kscale=o["kscale"].bfloat16()),
    "scales per page": lambda o: o.update(vscale=o["vscale"][:, :1].contiguous()),
    "strided scales": lambda o: o.update(vscale=strided(o["vscale"])),
    "strided store": lambda o: o.update(kcache=torch.cat([o["kcache"].view(torch.uint8)] * 2, dim=1)[:, :G].view(torch.float8_e4m3fn)),
    "table of 64-bit entries": lambda o: o.update(table=o["table"].long()),
    "flat table": lambda o: o.update(table=o["table"].view(-1)),
    "positions of 64 bits": lambda o: o.update(positions=o["positions"].long(), start_pos=o["start_pos"].long()),
    "float16 queries": lambda o: o.update({k: o[k].half() for k in ("q", "out", "k", "v")}),
    "out of another type": lambda o: o.update(out=o["out"].bfloat16()),
    "out of another shape": lambda o: o.update(out=o["out"][:, :-1]),
    "queries of another width": lambda o: o.update(q=torch.zeros(N, H * HD + 4)),
    "queries without dense rows": lambda o: o.update(q=strided(o["q"])),
}


@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("call", CALLS)
def test_refused(call, what):
    o = operands()
    BAD[what](o)
    with pytest.raises(KernelError) as e:
        CALLS[call](o)
    assert "CUDA device" not in str(e.value)          # looked at before the device is


@pytest.mark.parametrize("what,change", [
    ("k of another type", lambda o: o.update(k=o["k"].bfloat16())),
    ("v of another width", lambda o: o.update(v=o["v"][:, :HD])),
    ("k without dense rows", lambda o: o.update(k=strided(o["k"]))),
    ("angles in 64 bits", lambda o: o.update(cos_sin=o["cos_sin"].double())),
    ("an odd rotary width", lambda o: o.update(cos_sin=torch.zeros(40, 33))),
    ("a rotary width beyond the head", lambda o: o.update(cos_sin=torch.zeros(40, 2 * HD))),
    ("too few positions", lambda o: o.update(positions=o["positions"][:4])),
    ("no table row for a request", lambda o: o.update(table=o["table"][:2])),
    ("several tokens of a request without token_req", lambda o: o.update(token_req=None)),
    ("pages of 4097 tokens", lambda o: o.update({k: torch.zeros(2, G, 4097, HD, dtype=torch.uint8).view(torch.float8_e4m3fn)
                                                 for k in ("kcache", "vcache")} | dict(kscale=torch.ones(2, G), vscale=torch.ones(2, G)))),
])
def test_append_refuses(what, change):
    o = operands()
    change(o)
    with pytest.raises(KernelError) as e:
        append(o)
    assert "CUDA device" not in str(e.value)


def test_attention_refuses_missing_rows():
    o = operands()
    o.update(token_req=None)                       # five rows, three requests
    with pytest.raises(KernelError, match="per token"):
        decode(o)
    o = operands()
    o.update(q_start=o["q_start"][:3])
    with pytest.raises(KernelError, match="cover the requests"):
        prefill(o)


@pytest.mark.parametrize("tokens", [1, 2, 7, 64, 500])
@pytest.mark.parametrize("n_kv,group,hd", [(4, 8, 64), (8, 4, 128), (32, 1, 128), (1, 32, 128), (1, 1, 256), (8, 12, 256)])
@pytest.mark.parametrize("ctx", [1, 127, 128, 129, 2048, 131072, 2 ** 31 - 1])
def test_parts_of_a_context(tokens, n_kv, group, hd, ctx, monkeypatch):
    monkeypatch.setattr(kernels, "sm_count", lambda: 148)
    ranges, cluster = kernels.decode_q8_parts(tokens, n_kv, group, hd, ctx)
    assert cluster in (1, 2, 4, 8) and ranges >= 1
    assert ranges == 1 or cluster == 8
    blocks = -(-ctx // 128)
    assert ranges * cluster <= max(1, blocks), "a part for every 128 keys at most"


@pytest.mark.parametrize("tokens,requests", [(1, 1), (9, 9), (300, 1), (2048, 1), (700, 12), (100000, 3)])
@pytest.mark.parametrize("n_kv,group,hd", [(4, 8, 64), (8, 4, 128), (32, 1, 128), (1, 128, 64)])
@pytest.mark.parametrize("ctx", [0, 1, 128, 257, 8192, 2 ** 31 - 1])
def test_parts_of_portions(tokens, requests, n_kv, group, hd, ctx, monkeypatch):
    monkeypatch.setattr(kernels, "sm_count", lambda: 148)
    row_tiles, splits = kernels.prefill_q8_parts(tokens, requests, n_kv, group, max(ctx, tokens // requests), hd)
    assert row_tiles in (1, 2) and 1 <= splits <= 16
    assert splits == 1 or splits * 2 * 128 <= max(ctx, tokens) + 128, "two tiles of keys a part at least"


# ---- the manager and the options -----------------------------------------------------------------------------------------

def test_manager_keeps_pages_in_eight_bits():
    from kllm_b200.cache.manager import CacheManager
    from kllm_b200.parts.spec import PagedKVNeed
    full, near = PagedKVNeed(2, 64, eight_bits=True), PagedKVNeed(2, 64, window=32, eight_bits=True)
    m = CacheManager([full, near, full], 16, 5, max_requests=2, dtype=torch.bfloat16, cache_dtype=torch.float8_e4m3fn)
    tables = {g.index: torch.zeros(1, 1, dtype=torch.int32) for g in m.groups}
    for c in m.layer_caches(tables):
        assert c.k.dtype == c.v.dtype == torch.float8_e4m3fn and c.k.shape == (5, 2, 16, 64) and c.k.is_contiguous()
        assert c.k_scale.shape == c.v_scale.shape == (5, 2) and c.k_scale.dtype == torch.float32 and c.k_scale.is_contiguous()
    assert m.layer_caches(tables)[0].k_scale.data_ptr() != m.layer_caches(tables)[2].k_scale.data_ptr()
    assert m.bytes_per_page() == 3 * (16 * 2 * 2 * 64 + 2 * 2 * 4)
    assert m.bytes_per_token_full() == -(-2 * (16 * 2 * 2 * 64 + 2 * 2 * 4) // 16)
    wide = CacheManager([full, near, full], 16, 5, max_requests=2, dtype=torch.bfloat16)
    assert all(c.k_scale is None and c.k.dtype == torch.bfloat16 for c in wide.layer_caches(tables))
    assert wide.bytes_per_page() == 3 * 16 * 2 * 2 * 64 * 2 and wide.bytes_per_token_full() == 2 * 2 * 2 * 64 * 2
    budget = 100 * m.bytes_per_page()
    assert CacheManager.pages_within([full, near, full], 16, torch.bfloat16, budget, torch.float8_e4m3fn) == 100
    assert CacheManager.pages_within([full, near, full], 16, torch.bfloat16, budget) == 50


def test_manager_refuses_layers_that_cannot():
    from kllm_b200.cache.manager import CacheManager
    from kllm_b200.parts.spec import PagedKVNeed
    with pytest.raises(ValueError, match="does not take a cache in 8 bits"):
        CacheManager([PagedKVNeed(2, 64, eight_bits=True), PagedKVNeed(2, 64)], 16, 5, max_requests=2,
                     cache_dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="model's dtype"):
        CacheManager([PagedKVNeed(2, 64, eight_bits=True)], 16, 5, max_requests=2, dtype=torch.float32, cache_dtype=torch.bfloat16)


def test_which_layers_take_it():
    from kllm_b200.config.base import build_model_spec, parse_config
    from kllm_b200 import models  # noqa: F401
    from kllm_b200.parts.model import DecoderModel

    def needs(head_dim, **params):
        cfg = {"architectures": ["LlamaForCausalLM"], "num_hidden_layers": 1, "hidden_size": 64, "num_attention_heads": 4,
               "num_key_value_heads": 2, "head_dim": head_dim, "intermediate_size": 64, "vocab_size": 64, "max_position_embeddings": 64}
        spec = build_model_spec(parse_config(cfg))
        spec.blocks[0].mixer.params.update(params)
        return [n.eight_bits for n in DecoderModel(spec, torch.float32, "cpu").cache_needs()]
    assert needs(64) == [True] and needs(32, window=16) == [True] and needs(64, position=None) == [True]
    assert needs(16) == [False] and needs(48) == [False]
    for other in (dict(segment=8), dict(exact_weights=True), dict(v_head_dim=32), dict(score_slopes="geometric"),
                  dict(window=16, keep_first=2)):
        assert needs(64, **other) == [False], other


def test_a_reader_that_cannot_keeps_the_slot_wide():
    from kllm_b200 import models  # noqa: F401
    from kllm_b200.config.base import build_model_spec, parse_config
    from kllm_b200.parts.model import DecoderModel
    from kllm_b200.parts.spec import LayerCall
    cfg = {"architectures": ["LlamaForCausalLM"], "num_hidden_layers": 3, "hidden_size": 64, "num_attention_heads": 4,
           "num_key_value_heads": 2, "head_dim": 32, "intermediate_size": 64, "vocab_size": 64, "max_position_embeddings": 64}
    for reader, want in ((dict(score_slopes="geometric"), [False, True]), ({}, [True, True])):
        spec = build_model_spec(parse_config(cfg))
        spec.blocks[1].mixer.params.update(reader)
        spec.schedule = [LayerCall(0, 0), LayerCall(1, 0, writes_cache=False), LayerCall(2, 1)]
        assert [n.eight_bits for n in DecoderModel(spec, torch.float32, "cpu").cache_needs()] == want


def test_options_name_it():
    from kllm_b200.engine.engine import Options
    assert Options().fill().cache_dtype == "" and Options(cache_dtype="float8_e4m3fn").fill().cache_dtype == "float8_e4m3fn"
    with pytest.raises(ValueError, match="cache dtype"):
        Options(cache_dtype="int8").fill()


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("shape", [(-1,), (1, N, -1)])
def test_queries_that_are_no_matrix(call, shape):
    o = operands()
    o.update(q=o["q"].view(*shape), out=o["out"].view(*shape))
    with pytest.raises(KernelError, match="n, heads"):
        CALLS[call](o)


def test_angles_that_are_no_matrix():
    o = operands()
    o.update(cos_sin=o["cos_sin"].view(-1))
    with pytest.raises(KernelError, match="cos_sin"):
        append(o)


@pytest.mark.parametrize("window,kept", [(None, 0), (0, 0), (-3, 0), (7, 7), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 40 + 5, 2 ** 31 - 1)])
def test_windows_fit_the_kernels_integers(window, kept):
    assert kernels._q8_window(window) == kept


@pytest.mark.parametrize("library,defines,name", [
    ("cache_q8", None, "kllm_rope_append_q8"), ("attention_q8", {"KLLM_HD": 64}, "kllm_attention_decode_q8"),
    ("attention_q8", {"KLLM_HD": 64}, "kllm_attention_prefill_q8"), ("attention_q8_tcgen05", {"KLLM_HD": 64}, "kllm_attention_prefill_q8_tcgen05")])
def test_packed_calls_are_the_typed_ones(library, defines, name):
    """A head size of 35 or less is refused before a device is asked for, whatever the other arguments are: both forms say the same."""
    import ctypes
    import struct
    lib = kernels.load_library(library, defines)
    typed, packed, types = getattr(lib, name), lib.packed(name), lib._params[name]
    error = getattr(lib, "kllm_last_error_" + library)
    error.restype = ctypes.c_char_p
    floats = [t in (ctypes.c_float, ctypes.c_double) for t in types]
    base = [0.5 if f else 35 for f in floats]
    said = set()
    for at in range(len(types)):
        for value in (1, 3, 34, -2):
            args = list(base)
            args[at] = float(value) if floats[at] else value
            a, b = typed(*args), error()
            c, d = packed(*args), error()
            assert a == c and b == d, (at, value)
            said.add((a, b))
    assert len(said) >= 6
    with pytest.raises(struct.error):
        packed(*base[:-1])
    with pytest.raises(struct.error):
        packed(*base, 0)
