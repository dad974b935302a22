"""What is measured of the paged cache in 8 bits: the append that fills it, attention of single tokens and of portions.

The cache of a layer is two stores of e4m3 values [pages, kv heads, page, head size] and a float32 scale per page and kv
head for each, a power of two: a stored number stands for value * scale.

append   rotary encoding of a step's queries and keys, keys and values stored in their pages.  A page's scale is the
         smallest 2^e, -48 <= e <= 48, with max|x| <= 448 * 2^e over the rows that the step stores there, and not below the
         scale of the rows that it holds already; those are stored again under a scale that has grown.
decode   attention of one token per request over the request's pages.
prompt   attention of portions of prompts, behind what is cached of their requests, the portions' own keys included.
"""
import math

import torch

own = False

FLOAT8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def case(name, op, dtype, heads, kv_heads, head_dim, page, requests, new, cached, spread, window=0):
    """``requests`` portions of up to ``new`` tokens behind up to ``cached`` tokens; ``spread``: how much shorter the others
    are than the first (0: all alike)."""
    return dict(name=name, op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                requests=requests, new=new, cached=cached, spread=spread, window=window)


def listed():
    return [
        # a decode step of 8 requests on TinyLlama's layer (the benchmark's step): the smallest call, latency
        case("append_step_b8", "append", "bf16", 32, 4, 64, 64, 8, 1, 2047, 0.0),
        # TinyLlama's prompt of 2048 tokens, the benchmark's other workload
        case("append_prompt_2048", "append", "bf16", 32, 4, 64, 64, 1, 2048, 0, 0.0),
        # ragged portions behind odd lengths at Llama-2-7B's heads, pages of 16, float32: pages that earlier steps began
        case("append_ragged_f32", "append", "f32", 32, 32, 128, 16, 9, 701, 333, 0.9),
        # one request alone: latency
        case("decode_b1_2048", "decode", "bf16", 32, 4, 64, 64, 1, 1, 2047, 0.0),
        # the benchmark's decode step: 8 requests at 2048 tokens
        case("decode_b8_2048", "decode", "bf16", 32, 4, 64, 64, 8, 1, 2047, 0.0),
        # a full batch of unequal contexts at Llama-3-8B's heads, the default page of 16
        case("decode_b64_ragged", "decode", "bf16", 32, 8, 128, 16, 64, 1, 4094, 0.8),
        # one long document
        case("decode_b1_131072", "decode", "bf16", 32, 8, 128, 64, 1, 1, 131071, 0.0),
        # true 32-bit path, no shared heads, odd contexts
        case("decode_f32_b5_ragged", "decode", "f32", 32, 32, 128, 16, 5, 1, 1500, 0.7),
        # TinyLlama's prompt
        case("prompt_2048", "prompt", "bf16", 32, 4, 64, 64, 1, 2048, 0, 0.0),
        # a portion of a long prompt behind what earlier portions cached, Llama-3-8B's heads
        case("prompt_512_behind_7680", "prompt", "bf16", 32, 8, 128, 64, 1, 512, 7680, 0.0),
        # several requests' portions in one step, odd lengths, pages of 16
        case("prompt_ragged_7", "prompt", "bf16", 32, 8, 128, 16, 7, 613, 1201, 0.85),
        # a short prompt on the true 32-bit path
        case("prompt_f32_333", "prompt", "f32", 32, 4, 64, 16, 1, 333, 0, 0.0),
    ]


def draw(rng):
    def spread_over(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    heads, kv_heads, head_dim = rng.choice([(32, 4, 64), (32, 8, 128), (32, 32, 128), (32, 32, 64), (16, 1, 128), (24, 8, 96),
                                            (14, 2, 64), (16, 8, 256), (8, 8, 32), (20, 4, 160)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 24])
    window = rng.choice([0, 0, 0, spread_over(16, 4096)])
    spread = rng.choice([0.0, rng.uniform(0.1, 0.99)])
    if op == "decode":
        requests = spread_over(1, 64)
        most = max(16, min(131071, (1 << 28) // (requests * kv_heads * head_dim)))
        return case("", op, dtype, heads, kv_heads, head_dim, page, requests, 1, spread_over(1, most), spread, window) | {"name": ""}
    requests = spread_over(1, 12)
    new = spread_over(1, max(2, 2048 // requests))
    cached = rng.choice([0, spread_over(1, 4096)])
    if op == "append":
        return case("", op, dtype, heads, kv_heads, head_dim, page, requests, new, min(cached, 2048), spread)
    # the plain form holds every score: at most about what the largest listed case holds
    most = (1 << 27) // (requests * heads * new)
    return case("", op, dtype, heads, kv_heads, head_dim, page, requests, new, max(0, min(cached, most - new)), spread, window)


# ---- a case's lengths: from the case alone, the first request the longest --------------------------------------------

def lengths(c):
    """(cached, new) of every request."""
    out = []
    for i in range(c["requests"]):
        a, b = (i * 0.6180339887) % 1.0, (i * 0.4142135624) % 1.0
        out.append((int(round(c["cached"] * (1 - c["spread"] * a))), max(1, int(round(c["new"] * (1 - c["spread"] * b))))))
    return out


def work(c):
    es = 2 if c["dtype"] == "bf16" else 4
    H, G, hd, W = c["heads"], c["kv_heads"], c["head_dim"], c["window"]
    lens = lengths(c)
    n = sum(new for _, new in lens)
    if c["op"] == "append":
        pages = sum(-(-(old + new) // c["page"]) - old // c["page"] for old, new in lens)
        return {"bytes": n * (2 * H * hd * es + 2 * G * hd * (es + 1) + hd * 4 + 8) + pages * G * 16,
                "flops": n * (H + G) * hd * 3 + n * 2 * G * hd * 2}
    keys = pairs = 0
    for old, new in lens:
        ctx = old + new
        keys += min(ctx, W + new - 1) if W else ctx
        # row i of the portion sees old + i + 1 keys, at most W
        first, last = old + 1, ctx
        if W and last > W:
            pairs += W * (last - max(first, W + 1) + 1)
            last = W
        if last >= first:
            pairs += (first + last) * (last - first + 1) // 2
    pages = sum(-(-(old + new) // c["page"]) for old, new in lens)
    return {"bytes": keys * G * hd * 2 + pages * (G * 8 + 4) + 2 * n * H * hd * es + n * 4, "flops": 4 * pairs * H * hd}


# ---- inputs ------------------------------------------------------------------------------------------------------

def prepare(c, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype = TYPES[c["dtype"]]
    H, G, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens = lengths(c)
    R = len(lens)
    used = [-(-(old + new) // ps) for old, new in lens]
    width = max(used)
    pages = sum(used) + 3
    # pages are handed out in the order in which earlier requests gave them back
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32).cpu()
    table = torch.full((R, width), -1, dtype=torch.int32)
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = order[at:at + u]
        at += u
    rand = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
    # keys have channels of their own magnitudes, pages of different loudness
    channel = torch.exp(0.5 * rand(G, 1, hd))

    def store(loud):
        x = rand(pages, G, ps, hd)
        x *= channel if loud else 1.0
        x *= torch.exp(0.3 * rand(pages, G, 1, 1))
        scale = power_above(x.abs().amax(dim=(2, 3)))
        return (x / scale[:, :, None, None]).to(FLOAT8), scale
    k8, ks = store(True)
    v8, vs = store(False)
    n = sum(new for _, new in lens)
    q_start = [0]
    for _, new in lens:
        q_start.append(q_start[-1] + new)
    positions = torch.cat([torch.arange(old, old + new, dtype=torch.int32) for old, new in lens])
    token_req = torch.repeat_interleave(torch.arange(R, dtype=torch.int32), torch.tensor([new for _, new in lens]))
    ints = lambda v: torch.as_tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = dict(c=c, k8=k8, ks=ks, v8=v8, vs=vs, table=ints(table), positions=ints(positions), token_req=ints(token_req),
             q_start=ints(q_start), start=ints([old for old, _ in lens]), ctx=max(old + new for old, new in lens),
             new=max(new for _, new in lens), n=n, R=R, scale=1.0 / math.sqrt(hd))
    # the projections of one stacked product: q, k and v are slices of its rows
    qkv = rand(n, (H + 2 * G) * hd)
    qkv[:, :H * hd] *= 2.0
    qkv[:, H * hd:(H + G) * hd] *= (1.5 * channel).reshape(1, G * hd)
    qkv = qkv.to(dtype)
    s["q"], s["k"], s["v"] = qkv[:, :H * hd], qkv[:, H * hd:(H + G) * hd], qkv[:, (H + G) * hd:]
    s["out"] = torch.zeros(n, H * hd, dtype=dtype, device=dev)
    if c["op"] == "append":
        half = hd // 2
        ang = torch.arange(s["ctx"], dtype=torch.float64, device=dev)[:, None] * \
            torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=dev),
                      -2.0 * torch.arange(half, dtype=torch.float64, device=dev) / hd)[None, :]
        s["cos_sin"] = torch.cat([torch.cos(ang), torch.sin(ang)], dim=1).float().contiguous()
    return s


# ---- the plain forms: 32 bits, elementary operations -----------------------------------------------------------------

def power_above(amax):
    """The smallest 2^e, -48 <= e <= 48, with amax <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(amax)             # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -48)).clamp(-48, 48)
    return torch.ldexp(torch.ones_like(amax), e)


def rotated(x, cs, heads, hd):
    x = x.float().view(-1, heads, 2, hd // 2)
    cos, sin = cs[:, None, :hd // 2], cs[:, None, hd // 2:]
    a, b = x[:, :, 0], x[:, :, 1]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)


def append_into(store, scale, rows, page, slot, first, touched):
    """rows [n, G, hd] into store [pages, G, ps, hd] at (page, slot); ``first`` [pages]: the first slot that is written."""
    ps = store.shape[2]
    amax = torch.zeros_like(scale).index_reduce_(0, page, rows.abs().amax(dim=2), "amax")
    held = (first > 0) & touched
    grown = torch.maximum(power_above(amax), torch.where(held[:, None], scale, torch.zeros_like(scale)))
    grown = torch.where(touched[:, None], grown, scale)
    again = (store.float() * (scale / grown)[:, :, None, None]).to(FLOAT8).view(torch.uint8)
    earlier = torch.arange(ps, device=store.device)[None, :] < torch.where(held, first, torch.zeros_like(first))[:, None]
    bytes_ = torch.where(earlier[:, None, :, None], again, store.view(torch.uint8))
    bytes_[page, :, slot] = (rows / grown[page][:, :, None]).to(FLOAT8).view(torch.uint8)
    store.view(torch.uint8).copy_(bytes_)
    scale.copy_(grown)


def plain_append(s):
    c = s["c"]
    H, G, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    pos = s["positions"].long()
    page = s["table"].long()[s["token_req"].long(), pos // ps]
    slot = pos % ps
    cs = s["cos_sin"][pos]
    s["out"].copy_(rotated(s["q"], cs, H, hd).reshape(s["n"], H * hd))
    first = torch.full((s["k8"].shape[0],), ps, dtype=torch.int64, device=pos.device).index_reduce_(0, page, slot, "amin")
    touched = first < ps
    append_into(s["k8"], s["ks"], rotated(s["k"], cs, G, hd), page, slot, first, touched)
    append_into(s["v8"], s["vs"], s["v"].float().view(-1, G, hd), page, slot, first, touched)
    return s["out"], s["k8"], s["ks"], s["v8"], s["vs"]


def plain_attention(s):
    c = s["c"]
    H, G, hd, ps, W = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["window"]
    R, new, n = s["R"], s["new"], s["n"]
    table = s["table"].long().clamp(min=0)

    def held(store, scale):        # [R, G, places, hd]
        x = store.view(torch.uint8)[table].view(FLOAT8).float() * scale[table][:, :, :, None, None]
        return x.transpose(1, 2).reshape(R, G, -1, hd)
    keys, values = held(s["k8"], s["ks"]), held(s["v8"], s["vs"])
    req = s["token_req"].long()
    row = torch.arange(n, device=req.device) - s["q_start"].long()[req]
    q = torch.zeros(R, new, H * hd, device=req.device)
    q[req, row] = s["q"].float()
    q = q.view(R, new, G, H // G, hd).permute(0, 2, 3, 1, 4).reshape(R, G, -1, hd)
    scores = (q @ keys.transpose(2, 3)).view(R, G, H // G, new, -1) * s["scale"]
    at = s["start"].long()[:, None] + torch.arange(new, device=req.device)[None, :]      # a row's position
    j = torch.arange(keys.shape[2], device=req.device)
    seen = j[None, None, :] <= at[:, :, None]
    if W:
        seen = seen & (j[None, None, :] > at[:, :, None] - W)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(dim=-1, keepdim=True)
    weights = scores.exp_()
    total = weights.sum(dim=-1, keepdim=True)
    out = (weights.view(R, G, -1, keys.shape[2]) @ values).view(R, G, H // G, new, hd) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(R, new, H * hd)
    return out[req, row].to(s["q"].dtype)


def run(s):
    if own:
        from kllm_b200 import kernels
        c = s["c"]
        H, G, hd = c["heads"], c["kv_heads"], c["head_dim"]
        if c["op"] == "append":
            kernels.rope_append_q8(s["out"], s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["token_req"], s["q_start"],
                                   s["table"], s["k8"], s["v8"], s["ks"], s["vs"], H, G, hd)
            return s["out"], s["k8"], s["ks"], s["v8"], s["vs"]
        if c["op"] == "decode":
            kernels.attention_decode_q8(s["out"], s["q"], s["k8"], s["v8"], s["ks"], s["vs"], s["positions"], None, s["table"],
                                        H, G, hd, c["window"], s["scale"], s["ctx"])
        else:
            kernels.attention_prefill_q8(s["out"], s["q"], s["k8"], s["v8"], s["ks"], s["vs"], s["q_start"], s["start"],
                                         s["table"], s["R"], H, G, hd, c["window"], s["scale"], s["ctx"])
        return s["out"]
    return plain_append(s) if s["c"]["op"] == "append" else plain_attention(s)


# ---- from the definitions, in 64 bits, request by request ---------------------------------------------------------------

def nearest_e4m3(x):
    """The e4m3 value next to each number of x, ties to the even one: steps of 2^-9 below 2^-6, of an eighth of the binade above."""
    binade = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    binade = torch.where(torch.ldexp(torch.ones_like(x), binade.int()) > x.abs().clamp(min=2.0 ** -6), binade - 1, binade)
    step = torch.ldexp(torch.ones_like(x), (binade - 3).int())
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(c, seed):
    s = prepare(c, seed)
    H, G, hd, ps, W = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["window"]
    lens = lengths(c)
    if c["op"] == "append":
        half = hd // 2

        def turned(x, heads, pos):
            x = x.double().view(-1, heads, hd)
            cs = s["cos_sin"].double()[pos][:, None]
            lo, hi = x[..., :half], x[..., half:]
            return torch.cat((lo * cs[..., :half] - hi * cs[..., half:], hi * cs[..., :half] + lo * cs[..., half:]), -1)
        out = turned(s["q"], H, s["positions"].long()).view(s["n"], H * hd)
        stores = []
        for x, store, scale in ((turned(s["k"], G, s["positions"].long()), s["k8"], s["ks"]),
                                (s["v"].double().view(-1, G, hd), s["v8"], s["vs"])):
            store, scale = store.double(), scale.double()
            at = 0
            for r, (old, new) in enumerate(lens):
                for lp in range(old // ps, (old + new - 1) // ps + 1):
                    lo, hi = max(old, lp * ps), min(old + new, (lp + 1) * ps)
                    page, rows = int(s["table"][r, lp]), x[at + lo - old:at + hi - old].transpose(0, 1)     # [G, rows, hd]
                    need = rows.abs().amax(dim=(1, 2))
                    e = torch.ceil(torch.log2(need.clamp(min=1e-300) / 448.0)).clamp(-48, 48)
                    two = torch.ldexp(torch.ones_like(need), e.int())
                    kept = lo - lp * ps
                    if kept:
                        two = torch.maximum(two, scale[page])
                        store[page, :, :kept] = nearest_e4m3(store[page, :, :kept] * (scale[page] / two)[:, None, None])
                    store[page, :, kept:hi - lp * ps] = nearest_e4m3(rows / two[:, None, None])
                    scale[page] = two
                at += new
            stores += [store, scale]
        return out, stores[0], stores[1], stores[2], stores[3]
    out = torch.empty(s["n"], H * hd, dtype=torch.float64, device="cuda")
    at = 0
    for r, (old, new) in enumerate(lens):
        ctx = old + new
        low = max(0, old + 1 - W) // ps if W else 0          # the first page that a row of the portion sees
        pages = s["table"][r, low:-(-ctx // ps)].long()
        first = low * ps

        def held(store, scale):
            x = store.view(torch.uint8)[pages].view(FLOAT8).double() * scale[pages].double()[:, :, None, None]
            return x.transpose(0, 1).reshape(G, -1, hd)[:, :ctx - first]
        keys, values = held(s["k8"], s["ks"]), held(s["v8"], s["vs"])
        p = torch.arange(old, ctx, device="cuda")[:, None]
        j = torch.arange(first, ctx, device="cuda")[None, :]
        hidden = (j > p) | (j <= p - W) if W else j > p
        q = s["q"][at:at + new].double().view(new, H, hd)
        for h in range(H):
            z = q[:, h] @ keys[h // (H // G)].T / math.sqrt(hd)
            w = torch.softmax(z.masked_fill(hidden, -math.inf), dim=1)
            out[at:at + new, h * hd:(h + 1) * hd] = w @ values[h // (H // G)]
        at += new
    return out
