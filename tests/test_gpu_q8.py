"""The paged cache in 8 bits on the GPU: the append that fills it, attention of single tokens and of portions, against plain
operations in 64 bits (tests/q8_plain.py), with tolerances that count the roundings."""
import math

import pytest
import torch

import q8_plain as plain

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
NAN_BYTE = 0x7F


class Cache:
    """Stores of random numbers with pages handed out in a random order; what no request holds is NaN all over."""

    def __init__(self, starts, lens, G, hd, ps, seed, spread=0.5, fill=True):
        g = torch.Generator().manual_seed(seed)
        used = [max(0, -(-(a + b) // ps)) for a, b in zip(starts, lens)]
        self.pages = sum(used) + 2
        order = torch.randperm(self.pages, generator=g)
        width = max(used + [1])
        self.table = torch.full((len(starts), width), -1, dtype=torch.int32)
        at = 0
        for r, u in enumerate(used):
            self.table[r, :u] = order[at:at + u].int()
            at += u
        ek, ev = (torch.randn(self.pages, G, generator=g).mul(spread).round() for _ in range(2))
        k8 = (torch.randn(self.pages, G, ps, hd, generator=g) * 100).clamp(-448, 448).to(plain.E4M3)
        v8 = (torch.randn(self.pages, G, ps, hd, generator=g) * 100).clamp(-448, 448).to(plain.E4M3)
        ks, vs = torch.exp2(ek - 7), torch.exp2(ev - 7)
        if fill:
            held = torch.zeros(self.pages, ps, dtype=torch.bool)
            for r, (a, b) in enumerate(zip(starts, lens)):
                for j in range(max(0, a + b)):
                    held[int(self.table[r, j // ps]), j % ps] = True
            for t in (k8, v8):
                t.view(torch.uint8).masked_fill_(~held[:, None, :, None], NAN_BYTE)
            free = ~held.any(dim=1)
            ks[free], vs[free] = math.nan, math.nan
        self.k, self.v, self.ks, self.vs = (t.cuda() for t in (k8, v8, ks, vs))
        self.dev_table = self.table.cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def queries(n, H, hd, dtype, seed, loud=2.0, slack=24):
    """Rows of a wider tensor, as slices of a stacked projection are."""
    g = torch.Generator().manual_seed(seed + 1)
    wide = (torch.randn(n, H * hd + slack, generator=g) * loud).to(DT[dtype]).cuda()
    return wide[:, 8:8 + H * hd]


def decode(c, q, pos, H, G, hd, window=0, scale=None, req=None, bound=None, out=None):
    from kllm_b200 import kernels
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    kernels.attention_decode_q8(out, q, c.k, c.v, c.ks, c.vs, pos, req, c.dev_table, H, G, hd, window,
                                scale or hd ** -0.5, bound or int(pos.max()) + 1)
    return out


def prefill(c, q, starts, lens, H, G, hd, window=0, scale=None, out=None):
    from kllm_b200 import kernels
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    q_start = [0]
    for n in lens:
        q_start.append(q_start[-1] + n)
    kernels.attention_prefill_q8(out, q, c.k, c.v, c.ks, c.vs, ints(*q_start), ints(*starts), c.dev_table, len(lens), H, G, hd, window,
                                 scale or hd ** -0.5, max(a + b for a, b in zip(starts, lens)))
    assert int(kernels.status_word(q.device).item()) == 0
    return out


def check(got, q, c, starts, lens, H, G, hd, window=0, scale=None):
    want, err = plain.attention(q, c.k, c.v, c.ks, c.vs, c.table, starts, lens, H, G, hd, window, scale or hd ** -0.5)
    diff = (got.cpu().double() - want).abs()
    assert torch.isfinite(got.float()).all()
    over = diff > err
    assert not bool(over.any()), f"{int(over.sum())} of {over.numel()} beyond their bound, worst {float((diff / err.clamp(min=1e-300)).max()):.2f} times"


# ---- single tokens -----------------------------------------------------------------------------------------------------

HEADS = [(8, 1, 64), (32, 4, 64), (8, 8, 64), (8, 2, 128), (32, 2, 128), (3, 1, 32), (10, 2, 96), (6, 6, 160), (14, 1, 192),
         (4, 2, 224), (24, 2, 256), (7, 7, 32), (32, 1, 128)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd", HEADS)
def test_decode_head_layouts(dtype, H, G, hd):
    ctx = [1, 2, 31, 32, 33, 150]
    starts, lens = [n - 1 for n in ctx], [1] * len(ctx)
    c = Cache(starts, lens, G, hd, 16, seed=H + hd)
    q = queries(len(ctx), H, hd, dtype, seed=hd)
    check(decode(c, q, ints(*starts), H, G, hd), q, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 17, 32, 200])
def test_decode_pages_and_windows(dtype, page, window):
    H, G, hd = 8, 2, 64
    ctx = [1, 16, 63, 64, 65, 127, 128, 129, 300, 513]
    starts, lens = [n - 1 for n in ctx], [1] * len(ctx)
    c = Cache(starts, lens, G, hd, page, seed=page + window)
    q = queries(len(ctx), H, hd, dtype, seed=page)
    if window:                                   # pages behind the window may have been given back
        for r, n in enumerate(ctx):
            gone = max(0, n - window) // page
            c.table[r, :gone] = -1
        c.dev_table = c.table.cuda()
    check(decode(c, q, ints(*starts), H, G, hd, window), q, c, starts, lens, H, G, hd, window)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("tokens,ctx,H,G,hd", [(1, 3000, 8, 1, 64), (1, 20011, 4, 1, 128), (2, 5000, 4, 4, 64), (3, 1025, 32, 4, 64)])
def test_decode_contexts_in_parts(dtype, tokens, ctx, H, G, hd):
    """Clusters, ranges of clusters, parts that stay empty (the other contexts are short under the same bound)."""
    starts = [ctx - 1] + [11, 600][:tokens - 1]
    lens = [1] * tokens
    c = Cache(starts, lens, G, hd, 16, seed=ctx)
    q = queries(tokens, H, hd, dtype, seed=3)
    check(decode(c, q, ints(*starts), H, G, hd), q, c, starts, lens, H, G, hd)
    a = decode(c, q, ints(*starts), H, G, hd)
    assert torch.equal(a, decode(c, q, ints(*starts), H, G, hd)), "the same call twice"
    assert torch.equal(a[:1], decode(c, q, ints(*starts), H, G, hd, bound=ctx)[:1])
    # the bound only cuts: a larger one than any context gives the same within the roundings
    check(decode(c, q, ints(*starts), H, G, hd, bound=4 * ctx), q, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
def test_decode_scales_far_apart(dtype):
    """Pages whose scales differ by 2^40: loud keys decide alone, loud values stay in range, quiet ones are not lost."""
    H, G, hd = 8, 2, 64
    starts, lens = [199, 70], [1, 1]
    for spread in (6.0, 12.0):
        c = Cache(starts, lens, G, hd, 16, seed=5, spread=0.0)
        g = torch.Generator().manual_seed(9)
        e = (torch.randn(c.vs.shape, generator=g) * spread).round().clamp(-40, 40)
        c.vs = torch.where(torch.isnan(c.vs.cpu()), c.vs.cpu(), torch.exp2(e)).cuda()
        q = queries(2, H, hd, dtype, seed=6, loud=0.5)
        check(decode(c, q, ints(*starts), H, G, hd), q, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
def test_decode_queries_of_any_size(dtype):
    """Rows of very small and very large queries: the power of two that is taken out of a row."""
    H, G, hd = 8, 2, 64
    starts, lens = [40] * 6, [1] * 6
    c = Cache(starts, lens, G, hd, 16, seed=5)
    q = queries(6, H, hd, dtype, seed=6)
    for i, s in enumerate((2.0 ** -120, 2.0 ** -30, 2.0 ** -14, 1.0, 2.0 ** 10, 0.0)):
        q[i] *= s
    check(decode(c, q, ints(*starts), H, G, hd), q, c, starts, lens, H, G, hd)


def test_decode_rows_without_keys_and_requests():
    H, G, hd = 8, 2, 64
    starts, lens = [40, 20, 33, 64], [1] * 4
    c = Cache(starts, lens, G, hd, 16, seed=5)
    q = queries(4, H, hd, "bf16", seed=6)
    pos = ints(40, -1, -2147483648, 64)
    got = decode(c, q, pos, H, G, hd, bound=65)
    assert bool((got[1:3] == 0).all())
    check(got[:1], q[:1], c, [40], [1], H, G, hd)
    # a request that is none, in either direction
    got = decode(c, q, ints(*starts), H, G, hd, req=ints(2, 9, -1, 0), bound=65)
    assert bool((got[1:3] == 0).all()) and bool((got[0] != 0).any())


@pytest.mark.parametrize("dtype", DT)
def test_decode_keys_without_a_page(dtype):
    """Table entries that name no page, and places behind the table's end, are not seen."""
    H, G, hd = 8, 2, 64
    starts, lens = [99, 130], [1, 1]
    c = Cache(starts, lens, G, hd, 16, seed=5)
    c.table[0, 0], c.table[0, 3], c.table[0, 6] = -1, c.pages, 2 ** 31 - 1
    c.table[1, 1], c.table[1, 2] = -2 ** 31, c.pages + 5
    c.dev_table = c.table.cuda()
    q = queries(2, H, hd, dtype, seed=6)
    check(decode(c, q, ints(*starts), H, G, hd), q, c, starts, lens, H, G, hd)
    c.table = c.table[:, :4].contiguous()
    c.dev_table = c.table.cuda()
    check(decode(c, q, ints(*starts), H, G, hd), q, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("form", ["decode", "prefill"])
@pytest.mark.parametrize("dtype", DT)
def test_nan_reaches_the_rows_that_see_it(form, dtype):
    """A NaN key makes the rows that see it NaN and no others; a NaN or an infinity among a head's queries that head's row."""
    H, G, hd, W = 8, 2, 64, 48
    starts, lens = ([99, 99], [1, 1]) if form == "decode" else ([40, 0], [60, 33])
    c = Cache(starts, lens, G, hd, 16, seed=5)
    n = sum(lens)
    q = queries(n, H, hd, dtype, seed=6)
    bad = 45                                                  # of request 0: outside the window of later rows
    page, slot = int(c.table[0, bad // 16]), bad % 16
    c.k.view(torch.uint8)[page, 1, slot] = NAN_BYTE
    c.v.view(torch.uint8)[page, 1, slot] = 0
    q[n - 1, 3 * hd + 5] = math.inf
    q[n - 2, 0] = math.nan
    run = (lambda w: decode(c, q, ints(*starts), H, G, hd, w)) if form == "decode" else (lambda w: prefill(c, q, starts, lens, H, G, hd, w))
    clean_q = q.clone()
    clean_q[n - 1, 3 * hd + 5] = 1.0
    clean_q[n - 2, 0] = 1.0
    for w in (0, W):
        got = run(w).float().view(n, H, hd)
        expect = torch.zeros(n, H, dtype=torch.bool)
        at = 0
        for r, (a, m) in enumerate(zip(starts, lens)):
            for i in range(m):
                p = a + i
                if r == 0 and p >= bad and (not w or bad > p - w):
                    expect[at + i, H // G:] = True
            at += m
        expect[n - 1, 3] = expect[n - 2, 0] = True
        assert torch.equal(torch.isnan(got).all(dim=2).cpu(), expect)
        assert torch.equal(torch.isnan(got).any(dim=2).cpu(), expect)
        k2 = c.k.view(torch.uint8).clone()
        c.k.view(torch.uint8)[page, 1, slot] = 0
        want, err = plain.attention(clean_q, c.k, c.v, c.ks, c.vs, c.table, starts, lens, H, G, hd, w, hd ** -0.5)
        c.k.view(torch.uint8).copy_(k2)
        rest = (~expect)[:, :, None]
        diff = (got.cpu().double() - want.view(n, H, hd)).abs()
        assert bool(((diff <= err.view(n, H, hd)) | ~rest).all())


# ---- portions --------------------------------------------------------------------------------------------------------------

PORTIONS = [([0], [1]), ([0], [63]), ([0], [64]), ([0, 0], [65, 130]), ([64, 3, 0], [1, 62, 2]), ([127, 0, 128, 9], [1, 128, 2, 40])]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd", [(8, 2, 64), (32, 4, 64), (4, 4, 128), (8, 1, 128), (3, 1, 32), (10, 2, 96), (64, 1, 64)])
@pytest.mark.parametrize("starts,lens", PORTIONS)
def test_prefill_edges(dtype, H, G, hd, starts, lens):
    c = Cache(starts, lens, G, hd, 16, seed=H + hd)
    q = queries(sum(lens), H, hd, dtype, seed=hd)
    check(prefill(c, q, starts, lens, H, G, hd), q, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128, 160, 256])
@pytest.mark.parametrize("page", [1, 24, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_prefill_pages_and_windows(dtype, hd, page, window):
    H, G = 4, 2
    starts, lens = [100, 0, 37], [70, 90, 5]
    c = Cache(starts, lens, G, hd, page, seed=page + window)
    q = queries(sum(lens), H, hd, dtype, seed=page)
    if window:
        for r, n in enumerate(starts):
            c.table[r, :max(0, n + 1 - window) // page] = -1
        c.dev_table = c.table.cuda()
    check(prefill(c, q, starts, lens, H, G, hd, window), q, c, starts, lens, H, G, hd, window)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_long(dtype, hd):
    H, G = 4, 1
    starts, lens = [700, 0], [150, 333]
    c = Cache(starts, lens, G, hd, 64, seed=hd, spread=3.0)
    q = queries(sum(lens), H, hd, dtype, seed=hd)
    a = prefill(c, q, starts, lens, H, G, hd)
    check(a, q, c, starts, lens, H, G, hd)
    assert torch.equal(a, prefill(c, q, starts, lens, H, G, hd)), "the same call twice"


@pytest.mark.parametrize("hd", [64, 96])
def test_prefill_leaves_other_rows_alone_and_takes_empty_portions(hd):
    H, G = 8, 2
    starts, lens = [5, 9, 0, 30], [0, 20, 0, 3]
    c = Cache(starts, lens, G, hd, 16, seed=5)
    q = queries(sum(lens) + 9, H, hd, "bf16", seed=6)
    got = prefill(c, q, starts, lens, H, G, hd)
    assert bool((got[23:] == 7.0).all())
    check(got[:23], q[:23], c, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_keys_without_a_page(dtype, hd):
    H, G = 8, 2
    starts, lens = [90, 0], [40, 20]
    c = Cache(starts, lens, G, hd, 16, seed=5)
    c.table[0, 0], c.table[0, 3], c.table[0, 8] = -1, c.pages, 2 ** 31 - 1
    c.table[1, 0] = -5                                        # the first sixteen rows of request 1 see nothing
    c.dev_table = c.table.cuda()
    q = queries(60, H, hd, dtype, seed=6)
    got = prefill(c, q, starts, lens, H, G, hd)
    check(got, q, c, starts, lens, H, G, hd)
    assert bool((got[40:56] == 0).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_scales_far_apart(dtype, hd):
    H, G = 8, 2
    starts, lens = [100, 0], [50, 70]
    c = Cache(starts, lens, G, hd, 16, seed=5, spread=0.0)
    g = torch.Generator().manual_seed(9)
    e = (torch.randn(c.vs.shape, generator=g) * 12).round().clamp(-40, 40)
    c.vs = torch.where(torch.isnan(c.vs.cpu()), c.vs.cpu(), torch.exp2(e)).cuda()
    q = queries(120, H, hd, dtype, seed=6, loud=0.5)
    check(prefill(c, q, starts, lens, H, G, hd), q, c, starts, lens, H, G, hd)


# ---- append ---------------------------------------------------------------------------------------------------------------

def table_of_angles(positions, rot):
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * torch.pow(torch.tensor(10000.0, dtype=torch.float64),
                                                                             -2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)[None]
    return torch.cat([torch.cos(ang), torch.sin(ang)], dim=1).float().cuda()


def run_append(c, q, k, v, cs, starts, lens, H, G, hd, in_place=False, req=True, extra=0):
    from kllm_b200 import kernels
    pos = [a + i for a, n in zip(starts, lens) for i in range(n)] + [3] * extra
    token_req = [r for r, n in enumerate(lens) for _ in range(n)] + [0] * extra
    q_start = [0]
    for n in lens:
        q_start.append(q_start[-1] + n)
    q_out = q if in_place else torch.full((q.shape[0], q.shape[1] + 8), 7.0, dtype=q.dtype, device="cuda")[:, :q.shape[1]]
    kernels.rope_append_q8(q_out, q, k, v, cs, ints(*pos), ints(*token_req) if req else None, ints(*q_start), c.dev_table, c.k, c.v,
                           c.ks, c.vs, H, G, hd)
    return q_out, torch.tensor(pos)


def check_append(c, before, q_out, q, k, v, cs, pos, starts, lens, H, G, hd):
    n = sum(lens)
    kr, vr = plain.turned(k[:n], cs, pos[:n], G, hd), v[:n].cpu().double().view(n, G, hd)
    for name, is_key in (("key", True), ("value", False)):
        store, scale = (c.k, c.ks) if is_key else (c.v, c.vs)
        want, sc, written = plain.append(before[name][0], before[name][1], kr, vr, is_key, c.table, starts, lens)
        assert torch.equal(scale.cpu().double().nan_to_num(-1.0), sc.nan_to_num(-1.0)), name + " scales"
        got = store.cpu().float().double()
        if not is_key or cs is None:
            assert torch.equal(got.nan_to_num(1e6), want.nan_to_num(1e6)), name
            continue
        # a rotated key is rounded from float32: two products, one sum and, beside an e4m3 border, the other neighbour
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        away = ~written
        assert torch.equal(got[away].nan_to_num(1e6), want[away].nan_to_num(1e6)), "rows that were there"
        differ = (got != want) & ~torch.isnan(want)
        if bool(differ.any()):
            step = (got - want).abs()[differ]
            assert bool((step <= want.abs()[differ] * 2.0 ** -3 + 2.0 ** -9).all())
            assert int(differ.sum()) <= 2 + want.numel() * 2e-5
    want = plain.turned(q[:n], cs, pos[:n], H, hd).view(n, H * hd)
    size = q[:n].cpu().double().abs().amax(dim=1, keepdim=True)
    half = torch.finfo(q.dtype).eps / 2
    assert bool(((q_out[:n].cpu().double() - want).abs() <= want.abs() * half + size * 2.0 ** -22).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,rot", [(8, 2, 64, 64), (4, 4, 128, 128), (3, 1, 32, 32), (10, 2, 96, 48), (8, 1, 256, 256), (4, 2, 64, 6),
                                        (4, 2, 160, 0), (8, 8, 64, 2)])
@pytest.mark.parametrize("page,starts,lens", [(16, [0], [1]), (16, [0, 5, 31], [40, 12, 2]), (5, [3, 0], [17, 9]), (64, [10, 100, 0], [1, 1, 1]),
                                              (256, [0, 130], [200, 150]), (1, [2, 0], [3, 4])])
def test_append(dtype, H, G, hd, rot, page, starts, lens):
    c = Cache(starts, lens, G, hd, page, seed=page + hd, fill=False)
    n = sum(lens)
    q, k, v = queries(n, H, hd, dtype, 1), queries(n, G, hd, dtype, 2, loud=5.0), queries(n, G, hd, dtype, 3)
    cs = table_of_angles(400, rot) if rot else None
    before = dict(key=(c.k.clone(), c.ks.clone()), value=(c.v.clone(), c.vs.clone()))
    q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
    check_append(c, before, q_out, q, k, v, cs, pos, starts, lens, H, G, hd)
    # the same rows once more, rotated in place: nothing changes in the cache
    kept = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)]
    q2, _ = run_append(c, q, k, v, cs, starts, lens, H, G, hd, in_place=True, req=n != len(lens))
    assert torch.equal(q2, q_out)
    for a, b in zip(kept, (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
def test_append_grows_a_page(dtype):
    """Token after token of growing size into the same pages: earlier rows are stored again under the grown scale."""
    H, G, hd, ps, steps = 4, 2, 64, 16, 40
    c = Cache([0, 0], [steps, steps], G, hd, ps, seed=4, fill=False)
    for i in range(steps):
        k, v = queries(2, G, hd, dtype, 10 + i, loud=2.0 ** (i % 16 - 6)), queries(2, G, hd, dtype, 90 + i, loud=2.0 ** ((5 * i) % 21 - 9))
        q = queries(2, H, hd, dtype, 5)
        before = dict(key=(c.k.clone(), c.ks.clone()), value=(c.v.clone(), c.vs.clone()))
        q_out, pos = run_append(c, q, k, v, None, [i, i], [1, 1], H, G, hd, req=False)
        check_append(c, before, q_out, q, k, v, None, pos, [i, i], [1, 1], H, G, hd)


@pytest.mark.parametrize("dtype", DT)
def test_append_numbers_at_the_borders(dtype):
    """Zeros, numbers beyond the scales' range on either side, 448 2^e and what follows it, e4m3's subnormals."""
    H, G, hd, ps = 2, 1, 32, 16
    rows = [0.0, 448.0, 449.0, 450.0, 464.0, 2.0 ** -60, 2.0 ** -41, 448 * 2.0 ** 48, 1e18, 3e38, 2.0 ** -57]
    n = len(rows)
    starts, lens = [0] * n, [1] * n
    c = Cache(starts, lens, G, hd, ps, seed=4, fill=False)
    x = torch.tensor(rows)[:, None] * torch.cat([torch.ones(1), torch.rand(hd - 1, generator=torch.Generator().manual_seed(1)) - 0.5])[None]
    k, v = x.to(DT[dtype]).cuda(), (-x).to(DT[dtype]).cuda()
    q = queries(n, H, hd, dtype, 5)
    before = dict(key=(c.k.clone(), c.ks.clone()), value=(c.v.clone(), c.vs.clone()))
    q_out, pos = run_append(c, q, k, v, None, starts, lens, H, G, hd)
    check_append(c, before, q_out, q, k, v, None, pos, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rot", [0, 64])
def test_append_of_what_is_not_finite(dtype, rot):
    H, G, hd, ps = 4, 2, 64, 16
    starts, lens = [3, 0], [30, 20]
    c = Cache(starts, lens, G, hd, ps, seed=4, fill=False)
    n = sum(lens)
    q, k, v = queries(n, H, hd, dtype, 1), queries(n, G, hd, dtype, 2), queries(n, G, hd, dtype, 3)
    k[4, 7], k[9, hd + 3], v[12, 5], v[30, hd + 60], k[49, 63] = math.inf, math.nan, -math.inf, math.nan, math.nan
    for i in range(34, 50):
        v[i, 0] = math.inf                            # a page (the last of request 1) without one finite row of head 0
    cs = table_of_angles(64, rot) if rot else None
    before = dict(key=(c.k.clone(), c.ks.clone()), value=(c.v.clone(), c.vs.clone()))
    q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
    check_append(c, before, q_out, q, k, v, cs, pos, starts, lens, H, G, hd)


def test_append_leaves_out_what_has_no_place():
    """Rows behind the last request, negative positions, positions behind the angles, missing pages: nothing is touched."""
    from kllm_b200 import kernels
    H, G, hd, ps = 4, 2, 64, 16
    starts, lens = [0, 0, 0, 0], [1, 1, 1, 1]
    c = Cache([40] * 4, lens, G, hd, ps, seed=4, fill=False)
    c.table[2, 1] = -1
    c.table[3, 1] = c.pages
    c.dev_table = c.table.cuda()
    q, k, v = queries(6, H, hd, "bf16", 1), queries(6, G, hd, "bf16", 2), queries(6, G, hd, "bf16", 3)
    kept = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)]
    cs = table_of_angles(32, hd)
    q_out = torch.full_like(q, 7.0)
    kernels.rope_append_q8(q_out, q, k, v, cs, ints(-1, 32, 20, 21, 0, 0), ints(0, 1, 2, 3, 0, 1), ints(0, 1, 2, 3, 4), c.dev_table, c.k, c.v,
                           c.ks, c.vs, H, G, hd)
    assert bool((q_out[:2] == 7.0).all()) and bool((q_out[4:] == 7.0).all())
    want = plain.turned(q[2:4], cs, torch.tensor([20, 21]), H, hd).view(2, -1)
    assert bool(((q_out[2:4].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-4).all())
    for a, b in zip(kept, (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)):
        assert torch.equal(a, b)


# ---- together --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
def test_portions_then_tokens(dtype):
    """A run as an engine makes it: portions of three prompts, then single tokens, appended and attended to step by step; the
    attention of every step against the cache as it stands then, and the cache against the plain one."""
    H, G, hd, ps = 8, 2, 64, 16
    total = [50, 37, 90]
    c = Cache([0, 0, 0], [t + 8 for t in total], G, hd, ps, seed=11, fill=False)
    cs = table_of_angles(128, hd)
    length = [0, 0, 0]
    seed = 100
    for step in [(20, 37, 33), (30, 0, 1), (0, 0, 56)] + [(1, 1, 1)] * 8:
        lens, starts = list(step), list(length)
        n = sum(lens)
        seed += 10
        q, k, v = queries(n, H, hd, dtype, seed), queries(n, G, hd, dtype, seed + 1), queries(n, G, hd, dtype, seed + 2)
        before = dict(key=(c.k.clone(), c.ks.clone()), value=(c.v.clone(), c.vs.clone()))
        q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
        check_append(c, before, q_out, q, k, v, cs, pos, starts, lens, H, G, hd)
        rows = q_out.clone()
        got = decode(c, rows, ints(*pos.tolist()), H, G, hd) if all(m == 1 for m in lens) else prefill(c, rows, starts, lens, H, G, hd)
        check(got, rows, c, starts, lens, H, G, hd)
        length = [a + b for a, b in zip(length, lens)]


def test_on_another_stream_and_in_a_graph():
    """A step's three calls captured once and replayed with other inputs in the same buffers, beside eager calls on another stream."""
    from kllm_b200 import kernels
    H, G, hd, ps, n = 8, 2, 64, 16, 3
    start = [30, 2000, 64]
    c = Cache(start, [8] * n, G, hd, ps, seed=12)
    cs = table_of_angles(2100, hd)
    pos, q_start = ints(*start), ints(0, 1, 2, 3)
    q, k, v = (torch.zeros(n, w * hd, dtype=torch.bfloat16, device="cuda") for w in (H, G, G))
    out, rows = torch.zeros_like(q), torch.zeros_like(q)

    def step():
        kernels.rope_append_q8(rows, q, k, v, cs, pos, None, q_start, c.dev_table, c.k, c.v, c.ks, c.vs, H, G, hd)
        kernels.attention_decode_q8(out, rows, c.k, c.v, c.ks, c.vs, pos, None, c.dev_table, H, G, hd, 0, hd ** -0.5, 2100)
    saved = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    outs = []
    for use in ("graph", "stream"):
        for t, b in zip(saved, (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)):
            b.copy_(t)
        pos.copy_(ints(*start))
        seen = []
        side = torch.cuda.Stream()
        for i in range(4):
            for t, w in ((q, H), (k, G), (v, G)):
                t.copy_(queries(n, w, hd, "bf16", 40 * i + w))
            if use == "graph":
                graph.replay()
            else:
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
            seen.append(out.clone())
            check(out, rows, c, [s + i for s in start], [1] * n, H, G, hd)
            pos += 1
        outs.append(torch.stack(seen))
    assert torch.equal(outs[0], outs[1])


def test_refuses_what_the_kernels_do_not_take():
    from kllm_b200.kernels import KernelError
    c = Cache([10], [1], 1, 64, 16, seed=1)
    with pytest.raises(KernelError, match="at most 64"):
        prefill(c, queries(1, 128, 64, "f32", 1), [10], [1], 128, 1, 64)
    off = torch.zeros(c.k.numel() + 16, dtype=torch.uint8, device="cuda")[8:8 + c.k.numel()].view(plain.E4M3).view(c.k.shape)
    c.k = off
    with pytest.raises(KernelError, match="aligned"):
        decode(c, queries(1, 4, 64, "bf16", 1), ints(10), 4, 1, 64)


# ---- calls at the edges of what the faces allow -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40 + 5])
def test_windows_beyond_every_context(dtype, window):
    H, G, hd = 8, 2, 64
    c = Cache([90, 0], [20, 33], G, hd, 16, seed=21)
    rows = queries(53, H, hd, dtype, 22)
    assert torch.equal(prefill(c, rows, [90, 0], [20, 33], H, G, hd, window), prefill(c, rows, [90, 0], [20, 33], H, G, hd))
    pos = ints(109, 32)
    assert torch.equal(decode(c, rows[:2], pos, H, G, hd, window), decode(c, rows[:2], pos, H, G, hd))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("far", [2 ** 20, 2 ** 30, 2 ** 31 - 200])
def test_positions_far_behind_the_table(dtype, far):
    """A row sees what the table names of the keys before it, which is all of it, and walks no further."""
    H, G, hd = 8, 2, 64
    c = Cache([47], [1], G, hd, 16, seed=23)
    rows = queries(3, H, hd, dtype, 24)
    portion = prefill(c, rows, [far], [3], H, G, hd)
    single = decode(c, rows, ints(far, far + 1, far + 2), H, G, hd, req=ints(0, 0, 0))
    for i in range(3):
        for got in (portion, single):
            check(got[i:i + 1], rows[i:i + 1], c, [47], [1], H, G, hd)
    assert not prefill(c, rows, [far], [3], H, G, hd, window=20).any()
    assert not decode(c, rows, ints(far, far + 1, far + 2), H, G, hd, window=20, req=ints(0, 0, 0)).any()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 96])
def test_many_portions(dtype, hd):
    """More requests than a warp has lanes, some without rows, in tiles that end anywhere."""
    H, G, R = 4, 2, 171
    lens = [(7 * i) % 5 if i % 11 else 0 for i in range(R)]
    lens[40], lens[170] = 150, 90
    starts = [(13 * i) % 37 for i in range(R)]
    c = Cache(starts, lens, G, hd, 16, seed=25)
    rows = queries(sum(lens), H, hd, dtype, 26)
    check(prefill(c, rows, starts, lens, H, G, hd), rows, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("dtype", DT)
def test_calls_without_rows(dtype):
    from kllm_b200 import kernels
    H, G, hd = 4, 2, 64
    c = Cache([10], [1], G, hd, 16, seed=27)
    none = torch.zeros(0, H * hd, dtype=DT[dtype], device="cuda")
    flat = torch.zeros(0, dtype=torch.int32, device="cuda")
    decode(c, none, flat, H, G, hd, bound=1)
    kernels.attention_prefill_q8(none, none, c.k, c.v, c.ks, c.vs, ints(0, 0), ints(10), c.dev_table, 1, H, G, hd, 0, 0.1, 0)
    rows = queries(3, H, hd, dtype, 28)
    out = torch.full_like(rows, 7.0).contiguous()
    kernels.attention_prefill_q8(out, rows, c.k, c.v, c.ks, c.vs, ints(0), flat, c.dev_table[:0], 0, H, G, hd, 0, 0.1, 0)
    assert bool((out == 7.0).all())
    before = [t.clone() for t in (c.k.view(torch.uint8), c.ks)]
    kv = torch.zeros(0, G * hd, dtype=DT[dtype], device="cuda")
    kernels.rope_append_q8(none, none, kv, kv, None, flat, flat, ints(0, 0), c.dev_table, c.k, c.v, c.ks, c.vs, H, G, hd)
    torch.cuda.synchronize()
    assert torch.equal(before[0], c.k.view(torch.uint8)) and torch.equal(before[1].nan_to_num(3.0), c.ks.nan_to_num(3.0))


def test_two_graphs_that_share_their_workspace():
    """Contexts in several ranges and portions in several parts take room for their parts: two graphs of one memory pool are
    replayed in turn, on a stream of their own, beside eager calls."""
    from kllm_b200 import kernels
    H, G, hd = 32, 8, 128
    c = Cache([8000], [64], G, hd, 64, seed=29)
    one = Cache([20010], [1], 1, hd, 16, seed=30)
    assert kernels.decode_q8_parts(1, 1, 4, hd, 20011)[0] > 1 and kernels.prefill_q8_parts(64, 1, G, H // G, 8064, hd)[1] > 1
    rows, row = queries(64, H, hd, "bf16", 31), queries(1, 4, hd, "bf16", 32)
    q_start, start, pos = ints(0, 64), ints(8000), ints(20010)
    outs = [torch.zeros(64, H * hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 4 * hd, dtype=torch.bfloat16, device="cuda")]

    def portion(out):
        kernels.attention_prefill_q8(out, rows, c.k, c.v, c.ks, c.vs, q_start, start, c.dev_table, 1, H, G, hd, 0, 0.08, 8064)

    def single(out):
        kernels.attention_decode_q8(out, row, one.k, one.v, one.ks, one.vs, pos, None, one.dev_table, 4, 1, hd, 0, 0.08, 20011)
    eager = [torch.zeros_like(t) for t in outs]
    portion(eager[0]), single(eager[1])
    torch.cuda.synchronize()
    graphs, pool = [], torch.cuda.graph_pool_handle()
    for call, out in zip((portion, single), outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            call(out)
    side, again = torch.cuda.Stream(), [torch.zeros_like(t) for t in outs]
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for t in outs + again:
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
            graphs[1].replay()
        portion(again[0]), single(again[1])
        torch.cuda.current_stream().wait_stream(side)
        for got, eag, want in zip(outs, again, eager):
            assert torch.equal(got, want) and torch.equal(eag, want)


def test_stores_of_more_than_32_bits():
    """Pages whose bytes lie beyond 2^32 of a store: what is appended there is read from there."""
    from kllm_b200 import kernels
    H, G, hd, ps = 8, 8, 128, 64
    pages = (2 ** 32) // (G * ps * hd) + 40
    small = Cache([100], [30], G, hd, ps, seed=33)
    far = torch.tensor([[pages - 1, pages - 7, pages - 30]], dtype=torch.int32)
    k, v = (torch.zeros(pages, G, ps, hd, dtype=torch.uint8, device="cuda").view(plain.E4M3) for _ in range(2))
    ks, vs = (torch.ones(pages, G, device="cuda") for _ in range(2))
    x = [queries(130, G, hd, "bf16", 34 + i) for i in range(2)]
    pos = torch.arange(130, dtype=torch.int32, device="cuda")
    rows, turned = queries(130, H, hd, "bf16", 36), torch.zeros(130, H * hd, dtype=torch.bfloat16, device="cuda")
    outs = []
    for kc, vc, kss, vss, table in ((small.k, small.v, small.ks, small.vs, small.dev_table), (k, v, ks, vs, far.cuda())):
        kernels.rope_append_q8(turned, rows, x[0], x[1], table_of_angles(130, hd), pos, torch.zeros_like(pos), ints(0, 130), table, kc, vc,
                               kss, vss, H, G, hd)
        for dt in DT.values():
            q = turned.to(dt)
            out, one = torch.zeros_like(q), torch.zeros_like(q[:1])
            kernels.attention_prefill_q8(out, q, kc, vc, kss, vss, ints(0, 130), ints(0), table, 1, H, G, hd, 0, 0.09, 130)
            kernels.attention_decode_q8(one, q[129:], kc, vc, kss, vss, ints(129), None, table, H, G, hd, 0, 0.09, 130)
            outs.append((kc.view(torch.uint8)[table[0].long()], vc.view(torch.uint8)[table[0].long()], out, one))
    for near, there in zip(outs[:2], outs[2:]):
        assert bool(there[2].any())
        for i, (a, b) in enumerate(zip(near, there)):
            if i < 2:          # the last page's slots behind the 130th are not written
                a, b = (t.transpose(1, 2).reshape(3 * ps, G, hd)[:130] for t in (a, b))
            assert torch.equal(a, b)
    assert not bool(k.view(torch.uint8)[:pages - 40].any()) and not bool(v.view(torch.uint8)[:pages - 40].any())


def test_refuses_another_device_and_too_many_rows(monkeypatch):
    from kllm_b200 import kernels
    from kllm_b200.kernels import KernelError
    H, G, hd = 4, 1, 64
    c = Cache([10], [1], G, hd, 16, seed=37)
    rows, kv = queries(1, H, hd, "bf16", 38), queries(1, G, hd, "bf16", 39)
    calls = [lambda: decode(c, rows, ints(10), H, G, hd), lambda: prefill(c, rows, [10], [1], H, G, hd),
             lambda: kernels.rope_append_q8(rows, rows, kv, kv, None, ints(10), None, ints(0, 1), c.dev_table, c.k, c.v, c.ks, c.vs, H, G, hd)]
    many = torch.zeros(65536, H * hd, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError, match="at most 65535"):
        decode(c, many, torch.zeros(65536, dtype=torch.int32, device="cuda"), H, G, hd, req=torch.zeros(65536, dtype=torch.int32, device="cuda"))
    held = c.vs
    c.vs = held.cpu()
    for call in calls:
        with pytest.raises(KernelError, match="not on a CUDA device"):
            call()
    c.vs = held
    here = torch.cuda.current_device()
    with monkeypatch.context() as m:
        m.setattr(torch._C, "_cuda_getDevice", lambda: here + 1)
        for call in calls:
            with pytest.raises(KernelError, match="another than the current one"):
                call()
    for call in calls:
        call()


@pytest.mark.parametrize("dtype", DT)
def test_starts_outside_the_rows(dtype):
    """Portions that begin before the first row or end behind the last read and write nothing there."""
    from kllm_b200 import kernels
    H, G, hd = 4, 2, 64
    c = Cache([20, 20, 20], [40, 40, 40], G, hd, 16, seed=41)
    rows = queries(12, H, hd, dtype, 42)
    room = torch.full((36, H * hd), 7.0, dtype=rows.dtype, device="cuda")
    out = room[12:24]
    kernels.attention_prefill_q8(out, rows, c.k, c.v, c.ks, c.vs, ints(-9, 4, 8, 900), ints(20, 20, 20), c.dev_table, 3, H, G, hd, 0, 0.1, 60)
    assert bool((room[:12] == 7.0).all()) and bool((room[24:] == 7.0).all()) and bool((out != 7.0).any(dim=1).all())
    kept = [t.view(torch.uint8).clone() for t in (c.k, c.v)]
    kv = queries(12, G, hd, dtype, 43)
    pos = ints(*[3] * 12)
    kernels.rope_append_q8(rows, rows, kv, kv, None, pos, ints(*[0] * 12), ints(5, -3), c.dev_table, c.k, c.v, c.ks, c.vs, H, G, hd)
    assert torch.equal(kept[0], c.k.view(torch.uint8)) and torch.equal(kept[1], c.v.view(torch.uint8))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,rot,page,starts,lens", [
    (64, 32, 256, 256, 16, [0, 5, 31], [400, 92, 40]), (64, 64, 96, 48, 24, [7, 0], [600, 330]), (64, 64, 128, 0, 64, [70, 3, 0], [1, 440, 260]),
    (64, 64, 96, 40, 24, [7, 0], [600, 330])])
def test_append_many_numbers(dtype, H, G, hd, rot, page, starts, lens):
    """Calls of 2^24 numbers and more, which bfloat16 takes eight at a time where the rotary width is a multiple of 16."""
    n = sum(lens)
    assert n * (H + 2 * G) * hd >= 2 ** 24
    c = Cache(starts, lens, G, hd, page, seed=page + hd, fill=False)
    q, k, v = queries(n, H, hd, dtype, 1), queries(n, G, hd, dtype, 2, loud=5.0), queries(n, G, hd, dtype, 3)
    k[4, 7], k[9, hd + 3], v[12, 5], v[30, hd + 60], k[n - 1, 31] = math.inf, math.nan, -math.inf, math.nan, math.nan
    cs = table_of_angles(700, rot) if rot else None
    before = dict(key=(c.k.clone(), c.ks.clone()), value=(c.v.clone(), c.vs.clone()))
    q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
    check_append(c, before, q_out, q, k, v, cs, pos, starts, lens, H, G, hd)
    kept = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)]
    q2, _ = run_append(c, q, k, v, cs, starts, lens, H, G, hd, in_place=True)
    assert torch.equal(q2, q_out)
    for a, b in zip(kept, (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)):
        assert torch.equal(a.float().nan_to_num(-1.0), b.float().nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,rot,page,starts,lens", [(64, 64, 128, 128, 16, [3, 0], [400, 300]), (32, 32, 128, 128, 64, [9], [900]),
                                                         (32, 32, 96, 6, 16, [0], [500])])
@pytest.mark.parametrize("loud", [2.0, 2.0 ** -13])
def test_append_rounds_the_exact_rotation(dtype, H, G, hd, rot, page, starts, lens, loud):
    """Millions of keys without one that went to the wrong side of a border of e4m3, among its subnormals too (rows that one large
    number keeps small)."""
    c = Cache(starts, lens, G, hd, page, seed=5, fill=False)
    n = sum(lens)
    q, k, v = queries(n, H, hd, dtype, 1), queries(n, G, hd, dtype, 2, loud=loud), queries(n, G, hd, dtype, 3)
    if loud < 1:
        k[:, ::hd] = 1.5
    cs = table_of_angles(1600, rot)
    before = dict(key=(c.k.clone(), c.ks.clone()))
    q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
    kr, vr = plain.turned(k, cs, pos, G, hd), v.cpu().double().view(n, G, hd)
    want, scale, _ = plain.append(*before["key"], kr, vr, True, c.table, starts, lens)
    assert torch.equal(c.ks.cpu().double(), scale) and torch.equal(c.k.cpu().float().double(), want)
