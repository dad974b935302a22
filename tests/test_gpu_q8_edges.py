"""The cache in 8 bits where its kernels have to agree with the definition and with each other."""
import dataclasses
import math

import pytest
import torch

import q8_plain as plain
from test_gpu_q8 import DT, Cache, check, decode, ints, prefill, queries, run_append, table_of_angles

pytestmark = pytest.mark.gpu


# ---- rows that see no key --------------------------------------------------------------------------------------------------

@dataclasses.dataclass
class Rows:
    """A cache as one of its requests sees it."""
    c: Cache
    row: int = 0

    def __getattr__(self, name):
        return self.c.table[self.row:self.row + 1] if name == "table" else getattr(self.c, name)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("tokens,bound", [(40, 300), (12, 2000), (5, 3000), (2, 5000), (1, 20000)])
def test_decode_rows_without_keys_in_clusters(dtype, hd, tokens, bound):
    """Rows that see nothing beside rows that see some, and calls of such rows alone, with contexts in one part, in clusters of every size
    and in ranges of clusters."""
    from kllm_b200 import kernels
    H, G = 8, 8 if tokens > 2 else 1
    starts, lens = [(37 * i) % 300 for i in range(tokens)], [1] * tokens
    c = Cache(starts, lens, G, hd, 16, seed=tokens)
    q = queries(tokens, H, hd, dtype, seed=6)
    for every in (1, 2):
        pos = [-1 - i if i % every == 0 else s for i, s in enumerate(starts)]
        for _ in range(3):
            got = decode(c, q, ints(*pos), H, G, hd, bound=bound)
            assert not got[::every].any()
            for i in range(1, tokens, every) if every == 2 else ():
                check(got[i:i + 1], q[i:i + 1], Rows(c, i), [starts[i]], [1], H, G, hd)
    if tokens == 1:
        assert kernels.decode_q8_parts(1, G, H // G, hd, bound)[0] > 1


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("far", [30, 8000])
def test_rows_without_keys_are_zeros_whatever_their_queries(dtype, hd, far):
    H, G = 8, 2
    starts, lens = [far, -40, 20], [8, 30, 9]
    c = Cache(starts, lens, G, hd, 16, seed=5)
    c.table[2, 0] = -1                                     # places 0 to 15 of the last request
    c.dev_table = c.table.cuda()
    q = queries(sum(lens), H, hd, dtype, seed=6)
    q[8:38:2, 3] = math.nan
    q[9:38:2, 2 * hd + 1] = -math.inf
    got = prefill(c, q, starts, lens, H, G, hd)
    assert not got[8:38].any()
    single = decode(c, q, ints(*range(far, far + 8), *range(-40, -10), *range(20, 29)), H, G, hd, req=ints(*[0] * 8, *[1] * 30, *[2] * 9))
    assert not single[8:38].any()
    rest = [i for i in range(47) if not 8 <= i < 38]
    want, err = plain.attention(q[rest], c.k, c.v, c.ks, c.vs, c.table[[0, 2]], [far, 20], [8, 9], H, G, hd, 0, hd ** -0.5)
    for t in (got, single):
        assert bool(((t[rest].cpu().double() - want).abs() <= err).all())


# ---- loud scores -----------------------------------------------------------------------------------------------------------

PLACES = {"decode": ([99, 70, 200], [1, 1, 1]), "prefill": ([60, 0, 150], [40, 70, 51])}


def attend(form, c, q, starts, lens, H, G, hd):
    return decode(c, q, ints(*starts), H, G, hd) if form == "decode" else prefill(c, q, starts, lens, H, G, hd)


@pytest.mark.parametrize("form", PLACES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("loud", [2.0 ** 16, 2.0 ** 23, 2.0 ** 24, 2.0 ** 25, 2.0 ** 40, 2.0 ** 80])
def test_scores_beyond_what_float32_counts_in(form, dtype, hd, loud):
    """Scores near which neighbouring float32 numbers are whole units apart: one key has all the weight, where it is ahead by more than
    the scores' rounding and by 64 (weights of 2^-92), and the row is that key's values."""
    H, G = 8, 2
    starts, lens = PLACES[form]
    c = Cache(starts, lens, G, hd, 16, seed=5)
    q = queries(sum(lens), H, hd, dtype, seed=6, loud=loud)
    got = attend(form, c, q, starts, lens, H, G, hd).cpu().double().view(-1, H, hd)
    assert bool(torch.isfinite(got).all())
    k, v = plain.values(c.k, c.ks), plain.values(c.v, c.vs)
    half, at, alone = 2.0 ** -24 if dtype == "f32" else 2.0 ** -8, 0, 0
    for r, (old, new) in enumerate(zip(starts, lens)):
        j = torch.arange(old + new)
        page, slot = c.table[r].long()[j // 16], j % 16
        for i in range(new):
            for h in range(H):
                keys, vals = k[page[:old + i + 1], h // (H // G), slot[:old + i + 1]], v[page[:old + i + 1], h // (H // G), slot[:old + i + 1]]
                qh = q[at + i].cpu().double().view(H, hd)[h]
                s = keys @ qh * hd ** -0.5
                size = float((keys.abs() @ qh.abs()).max()) * hd ** -0.5
                top = torch.topk(s, min(2, s.numel()))
                if s.numel() > 1 and float(top.values[0] - top.values[1]) < 64 + size * 2.0 ** -16:
                    continue
                alone += 1
                want = vals[top.indices[0]]
                assert bool(((got[at + i, h] - want).abs() <= half * want.abs() + 2.0 ** -24 * vals.abs().amax(dim=0)).all())
        at += new
    assert alone > sum(lens) * H // 2


@pytest.mark.parametrize("form", PLACES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 96])
@pytest.mark.parametrize("top", range(22, 31))
@pytest.mark.parametrize("more", [2, 4, 6, 8, 16, 32])
def test_a_maximum_that_grows_where_numbers_are_far_apart(form, dtype, hd, top, more):
    """Two keys, tiles apart, at 2^top and a little more in units of log2; all the others are at 0.  The second one's weight is 2^-(their distance) of
    the first one's whatever the reference is, as far as float32 tells them apart: a distance below half a unit of 2^top's last place is any
    of 0 and that unit."""
    far = 130
    c = Cache([199], [1], 1, hd, 16, seed=1)
    k, v = (torch.zeros(200, hd) for _ in range(2))
    k[0, 0], k[far, 0], k[far, 1] = 256.0, 256.0, float(more)
    v[0], v[far] = 1.0, -1.0
    for store, rows in ((c.k, k), (c.v, v)):
        for j in range(200):
            store.view(torch.uint8)[int(c.table[0, j // 16]), 0, j % 16] = rows[j].to(plain.E4M3).view(torch.uint8).cuda()
    c.ks.fill_(1.0), c.vs.fill_(1.0)
    q = torch.zeros(1, hd)
    q[0, 0], q[0, 1] = 2.0 ** (top - 8), 1.0
    q = q.to(DT[dtype]).cuda()
    scale = 0.6931471805599453                              # its product with log2 e is 1 but for float32's rounding
    got = (decode(c, q, ints(199), 1, 1, hd, scale=scale, bound=1) if form == "decode" else prefill(c, q, [199], [1], 1, 1, hd, scale=scale))
    ulp = 2.0 ** max(top - 23, -9)
    out = lambda d: (1 - 2.0 ** d) / (1 + 2.0 ** d)  # noqa: E731
    lo, hi = out(more + 1.0 * ulp), out(max(more - 1.0 * ulp, 0.0))
    assert bool(torch.isfinite(got).all()) and bool((got.float() >= lo - 2.0 ** -8).all()) and bool((got.float() <= hi + 2.0 ** -8).all())


# ---- scales --------------------------------------------------------------------------------------------------------------

def cut(scale):
    """The power of two that the kernels take a scale for."""
    mantissa, exponent = torch.frexp(scale.abs().nan_to_num(math.inf, math.inf))
    exponent = torch.where(torch.isfinite(mantissa) & (mantissa > 0), exponent - 1, torch.where(mantissa > 0, 48, -48))
    return torch.ldexp(torch.ones_like(scale), exponent.clamp(-48, 48))


@pytest.mark.parametrize("form", PLACES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 96])
@pytest.mark.parametrize("which", ["ks", "vs"])
@pytest.mark.parametrize("odd", [0.0, 3.0, 2.0 ** -60, 2.0 ** -140, 2.0 ** 60, math.inf, math.nan])
def test_scales_that_the_append_does_not_leave(form, dtype, hd, which, odd):
    """Every form takes a scale for the power of two below it, 2^-48 to 2^48."""
    H, G = 8, 2
    starts, lens = PLACES[form]
    c = Cache(starts, lens, G, hd, 16, seed=5)
    held = c.table[c.table >= 0].long()
    getattr(c, which)[held[::3].cuda()] = odd
    q = queries(sum(lens), H, hd, dtype, seed=6)
    got = attend(form, c, q, starts, lens, H, G, hd)
    c.ks[held.cuda()], c.vs[held.cuda()] = cut(c.ks[held.cuda()]), cut(c.vs[held.cuda()])
    check(got, q, c, starts, lens, H, G, hd)


@pytest.mark.parametrize("form", PLACES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("spread", [3.0, 8.0])
@pytest.mark.parametrize("page", [16, 5])
def test_scales_of_keys_and_values_far_apart(form, dtype, hd, spread, page):
    """Pages whose keys' scales, and values', differ by more than a tile's step takes: the queries are as quiet as the keys are loud,
    so that no key decides alone."""
    H, G = 8, 2
    starts, lens = PLACES[form]
    c = Cache(starts, lens, G, hd, page, seed=5, spread=0.0)
    g = torch.Generator().manual_seed(9)
    for name in ("ks", "vs"):
        e = (torch.randn(c.ks.shape, generator=g) * spread).round().clamp(-30, 30) - 7
        setattr(c, name, torch.where(torch.isnan(getattr(c, name).cpu()), math.nan, torch.exp2(e)).cuda())
    q = queries(sum(lens), H, hd, dtype, seed=6, loud=2.0 ** (-2 * spread))
    check(attend(form, c, q, starts, lens, H, G, hd), q, c, starts, lens, H, G, hd)


# ---- append ---------------------------------------------------------------------------------------------------------------

def hold_append(c, before, k, v, cs, pos, starts, lens, G, hd):
    """Equality with the exact rotation rounded once, of every number and scale."""
    n = sum(lens)
    kr, vr = plain.turned(k[:n], cs, pos[:n], G, hd), v[:n].cpu().double().view(n, G, hd)
    for (store, scale), kept, is_key in (((c.k, c.ks), before[0], True), ((c.v, c.vs), before[1], False)):
        want, sc, _ = plain.append(*kept, kr, vr, is_key, c.table, starts, lens)
        assert torch.equal(scale.cpu().double().nan_to_num(-1.0), sc.nan_to_num(-1.0))
        assert torch.equal(store.cpu().float().double().nan_to_num(1e6), want.nan_to_num(1e6))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,rot", [(4, 2, 64, 64), (4, 2, 64, 6), (64, 64, 96, 48)])
@pytest.mark.parametrize("step", [0, 7])
@pytest.mark.parametrize("by", [1.0, 2.0 ** -9])
def test_a_pages_scale_follows_the_exact_rotation(dtype, H, G, hd, rot, step, by):
    """Keys that the rotation turns to 448 2^e and 2^-39 of it more, which float32 does not hold: they belong under the next scale.  As much
    less, they do not."""
    n = 32 if G < 64 else 960
    starts, lens = [step], [n]
    c = Cache(starts, lens, G, hd, 16, seed=3, fill=False)
    cs = torch.zeros(n + step, rot, device="cuda")
    cs[:, :rot // 2], cs[:, rot // 2:] = 1.0, 2.0 ** -20
    k = queries(n, G, hd, dtype, 2, loud=by)
    for g in range(G):
        for r in range(n):
            if r % 16 == 3 and g % 3 < 2:                 # a page's largest: just above, just below, none
                k[r, g * hd] = 448.0 * by
                k[r, g * hd + rot // 2] = (-2.0 ** -10 if g % 3 == 0 else 2.0 ** -10) * by
    q, v = queries(n, H, hd, dtype, 1), queries(n, G, hd, dtype, 3)
    before = [(c.k.clone(), c.ks.clone()), (c.v.clone(), c.vs.clone())]
    q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
    hold_append(c, before, k, v, cs, pos, starts, lens, G, hd)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,rot", [(8, 2, 64, 64), (4, 4, 128, 128), (3, 1, 32, 32), (10, 2, 96, 48), (8, 1, 256, 256), (4, 2, 64, 6),
                                        (8, 8, 64, 2)])
@pytest.mark.parametrize("page,starts,lens", [(16, [0], [1]), (16, [0, 5, 31], [40, 12, 2]), (5, [3, 0], [17, 9]), (64, [10, 100, 0], [1, 1, 1]),
                                              (256, [0, 130], [200, 150]), (1, [2, 0], [3, 4])])
def test_append_to_the_bit(dtype, H, G, hd, rot, page, starts, lens):
    for seed in range(3):
        c = Cache(starts, lens, G, hd, page, seed=page + hd + seed, fill=False)
        n = sum(lens)
        q, k, v = queries(n, H, hd, dtype, 7 * seed + 1), queries(n, G, hd, dtype, 7 * seed + 2, loud=5.0), queries(n, G, hd, dtype, 7 * seed + 3)
        cs = table_of_angles(400, rot)
        before = [(c.k.clone(), c.ks.clone()), (c.v.clone(), c.vs.clone())]
        q_out, pos = run_append(c, q, k, v, cs, starts, lens, H, G, hd)
        hold_append(c, before, k, v, cs, pos, starts, lens, G, hd)
