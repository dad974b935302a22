"""How far the attention kernels of the cache in 8 bits are from 64 bits beside float32 queries, held against float32 arithmetic that
adds one term after another.

Why that is a bound.  Float32 arithmetic rounds n times for a sum of n terms, by at most half a unit in the last place of the sum so far.
The tensor core takes 16 products at a time and cuts (up to a whole unit, always towards zero), once for each part of the
operands.  Added up in registers after every 32 products of a score, six cuts are of a sum of 32 terms and hd / 32 roundings of the
whole sum: rms 2.1 units at 256 dims where the long sum in the tensor core has 14 and float32 arithmetic 4.5 (simulated; 2.0, 7.4, 3.4
at 128 dims; 1.9, 3.6, 2.4 at 64).  Over keys, with a rounding per tile of 16 to 64 keys, the cuts of a tile stay in the tile.  Weights bring 2^-22
each from their exponential and their two float16 parts, 4 units, which scores of some size outweigh.  So the root mean square of the error has to be at most
1.25 times that of float32 arithmetic."""
import pytest
import torch

import q8_plain as plain

pytestmark = pytest.mark.gpu


class Keys:
    """One request's pages in their order, numbers in e4m3 with exponents of their own."""

    def __init__(self, ctx, G, hd, ps, seed, positive=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        pages = -(-ctx // ps)
        draw = lambda: torch.randn(pages, G, ps, hd, generator=g, device="cuda") * 100  # noqa: E731
        k, v = draw().clamp(-448, 448), draw().clamp(-448, 448)
        self.k, self.v = k.to(plain.E4M3), (v.abs() if positive else v).to(plain.E4M3)
        self.ks, self.vs = (torch.exp2(torch.randint(-8, -5, (pages, G), generator=g, device="cuda").float()) for _ in range(2))
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        self.ctx, self.G, self.hd = ctx, G, hd

    def rows(self, which):
        """float32 [G, ctx, hd], exact"""
        store, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        return (store.float() * scale[:, :, None, None]).transpose(0, 1).reshape(self.G, -1, self.hd)[:, :self.ctx]


def exact(c, q, H, scale, last):
    """float64 [n, H * hd]: row i sees the keys up to last[i]"""
    n, G, hd = q.shape[0], c.G, c.hd
    q = q.double().view(n, G, H // G, hd).permute(1, 0, 2, 3)
    s = torch.einsum("gnhd,gkd->gnhk", q, c.rows("k").double()) * scale
    hidden = torch.arange(c.ctx, device="cuda")[None, :] > last[:, None]
    w = torch.softmax(s.masked_fill(hidden[None, :, None, :], -torch.inf), dim=-1)
    return torch.einsum("gnhk,gkd->gnhd", w, c.rows("v").double()).permute(1, 0, 2, 3).reshape(n, H * hd)


def one_by_one(c, q, H, scale, last):
    """The same in float32, a term after the other."""
    n, G, hd = q.shape[0], c.G, c.hd
    q = q.view(n, G, H // G, hd).permute(1, 0, 2, 3)
    k, v = c.rows("k"), c.rows("v")
    s = torch.zeros(G, n, H // G, c.ctx, device="cuda")
    for d in range(hd):
        s += q[..., d, None] * k[:, None, None, :, d]
    s *= scale
    hidden = torch.arange(c.ctx, device="cuda")[None, :] > last[:, None]
    s.masked_fill_(hidden[None, :, None, :], -torch.inf)
    w = torch.exp(s - s.amax(dim=-1, keepdim=True))
    total, out = torch.zeros(G, n, H // G, device="cuda"), torch.zeros(G, n, H // G, hd, device="cuda")
    for j in range(c.ctx):
        total += w[..., j]
        out += w[..., j, None] * v[:, None, None, j]
    return (out / total[..., None]).permute(1, 0, 2, 3).reshape(n, H * hd)


def kernel(form, c, q, H, scale, last):
    from kllm_b200 import kernels
    ints = lambda v: torch.as_tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out, n = torch.empty_like(q), q.shape[0]
    if form == "decode":          # a bound of one key: one CTA walks a whole context
        kernels.attention_decode_q8(out, q, c.k, c.v, c.ks, c.vs, ints(last), ints([0] * n), c.table, H, c.G, c.hd, 0, scale, 1)
    else:
        kernels.attention_prefill_q8(out, q, c.k, c.v, c.ks, c.vs, ints([0, n]), ints([int(last[0])]), c.table, 1, H, c.G, c.hd, 0,
                                     scale, c.ctx)
    return out


def hold(form, c, q, H, scale, last):
    want = exact(c, q, H, scale, last)
    rms = lambda t: float((t.double() - want).square().mean().sqrt())  # noqa: E731
    here, other = rms(kernel(form, c, q, H, scale, last)), rms(one_by_one(c, q, H, scale, last))
    assert here <= 1.25 * other, f"{here:.3g} from 64 bits, float32 arithmetic {other:.3g}"


@pytest.mark.parametrize("form", ["decode", "prefill"])
@pytest.mark.parametrize("H,G,hd", [(8, 8, 64), (8, 2, 128), (4, 4, 160), (8, 2, 192), (4, 4, 256), (16, 2, 256)])
def test_scores_beside_float32_arithmetic(form, H, G, hd):
    """Scores of some size: their error is the weights'."""
    c = Keys(400, G, hd, 16, seed=hd)
    n = 12
    q = torch.randn(n, H * hd, generator=torch.Generator().manual_seed(hd + 1)).cuda()
    hold(form, c, q, H, 3.5 / hd ** 0.5, torch.arange(400 - n, 400, device="cuda"))


@pytest.mark.parametrize("H,G,hd", [(8, 2, 128), (4, 4, 160), (8, 2, 192), (4, 4, 256), (16, 2, 256)])
def test_portions_are_as_near_as_single_tokens(H, G, hd):
    """The same rows as single tokens and as a portion: their scores are sums of the same sums, of 32 or of 16 products, which are the error
    at scores of this size.  So they are within half as much again of each other."""
    c, n = Keys(400, G, hd, 16, seed=hd), 12
    q = torch.randn(n, H * hd, generator=torch.Generator().manual_seed(hd + 1)).cuda()
    last, scale = torch.arange(400 - n, 400, device="cuda"), 3.5 / hd ** 0.5
    want = exact(c, q, H, scale, last)
    one, portion = (float((kernel(form, c, q, H, scale, last).double() - want).square().mean().sqrt()) for form in ("decode", "prefill"))
    assert portion <= 1.5 * one, f"{portion:.3g} from 64 bits, single tokens {one:.3g}"


@pytest.mark.parametrize("form,H,G,hd,ctx", [("decode", 4, 4, 128, 16001), ("decode", 8, 2, 64, 16001), ("decode", 32, 2, 64, 9000),
                                             ("decode", 4, 1, 256, 9000), ("decode", 2, 2, 32, 30000), ("prefill", 8, 2, 64, 9000),
                                             ("prefill", 4, 1, 256, 5000)])
def test_long_contexts_beside_float32_arithmetic(form, H, G, hd, ctx):
    """Thousands of values of one sign: what a sum cuts off adds up."""
    c = Keys(ctx, G, hd, 64, seed=hd, positive=True)
    n = 3
    q = torch.randn(n, H * hd, generator=torch.Generator().manual_seed(hd + 1)).cuda()
    hold(form, c, q, H, 0.5 / hd ** 0.5, torch.arange(ctx - n, ctx, device="cuda"))


@pytest.mark.parametrize("H,G,hd,ctx", [(4, 4, 96, 131072), (4, 4, 160, 100000), (4, 4, 256, 60000)])
def test_long_contexts_of_bfloat16_portions(H, G, hd, ctx):
    """What is left of the error beside the output's rounding: weights, 2^-12 each, of many thousand keys, and a float32 rounding a tile, which
    are 2^-19 together.  A sum of the tensor core that all keys join is cut by up to 2^-23 at every sixteen of them, to one side."""
    c, n = Keys(ctx, G, hd, 64, seed=hd, positive=True), 16
    q = (torch.randn(n, H * hd, generator=torch.Generator().manual_seed(1)) * 0.05).bfloat16().cuda()
    last = torch.arange(ctx - n, ctx, device="cuda")
    want = exact(c, q, H, hd ** -0.5, last)
    far = lambda t: float(((t.double() - want) / want).square().mean().sqrt())  # noqa: E731
    here, rounding = far(kernel("prefill", c, q, H, hd ** -0.5, last)), far(want.bfloat16())
    assert here <= 1.01 * rounding, f"{here:.4g} from 64 bits, rounding alone {rounding:.4g}"


@pytest.mark.parametrize("form", ["decode", "prefill"])
@pytest.mark.parametrize("H,G,hd", [(2, 2, 64), (4, 1, 64), (2, 1, 128)])
def test_queries_keep_all_their_bits(form, H, G, hd):
    """Two keys whose scores differ by 1 / 2 in all, and only through the last bits of the queries' 24: with 22 of them (two float16 parts)
    the weights were 1 / 2 each.  Every sum here is a float32 number; the scores, near 2048, are rounded by 2^-13 on the way."""
    c = Keys(2, G, hd, 16, seed=1)
    k = torch.zeros(1, G, 16, hd)
    k[:, :, 0, 0::4], k[:, :, 0, 1::4] = 1.0, -1.0         # sees 1 against 1 + 2^-12 + 2^-23 of every four dims,
    k[:, :, 1, 2::4], k[:, :, 1, 3::4] = 1.0, -1.0         # ... 1 against 1 + 2^-12
    c.k = k.to(plain.E4M3).cuda()
    c.ks.fill_(1.0)
    q = torch.ones(1, H, hd)
    q[..., 1::4] += 2.0 ** -12 + 2.0 ** -23
    q[..., 3::4] += 2.0 ** -12
    q = q.view(1, H * hd).cuda()
    scale = 2.0 ** 22 / (hd // 4)                          # the scores are -(1024 + 1 / 2) and -1024
    last = torch.tensor([1], device="cuda")
    want = exact(c, q, H, scale, last)
    size = c.rows("v").abs().amax().double()
    assert bool(((kernel(form, c, q, H, scale, last).double() - want).abs() <= size * 4 * 2048 * 1.4427 * 2.0 ** -24).all())
