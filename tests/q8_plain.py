"""The paged cache in 8 bits in plain operations and 64 bits, request by request, for the tests of its kernels, with what
the kernels' roundings may add up to."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def exponent_for(amax: float) -> int:
    """The smallest e in [-48, 48] with amax <= 448 * 2^e."""
    e = -48
    while e < 48 and amax > math.ldexp(448.0, e):
        e += 1
    return e


def nearest(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 numbers next to x (float64), as float64; ties to even, +-448 at most, NaN stays."""
    mag = x.abs().clamp(min=2.0 ** -6)
    mantissa, exponent = torch.frexp(mag)            # [0.5, 1) * 2^exponent: steps of 2^(exponent - 4)
    step = torch.ldexp(torch.ones_like(mag), exponent - 4)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def values(store: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return store.cpu().float().double() * scale.cpu().double()[:, :, None, None]


def turned(x, cos_sin, positions, heads, hd):
    """rotate_half of the first rot dims of every head, float64 [n, heads, hd]."""
    x = x.cpu().double().view(x.shape[0], heads, hd).clone()
    if cos_sin is None:
        return x
    rot = cos_sin.shape[1]
    half = rot // 2
    cs = cos_sin.cpu().double()[positions.cpu().long().clamp(0, cos_sin.shape[0] - 1)][:, None]
    a, b = x[..., :half].clone(), x[..., half:rot].clone()
    x[..., :half] = a * cs[..., :half] - b * cs[..., half:]
    x[..., half:rot] = b * cs[..., :half] + a * cs[..., half:]
    return x


def append(store, scale, key_rows, value_rows, is_key, table, starts, lens):
    """float64 (numbers in e4m3 units, scales) after rows [n, G, hd] of requests' portions joined the pages; rows whose key
    or value is not finite are stored as NaN keys and zero values.  Also the units' places that were written."""
    out, sc = store.cpu().float().double().clone(), scale.cpu().double().clone()
    written = torch.zeros(out.shape, dtype=torch.bool)
    G, ps = store.shape[1], store.shape[2]
    fine = torch.isfinite(key_rows).all(dim=2) & torch.isfinite(value_rows).all(dim=2)      # [n, G]
    rows = key_rows if is_key else value_rows
    at = 0
    for r, (old, new) in enumerate(zip(starts, lens)):
        for lp in range(old // ps, -(-(old + new) // ps)):
            page = int(table[r][lp])
            lo, hi = max(old, lp * ps), min(old + new, (lp + 1) * ps)
            if not (0 <= page < store.shape[0]):
                continue
            for g in range(G):
                x, ok = rows[at + lo - old:at + hi - old, g], fine[at + lo - old:at + hi - old, g]
                amax = float(x[ok].abs().max()) if bool(ok.any()) else 0.0
                e = exponent_for(amax)
                kept = lo - lp * ps
                if kept:
                    before = int(math.log2(float(sc[page, g])))
                    if before >= e:
                        e = before
                    else:
                        out[page, g, :kept] = nearest(out[page, g, :kept] * math.ldexp(1.0, before - e))
                sc[page, g] = math.ldexp(1.0, e)
                y = nearest(x * math.ldexp(1.0, -e))
                y[~ok] = math.nan if is_key else 0.0
                out[page, g, kept:hi - lp * ps] = y
                written[page, g, kept:hi - lp * ps] = True
        at += new
    return out, sc, written


def attention(q, kcache, vcache, kscale, vscale, table, starts, lens, H, G, hd, window, scale):
    """(out, what the roundings may do to it) float64 [n, H*hd] of requests' portions (rows in order).

    The bound.  Keys, values and queries enter the products exactly (a float32 query as three float16: 2^-33).  A score in
    units of log2 is a sum in float32 whose partial sums are rounded or cut once per 16 products and part, each time by at
    most 2^-23 of the sum of the terms' magnitudes S = scale log2(e) sum |q k|; its factors, the reference and the exponent
    of the page's scale join in four float32 roundings, each of at most 2^-24 of 2 S, 15 and the exponents' size.  That
    error, times ln 2, is the weight's, with 2^-22 of the exponential and the weight's own rounding: float16, 2^-11,
    beside float32 queries two of them, 2^-22.  Weights enter numerator and denominator.  The sums over the keys are cut by
    2^-23 once per 16 keys, and in some 16 places where parts are joined.  Weights below 2^-32 of the row's largest are lost.
    Then the output's rounding."""
    wide = q.dtype == torch.float32
    kd, vd = values(kcache, kscale), values(vcache, vscale)
    exponents = torch.log2(vscale.cpu().double()).nan_to_num(0.0, 0.0, 0.0)
    q = q.cpu().double()
    n, ps, gs = q.shape[0], kcache.shape[2], H // G
    out = torch.zeros(n, H, hd, dtype=torch.float64)
    err = torch.zeros(n, H, hd, dtype=torch.float64)
    half = 2.0 ** -24 if wide else 2.0 ** -8
    at = 0
    for r, (old, new) in enumerate(zip(starts, lens)):
        j = torch.arange(max(old + new, 0))
        row = torch.as_tensor(table[r]).long()
        page = torch.where(j // ps < row.numel(), row[(j // ps).clamp(max=row.numel() - 1)], torch.full_like(j, -1))
        there = (page >= 0) & (page < kcache.shape[0])
        page = page.clamp(0, kcache.shape[0] - 1)
        for i in range(new):
            p = old + i
            seen = there & (j <= p)
            if window:
                seen = seen & (j > p - window)
            if p < 0 or not bool(seen.any()):
                continue
            where, slot = page[seen], j[seen] % ps
            for g in range(G):
                ks, vs = kd[where, g, slot], vd[where, g, slot]
                heads = slice(g * gs, (g + 1) * gs)
                qs = q[at + i].view(H, hd)[heads]
                w = torch.softmax((qs @ ks.T) * scale, dim=1)
                o = w @ vs
                S = (qs.abs() @ ks.abs().T).amax(dim=1, keepdim=True) * abs(scale) * 1.4427
                e = float(exponents[where, g].abs().max())
                dz = S * 2.0 ** -23 * (hd // 16) * (3 if wide else 1) + 4 * (2 * S + 15 + e) * 2.0 ** -24
                dw = dz * math.log(2.0) + 2.0 ** -22 + (2.0 ** -22 if wide else 2.0 ** -11)
                sums = (math.ceil(ks.shape[0] / 16) + 16) * 2.0 ** -23
                out[at + i, heads] = o
                err[at + i, heads] = half * o.abs() + (w @ vs.abs()) * (2 * dw + sums) * (1 + half) \
                    + ks.shape[0] * 2.0 ** -32 * vs.abs().amax(dim=0)
        at += new
    return out.view(n, H * hd), err.view(n, H * hd)
