"""Plain 64-bit forms of the 8-bit KV cache's operators, and random caches for their tests."""

from __future__ import annotations

import math

import torch

LARGEST = 448.0


def quantise(x):
    """(codes, scale bytes) of the rows x[..., :], by the definition: the smallest power of two 2^e, e >= -127, with
    amax <= 448 * 2^e over the finite values, and the nearest code of x / 2^e (ties to even), NaN for what is not finite."""
    wide = x.double()
    amax = torch.where(torch.isfinite(wide), wide, 0.0).abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)
    e = torch.where(mantissa > LARGEST / 512, exponent - 8, exponent - 9)
    e = torch.where(amax > 0, e, -127).clamp(min=-127).long()
    scale = ((e + 1023) << 52).view(torch.float64)
    y = torch.where(torch.isfinite(wide), wide / scale[..., None], math.nan)
    return y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def values(codes, scales):
    return codes.double() * scales.double()[..., None]


def random_cache(blocks, page, hkv, d, seed=0, layers=None, spread=3, device="cpu"):
    """Codes and scales of a pool ([blocks, layers, page, hkv(, d)], or a layer slice), scales over 2^-spread .. 2^spread."""
    g = torch.Generator().manual_seed(seed)
    shape = (blocks, page, hkv, d) if layers is None else (blocks, layers, page, hkv, d)
    out = []
    for _ in range(2):
        out.append((torch.randn(shape, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn))
    for _ in range(2):
        bytes_ = torch.randint(120 - spread, 121 + spread, shape[:-1], generator=g)
        out.append(bytes_.to(torch.uint8).view(torch.float8_e8m0fnu))
    return [t.to(device) for t in out]


def tables_for(lengths, page, seed=0, spare=3, pad=-1):
    """Random page tables of the given lengths: (int32 [rows, width], blocks of the pool)."""
    g = torch.Generator().manual_seed(seed + 1000)
    need = [-(-max(n, 0) // page) for n in lengths]
    perm = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    tables = torch.full((len(lengths), max(need + [1])), pad, dtype=torch.int32)
    used = 0
    for r, n in enumerate(need):
        tables[r, :n] = perm[used : used + n]
        used += n
    return tables, sum(need) + spare


def poison(cache, tables, lengths, page):
    """NaN codes and scales in every slot that no sequence owns, so that reading one shows."""
    kc, vc, ks, vs = cache
    live = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for r, n in enumerate(lengths):
        for p in range(-(-max(n, 0) // page)):
            live[int(tables[r, p]), : n - p * page] = True
    dead = ~live
    for codes, scales in ((kc, ks), (vc, vs)):
        codes.view(torch.uint8)[dead] = 0x7F
        scales.view(torch.uint8)[dead] = 0xFF


def attention(q, cache, table, limits, scale, p_unit):
    """64-bit attention of q [n, hq, d] over one sequence's pages, row i seeing keys below limits[i].

    Returns (out, bound): bound is how far a kernel may be off that keeps scores, sums
    and products in 32 bits and rounds each probability by at most p_unit, and the
    result by half a step of q's type:
    - a score is a sum of d products: off by (d + 8) 2^-24 of the sum of magnitudes (the
      8 for the scale factors and the exponent's argument), the probability by as much
      relative to it, in numerator and denominator alike: twice;
    - 2^-20 for the exponential, the sums over the keys and the joins of partial sums (each
      partial sum of at most some hundred terms, 2^-24 each, errors of both signs).
    """
    kc, vc, ks, vs = cache
    page, hkv = kc.shape[1:3]
    n, hq, d = q.shape
    longest = max(max(limits), 0)
    ids = table[: -(-longest // page)].long()
    ids = torch.where((ids >= 0) & (ids < kc.shape[0]), ids, 0)

    def rows(codes, scales):
        x = values(codes.view(torch.uint8)[ids].view(codes.dtype), scales.view(torch.uint8)[ids].view(scales.dtype))
        return x.flatten(0, 1)[:longest].transpose(0, 1).repeat_interleave(hq // hkv, 0)  # [hq, t, d]

    wide = q.double().transpose(0, 1)
    if longest == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    k, v = rows(kc, ks), rows(vc, vs)
    scores = wide @ k.transpose(1, 2) * scale
    size = (wide.abs() @ k.abs().transpose(1, 2)) * abs(scale)
    hidden = torch.arange(longest, device=q.device) >= torch.tensor(limits, device=q.device)[:, None]
    scores = scores.masked_fill(hidden, -math.inf)
    size = size.masked_fill(hidden, 0.0).amax(-1, keepdim=True)
    p = torch.softmax(scores, -1)
    p = torch.where(hidden.all(-1)[:, None], 0.0, p)
    v_seen = torch.nan_to_num(v, nan=0.0)
    out, spread = p @ v_seen, p @ v_seen.abs()
    unit = torch.finfo(q.dtype).eps / 2
    # Below the smallest normal number the type's step no longer shrinks: half of it is
    # smallest_normal * eps / 2 (fp16 2^-25), whatever the value.
    bound = unit * out.abs().clamp(min=torch.finfo(q.dtype).smallest_normal) + (2 * (d + 8) * 2.0**-24 * size + 2.0**-20 + p_unit) * spread
    return out.transpose(0, 1), bound.transpose(0, 1) + 1e-30


def assert_within(got, want, bound):
    off = (got.double() - want).abs() - bound
    bad = ~(off <= 0)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst by {off[bad].max().item():.3g} at {bad.nonzero()[0].tolist()}"
