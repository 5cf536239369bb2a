"""Plain forms of the block-scaled 8-bit cache's operators, and random caches for their tests."""

from __future__ import annotations

import math

import torch

SMALLEST = 2.0**-126
INVERSE_127 = torch.tensor(1.0) / 127  # in 32 bits


def append(cache, layer, blocks, offsets, k, v):
    """kv_append_int8 on CPU tensors by its definition, one (block, head) after another, in float32 steps."""
    kc, vc, ks, vs = cache
    nb, page, heads = kc.shape[0], kc.shape[2], kc.shape[3]
    groups = {}
    for i, (b, o) in enumerate(zip(blocks.tolist(), offsets.tolist())):
        if 0 <= b < nb and 0 <= o < page:
            groups.setdefault(b, []).append((o, i))
    for codes, scales, x in ((kc, ks, k.float()), (vc, vs, v.float())):
        for b, slots in groups.items():
            at, rows = [o for o, _ in slots], [i for _, i in slots]
            begins = 0 in at
            for h in range(heads):
                s0 = torch.tensor(0.0) if begins else scales[b, layer, h].clone()
                new = x[rows, h]
                if not new.isfinite().all() or s0.isnan():
                    s = torch.tensor(math.nan)
                else:
                    s = torch.maximum(torch.maximum(s0, new.abs().max() * INVERSE_127), torch.tensor(SMALLEST))
                    if s != s0 and not begins:
                        codes[b, layer, :, h] = torch.round(codes[b, layer, :, h].float() * (s0 / s)).to(torch.int8)
                scales[b, layer, h] = s
                codes[b, layer, at, h] = torch.round(new * (1 / s)).to(torch.int8) if s == s else torch.zeros((), dtype=torch.int8)


def values(codes, scales):
    """64-bit values of codes [..., page, heads, d] with scales [..., heads]."""
    return codes.double() * scales.double().unsqueeze(-2).unsqueeze(-1)


def random_cache(blocks, page, hkv, d, seed=0, layers=None, spread=2.0, device="cpu"):
    """Codes and scales of a pool ([blocks, layers, page, hkv, d]), or a layer slice; scales over 2^-spread .. 2^spread around 2^-6."""
    g = torch.Generator().manual_seed(seed)
    lead = (blocks,) if layers is None else (blocks, layers)
    codes = [(torch.randn((*lead, page, hkv, d), generator=g) * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [torch.exp2((torch.rand((*lead, hkv), generator=g) * 2 - 1) * spread - 6) for _ in range(2)]
    return [t.to(device) for t in (*codes, *scales)]


def poison(cache, tables, lengths, page):
    """NaN scales of every block that no sequence owns, the largest codes behind the last token of those that one does."""
    kc, vc, ks, vs = cache
    mine = torch.zeros(kc.shape[0], dtype=torch.bool)
    for r, n in enumerate(lengths):
        for p in range(-(-max(n, 0) // page)):
            block = int(tables[r, p])
            mine[block] = True
            for codes in (kc, vc):
                codes[block, n - p * page :] = 127
    for scales in (ks, vs):
        scales[~mine] = math.nan


def attention(q, cache, table, limits, scale, weight_unit=None):
    """64-bit attention of q [n, hq, d] over one sequence's blocks, row i seeing keys below limits[i].

    Returns (out, bound): bound is how far a kernel may be off that keeps scores, sums and
    products in 32 bits, rounds each weight p_j vs_j by at most weight_unit (default: half a
    step of fp16, 2^-11, or 2^-22 for float32, two parts of it), and the result by half a step
    of q's type:
    - a score is a sum of d products: off by (d + 8) 2^-24 of the sum of magnitudes (the
      8 for the scale factors and the exponent's argument), the probability by as much
      relative to it, in numerator and denominator alike: twice;
    - 2^-20 for the exponential, the sums over the keys and the joins of partial sums;
    - a weight is held relative to a power of two that puts the row's largest at 2^5 or more;
      one below 2^-14, fp16's smallest normal number, is off by up to 2^-25: 2^-30 of the
      largest, for every key whose weight is below 2^-19 of it.  (float32's second part is such a
      number beside weights below 2^-3: as much, for all its keys.)  Times codes of up to 128;
    - a key 126 binary orders below the largest weighs 0, as fp32's exponential does (its results
      below 2^-126, the smallest normal number, are 0): 2^(x - m) with m at most 1 above the
      largest x, so that the sum of these is at least 1/2 and a probability lost at most 2^-125.
    """
    kc, vc, ks, vs = cache
    page, hkv = kc.shape[1:3]
    n, hq, d = q.shape
    if weight_unit is None:
        weight_unit = 2.0**-22 if q.dtype == torch.float32 else 2.0**-11
    longest = max(max(limits), 0)
    ids = table[: -(-longest // page)].long()
    ids = torch.where((ids >= 0) & (ids < kc.shape[0]), ids, 0)

    def rows(x):  # [blocks, page, heads, ...] to [hq, t, ...]
        return x.flatten(0, 1)[:longest].transpose(0, 1).repeat_interleave(hq // hkv, 0)

    wide = q.double().transpose(0, 1)
    if longest == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    k, v = rows(values(kc[ids], ks[ids])), rows(values(vc[ids], vs[ids]))
    unit_v = rows(vs[ids].double()[:, None].expand(-1, page, -1)[..., None])[..., 0]  # [hq, t]
    scores = wide @ k.transpose(1, 2) * scale
    size = (wide.abs() @ k.abs().transpose(1, 2)) * abs(scale)
    hidden = torch.arange(longest, device=q.device) >= torch.tensor(limits, device=q.device)[:, None]
    scores = scores.masked_fill(hidden, -math.inf)
    size = size.masked_fill(hidden, 0.0).amax(-1, keepdim=True)
    p = torch.softmax(scores, -1)
    p = torch.where(hidden.all(-1)[:, None], 0.0, p)
    v_seen = torch.nan_to_num(v, nan=0.0)
    out, spread = p @ v_seen, p @ v_seen.abs()
    weights = p * torch.nan_to_num(unit_v, nan=0.0)[:, None]
    largest = weights.amax(-1, keepdim=True)
    small = (weights < largest * 2.0**-19) if q.dtype != torch.float32 else torch.ones_like(weights, dtype=torch.bool)
    floor = (small & ~hidden).sum(-1, keepdim=True) * largest * 128 * 2.0**-30
    lost = torch.where((p < 2.0**-125) & ~hidden, 2.0**-125, 0.0).double() @ v_seen.abs()
    unit = torch.finfo(q.dtype).eps / 2
    # Below the smallest normal number the type's step no longer shrinks: half of it is
    # smallest_normal * eps / 2 (fp16 2^-25), whatever the value.
    bound = unit * out.abs().clamp(min=torch.finfo(q.dtype).smallest_normal)
    bound = bound + (2 * (d + 8) * 2.0**-24 * size + 2.0**-20 + weight_unit) * spread + floor + lost
    return out.transpose(0, 1), bound.transpose(0, 1) + 1e-45
