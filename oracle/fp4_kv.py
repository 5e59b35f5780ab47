"""CPU oracle of the 4-bit KV cache and of page copies - TEST INFRASTRUCTURE ONLY.

Written from the format's definition in 64 bits (microserve_b200/csrc/fp4_kv.cuh):
codes e2m1, element 2i in the low nibble of byte i; one scale byte per 16 elements, an
unsigned float with 5 exponent and 3 mantissa bits (fp16 bits byte << 7); scale =
min(rn(max|x| / 6), 10240); code = rn(x / scale), saturating at 6; ties to even.
Caches: codes [NB, Hkv, BS, 64], scales [NB, Hkv, BS, 8], uint8.
"""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def scale_value(b: torch.Tensor) -> torch.Tensor:
    """fp64 value of scale bytes (248: inf, above: NaN)."""
    return (b.to(torch.int16) << 7).view(torch.float16).double()


def _nearest(v: torch.Tensor, points: torch.Tensor) -> torch.Tensor:
    """Index of the point nearest to v >= 0, ties to the even index (points ascending)."""
    mid = (points[1:] + points[:-1]) / 2  # exact: few bits
    hi = torch.bucketize(v, mid, right=True)
    lo = torch.bucketize(v, mid)
    return torch.where(hi % 2 == 0, hi, lo)


def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp16 [..., 128] -> (codes [..., 64], scale bytes [..., 8])."""
    g = x.double().unflatten(-1, (8, 16))
    nan = g.isnan().any(-1)
    g = g.nan_to_num(0.0).clamp(-65504, 65504)
    scales = scale_value(torch.arange(227, dtype=torch.uint8))  # up to 10240
    sc = _nearest(g.abs().amax(-1) / 6, scales)
    # a / 6 in 64 bits is within 2^-53 of the quotient; a midpoint has 5 bits and a 11, so
    # equality with a midpoint and its order are those of the exact quotient
    s = scales[sc]
    q = torch.where(s[..., None] > 0, g.abs() / s.clamp_min(2.0 ** -17)[..., None], torch.zeros_like(g))
    c = _nearest(q, GRID) + 8 * torch.signbit(x).unflatten(-1, (8, 16)).long()
    c = torch.where(nan[..., None], torch.zeros_like(c), c).flatten(-2)
    sc = torch.where(nan, torch.full_like(sc, 255), sc)
    return (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8), sc.to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp64 values [..., 128]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = GRID[c % 8] * (1 - 2 * (c // 8)).double()
    v = torch.where(c == 8, torch.full_like(v, -0.0), v)
    return (v.unflatten(-1, (8, 16)) * scale_value(scales)[..., None]).flatten(-2)


def store(k, v, kc, vc, ks, vs, slots) -> None:
    BS = kc.shape[2]
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        codes, sc = encode(x)
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                c[slot // BS, :, slot % BS] = codes[t]
                s[slot // BS, :, slot % BS] = sc[t]


def gather(c, s, table, n) -> torch.Tensor:
    """fp64 [Hkv, n, 128] of the first n tokens of a sequence."""
    BS = c.shape[2]
    pos = torch.arange(n)
    page = table.long()[pos // BS]
    return decode(c[page, :, pos % BS], s[page, :, pos % BS]).transpose(0, 1)


def attend(q, kc, vc, ks, vs, table, n, scale):
    """Queries q [Q, Hq, 128] at positions n - Q .. n - 1 over the first n cached tokens: (o, a), o the
    outputs and a the sums of p |v| that their error bounds are made of, both fp64 [Q, Hq, 128].
    A query that sees nothing gives 0."""
    Q, Hq, D = q.shape
    Hkv = kc.shape[1]
    o = torch.zeros(Q, Hq, D, dtype=torch.float64)
    a = torch.zeros_like(o)
    if n <= 0:
        return o, a
    k, v = gather(kc, ks, table, n), gather(vc, vs, table, n)
    G = Hq // Hkv
    at = n - Q + torch.arange(Q)
    seen = torch.arange(n)[None, :] <= at[:, None]
    for h in range(Hq):
        s = q[:, h].double() @ k[h // G].t() * scale
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1)
        p = torch.where((at >= 0)[:, None], p, torch.zeros_like(p))
        o[:, h] = p @ v[h // G]
        a[:, h] = p @ v[h // G].abs()
    return o, a


def decode_attention(q, kc, vc, ks, vs, lens, tables, scale):
    parts = [attend(q[b:b + 1], kc, vc, ks, vs, tables[b], int(lens[b]), scale) for b in range(q.shape[0])]
    return torch.cat([x[0] for x in parts]), torch.cat([x[1] for x in parts])


def prefill_attention(q, kc, vc, ks, vs, tables, cu, kv_lens, scale):
    parts = [attend(q[cu[s]:cu[s + 1]], kc, vc, ks, vs, tables[s], int(kv_lens[s]), scale)
             for s in range(len(kv_lens))]
    return torch.cat([x[0] for x in parts]), torch.cat([x[1] for x in parts])
