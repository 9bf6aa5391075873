"""CPU oracle of the 8-bit KV cache operators, in 64 bits and from their definitions: e4m3 codes with one power-of-two
scale per (block of slots, plane, KV head), attention over them, attention weights per token, and page eviction.
Test code only: no product path imports it."""
from __future__ import annotations

import math

import torch

# value of each of the 256 e4m3 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN
_E4M3 = torch.tensor([(-1.0 if c & 128 else 1.0) * (math.nan if c & 127 == 127 else (c & 7) * 2.0 ** -9 if c & 120 == 0 else
                                                     (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10)) for c in range(256)], dtype=torch.float64)


def values(kv: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """[pages,2,page,Hkv,D] float64 values of a pool (codes uint8 or float8) and its scale bytes [pages,2,page/block,Hkv]."""
    codes = kv.view(torch.uint8).long()
    block = kv.shape[2] // scales.shape[2]
    s = torch.where(scales == 0, torch.zeros((), dtype=torch.float64), 2.0 ** (scales.double() - 127))
    return _E4M3[codes] * s.repeat_interleave(block, 2)[..., None]


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of float64 x, ties to even, saturating at +-448; NaN stays."""
    a = x.abs().clamp(max=1e30)
    ex = torch.frexp(torch.where(a > 0, a, torch.ones_like(a)))[1].double() - 1
    step = 2.0 ** (ex.clamp(min=-6) - 3)
    y = (torch.round(x.clamp(-1e30, 1e30) / step) * step).clamp(-448, 448)
    return torch.where(torch.isnan(x), x, y)


def scale_exponent(amax: float) -> int:
    """Smallest e >= -126 with amax <= 448 * 2^e."""
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax / 448.0)[1] - 2)
        while amax > 448.0 * 2.0 ** e:
            e += 1
    return e


def append(kv: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos0, table) -> None:
    """The new tokens' K,V [B,T,Hkv,D] into copies of a pool, in place: kv float64 VALUES [pages,2,page,Hkv,D], scales
    int64 bytes.  pos0 and table per sequence (lists of slots and page ids)."""
    page, per_page = kv.shape[2], scales.shape[2]
    block = page // per_page
    for b in range(k.shape[0]):
        lo, hi = pos0[b], pos0[b] + k.shape[1]
        for s0 in range(lo // block * block, hi, block):
            pg, at = int(table[b][s0 // page]), s0 % page
            first, last = max(s0, lo), min(s0 + block, hi)
            for plane, new in ((0, k), (1, v)):
                rows = new[b, first - lo:last - lo].double()                                   # [n, Hkv, D]
                for h in range(kv.shape[3]):
                    x = rows[:, h]
                    before = int(scales[pg, plane, at // block, h]) - 127
                    fin = x[torch.isfinite(x)].abs()
                    e = scale_exponent(float(fin.max()) if fin.numel() else 0.0)
                    if first > s0:
                        e = max(e, before)
                        held = kv[pg, plane, at:at + first - s0, h]
                        kv[pg, plane, at:at + first - s0, h] = round_e4m3(held / 2.0 ** e) * 2.0 ** e
                    kv[pg, plane, at + first - s0:at + last - s0, h] = round_e4m3(x / 2.0 ** e) * 2.0 ** e
                    # codes behind the last new token keep their bits: what they stand for follows the scale
                    kv[pg, plane, at + last - s0:at + block, h] *= 2.0 ** (e - before)
                    scales[pg, plane, at // block, h] = e + 127


def attention(q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, sm: float, vscale: torch.Tensor | None = None):
    """One query row q [D] over K,V [n,D] (float64): (o, logits, lse, sum_j p_j |v_j|, max_j sum_d |q_d k_jd| sm) and, with
    the values' scales [n], max_j (p_j scale_j) * sum_j |v_j| / scale_j."""
    if K.shape[0] == 0:
        z = torch.zeros(q.shape[0], dtype=torch.float64)
        return (z, torch.zeros(0, dtype=torch.float64), -math.inf, z.clone(), 0.0) + (() if vscale is None else (z.clone(),))
    x = K @ q.double() * sm
    lse = torch.logsumexp(x, 0)
    p = torch.exp(x - lse)
    got = p @ V, x, float(lse), p @ V.abs(), float((K.abs() @ q.double().abs()).max() * sm)
    return got if vscale is None else got + ((p * vscale).max() * (V.abs() / vscale[:, None]).sum(0),)


def accumulate(scores, lse, weights, lens, decay):
    w = weights.double().clone()
    for b, n in enumerate(lens):
        z = lse[b].double()
        p = torch.exp(scores[b, :, :n].double() - z[:, None])
        w[b, :n] = decay * w[b, :n] + torch.where(torch.isinf(z[:, None]), torch.zeros((), dtype=torch.float64), p).sum(0)
    return w


def _order(x: float):
    """Sort key of a page weight: NaN above everything."""
    return math.inf if math.isnan(x) else x, math.isnan(x)


def evict(weights, table, lens, keep, page, sink, recent):
    """(weights, table, lens) after eviction; plain Python over lists."""
    weights, table, lens = weights.clone(), table.clone(), lens.clone()
    for r in range(weights.shape[0]):
        n = int(lens[r])
        used = -(-n // page)
        if used <= keep:
            continue
        w = weights[r, :n].clone()
        heavy = [float(w[i * page:(i + 1) * page].double().sum().float()) for i in range(used)]
        middle = sorted(range(sink, used - recent), key=lambda i: ([-c for c in _order(heavy[i])], i))
        stay = sorted(list(range(sink)) + middle[:keep - sink - recent] + list(range(used - recent, used)))
        gone = sorted(set(range(used)) - set(stay))
        table[r, :used] = table[r, torch.tensor(stay + gone, dtype=torch.long)]
        moved = torch.cat([w[i * page:(i + 1) * page] for i in stay])
        weights[r, :n] = 0
        weights[r, :moved.numel()] = moved
        lens[r] = moved.numel()
    return weights, table, lens
