"""Edges of the 8-bit KV cache operators: results to the last bit of their type, the ends of the ranges of scales, weights and
starts, and calls that come after an eviction.  Against the definitions in 64 bits (oracle/kv8_oracle.py)."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import kv8_oracle as K8

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LOG2E = 1.4426950408889634


@pytest.fixture(scope="module")
def T():
    import tidaldecode_b200.ops as ops
    return ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _half_step(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half the distance between the type's numbers in x's binade (of the subnormal numbers below the smallest normal one)."""
    info = torch.finfo(dtype)
    e = torch.frexp(x.abs().clamp(min=info.smallest_normal))[1].double() - 1
    return 2.0 ** e * info.eps / 2


# --------------------------------------------------------------- attention: last bits
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 12, 1), (128, 16, 1), (128, 8, 1), (64, 7, 1), (64, 6, 2), (128, 3, 3)])
def test_attention_rounds_16_bit_results_once(T, dt, D, Hq, Hkv):
    """A 16-bit result is the 64-bit one rounded to its type: off by half a step and by what 32-bit arithmetic loses.  The
    softmax weights have no rounding of their own beyond that: held in two fp16 terms they are off by 2^-22.  With
    dot = max_j sum_d |q_d k_jd| sm and A = sum_j p_j |v_j|, for up to 33 tokens:
        dx = 20 * 2^-23 * dot           logits (8 to 16 fp32 additions of exact products, the scale factors)
        de = dx + 2^-22 (2 + max|x| log2 e)     the exponential and its argument
        t  = A (2 de + 2^-22 + 40 * 2^-23) + 2^-38 U     weights and denominator, their two terms, sums, fp16's last step
    and the result lies within t + half a step, of the binade that holds |o| + t.  (One fp16 term: 2^-12 in place of 2^-22,
    ten times t here.)"""
    g = _gen(D + Hq)
    lens = list(range(1, 34))
    B, page, sm, G = len(lens), 16, 1 / math.sqrt(D), Hq // Hkv
    codes = torch.randint(0, 256, (3 * B, 2, page, Hkv, D), generator=g).to(torch.uint8)
    codes[codes & 127 == 127] = 0
    scales = torch.full((3 * B, 2, 1, Hkv), 121, dtype=torch.uint8)
    table = torch.randperm(3 * B, generator=g).view(B, 3).to(torch.int32)
    q = (0.1 * torch.randn(B, Hq, D, generator=g)).to(DT[dt])
    ws = T.Workspace(B, Hq, D, 1, 1)
    o = T.decode_attention_kv8(q.cuda(), codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), max(lens), ws, page_table=table.cuda(),
                               seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda")).cpu().double()
    assert ws.status() == 0
    vals = K8.values(codes, scales)
    for b, n in enumerate(lens):
        pos = torch.arange(n)
        kv = vals[table[b].long()[pos // page], :, pos % page]
        for h in range(Hq):
            want, x, _, A, dot, U = K8.attention(q[b, h], kv[:, 0, h // G], kv[:, 1, h // G], sm, torch.full((n,), 2.0 ** -6, dtype=torch.float64))
            de = 20 * 2.0 ** -23 * dot + 2.0 ** -22 * (2 + float(x.abs().max()) * LOG2E)
            t = A * (2 * de + 2.0 ** -22 + 40 * 2.0 ** -23) + 2.0 ** -38 * U
            tol = t + _half_step(want.abs() + t, DT[dt])
            assert ((o[b, h] - want).abs() <= tol).all(), (n, h, float(((o[b, h] - want).abs() / tol).max()))


# ------------------------------------------------------------------ append: any start
@pytest.mark.parametrize("page,block", [(1, 1), (4, 4), (6, 3)])
def test_append_starts_at_the_end_of_the_integers(T, page, block):
    """Starts on the device whose tokens run past 2^31 - 1: nothing is read or written for them, they are reported, and
    the other sequence is stored."""
    g = _gen(20)
    Hkv, D, n = 2, 64, 4
    top = 2 ** 31 - 1
    pos = torch.tensor([top, top - 1, 3, top - 2, top - 5], dtype=torch.int32)
    B, per_seq = len(pos), 12 // page
    codes = torch.randint(0, 127, (B * per_seq, 2, page, Hkv, D), generator=g).to(torch.uint8)
    scales = torch.full((B * per_seq, 2, page // block, Hkv), 121, dtype=torch.uint8)
    k = torch.randn(B * n, Hkv, D, generator=g)
    kv, sc, status = codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    T.append_kv8(k.cuda(), k.cuda(), kv, sc, batch=B, pos0_dev=pos.cuda(), status=status)
    want, want_s = K8.values(codes, scales), scales.long()
    mine = k.view(B, n, Hkv, D)[2:3]
    K8.append(want, want_s, mine, mine, [3], torch.arange(B * per_seq).view(B, per_seq)[2:3])
    assert torch.equal(sc.cpu().long(), want_s) and torch.equal(K8.values(kv.cpu(), sc.cpu()), want)
    assert int(status) == 2


@pytest.mark.parametrize("e", [-110, -16, -15, 15, 23, 24, 25, 26, 60, 119])
def test_append_f16_rows_behind_tokens_of_any_scale(T, e):
    """A block whose first token came in 32 bits and has scale 2^e, then 16-bit rows, among them the largest, infinite and
    NaN ones: codes and scales bit for bit.  From 2^25 on only magnitudes above 2^(e - 10) are more than zero."""
    g = _gen(21)
    D = 64
    first = torch.randn(1, 1, 1, D, generator=g)
    first[0, 0, 0, 0] = 448.0
    first = (first.clamp(-448, 448).double() * 2.0 ** e).float()
    rows = (torch.randn(1, 3, 1, D, generator=g) * 2.0 ** 10).half()
    rows[0, 0, 0, :8] = torch.tensor([65504.0, -65504.0, 40000.0, 32768.0, 32800.0, 2.0 ** -24, -0.0, 60000.0])
    rows[0, 1, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 50000.0])
    rows[0, 2] *= 2.0 ** -20
    codes, scales = torch.zeros(1, 2, 4, 1, D, dtype=torch.uint8), torch.zeros(1, 2, 1, 1, dtype=torch.uint8)
    want, want_s = K8.values(codes, scales), scales.long()
    kv, sc = codes.cuda().view(torch.float8_e4m3fn), scales.cuda()
    K8.append(want, want_s, first, first, [0], [[0]])
    assert want_s.eq(e + 127).all()
    T.append_kv8(first[0].cuda(), first[0].cuda(), kv, sc)
    K8.append(want, want_s, rows, rows, [1], [[0]])
    T.append_kv8(rows[0].cuda(), rows[0].cuda(), kv, sc, pos0=1)
    got = K8.values(kv.cpu(), sc.cpu())
    assert torch.equal(sc.cpu().long(), want_s) and torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# -------------------------------------------------------------------------- read-back
def test_read_leaves_rows_of_negative_lengths(T):
    """A length below zero, down to the smallest integer, holds no rows: they are left as they were."""
    g = _gen(22)
    codes, scales = torch.randint(0, 127, (40, 2, 1, 1, 64), generator=g).to(torch.uint8), torch.full((40, 2, 1, 1), 121, dtype=torch.uint8)
    lens = torch.tensor([-2 ** 31, -2 ** 31 + 6, -1, 9], dtype=torch.int32)
    out = torch.full((4, 3, 2, 1, 1, 64), -7.0, device="cuda")
    T.read_kv8(codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), 10, start=7, batch=4, seq_lens=lens.cuda(), out=out)
    want = torch.full((4, 3, 2, 64), -7.0, dtype=torch.float64)
    want[3, :2] = K8.values(codes, scales)[37:39, :, 0, 0]
    assert torch.equal(out.cpu().double()[:, :, :, 0, 0], want)


# ------------------------------------------------------------ attention: smallest results
def _attend_one(T, dt, q, codes, scales, n, sm):
    """One KV head, one-token pages in order: the output [Hq, D] in 64 bits and (want, A, U, x, dot) per query head."""
    Hq, D = q.shape
    ws = T.Workspace(1, Hq, D, 1, 1)
    o = T.decode_attention_kv8(q[None].cuda(), codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), n, ws, sm_scale=sm)[0].cpu().double()
    assert ws.status() == 0
    vals = K8.values(codes, scales)
    vs = 2.0 ** (scales[:, 1, 0, 0].double() - 127)
    per_head = []
    for h in range(Hq):
        want, x, _, A, dot, U = K8.attention(q[h], vals[:, 0, 0, 0], vals[:, 1, 0, 0], sm, vs)
        per_head.append((want, A, U, x, dot))
    return o, per_head


def _small_tolerance(want, A, U, x, dot, n, dtype):
    """Half a step of the result; logits, weights and sums as for ordinary values; 32-bit intermediate results that are
    subnormal are off by 2^-150 each, four to every pair of tiles, up to twice that after the division by the sum (>= 1/2)."""
    de = 20 * 2.0 ** -23 * dot + 2.0 ** -22 * (2 + float(x.abs().max()) * LOG2E)
    t = A * (2 * de + 2.0 ** -21 + (n / 4 + 32) * 2.0 ** -23) + 2.0 ** -38 * U + 8 * (n / 32 + 1) * 2.0 ** -150
    return t + _half_step(want.abs() + t, dtype)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,D", [(4, 128), (12, 64), (2, 64), (7, 128)])
@pytest.mark.parametrize("n", [5, 300, 3001])
@pytest.mark.parametrize("low,high", [(-126, -120), (-118, -112), (-110, -100), (-126, -90)])
def test_attention_over_the_smallest_values(T, dt, Hq, D, n, low, high):
    """Value scales from 2^low to 2^high, down to the smallest there is: results are held down to the type's smallest."""
    g = _gen(n + D - low)
    codes = torch.randint(0, 256, (n, 2, 1, 1, D), generator=g).to(torch.uint8)
    codes[codes & 127 == 127] = 0
    scales = torch.full((n, 2, 1, 1), 121, dtype=torch.uint8)
    scales[:, 1] = torch.randint(127 + low, 128 + high, (n, 1, 1), generator=g).to(torch.uint8)
    q = (0.3 * torch.randn(Hq, D, generator=g)).to(DT[dt])
    o, per_head = _attend_one(T, dt, q, codes, scales, n, 1 / math.sqrt(D))
    assert o.abs().max() > 0
    for h, (want, A, U, x, dot) in enumerate(per_head):
        tol = _small_tolerance(want, A, U, x, dot, n, DT[dt])
        assert ((o[h] - want).abs() <= tol).all(), (h, float(((o[h] - want).abs() / tol).max()))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,heavy", [(70, 0), (300, 299), (1500, 700), (9000, 8999)])
@pytest.mark.parametrize("logit", [70.0, 76.0, 84.0])
def test_attention_behind_a_token_of_nearly_all_the_weight(T, dt, n, heavy, logit):
    """The values of the heaviest token are zero, those of the others lie up to 121 binades of weight below it: the answer
    is theirs."""
    g = _gen(n)
    D = 64
    k, v = torch.zeros(n, 1, D), torch.randn(n, 1, D, generator=g)
    k[heavy, 0, 0] = logit
    v[heavy] = 0.0
    kv, sc = T.alloc_kv8(n, 1, 1, D)
    T.append_kv8(k.cuda(), v.cuda(), kv, sc)
    q = torch.zeros(2, D)
    q[:, 0] = 1.0
    o, per_head = _attend_one(T, dt, q.to(DT[dt]), kv.cpu().view(torch.uint8), sc.cpu(), n, 1.0)
    assert o.abs().max() > 0
    for h, (want, A, U, x, dot) in enumerate(per_head):
        # U counts the heaviest token's scale, which its values of zero do not use: 2^-126, out of account
        tol = _small_tolerance(want, A, torch.zeros_like(U), x, dot, n, DT[dt])
        assert ((o[h] - want).abs() <= tol).all(), float(((o[h] - want).abs() / tol).max())


# ----------------------------------------------- attention: tokens far below the heaviest
@pytest.mark.parametrize("D,Hq", [(64, 1), (128, 1), (64, 12), (128, 12), (64, 4), (128, 3), (64, 8), (128, 5)])
@pytest.mark.parametrize("n", [40, 300, 1000])
@pytest.mark.parametrize("logit", [16.0, 18.0, 20.0, 26.0])
def test_attention_keeps_the_bits_of_light_tokens(T, D, Hq, n, logit):
    """fp32.  One token of ordinary values holds nearly all the weight, but half its elements are zero: there the answer is
    what the other tokens carry, all of one weight 22 to 37 binades below, so that their roundings all go one way.  Off by
    at most, of sum p|v|: 2^-20 the rounding of an exponential's argument (up to 64: half a step, times ln 2, is 2^-19 only
    from 32 on), 2^-22 the exponential, 2^-22 a weight's two terms, 17 * 2^-24 a tile's product, 40 * 2^-24 the additions of a
    warp's tiles and of the parts, 4 * 2^-24 the denominator and the division: less than 2^-17.  (A second term without a
    factor of its own ends at 2^-24, 2^-38 of the heaviest weight: 2^-15 of a weight of 2^-24 of it, 2^-11 of 2^-28.)
    And 2^-50 U: the second term goes in times 2^12, so its steps of 2^-24 stand for 2^-36 and it is off by 2^-37, where the
    largest p_j 2^ev_j is scaled to more than 2^13; U = max_j (p_j 2^ev_j) * sum_j |code_j|."""
    g = _gen(D + n)
    k, v = torch.zeros(n, 1, D), torch.randn(n, 1, D, generator=g)
    heavy = n // 3
    k[:, 0, 0] = 0.34375
    k[heavy, 0, 0] = logit
    v[heavy, 0, :] = 1.0
    v[heavy, 0, : D // 2] = 0.0
    kv, sc = T.alloc_kv8(n, 1, 1, D)
    T.append_kv8(k.cuda(), v.cuda(), kv, sc)
    q = torch.zeros(Hq, D)
    q[:, 0] = 1.0
    o, per_head = _attend_one(T, "f32", q, kv.cpu().view(torch.uint8), sc.cpu(), n, 1.0)
    for h, (want, A, U, x, dot) in enumerate(per_head):
        off = ((o[h] - want).abs() / (2.0 ** -17 * A + 2.0 ** -50 * U)).max()
        assert off <= 1, float(off)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_read_over_all_scales_and_codes(T, dt):
    """Every code at every scale from zero and 2^-126 to 2^120: one rounding to the type, and what lies beyond its largest
    number saturates (32 bits hold every value but those of 2^128 and more, which codes from 256 on have at scale 2^120:
    the largest finite floats are stored so)."""
    n, D = 248, 128
    codes = torch.arange(256).view(1, 2, 1, 1, D).expand(n, 2, 1, 1, D).to(torch.uint8).contiguous()
    scales = torch.arange(n).view(n, 1, 1, 1).expand(n, 2, 1, 1).to(torch.uint8).contiguous()
    got = T.read_kv8(codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), n, dtype=DT[dt])[0, :, :, 0, 0].cpu()
    want = K8.values(codes, scales)[:, :, 0, 0]
    assert torch.equal(want[:247].float().double().nan_to_num(), want[:247].nan_to_num())
    most = torch.finfo(DT[dt]).max
    want = want.float().clamp(-most, most).to(DT[dt])
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~torch.isnan(got)], want[~torch.isnan(want)])


@pytest.mark.parametrize("Hq,D", [(1, 64), (8, 64), (8, 128), (12, 128), (4, 64), (3, 128)])
def test_attention_long_sums_of_ordinary_weights(T, Hq, D):
    """fp32, 20 000 tokens, many to a warp, ordinary softmax weights and values of both signs, in the root mean square of a
    result.  Queries and keys are few multiples of powers of two: the products' sums are exact.  What is left:
        2^-20.5   the argument of an exponential, below 32: half a step of 2^-19 times ln 2
        2^-22     the exponential; 2^-22 a weight's two terms; 2^-22 the merge and the division
        E         the common factor of all logits, sm log2 e, off by 2^-23 of itself: moves a weight by 2^-23 ln 2 (x - mean x)
        2 sqrt(n/16)/3 * 2^-24     additions rounded to nearest, as for equal weights."""
    g = _gen(D + Hq)
    n, page, B, sm = 20000, 16, 300, 2.0 ** -4 if D == 128 else 2.0 ** -3.5
    sm = float(torch.tensor(sm, dtype=torch.float32))
    k = torch.randint(-8, 9, (n, 1, D), generator=g) * 0.25
    codes = torch.randint(0, 256, (n // page, 2, page, 1, D), generator=g).to(torch.uint8)
    codes[codes & 127 == 127] = 0
    codes[:, 0] = k.to(torch.float8_e4m3fn).view(torch.uint8).view(n // page, page, 1, D)
    scales = torch.full((n // page, 2, 1, 1), 120, dtype=torch.uint8)
    scales[:, 0] = 127
    q = torch.randint(-8, 9, (B, Hq, D), generator=g) / 4.0
    ws = T.Workspace(B, Hq, D, 1, 1)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(B, -1).contiguous()
    o = T.decode_attention_kv8(q.cuda(), codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), n, ws, page_table=table, sm_scale=sm).double()
    assert ws.status() == 0
    vals = K8.values(codes, scales).cuda()
    K, V = vals[:, 0, :, 0].reshape(n, D), vals[:, 1, :, 0].reshape(n, D)
    assert torch.equal(K.cpu(), k[:, 0].double())
    worst = 0.0
    for b in range(0, B, 20):
        x = q[b:b + 20].cuda().double().view(-1, D) @ K.T * sm
        p = torch.softmax(x, 1)
        want = p @ V
        assert (x.amax(1) - x.amin(1)).max() * LOG2E + 1 < 32
        factor = (p * (x - (p * x).sum(1, keepdim=True))) @ V * 2.0 ** -23
        size = want.norm(dim=1)
        tol = 2.0 ** -20.5 + 3 * 2.0 ** -22 + factor.norm(dim=1) / size + 2 * math.sqrt(n / 16) / 3 * 2.0 ** -24
        off = (o[b:b + 20].view(-1, D) - want).norm(dim=1) / size
        worst = max(worst, float((off / tol).max()))
    assert worst <= 1, worst


@pytest.mark.parametrize("Hq,D", [(8, 64), (8, 128), (3, 128), (12, 64)])
def test_attention_of_one_token_is_its_value(T, Hq, D):
    """fp32, one token: the result is its value whatever the logit.  The weight and the denominator are the same exponential of
    the same argument, 2^(x - m), but for powers of two; what differs is the weight's two terms (2^-22), the division, the
    product with it and the scaling (2^-24 each), one to spare."""
    g = _gen(D + Hq)
    B = 64
    kv, sc = T.alloc_kv8(B, 1, 1, D)
    k, v = torch.randn(B, 1, D, generator=g).cuda(), torch.randn(B, 1, D, generator=g).cuda()
    T.append_kv8(k, v, kv, sc, batch=B)
    ws = T.Workspace(B, Hq, D, 1, 1)
    q = (3 * torch.rand(B, Hq, 1, generator=g) * torch.randn(B, Hq, D, generator=g)).cuda()
    o = T.decode_attention_kv8(q, kv, sc, 1, ws).cpu().double()
    want = K8.values(kv.cpu(), sc.cpu())[:, 1, 0]                                    # [B, 1, D]
    assert ws.status() == 0
    assert ((o - want).abs() <= (2.0 ** -22 + 4 * 2.0 ** -24) * want.abs()).all(), float(((o - want).abs() / want.abs().clamp(min=1e-30)).max().log2())
