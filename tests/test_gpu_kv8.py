"""The 8-bit KV cache operators against their definitions in 64 bits (oracle/kv8_oracle.py): quantised append, read-back,
decode attention, attention weights per token, page eviction, and a decode loop that uses all of them.

Tolerances.  Codes, scales, read-back values, moved weights, tables and lengths are exact.  For attention, with
A = sum_j p_j |v_j| and x the logits, a computed output may be off by
    eps(type)/2 * |o|                      the one rounding of the result; below the type's smallest normal number t its
                                           steps are t * eps(type) wide whatever |o|, so at least t * eps(type)/2
    2 * dx * A                             logits off by dx change every weight and the denominator by a factor 1 +- dx
    2^-11 A (16-bit types) or 2^-21 A      weights enter the product with V rounded to 11 (or twice 11) bits
    2^-38 U                                fp16's steps end at 2^-24, and weights are scaled so that the largest p_j 2^ev_j of
                                           the tokens lies in (2^13, 2^14]: a weight is off by 2^-25 at least, that is by up to
                                           2^-38 of the largest; U = max_j (p_j 2^ev_j) * sum_j |code_j|
    (n/4 + 32) * 2^-23 * A                 fp32 sums over n tokens, at least four to an addition, each step off by 2^-23
with dx = 20 * 2^-23 * max_j sum_d |q_d k_jd| sm (8 to 16 fp32 additions of exact products, the scale factors) plus
2^-22 * (2 + max|x| * log2 e) for the exponential and its argument.  Logits themselves are held to that dx."""
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


def _pool(g, pages, page, block, Hkv, D, spread=6):
    """A pool of random codes (no NaN) and scales of a few binades around 2^-6."""
    codes = torch.randint(0, 256, (pages, 2, page, Hkv, D), generator=g).to(torch.uint8)
    codes[codes & 127 == 127] = 0
    scales = torch.randint(121 - spread // 2, 122 + spread // 2, (pages, 2, page // block, Hkv), generator=g).to(torch.uint8)
    return codes, scales


def _table(g, B, per_seq, spare=3):
    n = B * per_seq + spare
    return torch.randperm(n, generator=g)[:B * per_seq].view(B, per_seq).to(torch.int32), n


def _same_values(got_codes, got_scales, want_values, want_scales):
    assert torch.equal(got_scales.cpu().long(), want_scales)
    got = K8.values(got_codes.cpu(), got_scales.cpu())
    assert torch.equal(torch.isnan(got), torch.isnan(want_values))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want_values))


# ------------------------------------------------------------------------- append
APPEND = [
    # dtype, B, T, pos0, Hkv, D, page, block
    ("bf16", 1, 1, 0, 8, 128, 16, 16), ("bf16", 5, 1, 19, 8, 128, 16, 16), ("f16", 2, 1, 15, 1, 64, 16, 8),
    ("f32", 3, 37, 5, 4, 64, 7, 7), ("f16", 1, 129, 0, 5, 128, 1, 1), ("bf16", 2, 65, 31, 2, 64, 1, 1),
    ("f32", 1, 33, 63, 3, 128, 64, 64), ("bf16", 2, 50, 7, 2, 128, 24, 3), ("f16", 1, 300, 100, 2, 64, 128, 128),
    ("f32", 2, 9, 1, 1, 128, 2, 2), ("f32", 1, 3, 2, 32, 128, 1, 1),
]


@pytest.mark.parametrize("dt,B,n,pos0,Hkv,D,page,block", APPEND)
@pytest.mark.parametrize("gain", [1.0, 0.01, 300.0])
def test_append(T, dt, B, n, pos0, Hkv, D, page, block, gain):
    """Codes and scales bit for bit; slots that are not written stay as they were.  A gain of 300 raises the scale of a
    block that already holds codes, 0.01 leaves it."""
    g = _gen(pos0 * 1000 + n + int(gain))
    table, pages = _table(g, B, -(-(pos0 + n) // page))
    codes, scales = _pool(g, pages, page, block, Hkv, D)
    k, v = (gain * torch.randn(B, n, Hkv, D, generator=g) * torch.rand(B, n, Hkv, 1, generator=g) for _ in range(2))
    k, v = k.to(DT[dt]), v.to(DT[dt])
    want, want_s = K8.values(codes, scales), scales.long()
    K8.append(want, want_s, k, v, [pos0] * B, table)
    kv, sc = codes.cuda().view(torch.float8_e4m3fn), scales.cuda()
    T.append_kv8(k.view(B * n, Hkv, D).cuda(), v.view(B * n, Hkv, D).cuda(), kv, sc, batch=B, pos0=pos0, page_table=table.cuda())
    _same_values(kv, sc, want, want_s)


def test_append_special_values(T):
    """Infinities saturate and do not set the scale, NaN stays NaN, a block of zeros takes the smallest scale, the
    largest and smallest magnitudes of 32 bits fit, and an amax exactly at 448 * 2^e does not raise e."""
    D = 64
    k = torch.zeros(8, 1, D)
    k[1, 0, :4] = torch.tensor([1.0, math.inf, -math.inf, math.nan])
    k[2, 0, :2] = torch.tensor([3.4028235e38, -3.0e38])
    k[3, 0, :2] = torch.tensor([1e-45, 1.2e-38])
    k[4, 0, 0] = 448.0
    k[5, 0, 0] = 448.00003
    k[6, 0, :3] = torch.tensor([math.nan, math.nan, math.inf])
    k[7, 0, :4] = torch.tensor([-0.0, 2.0 ** -9 * 1.75, 1.0, 17.0 * 2 ** -10])
    codes, scales = torch.zeros(8, 2, 1, 1, D, dtype=torch.uint8), torch.zeros(8, 2, 1, 1, dtype=torch.uint8)
    want, want_s = K8.values(codes, scales), scales.long()
    K8.append(want, want_s, k.view(1, 8, 1, D), k.view(1, 8, 1, D), [0], torch.arange(8)[None])
    kv, sc = codes.cuda().view(torch.float8_e4m3fn), scales.cuda()
    T.append_kv8(k.cuda(), k.cuda(), kv, sc, pos0=0)
    _same_values(kv, sc, want, want_s)
    assert sc[0, 0, 0, 0] == 1 and sc[4, 0, 0, 0] == 127 and sc[5, 0, 0, 0] == 128


@pytest.mark.parametrize("page,block", [(1, 1), (16, 16), (16, 4), (6, 3)])
def test_append_in_steps_equals_the_format(T, page, block):
    """Token by token, with starts on the device that differ between sequences: the scale of a block only grows, starts
    afresh when the block does, and ends at what the block's tokens ask for."""
    g = _gen(5)
    B, Hkv, D, n = 3, 2, 64, 21
    table, pages = _table(g, B, -(-(40 + n) // page))
    codes, scales = _pool(g, pages, page, block, Hkv, D)
    kv, sc, tab = codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), table.cuda()
    want, want_s = K8.values(codes, scales), scales.long()
    pos = torch.tensor([0, 17, 40], dtype=torch.int32)
    for t in range(n):
        k, v = (torch.randn(B, 1, Hkv, D, generator=g) * 2.0 ** (t % 7) for _ in range(2))
        K8.append(want, want_s, k, v, [int(x) + t for x in pos], table)
        T.append_kv8(k.view(B, Hkv, D).cuda(), v.view(B, Hkv, D).cuda(), kv, sc, batch=B, pos0_dev=(pos + t).cuda(), page_table=tab)
    _same_values(kv, sc, want, want_s)


def test_append_spaced_rows(T):
    """k and v as slices of one projection's output: the same codes as from contiguous rows."""
    g = _gen(6)
    B, Hkv, D = 4, 2, 128
    qkv = torch.randn(B, (4 + 2 * Hkv) * D, generator=g).to(torch.bfloat16).cuda()
    k = qkv[:, 4 * D:(4 + Hkv) * D].unflatten(1, (Hkv, D))
    v = qkv[:, (4 + Hkv) * D:].unflatten(1, (Hkv, D))
    assert not k.is_contiguous()
    pools = [T.alloc_kv8(B * 2, 8, Hkv, D, 8) for _ in range(2)]
    T.append_kv8(k, v, *pools[0], batch=B, pos0=3)
    T.append_kv8(k.contiguous(), v.contiguous(), *pools[1], batch=B, pos0=3)
    assert torch.equal(pools[0][0].view(torch.uint8), pools[1][0].view(torch.uint8)) and torch.equal(pools[0][1], pools[1][1])
    assert int(pools[0][1].count_nonzero()) == B * 2 * Hkv


def test_append_out_of_range_is_skipped(T):
    """A page outside the pool, a negative start and a start behind the table touch nothing and are reported; the other
    sequences are written."""
    g = _gen(7)
    Hkv, D = 2, 64
    codes, scales = _pool(g, 4, 2, 2, Hkv, D)
    k = torch.randn(4, Hkv, D, generator=g)
    table = torch.tensor([[9, 0], [1, 0], [2, 0], [3, 0]], dtype=torch.int32)
    pos = torch.tensor([1, -1, 4, 1], dtype=torch.int32)
    kv, sc = codes.cuda().view(torch.float8_e4m3fn), scales.cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    T.append_kv8(k.cuda(), k.cuda(), kv, sc, batch=4, pos0_dev=pos.cuda(), page_table=table.cuda(), status=status)
    want, want_s = K8.values(codes, scales), scales.long()
    K8.append(want, want_s, k[3:].view(1, 1, Hkv, D), k[3:].view(1, 1, Hkv, D), [1], table[3:])
    _same_values(kv, sc, want, want_s)
    assert int(status) == 2
    status.zero_()
    T.append_kv8(k.cuda()[:1], k.cuda()[:1], kv, sc, pos0_dev=torch.tensor([-5], dtype=torch.int32, device="cuda"), status=status)
    _same_values(kv, sc, want, want_s)
    assert int(status) == 2


# -------------------------------------------------------------------------- read
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,start,stop,Hkv,D,page,block", [(1, 0, 1, 1, 64, 1, 1), (2, 5, 44, 8, 128, 16, 16), (3, 13, 30, 3, 64, 7, 7), (1, 0, 300, 2, 128, 24, 3)])
def test_read(T, dt, B, start, stop, Hkv, D, page, block):
    g = _gen(stop)
    table, pages = _table(g, B, -(-stop // page))
    codes, scales = _pool(g, pages, page, block, Hkv, D)
    want = K8.values(codes, scales)
    pos = torch.arange(start, stop)
    want = want.transpose(1, 2)[table.long()[:, pos // page], pos % page]                       # [B, n, 2, Hkv, D]
    lens = torch.randint(start, stop + 1, (B,), generator=g).to(torch.int32)
    out = torch.full((B, stop - start, 2, 1, Hkv, D), -7.0, dtype=DT[dt], device="cuda")
    args = (codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), stop)
    got = T.read_kv8(*args, start=start, batch=B, page_table=table.cuda(), dtype=DT[dt])
    assert got.dtype == DT[dt] and torch.equal(got.cpu().double()[:, :, :, 0], want)
    T.read_kv8(*args, start=start, batch=B, page_table=table.cuda(), seq_lens=lens.cuda(), out=out)
    live = (pos < lens[:, None])[..., None, None, None]
    assert torch.equal(out.cpu().double()[:, :, :, 0], torch.where(live, want, torch.full_like(want, -7.0)))


def test_read_f16_saturates(T):
    kv, sc = T.alloc_kv8(1, 1, 1, 64)
    T.append_kv8(torch.full((1, 1, 64), 65504.0, dtype=torch.float16, device="cuda"), torch.full((1, 1, 64), -65504.0, dtype=torch.float16, device="cuda"), kv, sc)
    got = T.read_kv8(kv, sc, 1, dtype=torch.float16)
    assert got[0, 0, 0].eq(65504.0).all() and got[0, 0, 1].eq(-65504.0).all()
    assert T.read_kv8(kv, sc, 1, dtype=torch.float32)[0, 0, 0].eq(65536.0).all()
    assert T.read_kv8(kv, sc, 0).shape == (1, 0, 2, 1, 1, 64)


# --------------------------------------------------------------------- attention
def _attention_case(T, dt, B, Hq, Hkv, D, lens, page, block, lists="all", k=0, counts=None, gain=1.0, identity=False, want_logits=True, seed=0,
                    sm_scale=0.0, vspread=6):
    g = _gen(seed + sum(lens) + Hq)
    N = max(lens)
    dtype = DT[dt]
    per_seq = max(1, -(-N // page))
    table, pages = _table(g, B, per_seq)
    if identity:
        table, pages = torch.arange(B * per_seq, dtype=torch.int32).view(B, per_seq), B * per_seq
    codes, scales = _pool(g, pages, page, block, Hkv, D)
    scales[:, 1] = torch.randint(118 - vspread, 122 + vspread, scales[:, 1].shape, generator=g).to(torch.uint8)
    vals = K8.values(codes, scales)
    q = (gain * torch.randn(B, Hq, D, generator=g)).to(dtype)
    sm = sm_scale if sm_scale > 0 else 1 / math.sqrt(D)
    kw = {}
    if lists != "all":
        rows = 1 if lists == "shared" else Hq
        sel = torch.stack([torch.randint(0, max(lens[b], 1), (rows, k), generator=g) for b in range(B)]).to(torch.int32)
        kw["sel_idx"] = (sel[:, 0] if lists == "shared" else sel).contiguous().cuda()
        if counts is not None:
            cnt = torch.tensor(counts, dtype=torch.int32).view(B, 1).expand(B, rows).contiguous()
            kw["sel_counts"] = (cnt[:, 0] if lists == "shared" else cnt).contiguous().cuda()
    n_cols = N if lists == "all" else k
    scores = torch.full((B, Hq, max(n_cols, 1)), -123.0, device="cuda") if want_logits else None
    lse = torch.full((B, Hq), -123.0, device="cuda") if want_logits else None
    ws = T.Workspace(B, Hq, D, 1, 1)
    lens_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if identity:
        kw["pages_per_seq"] = per_seq
    else:
        kw["page_table"] = table.cuda()
    o = T.decode_attention_kv8(q.cuda(), codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), N, ws,
                               seq_lens=None if len(set(lens)) == 1 else lens_dev, scores=scores, lse=lse, sm_scale=sm_scale, **kw)
    torch.cuda.synchronize()
    assert ws.status() == 0
    o = o.cpu().double()
    eps = torch.finfo(dtype).eps / 2
    G = Hq // Hkv
    for b in range(B):
        for h in range(Hq):
            if lists == "all":
                pos = torch.arange(lens[b])
            else:
                n = k if counts is None else counts[b]
                pos = sel[b, 0 if lists == "shared" else h, :n].long()
            pg = table[b].long()[pos // page]
            vs = 2.0 ** (scales[pg, 1, pos % page // block, h // G].double() - 127)
            want, x, z, A, dot, U = K8.attention(q[b, h], vals[pg, 0, pos % page, h // G], vals[pg, 1, pos % page, h // G], sm, vs)
            n = pos.numel()
            top = float(x.abs().max()) if n else 0.0
            dx = 20 * 2.0 ** -23 * dot
            de = dx + 2.0 ** -22 * (2 + top * LOG2E)
            tol = eps * want.abs() + A * (2 * de + (2.0 ** -21 if dt == "f32" else 2.0 ** -11) + (n / 4 + 32) * 2.0 ** -23) + 2.0 ** -38 * U
            tol = torch.maximum(tol, torch.full_like(tol, torch.finfo(dtype).smallest_normal * eps) + tol - eps * want.abs())
            most = torch.finfo(dtype).max * (1 + eps)                    # from here on a result of the type is infinite
            over = want.abs() - tol >= most
            assert torch.equal(o[b, h][over], want[over].sign() * math.inf)
            near = (want.abs() + tol >= most) & ~over                   # either side of it is right
            err = torch.where(over | near, torch.zeros_like(want), (o[b, h] - want).abs())
            assert (err <= tol).all(), (b, h, n, float((err / tol).max()))
            if want_logits:
                got = scores[b, h].cpu().double()
                assert ((got[:n] - x).abs() <= dx + 2.0 ** -23 * x.abs()).all(), (b, h, float((got[:n] - x).abs().max()), dx)
                assert got[n:].eq(-123.0).all()
                if n == 0:
                    assert lse[b, h].item() == -math.inf
                else:
                    assert abs(lse[b, h].item() - z) <= de + (n / 4 + 32) * 2.0 ** -23 + 2.0 ** -22 * abs(z)
    return o


ATTEND = [
    # dtype, B, Hq, Hkv, D, lens, page, block
    ("bf16", 1, 32, 8, 128, [1], 16, 16), ("f16", 1, 4, 4, 64, [2], 1, 1), ("f32", 1, 8, 2, 128, [17], 16, 4),
    ("bf16", 2, 32, 8, 128, [131, 131], 16, 16), ("f16", 1, 32, 32, 128, [1000], 1, 1), ("f32", 5, 20, 4, 64, [503, 1, 0, 77, 250], 7, 7),
    ("bf16", 3, 16, 1, 128, [600, 15, 33], 3, 3), ("f16", 2, 40, 8, 64, [129, 300], 24, 8), ("f32", 1, 12, 6, 128, [777], 1, 1),
    ("bf16", 1, 64, 8, 128, [4099], 64, 32), ("f16", 1, 5, 5, 128, [2049], 16, 16), ("f32", 1, 48, 2, 64, [200], 16, 2),
    ("bf16", 1, 34, 1, 128, [100], 1, 1), ("f16", 7, 14, 2, 64, [0, 0, 1, 16, 17, 500, 31], 16, 16), ("bf16", 1, 4, 4, 128, [9001], 5, 5),
    ("bf16", 2, 1, 1, 64, [0, 0], 16, 16), ("f16", 33, 8, 8, 64, [3 * i for i in range(33)], 16, 16),
]


@pytest.mark.parametrize("dt,B,Hq,Hkv,D,lens,page,block", ATTEND)
def test_attention(T, dt, B, Hq, Hkv, D, lens, page, block):
    _attention_case(T, dt, B, Hq, Hkv, D, lens, page, block)


@pytest.mark.parametrize("dt,B,Hq,Hkv,D,lens,page,block", ATTEND[:6])
def test_attention_identity_pages_and_output_alone(T, dt, B, Hq, Hkv, D, lens, page, block):
    _attention_case(T, dt, B, Hq, Hkv, D, lens, page, block, identity=True, want_logits=False, sm_scale=0.3)


@pytest.mark.parametrize("lists", ["shared", "per_head"])
@pytest.mark.parametrize("dt,B,Hq,Hkv,D,lens,page,block,k,counts", [
    ("f16", 1, 32, 8, 128, [3000], 1, 1, 256, None), ("bf16", 2, 8, 8, 64, [500, 90], 16, 16, 33, None), ("f32", 3, 20, 4, 64, [64, 500, 7], 7, 7, 100, [100, 0, 3]),
    ("bf16", 1, 6, 1, 128, [40], 1, 1, 1, None), ("f16", 2, 16, 16, 128, [70000, 6], 1, 1, 2500, [2500, 17]),
])
def test_attention_lists(T, lists, dt, B, Hq, Hkv, D, lens, page, block, k, counts):
    """Lists in any order, positions listed twice among them."""
    _attention_case(T, dt, B, Hq, Hkv, D, lens, page, block, lists=lists, k=k, counts=counts)


def test_attention_many_lists(T):
    """More lists than a CTA adds up, and more sequences than ranges of tokens (warps that cross several lists)."""
    _attention_case(T, "f16", 130, 16, 4, 64, [50] * 130, 16, 16, lists="per_head", k=40, counts=[i % 41 for i in range(130)])
    _attention_case(T, "bf16", 300, 2, 1, 64, [1025 + (7 * i) % 300 if i % 5 else i % 3 for i in range(300)], 16, 16)


@pytest.mark.parametrize("B,Hq,Hkv,lens", [(1, 1, 1, [70001]), (2, 16, 16, [5000, 40001]), (1, 8, 1, [33333]), (3, 32, 2, [1500, 9000, 1]), (1, 24, 2, [20000])])
def test_attention_long(T, B, Hq, Hkv, lens):
    """Lists shared by many warps, merged in the order of their parts; units of 1, 8, 12 and 16 heads."""
    _attention_case(T, "bf16", B, Hq, Hkv, 128, lens, 16, 16)
    _attention_case(T, "f32", B, Hq, Hkv, 64, lens, 1, 1, want_logits=False)


@pytest.mark.parametrize("Hq,Hkv,D", [(1, 1, 64), (8, 1, 128), (12, 1, 128), (24, 1, 64)])
def test_attention_long_sums_are_rounded_to_nearest(T, Hq, Hkv, D):
    """fp32, many tokens to a warp (all sequences list the same pages), every weight equal and no value negative: the
    logits, the weights and a tile's 16 products are exact, so what is left are n / 16 additions.  Rounded to nearest,
    each is off by a uniform error of up to 2^-24 of a sum that grows evenly, sqrt(n / 16) / 3 * 2^-24 of the result in
    the root mean square; twice that is allowed, and 2^-22 for the merge and the division.  Sums that are cut off would
    be off by about n / 32 * 2^-24."""
    g = _gen(D + Hq)
    n, page, B = 20000, 16, 400
    table, pages = _table(g, 1, n // page)
    codes, scales = _pool(g, pages, page, page, Hkv, D)
    codes[:, 1] &= 127
    scales[:, 1] = 120
    want = K8.values(codes, scales)[table[0].long(), 1].view(n, Hkv, D).double().mean(0).repeat_interleave(Hq // Hkv, 0)
    ws = T.Workspace(B, Hq, D, 1, 1)
    o = T.decode_attention_kv8(torch.zeros(B, Hq, D, device="cuda"), codes.cuda().view(torch.float8_e4m3fn), scales.cuda(), n, ws,
                               page_table=table.cuda().expand(B, -1).contiguous())
    off = (o.cpu().double() - want).flatten(1).norm(dim=1) / want.norm()
    assert ws.status() == 0 and off.max() <= 2 * math.sqrt(n / 16) / 3 * 2.0 ** -24 + 2.0 ** -22, off.max()


def test_attention_empty_lists(T):
    """Lists of no entries are not "every token"; a sequence length of zero on the host."""
    kv, sc = T.alloc_kv8(4, 1, 1, 64)
    q = torch.randn(2, 3, 64, device="cuda")
    ws, lse = T.Workspace(2, 3, 64, 1, 1), torch.zeros(2, 3, device="cuda")
    for kw in (dict(seq_len=2, sel_idx=torch.zeros(2, 0, dtype=torch.int32, device="cuda")), dict(seq_len=2, sel_idx=torch.zeros(2, 3, 0, dtype=torch.int32, device="cuda")),
               dict(seq_len=0)):
        o = T.decode_attention_kv8(q, kv, sc, ws=ws, out=torch.full_like(q, 5.0), lse=lse.fill_(1.0), **kw)
        assert not o.any() and lse.eq(-math.inf).all()
    assert ws.status() == 0


def test_wrapper_refusals(T):
    kv, sc = T.alloc_kv8(4, 16, 2, 64, 16)
    q, ws = torch.zeros(1, 4, 64, device="cuda"), T.Workspace(1, 4, 64, 1, 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.zeros(3, 2, 64, device="cuda")
    for match, call in [
        ("float8", lambda: T.read_kv8(kv.view(torch.uint8), sc, 4)), ("uint8", lambda: T.read_kv8(kv, sc[:2], 4)), ("divide", lambda: T.read_kv8(kv, torch.zeros(4, 2, 3, 2, dtype=torch.uint8, device="cuda"), 4)),
        ("range", lambda: T.read_kv8(kv, sc, 4, start=5)), ("out must", lambda: T.read_kv8(kv, sc, 4, out=torch.zeros(4, device="cuda"))), ("page table", lambda: T.read_kv8(kv, sc, 40, page_table=torch.zeros(1, 2, **i32))),
        ("n_tokens", lambda: T.append_kv8(k, k, kv, sc, batch=2)), ("one dtype", lambda: T.append_kv8(k, k.half(), kv, sc)), ("contiguous", lambda: T.append_kv8(k.transpose(1, 2).contiguous().transpose(1, 2), k, kv, sc)),
        ("elements", lambda: T.append_kv8(k, k, kv, sc, pos0_dev=torch.zeros(2, **i32))), ("pages", lambda: T.append_kv8(k, k, kv, sc, pos0=62)), ("out of range", lambda: T.append_kv8(k, k, kv, sc, pos0=2 ** 31)),
        ("not q itself", lambda: T.decode_attention_kv8(q, kv, sc, 4, ws, out=q)), ("sel_idx", lambda: T.decode_attention_kv8(q, kv, sc, 4, ws, sel_counts=torch.zeros(1, **i32))),
        ("int32", lambda: T.decode_attention_kv8(q, kv, sc, 4, ws, sel_idx=torch.zeros(1, 2, dtype=torch.int64, device="cuda"))), ("scores", lambda: T.decode_attention_kv8(q, kv, sc, 4, ws, scores=torch.zeros(1, 4, device="cuda"))),
        ("score_stride", lambda: T.decode_attention_kv8(q, kv, sc, 4, ws, scores=torch.zeros(1, 4, 3, device="cuda"))), ("page table", lambda: T.decode_attention_kv8(q, kv, sc, 17, ws, page_table=torch.zeros(1, 1, **i32))),
        ("contiguous", lambda: T.decode_attention_kv8(q.expand(2, 4, 64), kv, sc, 4, ws)), ("one row per head", lambda: T.accumulate_weights(torch.zeros(1, 4, device="cuda"), q[0, :1], q[0, :1], 4)),
        ("shapes", lambda: T.evict_pages(torch.zeros(1, 8, device="cuda"), torch.zeros(1, 8, **i32), torch.zeros(1, **i32), 4, out=(torch.zeros(1, 7, device="cuda"), torch.zeros(1, 8, **i32), torch.zeros(1, **i32)))),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("gain,vspread", [(0.0, 0), (1e-4, 0), (40.0, 6), (300.0, 6), (1.0, 100)])
def test_attention_ranges(T, dt, gain, vspread):
    """Flat and one-hot softmax, query rows of any magnitude, value scales a hundred binades apart (a token of nearly all
    the weight whose values are nothing beside those of a token of little weight)."""
    _attention_case(T, dt, 1, 8, 2, 128, [700], 16, 16, gain=gain, vspread=vspread)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_attention_value_scales_do_not_hide_small_weights(T, dt):
    """The heaviest token's values are exactly zero; the answer is what tokens of weight 2^-40 and less carry."""
    D, n = 64, 70
    kv, sc = T.alloc_kv8(n, 1, 1, D)
    k, v = torch.zeros(n, 1, D), torch.randn(n, 1, D, generator=_gen(3))
    k[0, 0, 0] = 28.0                        # logit 28 = 40 binades over the others
    v[0] = 0.0
    T.append_kv8(k.cuda(), v.cuda(), kv, sc)
    q = torch.zeros(1, 1, D)
    q[0, 0, 0] = 1.0
    o = T.decode_attention_kv8(q.to(DT[dt]).cuda(), kv, sc, n, T.Workspace(1, 1, D, 1, 1), sm_scale=1.0)
    vals = K8.values(kv.cpu(), sc.cpu())
    want, x, z, A, dot = K8.attention(q[0, 0], vals[:, 0, 0, 0], vals[:, 1, 0, 0], 1.0)
    tiny = torch.finfo(DT[dt]).smallest_normal * torch.finfo(DT[dt]).eps / 2        # half a step of the subnormal outputs of f16
    de = 20 * 2.0 ** -23 * dot + 2.0 ** -22 * (2 + 28 * LOG2E)
    tol = torch.finfo(DT[dt]).eps / 2 * want.abs() + tiny + A * (2 * de + 2.0 ** -11 + 64 * 2.0 ** -23)
    assert ((o[0, 0].cpu().double() - want).abs() <= tol).all()


def test_attention_infinite_and_nan_keys(T):
    """A NaN code in a key or value poisons the heads that attend to it, and no other head, sequence or unlisted token;
    what lies in the pages behind the length does not matter."""
    g = _gen(9)
    D, Hkv, page = 64, 2, 16
    codes, scales = _pool(g, 8, page, page, Hkv, D)
    ws = T.Workspace(2, 4, D, 1, 1)
    q = torch.randn(2, 4, D, generator=g).cuda()
    table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
    lens = torch.tensor([50, 37], dtype=torch.int32, device="cuda")
    run = lambda c: T.decode_attention_kv8(q, c.cuda().view(torch.float8_e4m3fn), scales.cuda(), 64, ws, page_table=table, seq_lens=lens).cpu()   # noqa: E731
    clean = run(codes)
    assert torch.isfinite(clean).all()
    behind = codes.clone()
    behind[3, :, 2:] = 127                   # slots 50.. of sequence 0
    behind[6, :, 5:] = 255                   # slots 37.. of sequence 1
    behind[7] = 127
    assert torch.equal(run(behind), clean)
    for plane in (0, 1):
        bad = codes.clone()
        bad[1, plane, 3, 1, 5] = 127         # sequence 0, slot 19, KV head 1
        got = run(bad)
        assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :2], clean[0, :2])
        assert torch.isnan(got[0, 2:, 5]).all()


def test_attention_bad_entries_are_skipped(T):
    """Positions outside the sequence and pages outside the pool do not take part and are reported."""
    g = _gen(10)
    D, n = 64, 40
    codes, scales = _pool(g, n, 1, 1, 1, D)
    kv, sc = codes.cuda().view(torch.float8_e4m3fn), scales.cuda()
    q = torch.randn(1, 2, D, generator=g).cuda()
    ws = T.Workspace(1, 2, D, 1, 1)
    good = torch.tensor([[3, 9, 30]], dtype=torch.int32)
    bad = torch.tensor([[3, -1, 9, n, 2 ** 30, 30]], dtype=torch.int32)
    scores = torch.full((1, 2, 6), -5.0, device="cuda")
    a = T.decode_attention_kv8(q, kv, sc, n, ws, sel_idx=good.cuda())
    assert ws.status() == 0
    b = T.decode_attention_kv8(q, kv, sc, n, ws, sel_idx=bad.cuda(), scores=scores)
    assert ws.status() == 2
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-6) and scores[0, :, [1, 3, 4]].eq(-5.0).all() and scores[0, :, [0, 2, 5]].ne(-5.0).all()
    ws.reset()
    table = torch.arange(n, dtype=torch.int32)[None].clone()
    table[0, 5], table[0, 6] = -3, n
    keep = torch.tensor([[i for i in range(n) if i not in (5, 6)]], dtype=torch.int32).cuda()
    a = T.decode_attention_kv8(q, kv, sc, n, ws, sel_idx=keep)
    b = T.decode_attention_kv8(q, kv, sc, n, ws, page_table=table.cuda())
    assert ws.status() == 2 and torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_attention_repeats_bit_for_bit(T):
    g = _gen(11)
    codes, scales = _pool(g, 600, 16, 16, 8, 128)
    kv, sc = codes.cuda().view(torch.float8_e4m3fn), scales.cuda()
    q = torch.randn(3, 32, 128, generator=g).to(torch.bfloat16).cuda()
    ws = T.Workspace(3, 32, 128, 1, 1)
    lens = torch.tensor([3200, 100, 1777], dtype=torch.int32, device="cuda")
    runs = [T.decode_attention_kv8(q, kv, sc, 3200, ws, seq_lens=lens) for _ in range(4)]
    assert all(torch.equal(r, runs[0]) for r in runs)


# ----------------------------------------------------------------------- weights
@pytest.mark.parametrize("B,H,N,lens,decay", [(1, 1, 1, [1], 1.0), (1, 32, 1000, [1000], 1.0), (3, 20, 515, [515, 0, 77], 0.9), (2, 7, 4097, [4096, 3], 0.5),
                                              (2, 64, 131, [131, 130], 0.0), (1, 3, 40, [0], 1.0)])
def test_accumulate(T, B, H, N, lens, decay):
    """Each term is off by at most 2^-23 (1 + |s - lse| log2 e) (its argument, the exponential), their sum by H more steps."""
    g = _gen(N)
    s = 3 * torch.randn(B, H, N + 2, generator=g)
    lse = torch.stack([s[b, :, :lens[b]].double().logsumexp(1) for b in range(B)]).float()
    w = torch.rand(B, N + 1, generator=g)
    want = K8.accumulate(s, lse, w, lens, decay)
    got = w.clone().cuda()
    r = T.accumulate_weights(s.cuda(), lse.cuda(), got, N, seq_lens=None if set(lens) == {N} else torch.tensor(lens, dtype=torch.int32, device="cuda"), decay=decay)
    assert r is got
    far = (s[:, :, :N] - lse[..., None])[torch.isfinite(lse)].abs()
    steps = 4 + 2 * float(far.max()) * LOG2E + H if far.numel() else 4
    assert ((got.cpu().double() - want).abs() <= steps * 2.0 ** -23 * want.abs() + 1e-30).all()
    for b in range(B):
        assert torch.equal(got[b, lens[b]:].cpu(), w[b, lens[b]:])


def test_accumulate_of_a_selection_layer_is_one_per_head(T):
    """Weights of one step over an 8-bit and over a 16-bit cache add up to the number of query heads."""
    g = _gen(12)
    D, n, Hq, Hkv = 128, 1500, 8, 2
    kv, sc = T.alloc_kv8(n, 1, Hkv, D)
    k, v = (torch.randn(n, Hkv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    T.append_kv8(k, v, kv, sc)
    q = torch.randn(1, Hq, D, generator=g).to(torch.bfloat16).cuda()
    ws = T.Workspace(1, Hq, D, Hq, n)
    scores, lse = torch.empty(1, Hq, n, device="cuda"), torch.empty(1, Hq, device="cuda")
    T.decode_attention_kv8(q, kv, sc, n, ws, scores=scores, lse=lse)
    w = T.accumulate_weights(scores, lse, torch.zeros(1, n, device="cuda"), n)
    assert abs(float(w.double().sum()) - Hq) < Hq * 1e-5
    pool = T.read_kv8(kv, sc, n, dtype=torch.bfloat16)[0]
    m, l, o = (torch.empty(*s, device="cuda") for s in ((1, Hq), (1, Hq), (1, Hq, D)))
    T.decode_attention(q, pool, n, ws, scores=scores, partials=(m, l, o))
    w2 = T.accumulate_weights(scores, (m + l.log2()) * math.log(2), torch.zeros(1, n, device="cuda"), n)
    assert torch.allclose(w, w2, rtol=1e-4, atol=1e-7)


# ------------------------------------------------------------------------- evict
EVICT = [
    # rows, lens, page, keep, sink, recent
    (1, [100], 1, 60, 4, 8), (1, [1], 1, 1, 0, 1), (3, [300, 299, 120], 16, 9, 1, 2), (2, [5000, 4097], 1, 2048, 0, 1), (4, [77, 0, 16, 33], 16, 2, 0, 1),
    (2, [1025, 64], 3, 100, 2, 98), (1, [40000], 1, 39999, 1, 1), (1, [70001], 16, 3000, 0, 3000), (2, [130, 131], 64, 2, 1, 1), (1, [131072], 1, 1000, 4, 100),
    (1, [200000], 1, 150000, 0, 1), (1, [9], 100, 1, 0, 1),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
@pytest.mark.parametrize("R,lens,page,keep,sink,recent", EVICT)
def test_evict(T, R, lens, page, keep, sink, recent, kind, in_place):
    g = _gen(sum(lens) + keep)
    N = max(lens) + 5
    w = torch.exp(3 * torch.randn(R, N, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, (R, N), generator=g).float()
    elif kind == "odd":
        w = torch.randn(R, N, generator=g)
        w[:, ::7] = math.inf
        w[:, 3::11] = -math.inf
        w[:, 5::13] = math.nan
        w[:, 1::17] = -0.0
    pages = -(-N // page) + 2
    table = torch.stack([torch.randperm(5 * pages, generator=g)[:pages] for _ in range(R)]).to(torch.int32)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    if kind == "odd" and page > 1:
        w = torch.where(w.isinf(), torch.full_like(w, 1e30), w)          # a page with both infinities is NaN in any order of its sum
    want = K8.evict(w, table, lens_t, keep, page, sink, recent)
    src = [t.cuda() for t in (w, table, lens_t)]
    out = None if in_place else tuple(torch.full_like(t, 77) for t in src)
    if out is not None:
        out[1][:, -(-N // page):] = src[1][:, -(-N // page):]            # behind max_len nothing is written
    before = [t.clone() for t in src]
    got = T.evict_pages(*src, keep, page_size=page, sink_pages=sink, recent_pages=recent, out=out)
    if not in_place:
        assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(src, before))
    assert torch.equal(got[2].cpu(), want[2])
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu().view(torch.int32), want[0].view(torch.int32))


def test_evict_keeps_what_attention_needs(T):
    """Attention after an eviction equals attention over the list of kept tokens before it, with pages shared by no one,
    and the tokens appended next go into the dropped pages."""
    g = _gen(13)
    D, Hq, Hkv, page, n = 64, 4, 2, 8, 403
    per = -(-n // page) + 1
    kv, sc = T.alloc_kv8(per, page, Hkv, D, page)
    table = torch.randperm(per, generator=g)[None].to(torch.int32).cuda()
    k, v = (torch.randn(n, Hkv, D, generator=g).cuda() for _ in range(2))
    T.append_kv8(k, v, kv, sc, page_table=table)
    ws = T.Workspace(1, Hq, D, 1, 1)
    q = torch.randn(1, Hq, D, generator=g).cuda()
    w = torch.rand(1, per * page, generator=g).cuda()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    keep, heavy = 20, w[0, :n].cpu().double()
    sums = torch.stack([heavy[i * page:(i + 1) * page].sum() for i in range(per - 1)])
    stay = sorted([0] + (sums[1:-2].argsort(descending=True)[:keep - 3] + 1).tolist() + [per - 3, per - 2])
    listed = torch.tensor([[t for i in stay for t in range(i * page, min(n, (i + 1) * page))]], dtype=torch.int32).cuda()
    want = T.decode_attention_kv8(q, kv, sc, n, ws, page_table=table, sel_idx=listed)
    old = table.clone()
    T.evict_pages(w, table, lens, keep, page_size=page, max_len=n, sink_pages=1, recent_pages=2)
    left = int(lens)
    assert left == listed.shape[1] and sorted(table[0].tolist()) == sorted(old[0].tolist())
    got = T.decode_attention_kv8(q, kv, sc, left, ws, page_table=table)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)
    more = torch.randn(10, Hkv, D, generator=g).cuda()
    T.append_kv8(more, more, kv, sc, pos0=left, page_table=table)
    back = T.read_kv8(kv, sc, left + 10, page_table=table, dtype=torch.float32)
    assert ws.status() == 0 and (back[0, left:, 0, 0] - more).abs().max() < 0.25 * more.abs().max()


# ----------------------------------------------------------------- a run of them
def _decode_steps(T, state, steps):
    """append -> selection attention -> weights (-> top-k -> sparse attention): one layer's operators of a decode step."""
    s = state
    for _ in range(steps):
        T.append_kv8(s["k"], s["v"], s["kv"], s["sc"], batch=s["B"], pos0_dev=s["pos"], page_table=s["table"])
        s["o"] = T.decode_attention_kv8(s["q"], s["kv"], s["sc"], s["N"], s["ws"], page_table=s["table"], seq_lens=s["lens"], scores=s["scores"], lse=s["lse"])
        T.accumulate_weights(s["scores"], s["lse"], s["w"], s["N"], seq_lens=s["lens"], decay=0.9)
        T.topk(s["scores"], s["sel"].shape[-1], s["ws"], out_idx=s["sel"], row_len=s["rows"], out_count=s["counts"])
        s["o2"] = T.decode_attention_kv8(s["q"], s["kv"], s["sc"], s["N"], s["ws"], page_table=s["table"], seq_lens=s["lens"], sel_idx=s["sel"],
                                         sel_counts=s["counts"])
        for t in ("pos", "lens", "rows"):
            s[t].add_(1)


def _state(T, seed, ws=None):
    g = _gen(seed)
    B, Hq, Hkv, D, page, N = 2, 8, 4, 64, 4, 96
    s = dict(B=B, N=N, ws=ws or T.Workspace(B, Hq, D, B * Hq, N))
    s["kv"], s["sc"] = T.alloc_kv8(B * N // page + 3, page, Hkv, D, 4)
    s["table"] = torch.randperm(B * N // page + 3, generator=g)[:B * N // page].view(B, -1).to(torch.int32).cuda()
    s["k"], s["v"], s["q"] = (torch.randn(B, h, D, generator=g).to(torch.bfloat16).cuda() for h in (Hkv, Hkv, Hq))
    k, v = (torch.randn(B * 40, Hkv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    T.append_kv8(k, v, s["kv"], s["sc"], batch=B, page_table=s["table"])
    s["pos"] = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    s["lens"] = s["pos"] + 1
    s["rows"] = s["lens"].repeat_interleave(Hq).contiguous()
    s["scores"], s["lse"] = torch.zeros(B, Hq, N, device="cuda"), torch.zeros(B, Hq, device="cuda")
    s["w"] = torch.zeros(B, N, device="cuda")
    s["sel"], s["counts"] = torch.zeros(B, Hq, 16, dtype=torch.int32, device="cuda"), torch.zeros(B, Hq, dtype=torch.int32, device="cuda")
    return s


def _same_state(a, b):
    for n in ("o", "o2", "scores", "lse", "w", "sel", "counts", "sc"):
        assert torch.equal(a[n], b[n]), n
    assert torch.equal(a["kv"].view(torch.uint8), b["kv"].view(torch.uint8))


def test_decode_loop_eager_other_stream_and_graph(T):
    """The same ten steps eagerly, on a stream of their own, and as a captured step replayed: the same bits."""
    eager = _state(T, 1)
    _decode_steps(T, eager, 10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = _state(T, 1)
        _decode_steps(T, other, 10)
    stream.synchronize()
    captured = _state(T, 1)
    _decode_steps(T, captured, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _decode_steps(T, captured, 1)
    for _ in range(9):
        graph.replay()
    torch.cuda.synchronize()
    _same_state(eager, other)
    _same_state(eager, captured)
    assert eager["ws"].status() == 0 and other["ws"].status() == 0


def test_two_graphs_share_a_workspace(T):
    """Two captured steps on one workspace, replayed in turn on one stream, give what they give alone."""
    alone = [_state(T, i) for i in (1, 2)]
    for s in alone:
        _decode_steps(T, s, 6)
    both = [_state(T, i) for i in (1, 2)]
    both[1]["ws"] = both[0]["ws"]
    graphs = []
    for s in both:
        _decode_steps(T, s, 1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _decode_steps(T, s, 1)
        graphs.append(graph)
    for _ in range(5):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        _same_state(a, b)


def test_prefill_reads_the_cache_back(T):
    """A prompt in two chunks: append, read back, tidal_prefill over the rows — equal to attention over the stored values."""
    g = _gen(14)
    D, Hq, Hkv, n, n_q = 128, 4, 2, 300, 130
    kv, sc = T.alloc_kv8(20, 16, Hkv, D, 16)
    k, v = (torch.randn(n, Hkv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    T.append_kv8(k[:n - n_q], v[:n - n_q], kv, sc)
    T.append_kv8(k[n - n_q:], v[n - n_q:], kv, sc, pos0=n - n_q)
    pool = T.read_kv8(kv, sc, n, dtype=torch.bfloat16)[0]
    q = torch.randn(n_q, Hq, D, generator=g).to(torch.bfloat16).cuda()
    o = T.prefill(q, pool, torch.arange(n, dtype=torch.int32, device="cuda"), n).cpu().double()
    vals = K8.values(kv.cpu(), sc.cpu()).transpose(1, 2).reshape(-1, 2, Hkv, D)
    for i in (0, 57, n_q - 1):
        for h in range(Hq):
            m = n - n_q + i + 1
            want, _, _, A, _ = K8.attention(q[i, h].cpu(), vals[:m, 0, h // 2], vals[:m, 1, h // 2], 1 / math.sqrt(D))
            # bf16 result and bf16 softmax weights of the prefill kernel: half a step each
            assert ((o[i, h] - want).abs() <= 2.0 ** -8 * (want.abs() + 2 * A)).all()
