"""Workloads of the 8-bit KV cache operators: what a decode step does over a paged cache whose keys and values are held in
e4m3 with a power-of-two scale for every block of tokens and KV head, and what bounds such a cache (attention weights added
up per token, pages of little weight dropped).

    store    ops.append_kv8 of new tokens, then ops.read_kv8 of the blocks they touched (a prompt's prefill reads them)
    attend   ops.decode_attention_kv8: one query token per sequence over the cache, or over lists of cached tokens
    weigh    ops.accumulate_weights: softmax weights of a selection layer's logits, added per cached token
    evict    ops.evict_pages: the lightest pages leave the page table

`own` chooses between the framework's kernels and their plain form in elementary torch operations (32 bits).
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
WIDTH = {"f16": 2, "bf16": 2, "f32": 4}
# the pool keeps a few pages more than the sequences use, and hands them out in no order
SPARE_PAGES = 5


# --------------------------------------------------------------------------- cases
def _attend(name, batch, heads, kv_heads, head_dim, longest, ragged, page, block, dtype, logits=False, lists="all", selected=0):
    return dict(name=name, op="attend", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, longest=longest, ragged=ragged,
                page=page, block=block, dtype=dtype, logits=logits, lists=lists, selected=selected)


def _store(name, batch, tokens, start, kv_heads, head_dim, page, block, dtype):
    return dict(name=name, op="store", batch=batch, tokens=tokens, start=start, kv_heads=kv_heads, head_dim=head_dim, page=page, block=block,
                dtype=dtype)


def _weigh(name, batch, heads, longest, ragged, decay):
    return dict(name=name, op="weigh", batch=batch, heads=heads, longest=longest, ragged=ragged, decay=decay)


def _evict(name, rows, longest, ragged, page, keep, sink, recent):
    return dict(name=name, op="evict", rows=rows, longest=longest, ragged=ragged, page=page, keep=keep, sink=sink, recent=recent)


def listed():
    return [
        # the first tokens of a chat: one sequence, a context that ends inside a page; latency counts
        _attend("attend_short", 1, 32, 8, 128, 131, False, 16, 16, "bf16"),
        # a selection layer of a 32-head model at 32 K tokens, one token per page: the logits go on to the top-k
        _attend("attend_logits_32k", 1, 32, 32, 128, 32768, False, 1, 1, "f16", logits=True),
        # a serving batch of grouped-query sequences of very different lengths: the full layers of a decode step
        _attend("attend_ragged_batch", 64, 32, 8, 128, 32768, True, 16, 16, "bf16"),
        # a sparse layer: every query head has its own list of chosen tokens out of a long context
        _attend("attend_lists", 2, 32, 8, 128, 100003, False, 1, 1, "f16", lists="per_head", selected=2048),
        # a small model kept in 32 bits for comparisons: group of five, odd page size, ragged, logits wanted
        _attend("attend_f32_odd", 5, 20, 4, 64, 5003, True, 7, 7, "f32", logits=True),
        # a decode step's new token of 64 sequences, in the middle of a block that holds tokens already
        _store("store_token", 64, 1, 1003, 8, 128, 16, 16, "bf16"),
        # a chunk of a prompt for three sequences that already hold tokens; nothing is aligned
        _store("store_chunk", 3, 777, 1029, 4, 64, 7, 7, "f32"),
        # a long prompt in one go
        _store("store_prompt", 1, 32768, 0, 32, 128, 16, 16, "f16"),
        # weights of one sequence's selection layer in mid conversation
        _weigh("weigh_one", 1, 32, 4099, False, 1.0),
        # weights of a batch of long sequences, older steps fading
        _weigh("weigh_batch", 8, 32, 131072, True, 0.98),
        # one sequence over its budget of single-token pages
        _evict("evict_one", 1, 4096, False, 1, 2048, 4, 256),
        # a table per layer: 32 long rows of 16-token pages, halved
        _evict("evict_layers", 32, 131072, True, 16, 4096, 1, 64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _page_block(rng):
    page = rng.choice((1, 3, 7, 16, 24, 32, 64))
    return page, rng.choice([d for d in (1, 2, 3, 4, 7, 8, 16, 24, 32, 64) if page % d == 0])


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "store", "store", "weigh", "evict"))
    dtype = rng.choice(tuple(TYPES))
    if op == "attend":
        heads, kv = rng.choice(((32, 32), (32, 8), (8, 8), (20, 4), (16, 1), (64, 8), (40, 8), (12, 6), (4, 4), (14, 2), (48, 2)))
        dim = rng.choice((64, 128))
        page, block = _page_block(rng)
        lists = rng.choice(("all", "all", "shared", "per_head"))
        batch = _log(rng, 1, 32)
        longest = _log(rng, 1, min(131072, max(64, (400 << 20) // (batch * kv * dim))))
        selected = 0
        if lists != "all":
            batch = min(batch, 4)
            selected = _log(rng, 1, min(longest, 4096))
        return {k: v for k, v in _attend("", batch, heads, kv, dim, longest, rng.random() < 0.5, page, block, dtype, rng.random() < 0.4,
                                         lists, selected).items() if k != "name"}
    if op == "store":
        page, block = _page_block(rng)
        kv, dim = rng.choice((1, 2, 4, 5, 8, 16, 32)), rng.choice((64, 128))
        batch = _log(rng, 1, 64)
        tokens = 1 if rng.random() < 0.3 else _log(rng, 1, max(2, (128 << 20) // (batch * kv * dim * 8)))
        return {k: v for k, v in _store("", batch, tokens, rng.choice((0, _log(rng, 1, 4000))), kv, dim, page, block, dtype).items() if k != "name"}
    if op == "weigh":
        batch, heads = _log(rng, 1, 16), rng.choice((1, 4, 8, 20, 32, 64))
        longest = _log(rng, 1, min(131072, (1 << 25) // (batch * heads)))
        return {k: v for k, v in _weigh("", batch, heads, longest, rng.random() < 0.5, rng.choice((1.0, 0.9))).items() if k != "name"}
    page = rng.choice((1, 1, 3, 16, 64))
    rows, longest = _log(rng, 1, 32), _log(rng, 2 * page, 131072)
    pages = -(-longest // page)
    keep = max(1, int(pages * rng.uniform(0.2, 0.95)))
    recent = max(1, int(keep * rng.uniform(0.0, 0.5)))
    return {k: v for k, v in _evict("", rows, longest, rng.random() < 0.5, page, keep, min(rng.choice((0, 1, 4)), keep - recent), recent).items()
            if k != "name"}


# ------------------------------------------------------- the format, in plain torch
def _exponent(amax):
    """Smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the largest e4m3 value); an empty block takes the smallest scale."""
    f, x = torch.frexp(amax)                         # amax = f * 2^x, 0.5 <= f < 1
    e = x.to(torch.int32) - 9 + (f > 0.875).to(torch.int32)
    return torch.where(amax > 0, e.clamp(min=-126), torch.full_like(e, -126))


def _pow2(e):
    """2^e as a 32-bit float, from its exponent field."""
    return ((e.int().clamp(-126, 127) + 127) << 23).view(torch.float32)


def _magnitude(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


def _codes(x, e):
    """e4m3 codes of x at scale 2^e; infinities end at the largest value."""
    return (x * _pow2(-e)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, scale_bytes):
    return codes.view(torch.float8_e4m3fn).float() * (scale_bytes.int() << 23).view(torch.float32)


def _new_pool(c, pages, device):
    kv = torch.zeros(pages, 2, c["page"], c["kv_heads"], c["head_dim"], dtype=torch.uint8, device=device)
    return kv, torch.zeros(pages, 2, c["page"] // c["block"], c["kv_heads"], dtype=torch.uint8, device=device)


def _table(g, batch, per_seq, device):
    n = batch * per_seq + SPARE_PAGES
    return torch.randperm(n, generator=g, device=device)[: batch * per_seq].view(batch, per_seq).to(torch.int32), n


def _fill(g, c, kv, scales):
    """Keys and values as a model leaves them: keys with a few strong channels, values without; quantised block by block."""
    pages, _, page, heads, dim = kv.shape
    step = max(1, (1 << 26) // (page * heads * dim))
    gain = 1.0 + 3.0 * (torch.rand(heads, dim, generator=g, device=kv.device) > 0.97)
    for p0 in range(0, pages, step):
        part = kv[p0:p0 + step]
        x = torch.randn(part.shape, generator=g, device=kv.device)
        x[:, 0] *= gain
        x = x.view(part.shape[0], 2, page // c["block"], c["block"], heads, dim)
        e = _exponent(x.abs().amax(dim=(3, 5)))
        scales[p0:p0 + step] = (e + 127).to(torch.uint8)
        part.copy_(_codes(x, e[:, :, :, None, :, None]).view(part.shape))


def _lengths(g, n, longest, ragged, device):
    if not ragged:
        return torch.full((n,), longest, dtype=torch.int32, device=device)
    x = torch.rand(n, generator=g, device=device)
    lens = torch.exp(math.log(longest) * (0.4 + 0.6 * x)).round().clamp(1, longest).to(torch.int32)
    lens[0] = longest
    return lens


# ------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=c, **dict(attend=_prepare_attend, store=_prepare_store, weigh=_prepare_weigh, evict=_prepare_evict)[c["op"]](c, g, dev))
    if own and c["op"] == "attend":
        from tidaldecode_b200 import ops

        s["ws"] = ops.Workspace(c["batch"], c["heads"], c["head_dim"], 1, 1)
    return s


def _prepare_attend(c, g, dev):
    B, H, D, N = c["batch"], c["heads"], c["head_dim"], c["longest"]
    per_seq = -(-N // c["page"])
    table, pages = _table(g, B, per_seq, dev)
    kv, scales = _new_pool(c, pages, dev)
    _fill(g, c, kv, scales)
    s = dict(q=torch.randn(B, H, D, generator=g, device=dev).to(TYPES[c["dtype"]]), kv=kv.view(torch.float8_e4m3fn), scales=scales, table=table,
             lens=_lengths(g, B, N, c["ragged"], dev), sel=None, counts=None, logits=None)
    entries = N
    if c["lists"] != "all":
        entries = c["selected"]
        heads = () if c["lists"] == "shared" else (H,)
        lens = s["lens"].view(B, *(1 for _ in heads))
        if c["ragged"]:
            s["counts"] = lens.clamp(max=entries).expand(B, *heads).contiguous()
        # chosen positions, ascending; a list longer than its sequence is cut by its count
        x = torch.rand(B, *heads, N, generator=g, device=dev)
        x = torch.where(torch.arange(N, device=dev) < lens[..., None], x, torch.full_like(x, 2.0))
        idx = x.topk(entries, dim=-1, largest=False).indices
        s["sel"] = idx.sort(dim=-1).values.to(torch.int32)
    if c["logits"]:
        s["logits"] = torch.zeros(B, H, entries, device=dev)
        s["lse"] = torch.zeros(B, H, device=dev)
    return s


def _prepare_store(c, g, dev):
    B, T, end = c["batch"], c["tokens"], c["start"] + c["tokens"]
    table, pages = _table(g, B, -(-end // c["page"]), dev)
    kv, scales = _new_pool(c, pages, dev)
    _fill(g, c, kv, scales)
    shape = (B * T, c["kv_heads"], c["head_dim"])
    k, v = (torch.randn(shape, generator=g, device=dev) * (2.0 * torch.rand(shape[:2] + (1,), generator=g, device=dev)) for _ in range(2))
    return dict(k=k.to(TYPES[c["dtype"]]), v=v.to(TYPES[c["dtype"]]), kv=kv.view(torch.float8_e4m3fn), scales=scales, table=table)


def _prepare_weigh(c, g, dev):
    B, H, N = c["batch"], c["heads"], c["longest"]
    lens = _lengths(g, B, N, c["ragged"], dev)
    scores = 2.0 * torch.randn(B, H, N, generator=g, device=dev)
    live = torch.arange(N, device=dev) < lens[:, None, None]
    lse = torch.where(live, scores, torch.full_like(scores, -math.inf)).logsumexp(-1)
    return dict(scores=scores, lse=lse, lens=lens, weights=torch.rand(B, N, generator=g, device=dev))


def _prepare_evict(c, g, dev):
    R, N, page = c["rows"], c["longest"], c["page"]
    per_row = -(-N // page)
    # rows of one table per layer: every row lists pages of its own layer's pool
    table = torch.rand(R, per_row, generator=g, device=dev).argsort(dim=-1).to(torch.int32)
    w = torch.exp(3.0 * torch.randn(R, N, generator=g, device=dev))
    w = torch.where(torch.rand(R, N, generator=g, device=dev) < 0.1, torch.zeros_like(w), w)       # tokens nothing attended to
    return dict(weights=w, table=table, lens=_lengths(g, R, N, c["ragged"], dev), weights_out=w.clone(), table_out=table.clone(),
                lens_out=torch.zeros(R, dtype=torch.int32, device=dev))


# -------------------------------------------------------------------------- a pass
def run(state):
    return dict(attend=_run_attend, store=_run_store, weigh=_run_weigh, evict=_run_evict)[state["case"]["op"]](state)


def _run_attend(s):
    c = s["case"]
    if own:
        from tidaldecode_b200 import ops

        out = ops.decode_attention_kv8(s["q"], s["kv"], s["scales"], c["longest"], s["ws"], page_table=s["table"],
                                       seq_lens=s["lens"] if c["ragged"] else None, sel_idx=s["sel"], sel_counts=s["counts"],
                                       scores=s["logits"], lse=s.get("lse"))
        return dict(out=out, logits=s["logits"], lse=s.get("lse"))
    q, kv, scales, page = s["q"].float(), s["kv"].view(torch.uint8), s["scales"], c["page"]
    B, H, D = q.shape
    G = H // c["kv_heads"]
    dev = q.device
    sm = 1.0 / math.sqrt(D)
    if c["lists"] == "per_head":
        pos, live = s["sel"].long(), _live(s, c["selected"]).expand(B, H, -1)                        # [B, H, n]
        pages = torch.gather(s["table"].long()[:, None].expand(B, H, -1), 2, pos // page)
        head = (torch.arange(H, device=dev) // G)[None, :, None]
        k, v = (_values(kv[pages, j, pos % page, head], scales[pages, j, pos % page // c["block"], head][..., None]) for j in (0, 1))
        x = (k * q[:, :, None]).sum(-1) * sm
    else:
        n = c["longest"] if s["sel"] is None else c["selected"]
        pos = torch.arange(n, device=dev).expand(B, n) if s["sel"] is None else s["sel"].long()
        live = _live(s, n).expand(B, H, n)
        pages = torch.gather(s["table"].long(), 1, pos // page)
        k, v = (_values(kv[pages, j, pos % page], scales[pages, j, pos % page // c["block"]][..., None]) for j in (0, 1))      # [B, n, Hkv, D]
        x = (q.view(B, -1, G, D) @ k.permute(0, 2, 3, 1)).reshape(B, H, n) * sm
    y = torch.where(live, x, torch.full_like(x, -math.inf))
    top = y.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = torch.exp(y - top)
    total = p.sum(-1, keepdim=True)
    if c["lists"] == "per_head":
        o = (p[..., None] * v).sum(2)
    else:
        o = (p.view(B, -1, G, p.shape[-1]) @ v.permute(0, 2, 1, 3)).reshape(B, H, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).to(s["q"].dtype)
    if not c["logits"]:
        return dict(out=o, logits=None, lse=None)
    s["logits"].copy_(torch.where(live, x, s["logits"]))
    s["lse"].copy_((top + total.log())[..., 0])
    return dict(out=o, logits=s["logits"], lse=s["lse"])


def _live(s, n):
    """[B, 1 or H, n]: which entries of a list (or positions) count."""
    lens = s["counts"] if s["sel"] is not None and s["counts"] is not None else s["lens"] if s["sel"] is None else None
    if lens is None:
        return torch.ones(1, 1, n, dtype=torch.bool, device=s["q"].device)
    return torch.arange(n, device=lens.device) < (lens[:, None, None] if lens.dim() == 1 else lens[..., None])


def _run_store(s):
    c = s["case"]
    B, T, start, block, page = c["batch"], c["tokens"], c["start"], c["block"], c["page"]
    first, end = start // block * block, start + T
    if own:
        from tidaldecode_b200 import ops

        ops.append_kv8(s["k"], s["v"], s["kv"], s["scales"], batch=B, pos0=start, page_table=s["table"])
        return ops.read_kv8(s["kv"], s["scales"], end, start=first, batch=B, page_table=s["table"], dtype=s["k"].dtype)
    kv, scales, table = s["kv"].view(torch.uint8), s["scales"], s["table"].long()
    H, D = s["k"].shape[1:]
    n_blocks = -(-(end - first) // block)
    x = torch.stack((s["k"], s["v"])).float().view(2, B, T, H, D)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, start - first, n_blocks * block - (end - first)))
    at = torch.arange(first, first + n_blocks * block, block, device=kv.device)
    e = _exponent(_magnitude(x).view(2, B, n_blocks, block, H, D).amax(dim=(3, 5)))                    # [2, B, blocks, H]
    plane = torch.arange(2, device=kv.device)[:, None, None]
    held = start > first                                                                              # the first block holds tokens already
    if held:
        before = scales[table[None, :, first // page, None], plane, first % page // block].int() - 127   # [2, B, 1, H]
        e = torch.cat((torch.maximum(e[:, :, :1], before), e[:, :, 1:]), 2)
    pos = torch.arange(start, end, device=kv.device)
    wide = e.repeat_interleave(block, 2)[..., None]                                                   # [2, B, n, H, 1]
    new = _codes(x[:, :, start - first:end - first], wide[:, :, start - first:end - first])
    if held:
        old = torch.arange(first, start, device=kv.device)
        where = (table[None, :, old // page], plane, (old % page)[None, None])
        moved = kv[where].view(torch.float8_e4m3fn).float()
        kv[where] = _codes(moved, (e[:, :, :1] - before)[..., None])
    kv[table[None, :, pos // page], plane, (pos % page)[None, None]] = new
    scales[table[None, :, at // page], plane, (at % page // block)[None, None]] = (e + 127).to(torch.uint8)
    pos = torch.arange(first, end, device=kv.device)
    where = table[:, pos // page], (pos % page)[None]
    got = _values(kv[where[0][..., None], torch.arange(2, device=kv.device), where[1][..., None]],
                  scales[where[0][..., None], torch.arange(2, device=kv.device), where[1][..., None] // block][..., None])
    most = torch.finfo(s["k"].dtype).max
    return got.clamp(-most, most).to(s["k"].dtype)[:, :, :, None]                                       # [B, n, 2, 1, H, D]


def _run_weigh(s):
    c = s["case"]
    if own:
        from tidaldecode_b200 import ops

        return ops.accumulate_weights(s["scores"], s["lse"], s["weights"], c["longest"], seq_lens=s["lens"] if c["ragged"] else None,
                                      decay=c["decay"])
    w = torch.exp(s["scores"] - s["lse"][..., None]).sum(1)
    live = torch.arange(c["longest"], device=w.device) < s["lens"][:, None]
    s["weights"].copy_(torch.where(live, c["decay"] * s["weights"] + w, s["weights"]))
    return s["weights"]


def _run_evict(s):
    c = s["case"]
    w, table, lens, page, keep = s["weights"], s["table"], s["lens"], c["page"], c["keep"]
    if own:
        from tidaldecode_b200 import ops

        ops.evict_pages(w, table, lens, keep, page_size=page, max_len=c["longest"], sink_pages=c["sink"], recent_pages=c["recent"],
                        out=(s["weights_out"], s["table_out"], s["lens_out"]))
        return dict(weights=s["weights_out"], table=s["table_out"], lens=s["lens_out"])
    R, N = w.shape
    P = table.shape[1]
    dev = w.device
    tok = torch.arange(N, device=dev)
    pg = torch.arange(P, device=dev)
    used = (lens.long() + page - 1) // page                                                           # pages in use, [R]
    held = torch.where(tok < lens[:, None], w, torch.zeros_like(w)).double()
    heavy = torch.nn.functional.pad(held, (0, P * page - N)).view(R, P, page).sum(-1).float()         # a page's weight, summed in 64 bits
    sure = (pg < c["sink"]) | (pg >= used[:, None] - c["recent"])
    rank = torch.where(sure, torch.full_like(heavy, math.inf), heavy)
    rank = torch.where(pg < used[:, None], rank, torch.full_like(heavy, -math.inf))
    order = rank.argsort(dim=-1, descending=True, stable=True)                                        # ties: the lower page first
    stay = torch.zeros(R, P, dtype=torch.bool, device=dev).scatter_(1, order[:, :keep], True)
    stay = (stay | (used[:, None] <= keep)) & (pg < used[:, None])
    # kept pages first, dropped ones behind them, then what the row holds beyond its length
    group = torch.where(stay, 0, torch.where(pg < used[:, None], 1, 2))
    order = group.argsort(dim=-1, stable=True)
    s["table_out"].copy_(torch.gather(table, 1, order))
    dropped = used - stay.sum(1)
    s["lens_out"].copy_(lens - (dropped * page).to(torch.int32))
    kept_tok = torch.gather(stay, 1, (tok // page).expand(R, N)) & (tok < lens[:, None])
    order = torch.where(kept_tok, 0, torch.where(tok < lens[:, None], 1, 2)).argsort(dim=-1, stable=True)
    moved = torch.gather(torch.where(kept_tok | (tok >= lens[:, None]), w, torch.zeros_like(w)), 1, order)
    s["weights_out"].copy_(moved)
    return dict(weights=s["weights_out"], table=s["table_out"], lens=s["lens_out"])


# ----------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "attend":
        # lengths of a ragged batch are drawn like exp(log(longest) * u), u from 0.4 to 1, the first one the longest
        N, top = c["longest"], math.log(max(c["longest"], 2))
        mean = N if not c["ragged"] else (N + (c["batch"] - 1) * (math.exp(top) - math.exp(0.4 * top)) / (0.6 * top)) / c["batch"]
        rows = c["kv_heads"]
        if c["lists"] != "all":
            mean = min(c["selected"], mean)
            rows = c["heads"] if c["lists"] == "per_head" else rows
        read = c["batch"] * mean * rows * 2 * (c["head_dim"] + 1.0 / (c["block"] if c["lists"] == "all" else 1))
        per_token = 4.0 / c["page"] if c["lists"] == "all" else 8.0 * (c["heads"] if c["lists"] == "per_head" else 1)
        small = 2 * c["batch"] * c["heads"] * c["head_dim"] * WIDTH[c["dtype"]]
        logits = 4 * c["batch"] * c["heads"] * mean if c["logits"] else 0
        return {"bytes": read + c["batch"] * mean * per_token + small + logits, "flops": 4.0 * c["batch"] * c["heads"] * c["head_dim"] * mean}
    if c["op"] == "store":
        n = c["batch"] * 2 * c["kv_heads"]
        read = c["start"] % c["block"] + c["tokens"]
        values = n * c["head_dim"]
        return {"bytes": values * (WIDTH[c["dtype"]] * (c["tokens"] + read) + c["tokens"]) + n * read / c["block"], "flops": 2.0 * values * read}
    if c["op"] == "weigh":
        N, top = c["longest"], math.log(max(c["longest"], 2))
        total = c["batch"] * N if not c["ragged"] else N + (c["batch"] - 1) * (math.exp(top) - math.exp(0.4 * top)) / (0.6 * top)
        return {"bytes": 4.0 * total * (c["heads"] + 2) + 4.0 * c["batch"] * c["heads"], "flops": 3.0 * total * c["heads"]}
    N, top = c["longest"], math.log(max(c["longest"], 2))
    total = c["rows"] * N if not c["ragged"] else N + (c["rows"] - 1) * (math.exp(top) - math.exp(0.4 * top)) / (0.6 * top)
    return {"bytes": 8.0 * total + 8.0 * total / c["page"] + 8.0 * c["rows"], "flops": total}


# ----------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    by_op = dict(attend=_exact_attend, store=_exact_store, weigh=_exact_weigh, evict=_exact_evict)
    return by_op[case["op"]](prepare(case, seed))


def _two(e):
    """2^e in 64 bits, from its exponent field."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _decode64(codes, scale_bytes):
    """Value of every e4m3 code from its fields, times its scale, in 64 bits."""
    b = codes.long()
    frac, ex = (b & 7).double(), b >> 3 & 15
    mag = torch.where(ex > 0, (8.0 + frac) * _two(ex - 10), frac * 2.0 ** -9)
    mag = torch.where(b & 127 == 127, torch.full_like(mag, math.nan), mag)
    return torch.where(b >= 128, -mag, mag) * _two(scale_bytes.long() - 127)


def _exact_attend(s):
    c = s["case"]
    B, H, D = s["q"].shape
    G = H // c["kv_heads"]
    kv, page, block = s["kv"].view(torch.uint8), c["page"], c["block"]
    out = torch.zeros(B, H, D, dtype=torch.float64, device=kv.device)
    logits = s["logits"].double().clone() if c["logits"] else None
    lse = torch.zeros(B, H, dtype=torch.float64, device=kv.device) if c["logits"] else None
    for b in range(B):
        for h in range(c["kv_heads"]):
            for group in ([slice(h * G, (h + 1) * G)] if c["lists"] != "per_head" else [slice(i, i + 1) for i in range(h * G, (h + 1) * G)]):
                n = int(s["lens"][b])
                pos = torch.arange(n, device=kv.device)
                if c["lists"] != "all":
                    row = s["sel"][b] if c["lists"] == "shared" else s["sel"][b, group.start]
                    pos = row[: min(c["selected"], n)].long()
                pages, slot = s["table"][b].long()[pos // page], pos % page
                k, v = (_decode64(kv[pages, j, slot, h], s["scales"][pages, j, slot // block, h][:, None]) for j in (0, 1))
                x = s["q"][b, group].double() @ k.T / math.sqrt(D)
                z = x.logsumexp(-1, keepdim=True)
                out[b, group] = torch.exp(x - z) @ v
                if c["logits"]:
                    logits[b, group, : x.shape[1]] = x
                    lse[b, group] = z[:, 0]
    return dict(out=out, logits=logits, lse=lse)


def _round_e4m3(y):
    """To the nearest e4m3 value, ties to even, in 64 bits: 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    ex = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
    step = _two(ex - 3.0)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_store(s):
    c = s["case"]
    B, T, start, block, page = c["batch"], c["tokens"], c["start"], c["block"], c["page"]
    first, end = start // block * block, start + T
    kv = s["kv"].view(torch.uint8)
    got = []
    for plane, new in ((0, s["k"]), (1, s["v"])):
        new = new.double().view(B, T, c["kv_heads"], c["head_dim"])
        if start > first:
            old = torch.arange(first, start, device=kv.device)
            pages = s["table"].long()[:, old // page]
            scale = s["scales"][pages, plane, old % page // block]
            held = _decode64(kv[pages, plane, old % page], scale[..., None])
            floor = scale[:, :1].double() - 127.0
            x = torch.cat((held, new), 1)
        else:
            floor, x = None, new
        n = x.shape[1]
        full = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -n % block)).view(B, -1, block, c["kv_heads"], c["head_dim"])
        fresh = torch.nn.functional.pad(new, (0, 0, 0, 0, start - first, -n % block)).view_as(full)
        most = fresh.abs().amax(dim=(2, 4))                                                         # new tokens of each block
        e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -140) / 448.0))
        e = torch.where(most <= 448.0 * _two(e - 1.0), e - 1.0, e)
        e = torch.where(most > 448.0 * _two(e), e + 1.0, e).clamp(min=-126.0)
        if floor is not None:
            e[:, :1] = torch.maximum(e[:, :1], floor)
        unit = _two(e[:, :, None, :, None])
        got.append((_round_e4m3(full / unit) * unit).view(B, -1, c["kv_heads"], c["head_dim"])[:, :n])
    return torch.stack(got, 2)[:, :, :, None]


def _exact_weigh(s):
    c = s["case"]
    w = s["weights"].double()
    for b in range(c["batch"]):
        n = int(s["lens"][b])
        w[b, :n] = c["decay"] * w[b, :n] + torch.exp(s["scores"][b, :, :n].double() - s["lse"][b].double()[:, None]).sum(0)
    return w


def _exact_evict(s):
    c = s["case"]
    page, keep = c["page"], c["keep"]
    weights, table, lens = s["weights"].double(), s["table"].clone(), s["lens"].clone()
    for r in range(c["rows"]):
        n = int(s["lens"][r])
        used = -(-n // page)
        if used <= keep:
            continue
        w = s["weights"][r, :n].double()
        heavy = torch.zeros(used, dtype=torch.float64, device=w.device).index_add_(0, torch.arange(n, device=w.device) // page, w).float()
        lo, hi = c["sink"], used - c["recent"]
        middle = heavy[lo:hi]
        best = sorted(zip((-middle).tolist(), range(lo, hi)))[: keep - c["sink"] - c["recent"]]
        stay = torch.tensor(sorted(list(range(lo)) + [i for _, i in best] + list(range(hi, used))), device=w.device)
        gone = torch.ones(used, dtype=torch.bool, device=w.device)
        gone[stay] = False
        table[r, :used] = torch.cat((s["table"][r][stay], s["table"][r, :used][gone]))
        at = (stay[:, None] * page + torch.arange(page, device=w.device)).view(-1)
        at = at[at < n]
        weights[r, :n] = 0.0
        weights[r, : at.numel()] = w[at]
        lens[r] = at.numel()
    return dict(weights=weights, table=table, lens=lens)
