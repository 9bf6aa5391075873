"""What stands beside a bounded cache: Quest metadata that follow the cache, generation that runs on, eviction that has
something to go by."""
from __future__ import annotations

import pytest
import torch

from oracle import kv8_oracle as K8
from oracle import tidal_oracle as O
from tests.test_gpu_kv8_model import _controller
from tests.test_gpu_model import _tiny_model

pytestmark = pytest.mark.gpu


def _estimates_are_the_keys(c, U, q, layers, stored):
    """Pages hold one token, so the bound of a page is the token's logit itself: 64 products and their sum in 32 bits."""
    for layer in layers:
        got = U.decode_estimate(q, c, layer).cpu().double()
        keys = stored[layer][:got.shape[1]]                                          # [n - 1, Hkv, D]
        for h in range(q.shape[1]):
            terms = keys[:, h // 4].double() * q[0, h].cpu().double()
            assert ((got[h] - terms.sum(1)).abs() <= 64 * 2.0 ** -24 * terms.abs().sum(1)).all(), (layer, h)


def _in_order(c, layer):
    """The cached keys of sequence 0 in slot order."""
    pages = torch.tensor(c.kv_cache._indicies[0][:c.kv_cache.seqlen])
    return c.kv_cache.buf_layer(layer)[pages.cuda(), 0, 0].cpu()


@pytest.mark.parametrize("layer_alias", [1, 2])
def test_quest_metadata_of_a_controller(layer_alias):
    """append_kv keeps the per-page key bounds, decode_estimate reads them, per layer (or per pool that layers share)."""
    import tidaldecode_b200.utils as U
    g = torch.Generator().manual_seed(1)
    n = 70
    c = _controller(16, False, dtype=torch.float32, quest_metadata=True, layer_alias=layer_alias)
    for new in (n, 1, 1):
        c.prepare_metadata(new)
        c.begin_forward(new)
        for layer in range(2):
            k, v = (torch.randn(new, 2, 64, generator=g).cuda() for _ in range(2))
            U.append_kv(k, v, c, layer)
    q = torch.randn(1, 8, 64, generator=g).cuda()
    _estimates_are_the_keys(c, U, q, range(2), [_in_order(c, layer) for layer in range(2)])


@pytest.mark.parametrize("layer_alias", [1, 2])
def test_quest_metadata_follow_an_eviction(layer_alias):
    """After slots have been renumbered a page's bounds are those of the token it holds now, in every layer; so are those of
    the tokens appended next."""
    import tidaldecode_b200.utils as U
    g = torch.Generator().manual_seed(2)
    n, keep = 90, 40
    c = _controller(16, True, dtype=torch.float32, quest_metadata=True, layer_alias=layer_alias)
    q = torch.randn(1, 8, 64, generator=g).cuda()

    def append(new):
        c.prepare_metadata(new)
        c.begin_forward(new)
        for layer in range(2):
            k, v = (torch.randn(new, 2, 64, generator=g).cuda() for _ in range(2))
            U.append_kv(k, v, c, layer)

    append(n)
    append(1)
    U.decode_sparse_attn(q, c, 0, c.kv_indices_without_last, True)
    before = c.kv_cache._indicies[0][:n + 1]
    assert U.evict_kv(c, keep, 2, 5) == n + 1 - keep and c.kv_cache._indicies[0][:keep] != before[:keep]
    _estimates_are_the_keys(c, U, q, range(2), [_in_order(c, layer) for layer in range(2)])
    append(1)
    append(1)
    _estimates_are_the_keys(c, U, q, range(2), [_in_order(c, layer) for layer in range(2)])


def test_a_bounded_cache_generates_without_end():
    """170 tokens through a cache of 96, with evictions between the calls: replayed, eager and in calls of one token the same
    tokens, and what earlier calls returned stays as it was."""
    from tidaldecode_b200.runtime import GraphDecoder
    W = O.TinyLlamaWeights(vocab=512, hidden=512, layers=4, heads=8, kv_heads=2, ffn=352, seed=5, dtype=torch.bfloat16)
    prompt = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(3))
    runs = []
    for use_graph, at_once in ((True, True), (False, True), (True, False)):
        rt = GraphDecoder(_tiny_model(W, torch.bfloat16, (1, 3), "none", True, 2), max_seq_len=96, token_budget=16, kv_bits=8, track_weights=True)
        rt.prefill(prompt)
        parts, copies = [], []
        for steps in (20, 50, 50, 50):
            got = [rt.decode(steps, use_graph=use_graph)] if at_once else [rt.decode(1, use_graph=use_graph) for _ in range(steps)]
            assert torch.equal(got[-1][:, -1:], rt.tok)
            parts += got
            copies += [x.clone() for x in got]
            rt.evict(40, sink_tokens=2, recent_tokens=8)
            assert rt.c.kv_cache.seqlen == 40
        assert int(rt.pos) == 60 + 170 and int(rt.slot) == 40 and rt.c.workspace.status() == 0 and int(rt.lin_status) == 0
        with pytest.raises(RuntimeError, match="max_seq_len"):
            rt.decode(57, use_graph=use_graph)
        assert all(torch.equal(a, b) for a, b in zip(parts, copies))
        runs.append(torch.cat(parts, 1))
        assert runs[-1].shape == (1, 170)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    # a new conversation starts over
    rt.prefill(prompt)
    assert torch.equal(rt.decode(20), runs[0][:, :20])


def test_eviction_needs_weights():
    """Straight after a prompt no token has a weight: dropping "the lightest" is refused and changes nothing, while the first
    and the last tokens alone can be kept, and a cache within its budget is left alone."""
    import tidaldecode_b200.utils as U
    g = torch.Generator().manual_seed(4)
    c = _controller(8, True, B=2)
    c.prepare_metadata(100)
    c.begin_forward(100)
    k, v = (torch.randn(200, 2, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    U.append_kv(k, v, c, 0)
    pages = [list(x) for x in c.kv_cache._indicies]
    with pytest.raises(RuntimeError, match="attention weights"):
        U.evict_kv(c, 50, 4, 10)
    assert c.kv_cache.seqlen == 100 and c.kv_cache._indicies == pages and c.kv_cache.pos_base == 0
    assert U.evict_kv(c, 100, 4, 10) == 0
    assert U.evict_kv(c, 50, 10, 40) == 50
    assert [x[:50] for x in c.kv_cache._indicies] == [x[:10] + x[60:] for x in pages]
    c.prepare_metadata(1)
    c.begin_forward(1)
    U.append_kv(k[:2], v[:2], c, 0)
    U.decode_sparse_attn(torch.randn(2, 8, 64, generator=g).to(torch.bfloat16).cuda(), c, 0, c.kv_indices_without_last, True)
    assert U.evict_kv(c, 40, 4, 10) == 11
    c.clean_states()
    c.prepare_metadata(100)
    with pytest.raises(RuntimeError, match="attention weights"):
        U.evict_kv(c, 50, 4, 10)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv_bits", [8, 16])
def test_selection_layer_with_weights_against_its_definition(kv_bits, dtype):
    """With track_weights a selection layer's output, logits, log-sum-exp and weights are those of its definition over the
    cached values.  Logits: 128 roundings of fp32 sums of |q k| at most (64 products, any order, the scale).  Weights and
    output follow with twice their error, the output with half a step of its type and of the softmax weights' type."""
    import math
    import tidaldecode_b200.utils as U
    g = torch.Generator().manual_seed(6)
    B, n = 2, 180
    c = _controller(kv_bits, True, dtype=dtype, B=B)
    k, v = (torch.randn(B * n, 2, 64, generator=g).to(dtype).cuda() for _ in range(2))
    c.prepare_metadata(n)
    U.append_kv(k, v, c, 0)
    c.prepare_metadata(1)
    c.begin_forward(1)
    U.append_kv(k[:B], v[:B], c, 0)
    q = torch.randn(B, 8, 64, generator=g).to(dtype).cuda()
    o = U.decode_sparse_attn(q, c, 0, c.kv_indices_without_last, True)
    n += 1
    eps = torch.finfo(dtype).eps / 2
    for b in range(B):
        rows = c.kv_cache.buf_layer(0)[torch.tensor(c.kv_cache._indicies[b][:n]).cuda()]
        if kv_bits == 8:
            scales = c.kv_cache.scales_layer(0)[torch.tensor(c.kv_cache._indicies[b][:n]).cuda()]
            rows = K8.values(rows.cpu(), scales.cpu()).cuda()
        K, V = rows[:, 0, 0].double(), rows[:, 1, 0].double()                       # [n, Hkv, D]
        weights = torch.zeros(n, dtype=torch.float64, device="cuda")
        far = 0.0
        for h in range(8):
            kk, vv = K[:, h // 4], V[:, h // 4]
            x = kk @ q[b, h].double() / 8
            dx = 128 * 2.0 ** -24 * float((kk.abs() @ q[b, h].double().abs()).max()) / 8 + 2.0 ** -22 * (2 + float(x.abs().max()) * 1.4427)
            z = x.logsumexp(0)
            p = torch.exp(x - z)
            assert (c.qk_product[b, h, :n].double() - x).abs().max() <= dx
            assert abs(float(c.lse[b, h]) - float(z)) <= dx + (n + 8) * 2.0 ** -24 + 2.0 ** -22 * abs(float(z))
            A = p @ vv.abs()
            assert ((o[b, h].double() - p @ vv).abs() <= eps * (p @ vv).abs() + A * (2 * dx + (eps if dtype != torch.float32 else 0) + (n + 32) * 2.0 ** -23)).all()
            weights += p
            far = max(far, dx)
        assert ((c.weights[b, :n].double() - weights).abs() <= weights * (2 * far + (n + 16) * 2.0 ** -23)).all()
    assert c.workspace.status() == 0 and not c.weights[:, n:].any()
