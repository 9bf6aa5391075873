"""The 8-bit cache and its eviction behind the model's entry points: the operator façade and controller, the attention
modules, and the decoder replayed as a CUDA graph."""
from __future__ import annotations

import pytest
import torch

from oracle import kv8_oracle as K8
from oracle import tidal_oracle as O
from tests.test_gpu_model import _tiny_model

pytestmark = pytest.mark.gpu


def _controller(kv_bits, track, dtype=torch.bfloat16, B=1, N=256, budget=32, **kw):
    from tidaldecode_b200.utils import InferenceController
    return InferenceController(num_layers=2, num_heads=8, head_dim=64, page_size=1, token_budget=budget, max_seq_len=N, dtype=dtype,
                               device=torch.device("cuda"), num_kv_heads=2, batch_size=B, kv_bits=kv_bits, track_weights=track, **kw)


def _quantised(x):
    """What an 8-bit cache holds of x [n, Hkv, D] (a scale per token and head), in x's dtype."""
    flat = x.cpu().double()
    e = torch.tensor([[K8.scale_exponent(float(r.abs().max())) for r in t] for t in flat], dtype=torch.float64)
    return (K8.round_e4m3(flat / 2.0 ** e[..., None]) * 2.0 ** e[..., None]).to(x.dtype).to(x.device)


def test_facade_over_an_8_bit_cache_equals_the_model_dtype_cache_of_the_same_values():
    """Prefill is bit for bit the 16-bit cache's over the same (representable) values; decode attention, logits, the chosen
    set and the sparse layer agree with it within the two kernels' roundings (bf16 results: half a step each, 2^-9, and
    bf16 against fp16 softmax weights, 2^-9, of sum p|v| <= max|v|)."""
    import tidaldecode_b200.utils as U
    g = torch.Generator().manual_seed(0)
    n = 150
    a, b = _controller(8, False), _controller(16, False)
    k, v = (_quantised(torch.randn(n, 2, 64, generator=g).to(torch.bfloat16).cuda()) for _ in range(2))
    q = torch.randn(n, 8, 64, generator=g).to(torch.bfloat16).cuda()
    outs = []
    for c in (a, b):
        c.prepare_metadata(n)
        c.begin_forward(n)
        U.append_kv(k, v, c, 0)
        outs.append(U.prefill_forward(q, c, 0))
    assert torch.equal(*outs)
    k1, v1 = (_quantised(torch.randn(1, 2, 64, generator=g).to(torch.bfloat16).cuda()) for _ in range(2))
    res = []
    for c in (a, b):
        c.prepare_metadata(1)
        c.begin_forward(1)
        U.append_kv(k1, v1, c, 0)
        full = U.decode_sparse_attn(q[:1], c, 0, c.kv_indices_without_last, False)
        search = U.decode_sparse_attn(q[:1], c, 0, c.kv_indices_without_last, True)
        U.decode_topk(c)
        sparse = U.decode_sparse_attn(q[:1], c, 0, c.topk_dindices_buffer, False)
        res.append((full, search, sparse, c.qk_product[..., :n + 1].clone(), c.topk_dindices_buffer.clone()))
        assert c.workspace.status() == 0
    tol = 4 * 2.0 ** -9 * float(v.float().abs().max())
    for x, y in zip(res[0][:3], res[1][:3]):
        assert (x.float() - y.float()).abs().max() <= tol
    x, y = res[0][3], res[1][3]
    assert (x - y).abs().max() <= 2 * 20 * 2.0 ** -23 * float(k.float().abs().max()) * 64 * float(q.float().abs().max()) / 8
    assert torch.equal(res[0][4].sort(-1).values, res[1][4].sort(-1).values)
    with pytest.raises(RuntimeError, match="pool pages"):
        U.decode_sparse_attn(q[:1], a, 0, torch.zeros(8, 4, dtype=torch.int32, device="cuda"), False)


@pytest.mark.parametrize("kv_bits", [8, 16])
def test_weights_and_eviction_through_the_facade(kv_bits):
    """Weights of a selection layer add up to one per head; eviction keeps the first, the last and the heaviest tokens; what
    is appended next is rotated to its position, not its slot; clean_states starts over."""
    import tidaldecode_b200.utils as U
    g = torch.Generator().manual_seed(1)
    B, n, keep = 2, 100, 48
    c = _controller(kv_bits, True, dtype=torch.float32, B=B)
    c.prepare_metadata(n)
    k, v = (torch.randn(B * n, 2, 64, generator=g).cuda() for _ in range(2))
    U.append_kv(k, v, c, 0)
    q = torch.randn(B, 8, 64, generator=g).cuda()
    c.prepare_metadata(1)
    c.begin_forward(1)
    U.append_kv(k[:B], v[:B], c, 0)
    U.decode_sparse_attn(q, c, 0, c.kv_indices_without_last, True)
    assert (c.weights.double().sum(1) - 8).abs().max() < 8e-5
    before, pages = c.weights.cpu(), [list(x) for x in c.kv_cache._indicies]
    dropped = U.evict_kv(c, keep, 4, 10)
    assert dropped == n + 1 - keep and c.kv_cache.seqlen == keep and c.kv_cache.pos_base == dropped
    for b in range(B):
        middle = sorted(range(4, n + 1 - 10), key=lambda i: (-float(before[b, i]), i))[:keep - 14]
        stay = list(range(4)) + sorted(middle) + list(range(n + 1 - 10, n + 1))
        assert c.kv_cache._indicies[b][:keep] == [pages[b][i] for i in stay]
        assert torch.equal(c.weights[b, :keep].cpu(), before[b, stay]) and not c.weights[b, keep:].any()
        assert c.kv_cache.page_table[b, :n + 1].tolist() == c.kv_cache._indicies[b][:n + 1]
    assert U.evict_kv(c, keep, 4, 10) == 0
    # the next token: position n + 1, slot keep
    kn, vn, qn = (torch.randn(B, h, 64, generator=g).cuda() for h in (2, 2, 8))
    want = O.apply_rope_fp32(kn.cpu(), torch.full((B,), n + 1), 1e4)
    c.prepare_metadata(1)
    c.begin_forward(1)
    U.rope_append_kv(qn, kn.clone(), vn, c, 0)
    for b in range(B):
        page = c.kv_cache._indicies[b][keep]
        if kv_bits == 8:
            got = K8.values(c.kv_cache.buf_layer(0)[page:page + 1].cpu(), c.kv_cache.scales_layer(0)[page:page + 1, :, None][:, :, 0].cpu())[0, 0, 0]
            # half a step of e4m3: 2^-4 of the value, or of 2^-6 of the scale where values lie below that
            assert (got - want[b].double()).abs().max() <= 2.0 ** -4 * float(want.abs().max()) * (1 + 1e-5)
        else:
            assert torch.allclose(c.kv_cache.buf_layer(0)[page, 0, 0].cpu(), want[b], atol=1e-5, rtol=0)
    o = U.decode_sparse_attn(qn, c, 0, c.kv_indices_without_last, True)
    assert torch.isfinite(o).all() and c.workspace.status() == 0
    c.clean_states()
    assert c.kv_cache.seqlen == 0 and c.kv_cache.pos_base == 0 and not c.weights.any()


def test_refusals():
    for kw in (dict(kv_bits=4, track=False), dict(kv_bits=16, track=True, head_reduce="sum"), dict(kv_bits=8, track=False, head_reduce="sum"), dict(kv_bits=8, track=False, quest_metadata=True)):
        with pytest.raises(ValueError):
            _controller(**kw)
    import tidaldecode_b200.utils as U
    c = _controller(8, False)
    with pytest.raises(RuntimeError, match="track_weights"):
        U.evict_kv(c, 10)
    with pytest.raises(RuntimeError, match="keep_pages"):
        c = _controller(8, True)
        c.prepare_metadata(50)
        U.evict_kv(c, 20, 15, 15)


@pytest.mark.parametrize("dtype,fused", [(torch.bfloat16, True), (torch.float32, False)])
def test_graph_decoder_on_an_8_bit_cache_with_eviction(dtype, fused):
    """Replayed and eager decode steps give the same tokens, logits and weights, before and after an eviction between two
    decode() calls; generation goes on past the cache's capacity."""
    from tidaldecode_b200.runtime import GraphDecoder
    W = O.TinyLlamaWeights(vocab=512, hidden=512, layers=4, heads=8, kv_heads=2, ffn=352, seed=5, dtype=dtype)
    prompt = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(2))
    runs = []
    for use_graph in (True, False):
        rt = GraphDecoder(_tiny_model(W, dtype, (1, 3), "none", True, 2), max_seq_len=96, token_budget=16, kv_bits=8, track_weights=True,
                          fused_linear=fused)
        first = rt.prefill(prompt)
        toks = rt.decode(20, use_graph=use_graph).clone()
        assert rt.c.kv_cache.seqlen == 80
        dropped = rt.evict(40, sink_tokens=2, recent_tokens=8)
        assert dropped == 81 - 41 and rt.c.kv_cache.seqlen == 40
        with pytest.raises(RuntimeError, match="max_seq_len"):
            rt.decode(60, use_graph=use_graph)
        more = rt.decode(50, use_graph=use_graph).clone()
        assert rt.c.kv_cache.seqlen == 90 and int(rt.pos) == 60 + 70 and int(rt.slot) == 90
        assert rt.c.workspace.status() == 0 and int(rt.lin_status) == 0
        runs.append((first, toks, more, rt.logits.clone(), rt.c.weights.clone(), rt.c.kv_cache.page_table.clone()))
    for x, y in zip(*runs):
        assert torch.equal(x, y)


def test_model_on_an_8_bit_cache_eager():
    """LlamaForCausalLM with kv_bits=8: prefill, decode through full, selection and sparse layers; the same tokens twice."""
    W = O.TinyLlamaWeights(vocab=512, hidden=512, layers=4, heads=8, kv_heads=2, ffn=352, seed=5, dtype=torch.bfloat16)
    m = _tiny_model(W, torch.bfloat16, (1, 3), "none", True, 2)
    m.tidal_init(page_size=1, max_seq_len=128, token_budget=16, dtype=torch.bfloat16, device=torch.device("cuda"), kv_bits=8)
    prompt = torch.randint(0, 512, (1, 50), generator=torch.Generator().manual_seed(4)).cuda()
    a = m.greedy_generate(prompt, 12)
    m.tidal_clear()
    assert m.greedy_generate(prompt, 12) == a and m.model.iController.workspace.status() == 0
