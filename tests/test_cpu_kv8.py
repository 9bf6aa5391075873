"""CPU tier of the 8-bit KV cache operators: struct layouts, host-side refusals, and the oracle's own arithmetic."""
from __future__ import annotations

import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from oracle import kv8_oracle as K8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    from tidaldecode_b200 import build
    build.build()
    from tidaldecode_b200 import _lib
    return _lib


def test_struct_layouts(L, tmp_path):
    structs = {"tidal_append_kv8_args": L.AppendKv8Args, "tidal_read_kv8_args": L.ReadKv8Args, "tidal_attn_kv8_args": L.AttnKv8Args,
               "tidal_weights_args": L.WeightsArgs, "tidal_evict_args": L.EvictArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT}/include/tidal_b200.h"', "int main(void){"]
    for name, st in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in st._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = dict(x.split() for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, st in structs.items():
        assert int(got[name]) == C.sizeof(st)
        assert all(int(got[f"{name}.{f}"]) == getattr(st, f).offset for f, _ in st._fields_)


def _refused(L, fn, args, *rest, code=None, match=""):
    assert getattr(L.lib, fn)(C.byref(args), *rest) == (L.ERR_ARG if code is None else code)
    assert match in L.last_error(), L.last_error()


def _fill(a, **kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


APPEND = dict(d_k=256, d_v=256, d_kv=256, d_scales=256, k_stride=1024, v_stride=1024, page_table_stride=10, pos0=0, batch=1, tokens_per_seq=1, num_kv_heads=8,
              head_dim=128, page_size=16, block=16, dtype=1, num_pages=10)


@pytest.mark.parametrize("change,match", [
    (dict(d_k=0), "must be given"), (dict(d_scales=0), "must be given"), (dict(head_dim=96), "head_dim"), (dict(dtype=3), "dtype"), (dict(block=5), "divide"),
    (dict(block=0), "divide"), (dict(page_size=0), "page_size"), (dict(batch=0), "batch"), (dict(tokens_per_seq=0), "tokens_per_seq"), (dict(pos0=-1), "pos0"),
    (dict(pos0=2 ** 31 - 2), "pos0"), (dict(k_stride=1021), "aligned"), (dict(d_v=264), "aligned"), (dict(pos0=160), "pages"), (dict(tokens_per_seq=161), "pages"),
    (dict(batch=2, page_table_stride=9, pos0=130), "pool"), (dict(page_table_stride=0), "stride"),
])
def test_append_refusals(L, change, match):
    _refused(L, "tidal_append_kv8", _fill(L.AppendKv8Args(), **{**APPEND, **change}), None, match=match)


READ = dict(d_kv=256, d_scales=256, d_out=256, page_table_stride=10, start=0, stop=10, batch=1, num_kv_heads=8, head_dim=128, page_size=16, block=16, dtype=1,
            num_pages=10)


@pytest.mark.parametrize("change,match", [
    (dict(d_out=0), "must be given"), (dict(head_dim=32), "head_dim"), (dict(dtype=-1), "dtype"), (dict(block=3), "divide"), (dict(start=-1), "range"), (dict(start=11), "range"),
    (dict(d_out=8), "aligned"), (dict(stop=161), "pool"), (dict(stop=161, d_page_table=256), "table"), (dict(num_pages=0), "num_pages"),
])
def test_read_refusals(L, change, match):
    _refused(L, "tidal_read_kv8", _fill(L.ReadKv8Args(), **{**READ, **change}), None, match=match)


ATTN = dict(d_q=256, d_o=512, d_kv=256, d_scales=256, page_table_stride=10, seq_len=100, batch=1, num_qo_heads=8, num_kv_heads=2, head_dim=128, page_size=16,
            block=16, dtype=1, num_pages=10)


@pytest.mark.parametrize("change,match", [
    (dict(d_q=0), "must be given"), (dict(d_o=8), "aligned"), (dict(num_kv_heads=3), "multiple"), (dict(head_dim=256), "head_dim"), (dict(dtype=9), "dtype"),
    (dict(block=7), "divide"), (dict(seq_len=-1), "seq_len"), (dict(seq_len=161), "pool"), (dict(seq_len=161, d_page_table=256), "table"),
    (dict(num_pages=2 ** 27), "2^31"), (dict(d_sel_idx=256, sel_rows=2, sel_count=4, sel_stride=4), "sel_rows"),
    (dict(d_sel_idx=256, sel_rows=1, sel_count=5, sel_stride=4), "sel_count"), (dict(d_scores=256, score_stride=99), "score_stride"), (dict(batch=0), "batch"),
])
def test_attention_refusals(L, change, match):
    _refused(L, "tidal_decode_attention_kv8", _fill(L.AttnKv8Args(), **{**ATTN, **change}), 0x4000, 1 << 20, None, match=match)


def test_attention_needs_an_initialised_workspace(L):
    _refused(L, "tidal_decode_attention_kv8", _fill(L.AttnKv8Args(), **ATTN), 0x4000, 1 << 20, None, code=L.ERR_WORKSPACE, match="not initialised")


WEIGHTS = dict(d_scores=256, score_stride=100, d_lse=256, d_weights=256, weight_stride=100, seq_len=100, batch=1, heads=8, decay=1.0)


@pytest.mark.parametrize("change,match", [(dict(d_lse=0), "must be given"), (dict(batch=0), "batch"), (dict(heads=0), "heads"), (dict(batch=1025, d_seq_lens=256), "1024"), (dict(seq_len=101), "shorter"),
                                          (dict(weight_stride=99), "shorter"), (dict(seq_len=-1), "shorter")])
def test_weights_refusals(L, change, match):
    _refused(L, "tidal_accumulate_weights", _fill(L.WeightsArgs(), **{**WEIGHTS, **change}), None, match=match)


EVICT = dict(d_weights=0x10000, d_weights_out=0x20000, weight_stride=100, d_page_table=0x30000, d_page_table_out=0x40000, page_table_stride=100, d_seq_lens=0x50000,
             d_seq_lens_out=0x60000, max_len=100, rows=2, page_size=1, keep_pages=50, sink_pages=4, recent_pages=8)


@pytest.mark.parametrize("change,match", [
    (dict(d_weights=0), "must be given"), (dict(rows=0), "rows"), (dict(page_size=0), "page_size"), (dict(max_len=0), "max_len"), (dict(recent_pages=0), "recent_pages"),
    (dict(sink_pages=-1), "sink_pages"), (dict(keep_pages=11), "keep_pages"), (dict(max_len=101), "shorter"), (dict(page_table_stride=99), "shorter"),
    (dict(d_weights_out=0x10100), "overlap"), (dict(d_page_table_out=0x30000), "overlap"), (dict(d_seq_lens_out=0x50004), "overlap"),
])
def test_evict_refusals(L, change, match):
    _refused(L, "tidal_evict_pages", _fill(L.EvictArgs(), **{**EVICT, **change}), None, match=match)


def test_wrappers_refuse_cpu_tensors():
    import tidaldecode_b200.ops as T
    kv, sc = T.alloc_kv8(4, 16, 2, 64, 16, device="cpu")
    k = torch.zeros(1, 2, 64)
    for call in (lambda: T.append_kv8(k, k, kv, sc), lambda: T.read_kv8(kv, sc, 3), lambda: T.decode_attention_kv8(k, kv, sc, 3, None),
                 lambda: T.accumulate_weights(torch.zeros(1, 2, 3), torch.zeros(1, 2), torch.zeros(1, 3), 3),
                 lambda: T.evict_pages(torch.zeros(1, 3), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="divide"):
        T.alloc_kv8(4, 16, 2, 64, 5, device="cpu")


def test_oracle_rounding_is_torchs():
    """The oracle's e4m3 rounding against torch's cast on every float16 up to 448, and its table against torch's values."""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    assert torch.equal(K8.round_e4m3(x.double()), x.float().to(torch.float8_e4m3fn).double())
    codes = torch.arange(256, dtype=torch.uint8)
    t = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(K8._E4M3, nan=-1.0), torch.nan_to_num(t, nan=-1.0))
    for amax, e in ((448.0, 0), (448.5, 1), (0.0, -126), (1.0, -8), (1.75, -8), (1.7500001, -7), (3.4028234e38, 120), (1e-45, -126)):
        assert K8.scale_exponent(amax) == e, amax
    assert math.isnan(float(K8.round_e4m3(torch.tensor(math.nan, dtype=torch.float64))))
