"""What the C entry points of paged decode attention and windowed prefill refuse before any launch."""
from __future__ import annotations

import ctypes

import pytest

from racetrack_b200 import _lib, build as rt_build

BAD, UNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def lib():
    rt_build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def memory():
    buf = ctypes.create_string_buffer(4096)
    return ctypes.addressof(buf) // 16 * 16 + 16, buf


DECODE = dict(q_abs=0, q_pe=0, kv=0, pe=0, table=0, lens=0, seqs=None, out=0, workspace=0, batch=1, heads=16, slots=1, width=4,
              pages=8, page_size=64, qa_batch=16 * 512, qa_head=512, qp_batch=16 * 64, qp_head=64, kv_page=64 * 512,
              kv_row=512, pe_page=64 * 64, pe_row=64, table_stride=4, window=0, sinks=0, scale=0.1, stream=None)
POINTERS = ("q_abs", "q_pe", "kv", "pe", "table", "lens", "out", "workspace", "q", "k_nope", "k_pe", "v")


def call(fn, defaults, at, change):
    args = {k: at if k in POINTERS else v for k, v in defaults.items()}
    args.update({k: at + v if k in POINTERS and v is not None else v for k, v in change.items()})
    return fn(*args.values())


@pytest.mark.parametrize("change, code, says", [
    (dict(batch=-1), BAD, b"bad shape"),
    (dict(heads=0), BAD, b"bad shape"),
    (dict(page_size=8), UNSUPPORTED, b"power of two"),
    (dict(page_size=48), UNSUPPORTED, b"power of two"),
    (dict(page_size=1 << 21), UNSUPPORTED, b"power of two"),
    (dict(q_abs=None), BAD, b"null"),
    (dict(table=None), BAD, b"null"),
    (dict(lens=None), BAD, b"null"),
    (dict(workspace=None), BAD, b"null"),
    (dict(kv=8), BAD, b"16-byte"),
    (dict(out=2), BAD, b"16-byte"),
    (dict(qa_head=500), BAD, b"multiples of 8"),
    (dict(kv_row=-512), BAD, b"multiples of 8"),
    (dict(window=-1), BAD, b"negative"),
    (dict(sinks=-1), BAD, b"negative"),
    (dict(pages=0), BAD, b"no page"),
    (dict(batch=65536), UNSUPPORTED, b"too large"),
    (dict(heads=1025), UNSUPPORTED, b"too large"),
    (dict(width=1 << 26), UNSUPPORTED, b"too large"),
    (dict(batch=60000, width=1 << 20), UNSUPPORTED, b"too large"),
])
def test_decode(lib, memory, change, code, says):
    assert call(lib.rt_mla_paged_decode, DECODE, memory[0], change) == code
    assert says in lib.rt_last_error()


def test_a_decode_without_rows_does_nothing(lib, memory):
    assert call(lib.rt_mla_paged_decode, DECODE, memory[0], dict(batch=0)) == 0


def test_workspace_sizes(lib):
    assert lib.rt_mla_paged_decode_workspace_bytes(0) == 0 and lib.rt_mla_paged_decode_workspace_bytes(-3) == 0


PREFILL = dict(q=0, k_nope=0, k_pe=0, v=0, out=0, out_codes=None, out_scales=None, tokens=4, heads=2, layer_heads=2, nope=128,
               rope=64, v_dim=128, q_token=384, q_head=192, kn_token=256, kn_head=128, kp_token=64, kp_head=0,
               v_token=256, v_head=128, o_token=256, o_head=128, window=2, sinks=0, scale=0.1, stream=None)


@pytest.mark.parametrize("change, code, says", [
    (dict(window=0), BAD, b"window must be positive"),
    (dict(window=-5), BAD, b"window must be positive"),
    (dict(sinks=-1), BAD, b"sinks not negative"),
    (dict(layer_heads=1), BAD, b"layer_heads"),
    (dict(out=None), BAD, b"null"),
    (dict(q=None), BAD, b"null"),
    (dict(k_nope=4), BAD, b"16-byte"),
    (dict(nope=100), UNSUPPORTED, b"multiples of 8"),
    (dict(v_dim=136), UNSUPPORTED, b"multiples of 8"),
    (dict(q_token=380), BAD, b"multiples of 8"),
    (dict(tokens=-1), BAD, b"bad shape"),
    (dict(tokens=1 << 31), UNSUPPORTED, b"too large"),
])
def test_windowed_prefill(lib, memory, change, code, says):
    assert call(lib.rt_attn_window_prefill, PREFILL, memory[0], change) == code
    assert says in lib.rt_last_error()


def test_a_prefill_without_tokens_does_nothing(lib, memory):
    assert call(lib.rt_attn_window_prefill, PREFILL, memory[0], dict(tokens=0)) == 0


@pytest.mark.parametrize("change", [{}, dict(out=None, out_codes=None, out_scales=None),
                                    dict(q=None, k_nope=None, k_pe=None, v=None, out=None), dict(out=None, nope=64, v_dim=64)])
def test_a_prefill_without_tokens_needs_no_memory(lib, memory, change):
    """Tensors without elements have no address: no tokens is no error, under a window or without one."""
    args = dict(change, tokens=0)
    assert call(lib.rt_attn_window_prefill, PREFILL, memory[0], args) == 0
    share = {k: v for k, v in PREFILL.items() if k not in ("window", "sinks")}
    assert call(lib.rt_attn_causal_prefill_share, share, memory[0], args) == 0
    causal = {k: v for k, v in share.items() if k not in ("out_codes", "out_scales", "layer_heads")}
    args = {k: v for k, v in args.items() if k in causal}
    assert call(lib.rt_attn_causal_prefill, causal, memory[0], args) == 0


@pytest.mark.parametrize("change", [dict(kv_row=0), dict(kv_row=504), dict(pe_row=0), dict(kv_page=0), dict(pe_page=56),
                                    dict(qa_head=0), dict(qp_head=0), dict(batch=2, qa_batch=0), dict(batch=2, qp_batch=8)])
def test_decode_refuses_rows_that_overlap(lib, memory, change):
    assert call(lib.rt_mla_paged_decode, DECODE, memory[0], change) == BAD
    assert b"overlap" in lib.rt_last_error()
