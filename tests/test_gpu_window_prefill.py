"""Causal attention under a sliding window with sinks against its definition in 64 bits.

Tolerance, for an element o = sum p_j v_j with a = sum p_j |v_j|: bf16 rounding of the probabilities (2^-8 of
a) and of the output (2^-8 of |o|); fp32 scores of 192 exact products, off by at most 196 * 2^-24 * c with c
= scale * sum_d |q_d k_d| (largest over the visible keys; the scale and maximum folded into the exponent are in
the 196), a factor expm1(2 e) on the probabilities; 2^x by a polynomial or ex2 (4 * 2^-24) and sums over n
keys: (2 n + 64) 2^-24 of a. The FP8 epilogue is compared with the quantiser bit for bit instead.
"""
from __future__ import annotations

import pytest
import torch

from racetrack_b200 import ops

pytestmark = pytest.mark.gpu


def inputs(tokens, heads, seed, nope=128, rope=64, v_dim=128, spread=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    mk = lambda *s: (torch.randn(*s, device="cuda", generator=g) * spread).bfloat16()
    return mk(tokens, heads, nope + rope), mk(tokens, heads, nope), mk(tokens, rope) if rope else None, mk(tokens, heads, v_dim)


def seen(tokens, window, sinks):
    i = torch.arange(tokens, device="cuda")[:, None]
    j = torch.arange(tokens, device="cuda")[None, :]
    return (j <= i) & ((j > i - window) | (j < sinks))


def check(got, q, k_nope, k_pe, v, window, sinks, scale=None):
    tokens, heads, qk = q.shape
    scale = qk ** -0.5 if scale is None else scale
    hidden = ~seen(tokens, window, sinks)
    n = int((~hidden).sum(1).max())
    u = 2.0 ** -24
    assert got.shape == (tokens, heads, v.shape[-1])
    for h in range(heads):
        pe = [] if k_pe is None else [k_pe if k_pe.dim() == 2 else k_pe[:, h]]
        k, qh, vh = torch.cat([k_nope[:, h], *pe], 1).double(), q[:, h].double(), v[:, h].double()
        p = torch.softmax((qh @ k.T * scale).masked_fill(hidden, float("-inf")), 1)
        o, a = p @ vh, p @ vh.abs()
        c = abs(scale) * (qh.abs() @ k.abs().T).masked_fill(hidden, 0.0).amax(1, keepdim=True)
        tol = 2.0 ** -8 * (a + o.abs()) + a * (torch.expm1(2 * 196 * u * c) + (2 * n + 64) * u)
        off = (got[:, h].double() - o).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (f"head {h}: {int(bad.sum())} off, worst {float((off / tol).max()):.3g} of the tolerance, "
                               f"first at {bad.nonzero()[0].tolist()}")
    ops.tc_error_state()


@pytest.mark.parametrize("tokens", [1, 2, 127, 128, 129, 255, 257, 384, 520, 777])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (5, 0), (127, 3), (128, 0), (128, 128), (129, 1), (200, 4),
                                           (256, 300), (300, 129), (500, 1000)])
def test_windows_around_tiles(tokens, window, sinks):
    q, kn, kp, v = inputs(tokens, 2, tokens + window)
    got = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks)
    check(got, q, kn, kp, v, window, sinks)


@pytest.mark.parametrize("tokens, heads, window, sinks", [(2000, 3, 700, 4), (4000, 1, 64, 0), (1500, 5, 1024, 64)])
def test_longer_prompts(tokens, heads, window, sinks):
    q, kn, kp, v = inputs(tokens, heads, 9)
    got = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks)
    check(got, q, kn, kp, v, window, sinks)
    again = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("nope, rope, v_dim", [(32, 16, 32), (64, 64, 64), (128, 0, 128), (96, 32, 72), (48, 0, 16)])
def test_other_head_shapes(nope, rope, v_dim):
    q, kn, kp, v = inputs(400, 2, nope, nope, rope, v_dim)
    check(ops.attention_prefill(q, kn, kp, v, window=70, sinks=5), q, kn, kp, v, 70, 5)


def test_strided_operands_and_a_rope_key_a_head():
    tokens, heads = 300, 3
    q, _, kp, _ = inputs(tokens, heads, 1)
    kv = torch.randn(tokens, heads, 256, device="cuda").bfloat16()
    per_head = torch.randn(tokens, heads, 64, device="cuda").bfloat16()
    for pe in (kp, per_head, kp[:, None].expand(-1, heads, -1)):
        got = ops.attention_prefill(q, kv[..., :128], pe, kv[..., 128:], window=90, sinks=2)
        check(got, q, kv[..., :128], pe, kv[..., 128:], 90, 2)


@pytest.mark.parametrize("window", [300, 301, 2 ** 31, 2 ** 62])
def test_a_window_over_everything_is_the_causal_call(window):
    q, kn, kp, v = inputs(300, 4, 3)
    a, b = ops.attention_prefill(q, kn, kp, v), ops.attention_prefill(q, kn, kp, v, window=window, sinks=7)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("special", [float("nan"), float("inf"), float("-inf"), 3.0e38])
def test_hidden_keys_weigh_nothing(special):
    """Keys that a query does not see do not reach it, whatever they are; nor do their values, however large."""
    tokens, window, sinks = 600, 130, 3
    q, kn, kp, v = inputs(tokens, 2, 4)
    clean = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks)
    for at in (3, 127, 128, 250, 400):
        kn2, v2 = kn.clone(), v.clone()
        kn2[at] = special
        v2[at] = 3.0e38
        got = ops.attention_prefill(q, kn2, kp, v2, window=window, sinks=sinks)
        blind = ~seen(tokens, window, sinks)[:, at]
        assert torch.equal(got[blind].view(torch.int16), clean[blind].view(torch.int16)), at


@pytest.mark.parametrize("tokens, window, sinks", [(257, 100, 4), (700, 256, 128)])
def test_fp8_epilogue_is_the_quantiser(tokens, window, sinks):
    q, kn, kp, v = inputs(tokens, 5, 6)
    plain = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks)
    codes, scales = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks, quantized=True)
    want, want_scales = ops.fused_act_quant(plain.view(tokens, -1))
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)
    # another head shape takes the quantiser behind the kernel
    q, kn, kp, v = inputs(tokens, 2, 6, 64, 32, 128)
    codes, _ = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks, quantized=True)
    want, _ = ops.fused_act_quant(ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks).view(tokens, -1))
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))


def test_sharp_scores_and_other_scales():
    q, kn, kp, v = inputs(500, 2, 8, spread=3.0)
    for scale in (192 ** -0.5, 0.01, 0.5):
        check(ops.attention_prefill(q, kn, kp, v, scale, window=150, sinks=20), q, kn, kp, v, 150, 20, scale)


def test_a_prompt_then_a_token_agree():
    """The last query of a windowed prefill is what decoding that token under the same window computes: one
    head shape in two forms, the second over latent rows with the key half of the projection absorbed."""
    tokens, heads, window, sinks = 333, 16, 100, 4
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    mk = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).bfloat16()
    kv, pe, q = mk(tokens, 512), mk(tokens, 64), mk(tokens, heads, 192)
    w = mk(heads, 256, 512, std=512 ** -0.5)
    both = torch.einsum("tc,hdc->thd", kv.double(), w.double())
    prefill = ops.attention_prefill(q, both[..., :128].bfloat16(), pe, both[..., 128:].bfloat16(), window=window, sinks=sinks)
    q_abs = torch.einsum("hd,hdc->hc", q[-1, :, :128].double(), w[:, :128].double()).bfloat16()
    pages = -(-tokens // 64)
    kvp, pep = torch.zeros(pages, 64, 512, device="cuda").bfloat16(), torch.zeros(pages, 64, 64, device="cuda").bfloat16()
    kvp.view(-1, 512)[:tokens], pep.view(-1, 64)[:tokens] = kv, pe
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    latent = ops.mla_paged_decode(q_abs[None], q[-1:, :, 128:], kvp, pep, i32([list(range(pages))]), i32([tokens]), 192 ** -0.5,
                                  window=window, sinks=sinks)
    decode = torch.einsum("hc,hdc->hd", latent[0].double(), w[:, 128:].double())
    # roundings of the keys, the absorbed query, the values, the latent row and the probabilities, 2^-8 each
    # and of independent sign: 2 % of the largest element is 5 of them
    assert (decode - prefill[-1].double()).abs().max() <= 0.02 * prefill[-1].double().abs().max()


def test_captured_and_on_another_stream():
    q, kn, kp, v = inputs(300, 2, 5)
    want = ops.attention_prefill(q, kn, kp, v, window=64, sinks=1)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        with torch.cuda.graph(graph, stream=side):
            got = ops.attention_prefill(q, kn, kp, v, window=64, sinks=1)
    v.mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want * 2)                      # a power of two: every rounding scales with it


@pytest.mark.parametrize("kw, says", [({"window": 0}, "positive"), ({"window": -1}, "positive"), ({"sinks": 3}, "go with"),
                                      ({"window": 4, "sinks": -1}, "negative"), ({"window": 4, "layer_heads": 1}, "layer_heads")])
def test_what_is_refused(kw, says):
    q, kn, kp, v = inputs(20, 2, 5)
    with pytest.raises(RuntimeError, match=says):
        ops.attention_prefill(q, kn, kp, v, **kw)


@pytest.mark.parametrize("scale", [-192 ** -0.5, -0.3, 0.0, -0.0])
@pytest.mark.parametrize("tokens, heads, window, sinks", [(300, 2, 100, 3), (300, 60, 100, 3), (300, 60, 30, 140)])
def test_scales_that_are_not_positive(tokens, heads, window, sinks, scale):
    """A negative scale turns the order of the scores, 0 weighs what is seen alike; 2 and 60 heads are the two
    tilings. Hidden keys weigh nothing, NaN included."""
    q, kn, kp, v = inputs(tokens, heads, 11)
    got = ops.attention_prefill(q, kn, kp, v, scale, window=window, sinks=sinks)
    check(got, q, kn, kp, v, window, sinks, scale)
    at = 200
    kn2 = kn.clone()
    kn2[at] = float("nan")
    blind = ~seen(tokens, window, sinks)[:, at]
    again = ops.attention_prefill(q, kn2, kp, v, scale, window=window, sinks=sinks)
    assert torch.equal(again[blind].view(torch.int16), got[blind].view(torch.int16))
    codes, scales = ops.attention_prefill(q, kn, kp, v, scale, window=window, sinks=sinks, quantized=True)
    want, want_scales = ops.fused_act_quant(got.view(tokens, -1))
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)


@pytest.mark.parametrize("scale", [-192 ** -0.5, -0.3, 0.0])
@pytest.mark.parametrize("schedule", [1, 2])
def test_scales_that_are_not_positive_without_a_window(schedule, scale):
    q, kn, kp, v = inputs(300, 3, 12)
    previous = ops.attention_prefill_schedule(schedule)
    try:
        got = ops.attention_prefill(q, kn, kp, v, scale)
    finally:
        ops.attention_prefill_schedule(previous)
    check(got, q, kn, kp, v, 300, 0, scale)


@pytest.mark.parametrize("window, sinks", [(None, 0), (5, 1)])
@pytest.mark.parametrize("nope, rope, v_dim", [(128, 64, 128), (64, 32, 64)])
def test_a_prompt_without_tokens(nope, rope, v_dim, window, sinks):
    q, kn, kp, v = inputs(0, 4, 1, nope, rope, v_dim)
    got = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks)
    assert got.shape == (0, 4, v_dim) and got.dtype == torch.bfloat16
    codes, scales = ops.attention_prefill(q, kn, kp, v, window=window, sinks=sinks, quantized=True)
    assert codes.shape == (0, 4 * v_dim) and codes.dtype == torch.float8_e4m3fn
    assert scales.shape == (0, 4 * v_dim // 128) and scales.dtype == torch.float32


@pytest.mark.parametrize("tokens, heads", [(1, 3), (300, 2), (300, 60)])
@pytest.mark.parametrize("spread", [0.1, 1.0, 2.0])
@pytest.mark.parametrize("window, sinks", [(1, 0), (2, 0), (40, 3)])
def test_a_key_that_is_seen_alone_gives_its_value(tokens, heads, spread, window, sinks):
    """Its probability is 1: the output is the value itself, to the bit (scores up to 100 in size). Two and 60 heads
    are the two tilings; a single token takes the causal call, so it is asked for under a window in two."""
    q, kn, kp, v = inputs(max(tokens, 2), heads, tokens + 13, spread=spread)
    got = ops.attention_prefill(q, kn, kp, v, window=1 if tokens == 1 else window, sinks=sinks)
    alone = seen(max(tokens, 2), 1 if tokens == 1 else window, sinks).sum(1) == 1
    assert alone[0] and (window > 1 or sinks or bool(alone.all()))
    assert torch.equal(got[alone].view(torch.int16), v[alone].view(torch.int16))


@pytest.mark.parametrize("scale", [None, -0.05])
@pytest.mark.parametrize("window, sinks", [(200, 0), (200, 4), (300, 300), (129, 129), (128, 128), (1, 0), (600, 128)])
@pytest.mark.parametrize("tokens, heads, share", [(777, 32, 4), (700, 40, 1)])
def test_a_share_of_the_heads_has_the_bits_of_the_whole(tokens, heads, share, window, sinks, scale):
    """All heads fill more than one wave with blocks of 256 queries, a share takes blocks of 128: the same bits,
    whatever the share says of its layer."""
    q, kn, kp, v = inputs(tokens, heads, 17)
    kw = dict(softmax_scale=scale, window=window, sinks=sinks)
    whole = ops.attention_prefill(q, kn, kp, v, **kw)
    codes, scales = ops.attention_prefill(q, kn, kp, v, quantized=True, **kw)
    for lo in (0, heads - share):
        mine = slice(lo, lo + share)
        for layer_heads in (heads, share):
            part = ops.attention_prefill(q[:, mine], kn[:, mine], kp, v[:, mine], layer_heads=layer_heads, **kw)
            assert torch.equal(part.view(torch.int16), whole[:, mine].contiguous().view(torch.int16))
            c, s = ops.attention_prefill(q[:, mine], kn[:, mine], kp, v[:, mine], quantized=True, layer_heads=layer_heads, **kw)
            assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8)[:, lo * 128:(lo + share) * 128])
            assert torch.equal(s, scales[:, mine])
