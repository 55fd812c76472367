"""The paged decode layer against the layer it stands beside: prompts by RealisticLayer, steps by DecodeLayer
where its sparse selection takes every position. Attention halves agree to 2e-2 of the largest element, the
tolerance of test_gpu_decode.py for the same projections (roundings of the absorbed query, the latent row and
the probabilities, 2^-8 each, through two more bf16 products)."""
from __future__ import annotations

import pytest
import torch

from helpers import rel_err
from racetrack_b200 import decode, layer, ops, paging

pytestmark = pytest.mark.gpu

SHAPE = layer.DSV32.scaled(name="small_paged", hidden=512, heads=16, q_lora=128, kv_lora=512, nope=32, rope=64,
                           v_dim=32, moe_inter=256, n_experts=16, topk=4)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def weights(rank=0, world=1):
    return {k: v.cuda() for k, v in layer.make_weights(SHAPE, rank, world, "cpu", std=0.05).items()}


def model(page=32, window=None, sinks=0, pages=64, rank=0, world=1):
    caches = paging.PagedCaches(SHAPE, pages, page, 6, 20, "cuda")
    m = decode.PagedDecodeLayer(SHAPE, weights(rank, world), rank, world, caches=caches, window=window, sinks=sinks)
    m.reduce = False
    return m


def prompt(tokens, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(tokens, SHAPE.hidden, device="cuda", generator=g) * 0.5).bfloat16()


def attention_rows(m, hidden):
    """The attention half of the plain layer over a whole prompt."""
    normed = ops.fused_rms_norm(hidden, m.ones_h, eps=SHAPE.eps)
    return m.attention(normed, torch.arange(hidden.shape[0], device="cuda"))


@pytest.mark.parametrize("window, sinks", [(None, 0), (40, 3)])
def test_steps_continue_their_prompts(window, sinks):
    """Prompts of different lengths, then three tokens each: every step's attention is the last row of the
    prompt with these tokens appended."""
    m = model(window=window, sinks=sinks)
    plain = layer.RealisticLayer(SHAPE, weights(), window=window, sinks=sinks)
    lengths, order = [70, 1, 129], [2, 5, 0]
    text = {s: prompt(n + 3, 10 + s) for s, n in zip(order, lengths)}
    for s, n in zip(order, lengths):
        out = m.prefill(text[s][:n], ints([s]), 1)
        assert torch.equal(out, plain.forward_stack(text[s][:n], torch.arange(n, device="cuda"), 1))
    for step in range(3):
        batch = [5, 0, 2]
        hidden = torch.stack([text[s][lengths[order.index(s)] + step] for s in batch])
        normed = ops.fused_rms_norm(hidden, m.ones_h, eps=SHAPE.eps)
        seqs = ints(batch + [-1])
        slots = m.caches.extend(4, seqs)
        pos = torch.tensor([lengths[order.index(s)] + step for s in batch] + [0], device="cuda")
        got = m.decode_attention(torch.cat((normed, normed[:1])), seqs, slots, pos)
        for b, s in enumerate(batch):
            n = lengths[order.index(s)] + step + 1
            want = attention_rows(plain, text[s][:n])[-1]
            assert rel_err(got[b], want) <= 2e-2, (step, s, rel_err(got[b], want))
    m.caches.check()
    ops.tc_error_state()
    assert m.caches.seq_lens.tolist() == [132, 0, 73, 0, 0, 4]


def test_a_step_is_the_sparse_layers_where_that_takes_every_position():
    batch, start = 5, 100
    m = model(page=64)
    contiguous = decode.DecodeCaches(SHAPE, batch, 128, "cuda", fill=start)
    sparse = decode.DecodeLayer(SHAPE, weights(), index_weights=decode.make_indexer_weights(SHAPE, "cuda", std=0.05),
                                caches=contiguous, index_topk=2048)
    sparse.reduce = False
    offsets = torch.arange(batch + 1, device="cuda", dtype=torch.int32) * start
    m.caches.append((contiguous.kv[:, :start].reshape(-1, 512), contiguous.pe[:, :start].reshape(-1, 64)),
                    ints(range(batch)), offsets=offsets)
    hidden = prompt(batch, 3)
    normed = ops.fused_rms_norm(hidden, m.ones_h, eps=SHAPE.eps)
    want = sparse.decode_attention(normed, start)
    seqs = ints(range(batch))
    slots = m.caches.extend(batch, seqs)
    got = m.decode_attention(normed, seqs, slots, torch.full((batch,), start, device="cuda"))
    assert rel_err(got, want) <= 2e-2
    # the new rows are the same bits in both caches
    kv = m.caches.kv.view(-1, 512)[slots.long()]
    assert torch.equal(kv.view(torch.int16), contiguous.kv[:, start].view(torch.int16))
    assert torch.equal(m.caches.pe.view(-1, 64)[slots.long()].view(torch.int16), contiguous.pe[:, start].view(torch.int16))
    ops.tc_error_state()


def test_a_captured_step_replays_and_grows():
    m = model(window=50, sinks=2)
    twin = model(window=50, sinks=2)
    for x in (m, twin):
        x.prefill(prompt(31, 1), ints([0]), 1)
        x.prefill(prompt(64, 2), ints([3]), 1)
    hidden, seqs = prompt(2, 5), ints([3, 0])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        with torch.cuda.graph(graph, stream=side):
            out = m.decode_stack(hidden, seqs, 2)
    torch.cuda.synchronize()
    assert m.caches.seq_lens.tolist() == twin.caches.seq_lens.tolist()       # capturing runs nothing
    for _ in range(4):
        graph.replay()
        want = twin.decode_stack(hidden, seqs, 2)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert m.caches.seq_lens.tolist() == [35, 0, 0, 68, 0, 0]
    assert torch.equal(m.caches.block_table, twin.caches.block_table)
    ops.tc_error_state()


def test_forked_samples_share_their_prompt():
    """Two samples of one prompt decode like two copies of it."""
    m, twin = model(), model()
    text = prompt(75, 4)
    m.prefill(text, ints([0]), 1)
    m.caches.fork(ints([0]), ints([4]))
    for s in (0, 4):
        twin.prefill(text, ints([s]), 1)
    used = int((m.caches.refcount > 0).sum())
    assert used == 4 and int((twin.caches.refcount > 0).sum()) == 6
    for step in range(3):
        hidden = prompt(2, 20 + step)
        a, b = m.decode_stack(hidden, ints([0, 4]), 1), twin.decode_stack(hidden, ints([0, 4]), 1)
        assert torch.equal(a, b)
        if step == 1:
            m.caches.compact()
    m.caches.free(ints([0]))
    assert torch.equal(m.decode_stack(hidden[:1], ints([4]), 1), twin.decode_stack(hidden[:1], ints([4]), 1))
    m.caches.check()


def test_two_rank_partials_sum_to_the_single_rank_result():
    whole = model()
    whole.prefill(prompt(40, 6), ints([1]), 1)
    normed = ops.fused_rms_norm(prompt(1, 7), whole.ones_h, eps=SHAPE.eps)
    parts = []
    for m in (whole, model(rank=0, world=2), model(rank=1, world=2)):
        if m is not whole:                                  # the caches are those of every rank alike
            m.caches = paging.PagedCaches(SHAPE, 64, 32, 6, 20, "cuda")
            m.caches.append((whole.caches.kv.view(-1, 512)[:40], whole.caches.pe.view(-1, 64)[:40]), ints([1]),
                            offsets=ints([0, 40]))
        slots = m.caches.extend(1, ints([1]))
        parts.append(m.decode_attention(normed, ints([1]), slots, torch.tensor([40], device="cuda")).float())
    assert rel_err(parts[1] + parts[2], parts[0]) <= 2e-2
    ops.tc_error_state()


def test_a_pool_that_is_full_is_reported():
    m = model(pages=2)
    m.prefill(prompt(64, 8), ints([0]), 1)
    m.decode_stack(prompt(1, 9), ints([0]), 1)
    with pytest.raises(RuntimeError, match="1 pages were lacking"):
        m.caches.check()
    assert m.caches.seq_lens.tolist()[0] == 64


def test_a_prompt_for_a_sequence_that_holds_tokens_is_refused():
    """Positions and attention of a prompt begin at 0, so a second one has no place behind the first."""
    m, twin = model(), model()
    for x in (m, twin):
        x.prefill(prompt(40, 1), ints([1]), 1)
        x.prefill(prompt(20, 3), ints([0]), 1)
    m.prefill(prompt(24, 2), ints([1]), 1)
    with pytest.raises(RuntimeError, match="1 entries were refused .0 pages"):
        m.caches.check()
    for name in ("kv", "pe", "block_table", "seq_lens", "refcount"):
        a, b = getattr(m.caches, name), getattr(twin.caches, name)
        assert torch.equal(a, b), name
    # padding is not refused, a number out of range is; a sequence that was given back takes a new prompt
    m.prefill(prompt(24, 2), ints([-1]), 1)
    m.caches.check()
    m.prefill(prompt(24, 2), ints([6]), 1)
    with pytest.raises(RuntimeError, match="1 entries were refused"):
        m.caches.check()
    m.caches.free(ints([1]))
    again = m.prefill(prompt(24, 2), ints([1]), 1)
    m.caches.check()
    assert m.caches.seq_lens.tolist() == [20, 24, 0, 0, 0, 0]
    assert torch.equal(again, twin.prefill(prompt(24, 2), ints([4]), 1))


def test_a_captured_prompt_is_refused_on_its_second_replay():
    m = model()
    hidden, seq = prompt(33, 1), ints([2])
    m.prefill(hidden, ints([3]), 1)
    m.caches.free(ints([3]))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        with torch.cuda.graph(graph, stream=side):
            m.prefill(hidden, seq, 1)
    torch.cuda.synchronize()
    graph.replay()
    m.caches.check()
    assert m.caches.seq_lens.tolist() == [0, 0, 33, 0, 0, 0]
    graph.replay()
    with pytest.raises(RuntimeError, match="1 entries were refused"):
        m.caches.check()
    assert m.caches.seq_lens.tolist() == [0, 0, 33, 0, 0, 0]


def test_the_attention_half_of_a_step_without_sequences():
    m = model()
    none = ints([])
    normed = ops.fused_rms_norm(prompt(1, 1), m.ones_h, eps=SHAPE.eps)[:0]
    out = m.decode_attention(normed, none, m.caches.extend(0, none), torch.zeros(0, device="cuda", dtype=torch.int64))
    assert out.shape == (0, SHAPE.hidden)
    m.caches.check()
    assert not m.caches.seq_lens.any()
