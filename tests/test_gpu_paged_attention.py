"""Attention of new tokens over a paged latent cache against its definition in 64 bits.

Tolerance, for an element with value o = sum p_j v_j and a = sum p_j |v_j|: the probabilities are rounded to
bf16 before they multiply the rows (2^-8 of a), the output is rounded to bf16 (2^-8 of |o|), and the scores
are fp32 sums of 576 products that are exact in fp32: off by at most 577 * 2^-24 * c with c = |scale| max_j
sum_d |q_d k_d|, a factor exp(2 e) on the probabilities; the exponential's argument s * log2(e) - m is formed
with three more roundings of the magnitude |s| <= c, and ex2 itself, the sums of p and of p v over up to n
positions add n * 2^-24 (worst order). All of it: (2^-8 (a + |o|)) + a (expm1(2 * 580 * 2^-24 * c) + (2 n + 64)
2^-24).
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from racetrack_b200 import layer, ops, paging

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def visible(n, window, sinks):
    pos = torch.arange(n, device="cuda")
    if window is None:
        return pos
    return pos[(pos >= n - window) | (pos < sinks)]


def expected(q_abs, q_pe, kv, pe, table, length, scale, window, sinks):
    """(value, tolerance) of one row in 64 bits; table: its pages as a list."""
    page = kv.shape[1]
    pos = visible(length, window, sinks)
    ids = torch.tensor(table, device="cuda", dtype=torch.int64)
    at = ids[pos // page]
    ok = (at >= 0) & (at < kv.shape[0])
    pos, at = pos[ok], at[ok]
    if not len(pos):
        zero = torch.zeros(q_abs.shape[0], 512, device="cuda", dtype=torch.float64)
        return zero, zero
    v = kv[at, pos % page].double()
    k = torch.cat((v, pe[at, pos % page].double()), 1)
    q = torch.cat((q_abs.double(), q_pe.double()), 1)
    p = torch.softmax(q @ k.T * scale, 1)
    o, a = p @ v, p @ v.abs()
    c = abs(scale) * (q.abs() @ k.abs().T).amax(1, keepdim=True)
    u = 2.0 ** -24
    return o, 2.0 ** -8 * (a + o.abs()) + a * (torch.expm1(2 * 580 * u * c) + (2 * len(pos) + 64) * u)


def make(lengths, heads, page, *, spare=3, seed=0, fill=float("nan"), width=None, combined=False, spread=1.0):
    """Caches whose pages lie anywhere, unwritten rows and free pages holding `fill`."""
    r = random.Random(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    ids = r.sample(range(pages), sum(need))
    width = width or max(need + [1]) + 1
    if combined:
        both = torch.full((pages, page, 576), fill, device="cuda", dtype=torch.bfloat16)
        kv, pe = both[..., :512], both[..., 512:]
    else:
        kv = torch.full((pages, page, 512), fill, device="cuda", dtype=torch.bfloat16)
        pe = torch.full((pages, page, 64), fill, device="cuda", dtype=torch.bfloat16)
    table = []
    for n, k in zip(lengths, need):
        row, ids = ids[:k], ids[k:]
        # entries behind the end: valid numbers of other pages, -1, and numbers out of range
        table.append(row + [r.choice([-1, 0, pages - 1, pages + 5, 2 ** 31 - 1]) for _ in range(width - k)])
        if n:
            pos = torch.arange(n, device="cuda")
            at = torch.tensor(row, device="cuda")[pos // page]
            kv[at, pos % page] = (torch.randn(n, 512, device="cuda", generator=g) * spread).bfloat16()
            pe[at, pos % page] = (torch.randn(n, 64, device="cuda", generator=g) * spread).bfloat16()
    rows = len(lengths)
    q_abs = (torch.randn(rows, heads, 512, device="cuda", generator=g) * 0.5).bfloat16()
    q_pe = torch.randn(rows, heads, 64, device="cuda", generator=g).bfloat16()
    return kv, pe, table, q_abs, q_pe


def check(got, kv, pe, table, lengths, q_abs, q_pe, scale=SCALE, window=None, sinks=0, seqs=None):
    assert got.shape == q_abs.shape and got.dtype == torch.bfloat16 and got.is_contiguous()
    for b in range(q_abs.shape[0]):
        s = seqs[b] if seqs is not None else b
        n = lengths[s] if 0 <= s < len(lengths) else 0
        want, tol = expected(q_abs[b], q_pe[b], kv, pe, table[s] if n else [], n, scale, window, sinks)
        off = (got[b].double() - want).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (f"row {b} (length {n}): {int(bad.sum())} of {bad.numel()} off, worst "
                               f"{float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance, first at {bad.nonzero()[0].tolist()}")
    ops.tc_error_state()


LENGTHS = [1, 64, 0, 63, 65, 17, 128, 129, 16, 15, 700, 191, 192]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [16, 128])
def test_lengths_around_tiles_and_pages(page, heads):
    kv, pe, table, q_abs, q_pe = make(LENGTHS, heads, page)
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(LENGTHS), SCALE)
    check(got, kv, pe, table, LENGTHS, q_abs, q_pe)


@pytest.mark.parametrize("heads", [1, 3, 8, 9, 15, 16, 17, 24, 31, 32, 33, 40, 63, 64, 65, 96, 100, 127, 128, 129, 192, 256])
def test_head_counts(heads):
    lengths = [200, 1, 77, 1000]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 64, seed=heads)
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    check(got, kv, pe, table, lengths, q_abs, q_pe)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("heads", [16, 64])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (15, 4), (64, 0), (64, 64), (65, 3), (100, 200), (256, 100),
                                           (700, 1), (10000, 5), (2 ** 40, 0)])
def test_window_and_sinks(page, heads, window, sinks):
    lengths = [1, 64, 65, 0, 300, 699, 700, 701, 1111]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, page, seed=window % 1000 + sinks)
    # what the window hides may be anything: pages that were given back, or rows of NaN
    for s, n in enumerate(lengths):
        hidden = sorted(set(range(n)) - set(visible(n, window, sinks).tolist()))
        for i in hidden[:: 7]:
            kv[table[s][i // page], i % page] = float("nan")
            pe[table[s][i // page], i % page] = float("inf")
        for m in range(-(-n // page)):
            if set(range(m * page, min(n, m * page + page))) <= set(hidden):
                table[s][m] = -1
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE, window=window, sinks=sinks)
    check(got, kv, pe, table, lengths, q_abs, q_pe, window=window, sinks=sinks)


@pytest.mark.parametrize("heads", [16, 128])
def test_rows_of_any_slots_and_padding(heads):
    lengths = [70, 3, 0, 500, 64]
    kv, pe, table, _, _ = make(lengths, heads, 32)
    seqs = [3, -1, 0, 3, 4, 99, 2, -7, 1]
    q_abs = torch.randn(len(seqs), heads, 512, device="cuda").bfloat16() * 0.5
    q_pe = torch.randn(len(seqs), heads, 64, device="cuda").bfloat16()
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE, seqs=ints(seqs))
    check(got, kv, pe, table, lengths, q_abs, q_pe, seqs=seqs)
    assert not got[1].any() and not got[5].any() and not got[6].any()


@pytest.mark.parametrize("heads", [16, 128])
def test_nothing_to_attend_to(heads):
    kv, pe, table, q_abs, q_pe = make([0, 0, 0], heads, 64)
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints([0, -5, 0]), SCALE)
    assert not got.any()
    none = ops.mla_paged_decode(q_abs[:0], q_pe[:0], kv, pe, ints(table), ints([0, 0, 0]), SCALE)
    assert none.shape == (0, heads, 512)
    # a table without a column, and lengths beyond the table, which are cut to it
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, torch.zeros(3, 0, dtype=torch.int32, device="cuda"), ints([5, 6, 7]), SCALE)
    assert not got.any()


@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("page, width", [(16, 1), (64, 1), (64, 2), (128, 1), (16, 9)])
@pytest.mark.parametrize("length", [0, 1, 15, 16])
def test_tables_of_few_tiles(heads, page, width, length):
    """Less than a CTA each: with one tile there is nothing to join."""
    lengths = [length if width == 1 else length * page * width // 16]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, page, width=width, seed=length)
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    check(got, kv, pe, table, lengths, q_abs, q_pe)


def test_lengths_beyond_the_table_are_cut():
    lengths = [128, 64]
    kv, pe, table, q_abs, q_pe = make(lengths, 16, 64, width=2)
    table[1] = table[1][:1] + [-1]
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints([2 ** 31 - 1, 128]), SCALE)
    check(got, kv, pe, table, lengths, q_abs, q_pe)


@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_out_of_the_pool_weigh_nothing(page, heads):
    lengths = [500, 300, 64, 40]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, page)
    for s, m, bad in ((0, 0, -1), (0, 3, 10 ** 6), (1, 1, -2 ** 31), (1, 300 // page, 2 ** 31 - 1)):
        table[s][m] = bad
    table[2] = [-1] * len(table[2])                       # a row all of whose pages are missing
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    check(got, kv, pe, table, lengths, q_abs, q_pe)
    assert not got[2].any()


@pytest.mark.parametrize("heads", [16, 32, 128])
def test_one_long_sequence_is_cut_over_the_gpu(heads):
    lengths = [50_001]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 128)
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    check(got, kv, pe, table, lengths, q_abs, q_pe)
    again = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("heads", [8, 128])
def test_many_short_sequences(heads):
    r = random.Random(1)
    lengths = [r.choice([0, 1, 5, 64, 90, 130]) for _ in range(1500)]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 16)
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    for part in range(0, 1500, 500):
        sl = slice(part, part + 500)
        check(got[sl], kv, pe, table[sl], lengths[sl], q_abs[sl], q_pe[sl])


@pytest.mark.parametrize("heads", [16, 128])
def test_strided_caches_and_queries(heads):
    """kv and pe as slices of one buffer with layers between its pages, queries as slices of projections."""
    lengths = [333, 64, 10]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 64, combined=True)
    layers = torch.full((kv.shape[0], 3, 64, 640), float("nan"), device="cuda", dtype=torch.bfloat16)
    layers[:, 1, :, 32:544], layers[:, 1, :, 560:624] = kv, pe
    wide = torch.zeros(3, heads, 700, device="cuda", dtype=torch.bfloat16)
    wide[..., 64:576], wide[..., 600:664] = q_abs, q_pe
    big = torch.full((3, len(table[0]) + 9), -1, dtype=torch.int32, device="cuda")
    big[:, 4:4 + len(table[0])] = ints(table)
    for kv_, pe_ in ((kv, pe), (layers[:, 1, :, 32:544], layers[:, 1, :, 560:624])):
        got = ops.mla_paged_decode(wide[..., 64:576], wide[..., 600:664], kv_, pe_, big[:, 4:4 + len(table[0])],
                                   ints(lengths), SCALE)
        check(got, kv, pe, table, lengths, q_abs, q_pe)
    # queries that every row shares (stride 0) or that lie at odd addresses are copied
    got = ops.mla_paged_decode(q_abs[:1].expand(3, -1, -1), wide[..., 1:65], kv, pe, ints(table), ints(lengths), SCALE)
    check(got, kv, pe, table, lengths, q_abs[:1].expand(3, -1, -1), wide[..., 1:65])


@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("scale", [SCALE, 1.0, -0.3, 0.0])
def test_sharp_and_flat_scores(heads, scale):
    """Scores over a wide range: the running maximum grows late, early or not at all."""
    lengths = [400, 129]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 64, seed=7, spread=3.0 if scale == SCALE else 1.0)
    ramp = torch.linspace(-4, 4, 400, device="cuda")
    pos = torch.arange(400, device="cuda")
    at = torch.tensor(table[0], device="cuda")[pos // 64]
    kv[at, pos % 64] += (ramp[:, None] * q_abs[0, 0].float()).bfloat16()
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), scale)
    check(got, kv, pe, table, lengths, q_abs, q_pe, scale=scale)


@pytest.mark.parametrize("heads", [16, 128])
def test_nan_and_infinity_that_are_seen_stay_in_their_row(heads):
    lengths = [200, 200, 200]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 64)
    q_pe[..., 3] = 1.0
    pe[table[1][1], 5, 3] = float("nan")
    pe[table[2][2], 7, 3] = float("inf")
    got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints(lengths), SCALE)
    check(got[:1], kv, pe, table, lengths, q_abs[:1], q_pe[:1])
    assert got[1:].isnan().all()                          # as torch's softmax


def test_offsets_beyond_32_bits():
    pages = (1 << 31) // (64 * 512) + 40                  # the last pages begin behind 2^31 elements
    kv = torch.empty(pages, 64, 512, device="cuda", dtype=torch.bfloat16)
    pe = torch.empty(pages, 64, 64, device="cuda", dtype=torch.bfloat16)
    table = [[pages - 1, 0, pages - 30, 5]]
    for p in table[0]:
        kv[p].normal_()
        pe[p].normal_()
    for heads in (16, 128):
        q_abs, q_pe = torch.randn(1, heads, 512, device="cuda").bfloat16(), torch.randn(1, heads, 64, device="cuda").bfloat16()
        got = ops.mla_paged_decode(q_abs, q_pe, kv, pe, ints(table), ints([250]), SCALE)
        check(got, kv, pe, table, [250], q_abs, q_pe)


@pytest.mark.parametrize("heads", [16, 128])
def test_a_captured_step_grows_its_cache(heads):
    """Append and attention in one graph, replayed while lengths cross pages; beside it a second graph."""
    lengths = [62, 1, 127]
    caches = paging.PagedCaches(layer.DSV32, 20, 64, 4, 5, "cuda")
    rows = lambda n: (torch.randn(n, 512, device="cuda").bfloat16(), torch.randn(n, 64, device="cuda").bfloat16())
    caches.append(rows(190), ints([0, 1, 3]), offsets=ints([0, 62, 63, 190]))
    seqs = ints([3, -1, 0, 1])
    state = [(rows(4), torch.randn(4, heads, 512, device="cuda").bfloat16(), torch.randn(4, heads, 64, device="cuda").bfloat16())
             for _ in range(2)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for new, q_abs, q_pe in state:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            with torch.cuda.graph(graph, stream=side):
                caches.append(new, seqs)
                outs.append(ops.mla_paged_decode(q_abs, q_pe, caches.kv, caches.pe, caches.block_table, caches.seq_lens,
                                                 SCALE, seqs=seqs, window=100, sinks=2))
        graphs.append(graph)
    torch.cuda.synchronize()
    want_len = {3: 127, 0: 62, 1: 1}
    for step in range(6):
        k = step % 2
        graphs[k].replay()
        torch.cuda.synchronize()
        want_len = {s: n + 1 for s, n in want_len.items()}
        lens, table = caches.seq_lens.tolist(), caches.block_table.tolist()
        assert {s: lens[s] for s in want_len} == want_len
        new, q_abs, q_pe = state[k]
        check(outs[k], caches.kv, caches.pe, table, lens, q_abs, q_pe, window=100, sinks=2, seqs=seqs.tolist())
    caches.check()


def test_two_streams_at_once():
    lengths = [3000, 50, 700]
    kv, pe, table, q_abs, q_pe = make(lengths, 128, 64)
    t, n = ints(table), ints(lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                h = 128 if k == 0 else 16
                outs[k].append(ops.mla_paged_decode(q_abs[:, :h], q_pe[:, :h], kv, pe, t, n, SCALE))
    torch.cuda.synchronize()
    for k, h in ((0, 128), (1, 16)):
        check(outs[k][0], kv, pe, table, lengths, q_abs[:, :h], q_pe[:, :h])
        assert all(torch.equal(o.view(torch.int16), outs[k][0].view(torch.int16)) for o in outs[k])


def test_a_cache_through_its_life():
    """Prompts come in, samples fork and grow apart, some end, the pool is packed: attention over it is that
    over the rows themselves."""
    caches = paging.PagedCaches(layer.DSV32, 60, 16, 8, 20, "cuda")
    kept = {}
    r = random.Random(3)

    def append(seqs, counts):
        kv, pe = torch.randn(sum(counts), 512, device="cuda").bfloat16(), torch.randn(sum(counts), 64, device="cuda").bfloat16()
        starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
        caches.append((kv, pe), ints(seqs), offsets=ints(starts))
        for i, s in enumerate(seqs):
            old = kept.get(s, (kv[:0], pe[:0]))
            kept[s] = tuple(torch.cat((o, x[starts[i]:starts[i + 1]])) for o, x in zip(old, (kv, pe)))

    append([0, 5], [100, 33])
    for step in range(12):
        if step == 1:
            caches.fork(ints([0, 0, 5]), ints([1, 2, 6]))
            kept.update({1: kept[0], 2: kept[0], 6: kept[5]})
        if step == 5:
            caches.free(ints([0, 6]))
            kept.pop(0), kept.pop(6)
        if step in (6, 9):
            caches.compact()
        if step == 8:
            caches.fork(ints([2, 1]), ints([1, 2]))          # two beams change places
            kept[1], kept[2] = kept[2], kept[1]
        live = sorted(kept)
        append(live, [r.randint(1, 9) for _ in live])
        q_abs = torch.randn(len(live), 16, 512, device="cuda").bfloat16()
        q_pe = torch.randn(len(live), 16, 64, device="cuda").bfloat16()
        got = ops.mla_paged_decode(q_abs, q_pe, caches.kv, caches.pe, caches.block_table, caches.seq_lens, SCALE,
                                   seqs=ints(live))
        for b, s in enumerate(live):
            kv, pe = kept[s]
            want, tol = expected(q_abs[b], q_pe[b], kv[None], pe[None], [0], len(kv), SCALE, None, 0)
            assert ((got[b].double() - want).abs() <= tol).all(), (step, s)
    caches.check()


def _call(**change):
    kv, pe, table, q_abs, q_pe = make([70, 3], 16, 64)
    args = dict(q_abs=q_abs, q_pe=q_pe, kv_pages=kv, pe_pages=pe, block_table=ints(table), seq_lens=ints([70, 3]),
                softmax_scale=SCALE)
    for name, f in change.items():
        args[name] = f(args.get(name))
    return ops.mla_paged_decode(**args)


@pytest.mark.parametrize("change, says", [
    (dict(q_abs=lambda t: t.float()), "bf16"),
    (dict(q_abs=lambda t: t[0]), "three dimensions"),
    (dict(q_abs=lambda t: t[..., :256]), "shapes must be"),
    (dict(q_pe=lambda t: t[:, :8]), "shapes must be"),
    (dict(pe_pages=lambda t: t[:, :16]), "shapes must be"),
    (dict(kv_pages=lambda t: t.cpu()), "one device"),
    (dict(kv_pages=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
    (dict(kv_pages=lambda t: t[:, :48].contiguous(), pe_pages=lambda t: t[:, :48].contiguous()), "power of two"),
    (dict(kv_pages=lambda t: t[:, :8].contiguous(), pe_pages=lambda t: t[:, :8].contiguous()), "power of two"),
    (dict(block_table=lambda t: t.long()), "int32"),
    (dict(block_table=lambda t: t.t()), "contiguous"),
    (dict(seq_lens=lambda t: t[:1]), "one entry"),
    (dict(seq_lens=lambda t: t.cpu()), "on the device"),
    (dict(seqs=lambda t: ints([0, 1, 0])), "an entry"),
    (dict(block_table=lambda t: t[:1], seq_lens=lambda t: t[:1]), "row for each query"),
    (dict(window=lambda t: 0), "window must be positive"),
    (dict(window=lambda t: -3), "window must be positive"),
    (dict(sinks=lambda t: 4), "sinks go with a window"),
    (dict(window=lambda t: 4, sinks=lambda t: -1), "sinks"),
])
def test_what_is_refused(change, says):
    with pytest.raises(RuntimeError, match=says):
        _call(**change)


@pytest.mark.parametrize("name, width", [("kv_pages", 512), ("pe_pages", 64)])
def test_pages_whose_rows_overlap_are_refused(name, width):
    for view in (lambda t: t[:1].expand(t.shape[0], -1, -1), lambda t: t[:, :1].expand(-1, t.shape[1], -1),
                 lambda t: t.as_strided(t.shape, (t.stride(0), width - 8, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            _call(**{name: view})


@pytest.mark.parametrize("heads", [1, 16, 128])
def test_rows_of_one_head_or_sequence_and_pages_of_interleaved_rows(heads):
    """What a dimension of 1 has for a stride does not matter; page p's row r may lie at row r * pages + p."""
    lengths = [130]
    kv, pe, table, q_abs, q_pe = make(lengths, heads, 64)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    odd = lambda t: t.as_strided(t.shape, (3, t.stride(1) if heads > 1 else 5, 1))
    got = ops.mla_paged_decode(odd(q_abs), odd(q_pe), turned(kv), turned(pe), ints(table), ints(lengths), SCALE)
    check(got, kv, pe, table, lengths, q_abs, q_pe)
