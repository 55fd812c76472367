"""Upkeep of paged caches against a plain Python model: tables, counts and every byte of the pages."""
from __future__ import annotations

import random

import pytest
import torch

from paged_model import Model
from racetrack_b200 import layer, ops, paging

pytestmark = pytest.mark.gpu

SHAPE = layer.DSV32
EXTRA = {"index_k": ((128,), torch.float8_e4m3fn), "index_scale": ((), torch.float32)}


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(n_pages, page, max_seqs, width, extra=EXTRA):
    c = paging.PagedCaches(SHAPE, n_pages, page, max_seqs, width, "cuda", extra=extra)
    for b in c.buffers:                                   # a recognisable byte everywhere
        b.view(torch.uint8).fill_(0x35)
    return c, Model(c.buffers, n_pages, page, max_seqs, width)


def rows(c, tokens, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(tokens, *b.shape[2:], device="cuda", generator=g).to(b.dtype) for b in c.buffers]


def same(c, m):
    m.assert_same(c.block_table, c.seq_lens, c.refcount, c.status, c.buffers)


def append(c, m, seqs, counts, seed=0, offsets=True):
    r = rows(c, sum(counts), seed)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    slots = c.append(r, ints(seqs), offsets=ints(starts) if offsets else None)
    want = m.extend(seqs, counts)
    m.write(r, want)
    assert slots.tolist() == want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_by_chunks_and_single_tokens(page):
    c, m = make(40, page, 6, 9)
    append(c, m, [3, 0, 5], [page + 1, 1, 3 * page], 1)
    append(c, m, [0, 3, 4, 5], [1, 1, 1, 1], 2, offsets=False)
    append(c, m, [4, 1, 0], [page - 1, 2 * page - 1, 0], 3)
    append(c, m, [1, 4], [1, 1], 4, offsets=False)
    same(c, m)
    m.assert_consistent()
    c.check()


def test_append_of_every_sequence_without_a_list():
    c, m = make(10, 16, 3, 4)
    r = rows(c, 3, 5)
    assert c.append(r).tolist() == m.extend([0, 1, 2], [1, 1, 1])
    m.write(r, [0, 16, 32])
    same(c, m)


def test_padding_repeats_and_numbers_out_of_range_are_refused_one_by_one():
    c, m = make(12, 16, 4, 3)
    append(c, m, [2, -1, 2, 7, 1, -5], [5, 3, 4, 2, 17, 1], 6)
    same(c, m)
    assert c.status.tolist() == [2, 0]                    # the second mention of 2, and 7
    append(c, m, [1], [2 * 16], 7)                        # 17 + 32 = 49 positions are four pages: one too many
    same(c, m)
    with pytest.raises(RuntimeError, match="3 entries"):
        c.check()
    c.check()


def test_a_full_pool_refuses_what_does_not_fit_and_serves_the_rest():
    c, m = make(4, 16, 5, 8)
    append(c, m, [0, 1], [33, 16], 8)                     # three pages and one: the pool is full
    append(c, m, [1, 0, 2], [1, 5, 0], 9)                 # 1 needs a page; 0 has room left; 2 needs none
    same(c, m)
    assert c.status.tolist() == [1, 1]
    c.free(ints([0]))
    m.free([0])
    append(c, m, [1, 2, 3], [20, 16, 17], 10)             # two pages, one, and two more than are left
    same(c, m)
    m.assert_consistent()


def test_offsets_beyond_the_rows_stay_inside():
    c, m = make(8, 16, 3, 4)
    r = rows(c, 5, 11)
    # rows 0-1 to sequence 0, rows 2-4 to 1 (whose end lies beyond the rows), none to 2
    slots = c.append(r, ints([0, 1, 2]), offsets=ints([0, 2, 400, 500]))
    want = m.extend([0, 1, 2], [2, 3, 0])
    m.write(r, want)
    assert slots.tolist() == want
    same(c, m)
    # overlapping offsets ask for more pages than there are tokens: whatever is served, tables stay whole
    c2, _ = make(64, 16, 8, 8)
    c2.append(rows(c2, 16, 12), ints([0, 1, 2, 3]), offsets=ints([0, 16, 0, 16, 0]))
    table = c2.block_table.cpu()
    count = torch.bincount(table[table >= 0], minlength=64)
    assert torch.equal(count, c2.refcount.cpu().long())


def test_rows_at_any_pitch_and_slots_outside():
    c, m = make(6, 16, 2, 3, extra=None)
    wide = torch.randn(7, 600, device="cuda").to(torch.bfloat16)
    r = [wide[:, 8:520], wide[:, 521:585]]                # the second starts at an odd 2-byte offset
    slots = ints([0, -1, 95, 96, 40, 2 ** 31 - 1, 17])
    ops.page_write(c.buffers, r, slots)
    m.write(r, slots.tolist())
    same(c, m)


@pytest.mark.parametrize("page", [16, 64])
def test_fork_shares_full_pages_and_copies_the_tail(page):
    c, m = make(40, page, 10, 6)
    append(c, m, [0, 1, 2, 3], [2 * page + 5, 3 * page, 7, 0], 20)
    append(c, m, [8, 9], [page + 1, 2], 21)
    pairs = ([0, 0, 1, 2, 3, 1], [4, 8, 5, 9, 6, 7])
    c.fork(ints(pairs[0]), ints(pairs[1]))
    m.fork(*pairs)
    same(c, m)
    m.assert_consistent()
    append(c, m, [0, 4, 8, 9, 2], [1, 2, 3, page, 1], 22)     # holders of the same pages grow apart
    same(c, m)
    c.free(ints([0, 4, 0, -1, 99]))                       # one named twice, padding, out of range
    m.free([0, 4])
    same(c, m)
    m.assert_consistent()


def test_fork_lets_beams_change_places():
    c, m = make(20, 16, 4, 4)
    append(c, m, [0, 1, 2, 3], [20, 33, 16, 5], 23)
    pairs = ([1, 0, 2, 0], [0, 1, 2, 3])                  # 0 and 1 swap, 2 stays, 3 becomes a second 0
    c.fork(ints(pairs[0]), ints(pairs[1]))
    m.fork(*pairs)
    same(c, m)
    m.assert_consistent()


def test_fork_refuses_repeats_numbers_out_of_range_and_a_full_pool():
    c, m = make(6, 16, 5, 4)
    append(c, m, [0, 1], [20, 17], 24)                    # four pages of six
    pairs = ([0, 1, 7, 0, -1, 1, 0], [2, 2, 3, 9, 4, 3, 4])
    c.fork(ints(pairs[0]), ints(pairs[1]))                # 2, 3 take the last two tails; 4 finds none
    m.fork(*pairs)
    same(c, m)
    m.assert_consistent()
    assert c.status.tolist() == [4, 1]


def test_compact_packs_the_pages_in_use():
    c, m = make(50, 16, 8, 10)
    append(c, m, list(range(8)), [40, 7, 100, 1, 33, 64, 16, 90], 25)
    c.fork(ints([2]), ints([1]))
    m.fork([2], [1])
    c.free(ints([0, 3, 5]))
    m.free([0, 3, 5])
    for _ in range(2):                                    # the second time nothing is left to move
        assert c.compact().tolist() == list(m.compact())
        same(c, m)
        m.assert_consistent()


def test_compact_of_an_empty_and_of_a_full_pool():
    c, m = make(4, 16, 2, 4)
    assert c.compact().tolist() == [0, 0]
    append(c, m, [0, 1], [33, 16], 26)
    assert c.compact().tolist() == [4, 0]
    same(c, m)


def test_copy_of_pages():
    c, m = make(9, 16, 2, 4)
    append(c, m, [0, 1], [40, 20], 27)
    src, dst = [0, 0, 2, -1, 9, 3], [5, 6, 7, 8, 8, 9]    # the last three name no page
    ops.page_copy(c.buffers, ints(src), ints(dst))
    for b in m.buffers:
        for s, d in ((0, 5), (0, 6), (2, 7)):
            b[d] = b[s]
    same(c, m)


@pytest.mark.parametrize("seed", range(4))
def test_a_long_run_of_all_of_them(seed):
    r = random.Random(seed)
    page, n_seqs, width = r.choice([16, 32, 64]), 12, 7
    c, m = make(45, page, n_seqs, width)
    for step in range(25):
        what = r.choice(["append", "append", "step", "fork", "free", "compact"])
        if what == "append":
            seqs = r.sample(range(n_seqs), r.randint(1, 4))
            append(c, m, seqs, [r.randint(0, 2 * page + 3) for _ in seqs], 100 * seed + step)
        elif what == "step":
            seqs = r.sample(range(n_seqs), n_seqs) + [-1]
            append(c, m, seqs, [1] * len(seqs), 100 * seed + step, offsets=False)
        elif what == "fork":
            k = r.randint(1, 5)
            src, dst = [r.randrange(n_seqs) for _ in range(k)], r.sample(range(n_seqs), k)
            c.fork(ints(src), ints(dst))
            m.fork(src, dst)
        elif what == "free":
            seqs = r.sample(range(n_seqs), r.randint(1, 3))
            c.free(ints(seqs))
            m.free(seqs)
        else:
            assert c.compact().tolist() == list(m.compact())
        m.assert_consistent()
    same(c, m)


def test_long_lists_take_several_passes_of_the_block():
    """More entries, sequences, pages and tokens than the planning block has threads."""
    n = 2500
    c, m = make(9000, 16, n, 3, extra={})
    c.kv, m.buffers = c.kv[:, :, :8].contiguous(), m.buffers   # narrow rows: the tables are what is tested
    m.buffers[0] = c.kv.cpu()
    r = random.Random(5)
    order = r.sample(range(n), n)
    append(c, m, order, [r.randint(0, 40) for _ in range(n)], 30)
    pairs = (r.sample(range(n), n), r.sample(range(n), n))
    c.fork(ints(pairs[0]), ints(pairs[1]))
    m.fork(*pairs)
    same(c, m)
    c.free(ints(order[::2]))
    m.free(order[::2])
    assert c.compact().tolist() == list(m.compact())
    same(c, m)


@pytest.mark.parametrize("tokens, forks", [(1, 1), (63, 3), (64, 4), (65, 5), (129, 9)])
def test_lists_on_both_sides_of_the_single_launch(tokens, forks):
    c, m = make(700, 16, tokens + 10, 4)
    append(c, m, list(range(tokens)), [1 + 7 * i % 31 for i in range(tokens)], 40)
    for step in range(3):
        append(c, m, list(range(tokens)), [1] * tokens, 41 + step, offsets=False)
    append(c, m, [0], [min(tokens, 33)], 44)                    # all of the rows to one sequence
    pairs = ([i % tokens for i in range(forks)], [tokens + i for i in range(forks)])
    c.fork(ints(pairs[0]), ints(pairs[1]))
    m.fork(*pairs)
    c.fork(ints(pairs[1]), ints(pairs[0][:1] + pairs[1][:-1]))  # each to its neighbour's place
    m.fork(pairs[1], pairs[0][:1] + pairs[1][:-1])
    same(c, m)
    m.assert_consistent()


def test_wide_tables_and_long_pages_fork():
    """One entry whose row of the table, and one whose pages, are more than a single block is given."""
    c, m = make(30, 16, 4, 5000, extra=None)
    append(c, m, [0, 1], [70, 33], 45)
    c.fork(ints([0]), ints([2]))
    m.fork([0], [2])
    same(c, m)
    c, m = make(3, 1024, 3, 2, extra=None)
    append(c, m, [0], [1023], 46)
    c.fork(ints([0]), ints([2]))
    m.fork([0], [2])
    same(c, m)


def test_many_buffers_at_once():
    """All layers' buffers under one table."""
    c, m = make(8, 16, 3, 3, extra={f"layer{i}": ((8,), torch.bfloat16) for i in range(60)})
    append(c, m, [0, 1], [20, 9], 31)
    c.fork(ints([0]), ints([2]))
    m.fork([0], [2])
    c.free(ints([0]))
    m.free([0])
    c.compact()
    m.compact()
    same(c, m)


def test_tables_and_buffers_may_be_slices():
    big_table = torch.full((4, 10), -1, dtype=torch.int32, device="cuda")
    table, lens = big_table[:, 3:8], torch.zeros(4, dtype=torch.int32, device="cuda")
    refs, status = torch.zeros(9, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    both = torch.zeros(9, 2, 16, 24, device="cuda", dtype=torch.bfloat16)     # two buffers page by page
    pages = (both[:, 0], both[:, 1])
    m = Model(pages, 9, 16, 4, 5)
    r = [torch.randn(30, 24, device="cuda").to(torch.bfloat16) for _ in pages]
    ops.page_append(pages, r, table, lens, refs, status, ints([1, 2]), offsets=ints([0, 18, 30]))
    m.write(r, m.extend([1, 2], [18, 12]))
    ops.page_fork(pages, table, lens, refs, status, ints([1]), ints([0]))
    m.fork([1], [0])
    ops.page_free(table, lens, refs, ints([1]))
    m.free([1])
    ops.page_compact(pages, table, refs)
    m.compact()
    m.assert_same(table, lens, refs, status, pages)
    assert (big_table[:, :3] == -1).all() and (big_table[:, 8:] == -1).all()


def test_a_captured_step_replays():
    """Growth in a graph: every replay takes the next positions, and pages when they are due."""
    c, m = make(12, 16, 3, 4)
    append(c, m, [0, 2], [14, 31], 32)
    r, seqs = rows(c, 3, 33), ints([2, 0, -1])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        with torch.cuda.graph(graph, stream=side):
            slots = c.append(r, seqs)
    torch.cuda.synchronize()
    same(c, m)                                            # capturing runs nothing
    for _ in range(4):
        graph.replay()
        want = m.extend([2, 0, -1], [1, 1, 1])
        m.write(r, want)
        torch.cuda.synchronize()
        assert slots.tolist() == want
    same(c, m)


@pytest.mark.parametrize("call, says", [
    (lambda c: c.append(rows(c, 2, 0)[:2], ints([0, 1])), "one tensor of rows"),
    (lambda c: c.append([x.float() for x in rows(c, 2, 0)], ints([0, 1])), "type and device"),
    (lambda c: c.append([x[:, None] if x.dim() > 1 else x for x in rows(c, 2, 0)], ints([0, 1])), "rows of their"),
    (lambda c: c.append(rows(c, 2, 0), ints([0, 1, 2])), "one token"),
    (lambda c: c.append(rows(c, 2, 0), ints([0, 1]), offsets=ints([0, 1, 2, 2])), "one entry more"),
    (lambda c: c.append(rows(c, 2, 0), torch.tensor([0, 1], device="cuda")), "int32"),
    (lambda c: c.append(rows(c, 2, 0), torch.tensor([0, 1], dtype=torch.int32)), "on the device"),
    (lambda c: c.append(rows(c, 9, 0)), "more entries"),
    (lambda c: c.fork(ints([0]), ints([1, 2])), "as many"),
    (lambda c: ops.page_free(c.block_table, c.seq_lens[:2], c.refcount, ints([0])), "one entry for each row"),
    (lambda c: ops.page_compact([c.kv[:3]], c.block_table, c.refcount), "one entry of refcount"),
    (lambda c: ops.page_compact([c.kv.transpose(1, 2)], c.block_table, c.refcount), "contiguous"),
    (lambda c: ops.page_compact([], c.block_table, c.refcount), "at least one"),
    (lambda c: ops.page_copy([c.kv[:, :, :256]], ints([0]), ints([1])), "contiguous"),
    (lambda c: ops.page_free(c.block_table.t(), c.seq_lens, c.refcount, ints([0])), "contiguous"),
])
def test_what_is_refused(call, says):
    c, m = make(6, 16, 4, 4)
    with pytest.raises(RuntimeError, match=says):
        call(c)
    same(c, m)


@pytest.mark.parametrize("seed", range(6))
def test_lists_whose_offsets_overlap_keep_tables_and_counts_together(seed):
    """Offsets that do not ascend are nobody's list, but every page that is named is counted, none is named twice,
    and no sequence has more entries than its length asks for."""
    r = random.Random(seed)
    c, _ = make(200, 16, 40, 12, extra=None)
    c.append(rows(c, 60, seed), ints(range(40)[::2]), offsets=ints([3 * i for i in range(21)]))
    n, tokens = 40, r.choice([30, 64, 500])
    offsets = [r.randrange(-20, tokens + 40) for _ in range(n + 1)]
    order = r.sample(range(40), n)
    c.append(rows(c, tokens, seed + 1), ints(order), offsets=ints(offsets))
    table, lens = c.block_table.cpu(), c.seq_lens.tolist()
    named = table[table >= 0]
    assert torch.equal(torch.bincount(named, minlength=200), c.refcount.cpu().long())
    assert len(set(named.tolist())) == named.numel()
    for s in range(40):
        assert int((table[s] >= 0).sum()) <= -(-lens[s] // 16) and lens[s] <= 12 * 16
