"""The paged-cache operators of racetrack_b200 as cases to time: attention of new tokens over a paged
latent cache (MLA), causal attention with a sliding window and sinks, and the upkeep of a cache's
pages. Sizes are those of the DeepSeek-V3.2 block this package serves (128 heads, 16 on each of
eight ranks; latent 512, rope 64, values 128) and of the batches and contexts bench.py runs it at.
"""
from __future__ import annotations

import math
import random

import torch

own = False

LATENT, ROPE, NOPE, V_DIM = 512, 64, 128, 128
SCALE = (NOPE + ROPE) ** -0.5
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def listed() -> list[dict]:
    return [
        # one sequence at its first positions on a rank with 16 heads: latency alone
        {"name": "paged_1x17_h16", "op": "decode", "batch": 1, "longest": 17, "spread": False, "heads": 16,
         "page": 64, "window": 0, "sinks": 0, "padding": 0},
        # a full decode batch on one GPU with all heads, contexts of 4096 (bench.py's decode workload)
        {"name": "paged_64x4096_h128", "op": "decode", "batch": 64, "longest": 4096, "spread": False, "heads": 128,
         "page": 64, "window": 0, "sinks": 0, "padding": 0},
        # continuous batching on a rank with 16 heads: contexts of very different lengths, sequences in
        # any order of their slots, three padding rows behind the batch
        {"name": "paged_ragged_h16", "op": "decode", "batch": 48, "longest": 32768, "spread": True, "heads": 16,
         "page": 64, "window": 0, "sinks": 0, "padding": 3},
        # many long chats under a window of the last 1024 positions and the first 4, small pages
        {"name": "paged_window_h32", "op": "decode", "batch": 128, "longest": 8192, "spread": True, "heads": 32,
         "page": 16, "window": 1024, "sinks": 4, "padding": 0},
        # a short ragged prompt on a rank, window shorter than a key tile's end
        {"name": "window_777_h16", "op": "prefill", "tokens": 777, "heads": 16, "window": 200, "sinks": 4},
        # the prompt size of bench.py on a rank of four, the window an eighth of it
        {"name": "window_8192_h32", "op": "prefill", "tokens": 8192, "heads": 32, "window": 1024, "sinks": 64},
        # a decode step's rows of 64 sequences; a few of them cross into a new page
        {"name": "append_64x1", "op": "append", "seqs": 64, "longest": 4096, "page": 64, "new": 64, "pages": 6000},
        # chunks of prompts of odd lengths, 8192 tokens in all
        {"name": "append_8192", "op": "append", "seqs": 12, "longest": 4096, "page": 64, "new": 8192, "pages": 2000},
        # a few samples of one prompt take the slots of finished ones
        {"name": "fork_4", "op": "fork", "parents": 1, "children": 4, "longest": 1500, "page": 64, "pages": 600},
        # parallel sampling of many prompts
        {"name": "fork_512", "op": "fork", "parents": 32, "children": 16, "longest": 8192, "page": 64, "pages": 16000},
        # a nearly idle pool is packed, and a large fragmented one
        {"name": "compact_500", "op": "compact", "seqs": 9, "longest": 800, "page": 64, "pages": 500},
        {"name": "compact_16384", "op": "compact", "seqs": 128, "longest": 8192, "page": 64, "pages": 16384},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["decode", "decode", "decode", "prefill", "prefill", "append", "fork", "compact"])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "decode":
        batch = _log_int(rng, 1, 128)
        longest = _log_int(rng, 1, min(32768, 400_000 // batch))
        heads = rng.choice([5, 8, 16, 16, 24, 32, 64, 100, 128])
        windowed = rng.random() < 0.4
        return {"op": op, "batch": batch, "longest": longest, "spread": rng.random() < 0.6, "heads": heads,
                "page": page, "window": _log_int(rng, 1, 8192) if windowed else 0,
                "sinks": rng.choice([0, 1, 4, 64, 100]) if windowed else 0, "padding": rng.choice([0, 0, 1, 5])}
    if op == "prefill":
        tokens, heads = _log_int(rng, 1, 8192), rng.choice([8, 16, 32])
        return {"op": op, "tokens": tokens, "heads": heads, "window": _log_int(rng, 1, 1024),
                "sinks": rng.choice([0, 1, 4, 64, 64, 300]) if tokens < 4096 else rng.choice([0, 4, 64])}
    if op == "append":
        seqs = _log_int(rng, 1, 256)
        return {"op": op, "seqs": seqs, "longest": _log_int(rng, 1, 4096 if seqs <= 128 else 1024), "page": page,
                "new": seqs if rng.random() < 0.5 else _log_int(rng, seqs, 8192), "pages": 0}
    if op == "fork":
        return {"op": op, "parents": _log_int(rng, 1, 32), "children": _log_int(rng, 1, 16),
                "longest": _log_int(rng, 1, 4096), "page": page, "pages": 0}
    return {"op": op, "seqs": _log_int(rng, 1, 128), "longest": _log_int(rng, 1, 4096), "page": page, "pages": 0}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _normal(gen, *size):
    return torch.empty(*size, device="cuda", dtype=BF16).normal_(generator=gen)


def _lengths(n: int, longest: int, spread: bool = True) -> list[int]:
    """The n lengths of a case: all `longest`, or spread over their logarithm, the longest among them."""
    if not spread:
        return [longest] * n
    r = random.Random(n * 1_000_003 + longest)
    lo = max(1, longest // 64)
    return [longest] + [_log_int(r, lo, longest) for _ in range(n - 1)]


def _cut(total: int, n: int) -> list[int]:
    """n odd-sized shares of `total`, one at least each."""
    r = random.Random(n * 1_000_003 + total)
    w = [r.uniform(0.3, 1.7) for _ in range(n)]
    shares = [1 + int((total - n) * x / sum(w)) for x in w]
    shares[-1] += total - sum(shares)
    return shares


def _pool_pages(case: dict) -> int:
    """Pages of the pool: as the case says, or twice what its sequences and one call can need."""
    page = case["page"]
    if case["op"] == "append":
        need = sum(-(-n // page) for n in _lengths(case["seqs"], case["longest"])) + case["new"] // page + case["seqs"]
    elif case["op"] == "fork":
        need = sum(-(-n // page) for n in _lengths(case["parents"], case["longest"]))
        need += case["parents"] * case["children"] * (1 + -(-case["longest"] // (8 * page)))
    else:
        need = sum(-(-n // page) for n in _lengths(case["seqs"], case["longest"]))
    return max(case.get("pages", 0), 2 * need)


def _table(r, lengths: list[int], page: int, pages: int, width: int):
    """block_table, seq_lens, refcount of sequences whose pages lie anywhere in the pool."""
    ids = r.sample(range(pages), sum(-(-n // page) for n in lengths))
    table = torch.full((len(lengths), width), -1, dtype=I32)
    count = torch.zeros(pages, dtype=I32)
    for s, n in enumerate(lengths):
        k = -(-n // page)
        mine = torch.tensor([ids.pop() for _ in range(k)], dtype=I32)
        table[s, :k] = mine
        count[mine.long()] = 1
    return table.cuda(), torch.tensor(lengths, dtype=I32).cuda(), count.cuda()


def _prepare_decode(case: dict, gen, r) -> dict:
    lengths = _lengths(case["batch"], case["longest"], case["spread"])
    r.shuffle(lengths)
    page, heads, rows = case["page"], case["heads"], case["batch"] + case["padding"]
    pages = sum(-(-n // page) for n in lengths) + 3
    table, lens, _ = _table(r, lengths, page, pages, -(-case["longest"] // page) + 1)
    order = list(range(case["batch"]))
    r.shuffle(order)
    s = {"kv": _normal(gen, pages, page, LATENT), "pe": _normal(gen, pages, page, ROPE),
         # what the absorbed projection leaves: wide rows of moderate size
         "q_abs": _normal(gen, rows, heads, LATENT) * 0.5, "q_pe": _normal(gen, rows, heads, ROPE),
         "table": table, "lens": lens}
    # slots in the order of the batch, padding rows behind it; None: row b is slot b
    s["seqs"] = torch.tensor(order + [-1] * case["padding"], dtype=I32).cuda() if case["padding"] else None
    return s


def _prepare_append(case: dict, gen, r) -> dict:
    n, page = case["seqs"], case["page"]
    lengths, shares = _lengths(n, case["longest"]), _cut(case["new"], n)
    r.shuffle(lengths)
    pages = _pool_pages(case)
    width = -(-(case["longest"] + max(shares)) // page) + 1
    table, lens, count = _table(r, lengths, page, pages, width)
    order = list(range(n))
    r.shuffle(order)
    s = {"kv": _normal(gen, pages, page, LATENT), "pe": _normal(gen, pages, page, ROPE), "table": table,
         "lens": lens, "count": count, "seqs": torch.tensor(order, dtype=I32).cuda(),
         "new_kv": _normal(gen, case["new"], LATENT), "new_pe": _normal(gen, case["new"], ROPE)}
    starts = [0]
    for k in shares:
        starts.append(starts[-1] + k)
    s["offsets"] = None if case["new"] == n else torch.tensor(starts, dtype=I32).cuda()
    return s


def _prepare_fork(case: dict, gen, r) -> dict:
    # parents in the first slots, what their children replace (shorter finished sequences) behind them
    parents, kids, page = case["parents"], case["parents"] * case["children"], case["page"]
    lengths = _lengths(parents, case["longest"])
    r.shuffle(lengths)
    old = [max(1, case["longest"] // 8 - k % 7) for k in range(kids)]
    pages = _pool_pages(case)
    table, lens, count = _table(r, lengths + old, page, pages, -(-case["longest"] // page) + 1)
    src = [k // case["children"] for k in range(kids)]
    dst = list(range(parents, parents + kids))
    r.shuffle(dst)
    return {"kv": _normal(gen, pages, page, LATENT), "pe": _normal(gen, pages, page, ROPE), "table": table,
            "lens": lens, "count": count, "src": torch.tensor(src, dtype=I32).cuda(),
            "dst": torch.tensor(dst, dtype=I32).cuda()}


def _prepare_compact(case: dict, gen, r) -> dict:
    lengths = _lengths(case["seqs"], case["longest"])
    r.shuffle(lengths)
    pages = _pool_pages(case)
    table, lens, count = _table(r, lengths, case["page"], pages, -(-case["longest"] // case["page"]))
    return {"kv": _normal(gen, pages, case["page"], LATENT), "pe": _normal(gen, pages, case["page"], ROPE),
            "table": table, "lens": lens, "count": count}


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = random.Random(seed)
    op = case["op"]
    if op == "decode":
        s = _prepare_decode(case, gen, r)
    elif op == "prefill":
        t, h = case["tokens"], case["heads"]
        s = {"q": _normal(gen, t, h, NOPE + ROPE), "kv_b": _normal(gen, t, h, NOPE + V_DIM),
             "k_pe": _normal(gen, t, ROPE)}
    else:
        s = {"append": _prepare_append, "fork": _prepare_fork, "compact": _prepare_compact}[op](case, gen, r)
        # refused entries and the pages they lacked
        s["status"] = torch.zeros(2, dtype=I32, device="cuda")
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------

def _softmax(scores: torch.Tensor) -> torch.Tensor:
    """Softmax over the last dimension with -inf for what is masked; a row without any key is zero."""
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_decode(s: dict) -> torch.Tensor:
    case, table, lens = s["case"], s["table"], s["lens"]
    if s["seqs"] is not None:
        slot = s["seqs"].clamp(min=0).long()
        table, lens = table[slot], torch.where(s["seqs"] < 0, 0, lens[slot])
    rows, width = table.shape
    where = table.clamp(min=0).long()
    kv = s["kv"][where].reshape(rows, -1, LATENT).float()
    pe = s["pe"][where].reshape(rows, -1, ROPE).float()
    scores = torch.matmul(s["q_abs"].float(), kv.transpose(1, 2))
    scores = (scores + torch.matmul(s["q_pe"].float(), pe.transpose(1, 2))) * SCALE
    pos = torch.arange(kv.shape[1], device=kv.device)
    seen = pos < lens[:, None]
    if case["window"]:
        seen = seen & ((pos >= lens[:, None] - case["window"]) | (pos < case["sinks"]))
    scores = scores.masked_fill(~seen[:, None, :], -math.inf)
    # rows behind a sequence's end are whatever the pages hold
    kv = kv.masked_fill(~seen[:, :, None], 0.0)
    return torch.matmul(_softmax(scores), kv).to(BF16)


def _plain_prefill(s: dict) -> torch.Tensor:
    case, kv_b = s["case"], s["kv_b"].float()
    t = kv_b.shape[0]
    k = torch.cat((kv_b[..., :NOPE], s["k_pe"].float()[:, None, :].expand(-1, kv_b.shape[1], -1)), dim=-1)
    scores = torch.matmul(s["q"].float().transpose(0, 1), k.permute(1, 2, 0)) * SCALE
    i = torch.arange(t, device=kv_b.device)[:, None]
    j = torch.arange(t, device=kv_b.device)[None, :]
    seen = (j <= i) & ((j > i - case["window"]) | (j < case["sinks"]))
    p = _softmax(scores.masked_fill_(~seen, -math.inf))
    return torch.matmul(p, kv_b[..., NOPE:].transpose(0, 1)).transpose(0, 1).to(BF16).contiguous()


def _plain_append(s: dict, table, lens, count) -> None:
    page, width = s["kv"].shape[1], table.shape[1]
    seqs = s["seqs"].long()
    n = seqs.numel()
    offsets = s["offsets"] if s["offsets"] is not None else torch.arange(n + 1, dtype=I32, device=table.device)
    old, new = lens[seqs], offsets[1:] - offsets[:-1]
    have, want = (old + page - 1) // page, (old + new + page - 1) // page
    # the lowest free pages, in the order of the list
    slot = torch.arange(width, device=table.device)
    fresh = (slot >= have[:, None]) & (slot < want[:, None])
    pick = torch.nonzero(count == 0)[:, 0][:int(fresh.sum())].to(I32)
    rows = table[seqs]
    rows[fresh] = pick
    table[seqs] = rows
    count[pick.long()] = 1
    lens[seqs] = old + new
    token = torch.arange(s["new_kv"].shape[0], device=table.device)
    of = torch.searchsorted(offsets[1:].contiguous(), token.to(I32), right=True)
    pos = old[of] + (token - offsets[of])
    at = rows[of, pos // page].long()
    s["kv"][at, pos % page] = s["new_kv"]
    s["pe"][at, pos % page] = s["new_pe"]


def _plain_free(table, lens, count, seqs) -> None:
    rows = table[seqs.long()]
    gone = rows[rows >= 0].long()
    count.index_add_(0, gone, torch.full_like(gone, -1, dtype=I32))
    table[seqs.long()] = -1
    lens[seqs.long()] = 0


def _plain_fork(s: dict, table, lens, count) -> None:
    page = s["kv"].shape[1]
    src, dst = s["src"].long(), s["dst"].long()
    size, rows = lens[src], table[src]
    full, tail = size // page, size % page
    slot = torch.arange(table.shape[1], device=table.device)
    shared = slot < full[:, None]
    kept = rows[shared].long()
    count.index_add_(0, kept, torch.ones_like(kept, dtype=I32))
    # a partial last page is copied, so that parent and child write into their own
    has = torch.nonzero(tail > 0)[:, 0]
    pick = torch.nonzero(count == 0)[:, 0][:has.numel()]
    count[pick] = 1
    last = rows[has, full[has]].long()
    new = torch.where(shared, rows, torch.full_like(rows, -1))
    new[has, full[has]] = pick.to(I32)
    r = torch.arange(page, device=table.device)
    which, row = torch.nonzero(r < tail[has][:, None], as_tuple=True)
    for buf in (s["kv"], s["pe"]):
        buf[pick[which], row] = buf[last[which], row]
    table[dst] = new
    lens[dst] = size


def _plain_compact(s: dict, table, count) -> None:
    page_id = torch.arange(count.numel(), device=count.device)
    live = count > 0
    n = live.sum()
    src, dst = torch.nonzero(live & (page_id >= n))[:, 0], torch.nonzero(~live & (page_id < n))[:, 0]
    to = page_id.clone()
    to[src] = dst
    s["kv"][dst] = s["kv"][src]
    s["pe"][dst] = s["pe"][src]
    count[dst] = count[src]
    count[src] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(I32), table))


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def _decode(s: dict):
    if not own:
        return _plain_decode(s)
    from racetrack_b200 import ops
    case = s["case"]
    return ops.mla_paged_decode(s["q_abs"], s["q_pe"], s["kv"], s["pe"], s["table"], s["lens"], SCALE, seqs=s["seqs"],
                                window=case["window"] or None, sinks=case["sinks"])


def _prefill(s: dict):
    if not own:
        return _plain_prefill(s)
    from racetrack_b200 import ops
    case, kv_b = s["case"], s["kv_b"]
    return ops.attention_prefill(s["q"], kv_b[..., :NOPE], s["k_pe"], kv_b[..., NOPE:], SCALE,
                                 window=case["window"], sinks=case["sinks"])


def _upkeep(s: dict) -> tuple:
    """Upkeep starts from the tables as they were, in every pass: the call changes them in place, and
    what it writes into the pages are rows that no sequence those tables keep has."""
    op, pages = s["case"]["op"], (s["kv"], s["pe"])
    table, lens, count = s["table"].clone(), s["lens"].clone(), s["count"].clone()
    if not own:
        if op == "append":
            _plain_append(s, table, lens, count)
        elif op == "fork":
            _plain_free(table, lens, count, s["dst"])
            _plain_fork(s, table, lens, count)
        else:
            _plain_compact(s, table, count)
    else:
        from racetrack_b200 import ops
        if op == "append":
            ops.page_append(pages, (s["new_kv"], s["new_pe"]), table, lens, count, s["status"], s["seqs"],
                            offsets=s["offsets"])
        elif op == "fork":
            ops.page_free(table, lens, count, s["dst"])
            ops.page_fork(pages, table, lens, count, s["status"], s["src"], s["dst"])
        else:
            ops.page_compact(pages, table, count)
    return table, lens, count, s["status"], *pages


def run(state: dict):
    op = state["case"]["op"]
    return _decode(state) if op == "decode" else _prefill(state) if op == "prefill" else _upkeep(state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------

def _seen(n: int, window: int, sinks: int) -> int:
    """Positions that the newest of n positions attends to."""
    return n if not window or window >= n else window + min(sinks, n - window)


def _prefill_pairs(case: dict) -> int:
    return sum(_seen(i + 1, case["window"], case["sinks"]) for i in range(case["tokens"]))


ROW = 2 * (LATENT + ROPE)       # bytes of a cached position


def work(case: dict) -> dict:
    op = case["op"]
    if op == "decode":
        seen = sum(_seen(n, case["window"], case["sinks"]) for n in _lengths(case["batch"], case["longest"], case["spread"]))
        rows = (case["batch"] + case["padding"]) * case["heads"]
        return {"bytes": seen * ROW + rows * (ROW + 2 * LATENT), "flops": 2 * seen * case["heads"] * (2 * LATENT + ROPE)}
    if op == "prefill":
        t, h = case["tokens"], case["heads"]
        return {"bytes": 2 * t * (h * (NOPE + ROPE + NOPE + 2 * V_DIM) + ROPE),
                "flops": 2 * _prefill_pairs(case) * h * (NOPE + ROPE + V_DIM)}
    page, pages = case["page"], _pool_pages(case)
    if op == "append":
        lengths, n = _lengths(case["seqs"], case["longest"]), case["seqs"]
        return {"bytes": 2 * case["new"] * ROW + 4 * (4 * n + case["new"] // page), "flops": 0}
    if op == "fork":
        lengths = _lengths(case["parents"], case["longest"])
        kids = case["children"]
        tails = kids * sum(n % page for n in lengths)
        entries = kids * sum(-(-n // page) for n in lengths)
        return {"bytes": 2 * tails * ROW + 4 * 4 * entries, "flops": 0}
    live = sum(-(-n // page) for n in _lengths(case["seqs"], case["longest"]))
    moved = live * (pages - live) // pages          # pages lie anywhere: this share of the live ones is out of place
    return {"bytes": 2 * moved * page * ROW + 4 * (2 * pages + 2 * live), "flops": 0}


# ---------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    """Attention from its definition, a sequence or a head at a time. Upkeep moves values and computes none."""
    if case["op"] not in ("decode", "prefill"):
        return None
    s = prepare(case, seed)
    if case["op"] == "decode":
        lens = s["lens"].tolist()
        rows, heads = s["q_abs"].shape[:2]
        slots = s["seqs"].tolist() if s["seqs"] is not None else range(rows)
        out = torch.zeros(rows, heads, LATENT, device="cuda", dtype=torch.float64)
        for b, slot in enumerate(slots):
            n = lens[slot] if slot >= 0 else 0
            if n == 0:
                continue
            pos = torch.arange(n, device="cuda")
            if case["window"]:
                pos = pos[(pos >= n - case["window"]) | (pos < case["sinks"])]
            at, row = s["table"][slot].long()[pos // case["page"]], pos % case["page"]
            kv = s["kv"][at, row].double()
            key = torch.cat((kv, s["pe"][at, row].double()), dim=1)
            q = torch.cat((s["q_abs"][b].double(), s["q_pe"][b].double()), dim=1)
            out[b] = torch.softmax(q @ key.T * SCALE, dim=1) @ kv
        return out
    t, heads = case["tokens"], case["heads"]
    out = torch.empty(t, heads, V_DIM, device="cuda", dtype=torch.float64)
    ago = torch.arange(t, device="cuda")[:, None] - torch.arange(t, device="cuda")[None, :]
    hidden = (ago < 0) | ((ago >= case["window"]) & (torch.arange(t, device="cuda")[None, :] >= case["sinks"]))
    for h in range(heads):
        k = torch.cat((s["kv_b"][:, h, :NOPE], s["k_pe"]), dim=1).double()
        scores = s["q"][:, h].double() @ k.T * SCALE
        scores[hidden] = -math.inf
        out[:, h] = torch.softmax(scores, dim=1) @ s["kv_b"][:, h, NOPE:].double()
    return out
