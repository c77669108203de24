"""The operators of the device-planned paged decode, as cases that can be measured.

A serving decoder keeps the self-attention keys and values of its requests in
a pool of pages, drafts a tree of tokens for each request and has the large
model check the whole tree at once. Four operators make up such a step:

  plan    block tables, slot maps, positions and tree masks from the requests'
          lengths, on the device: pages are taken from a free stack and given
          back to it;
  write   the new rows' keys and values into their pages;
  attend  attention of every drafted row over its request's cached keys and
          its own ancestors in the tree;
  accept  the longest path of drafts that the model agrees with, the
          accepted rows' keys and values moved together, the lengths advanced.

``own`` False: the plain form of each in elementary torch operations. ``own``
True: the calls of the ``wattn`` package. Both take the same state and update
it in place where the operator does.
"""
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEAD = 64           # head dimension
VOCAB = 51866       # tokens are drawn below this
MASK_WORDS = 2      # 32-bit mask words of a row's tree: up to 64 drafts a request


def _wattn():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "whisper.rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import wattn
    return wattn


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One request's draft of 16 tokens: what a single user waits for.
        {"name": "plan_one", "op": "plan", "seqs": 1, "ctx": 448, "rows": 16, "tree": True,
         "page": 64, "shape": 1},
        # 64 utterances x 5 beams, one token each, contexts of 1 to 448 tokens.
        {"name": "plan_beams", "op": "plan", "seqs": 320, "ctx": 448, "rows": 1, "tree": False,
         "page": 64, "shape": 2},
        # Many new requests with prompts of 1 to 224 tokens, in small pages.
        {"name": "plan_prompts", "op": "plan", "seqs": 2048, "ctx": 0, "rows": 224, "tree": False,
         "page": 16, "shape": 3},
        # The decode step of 320 beams, 20 heads: one layer's new rows.
        {"name": "write_step", "op": "write", "seqs": 320, "ctx": 448, "rows": 1, "tree": False,
         "page": 64, "heads": 20, "layers": 4, "src": "f16", "dtype": "f16", "shape": 2},
        # Prompts of 64 requests, f32 rows into a bf16 pool.
        {"name": "write_prompts", "op": "write", "seqs": 64, "ctx": 0, "rows": 224, "tree": False,
         "page": 64, "heads": 20, "layers": 4, "src": "f32", "dtype": "bf16", "shape": 4},
        # A single user's draft of 16 tokens over a full context, 6 heads.
        {"name": "tree_one", "op": "attend", "seqs": 1, "ctx": 448, "rows": 16, "tree": True,
         "page": 64, "heads": 6, "layers": 4, "dtype": "f16", "shape": 1},
        # Plain decode of 320 beams, one row each: the memory-bound case.
        {"name": "decode_beams", "op": "attend", "seqs": 320, "ctx": 448, "rows": 1,
         "tree": False, "page": 64, "heads": 20, "layers": 2, "dtype": "bf16", "shape": 2},
        # A batch of 64 requests with up to 33 drafts each, 20 heads.
        {"name": "tree_batch", "op": "attend", "seqs": 64, "ctx": 448, "rows": 33, "tree": True,
         "page": 64, "heads": 20, "layers": 2, "dtype": "f16", "shape": 5},
        # Long contexts and the widest trees: few rows over many keys.
        {"name": "tree_long", "op": "attend", "seqs": 8, "ctx": 32768, "rows": 64, "tree": True,
         "page": 128, "heads": 8, "layers": 1, "dtype": "bf16", "shape": 6},
        # The f32 cache (the reference's precision), 8 heads, odd tree sizes.
        {"name": "tree_f32", "op": "attend", "seqs": 16, "ctx": 448, "rows": 13, "tree": True,
         "page": 64, "heads": 8, "layers": 2, "dtype": "f32", "shape": 7},
        # One request's verified draft: 4 layers.
        {"name": "accept_one", "op": "accept", "seqs": 1, "ctx": 448, "rows": 16, "tree": True,
         "page": 64, "heads": 20, "layers": 4, "dtype": "f16", "shape": 1},
        # 32 requests with up to 64 drafts, 32 layers of 20 heads.
        {"name": "accept_batch", "op": "accept", "seqs": 32, "ctx": 448, "rows": 64, "tree": True,
         "page": 64, "heads": 20, "layers": 32, "dtype": "bf16", "shape": 8},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "accept"])
    c = {"op": op, "page": rng.choice([16, 32, 48, 64, 64, 128]), "shape": rng.randrange(1 << 20)}
    c["tree"] = op == "accept" or rng.random() < 0.6
    c["rows"] = _log(rng, 1, 64) if c["tree"] else _log(rng, 1, 224)
    if op == "plan":
        c["seqs"] = _log(rng, 1, 2048)
        c["ctx"] = rng.choice([0, _log(rng, 1, 448)])
        return c
    c["heads"] = rng.choice([1, 3, 6, 8, 12, 16, 20])
    c["dtype"] = rng.choice(["f32", "f16", "bf16"])
    if op == "write":
        c["src"] = rng.choice(["f32", "f16", "bf16"])
        c["layers"] = rng.choice([1, 2, 4])
        c["seqs"] = _log(rng, 1, 64)
        c["ctx"] = _log(rng, 1, 448)
    elif op == "attend":
        c["layers"] = rng.choice([1, 2])
        c["ctx"] = _log(rng, 1, 32768)
        # at most the keys of the largest listed case, and the rows that go with them
        c["seqs"] = _log(rng, 1, max(1, min(320, (8 * 32768 * 8) // (2 * (c["ctx"] + 64) *
                                                                    c["heads"]))))
        if c["dtype"] == "f32":  # the products of f32 rows cost several times those of 16 bits
            c["rows"] = min(c["rows"], 32)
    else:
        c["layers"] = rng.choice([1, 4, 6, 32])
        c["ctx"] = _log(rng, 1, 448)
        c["seqs"] = _log(rng, 1, 32)
        c["dtype"] = rng.choice(["f16", "bf16"])
    return c


def _shape(case):
    """The case's request lengths, new rows and parents (host arrays): they
    depend on the case alone, so that every seed has the same work."""
    r = np.random.RandomState(case["shape"])
    n, ctx, rows = case["seqs"], case["ctx"], case["rows"]
    lens = r.randint(1, ctx + 1, n) if ctx else np.zeros(n, np.int64)
    new = r.randint(1, rows + 1, n)
    if n == 1:
        lens[0], new[0] = ctx, rows  # a single request has the whole size
    else:
        lens[0], new[0], new[-1] = ctx, rows, 0 if n > 2 else 1  # one request rests
    start = np.concatenate([[0], np.cumsum(new)])
    within = np.arange(start[-1]) - np.repeat(start[:-1], new)
    if case["tree"]:
        # each draft hangs below one of the four rows before it or the root
        parent = np.maximum(within - 1 - r.randint(0, 4, len(within)) * (r.rand(len(within)) < .7), 0)
        parent = np.where(within == 0, -1, parent)
    else:
        parent = within - 1
    return lens.astype(np.int64), new.astype(np.int64), start, within, parent


def _ancestors(parent, start):
    """[rows][rows of the longest draft] truth values: itself and its ancestors."""
    n = int(start[-1])
    seq_start = np.repeat(start[:-1], np.diff(start))
    m = np.zeros((n, int(np.diff(start).max()) if n else 0), bool)
    for i in range(n):
        if parent[i] >= 0:
            m[i] = m[seq_start[i] + parent[i]]
        m[i, i - seq_start[i]] = True
    return m


def _words(m, width):
    """Truth values [rows][n] as 32-bit words [rows][width]."""
    out = np.zeros((m.shape[0], width * 32), np.uint64)
    out[:, :m.shape[1]] = m
    w = (out.reshape(-1, width, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32).view(np.int32)


def work(case):
    lens, new, start, within, parent = _shape(case)
    rows = int(start[-1])
    es = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "plan":
        # lengths, new rows, held pages and parents read; held pages, row starts and each
        # row's position, slot and mask written; each page moved once out and once back
        pages = int((-(-(lens + new) // case["page"]) - -(-lens // case["page"])).sum())
        per_row = 8 + (4 + 4 * MASK_WORDS if case["tree"] else 0)
        return {"bytes": 2 * (16 * case["seqs"]) + rows * per_row + 16 * pages, "flops": 0}
    width = case["heads"] * HEAD
    if case["op"] == "write":
        return {"bytes": rows * (2 * width * (es[case["src"]] + es[case["dtype"]]) + 4), "flops": 0}
    if case["op"] == "attend":
        seen = int((new * lens).sum()) + int(_ancestors(parent, start).sum())
        kv = int((lens + new)[new > 0].sum()) * 2 * width * es[case["dtype"]]
        return {"bytes": kv + 2 * rows * width * es[case["dtype"]], "flops": 4 * seen * width}
    # accept: parents, tokens and picks read, the path written; each moved row read and written
    moved = _accept_host(case)[2]
    return {"bytes": rows * 16 + 2 * moved * case["layers"] * 2 * width * es[case["dtype"]],
            "flops": 0}


# ------------------------------------------------------------------ inputs

def _drafts(case):
    """Drafted and picked tokens (host): most rows have a child that the model
    agrees with, so that paths of several tokens are accepted."""
    lens, new, start, within, parent = _shape(case)
    r = np.random.RandomState(case["shape"] + 1)
    rows = int(start[-1])
    tokens, picked = r.randint(0, VOCAB, rows), r.randint(0, VOCAB, rows)
    base = np.repeat(start[:-1], new)
    for i in np.nonzero((r.rand(rows) < 0.75) & (parent >= 0))[0]:
        picked[base[i] + parent[i]] = tokens[i]
    return tokens, picked


def _accept_host(case):
    """(path of each request, row after row; accepted rows; moved rows), walked on the host."""
    lens, new, start, within, parent = _shape(case)
    tokens, picked = _drafts(case)
    paths, moved = [], 0
    for s in range(len(new)):
        a, b = start[s], start[s + 1]
        path = [0] if b > a else []
        while path:
            cur = path[-1]
            nxt = [c for c in range(cur + 1, b - a)
                   if parent[a + c] == cur and tokens[a + c] == picked[a + cur]]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path)
        moved += sum(p != j for j, p in enumerate(path))
    return paths, sum(len(p) for p in paths), moved


def prepare(case, seed):
    lens, new, start, within, parent = _shape(case)
    n, P, rows = case["seqs"], case["page"], int(start[-1])
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 31))
    dev = lambda a: torch.as_tensor(np.ascontiguousarray(a), device="cuda").to(torch.int32)  # noqa: E731
    need = -(-(lens + new) // P)
    held = -(-lens // P) if case["op"] == "plan" else need
    max_pages = int(need.max()) + 1
    n_pages = int(need.sum()) + 8
    order = r.permutation(n_pages)
    table = np.full((n, max_pages), -1, np.int64)
    table[np.arange(max_pages)[None] < held[:, None]] = order[:held.sum()]
    free = np.zeros(n_pages, np.int64)
    n_free = n_pages - int(held.sum())
    free[:n_free] = order[held.sum():]
    st = {"case": case, "page": P, "rows": rows, "nmax": int(new.max()), "lmax": int((lens + new).max()),
          "lens": dev(lens), "new": dev(new), "table": dev(table), "parent": dev(parent)}
    if case["op"] == "plan":
        max_rows = rows + 5  # the buffers of a captured step are a little larger than it needs
        st.update(zero=torch.zeros_like(st["new"]), held=dev(held), free=dev(free),
                  n_free=dev([n_free]), parent=dev(np.concatenate([parent, np.full(5, -1)])),
                  row_start=dev(np.zeros(n + 1)), row_pos=dev(np.zeros(max_rows)),
                  row_slot=dev(np.zeros(max_rows)), status=dev([0, 0]),
                  row_mask=dev(np.zeros((max_rows, MASK_WORDS))), back=dev(np.zeros(n + 1)),
                  back_pos=dev(np.zeros(max_rows)), back_slot=dev(np.zeros(max_rows)))
        return st
    pos = np.repeat(lens, new) + within
    slot = table[np.repeat(np.arange(n), new), pos // P] * P + pos % P
    dt = DTYPES[case["dtype"]]
    st["pool"] = torch.randn((n_pages, case["layers"], 2, case["heads"], P, HEAD), generator=g,
                             device="cuda", dtype=torch.float32 if case["dtype"] == "f32" else dt)
    st["layer"] = case["layers"] - 1
    st.update(row_start=dev(start), row_slot=dev(slot))
    width = case["heads"] * HEAD
    if case["op"] == "write":
        src = DTYPES[case["src"]]
        st["kv"] = torch.randn((rows, 2, width), generator=g, device="cuda").to(src)
    elif case["op"] == "attend":
        # the queries are the first third of the fused projection's rows
        st["q"] = torch.randn((rows, 3 * width), generator=g, device="cuda").to(dt)[:, :width]
        st["out"] = torch.empty((rows, width), device="cuda", dtype=dt)
        st["row_mask"] = (torch.as_tensor(_words(_ancestors(parent, start), MASK_WORDS),
                                          device="cuda") if case["tree"] else None)
    else:
        tokens, picked = _drafts(case)
        shift = r.randint(0, VOCAB)  # other tokens for each seed, the same agreement
        st.update(tokens=dev((tokens + shift) % VOCAB), picked=dev((picked + shift) % VOCAB),
                  accepted=dev(np.zeros(n)), path=dev(np.zeros(rows)), next=dev(np.zeros(n)))
    return st


# ------------------------------------------------------------------ plain forms

def _row_seq(row_start, n_rows, n_seqs):
    """The request of each row; rows past the last request give the last one."""
    r = torch.arange(n_rows, device=row_start.device)
    return torch.searchsorted(row_start[1:].contiguous(), r, right=True).clamp(max=n_seqs - 1), r


def _plain_plan(lens, new, table, held, free, n_free, page, max_rows, parent):
    """Updates table, held, free and n_free; returns row starts, positions, slots and masks."""
    n, max_pages = table.shape
    need = (lens + new + page - 1) // page
    col = torch.arange(max_pages, device=table.device)
    gone = (col >= need[:, None]) & (col < held[:, None])
    more = (col >= held[:, None]) & (col < need[:, None])
    # given back: the first of them ends on top of the stack
    ext = torch.cat([free, free[:1]])  # one place more, for what goes nowhere
    n_gone = gone.sum()
    at = torch.where(gone.view(-1), n_free + n_gone - gone.view(-1).cumsum(0), len(free))
    ext.scatter_(0, at, table.view(-1))
    top = n_free + n_gone
    # taken: from the top of the stack down
    at = torch.where(more.view(-1), top - more.view(-1).cumsum(0), len(free))
    new_table = torch.where(more, ext[at].view(n, max_pages), torch.where(gone, -1, table))
    table.copy_(new_table)
    free.copy_(ext[:-1])
    n_free.copy_(top - more.sum())
    held.copy_(need)
    row_start = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0).to(torch.int32)])
    seq, r = _row_seq(row_start, max_rows, n)
    live = r < row_start[-1]
    within = r - row_start[seq]
    at = torch.where(live, lens[seq] + within, 0)
    page_of = table[seq, (at // page).clamp(max=max_pages - 1)]
    slot = torch.where(live, page_of * page + at % page, -1).to(torch.int32)
    if parent is None:
        return row_start, torch.where(live, at, -1).to(torch.int32), slot, None
    # ancestors: each row joins its own bits to those of the row that it points to, and then
    # points twice as far
    width = MASK_WORDS * 32
    bit = torch.arange(width, device=table.device)
    m = torch.zeros((max_rows + 1, width), dtype=torch.bool, device=table.device)
    m[:-1] = (within[:, None] == bit) & live[:, None]
    up = torch.full((max_rows + 1,), max_rows, device=table.device)
    up[:-1] = torch.where(live & (parent >= 0), row_start[seq] + parent, max_rows)
    for _ in range(6):  # 2^6 = 64 rows are the longest way up
        m = m | m[up]
        up = up[up]
    m = m[:-1]
    depth = m.sum(1) - 1
    words = (m.view(-1, MASK_WORDS, 32).long() << bit[:32]).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return row_start, torch.where(live, lens[seq] + depth, -1).to(torch.int32), slot, words


def _plan_plain(s):
    parent = s["parent"] if s["case"]["tree"] else None
    a = _plain_plan(s["lens"], s["new"], s["table"], s["held"], s["free"], s["n_free"], s["page"],
                    len(s["row_pos"]), parent)
    b = _plain_plan(s["lens"], s["zero"], s["table"], s["held"], s["free"], s["n_free"],
                    s["page"], len(s["row_pos"]), None)
    return a, b[:3], torch.zeros_like(s["status"])


def _write_plain(s):
    pool, page, slot = s["pool"], s["page"], s["row_slot"].long()
    kv = s["kv"].float().to(pool.dtype).view(s["rows"], 2, s["case"]["heads"], HEAD)
    pool[slot // page, s["layer"], :, :, slot % page] = kv
    return pool


def _attend_plain(s):
    c, pool, page = s["case"], s["pool"], s["page"]
    n, N, L, H = c["seqs"], s["nmax"], s["lmax"], c["heads"]
    lens, start = s["lens"].long(), s["row_start"].long()
    seq, r = _row_seq(start, s["rows"], n)
    within = r - start[seq]
    at = torch.arange(L, device=pool.device)
    valid = at < (lens + s["new"])[:, None]                       # [seqs][keys]
    where = torch.where(valid, s["table"][:, at // page], 0).long()
    k = pool[where, s["layer"], 0, :, at % page].float()          # [seqs][keys][heads][64]
    v = torch.where(valid[..., None, None], pool[where, s["layer"], 1, :, at % page].float(), 0.)
    q = torch.zeros((n, N, H, HEAD), device=pool.device)
    q[seq, within] = s["q"].float().reshape(-1, H, HEAD)
    score = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * 0.125  # [seqs][heads][rows][keys]
    off = at - lens[:, None]                                      # the draft at each key
    own_row = torch.arange(N, device=pool.device)[:, None]
    if s["row_mask"] is None:
        draft = off[:, None, :] <= own_row
    else:
        bits = torch.zeros((n, N, MASK_WORDS), dtype=torch.int64, device=pool.device)
        bits[seq, within] = s["row_mask"].long()
        word = (off // 32).clamp(0, MASK_WORDS - 1)
        draft = (torch.gather(bits, 2, word[:, None, :].expand(n, N, L)) >> (off % 32)[:, None, :]) & 1 > 0
    seen = valid[:, None, :] & ((off < 0)[:, None, :] | draft)    # [seqs][rows][keys]
    score = torch.where(seen[:, None], score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0., top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.transpose(1, 2)) / torch.where(total == 0, 1., total)
    s["out"].copy_(o.transpose(1, 2)[seq, within].reshape(s["rows"], H * HEAD))
    return s["out"]


def _accept_plain(s):
    pool, page, start = s["pool"], s["page"], s["row_start"].long()
    n, rows = s["case"]["seqs"], s["rows"]
    seq, r = _row_seq(start, rows, n)
    base, parent = start[seq], s["parent"].long()
    above = torch.where(parent >= 0, base + parent, r)            # a root points to itself
    fits = (parent >= 0) & (s["tokens"] == s["picked"][above])
    # of a row's children that fit, the first counts
    first = torch.full((rows,), rows, device=r.device).scatter_reduce(
        0, above, torch.where(fits, r, rows), "amin")
    ok = (fits & (first[above] == r)) | (r == base)
    up = above
    for _ in range(6):  # 2^6 = 64 rows are the longest way up
        ok = ok & ok[up]
        up = up[up]
    rank = ok.cumsum(0) - 1
    rank = rank - rank[base]
    accepted = torch.zeros(n, dtype=torch.int64, device=r.device).scatter_add(0, seq, ok.long())
    last = torch.full((n,), -1, device=r.device).scatter_reduce(0, seq, torch.where(ok, r, -1), "amax")
    nxt = torch.where(last >= 0, s["picked"][last.clamp(min=0)], -1)
    # rows that are not accepted move the root onto itself, which changes nothing
    path = torch.full((rows,), -1, device=r.device)
    path.scatter_(0, torch.where(ok, base + rank, base), torch.where(ok, r - base, 0))
    slot = s["row_slot"].long()
    src, dst = slot[torch.where(ok, r, base)], slot[torch.where(ok, base + rank, base)]
    pool[dst // page, :, :, :, dst % page] = pool[src // page, :, :, :, src % page]
    s["lens"].add_(accepted.to(torch.int32))
    return [accepted.to(torch.int32), path.to(torch.int32), nxt.to(torch.int32), s["lens"], pool]


# ------------------------------------------------------------------ one pass

def run(s):
    op = s["case"]["op"]
    if not own:
        if op == "plan":
            # a draft step's plan, and the plan that gives its pages back
            a, b, status = _plan_plain(s)
            return {"first": [x for x in a if x is not None], "back": list(b), "table": s["table"],
                    "held": s["held"], "free": s["free"], "n_free": s["n_free"], "status": status}
        if op == "write":
            return _write_plain(s)
        return _attend_plain(s) if op == "attend" else _accept_plain(s)
    W = _wattn()
    if op == "plan":
        tree = s["case"]["tree"]
        W.paged_plan(s["lens"], s["new"], s["table"], s["held"], s["free"], s["n_free"],
                     s["row_start"], s["row_pos"], s["row_slot"], s["status"][:1],
                     page_rows=s["page"], parents=s["parent"] if tree else None,
                     row_mask=s["row_mask"] if tree else None)
        W.paged_plan(s["lens"], s["zero"], s["table"], s["held"], s["free"], s["n_free"],
                     s["back"], s["back_pos"], s["back_slot"], s["status"][1:],
                     page_rows=s["page"])
        first = [s["row_start"], s["row_pos"], s["row_slot"]] + ([s["row_mask"]] if tree else [])
        return {"first": first, "back": [s["back"], s["back_pos"], s["back_slot"]],
                "table": s["table"], "held": s["held"], "free": s["free"], "n_free": s["n_free"],
                "status": s["status"]}
    if op == "write":
        W.paged_write(s["pool"], s["layer"], s["row_slot"], s["kv"][:, 0], s["kv"][:, 1])
        return s["pool"]
    if op == "attend":
        W.paged_attend(s["pool"], s["layer"], s["table"], s["lens"], s["row_start"], s["q"],
                       s["out"], row_mask=s["row_mask"])
        return s["out"]
    W.paged_accept(s["pool"], s["row_start"], s["row_slot"], s["tokens"], s["picked"], s["lens"],
                   s["accepted"], s["path"], s["next"], parents=s["parent"])
    return [s["accepted"], s["path"], s["next"], s["lens"], s["pool"]]


def exact(case, seed):
    """The attention from its definition in 64 bits, request by request; the
    other operators give whole numbers or move values as they are."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
    lens, new, start, within, parent = _shape(case)
    seen_by = torch.as_tensor(_ancestors(parent, start), device="cuda")
    out = torch.zeros((s["rows"], case["heads"] * HEAD), dtype=torch.float64, device="cuda")
    table = s["table"].cpu().numpy()
    for i in range(case["seqs"]):
        a, b, ln = int(start[i]), int(start[i + 1]), int(lens[i])
        if a == b:
            continue
        at = np.arange(ln + b - a)
        rows = torch.as_tensor(table[i][at // case["page"]].astype(np.int64), device="cuda")
        off = torch.as_tensor(at % case["page"], device="cuda")
        kv = s["pool"][:, s["layer"]][rows, :, :, off].double()   # [keys][2][heads][64]
        q = s["q"][a:b].double().reshape(b - a, case["heads"], HEAD)
        z = torch.einsum("nhd,khd->hnk", q, kv[:, 0]) / 8
        z[:, :, ln:].masked_fill_(~seen_by[a:b, :b - a], -torch.inf)
        w = torch.softmax(z, -1)
        out[a:b] = torch.einsum("hnk,khd->nhd", w, kv[:, 1]).reshape(b - a, -1)
    return out
