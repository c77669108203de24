"""The device-planned paged cache where its attention can go wrong quietly:
values that are not finite, long flat tails, lengths near 2^31, row buffers
larger than the step, and what the device status word says of whom."""
import numpy as np
import pytest

from tests.test_gpu_paged import WIDE, Batch, W, bound, clean_status, cu, tdt, tree  # noqa: F401

pytestmark = pytest.mark.gpu


def seen_by(b, s):
    """[new rows][new rows] truth values: which drafts of request s each of its rows sees."""
    a, n = int(b.start[s]), int(b.new[s])
    if b.parents is None:
        return np.tril(np.ones((n, n), bool))
    bits = np.unpackbits(np.ascontiguousarray(b.mask[a:a + n]).view(np.uint8), axis=1, bitorder="little")
    return bits[:, :n].astype(bool)


def formula(b, layer, scale=0.125):
    """(o, sum of the weights times |v|, bound on the scores' magnitudes), the
    attention's definition in float64 on the device."""
    import torch
    rows, w = int(b.start[-1]), b.heads * 64
    out = np.zeros((3, rows, w))
    for s in range(len(b.lens)):
        a, n, ln = int(b.start[s]), int(b.new[s]), int(b.lens[s])
        if n == 0:
            continue
        at = np.arange(ln + n)
        pages = torch.as_tensor(b.st.table[s, at // b.P].astype(np.int64), device="cuda")
        kv = b.pool[:, layer][pages, :, :, torch.as_tensor(at % b.P, device="cuda")].double()
        q = b.q[a:a + n].double().view(n, b.heads, 64)
        seen = torch.ones(n, ln + n, dtype=torch.bool, device="cuda")
        seen[:, ln:] = torch.as_tensor(seen_by(b, s), device="cuda")
        z = torch.einsum("nhd,khd->hnk", q, kv[:, 0]) * scale
        z = z.masked_fill(~seen, -torch.inf)
        p = torch.softmax(z, -1).masked_fill(~seen.any(-1)[:, None], 0)
        big = torch.einsum("nhd,khd->hnk", q.abs(), kv[:, 0].abs()).masked_fill(~seen, 0) * scale
        for i, x in enumerate((torch.einsum("hnk,khd->nhd", p, kv[:, 1]),
                               torch.einsum("hnk,khd->nhd", p, kv[:, 1].abs()),
                               big.amax(-1).T[:, :, None].expand(n, b.heads, 64))):
            out[i, a:a + n] = x.reshape(n, w).cpu().numpy()
    return out


def units(lens, new, heads, words):
    """(units of the narrow, of the wide kernel) that a step of f16 counts for;
    words: mask words, 0 without masks."""
    total = [0, 0]
    for k, (keys, rows, stage, item) in enumerate(((32, 32, 5, 12), (128, 128, 2, 3))):
        for ln, n in zip(lens, new):
            for first in range(0, n, rows):
                end = ln + min(n, 32 * words if words else first + rows)
                total[k] += -(-end // keys) * (4 if k == 0 and n - first <= 16 else stage) + item
    return total[0] * heads, total[1] * heads


def wide(seed, lens, new, heads, page_rows, kind="tree", dead=0.0, **kw):
    """A step that the kernel for many rows takes, as the numbers of its work say."""
    rng = np.random.default_rng(seed)
    par = sum((tree(rng, k, dead) for k in new), []) if kind == "tree" else None
    words = -(-max(new) // 32)
    kw = {"layers": 1, **kw}
    b = Batch(seed, "f16", lens, new, heads, page_rows, par, words=words, **kw)
    narrow, many = units(lens, new, heads, words if par else 0)
    assert narrow > 33 * many and narrow >= 150 * 148 * 8 and b.max_rows // len(lens) > 96
    return b


def place(b, s, at):
    """Index of position `at` of request s in the pool's first and fifth dimension."""
    return int(b.st.table[s, at // b.P]), at % b.P


# ------------------------------------------------------------------ values and keys that are not finite

@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_wide_value_that_is_not_finite_where_the_maximum_grows(W, value):
    """Tiles in which the running maximum grows by more than 2^8 and a draft's
    value is not finite: the sums so far are rescaled once, in all dimensions
    but the value's own."""
    b = wide(66, [15000], [128], 20, 64)
    b.q += 1
    # scores of about 32 in the tile of the first drafts, of about 64 in the next
    # (every row sees that draft)
    jumps = [(14999, 4.0), (15110, 8.0)]
    for at, k in jumps:
        page, row = place(b, 0, at)
        b.pool[page, 0, 0, :, row] = k
    b.mask[:128, 3] |= np.int32(1 << 14)
    o, mag, top = formula(b, 0)
    sees = seen_by(b, 0)
    hit = sees[:, 4] | sees[:, 108]
    assert hit.any() and not hit.all()
    for at in (15004, 15108):
        page, row = place(b, 0, at)
        b.pool[page, 0, 1, :, row, 37] = value
    got = b.attend(W, 0, "f32")
    want = got[hit, 37::64]
    assert np.isnan(want).all() if value != value else (want == value).all()
    got[hit, 37::64] = o[hit, 37::64]
    lim = bound("f16", "f32", o, mag, top, 15128, 6.0) + WIDE * mag
    assert (np.abs(got - o) <= lim).all()


@pytest.mark.parametrize("dtype,many", [("f16", True), ("f16", False), ("bf16", False), ("f32", False)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_key_that_is_not_finite_is_seen(W, dtype, many, bad):
    """One element of one draft's key, at each of nine neighbouring positions: a
    row that sees it has a score that is NaN or +inf there and is NaN, or one
    of -inf and does without that key; the others are as they were."""
    lens, new = ([15000], [128]) if many else ([70], [40])
    b = wide(67, lens, new, 20, 64) if many else Batch(
        67, dtype, lens, new, 2, 64, [-1] + [max(0, i - 2) for i in range(1, new[0])], layers=1)
    clean, mask = b.attend(W, 0, "f32"), b.mask.copy()
    n_lost = n_without = 0
    for j in range(3, 12):
        page, row = place(b, 0, lens[0] + j)
        keep = b.pool[page, 0, 0, 1, row, 5].clone()
        b.pool[page, 0, 0, 1, row, 5] = bad
        got = b.attend(W, 0, "f32")
        sees = seen_by(b, 0)[:, j]
        positive = (b.q[:new[0], 64 + 5] > 0).cpu().numpy()
        lost = sees if bad != bad else sees & positive
        n_lost += lost.sum()
        assert not sees.all()
        assert np.isnan(got[lost, 64:128]).all(), j
        same = ~sees
        assert np.array_equal(got[same], clean[same])
        assert np.array_equal(got[:, :64], clean[:, :64]) and np.array_equal(got[:, 128:], clean[:, 128:])
        if bad == bad:  # without that key
            without = sees & ~positive
            b.pool[page, 0, 0, 1, row, 5] = keep
            b.mask[:new[0], 0] &= ~np.int32(1 << j)
            o, mag, top = formula(b, 0)
            b.mask = mask.copy()
            lim = bound(dtype, "f32", o, mag, top, 1200, 6.0) + (WIDE if many else 0) * mag
            n_without += without.sum()
            assert (np.abs(got - o) <= lim)[without, 64:128].all()
        b.pool[page, 0, 0, 1, row, 5] = keep
    assert n_lost > 0 and (n_without > 0 or bad != bad)


# ------------------------------------------------------------------ what 16-bit weights keep

TAIL_KEYS = 131072


@pytest.mark.parametrize("rows", [1, 12, 20, 128])
def test_a_flat_tail_keeps_its_weight(W, rows):
    """One key that outweighs each of 131072 others 2^25.5 times, whose values
    are small where theirs are not: theirs are the output. (Requests of the
    same pages, as many as give each share of the work a whole request's keys.)

    Weights in f16 relative to 2^-7 of the largest: 2^-18.5 in steps of 2^-24,
    off by 2^-6.5 of themselves at most and all alike; the sums of 131072 of
    them on the tensor cores, which cut off, by 8192 * 2^-23."""
    import torch
    heads, page_rows, n = 8, 128, 40 if rows > 64 else 160
    pages = TAIL_KEYS // page_rows + 1
    pool = torch.zeros(pages, 1, 2, heads, page_rows, 64, dtype=torch.float16, device="cuda")
    c = (0.5 + torch.arange(64, device="cuda") / 64).half()
    pool[:, :, 1] = c
    sink = 25.5 * float(np.log(2.0))
    pool[0, 0, 0, :, 0, 0] = sink
    pool[0, 0, 1, :, 0] = 0
    q = torch.zeros(n * rows, heads, 64, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 8
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(n, pages).contiguous()
    o = torch.empty(n * rows, heads * 64, device="cuda")
    W.paged_attend(pool, 0, table, cu(np.full(n, TAIL_KEYS)), cu(np.arange(n + 1) * rows),
                   q.view(n * rows, heads * 64), o)
    r = float(np.exp(-float(pool[0, 0, 0, 0, 0, 0])))
    tail = torch.arange(TAIL_KEYS, TAIL_KEYS + rows, device="cuda").double().repeat(n)[:, None, None] * r
    want = (tail / (1 + tail) * c.double()).expand(n * rows, heads, 64).reshape(n * rows, -1)
    assert 2e-3 < float(want.max()) < 6e-3
    err = (o.double() - want).abs()
    assert float((err / want).max()) <= 2.0 ** -6.5 + 2.0 ** -10 + 2 * 7.5e-5 + 2.0 ** -16


@pytest.mark.parametrize("lens,new", [([5], [1]), ([448, 17, 300], [8, 1, 3]), ([40] * 30, [2] * 30),
                                      ([9000], [5])])
def test_up_to_8_rows_carry_the_weights_residuals(W, lens, new):
    """f16 pools, f32 outputs, at most 8 rows to a request: the weights are two
    f16 numbers and 22 bits, of which those below 2^-25 in the unit of 2^7
    above the largest are lost."""
    b = Batch(68, "f16", lens, new, 6, 64)
    o, mag, top = formula(b, 1)
    got = b.attend(W, 1, "f32")
    keys = int((b.lens + b.new).max())
    lim = (2 * 64 * 2.0 ** -24 * top + 2.0 ** -22 + 2.0 ** -18) * mag + keys * 2.0 ** -32 * 6 + 1e-7
    assert (np.abs(got - o) <= lim + 2.0 ** -24 * np.abs(o)).all()


# ------------------------------------------------------------------ sizes

@pytest.mark.parametrize("dtype,rows", [("f16", 130), ("f16", 3), ("bf16", 130), ("f32", 3)])
def test_lengths_near_2_31(W, dtype, rows):
    """A table of 2^31 positions and a length close to them: out of range, and
    the other request's rows are written."""
    import torch
    P_, heads, ln = 4096, 2, 600
    g = torch.Generator(device="cuda").manual_seed(69)
    pool = torch.randn(2, 1, 2, heads, P_, 64, generator=g, device="cuda").to(tdt(dtype))
    table = torch.zeros(2, (1 << 31) // P_, dtype=torch.int32, device="cuda")
    table[0, 0] = 1
    q = torch.randn(2 * rows, heads * 64, generator=g, device="cuda").to(tdt(dtype))
    o = torch.full((2 * rows, heads * 64), 7.0, device="cuda")
    W.paged_attend(pool, 0, table, cu(np.array([ln, 2 ** 31 - 1 - 64 - rows])),
                   cu(np.array([0, rows, 2 * rows])), q, o)
    torch.cuda.synchronize()
    assert W.device_status() == -6
    assert (o[rows:] == 7).all()
    kv = pool[1, 0, :, :, :ln + rows].double()
    z = torch.einsum("nhd,hkd->hnk", q[:rows].double().view(rows, heads, 64), kv[0]) / 8
    z.masked_fill_(torch.arange(ln + rows, device="cuda") > ln + torch.arange(rows, device="cuda")[:, None],
                   -torch.inf)
    ref = torch.einsum("hnk,hkd->nhd", torch.softmax(z, -1), kv[1]).reshape(rows, -1)
    assert float((o[:rows] - ref).abs().max()) <= (1e-5 if dtype == "f32" else 2e-3)


@pytest.mark.parametrize("n,heads", [(4, 6), (64, 20)])
def test_row_buffers_larger_than_the_step(W, n, heads):
    """Single rows in a buffer for 120 rows a request (a graph captured once
    for steps of every length) are computed as in a buffer of their own."""
    import torch
    lens = ([1000, 300, 700, 80] * n)[:n]
    b = Batch(70, "f16", lens, [1] * n, heads, 64, spare_rows=n * 119)
    table, seq, start, _ = b.device()
    small = torch.zeros(n, heads * 64, device="cuda")
    large = torch.zeros(b.max_rows, heads * 64, device="cuda")
    W.paged_attend(b.pool, 1, table, seq, start, b.q[:n], small)
    W.paged_attend(b.pool, 1, table, seq, start, b.q, large)
    assert torch.equal(small, large[:n])
    assert (large[n:] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masks_narrower_than_the_step(W, dtype):
    """Mask words for fewer drafts than the request has rows: those behind are seen by none."""
    import torch
    b = Batch(72, dtype, [40, 0, 5], [70, 33, 3], 3, 32, sum((tree(np.random.default_rng(72), k) for k in (70, 33, 3)), []),
              words=3, layers=1)
    b.mask[:, 1:] = 0
    table, seq, start, _ = b.device()
    o = torch.zeros(b.max_rows, 192, device="cuda")
    W.paged_attend(b.pool, 0, table, seq, start, b.q, o, row_mask=cu(b.mask[:, :1]))
    ref, mag, top = formula(b, 0)
    assert (np.abs(o[:106].cpu().numpy() - ref) <= bound(dtype, "f32", ref, mag, top, 110, 6.0)).all()


# ------------------------------------------------------------------ steps that the wide kernel takes

WIDE_STEPS = [
    # lens, new, heads, page_rows
    ([15000], [128], 20, 64), ([9000, 0, 33, 1000], [256, 1, 2, 127], 20, 128),
    ([2500] * 8, [120] * 8, 16, 48), ([4000], [1000], 16, 16), ([7000, 1, 6501, 513], [124, 0, 253, 113], 20, 80),
    ([0, 0], [2040, 2048], 20, 32),
]


@pytest.mark.parametrize("step", range(len(WIDE_STEPS)))
@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_wide_steps(W, step, kind, out):
    """Rows that fill tiles of 128 nearly, next to requests that do not."""
    b = wide(80 + step, *WIDE_STEPS[step], kind, dead=0.02, stride=8 * step)
    got = b.attend(W, 0, out, stride=8 * step)
    o, mag, top = formula(b, 0)
    lim = bound("f16", out, o, mag, top, int((b.lens + b.new).max()), 6.0) + WIDE * mag
    assert (np.abs(got - o) <= lim).all()
    assert np.array_equal(got, b.attend(W, 0, out, stride=8 * step))


def test_the_work_decides_which_kernel(W):
    """The same request alone, and beside so many that rest that the buffers
    cannot be full: other sums, to their rounding the same."""
    import torch
    b = wide(90, [15000], [128], 20, 64, "chain")
    alone = b.attend(W, 0, "f32")
    table, _, _, _ = b.device()
    o = torch.zeros(b.max_rows, 1280, device="cuda")
    W.paged_attend(b.pool, 0, table.expand(9, -1).contiguous(), cu(np.array([15000] + [0] * 8)),
                   cu(np.array([0] + [128] * 9)), b.q, o)
    o = o[:128].cpu().numpy()
    assert not np.array_equal(o, alone)
    ref, mag, top = formula(b, 0)
    assert (np.abs(o - ref) <= bound("f16", "f32", ref, mag, top, 15128, 6.0)).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), "lowest"])
def test_wide_steps_masked_places_have_no_influence(W, bad):
    """Drafts that hold NaN, infinities or the lowest value reach only the rows that see them."""
    import torch
    bad = torch.finfo(torch.float16).min if bad == "lowest" else bad
    b = wide(91, [9000, 0, 33, 1000], [256, 1, 2, 127], 20, 128)
    clean = b.attend(W, 0, "f32")
    hit = np.zeros(int(b.start[-1]), bool)
    for s, j in [(0, 5), (0, 250), (3, 60), (2, 1)]:
        page, row = place(b, s, int(b.lens[s]) + j)
        b.pool[page, :, :, :, row] = bad
        a = int(b.start[s])
        hit[a:a + b.new[s]] |= seen_by(b, s)[:, j]
    got = b.attend(W, 0, "f32")
    assert hit.any() and not hit.all()
    assert np.array_equal(got[~hit], clean[~hit])
    if not np.isfinite(bad):
        assert np.isnan(got[hit]).any(axis=1).all()


def test_wide_steps_rows_that_see_nothing_are_zero(W):
    b = wide(92, [9000, 0], [256, 120], 20, 128)
    b.mask[[256, 300, 375]] = 0        # rows of the request without context
    b.mask[40] = 0                     # this one still sees its context
    got = b.attend(W, 0, "f32")
    o, mag, top = formula(b, 0)
    assert (got[[256, 300, 375]] == 0).all() and (got[40] != 0).any()
    assert (np.abs(got - o) <= bound("f16", "f32", o, mag, top, 9256, 6.0) + WIDE * mag).all()


def either_kernel():
    """A step for the wide kernel, and one of single rows in buffers for many."""
    many = wide(93, [9000, 0, 33, 1000], [256, 1, 2, 127], 20, 128)
    single = Batch(94, "f16", [1000, 300, 700, 80] * 16, [1] * 64, 20, 64, spare_rows=64 * 119, layers=1)
    return many, single


def test_either_kernel_repeats_beside_another(W):
    """The same calls 100 times while attention of its own runs on another stream."""
    import torch
    x = torch.randn(4 * 700 * 384, device="cuda").half()
    y = torch.empty_like(x)
    ws = torch.zeros(W.paged_attend_workspace_bytes(1, 1, 1), dtype=torch.uint8, device="cuda")
    work = []
    for b in either_kernel():
        a = dict(zip(("block_table", "seq_lens", "row_start", "row_mask"), b.device()))
        want = torch.zeros(b.max_rows, b.heads * 64, device="cuda")
        W.paged_attend(b.pool, 0, q=b.q, o=want, **a)
        work.append((b, a, want, torch.empty_like(want)))
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    side, main = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(100):
        W.attention_fwd(x, x, x, y, batch=4, t_q=700, t_kv=700, n_heads=6, scale=0.125, stream=side)
        with torch.cuda.stream(main):
            for b, a, want, o in work:
                o.zero_()
                W.paged_attend(b.pool, 0, q=b.q, o=o, workspace=ws, **a)
                differ += (o != want).any()
    torch.cuda.synchronize()
    assert int(differ) == 0
    assert (ws[:65536 * 4] == 0).all()


def test_either_kernel_from_one_graph(W):
    """A graph captured once, without a workspace, replayed with lengths for
    the one kernel and for the other, on two streams at once."""
    import torch
    long = Batch(95, "f16", [9000, 1000], [256, 127], 20, 64, layers=1)
    single, n = either_kernel()[1], 64
    rows, pages = single.max_rows, long.st.table.shape[1]
    narrow, many = units(long.lens, long.new, 20, 0)
    assert narrow > 33 * many and narrow >= 150 * 148 * 8 and rows // n > 96
    graphs = []
    for _ in range(2):
        g = dict(pool=torch.zeros(max(long.n_pages, single.n_pages), 1, 2, 20, 64, 64,
                                  dtype=torch.float16, device="cuda"),
                 block_table=torch.zeros(n, pages, dtype=torch.int32, device="cuda"),
                 seq_lens=torch.zeros(n, dtype=torch.int32, device="cuda"),
                 row_start=torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
                 q=torch.zeros(rows, 1280, dtype=torch.float16, device="cuda"),
                 o=torch.zeros(rows, 1280, device="cuda"))
        s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            W.paged_attend(layer=0, **g)
        graphs.append((g, s, graph))
    for steps in ((long, single), (single, long), (long, long)):
        for (g, s, graph), b in zip(graphs, steps):
            k = len(b.lens)
            g["pool"][:b.n_pages] = b.pool
            g["block_table"][:k, :b.st.table.shape[1]] = cu(b.st.table)
            g["seq_lens"][:k] = cu(b.lens)
            g["row_start"][:k + 1] = cu(b.start)
            g["row_start"][k + 1:] = int(b.start[-1])
            g["q"][:b.max_rows] = b.q
            g["o"].fill_(7)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s, graph in graphs:
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (g, s, graph), b in zip(graphs, steps):
            end = int(b.start[-1])
            o, mag, top = formula(b, 0)
            lim = bound("f16", "f32", o, mag, top, 9300, 6.0) + WIDE * mag
            assert (np.abs(g["o"][:end].cpu().numpy() - o) <= lim).all()
            assert (g["o"][end:] == 7).all()


# ------------------------------------------------------------------ the status word

def bad_length(W):
    b = Batch(71, "f16", [100, 40], [3, 2], 2, 16)
    b.lens[1] = 2 ** 31 - 1
    b.attend(W, 1, "f32")


def test_a_range_report_is_its_callers_alone(W, oracle):
    """A length out of range in a paged call, then a call of host buffers:
    that one succeeds, and the report is still there for who asks."""
    bad_length(W)
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal(100 * 128).astype(np.float32) for _ in range(3))
    out = np.empty_like(q)
    W.flash_attention_2(q, k, v, 100, 100, 2, 128, False, out)
    assert np.abs(out - oracle.flash_attention_2(q, k, v, 100, 100, 2, 128, False)).max() <= 1e-5
    assert W.device_status() == -6 and W.device_status() == 0


def test_a_range_report_does_not_hide_a_timeout(W):
    bad_length(W)
    assert W.selftest_bounded_wait(2000) == -4   # a flag that nothing sets: 2 ms
    assert W.device_status() == -6 and W.device_status() == 0
