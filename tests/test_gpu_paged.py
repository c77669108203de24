"""The device-planned paged cache on the GPU against its host model: whole
numbers and moved values exactly, the attention against float64."""
import numpy as np
import pytest

from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

DT = {"f32": 0, "f16": 1, "bf16": 2}


@pytest.fixture(scope="module")
def W():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import wattn
    return wattn


@pytest.fixture(autouse=True)
def clean_status(W):
    yield
    assert W.device_status() == 0


def cu(a):
    import torch
    return torch.as_tensor(np.ascontiguousarray(a), device="cuda").to(torch.int32)


def tdt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def tree(rng, n, dead=0.0):
    """Parents of n rows: a root first, further roots and dead rows here and there."""
    par = [int(rng.integers(max(-1, i - 5), i)) if i else -1 for i in range(n)]
    for i in range(1, n):
        if rng.random() < dead:
            par[i] = int(rng.choice([i, i + 1, -2, 1000]))
    return par


# ------------------------------------------------------------------ plan

class Plan:
    """The device arrays of a plan next to the host model's."""

    def __init__(self, W, rng, n_seqs, n_pages, max_pages, max_rows, page_rows, words=0, stride=0):
        import torch
        self.W, self.page_rows, self.max_rows, self.words = W, page_rows, max_rows, words
        self.st = P.PlanState(n_seqs, n_pages, max_pages, rng.permutation(n_pages))
        wide = torch.full((n_seqs, max_pages + stride), -7, dtype=torch.int32, device="cuda")
        self.wide, self.table = wide, wide[:, :max_pages]
        self.table.copy_(cu(self.st.table))
        self.held, self.free, self.n_free = cu(self.st.held), cu(self.st.free), cu([n_pages])
        junk = lambda *s: torch.full(s, 99, dtype=torch.int32, device="cuda")  # noqa: E731
        self.start, self.pos, self.slot = junk(n_seqs + 1), junk(max_rows), junk(max_rows)
        self.mask, self.status = junk(max_rows, max(1, words)), junk(1)

    def step(self, lens, new, parents=None):
        """One plan on both sides, compared whole; the model's (status, start, pos, slot, mask)."""
        par = None
        if parents is not None:
            par = np.full(self.max_rows, -5)
            par[:len(parents)] = parents
        self.W.paged_plan(cu(lens), cu(new), self.table, self.held, self.free, self.n_free,
                          self.start, self.pos, self.slot, self.status, page_rows=self.page_rows,
                          parents=None if par is None else cu(par),
                          row_mask=None if par is None else self.mask)
        want = P.plan(self.st, lens, new, self.page_rows, self.max_rows, par,
                      self.words if par is not None else 0)
        assert self.status.item() == want[0]
        for got, exp, what in ((self.start, want[1], "row_start"), (self.pos, want[2], "row_pos"),
                               (self.slot, want[3], "row_slot"), (self.table, self.st.table, "table"),
                               (self.held, self.st.held, "held")):
            assert np.array_equal(got.cpu().numpy(), exp), what
        if par is not None:
            assert np.array_equal(self.mask.cpu().numpy(), want[4]), "row_mask"
        assert self.n_free.item() == self.st.n_free
        assert np.array_equal(self.free.cpu().numpy()[:self.st.n_free],
                              self.st.free[:self.st.n_free])
        assert (self.wide[:, self.st.table.shape[1]:] == -7).all()
        return want


@pytest.mark.parametrize("n_seqs,page_rows,words,stride", [
    (1, 64, 1, 0), (3, 16, 2, 5), (37, 48, 2, 0), (1023, 16, 1, 1), (1024, 64, 0, 0),
    (1025, 32, 2, 0), (2500, 16, 1, 3)])
def test_plan_history(W, n_seqs, page_rows, words, stride):
    """Steps of growing, shrinking, resting and finishing requests."""
    rng = np.random.default_rng(n_seqs + page_rows)
    most = 20 if n_seqs < 100 else 6
    max_pages = 8
    cap = max_pages * page_rows
    pl = Plan(W, rng, n_seqs, n_seqs * 5 + 8, max_pages, n_seqs * most, page_rows, words, stride)
    lens = rng.integers(0, 3 * page_rows, n_seqs)
    for step in range(6):
        new = rng.integers(0, most + 1, n_seqs)
        par = sum((tree(rng, int(k), 0.1) for k in new), []) if words else None
        status, *_ = pl.step(lens, new, par)
        assert status in (0, P.NOMEM)
        if status == 0:
            lens = np.minimum(lens + rng.integers(0, new + 1), cap - most)
        lens[rng.random(n_seqs) < 0.2] = 0
        lens = np.where(rng.random(n_seqs) < 0.2, rng.integers(0, 3 * page_rows, n_seqs), lens)
    pl.step(np.zeros(n_seqs, int), np.zeros(n_seqs, int), [] if words else None)
    assert pl.st.n_free == len(pl.st.free)  # every page came back


def test_plan_undo_restores_the_stack(W):
    rng = np.random.default_rng(3)
    pl = Plan(W, rng, 20, 300, 12, 400, 16)
    lens = rng.integers(0, 100, 20)
    pl.step(lens, np.zeros(20, int))
    table, free = pl.table.clone(), pl.free.clone()
    pl.step(lens, rng.integers(0, 20, 20))
    pl.step(lens, np.zeros(20, int))
    n = pl.st.n_free
    assert (pl.table == table).all() and (pl.free[:n] == free[:n]).all()


def test_plan_long_requests(W):
    """Many pages for one request, a deep chain as a tree, rows beyond one launch block."""
    rng = np.random.default_rng(4)
    pl = Plan(W, rng, 3, 9000, 4200, 5000, 16, words=64)
    n = 2000
    pl.step([65000, 0, 7], [n, 1, 2000], list(range(-1, n - 1)) + [-1] + tree(rng, 2000))
    pl.step([100, 0, 0], [1, 0, 0], [-1])


@pytest.mark.parametrize("lens,new,status", [
    ([0, -1, 0], [1, 1, 1], -1), ([0, 0, 0], [1, -1, 1], -1), ([64 * 5, 0, 0], [1, 1, 1], -6),
    ([0, 0, 0], [30, 30, 30], -6), ([0, 0, 0], [1, 33, 1], -6), ([320, 320, 1], [0, 0, 0], -5),
    ([2**31 - 1, 2**31 - 1, 2**31 - 1], [2**31 - 1] * 3, -6)])
def test_plan_refusals_change_nothing(W, lens, new, status):
    rng = np.random.default_rng(5)
    pl = Plan(W, rng, 3, 10, 5, 64, 64, words=1)
    pl.step([70, 1, 0], [3, 0, 20], sum((tree(rng, k) for k in (3, 0, 20)), []))
    assert pl.step(lens, new, tree(rng, 64))[0] == status
    pl.step([70, 1, 0], [3, 0, 20], sum((tree(rng, k) for k in (3, 0, 20)), []))


def test_plan_bad_counts(W):
    rng = np.random.default_rng(6)
    for what, value in (("held", 9), ("held", -1), ("n_free", 11), ("n_free", -1)):
        pl = Plan(W, rng, 2, 10, 5, 64, 64)
        if what == "held":
            pl.st.held[1] = value
            pl.held.copy_(cu(pl.st.held))
        else:
            pl.st.n_free = value
            pl.n_free.fill_(value)
        pl.W.paged_plan(cu([1, 2]), cu([3, 4]), pl.table, pl.held, pl.free, pl.n_free, pl.start,
                        pl.pos, pl.slot, pl.status, page_rows=64)
        assert pl.status.item() == -1 and (pl.start == 0).all() and (pl.slot == -1).all()


def test_plan_without_requests_or_rows(W):
    rng = np.random.default_rng(7)
    Plan(W, rng, 0, 4, 3, 5, 16).step([], [])
    Plan(W, rng, 2, 4, 3, 0, 16).step([3, 17], [0, 0])


# ------------------------------------------------------------------ write

@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dst", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,page_rows,pad", [(1, 16, 0), (5, 48, 3), (20, 64, 64)])
def test_write(W, src, dst, heads, page_rows, pad):
    import torch
    g = torch.Generator(device="cuda").manual_seed(heads)
    n_pages, layers, n, w = 7, 3, 41, heads * 64
    pool = torch.randn(n_pages, layers, 2, heads, page_rows, 64, generator=g, device="cuda").to(tdt(dst))
    want = pool.clone()
    slots = torch.randperm(n_pages * page_rows, generator=g, device="cuda")[:n].to(torch.int32)
    slots[::7] = -1
    slots[3] = n_pages * page_rows          # outside the pool: skipped
    k = torch.randn(n, w + pad, generator=g, device="cuda").to(tdt(src))[:, pad // 3:pad // 3 + w]
    v = torch.randn(n, w + pad, generator=g, device="cuda").to(tdt(src))[:, :w]
    ok = (slots >= 0) & (slots < n_pages * page_rows)
    at = slots[ok].long()
    want[at // page_rows, 1, 0, :, at % page_rows] = k[ok].float().to(tdt(dst)).view(-1, heads, 64)
    want[at // page_rows, 1, 1, :, at % page_rows] = v[ok].float().to(tdt(dst)).view(-1, heads, 64)
    W.paged_write(pool, 1, slots, k, v)
    assert torch.equal(pool, want)


# ------------------------------------------------------------------ attend

def bound(dtype, out, o, mag, top, keys, vmax):
    """How far an output may be from float64, by its roundings: the scores are
    sums of 64 products in f32 (64 roundings of 2^-24 relative to the sum of
    magnitudes; `d` moves a weight by a factor exp(d) and the normaliser by
    another), the weights enter the second product in f16 (2^-11, below
    2^-14 of the largest by 2^-25 each), in bf16 with their rounding's residual
    (2^-16), or in f32; its sum and the exponentials cost 2^-18 at most, and
    the store half a step."""
    d = 64 * 2.0 ** -24 * top
    w = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -16}[dtype]
    t = (2 * d + w + 2.0 ** -18) * mag + (keys * 2.0 ** -25 * vmax if dtype == "f16" else 0) + 1e-7
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[out]
    return t + half * (np.abs(o) + t) + (2.0 ** -25 if out == "f16" else 0)


class Batch:
    """Requests with pages in random places; everything in the pool that no
    request holds is NaN."""

    def __init__(self, seed, dtype, lens, new, heads, page_rows, parents=None, words=2, layers=2,
                 spare_rows=3, stride=0, order=None, n_pages=None):
        import torch
        self.rng = np.random.default_rng(seed)
        self.dtype, self.heads, self.layers, self.P = dtype, heads, layers, page_rows
        self.lens, self.new = np.array(lens), np.array(new)
        need = -(-(self.lens + self.new) // page_rows)
        self.n_pages = n_pages or int(need.sum()) + 2
        order = self.rng.permutation(self.n_pages) if order is None else order
        self.st = P.PlanState(len(lens), self.n_pages, int(need.max(initial=0)) + 1, order)
        self.max_rows = int(self.new.sum()) + spare_rows
        par = None if parents is None else np.concatenate([parents, np.full(spare_rows, -1)]).astype(int)
        status, self.start, _, self.slot, self.mask = P.plan(
            self.st, lens, new, page_rows, self.max_rows, par, words if parents is not None else 0)
        assert status == 0
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pool = torch.full((self.n_pages, layers, 2, heads, page_rows, 64), float("nan"),
                               dtype=tdt(dtype), device="cuda")
        for s in range(len(lens)):
            at = np.arange(self.lens[s] + self.new[s])
            if len(at):
                pg = torch.as_tensor(self.st.table[s, at // page_rows].astype(np.int64), device="cuda")
                ro = torch.as_tensor(at % page_rows, device="cuda")
                self.pool[pg, :, :, :, ro] = torch.randn(
                    (len(at), layers, 2, heads, 64), generator=g, device="cuda").to(tdt(dtype))
        w = heads * 64
        self.q_wide = torch.full((self.max_rows, w + stride), float("nan"), dtype=tdt(dtype), device="cuda")
        self.q = self.q_wide[:, :w]
        self.q.copy_(torch.randn((self.max_rows, w), generator=g, device="cuda"))
        self.parents = parents

    def device(self):
        return (cu(self.st.table), cu(self.lens), cu(self.start),
                None if self.parents is None else cu(self.mask))

    def attend(self, W, layer, out, stride=0, scale=0.125, workspace=None):
        import torch
        w = self.heads * 64
        wide = torch.full((self.max_rows, w + stride), 777.0, dtype=tdt(out), device="cuda")
        table, lens, start, mask = self.device()
        W.paged_attend(self.pool, layer, table, lens, start, self.q, wide[:, :w], row_mask=mask,
                       scale=scale, workspace=workspace)
        assert (wide[self.start[-1]:] == 777).all(), "padding rows"
        assert (wide[:, w:] == 777).all(), "columns behind the rows"
        return wide[:self.start[-1], :w].float().cpu().numpy().astype(np.float64)

    def check(self, W, layer=1, out=None, stride=0, scale=0.125, workspace=None, more=0.0):
        out = out or self.dtype
        got = self.attend(W, layer, out, stride, scale, workspace)
        rows = int(self.start[-1])
        o, mag, top = P.attend(self.pool.float().cpu().numpy(), layer, self.st.table, self.lens,
                               self.start, self.q.float().cpu().numpy()[:rows], self.heads, scale,
                               None if self.parents is None else self.mask)
        err = np.abs(got - o)
        lim = bound(self.dtype, out, o, mag, top, int((self.lens + self.new).max(initial=0)), 6.0)
        lim = lim + more * mag
        assert np.isfinite(got).all()
        worst = float((err / lim).max(initial=0))
        assert worst <= 1, f"{worst:.2f} of the bound, error {err.max():.3g}"
        # the framework's own bars, with half a step of a 16-bit store
        bar = 1e-5 if self.dtype == "f32" else 2e-3
        half = {"f32": 0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[out]
        assert (err - half * np.abs(o)).max(initial=0) <= bar
        return got


SHAPES = [
    # lens, new, heads, page_rows
    ([0], [1], 1, 16), ([5], [1], 3, 64), ([448], [16], 6, 64), ([63, 64, 65], [1, 1, 1], 2, 64),
    ([0, 0, 7], [4, 0, 2], 3, 48), ([127, 1, 1000], [7, 8, 9], 2, 16),
    ([33, 200, 64, 0], [31, 32, 33, 40], 4, 32), ([700, 30], [64, 63], 2, 128),
    ([16] * 40, [1] * 40, 20, 16), ([2100, 3], [17, 1], 1, 48),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_attend(W, dtype, shape, kind):
    lens, new, heads, page_rows = SHAPES[shape]
    rng = np.random.default_rng(shape)
    par = sum((tree(rng, k) for k in new), []) if kind == "tree" else None
    b = Batch(100 + shape, dtype, lens, new, heads, page_rows, par)
    b.check(W)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_f32_output_and_strides(W, dtype):
    rng = np.random.default_rng(9)
    new = [5, 40, 1, 0, 20]
    par = sum((tree(rng, k) for k in new), [])
    b = Batch(9, dtype, [100, 450, 2, 77, 0], new, 5, 64, par, stride=640)
    b.check(W, out="f32")
    b.check(W, layer=0, stride=320)
    b.check(W, scale=0.05)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_long_chain(W, dtype):
    """A prompt longer than any row tile, next to single rows."""
    b = Batch(10, dtype, [0, 300, 64], [224, 1, 130], 3, 64)
    b.check(W)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_many_keys(W, dtype):
    rng = np.random.default_rng(11)
    new = [3, 64, 12]
    b = Batch(11, dtype, [9000, 5001, 17], new, 2, 48, sum((tree(rng, k) for k in new), []), layers=2)
    b.check(W)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_wide_trees(W, dtype):
    """More than 64 rows to a tree: masks of several words, rows over several tiles."""
    rng = np.random.default_rng(12)
    new = [130, 2, 97]
    b = Batch(12, dtype, [70, 500, 0], new, 2, 64, sum((tree(rng, k) for k in new), []), words=5)
    b.check(W)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), "lowest"])
def test_masked_places_have_no_influence(W, dtype, bad):
    """Rows of the tree that others do not see hold NaN, infinities or the
    type's lowest value: only rows that see them may notice."""
    import torch
    bad = torch.finfo(tdt(dtype)).min if bad == "lowest" else bad
    new = [12, 3, 50]
    lens = [60, 5, 130]
    rng = np.random.default_rng(13)
    par = sum((tree(rng, k) for k in new), [])
    b = Batch(13, dtype, lens, new, 3, 64, par)
    clean = b.attend(W, 1, "f32")
    b.check(W)
    victims = [(0, 5), (0, 11), (2, 40), (2, 7)]
    hit = np.zeros(int(b.start[-1]), bool)
    for s, j in victims:
        at = lens[s] + j
        b.pool[int(b.st.table[s, at // 64]), 1, :, :, at % 64] = bad
        for i in range(new[s]):
            r = b.start[s] + i
            hit[r] |= bool(b.mask[r].view(np.uint32)[j // 32] >> np.uint32(j % 32) & np.uint32(1))
    got = b.attend(W, 1, "f32")
    assert hit.any() and not hit.all()
    assert np.array_equal(got[~hit], clean[~hit])
    if not np.isfinite(bad):
        assert np.isnan(got[hit]).all(axis=1).any() or not np.isfinite(got[hit]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_value_that_is_not_finite_reaches_those_who_see_it(W, dtype, value):
    """One value element of one draft: in the rows that see it that one
    dimension is not finite, as in the formula, and nothing else changes."""
    lens, new = [40, 9], [20, 6]
    rng = np.random.default_rng(14)
    b = Batch(14, dtype, lens, new, 2, 32, sum((tree(rng, k) for k in new), []))
    clean = b.attend(W, 0, "f32")
    at = lens[0] + 4
    b.pool[int(b.st.table[0, at // 32]), 0, 1, 1, at % 32, 37] = value
    got = b.attend(W, 0, "f32")
    sees = np.zeros(26, bool)
    sees[:20] = [(int(b.mask[i, 0]) >> 4) & 1 for i in range(20)]
    assert sees.any() and not sees[:20].all()
    want = got[sees][:, 64 + 37]
    assert np.isnan(want).all() if value != value else (want == value).all()
    got[sees, 64 + 37] = clean[sees, 64 + 37]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_that_see_nothing_are_zero(W, dtype):
    b = Batch(15, dtype, [0, 30, 0], [3, 2, 40], 2, 16, [-1, 0, 0] + [-1, 0] + [-1] * 40)
    b.mask[[1, 10, 44]] = 0            # rows of requests without context
    b.mask[4] = 0                      # this one still sees its context
    got = b.check(W)
    assert (got[[1, 10, 44]] == 0).all() and (got[4] != 0).any()


def test_mask_bits_behind_the_request_are_ignored(W):
    b = Batch(16, "f16", [20, 40], [3, 5], 2, 16, [-1, 0, 1, -1, 0, 1, 2, 3])
    plain = b.attend(W, 0, "f16")
    keep = b.mask.copy()
    b.mask[:3] |= np.int32(0x7ffffff8)
    b.mask[:3, 1] = -1
    got = b.attend(W, 0, "f16")
    b.mask = keep
    assert np.array_equal(got, plain)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_large_scores(W, dtype):
    """Scores in the thousands: the running maximum jumps from tile to tile."""
    b = Batch(17, dtype, [600, 10], [20, 3], 2, 64)
    b.pool *= 20
    b.q *= 20
    got = b.attend(W, 1, "f32")
    rows = int(b.start[-1])
    o, mag, top = P.attend(b.pool.float().cpu().numpy(), 1, b.st.table, b.lens, b.start,
                           b.q.float().cpu().numpy()[:rows], 2, 0.125)
    lim = bound(dtype, "f32", o, mag, top, 700, 120.0)
    assert (np.abs(got - o) <= lim).all()


@pytest.mark.parametrize("seed", range(12))
def test_attend_random(W, seed):
    rng = np.random.default_rng(1000 + seed)
    dtype = ["f32", "f16", "bf16"][seed % 3]
    n = int(rng.integers(1, 20))
    lens = (2 ** rng.uniform(0, 10, n)).astype(int) - 1
    new = np.where(rng.random(n) < .2, 0, (2 ** rng.uniform(0, 6.2, n)).astype(int))
    words = 3
    par = sum((tree(rng, int(k), 0.05) for k in new), []) if rng.random() < .7 else None
    b = Batch(2000 + seed, dtype, lens, new, int(rng.integers(1, 8)),
              int(rng.choice([16, 32, 48, 64, 80, 128])), par, words, stride=int(rng.integers(0, 3)) * 8)
    b.check(W, out="f32" if seed % 2 else dtype, stride=int(rng.integers(0, 3)) * 8)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_offsets_beyond_32_bits(W, dtype):
    """Pages more than 4 GiB apart in the pool."""
    import torch
    heads, page_rows, layers = 4, 64, 1
    page = heads * 2 * 64 * page_rows * (2 if dtype == "f16" else 4)
    n_pages = (6 << 30) // page
    order = np.concatenate([np.arange(3, n_pages - 6), [1, n_pages - 1, 0, n_pages - 2, 2, n_pages - 4]])
    pad = np.setdiff1d(np.arange(n_pages), order)
    b = Batch(18, dtype, [250, 100], [9, 2], heads, page_rows, tree(np.random.default_rng(1), 9) + [-1, 0],
              layers=layers, order=np.concatenate([pad, order]), n_pages=n_pages)
    assert b.st.table.max() >= n_pages - 4
    table, lens, start, mask = b.device()
    o = torch.empty(b.max_rows, heads * 64, device="cuda")
    W.paged_attend(b.pool, 0, table, lens, start, b.q, o, row_mask=mask)
    used = sorted(set(b.st.table[b.st.table >= 0].tolist()))
    small = b.pool[used].float().cpu().numpy()
    local = np.where(b.st.table >= 0, np.searchsorted(used, np.maximum(b.st.table, 0)), -1)
    rows = int(b.start[-1])
    ref, mag, top = P.attend(small, 0, local, b.lens, b.start, b.q.float().cpu().numpy()[:rows], heads,
                             0.125, b.mask)
    lim = bound(dtype, "f32", ref, mag, top, 300, 6.0)
    assert (np.abs(o.cpu().numpy()[:rows] - ref) <= lim).all()
    # rows written there land there
    k = torch.randn(b.max_rows, heads * 64, device="cuda").to(tdt(dtype))
    W.paged_write(b.pool, 0, cu(b.slot), k, k)
    for r in range(rows):
        got = b.pool[int(b.slot[r]) // 64, 0, :, :, int(b.slot[r]) % 64]
        assert torch.equal(got, k[r].view(1, heads, 64).expand(2, heads, 64))
    # and moved from there
    tok = cu(np.zeros(b.max_rows))
    want = b.pool[used].cpu().numpy()
    par = np.concatenate([b.parents, np.full(3, -1)])
    paths, _ = P.accept(b.start, par, np.zeros(b.max_rows), np.zeros(b.max_rows))
    P.move(want, b.start, np.array([local.ravel()[np.where(b.st.table.ravel() == sl // 64)[0][0]] * 64
                                    + sl % 64 if sl >= 0 else -1 for sl in b.slot]), paths)
    n = len(b.lens)
    W.paged_accept(b.pool, start, cu(b.slot), tok, tok, lens, cu(np.zeros(n)), cu(np.zeros(b.max_rows)),
                   cu(np.zeros(n)), parents=cu(par))
    same = np.array_equal(b.pool[used].cpu().numpy(), want, equal_nan=True)
    assert same


# ------------------------------------------------------------------ accept

@pytest.mark.parametrize("dtype,layers,heads,page_rows", [("f16", 1, 1, 16), ("bf16", 3, 5, 48),
                                                          ("f32", 2, 20, 64)])
@pytest.mark.parametrize("kind", ["tree", "chain", "dead"])
def test_accept(W, dtype, layers, heads, page_rows, kind):
    import torch
    rng = np.random.default_rng(layers * 7 + heads)
    new = [1, 0, 70, 5, 33, 64, 2, 40]
    lens = rng.integers(0, 200, len(new))
    par = None if kind == "chain" else sum((tree(rng, k, 0.1 if kind == "dead" else 0) for k in new), [])
    if kind == "dead":
        par[int(np.cumsum(new)[3]) - 5] = 3     # request 3 has no root
    b = Batch(50, dtype, lens, new, heads, page_rows, par, words=3, layers=layers)
    tokens = rng.integers(0, 4, b.max_rows)      # few tokens: several children fit
    picked = rng.integers(0, 4, b.max_rows)
    full = None if par is None else np.concatenate([par, np.full(3, -1)])
    paths, nxt = P.accept(b.start, full, tokens, picked)
    want = b.pool.cpu().float().numpy()
    P.move(want, b.start, b.slot, paths)
    d_lens, acc, path, nx = cu(lens), cu(np.full(8, 9)), cu(np.full(b.max_rows, 9)), cu(np.full(8, 9))
    W.paged_accept(b.pool, cu(b.start), cu(b.slot), cu(tokens), cu(picked), d_lens, acc, path, nx,
                   parents=None if full is None else cu(full))
    assert acc.tolist() == [len(p) for p in paths] and nx.tolist() == nxt
    assert d_lens.tolist() == [int(x) + len(p) for x, p in zip(lens, paths)]
    exp = np.full(b.max_rows, -1)
    for s, p in enumerate(paths):
        exp[b.start[s]:b.start[s] + len(p)] = p
    assert path.tolist() == exp.tolist()
    same = np.array_equal(b.pool.cpu().float().numpy(), want, equal_nan=True)
    assert same
    assert max(len(p) for p in paths) >= 2


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_speculative_steps(W, dtype, captured):
    """Steps of plan, write, attend and accept over two layers, eagerly or as
    one captured graph replayed with other lengths, trees and tokens: pages,
    masks and paths equal the model's, and the attention is float64's."""
    import torch
    rng = np.random.default_rng(20)
    n, heads, page_rows, layers, max_rows, words, max_pages = 5, 3, 16, 2, 60, 1, 12
    w = heads * 64
    n_pages = n * max_pages
    st = P.PlanState(n, n_pages, max_pages, rng.permutation(n_pages))
    dev = {k: cu(v) for k, v in dict(
        lens=np.zeros(n), new=np.zeros(n), table=st.table, held=st.held, free=st.free,
        n_free=[n_pages], par=np.full(max_rows, -1), start=np.zeros(n + 1), pos=np.zeros(max_rows),
        slot=np.zeros(max_rows), mask=np.zeros((max_rows, words)), status=[0],
        tok=np.zeros(max_rows), pick=np.zeros(max_rows), acc=np.zeros(n), path=np.zeros(max_rows),
        nxt=np.zeros(n)).items()}
    pool = torch.full((n_pages, layers, 2, heads, page_rows, 64), float("nan"), dtype=tdt(dtype), device="cuda")
    qkv = [torch.zeros(max_rows, 3 * w, dtype=tdt(dtype), device="cuda") for _ in range(layers)]
    out = [torch.zeros(max_rows, w, device="cuda") for _ in range(layers)]
    ws = torch.zeros(max(16, W.paged_attend_workspace_bytes(n, max_rows, heads)), dtype=torch.uint8,
                     device="cuda")

    def step():
        W.paged_plan(dev["lens"], dev["new"], dev["table"], dev["held"], dev["free"], dev["n_free"],
                     dev["start"], dev["pos"], dev["slot"], dev["status"], page_rows=page_rows,
                     parents=dev["par"], row_mask=dev["mask"])
        for i in range(layers):
            W.paged_write(pool, i, dev["slot"], qkv[i][:, w:2 * w], qkv[i][:, 2 * w:])
            W.paged_attend(pool, i, dev["table"], dev["lens"], dev["start"], qkv[i][:, :w], out[i],
                           row_mask=dev["mask"], workspace=ws)
        W.paged_accept(pool, dev["start"], dev["slot"], dev["tok"], dev["pick"], dev["lens"],
                       dev["acc"], dev["path"], dev["nxt"], parents=dev["par"])

    if captured:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            step()  # no rows: loads the kernels
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        run = graph.replay
    else:
        run = step
    lens = np.zeros(n, int)
    rows_of = {}  # (request, layer) -> the kept rows' K and V
    g = torch.Generator(device="cuda").manual_seed(1)
    for turn in range(8):
        new = rng.integers(0, 12, n) if turn else np.array([11, 12, 1, 0, 12])
        if turn == 5:
            lens[1] = 0  # request 1 is replaced by a new one
            dev["lens"][1] = 0
        par = sum((tree(rng, int(k)) for k in new), [])
        full = np.concatenate([par, np.full(max_rows - len(par), -1)]).astype(int)
        tok, pick = rng.integers(0, 3, max_rows), rng.integers(0, 3, max_rows)
        for key, val in (("new", new), ("par", full), ("tok", tok), ("pick", pick)):
            dev[key].copy_(cu(val))
        for x in qkv:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        status, start, pos, slot, mask = P.plan(st, lens, new, page_rows, max_rows, full, words)
        assert status == 0 and dev["status"].item() == 0
        for key, val in (("start", start), ("pos", pos), ("slot", slot), ("mask", mask),
                         ("table", st.table), ("held", st.held)):
            assert np.array_equal(dev[key].cpu().numpy(), val), (turn, key)
        paths, nxt = P.accept(start, full, tok, pick)
        assert dev["nxt"].tolist() == nxt
        # the rows each request should hold now, from the model
        for i in range(layers):
            x = qkv[i].float().cpu().numpy().astype(np.float64)
            got = out[i].cpu().numpy()
            for s in range(n):
                if lens[s] == 0:
                    rows_of[s, i] = np.zeros((0, 2, heads, 64))
                a, b = int(start[s]), int(start[s + 1])
                kv = np.concatenate([rows_of[s, i], x[a:b, w:].reshape(-1, 2, heads, 64)])
                one = np.zeros((1, 1, 2, heads, len(kv), 64))
                one[0, 0] = kv.transpose(1, 2, 0, 3)
                if b > a:
                    o, mag, top = P.attend(one, 0, np.zeros((1, 1), int), [lens[s]], [0, b - a],
                                           x[a:b, :w], heads, 0.125, mask[a:b])
                    lim = bound(dtype, "f32", o, mag, top, len(kv), 6.0)
                    assert (np.abs(got[a:b] - o) <= lim).all(), (turn, i, s)
                rows_of[s, i] = kv[list(range(lens[s])) + [lens[s] + p for p in paths[s]]]
        lens = lens + [len(p) for p in paths]
        assert dev["lens"].tolist() == lens.tolist()
    # what is in the pool at the end is what was kept
    host = pool.float().cpu().numpy()
    for (s, i), kv in rows_of.items():
        at = np.arange(lens[s])
        kept = host[st.table[s, at // page_rows], i, :, :, at % page_rows]
        assert np.array_equal(kept, kv.astype(np.float32))


def test_decode_agrees_with_the_host_planned_cache(W):
    """One new token per request: the same rows through DeviceKvCache and the
    device-planned cache give the same attention to rounding."""
    import torch
    rng = np.random.default_rng(21)
    lens, heads = rng.integers(1, 300, 24), 6
    b = Batch(21, "f16", lens, [1] * 24, heads, 64)
    got = b.attend(W, 1, "f32")
    c = W.DeviceKvCache(1, 24, heads, 448, page_rows=64, dtype=W.F16)
    w = heads * 64
    for s in range(24):
        at = np.arange(lens[s] + 1)
        kv = b.pool[torch.as_tensor(b.st.table[s, at // 64].astype(np.int64)), 1, :, :,
                    torch.as_tensor(at % 64)]
        c.append(0, [s], [len(at)], kv[:, 0].reshape(-1, w), kv[:, 1].reshape(-1, w))
    c.advance(list(range(24)), [int(x) for x in lens])
    o = torch.empty(24, w, device="cuda")
    c.attend(0, list(range(24)), [1] * 24, b.q[:24].contiguous(), o)
    torch.cuda.synchronize()
    assert np.abs(o.cpu().numpy() - got).max() <= 2e-3
    c.close()


def test_runs_on_the_callers_stream(W):
    """Calls on two streams at once, each with its own workspace."""
    import torch
    batches = [Batch(30 + i, "bf16", [400, 30, 1800], [20, 3, 7], 4, 64) for i in range(2)]
    want = [b.attend(W, 1, "bf16") for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    n = max(16, W.paged_attend_workspace_bytes(3, 33, 4))
    for _ in range(5):
        outs = []
        for b, s in zip(batches, streams):
            table, lens, start, _ = b.device()
            ws, o = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.empty(33, 256, dtype=torch.bfloat16, device="cuda")
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                for _ in range(3):
                    W.paged_attend(b.pool, 1, table, lens, start, b.q, o, workspace=ws)
            outs.append((o, table, lens, start, ws))
        torch.cuda.synchronize()
        for (o, *_), x, b in zip(outs, want, batches):
            assert np.array_equal(o[:30].float().cpu().numpy(), x)


@pytest.mark.parametrize("kind", ["cut", "taken", "wide"])
def test_graphs_without_a_workspace(W, kind):
    """Two graphs captured without a workspace, replayed at once on two streams
    and next to an eager call, which uses the thread's."""
    import torch
    if kind == "cut":
        batches = [Batch(80 + i, "bf16", [400, 30, 1800], [20, 3, 7], 4, 64) for i in range(2)]
    elif kind == "taken":
        batches = [many(82 + i, "f16") for i in range(2)]
    else:
        batches = [wide_batch(84 + i, [600, 20, 0], [150, 190, 1], 3, 64) for i in range(2)]
    work = []
    for b in batches:
        want = torch.zeros(b.max_rows, b.heads * 64, device="cuda")
        a = dict(zip(("block_table", "seq_lens", "row_start", "row_mask"), b.device()))
        W.paged_attend(b.pool, 0, q=b.q, o=want, **a)
        o, s, g = torch.zeros_like(want), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            for _ in range(3):
                W.paged_attend(b.pool, 0, q=b.q, o=o, **a)
        work.append((b, a, want, o, s, g))
    for _ in range(4):
        for b, a, want, o, s, g in work:
            with torch.cuda.stream(s):
                o.zero_()
                g.replay()
        b, a, want, *_ = work[0]
        again = torch.zeros_like(want)
        W.paged_attend(b.pool, 0, q=b.q, o=again, **a)
        torch.cuda.synchronize()
        assert torch.equal(again, want)
        for b, a, want, o, s, g in work:
            assert torch.equal(o, want)


CONCURRENT = {
    "cut": lambda: Batch(90, "f16", [700, 30, 1801, 77] * 12, [20, 3, 7, 33] * 12, 6, 64),
    "bf16": lambda: Batch(91, "bf16", [70, 204, 76] * 30, [1, 2, 17] * 30, 20, 48),
    "f32": lambda: Batch(92, "f32", [70, 204, 1000] * 8, [1, 20, 7] * 8, 6, 16),
    "taken": lambda: many(93, "bf16"),
    "wide": lambda: wide_batch(94, [600, 20, 0, 1030], [150, 190, 1, 131], 8, 32),
}


@pytest.mark.parametrize("kind", CONCURRENT)
def test_repeats_beside_another_kernel(W, kind):
    """The same call 200 times while attention of its own runs on another stream."""
    import torch
    b = CONCURRENT[kind]()
    a = dict(zip(("block_table", "seq_lens", "row_start", "row_mask"), b.device()))
    want = torch.zeros(b.max_rows, b.heads * 64, device="cuda")
    W.paged_attend(b.pool, 0, q=b.q, o=want, **a)
    x = torch.randn(4 * 700 * 384, device="cuda").half()
    y = torch.empty_like(x)
    ws = torch.zeros(max(16, W.paged_attend_workspace_bytes(len(b.lens), b.max_rows, b.heads)),
                     dtype=torch.uint8, device="cuda")
    o, differ = torch.empty_like(want), torch.zeros((), dtype=torch.int64, device="cuda")
    side, main = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(200):
        W.attention_fwd(x, x, x, y, batch=4, t_q=700, t_kv=700, n_heads=6, scale=0.125, stream=side)
        with torch.cuda.stream(main):
            o.copy_(want)
            o[:int(b.start[-1])] = 0
            W.paged_attend(b.pool, 0, q=b.q, o=o, workspace=ws, **a)
            differ += (o != want).any()
    torch.cuda.synchronize()
    assert int(differ) == 0


def test_repeats_are_bit_exact(W):
    rng = np.random.default_rng(40)
    new = [20, 1, 33, 64]
    b = Batch(40, "bf16", [3000, 64, 500, 129], new, 6, 64, sum((tree(rng, k) for k in new), []))
    first = b.attend(W, 1, "f32")
    for _ in range(5):
        assert np.array_equal(b.attend(W, 1, "f32"), first)


# ------------------------------------------------------------------ many new rows a request (f16)

# A quarter of the exponentials is a polynomial, 7.5e-5 off at most, in the
# weights and in their sum.
WIDE = 2 * 7.5e-5
WIDE_SHAPES = [
    # lens, new, heads, page_rows
    ([600], [128], 1, 64), ([0, 700, 33], [260, 2, 130], 3, 64), ([1500, 511], [129, 127], 2, 48),
    ([513] * 3, [112] * 3, 5, 16), ([5000], [224], 2, 128), ([900, 0, 0, 0], [500, 0, 1, 3], 2, 32),
    ([400] * 10, [115] * 10, 12, 64), ([127, 700, 129], [256, 100, 20], 2, 32),
]


def wide_batch(seed, lens, new, heads, page_rows, kind="tree", dead=0.0, **kw):
    rng = np.random.default_rng(seed)
    par = sum((tree(rng, k, dead) for k in new), []) if kind == "tree" else None
    b = Batch(seed, "f16", lens, new, heads, page_rows, par, words=-(-max(new) // 32), **kw)
    rows = b.max_rows // len(lens)  # the rule by which the kernel for many rows is chosen
    assert rows * 8 >= 7 * 128 * ((rows + 119) // 128) and b.st.table.shape[1] * page_rows - rows >= 448
    return b


@pytest.mark.parametrize("shape", range(len(WIDE_SHAPES)))
@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_wide_attend(W, shape, kind, out):
    wide_batch(50 + shape, *WIDE_SHAPES[shape], kind).check(W, out=out, more=WIDE)


def test_wide_strides_scales_layers(W):
    b = wide_batch(60, [600, 20, 0], [150, 190, 1], 3, 64, stride=72)
    b.check(W, out="f32", stride=320, more=WIDE)
    b.check(W, layer=0, stride=64, more=WIDE)
    b.check(W, scale=0.05, more=WIDE)


@pytest.mark.parametrize("seed", range(6))
def test_wide_random(W, seed):
    rng = np.random.default_rng(1100 + seed)
    n = int(rng.integers(1, 8))
    lens = (2 ** rng.uniform(0, 10, n)).astype(int) - 1
    lens[0] = 600
    new = np.where(rng.random(n) < .2, 0, rng.integers(1, 130, n))
    new[-1] += 120 * n - int(new.sum())
    b = wide_batch(2100 + seed, lens, new, int(rng.integers(1, 6)), int(rng.choice([16, 32, 48, 64, 80, 128])),
                   "tree" if seed % 3 else "chain", 0.05, stride=int(rng.integers(0, 3)) * 8)
    b.check(W, out="f32" if seed % 2 else "f16", stride=int(rng.integers(0, 3)) * 8, more=WIDE)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), "lowest"])
def test_wide_masked_places_have_no_influence(W, bad):
    import torch
    bad = torch.finfo(torch.float16).min if bad == "lowest" else bad
    lens, new = [600, 5, 130], [140, 3, 230]
    b = wide_batch(61, lens, new, 2, 64)
    clean = b.attend(W, 1, "f32")
    hit = np.zeros(int(b.start[-1]), bool)
    for s, j in [(0, 5), (0, 139), (2, 40), (2, 200)]:
        at = lens[s] + j
        b.pool[int(b.st.table[s, at // 64]), 1, :, :, at % 64] = bad
        for i in range(new[s]):
            r = b.start[s] + i
            hit[r] |= bool(b.mask[r].view(np.uint32)[j // 32] >> np.uint32(j % 32) & np.uint32(1))
    got = b.attend(W, 1, "f32")
    assert hit.any() and not hit.all()
    assert np.array_equal(got[~hit], clean[~hit])
    if not np.isfinite(bad):
        assert not np.isfinite(got[hit]).all()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_wide_value_that_is_not_finite_reaches_those_who_see_it(W, value):
    lens, new = [530, 9], [220, 40]
    b = wide_batch(62, lens, new, 2, 32)
    clean = b.attend(W, 0, "f32")
    at = lens[0] + 4
    b.pool[int(b.st.table[0, at // 32]), 0, 1, 1, at % 32, 37] = value
    got = b.attend(W, 0, "f32")
    sees = np.zeros(260, bool)
    sees[:220] = [(int(b.mask[i, 0]) >> 4) & 1 for i in range(220)]
    assert sees.any() and not sees[:220].all()
    want = got[sees][:, 64 + 37]
    assert np.isnan(want).all() if value != value else (want == value).all()
    got[sees, 64 + 37] = clean[sees, 64 + 37]
    assert np.array_equal(got, clean)


def test_wide_rows_that_see_nothing_are_zero(W):
    b = wide_batch(63, [0, 600, 0], [3, 130, 220], 2, 16)
    b.mask[[1, 140, 300]] = 0
    b.mask[40] = 0  # this one still sees its context
    got = b.check(W, more=WIDE)
    assert (got[[1, 140, 300]] == 0).all() and (got[40] != 0).any()


def test_wide_large_scores(W):
    b = wide_batch(64, [600, 10], [200, 60], 2, 64, "chain")
    b.pool *= 20
    b.q *= 20
    got = b.attend(W, 1, "f32")
    rows = int(b.start[-1])
    o, mag, top = P.attend(b.pool.float().cpu().numpy(), 1, b.st.table, b.lens, b.start,
                           b.q.float().cpu().numpy()[:rows], 2, 0.125)
    lim = bound("f16", "f32", o, mag, top, 800, 120.0) + WIDE * mag
    assert (np.abs(got - o) <= lim).all()


def test_wide_bad_tables_are_reported_and_harmless(W):
    import torch
    for what in ("page", "len", "len_low", "start", "start_back"):
        b = wide_batch(65, [600, 40, 70], [130, 120, 100], 2, 16, "chain")
        ref, mag, top = P.attend(b.pool.float().cpu().numpy(), 1, b.st.table, b.lens, b.start,
                                 b.q.float().cpu().numpy()[:350], 2, 0.125)
        lim = bound("f16", "f32", ref, mag, top, 730, 6.0) + WIDE * mag
        if what == "page":
            b.st.table[1, 0] = b.n_pages
        elif what == "len":
            b.lens[1] = 2 ** 31 - 1
        elif what == "len_low":
            b.lens[1] = -5
        elif what == "start":
            b.start[3] = 1 << 30
        else:
            b.start[2] = 1 << 29
        table, lens, start, _ = b.device()
        o = torch.zeros(b.max_rows, 128, device="cuda")
        W.paged_attend(b.pool, 1, table, lens, start, b.q, o)
        torch.cuda.synchronize()
        assert W.device_status() == -6, what
        assert (np.abs(o[:130].cpu().numpy() - ref[:130]) <= lim[:130]).all(), what


# ------------------------------------------------------------------ many small items

def many(seed, dtype, kind="chain", n=520, heads=12, top=200):
    """More items than four to a warp: they are taken one by one."""
    rng = np.random.default_rng(seed)
    lens, new = rng.integers(0, top, n), rng.integers(1, 4, n)
    lens[rng.random(n) < .1] = 0
    new[rng.random(n) < .1] = 0
    lens[[3, 200]], new[[3, 200]] = 20, 40  # two row tiles and more
    par = sum((tree(rng, int(k), 0.05) for k in new), []) if kind == "tree" else None
    return Batch(seed, dtype, lens, new, heads, 32, par, layers=1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_many_small_items(W, dtype, kind):
    many(70, dtype, kind).check(W, layer=0)


def test_many_requests(W):
    """More requests than a thread looks at one by one."""
    many(71, "f16", n=9000, heads=1, top=24).check(W, layer=0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_small_items_repeat(W, dtype):
    """The workspace is ready again after each call, eager or replayed, and the
    bits do not depend on which warp takes what."""
    import torch
    b = many(72, dtype)
    table, lens, start, _ = b.device()
    ws = torch.zeros(max(16, W.paged_attend_workspace_bytes(520, b.max_rows, 12)), dtype=torch.uint8, device="cuda")
    outs = [torch.zeros(b.max_rows, 768, device="cuda") for _ in range(4)]
    for o in outs[:3]:
        W.paged_attend(b.pool, 0, table, lens, start, b.q, o, workspace=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            W.paged_attend(b.pool, 0, table, lens, start, b.q, outs[3], workspace=ws)
    for _ in range(3):
        outs[3].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[3])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert (ws[:65536 * 4] == 0).all()


def test_many_small_items_bad_tables(W):
    import torch
    for what in ("page", "len", "start_back"):
        b = many(73, "f16")
        rows = int(b.start[-1])
        ref, mag, top = P.attend(b.pool.float().cpu().numpy(), 0, b.st.table, b.lens, b.start,
                                 b.q.float().cpu().numpy()[:rows], 12, 0.125)
        lim = bound("f16", "f32", ref, mag, top, 300, 6.0)
        s = int(np.nonzero((b.new > 0) & (b.lens > 0))[0][100])
        if what == "page":
            b.st.table[s, 0] = b.n_pages
        elif what == "len":
            b.lens[s] = 2 ** 31 - 1
        else:
            b.start[s + 1] = 1 << 29
        table, lens, start, _ = b.device()
        o = torch.zeros(b.max_rows, 768, device="cuda")
        W.paged_attend(b.pool, 0, table, lens, start, b.q, o)
        torch.cuda.synchronize()
        assert W.device_status() == -6, what
        ok = np.r_[0:b.start[s], b.start[s] + b.new[s:s + 2].sum():rows]
        assert (np.abs(o[:rows].cpu().numpy() - ref)[ok] <= lim[ok]).all(), what


# ------------------------------------------------------------------ bad device data

def test_bad_tables_are_reported_and_harmless(W):
    """Entries outside the pool, lengths beyond the table, rows out of order:
    the other requests are right and the status word says so."""
    for what in ("page", "page_low", "len", "len_low", "start", "start_back"):
        b = Batch(41, "f16", [100, 40, 70], [3, 2, 4], 2, 16)
        ref, mag, top = (x[:3] for x in P.attend(
            b.pool.float().cpu().numpy(), 1, b.st.table, b.lens, b.start,
            b.q.float().cpu().numpy()[:9], 2, 0.125))
        lim = bound("f16", "f32", ref, mag, top, 110, 6.0)
        if what == "page":
            b.st.table[1, 0] = b.n_pages
        elif what == "page_low":
            b.st.table[1, 1] = -(2 ** 31)
        elif what == "len":
            b.lens[1] = 2 ** 31 - 1
        elif what == "len_low":
            b.lens[1] = -5
        elif what == "start":
            b.start[3] = 1 << 30
        else:
            b.start[2] = 1 << 29
        import torch
        table, lens, start, _ = b.device()
        o = torch.zeros(b.max_rows, 128, device="cuda")
        W.paged_attend(b.pool, 1, table, lens, start, b.q, o)
        torch.cuda.synchronize()
        assert W.device_status() == -6, what
        # (not bit for bit: the lengths of the others move the cuts of the keys)
        assert (np.abs(o[:3].cpu().numpy() - ref) <= lim).all(), what


@pytest.mark.parametrize("dtype,rows", [("f16", 3), ("f16", 130), ("f32", 3)])
def test_more_work_than_can_be_counted(W, dtype, rows):
    """Lengths that are in range but make 2^31 units of work: reported, and
    no row is written."""
    import torch
    P_, heads = 4096, 64
    pages = (1 << 30) // P_
    pool = torch.zeros(1, 1, 2, heads, P_, 64, dtype=tdt(dtype), device="cuda")
    table = torch.zeros(1, pages, dtype=torch.int32, device="cuda")
    q = torch.zeros(rows, heads * 64, dtype=tdt(dtype), device="cuda")
    o = torch.full((rows, heads * 64), 7.0, device="cuda")
    W.paged_attend(pool, 0, table, cu(np.array([(1 << 30) - rows])), cu(np.array([0, rows])), q, o)
    torch.cuda.synchronize()
    assert W.device_status() == -6
    assert (o == 7).all()
    W.paged_attend(pool, 0, table, cu(np.array([50])), cu(np.array([0, rows])), q, o)
    torch.cuda.synchronize()
    assert W.device_status() == 0 and (o == 0).all()


def test_refusals(W):
    import torch
    b = Batch(42, "f16", [10], [2], 2, 16)
    table, lens, start, _ = b.device()
    o = torch.zeros(b.max_rows, 128, device="cuda")

    def bad(status, **kw):
        a = dict(pool=b.pool, layer=0, block_table=table, seq_lens=lens, row_start=start, q=b.q, o=o)
        a.update(kw)
        with pytest.raises(W.WattnError) as e:
            W.paged_attend(**a)
        assert e.value.status == status

    bad(-6, layer=2)
    bad(-1, q=b.q.float())
    bad(-1, o=o[:, :64])
    bad(-1, o=torch.zeros(b.max_rows, 129, device="cuda")[:, :128])
    bad(-1, row_start=start[:1])
    bad(-1, block_table=table[:0])
    bad(-1, pool=b.pool[:, :, :, :, :8].contiguous())
    bad(-1, pool=b.pool.transpose(0, 1))
    bad(-1, o=o.to(torch.bfloat16))
    bad(-1, scale=0.0)
    bad(-1, row_mask=torch.zeros(b.max_rows - 1, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        W.paged_attend(b.pool, 0, table.long(), lens, start, b.q, o)
    n = W.paged_attend_workspace_bytes(1, b.max_rows, 2)
    if n > 16:
        bad(-1, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
