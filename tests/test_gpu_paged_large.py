"""The device-planned paged cache at sizes that take its other paths: more
requests than a plan's threads and tables hold at a time, trees and accepted
paths longer than what an acceptance keeps at hand."""
import numpy as np
import pytest

from oracle import paged_oracle as P
from tests.test_gpu_paged import Batch, Plan, W, clean_status, cu, tree  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seqs,most,words", [(20000, 1, 1), (20000, 1, 0), (9000, 4, 2), (17000, 3, 0)])
def test_plan_many_requests(W, n_seqs, most, words):
    """Steps of growing, shrinking and finishing requests, many to a thread."""
    rng = np.random.default_rng(n_seqs + words)
    pl = Plan(W, rng, n_seqs, n_seqs * 3, 4, n_seqs * most * 3 // 4, 16, words)
    lens = rng.integers(0, 40, n_seqs)
    for step in range(3):
        new = np.where(rng.random(n_seqs) < 0.4, rng.integers(1, most + 1, n_seqs), 0)
        par = sum((tree(rng, int(k), 0.1) for k in new), []) if words else None
        assert pl.step(lens, new, par)[0] == 0
        lens = lens + rng.integers(0, new + 1)
        lens[rng.random(n_seqs) < 0.3] = 0
    pl.step(np.zeros(n_seqs, int), np.zeros(n_seqs, int), [] if words else None)
    assert pl.st.n_free == len(pl.st.free)


@pytest.mark.parametrize("kind", ["chain", "every other row", "stops"])
@pytest.mark.parametrize("rows", [256, 257, 512, 1024, 1025, 1500])
def test_accept_long_paths(W, rows, kind):
    """Paths of hundreds of rows, moved in several turns."""
    new = [rows, 0, 5, rows - 1]
    lens = np.array([7, 9, 0, 100])
    par = None
    tokens = np.zeros(sum(new) + 3, int)
    if kind != "chain":
        one = lambda n: [-1] + [i - 1 if i % 2 else i - 2 for i in range(1, n)]  # noqa: E731
        par = sum((one(n) for n in new if n), [])
        tokens[:sum(new)] = np.concatenate([np.arange(n) % 2 for n in new])
    picked = np.zeros(len(tokens), int)
    if kind == "stops":
        picked[260], picked[sum(new[:3]) + 130] = 2, 1
    b = Batch(60, "f16", lens, new, 2, 48, par, words=-(-rows // 32), layers=2)
    full = None if par is None else np.concatenate([par, np.full(3, -1)])
    paths, nxt = P.accept(b.start, full, tokens, picked)
    want = b.pool.cpu().float().numpy()
    P.move(want, b.start, b.slot, paths)
    d_lens, acc, nx = cu(lens), cu(np.full(4, 9)), cu(np.full(4, 9))
    path = cu(np.full(b.max_rows, 9))
    W.paged_accept(b.pool, cu(b.start), cu(b.slot), cu(tokens), cu(picked), d_lens, acc, path, nx,
                   parents=None if full is None else cu(full))
    assert acc.tolist() == [len(p) for p in paths] and nx.tolist() == nxt
    assert d_lens.tolist() == [int(x) + len(p) for x, p in zip(lens, paths)]
    exp = np.full(b.max_rows, -1)
    for s, p in enumerate(paths):
        exp[b.start[s]:b.start[s] + len(p)] = p
    assert path.tolist() == exp.tolist()
    assert np.array_equal(b.pool.cpu().float().numpy(), want, equal_nan=True)
