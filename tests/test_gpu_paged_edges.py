"""The device-planned paged cache where its attention can go wrong quietly:
values that are not finite, long flat tails, lengths near 2^31, row buffers
larger than the step, and what the device status word says of whom."""
import numpy as np
import pytest

from tests.test_gpu_paged import WIDE, W, bound, clean_status, wide_batch  # noqa: F401

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
        p = torch.softmax(z, -1)
        big = torch.einsum("nhd,khd->hnk", q.abs(), kv[:, 0].abs()).masked_fill(~seen, 0) * scale
        for i, x in enumerate((torch.einsum("hnk,khd->nhd", p, kv[:, 1]),
                               torch.einsum("hnk,khd->nhd", p, kv[:, 1].abs()),
                               big.amax(-1).T[:, :, None].expand(n, b.heads, 64))):
            out[i, a:a + n] = x.reshape(n, w).cpu().numpy()
    return out


def place(b, s, at):
    """Index of position `at` of request s in the pool's first and fifth dimension."""
    return int(b.st.table[s, at // b.P]), at % b.P


# ------------------------------------------------------------------ values and keys that are not finite

@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_wide_value_that_is_not_finite_where_the_maximum_grows(W, value):
    """Tiles in which the running maximum grows by more than 2^8 and a draft's
    value is not finite: the sums so far are rescaled once, in all dimensions
    but the value's own."""
    b = wide_batch(66, [1000], [128], 2, 64, layers=1)
    b.q += 1
    # scores of about 32 in the tile of the first drafts, of about 64 in the next
    # (every row sees that draft)
    jumps = [(999, 4.0), (1030, 8.0)]
    for at, k in jumps:
        page, row = place(b, 0, at)
        b.pool[page, 0, 0, :, row] = k
    b.mask[:128, 0] |= np.int32(1 << 30)
    o, mag, top = formula(b, 0)
    sees = seen_by(b, 0)
    hit = sees[:, 4] | sees[:, 40]
    assert hit.any() and not hit.all()
    for at in (1004, 1040):
        page, row = place(b, 0, at)
        b.pool[page, 0, 1, 1, row, 37] = value
    got = b.attend(W, 0, "f32")
    want = got[hit, 64 + 37]
    assert np.isnan(want).all() if value != value else (want == value).all()
    got[hit, 64 + 37] = o[hit, 64 + 37]
    lim = bound("f16", "f32", o, mag, top, 1128, 6.0) + WIDE * mag
    assert (np.abs(got - o) <= lim).all()
