"""Host model of the device-planned paged cache (test infrastructure).

Plain loops over requests and rows, whole numbers exact and the attention in
float64: the definitions of include/wattn.h's "Device-planned paged cache",
written out. ``pool`` is a numpy array [n_pages][n_layers][2][n_heads]
[page_rows][64].
"""
import numpy as np

OK, INVALID, NOMEM, RANGE = 0, -1, -5, -6


class PlanState:
    """Block table, pages held and free stack of a set of requests."""

    def __init__(self, n_seqs, n_pages, max_pages, order=None):
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        self.held = np.zeros(n_seqs, np.int32)
        self.free = np.array(range(n_pages) if order is None else order, np.int32)
        self.n_free = n_pages


def plan(st, lens, new, page_rows, max_rows, parents=None, mask_words=0):
    """(status, row_start, row_pos, row_slot, row_mask); updates ``st``."""
    n, max_pages = st.table.shape
    n_pages = len(st.free)
    start = np.zeros(n + 1, np.int32)
    pos, slot = np.full(max_rows, -1, np.int32), np.full(max_rows, -1, np.int32)
    mask = np.zeros((max_rows, mask_words), np.uint32)
    lens, new = [int(x) for x in lens], [int(x) for x in new]
    need = [-(-(a + b) // page_rows) for a, b in zip(lens, new)]
    give = sum(max(0, int(h) - m) for h, m in zip(st.held, need))
    take = sum(max(0, m - int(h)) for h, m in zip(st.held, need))
    status = OK
    if (min(lens + [0]) < 0 or min(new + [0]) < 0 or np.any(st.held < 0)
            or np.any(st.held > max_pages) or not 0 <= st.n_free <= n_pages
            or st.n_free + give > n_pages):
        status = INVALID
    elif (max(need + [0]) > max_pages or sum(new) > max_rows
          or (parents is not None and max(new + [0]) > 32 * mask_words)):
        status = RANGE
    elif take > st.n_free + give:
        status = NOMEM
    if status != OK:
        return status, start, pos, slot, mask.view(np.int32)
    back = []
    for s in range(n):
        for i in range(need[s], st.held[s]):
            back.append(st.table[s, i])
            st.table[s, i] = -1
    for g, p in enumerate(back):
        st.free[st.n_free + len(back) - 1 - g] = p
    st.n_free += len(back)
    for s in range(n):
        for i in range(st.held[s], need[s]):
            st.n_free -= 1
            st.table[s, i] = st.free[st.n_free]
        st.held[s] = need[s]
    start[1:] = np.cumsum(new)
    for s in range(n):
        a = start[s]
        for t in range(new[s]):
            up, j = [t], t
            while parents is not None:
                k = int(parents[a + j])
                if k == -1:
                    break
                if k < -1 or k >= j:
                    up = None
                    break
                up.append(k)
                j = k
            at = lens[s] + t
            slot[a + t] = st.table[s, at // page_rows] * page_rows + at % page_rows
            if up is None:
                continue
            pos[a + t] = at if parents is None else lens[s] + len(up) - 1
            if parents is not None:
                for j in up:
                    mask[a + t, j // 32] |= np.uint32(1 << (j % 32))
    return status, start, pos, slot, mask.view(np.int32)


def attend(pool, layer, table, lens, start, q, n_heads, scale, row_mask=None):
    """(o, sum of the weights times |v|, bound on the scores' magnitudes) in
    float64 for the packed rows; q [rows][n_heads*64]."""
    page_rows = pool.shape[4]
    rows, w = q.shape
    o, mag, top = np.zeros((rows, w)), np.zeros((rows, w)), np.zeros((rows, n_heads))
    for s in range(len(lens)):
        a, n, ln = int(start[s]), int(start[s + 1] - start[s]), int(lens[s])
        if n == 0:
            continue
        at = np.arange(ln + n)
        kv = pool[table[s, at // page_rows], layer, :, :, at % page_rows].astype(np.float64)
        for i in range(n):
            if row_mask is None:
                seen = at <= ln + i
            else:
                bits = row_mask[a + i].view(np.uint32)
                seen = np.array([p < ln or ((p - ln) // 32 < len(bits)
                                            and bool(bits[(p - ln) // 32] >> np.uint32((p - ln) % 32) & np.uint32(1)))
                                 for p in at])
            k, v = kv[seen, 0], kv[seen, 1]  # [keys][heads][64]
            if len(k) == 0:
                continue
            qi = q[a + i].astype(np.float64).reshape(n_heads, 64)
            z = np.einsum("hd,khd->hk", qi, k) * scale
            p = np.exp(z - z.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            o[a + i] = np.einsum("hk,khd->hd", p, v).ravel()
            mag[a + i] = np.einsum("hk,khd->hd", p, np.abs(v)).ravel()
            top[a + i] = (np.einsum("hd,khd->hk", np.abs(qi), np.abs(k)) * scale).max(1)
    return o, mag, np.repeat(top, 64, axis=1)


def accept(start, parents, tokens, picked):
    """(paths of each request, next tokens)."""
    paths, nxt = [], []
    for s in range(len(start) - 1):
        a, n = int(start[s]), int(start[s + 1] - start[s])
        par = [t - 1 for t in range(n)] if parents is None else [int(x) for x in parents[a:a + n]]
        path = [0] if n and par[0] == -1 else []
        while path:
            cur = path[-1]
            kids = [c for c in range(cur + 1, n)
                    if par[c] == cur and tokens[a + c] == picked[a + cur]]
            if not kids:
                break
            path.append(kids[0])
        paths.append(path)
        nxt.append(int(picked[a + path[-1]]) if path else -1)
    return paths, nxt


def move(pool, start, slots, paths):
    """The accepted rows of every layer moved together, in place."""
    page_rows = pool.shape[4]
    for s, path in enumerate(paths):
        a = int(start[s])
        for j, p in enumerate(path):
            src, dst = int(slots[a + p]), int(slots[a + j])
            pool[dst // page_rows, :, :, :, dst % page_rows] = \
                pool[src // page_rows, :, :, :, src % page_rows]
