"""The host model of the device-planned paged cache on cases small enough to
follow by hand."""
import numpy as np

from oracle import paged_oracle as P


def test_plan_takes_and_gives_back_pages():
    st = P.PlanState(2, 6, 4)
    status, start, pos, slot, _ = P.plan(st, [0, 5], [3, 4], 4, 8)
    # request 0 needs 1 page, request 1 (9 tokens) 3: taken from the top of 0..5
    assert status == 0 and st.table[0].tolist() == [5, -1, -1, -1]
    assert st.table[1].tolist() == [4, 3, 2, -1] and st.n_free == 2
    assert start.tolist() == [0, 3, 7]
    assert pos.tolist() == [0, 1, 2, 5, 6, 7, 8, -1]
    assert slot.tolist() == [20, 21, 22, 3 * 4 + 1, 3 * 4 + 2, 3 * 4 + 3, 2 * 4, -1]
    # undone: the stack is as it was
    assert P.plan(st, [0, 0], [0, 0], 4, 8)[0] == 0
    assert st.n_free == 6 and st.free.tolist() == [0, 1, 2, 3, 4, 5] and (st.table == -1).all()


def test_plan_refuses_whole():
    st = P.PlanState(2, 3, 4)
    before = st.table.copy()
    assert P.plan(st, [0, 0], [8, 8], 4, 16)[0] == P.NOMEM
    assert P.plan(st, [0, 0], [17, 0], 4, 32)[0] == P.RANGE
    assert P.plan(st, [0, 0], [2, 2], 4, 3)[0] == P.RANGE
    assert P.plan(st, [-1, 0], [2, 2], 4, 8)[0] == P.INVALID
    assert (st.table == before).all() and st.n_free == 3


def test_tree_masks_and_dead_rows():
    st = P.PlanState(1, 3, 3)
    #            root 0   1   1   dead  below it
    par = np.array([-1, 0, 1, 1, 4, 4])
    _, _, pos, slot, mask = P.plan(st, [10], [6], 16, 7, par, 1)
    assert pos.tolist() == [10, 11, 12, 12, -1, -1, -1]
    assert mask[:, 0].tolist() == [1, 3, 7, 11, 0, 0, 0]
    assert slot[3] == st.table[0, 0] * 16 + 13 and slot[4] == st.table[0, 0] * 16 + 14


def test_accept_takes_the_lowest_fitting_child():
    start = np.array([0, 5, 5, 6])
    par = np.array([-1, 0, 0, 2, 2, 0])
    tok = np.array([1, 7, 8, 9, 9, 3])
    pick = np.array([8, 0, 9, 4, 5, 6])
    paths, nxt = P.accept(start, par, tok, pick)
    assert paths == [[0, 2, 3], [], []] and nxt == [4, -1, -1]
    assert P.accept(start, None, np.array([1, 8, 0, 0, 0, 3]), pick)[0] == [[0, 1, 2], [], [0]]


def test_attention_of_an_empty_row_is_zero():
    r = np.random.default_rng(0)
    pool = r.standard_normal((2, 1, 2, 1, 16, 64))
    table, q = np.array([[1, -1]]), r.standard_normal((2, 64))
    o, _, _ = P.attend(pool, 0, table, [0], [0, 2], q, 1, 0.125,
                       np.array([[0], [2]], np.int32))
    assert (o[0] == 0).all()
    assert np.allclose(o[1], pool[1, 0, 1, 0, 1])  # it sees itself alone
