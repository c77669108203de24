"""Refusals of the wattn_paged_* entry points: bad arguments come back as
error codes from the host-side checks, before any launch. The addresses are
made up and never dereferenced; on a machine with a GPU the tests stand aside
(a check that let one through would hand it to a kernel there)."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="made-up device addresses are only passed where no GPU is")

A = 1 << 20  # an aligned made-up address


@pytest.fixture(scope="module")
def W():
    import wattn
    return wattn


def refused(W, fn, base, at, value, status, text):
    args = list(base)
    args[at] = value
    assert fn(*args) == status, (at, value)
    buf = ctypes.create_string_buffer(512)
    assert W.lib.wattn_last_error(buf, 512) == status
    assert text in buf.value, buf.value


#                0  1  2  3   4   5  6  7  8  9  10 11 12 13 14 15 16 17  18 19
PLAN = [A, A, 2, 64, 8, A, 4, 4, A, A, A, A, A, A, A, A, 1, 32, A, None]


@pytest.mark.parametrize("at,value,status,text", [
    (2, -1, -1, b"sizes"), (3, 0, -1, b"sizes"), (4, 0, -1, b"sizes"), (7, 0, -1, b"sizes"),
    (17, -1, -1, b"sizes"), (4, 1 << 26, -2, b"2^31"), (6, 3, -1, b"table_stride"),
    (11, None, -1, b"together"), (15, None, -1, b"together"), (16, 0, -1, b"mask_words"),
    (0, None, -1, b"NULL"), (5, None, -1, b"NULL"), (8, None, -1, b"NULL"), (9, None, -1, b"NULL"),
    (10, None, -1, b"NULL"), (12, None, -1, b"NULL"), (13, None, -1, b"NULL"),
    (14, None, -1, b"NULL"), (18, None, -1, b"NULL"), (0, A + 2, -1, b"aligned"),
    (18, A + 1, -1, b"aligned")])
def test_plan(W, at, value, status, text):
    refused(W, W.lib.wattn_paged_plan, PLAN, at, value, status, text)


#       pool dt pages layers heads rows layer slot n  k  v src stride stream
WRITE = [A, 1, 8, 2, 3, 64, 0, A, 4, A, A, 1, 192, None]
POOL = [(0, None, -1, b"16-byte"), (0, A + 8, -1, b"16-byte"), (1, 7, -1, b"dtype"),
        (2, 0, -1, b"sizes"), (3, 0, -1, b"sizes"), (4, 0, -1, b"sizes"), (4, 70000, -1, b"sizes"),
        (5, 24, -1, b"multiple of 16"), (5, 0, -1, b"multiple of 16"), (2, 1 << 23, -2, b"2^31")]


@pytest.mark.parametrize("at,value,status,text", POOL + [
    (6, 2, -6, b"layer"), (6, -1, -6, b"layer"), (11, 3, -1, b"dtype"), (8, -1, -1, b"n_rows"),
    (12, 191, -1, b"row_stride"), (7, None, -1, b"NULL"), (9, None, -1, b"NULL"),
    (10, None, -1, b"NULL"), (9, A + 1, -1, b"aligned"), (7, A + 2, -1, b"aligned")])
def test_write(W, at, value, status, text):
    refused(W, W.lib.wattn_paged_write, WRITE, at, value, status, text)


#        0  1  2  3  4  5   6  7  8  9  10 11 12 13 14 15 16   17 18 19  20  21  22 23 24
ATTEND = [A, 1, 8, 2, 3, 64, 0, A, 4, 4, A, A, 2, A, 1, A, 192, A, 1, 192, 32, .125, None, 0, None]


@pytest.mark.parametrize("at,value,status,text", POOL + [
    (6, 2, -6, b"layer"), (18, 2, -1, b"out_dtype"), (18, 5, -1, b"out_dtype"),
    (12, -1, -1, b"sizes"), (20, -1, -1, b"sizes"), (9, 0, -1, b"sizes"), (8, 3, -1, b"sizes"),
    (14, 0, -1, b"mask_words"), (21, 0., -1, b"scale"), (21, float("nan"), -1, b"scale"),
    (21, float("inf"), -1, b"scale"), (16, 184, -1, b"stride"), (19, 128, -1, b"stride"),
    (7, None, -1, b"NULL"), (10, None, -1, b"NULL"), (11, None, -1, b"NULL"),
    (15, None, -1, b"NULL"), (17, None, -1, b"NULL"), (10, A + 2, -1, b"4-byte"),
    (13, A + 1, -1, b"4-byte"), (15, A + 8, -1, b"16-byte"), (17, A + 2, -1, b"16-byte"),
    (16, 196, -1, b"16 "), (19, 193, -1, b"16 ")])
def test_attend(W, at, value, status, text):
    refused(W, W.lib.wattn_paged_attend, ATTEND, at, value, status, text)


#        0  1  2  3  4  5   6  7  8   9  10 11 12 13 14 15 16 17
ACCEPT = [A, 1, 8, 2, 3, 64, A, 2, 32, A, A, A, A, A, A, A, A, None]


@pytest.mark.parametrize("at,value,status,text", POOL + [
    (7, -1, -1, b"sizes"), (8, -1, -1, b"sizes"), (6, None, -1, b"NULL"), (10, None, -1, b"NULL"),
    (11, None, -1, b"NULL"), (12, None, -1, b"NULL"), (13, None, -1, b"NULL"),
    (14, None, -1, b"NULL"), (15, None, -1, b"NULL"), (16, None, -1, b"NULL"),
    (9, A + 2, -1, b"aligned"), (13, A + 1, -1, b"aligned")])
def test_accept(W, at, value, status, text):
    refused(W, W.lib.wattn_paged_accept, ACCEPT, at, value, status, text)


def test_nothing_to_do_is_no_error(W):
    L = W.lib
    assert L.wattn_paged_write(*[0 if i == 8 else x for i, x in enumerate(WRITE)]) == 0
    assert L.wattn_paged_attend(*[0 if i == 12 else x for i, x in enumerate(ATTEND)]) == 0
    assert L.wattn_paged_attend(*[0 if i == 20 else x for i, x in enumerate(ATTEND)]) == 0
    assert L.wattn_paged_accept(*[0 if i == 7 else x for i, x in enumerate(ACCEPT)]) == 0
    assert W.paged_attend_workspace_bytes(0, 4, 4) == 0


def test_host_tensors_are_refused(W):
    pool = torch.zeros(2, 1, 2, 1, 16, 64)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(TypeError):
        W.paged_write(pool, 0, i, torch.zeros(4, 64), torch.zeros(4, 64))
    with pytest.raises(TypeError):
        W.paged_plan(i, i, i.view(2, 2), i, i, i, i, i, i, i, page_rows=16)
