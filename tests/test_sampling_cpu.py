"""What qg_sample and qg_sampling_softmax refuse, before any device call."""
import ctypes as C

import pytest

from nebula_amd import qg

INVALID = 1  # hipErrorInvalidValue
A = 1 << 20   # a well-aligned address that is never read
W, N = 22 * A, 1 << 40


@pytest.fixture(scope="module")
def lib():
    return qg.lib()


def ask(**kw):
    return C.byref(qg.Sampling(**(dict(temperature=10 * A, top_k=11 * A, top_p=12 * A, min_p=13 * A) | kw)))


# token, logprob, x, rows, cols, draws, sampling, u, workspace, bytes
GOOD = [A, 2 * A, 3 * A, 5, 1000, 2, None, 8 * A, W, N]
BAD = [(0, None), (0, A + 2), (1, 2 * A + 1), (2, None), (2, 3 * A + 2), (3, 0), (3, -1), (3, 65537), (4, 0), (4, (1 << 24) + 1), (5, 0), (5, 65), (7, None),
       (7, 8 * A + 1), (8, None), (8, W + 8), (9, 0), (9, 15), (1, A), (1, A + 36), (0, 3 * A), (0, 3 * A + 4 * 4999), (1, 3 * A + 400), (0, 8 * A + 36), (1, 8 * A),
       (0, 10 * A), (0, 11 * A + 16), (1, 12 * A), (1, 13 * A + 16), (8, 3 * A), (8, 3 * A + 16000), (8, 8 * A), (8, 10 * A), (8, 13 * A), (8, A), (8, 2 * A + 32)]


@pytest.mark.parametrize("at,value", BAD)
def test_refused_samples(lib, at, value):
    args = list(GOOD)
    args[6] = ask()
    args[at] = value
    if at == 3 and value == 65537 or at == 4 and value:
        assert lib.qg_sample_workspace_bytes(args[3], args[4]) == 0
    assert lib.qg_sample(*args) == INVALID


@pytest.mark.parametrize("kw", [dict(temperature=10 * A + 2), dict(top_k=11 * A + 1), dict(top_p=12 * A + 3), dict(min_p=13 * A + 2)])
def test_refused_requests(lib, kw):
    args = list(GOOD)
    args[6] = ask(**kw)
    assert lib.qg_sample(*args) == INVALID
    assert lib.qg_sampling_softmax(A, 3 * A, 5, 1000, ask(**kw), W, N) == INVALID
    args[6] = None
    assert lib.qg_sample(*args) == INVALID
    assert lib.qg_sampling_softmax(A, 3 * A, 5, 1000, None, W, N) == INVALID


@pytest.mark.parametrize("args", [
    (None, 3 * A, 5, 1000, W, N), (A, None, 5, 1000, W, N), (A + 2, 3 * A, 5, 1000, W, N), (A, 3 * A + 1, 5, 1000, W, N), (A, 3 * A, 0, 1000, W, N),
    (A, 3 * A, 5, 0, W, N), (A, 3 * A, 65536, 1 << 24, W, N), (A, 3 * A, 5, 1000, None, N), (A, 3 * A, 5, 1000, W + 4, N), (A, 3 * A, 5, 1000, W, 15),
    (3 * A + 4, 3 * A, 5, 1000, W, N), (3 * A - 19996, 3 * A, 5, 1000, W, N), (A, 3 * A, 5, 1000, 3 * A + 16, N), (A, 3 * A, 5, 1000, A, N),
    (10 * A, 3 * A, 5, 1000, W, N), (11 * A - 19984, 3 * A, 5, 1000, W, N), (12 * A, 3 * A, 5, 1000, W, N), (13 * A, 3 * A, 5, 1000, W, N),
    (A, 3 * A, 5, 1000, 10 * A, N), (A, 3 * A, 5, 1000, 13 * A, N)])
def test_refused_probabilities(lib, args):
    out, x, rows, cols, ws, n = args
    assert lib.qg_sampling_softmax(out, x, rows, cols, ask(), ws, n) == INVALID


def test_workspace_sizes(lib):
    for rows, cols in ((0, 5), (5, 0), (65537, 5), (5, (1 << 24) + 1), (-1, -1), (4096, 1 << 24)):
        assert lib.qg_sample_workspace_bytes(rows, cols) == 0
    for cols in (1, 1000, 4096, 4097, 151936, 1 << 24):
        sizes = [lib.qg_sample_workspace_bytes(r, cols) for r in (1, 2, 3, 17, 64, 255, 256, 257, 1000, 2048)]
        assert sizes[0] >= 16 and sizes == sorted(sizes)
        assert lib.qg_sample(*[A, None, 3 * A, 2, cols, 1, ask(), 2 * A, 1 << 42, sizes[1] - 1]) == INVALID
