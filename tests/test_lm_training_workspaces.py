"""Workspace queries of the output-layer loss and the orthogonalised update: what a call asks for covers every launch it makes.
None of this needs a GPU."""
import ctypes

import pytest

from origindl_amd import _lib

KGROUP, GROUP_BYTES = 32, 2 << 30  # matrices per launch, and the workspace that bounds their number


@pytest.fixture(scope="module")
def l():
    return _lib.lib()


def schulz(l, batch, rows, cols):
    return l.query("odl_hip_newton_schulz_workspace_bytes", batch, rows, cols)


def muon(l, count, rows, cols):
    return l.query("odl_hip_muon_step_multi_workspace_bytes", count, (ctypes.c_int64 * count)(*[rows] * count), (ctypes.c_int64 * count)(*[cols] * count))


def padded(n):
    tile = 128 if n > 64 else 64
    return -(-n // tile) * tile


def group_of(count, rows, cols):
    """How many of `count` equal matrices share a launch: two copies of X in two layouts and two square matrices each, 4 bytes an
    element. (With a short side up to 128 they need far less than this, and 32 always fit.)"""
    m, n = padded(min(rows, cols)), padded(max(rows, cols))
    if min(rows, cols) <= 128 and max(rows, cols) <= 4096:
        return min(count, KGROUP)
    return max(1, min(count, KGROUP, GROUP_BYTES // (16 * m * n + 8 * m * m)))


SIDES = (40, 128, 200, 256, 320, 384, 512, 640, 768, 1000, 1024, 1536, 1920, 2048, 2560, 3000, 4096, 6000, 8192, 11008, 16384, 50000)


@pytest.mark.parametrize("rows", SIDES)
def test_a_batch_asks_for_what_each_of_its_groups_needs(l, rows):
    """A group smaller than the full one may cut its products into more runs, whose sums need more room than the matrices left out."""
    for cols in SIDES:
        if cols < rows or rows * cols > 1 << 28:
            continue
        for count in range(1, 65):
            group = group_of(count, rows, cols)
            rest = count % group
            asked = schulz(l, count, rows, cols)
            for part in (group, rest):
                # alone, `part` matrices are one group: the query is what that group lays out
                assert part == 0 or asked >= schulz(l, part, rows, cols), (count, rows, cols, part)
            if count in (31, 33, 61, 63, 64):
                assert muon(l, count, rows, cols) == asked and muon(l, count, cols, rows) == schulz(l, count, cols, rows)


def test_shapes_whose_last_group_needs_the_most(l):
    for count, rows, cols, rest in ((63, 384, 1920, 31), (63, 320, 1920, 31), (62, 512, 4096, 30), (63, 512, 4096, 31)):
        assert schulz(l, rest, rows, cols) > schulz(l, 32, rows, cols)
        assert schulz(l, count, rows, cols) == muon(l, count, rows, cols) == schulz(l, rest, rows, cols)


def test_a_workspace_for_the_full_group_alone_is_refused(l):
    some, count, rows, cols = ctypes.c_void_p(256), 63, 384, 1920  # never dereferenced
    nb = schulz(l, 32, rows, cols)
    coef = (3.4445, -4.7750, 2.0315)
    assert l.cdll.odl_hip_newton_schulz(some, count, rows, cols, 5, *coef, 1e-7, some, some, nb, None) == _lib.ODL_ERR_INVALID_ARG
    assert "workspace" in l.last_error()


@pytest.mark.parametrize("N", [1, 32, 64, 128, 200, 256, 257, 4096])
def test_backward_goes_over_the_vocabulary_in_pieces_whatever_the_rows(l, N):
    """softmax - one-hot never lies in the workspace whole: what a call asks for has a bound in V."""
    q = lambda K, V: l.query("odl_hip_linear_softmax_ce_backward_workspace_bytes", N, K, V)
    for K in (1, 64, 1024):
        sizes = [q(K, V) for V in (10_000_000, 100_000_000, 1 << 30)]
        assert max(sizes) < 1 << 30, (K, sizes)
        assert max(sizes) - min(sizes) < 64 << 20, (K, sizes)  # pieces of equal size, up to a tile
    assert q(1024, 1_000_000) < 1 << 30
