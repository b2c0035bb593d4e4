"""What the output-layer loss and the orthogonalised update refuse before anything reaches the device, and their workspace
queries. None of this needs a GPU: a refused call must not look at one."""
import ctypes

import pytest

from origindl_amd import _lib

OK, BAD = _lib.ODL_OK, _lib.ODL_ERR_INVALID_ARG
SOME = ctypes.c_void_p(256)  # never dereferenced: the calls below are refused or empty
COEF = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def l():
    return _lib.lib()


def forward(l, N=4, K=8, V=16, x=SOME, w=SOME, b=None, t=SOME, saved=SOME, rows=SOME, ws=SOME, nb=None):
    nb = l.query("odl_hip_linear_softmax_ce_forward_workspace_bytes", N, K, V) if nb is None else nb
    return l.cdll.odl_hip_linear_softmax_ce_forward(x, w, 0, b, t, 1, -100, N, K, V, saved, rows, ws, nb, None)


def backward(l, N=4, K=8, V=16, x=SOME, w=SOME, t=SOME, saved=SOME, rows=SOME, gx=SOME, gw=SOME, gb=SOME, ws=SOME, nb=None):
    nb = l.query("odl_hip_linear_softmax_ce_backward_workspace_bytes", N, K, V) if nb is None else nb
    return l.cdll.odl_hip_linear_softmax_ce_backward(None, x, w, 0, None, t, 1, -100, N, K, V, saved, rows, gx, gw, gb, ws, nb, None)


@pytest.mark.parametrize("call", [forward, backward])
def test_output_layer_refuses_bad_arguments(l, call):
    for sizes in ({"N": -1}, {"K": 0}, {"V": 0}, {"V": -5}, {"N": (1 << 20) + 1}, {"K": (1 << 20) + 1}, {"V": (1 << 30) + 1}):
        assert call(l, nb=1 << 40, **sizes) == BAD, sizes
        assert any(k in l.last_error() for k in ("needs", "up to")), l.last_error()
    for null in ("x", "w", "t", "saved", "rows"):
        assert call(l, **{null: None}) == BAD, null
        assert "null" in l.last_error()
    assert call(l, ws=None) == BAD and "workspace" in l.last_error()
    assert call(l, nb=64) == BAD and "workspace" in l.last_error()
    assert call(l, ws=ctypes.c_void_p(260)) == BAD and "aligned" in l.last_error()


def test_output_layer_backward_without_outputs_does_nothing(l):
    assert backward(l, gx=None, gw=None, gb=None) == OK


def test_output_layer_workspaces_are_bounded(l):
    """The vocabulary goes through in pieces: the workspace does not grow with V beyond the partial maxima and sums."""
    for which, per_entry in (("forward", 8 * 8192 / 64 + 4), ("backward", 0)):
        q = lambda N, K, V: l.query("odl_hip_linear_softmax_ce_%s_workspace_bytes" % which, N, K, V)
        assert q(0, 8, 8) == 0 and q(8, 0, 8) == 0 and q(8, 8, -1) == 0
        assert 0 < q(1, 1, 1) < 1 << 20
        assert q(8192, 2048, 128000) < 3 << 30
        assert q(8192, 2048, 512000) - q(8192, 2048, 128000) <= per_entry * 384000 + (64 << 20)


def test_row_statistics_hold_logits_only_where_they_are_small(l):
    q = lambda N, K, V: l.query("odl_hip_linear_softmax_ce_row_stats_floats", N, K, V)
    assert q(0, 8, 8) == q(4, 0, 8) == q(4, 8, -1) == 0
    assert q(4, 8, 16) == 8 and q(4096, 1024, 32000) == 8192  # small weights; many rows
    assert q(256, 515, 12007) == 512                          # few rows whose logits are half the weights
    for N, K, V in ((1, 2048, 32000), (7, 129, 50003), (64, 2000, 4001), (128, 1031, 60021), (256, 1024, 100000)):
        assert 2 * N + N * V <= q(N, K, V) <= 2 * N + (K * V) // 4 + 128 * 256, (N, K, V)


def schulz(l, batch=1, rows=4, cols=8, steps=5, coef=COEF, eps=1e-7, g=SOME, out=SOME, ws=SOME, nb=None):
    nb = l.query("odl_hip_newton_schulz_workspace_bytes", batch, rows, cols) if nb is None else nb
    return l.cdll.odl_hip_newton_schulz(g, batch, rows, cols, steps, *coef, eps, out, ws, nb, None)


def test_newton_schulz_refuses_bad_arguments(l):
    for bad in ({"batch": -1}, {"rows": -1}, {"cols": -1}, {"rows": (1 << 20) + 1}, {"steps": 0}, {"steps": 101}, {"eps": -1.0},
                {"g": None}, {"out": None}, {"ws": None}, {"nb": 64}, {"ws": ctypes.c_void_p(264)}):
        assert schulz(l, **bad) == BAD, bad
        assert l.last_error()
    nan, inf = float("nan"), float("inf")
    # coefficients that drive singular values, or the polynomial's factor, out of the operands' range; also NaN
    for coef in ((10.0, 0.0, 0.0), (3.4445, -4.775, 20.0), (1.5, -9.0, 0.0), (nan, 0.0, 0.0), (1.0, inf, 0.0)):
        assert schulz(l, coef=coef) == BAD and "coefficients" in l.last_error(), coef
    # the usual ones, the cubic one and the convergent quintic one are taken: the call then stops at its null argument
    for coef in (COEF, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)):
        assert schulz(l, coef=coef, g=None) == BAD and "null" in l.last_error()
    for empty in ({"batch": 0}, {"rows": 0}, {"cols": 0}):
        assert schulz(l, g=None, out=None, ws=None, nb=0, **empty) == OK, empty


def muon(l, shapes, ptr=256, steps=5, coef=COEF, ws=SOME, nb=None, lists=True):
    n = len(shapes)
    rows, cols = (ctypes.c_int64 * max(n, 1))(*[s[0] for s in shapes]), (ctypes.c_int64 * max(n, 1))(*[s[1] for s in shapes])
    ptrs = (ctypes.c_void_p * max(n, 1))(*[ptr] * n) if lists else None
    nb = l.query("odl_hip_muon_step_multi_workspace_bytes", n, rows, cols) if nb is None else nb
    return l.cdll.odl_hip_muon_step_multi(n, ptrs, ptrs, ptrs, rows, cols, 0.02, 0.95, 1, 0.0, steps, *coef, 1e-7, ptrs, ws, nb, None)


def test_muon_step_refuses_bad_arguments(l):
    assert muon(l, []) == OK
    assert muon(l, [(4, 8)], lists=False) == BAD and "null" in l.last_error()
    assert muon(l, [(4, 8)], ptr=None) == BAD and "entry 0" in l.last_error()
    assert muon(l, [(4, 8), (-1, 8)]) == BAD and "sides" in l.last_error()
    assert muon(l, [(4, 8)], steps=0) == BAD and "steps" in l.last_error()
    assert muon(l, [(4, 8)], coef=(10.0, 0.0, 0.0)) == BAD and "coefficients" in l.last_error()
    assert muon(l, [(4, 8)], ws=None) == BAD and "workspace" in l.last_error()
    assert muon(l, [(4, 8)], nb=64) == BAD and "workspace" in l.last_error()
    # one momentum for two matrices (an empty one between them writes nothing)
    assert muon(l, [(4, 8), (0, 8), (8, 4)]) == BAD and "entries 0 and 2" in l.last_error()


def test_muon_workspace_is_that_of_the_largest_group(l):
    q = lambda shapes: l.query("odl_hip_muon_step_multi_workspace_bytes", len(shapes), (ctypes.c_int64 * len(shapes))(*[s[0] for s in shapes]),
                               (ctypes.c_int64 * len(shapes))(*[s[1] for s in shapes]))
    one, two = q([(300, 500)]), q([(300, 500), (300, 500)])
    assert 0 < one < two <= 2 * one
    assert q([(300, 500), (64, 64), (300, 500)]) == two
    assert q([(300, 500)] * 40) == q([(300, 500)] * 32)


def test_a_valid_call_without_a_gpu_is_a_runtime_error(l):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    for rc in (forward(l), forward(l, N=0), backward(l), schulz(l), muon(l, [(4, 8)])):
        assert rc == _lib.ODL_ERR_RUNTIME
