"""What linear_cross_entropy refuses, without a GPU: Python's checks and the C entries' own, which launch nothing."""
import ctypes

import pytest
import torch


def test_python_refusals():
    from recommender_amd import ops
    x, w, t = torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_cross_entropy_grad(x, w, t)
    with pytest.raises(ValueError, match="reduction"):
        ops.linear_cross_entropy(x, w, t, reduction="batchmean")
    with pytest.raises(TypeError, match="ignore_index"):
        ops.linear_cross_entropy(x, w, t, ignore_index=None)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.linear_cross_entropy([[0.0]], w, t)


def test_c_refusals():
    from recommender_amd import _lib
    L = _lib.lib()
    some = ctypes.c_void_p(256)                              # never read: every call below is refused before a launch
    ok = dict(x=some, ldx=8, w=some, ldw=8, bias=None, dtype=0, T=4, V=9, D=8, target=some, reduction=1, loss=some, state=some, unit=some, dloss=some, dx=some,
              dw=some, db=None, ws=some)
    need = L.reco_linear_xent_workspace_bytes(some, 8, some, 8, 0, 4, 9, 8, 1)
    need_grad = L.reco_linear_xent_grad_workspace_bytes(some, 8, some, 8, 0, 4, 9, 8)
    assert need > 0 and need_grad > 0

    def forward(nbytes=need, **k):
        a = {**ok, **k}
        return L.reco_linear_xent(a["x"], a["ldx"], a["w"], a["ldw"], a["bias"], a["dtype"], a["T"], a["V"], a["D"], a["target"], -100, a["reduction"],
                                  a["loss"], a["state"], a["unit"], None, a["ws"], nbytes, None)

    def grad(nbytes=need_grad, **k):
        a = {**ok, **k}
        return L.reco_linear_xent_grad(a["x"], a["ldx"], a["w"], a["ldw"], a["bias"], a["dtype"], a["T"], a["V"], a["D"], a["target"], -100, a["reduction"],
                                       a["state"], a["unit"], a["dloss"], a["dx"], a["dw"], a["db"], a["ws"], nbytes, None)
    shared = [dict(x=None), dict(w=None), dict(target=None), dict(state=None), dict(ws=None), dict(ws=ctypes.c_void_p(8)), dict(T=0), dict(T=2 ** 31), dict(V=0),
              dict(V=2 ** 31), dict(D=0), dict(D=2 ** 20 + 1, ldx=2 ** 21, ldw=2 ** 21), dict(ldx=7), dict(ldw=7), dict(dtype=3), dict(dtype=-1),
              dict(reduction=3), dict(reduction=-1)]
    for k in shared + [dict(loss=None)]:
        assert forward(**k) == _lib.EINVAL, k
    for k in shared + [dict(dloss=None), dict(unit=None)]:
        assert grad(**k) == _lib.EINVAL, k
    assert forward(nbytes=need - 1) == _lib.ENOMEM and grad(nbytes=need_grad - 1) == _lib.ENOMEM
    assert grad(dx=None, dw=None, db=None) == _lib.OK         # nothing wanted, nothing launched


def test_workspace_does_not_hold_the_logits():
    from recommender_amd import _lib
    L = _lib.lib()
    some = ctypes.c_void_p(256)
    T, V, D = 8192, 100003, 128
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        assert L.reco_linear_xent_workspace_bytes(some, D, some, D, dtype, T, V, D, 1) < T * V * size // 8
        assert L.reco_linear_xent_grad_workspace_bytes(some, D, some, D, dtype, T, V, D) < T * V * size // 2
    aligned = L.reco_linear_xent_workspace_bytes(some, D, some, D, 1, T, V, D, 0)
    assert L.reco_linear_xent_workspace_bytes(ctypes.c_void_p(258), D, some, D, 1, T, V, D, 0) >= aligned + 2 * T * D       # a copy of x
    assert L.reco_linear_xent_workspace_bytes(some, D, some, D + 1, 1, T, V, D, 0) >= aligned + 2 * V * D                  # a copy of w


def test_what_is_kept_for_the_gradient():
    from recommender_amd import _lib
    kept = _lib.lib().reco_linear_xent_kept_floats
    assert kept(0, 70, 900, 128, 1) == 70 * 128 and kept(0, 70, 900, 128, 0) == 0                 # narrow rows: dx
    assert kept(1, 70, 900, 256, 1) == 70 * 256
    assert kept(0, 70, 900, 129, 1) == kept(0, 70, 900, 129, 0) == 128 * 1024                     # the logits, in whole tiles
    assert kept(1, 70, 900, 257, 1) == kept(2, 70, 900, 600, 1) == 0
    assert kept(0, 16384, 8192, 300, 1) == 2 ** 27 and kept(0, 16384, 8193, 300, 1) == kept(0, 16385, 8192, 300, 1) == 0
    assert kept(0, 2 ** 31 - 1, 2 ** 31 - 1, 300, 1) == 0 and kept(3, 70, 900, 8, 1) == kept(0, 0, 900, 8, 1) == 0
    some = ctypes.c_void_p(256)
    assert _lib.lib().reco_linear_xent(some, 200, some, 200, None, 0, 4, 9, 200, some, -100, 1, some, some, ctypes.c_void_p(264), None, some, 1 << 30,
                                       None) == _lib.EINVAL
    assert _lib.lib().reco_linear_xent_grad(some, 200, some, 200, None, 0, 4, 9, 200, some, -100, 1, some, ctypes.c_void_p(264), some, some, some, None, some,
                                            1 << 30, None) == _lib.EINVAL


def test_the_last_piece_of_the_vocabulary_has_room():
    """Fewer units of work can mean shorter shares and more workgroups, each of which has two places of 128 x 128 sums."""
    from recommender_amd import _lib
    L = _lib.lib()
    some = ctypes.c_void_p(256)
    # 600 columns: 5 x 3 tiles of dw with 57 steps each are 855 units, 2 to each of 428 workgroups (768 would be 1026, 3 to each of 342)
    T, V, D = 7296, 600, 384
    assert L.reco_linear_xent_grad_workspace_bytes(some, D, some, D, 0, T, V, D) >= 428 * 2 * 128 * 128 * 4 + T * V * 4 + T * D * 4


def test_a_tangent_is_refused():
    from torch.autograd import forward_ad
    from recommender_amd import ops
    x = torch.zeros(2, 3)
    ops._no_tangent(x, "input")
    with forward_ad.dual_level():
        ops._no_tangent(x, "input")
        for t in (forward_ad.make_dual(x, x), 2 * forward_ad.make_dual(x, x)):
            with pytest.raises(NotImplementedError, match="input.*forward"):
                ops._no_tangent(t, "input")
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            ops._no_tangent(forward_ad.make_dual(x, x), "input")


def test_ignore_index_fits_a_target():
    """A longer one would be cut to its low 64 bits on its way into the library, and could name a column."""
    from recommender_amd import ops
    x, w, t = torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=torch.int64)
    for call in (ops.linear_cross_entropy, ops.linear_cross_entropy_grad):
        for bad in (2 ** 64 + 5, 2 ** 63, -2 ** 63 - 1):
            with pytest.raises(ValueError, match="ignore_index"):
                call(x, w, t, ignore_index=bad)
        for good in (2 ** 63 - 1, -2 ** 63):
            with pytest.raises(ValueError, match="GPU"):
                call(x, w, t, ignore_index=good)
