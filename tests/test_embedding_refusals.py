"""What embedding / embedding_grad refuse, without a GPU: Python's checks and the C entries' own, which launch nothing."""
import ctypes

import pytest
import torch


def test_python_refusals(monkeypatch):
    from recommender_amd import ops
    cpu = torch.zeros(4, 3)
    with pytest.raises(ValueError, match="GPU"):
        ops.embedding(torch.tensor([1]), cpu)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.embedding(torch.tensor([1]), [[1.0]])
    with pytest.raises(TypeError, match="number"):
        ops.embedding(torch.tensor([1]), cpu, scale=torch.tensor(2.0))
    with pytest.raises(ValueError, match="GPU"):
        ops.embedding_grad(torch.tensor([1]), cpu, 4)
    # nn.Embedding's rule for padding_idx
    assert ops._padding(None, 5) == -1 and ops._padding(0, 5) == 0 and ops._padding(-1, 5) == 4 and ops._padding(-5, 5) == 0
    for bad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            ops._padding(bad, 5)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        ops._no_captured_graph("embedding", "embedding_grad")


def test_c_refusals():
    from recommender_amd import _lib
    L = _lib.lib()
    some = ctypes.c_void_p(64)                               # never read: every call below is refused before a launch
    ok = dict(table=some, rows=10, ld=4, dim=4, dtype=0, ids=some, n=3, out=some)

    def lookup(**k):
        a = {**ok, **k}
        return L.reco_embedding(a["table"], a["rows"], a["ld"], a["dim"], a["dtype"], a["ids"], a["n"], 1.0, a["out"], None, None)
    for k in (dict(table=None), dict(ids=None), dict(out=None), dict(rows=0), dict(dim=0), dict(ld=3), dict(dtype=3), dict(dtype=-1)):
        assert lookup(**k) == _lib.EINVAL, k
    assert lookup(n=0, table=None) == _lib.OK

    need = L.reco_embedding_grad_workspace_bytes(3, 10, 4)
    assert need > 0 and L.reco_embedding_grad_workspace_bytes(0, 10, 4) == 0
    okg = dict(ids=some, n=3, grad=some, ldg=4, dim=4, dtype=0, rows=10, out=some, ws=some, nbytes=need)

    def grad(**k):
        a = {**okg, **k}
        return L.reco_embedding_grad(a["ids"], a["n"], a["grad"], a["ldg"], a["dim"], a["dtype"], a["rows"], 1.0, -1, a["out"], a["ws"], a["nbytes"], None)
    for k in (dict(ids=None), dict(grad=None), dict(out=None), dict(ws=None), dict(rows=0), dict(rows=2 ** 31 - 1), dict(n=2 ** 31), dict(n=-1), dict(dim=0),
              dict(ldg=3), dict(dtype=7), dict(out=ctypes.c_void_p(72)), dict(ws=ctypes.c_void_p(72))):
        assert grad(**k) == _lib.EINVAL, k
    assert grad(nbytes=need - 1) == _lib.ENOMEM
    with pytest.raises(MemoryError):
        _lib.check(_lib.ENOMEM)


@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (4096, 6038, 64), (4097, 6038, 64), (10 ** 6, 10 ** 6, 128), (2 ** 31 - 1, 2 ** 31 - 2, 512)])
def test_workspace_holds_both_lists_and_the_partial_rows(n, rows, dim):
    from recommender_amd import _lib
    got = _lib.lib().reco_embedding_grad_workspace_bytes(n, rows, dim)
    assert got >= 8 * n + 2 * 4 * dim * (n // 128)


def test_whole_numbers_are_asked_for():
    from recommender_amd import ops
    for bad in (1.0, 0.5, "1", torch.tensor([1, 2])):
        with pytest.raises(TypeError):
            ops._padding(bad, 4)
    assert ops._padding(torch.tensor(3), 4) == 3
    with pytest.raises(TypeError):
        ops.embedding_grad(torch.zeros(2, dtype=torch.int64), torch.zeros(2, 3), 4.5)


def test_rows_too_wide_for_the_library_are_refused():
    """Refused before anything is allocated (the wide row here is one value, expanded): its width would be cut to 32 bits."""
    from recommender_amd import ops
    wide = torch.zeros(1, 1).expand(1, 2 ** 31 + 8)
    with pytest.raises(ValueError, match="2147483656"):
        ops._embedding(torch.zeros(1, dtype=torch.int64), wide, 1.0, False)
    with pytest.raises(ValueError, match="2147483656"):
        ops._embedding_grad(torch.zeros(1, dtype=torch.int64), wide, 4, 1.0, -1)
    assert ops._width(2 ** 31 - 1) == 2 ** 31 - 1
