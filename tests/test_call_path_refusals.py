"""Both forms of the Python call path refuse integers where a collective or the expert exchange takes buffers.  The integers are addresses of
memory that is there, so that a call that takes them is seen to."""
import numpy as np
import pytest

import cann_hccl_b200 as H
from cann_hccl_b200 import _calls
from cann_hccl_b200 import _lib as L


@pytest.fixture(params=["extension", "ctypes"])
def path(request, monkeypatch):
    L.lib()
    if request.param == "ctypes":
        calls = _calls.Calls(L.lib())
        from cann_hccl_b200.utils.dtypes import dtype_table
        calls.setup(dtype_table(False), None, None)
        monkeypatch.setattr(L, "fast", calls)
    return L.fast


CALLS = {"all_reduce": lambda c, x, y: c.all_reduce(x, y), "all_gather": lambda c, x, y: c.all_gather(x, y), "reduce_scatter": lambda c, x, y: c.reduce_scatter(x, y),
         "reduce": lambda c, x, y: c.reduce(x, y, 0), "broadcast": lambda c, x, y: c.broadcast(y, 0), "scatter": lambda c, x, y: c.scatter(x, y, 0),
         "gather": lambda c, x, y: c.gather(x, y, 0), "all_to_all": lambda c, x, y: c.all_to_all(x, y),
         "collective": lambda c, x, y: c.collective(L.ALLREDUCE, x, y, 4, L.FP32),
         "all_gather_v": lambda c, x, y: c.all_gather_v(x, y, [4] * c.nranks, [4 * r for r in range(c.nranks)]),
         "reduce_scatter_v": lambda c, x, y: c.reduce_scatter_v(x, y, [4] * c.nranks, [4 * r for r in range(c.nranks)]),
         "all_to_all_v": lambda c, x, y: c.all_to_all_v(x, [[4] * c.nranks] * c.nranks, [[0] * c.nranks] * c.nranks, y, [[4] * c.nranks] * c.nranks, [[0] * c.nranks] * c.nranks)}


@pytest.mark.parametrize("p", [1, 2])
@pytest.mark.parametrize("name", list(CALLS))
def test_collectives(path, name, p):
    c = H.Communicator.init_local(p, device=False)
    good = [np.ones(64, np.float32) for _ in range(p)]
    out = [np.zeros(256, np.float32) for _ in range(p)]
    at = [o.ctypes.data for o in out]
    bad = [at] if p > 1 else [at, at[0]]
    for b in bad:
        with pytest.raises((AttributeError, TypeError)):
            CALLS[name](c, good, b)
        if name != "broadcast":
            with pytest.raises((AttributeError, TypeError)):
                CALLS[name](c, b, out)
    if p > 1:
        with pytest.raises((AttributeError, TypeError)):
            CALLS[name](c, good, [out[0], at[1]])
    assert all((o == 0).all() for o in out)
    assert c.destroy() == L.SUCCESS


def test_exchange(path):
    x = [np.zeros(64, np.float32)]
    at = [x[0].ctypes.data]
    for bad in (at, at[0]):
        for a in ((bad, x), (x, bad)):
            with pytest.raises((AttributeError, TypeError)):
                path.moe_dispatch(0, 1, 0, *a, 0)
        for i in range(3):
            a = [x, x, x]
            a[i] = bad
            with pytest.raises((AttributeError, TypeError)):
                path.moe_combine(0, 1, 0, 0, *a, 0)


def test_operators_around_the_layers(path):
    """Only the parts of a Gate, which have no tensors of their own, are addresses."""
    t = np.zeros(64, np.float32)
    at = t.ctypes.data
    for i in (0, 3, 10):
        a = [t, L.INT64, -1, t, 8, 8, 0, 8, L.FP32, 1.0, t, 0]
        assert path.embedding(*a) == L.E_PARA
        a[i] = at
        with pytest.raises((AttributeError, TypeError)):
            path.embedding(*a)
    for i in (0, 3, 10, 13):
        a = [t, L.INT64, -1, t, 8, 8, 0, 8, L.FP32, 1.0, t, L.FP32, 0, t, 0]
        assert path.embedding_grad(*a) == L.E_PARA
        a[i] = at
        with pytest.raises((AttributeError, TypeError)):
            path.embedding_grad(*a)
    for i in (0, 7, 14):
        a = [t, L.FP32, -1, 8, 8, 2, 1, t, at, at, at, at, at, at, t, 0]
        assert path.gate(*a) == L.E_PARA
        a[i] = at
        with pytest.raises((AttributeError, TypeError)):
            path.gate(*a)
    for i in (0, 7, 9, 13):
        a = [t, L.FP32, -1, 8, 8, 2, 1, t, at, t, at, at, 0.0, t, 0]
        assert path.gate_grad(*a) == L.E_PARA
        a[i] = at
        with pytest.raises((AttributeError, TypeError)):
            path.gate_grad(*a)
