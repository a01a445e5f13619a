"""Calls of the operators around the layers from several threads at once, of sizes that need different amounts of shared memory."""
import threading

import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200.parallel import moe, vocab  # noqa: E402

pytestmark = pytest.mark.gpu


def at_once(calls, rounds):
    """Every call in a thread of its own, with a stream of its own, over and over; the first results, compared with each later one."""
    errors, start = [], threading.Barrier(len(calls))

    def work(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                want = call()
                start.wait()
                for i in range(rounds):
                    got = call()
                    if i % 50 == 0:
                        assert all(torch.equal(a, b) for a, b in zip(got, want))
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:  # a thread's error is the test's
            errors.append(e)
            start.abort()
    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(6)


def test_embedding_gradient():
    """Up to 4096 tokens one kernel sorts, with four bytes of shared memory more for each."""
    def call(T):
        ids, dy = torch.randint(0, 100, (T,), device="cuda"), torch.randn(T, 8, device="cuda")
        torch.cuda.synchronize()
        return lambda: (vocab.embedding_grad(ids, dy, 100),)
    at_once([call(T) for T in (4096, 1, 4090, 700)], 1500)


@pytest.mark.parametrize("sizes", [(512, 257, 300, 400), (1024, 513, 600, 900), (4096, 2049, 2100, 3000)])
def test_router(sizes):
    """One kernel for a range of expert counts."""
    def call(E):
        l = torch.randn(64, E, device="cuda")
        torch.cuda.synchronize()
        return lambda: tuple(moe.gate(l, 4))
    at_once([call(E) for E in sizes], 1500)


@pytest.mark.parametrize("sizes", [(4096, 2049, 2100, 3000)])
def test_router_gradient(sizes):
    def call(E):
        l = torch.randn(64, E, device="cuda")
        g = moe.gate(l, 4)
        torch.cuda.synchronize()
        return lambda: (moe.gate_grad(l, g, None, 1.0),)
    at_once([call(E) for E in sizes], 1500)
