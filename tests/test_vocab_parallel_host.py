"""Host side of the vocabulary-parallel operators for one rank per process: which shard, which exchange, in which order.  The library's
launches are stood in for by functions that write down their arguments."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import vocab  # noqa: E402


class Comm:
    nranks, nlocal = 4, 1

    def __init__(self, rank, log):
        self.rank, self.log = rank, log

    def all_gather(self, send, recv):
        self.log.append(("all_gather", send[0].numel(), tuple(recv[0].shape)))

    def all_reduce(self, send, recv):
        assert send[0] is recv[0]
        self.log.append(("all_reduce", tuple(send[0].shape), send[0].dtype))


class Lib:
    def __init__(self, log, chunk):
        self.log, self.chunk = log, chunk

    def HcclB200VocabLossChunk(self, v, grad):
        return self.chunk

    def HcclB200VocabLossScratchBytes(self, tokens, v, h, grad):
        return 1000

    def __getattr__(self, name):
        def call(p, *a):
            s = C.cast(p, C.POINTER(L.VocabLoss)).contents
            self.log.append((name.replace("HcclB200VocabLoss", ""), s.tokens, s.firstId, s.vocab, s.wholeVocab, s.targets, a))
            return 0
        return call


@pytest.fixture
def host(monkeypatch):
    log = []
    monkeypatch.setattr(vocab, "_check_loss", lambda *a: None)
    monkeypatch.setattr(vocab, "on_device_of", lambda t: __import__("contextlib").nullcontext())
    monkeypatch.setattr(vocab, "_raw_stream", lambda: 0)
    lib = Lib(log, 8)
    monkeypatch.setattr(vocab.L, "lib", lambda: lib)
    return log


def tensors(T=20, V=6, hidden=16):
    return torch.zeros(T, hidden, dtype=torch.bfloat16), torch.zeros(V, hidden, dtype=torch.bfloat16), torch.zeros(T, dtype=torch.int64)


@pytest.mark.parametrize("rank", [0, 3])
def test_a_rank_of_four(host, rank):
    x, w, y = tensors()
    loss, dx, dw = vocab.vocab_parallel_cross_entropy_grad(Comm(rank, host), x, w, y)
    assert dx.shape == x.shape and dw.shape == w.shape and dw.dtype == torch.bfloat16
    names = [e[0] for e in host]
    chunk = ["Scores", "all_gather", "Combine", "Grad"]
    assert names == ["Total"] + chunk * 3 + ["all_reduce", "Sum"]                  # 20 tokens in chunks of 8, 8 and 4
    for e in host:
        if e[0] in ("Scores", "Combine", "Grad", "Total", "Sum"):
            assert e[2:5] == (rank * 6, 6, 24)
    assert [e[1] for e in host if e[0] == "Scores"] == [8, 8, 4] and [e[1:] for e in host if e[0] == "all_gather"] == [(2 * n, (4, 2, n)) for n in (8, 8, 4)]
    assert [e[5] - y.data_ptr() for e in host if e[0] == "Grad"] == [0, 64, 128]
    for e in host:
        if e[0] == "Scores":
            assert e[6][3] is None                                                 # a shard has no losses of its own
        if e[0] == "Combine":
            assert e[6][1] == 4
    assert [e[6][7] for e in host if e[0] == "Grad"] == [1, 2, 3]                  # fp32 sum written, added to, added to and rounded
    lse = [e[6][0] for e in host if e[0] == "Grad"]
    assert lse == [e[6][2] for e in host if e[0] == "Combine"]                      # the joint one, not the shard's
    assert host[-2][1:] == ((20, 16), torch.bfloat16)


def test_sums_given_by_the_caller(host):
    x, w, y = tensors()
    acc = torch.zeros(6, 16)
    assert vocab.vocab_parallel_cross_entropy_grad(Comm(1, host), x, w, y, reduction="sum", dw=acc)[2] is acc
    assert [e[6][7] for e in host if e[0] == "Grad"] == [2, 2, 2] and "Total" not in [e[0] for e in host]
    assert all(e[6][6] == acc.data_ptr() for e in host if e[0] == "Grad")


def test_losses_without_gradients(host):
    x, w, y = tensors(5)
    out = vocab.vocab_parallel_cross_entropy(Comm(2, host), x, w, y, reduction="none")
    assert out.shape == (5,) and [e[0] for e in host] == ["Scores", "all_gather", "Combine"]


def test_no_tokens_exchange_nothing(host):
    x, w, y = tensors(0)
    loss, dx, dw = vocab.vocab_parallel_cross_entropy_grad(Comm(1, host), x, w, y)
    assert [e[0] for e in host] == ["Total", "Sum"] and dx.shape == (0, 16) and not bool(dw.any())


def test_arguments_of_ranks():
    x, w, y = tensors()

    class Two:
        nranks = nlocal = 2
        rank = 0
    with pytest.raises(ValueError):
        vocab.vocab_parallel_cross_entropy(Two(), [x], [w, w], [y, y])
    with pytest.raises(ValueError):
        vocab.vocab_parallel_embedding(Two(), [y], [w])
    assert vocab.first_ids(Two(), 7) == [0, 7]
    assert np.array_equal(vocab.first_ids(type("C", (), {"nlocal": 1, "rank": 3, "nranks": 4})(), 5), [15])
