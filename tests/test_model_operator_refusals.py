"""What the embedding and the router refuse on the host, before anything is launched."""
import ctypes as C

import pytest

from cann_hccl_b200 import _lib as L

MEM = C.create_string_buffer(4096)
AT = (C.addressof(MEM) + 63) // 64 * 64


def embed(grad=False, ids=AT, id_type=L.INT64, tokens=4, rows=AT, stride=8, vocab=16, first=0, hidden=8, dtype=L.BFP16, out=AT, out_type=None, add=0, scratch=AT):
    lib = L.lib()
    if not grad:
        return lib.HcclB200Embedding(ids, id_type, tokens, rows, stride, vocab, first, hidden, dtype, 1.0, out, None)
    return lib.HcclB200EmbeddingGrad(ids, id_type, tokens, rows, stride, vocab, first, hidden, dtype, 1.0, out, dtype if out_type is None else out_type, add,
                                     scratch, None)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("bad,want", [({"ids": None}, "PTR"), ({"rows": None}, "PTR"), ({"out": None}, "PTR"), ({"id_type": L.FP32}, "NOT_SUPPORT"),
                                      ({"dtype": L.INT32}, "NOT_SUPPORT"), ({"dtype": L.FP64}, "NOT_SUPPORT"), ({"tokens": -1}, "PARA"), ({"tokens": 1 << 31}, "PARA"),
                                      ({"vocab": 0}, "PARA"), ({"vocab": (1 << 31) - 1}, "PARA"), ({"hidden": 0}, "PARA"), ({"first": -1}, "PARA"),
                                      ({"stride": 7}, "PARA"), ({"ids": AT + 4}, "PARA"), ({"rows": AT + 1}, "PARA"), ({"out": AT + 1}, "PARA")])
def test_embedding(grad, bad, want):
    assert embed(grad, **bad) == getattr(L, "E_" + want)


def test_embedding_gradient():
    assert embed(True, scratch=None) == L.E_PTR
    assert embed(True, scratch=AT + 8) == L.E_PARA
    assert embed(True, out_type=L.FP32) == L.E_NOT_SUPPORT                 # fp32 sums are added to, or the rows are fp32
    assert embed(True, add=1) == L.E_NOT_SUPPORT
    assert embed(True, add=1, out_type=L.FP32, out=AT + 2) == L.E_PARA
    lib = L.lib()
    assert lib.HcclB200EmbeddingGradScratchBytes(-1, 10, 8) == -1 and lib.HcclB200EmbeddingGradScratchBytes(10, 0, 8) == -1
    assert lib.HcclB200EmbeddingGradScratchBytes(10, 10, 0) == -1 and lib.HcclB200EmbeddingGradScratchBytes(0, 10, 8) > 0
    assert embed(False, tokens=0, ids=None, out=None) == L.SUCCESS
    assert embed(True, tokens=(1 << 24) + 1) == L.E_PARA and lib.HcclB200EmbeddingGradScratchBytes((1 << 24) + 1, 10, 8) == -1


def gate(grad=False, logits=AT, dtype=L.FP32, tokens=4, experts=8, stride=8, topk=2, idx=AT, gates=AT, counts=AT, prob=AT, routed=AT, balance=AT, scratch=AT,
         d_gates=None, out=AT):
    lib = L.lib()
    if not grad:
        return lib.HcclB200MoeGate(logits, dtype, tokens, experts, stride, topk, 1, None, idx, gates, counts, prob, routed, balance, scratch, None)
    return lib.HcclB200MoeGateGrad(logits, dtype, tokens, experts, stride, topk, 1, None, idx, d_gates, counts, routed, 0.0, out, None)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("bad,want", [({"logits": None}, "PTR"), ({"idx": None}, "PTR"), ({"counts": None}, "PTR"), ({"routed": None}, "PTR"),
                                      ({"dtype": L.INT32}, "NOT_SUPPORT"), ({"experts": 4097, "stride": 4097}, "NOT_SUPPORT"), ({"experts": 64, "stride": 64, "topk": 33}, "NOT_SUPPORT"),
                                      ({"topk": 9}, "PARA"), ({"topk": 0}, "PARA"), ({"experts": 0}, "PARA"), ({"tokens": -1}, "PARA"), ({"stride": 7}, "PARA"),
                                      ({"logits": AT + 2}, "PARA"), ({"idx": AT + 2}, "PARA"), ({"counts": AT + 1}, "PARA")])
def test_gate(grad, bad, want):
    assert gate(grad, **bad) == getattr(L, "E_" + want)


def test_gate_outputs():
    for name in ("gates", "prob", "balance"):
        assert gate(**{name: None}) == L.E_PTR and gate(**{name: AT + 2}) == L.E_PARA, name
    assert gate(scratch=AT + 2) == L.E_PARA and gate(scratch=None, tokens=1000) == L.E_PTR   # a decode batch needs none
    assert gate(True, out=None) == L.E_PTR and gate(True, out=AT + 2) == L.E_PARA and gate(True, d_gates=AT + 2) == L.E_PARA
    lib = L.lib()
    assert lib.HcclB200MoeBalance(None, AT, AT, 8, 2, AT, None) == L.E_PTR and lib.HcclB200MoeBalance(AT, AT, AT, 8, 9, AT, None) == L.E_PARA
    assert lib.HcclB200MoeGateScratchBytes(4, 0) == -1 and lib.HcclB200MoeGateScratchBytes(4, 5000) == -1 and lib.HcclB200MoeGateScratchBytes(0, 8) == 0
    assert lib.HcclB200MoeGateScratchBytes(1000, 8) > 0


def loss(entry="Scores", args=None, **bad):
    """The entry of a loss call whose structure has the fields `bad`, whose pointers after it those of `args`."""
    d = dict(x=AT, w=AT, xStride=8, wStride=8, targets=AT, weights=None, tokens=4, vocab=16, firstId=0, wholeVocab=16, ignoreId=-100, hidden=8, targetType=L.INT64)
    d.update(bad)
    p = C.byref(L.VocabLoss(**d))
    a = dict(lse=AT, target=AT, losses=AT, scratch=AT0, parts=AT, shards=2, total=AT, loss=AT, dx=AT, dw=AT, sum=AT, kind=0)
    a.update(args or {})
    lib = L.lib()
    return {"Scores": lambda: lib.HcclB200VocabLossScores(p, 1, a["lse"], a["target"], a["losses"], a["scratch"], None),
            "Combine": lambda: lib.HcclB200VocabLossCombine(p, a["parts"], a["shards"], a["lse"], a["losses"], None),
            "Total": lambda: lib.HcclB200VocabLossTotal(p, a["total"], None),
            "Step": lambda: lib.HcclB200VocabLossStep(p, 1, 1.0, a["loss"], a["dx"], a["dw"], a["sum"], a["kind"], a["scratch"], None),
            "Sum": lambda: lib.HcclB200VocabLossSum(p, a["losses"], a["total"], a["loss"], None),
            "Grad": lambda: lib.HcclB200VocabLossGrad(p, a["lse"], a["target"], a["total"], 1.0, a["dx"], a["dw"], a["sum"], a["kind"], a["scratch"], None)}[entry]()


AT0 = (C.addressof(MEM) + 255) // 256 * 256


@pytest.mark.parametrize("entry", ["Scores", "Grad", "Step"])
@pytest.mark.parametrize("bad,want", [({"x": None}, "PTR"), ({"w": None}, "PTR"), ({"targets": None}, "PTR"), ({"targetType": L.FP32}, "NOT_SUPPORT"),
                                      ({"hidden": 12}, "PARA"), ({"hidden": 0}, "PARA"), ({"hidden": 16}, "PARA"), ({"xStride": 12}, "PARA"), ({"wStride": 0}, "PARA"),
                                      ({"vocab": 0}, "PARA"), ({"vocab": 17}, "PARA"), ({"firstId": 1}, "PARA"), ({"firstId": -1}, "PARA"), ({"wholeVocab": 15}, "PARA"),
                                      ({"tokens": -1}, "PARA"), ({"tokens": (1 << 20) + 1}, "PARA"), ({"x": AT + 8}, "PARA"), ({"w": AT + 2}, "PARA"),
                                      ({"targets": AT + 4}, "PARA"), ({"weights": AT + 2}, "PARA")])
def test_vocab_loss(entry, bad, want):
    assert loss(entry, **bad) == getattr(L, "E_" + want)


def test_vocab_loss_outputs():
    assert loss("Scores", vocab=8) == L.E_PARA                              # a shard has no losses of its own
    for entry, names in (("Scores", ("lse", "target", "scratch")), ("Combine", ("parts", "lse", "losses")), ("Total", ("total",)), ("Sum", ("losses", "loss")),
                         ("Grad", ("lse", "target", "dx", "dw", "scratch")), ("Step", ("loss", "dx", "dw", "scratch"))):
        for n in names:
            assert loss(entry, {n: None}) == L.E_PTR and loss(entry, {n: AT0 + 2}) == L.E_PARA, (entry, n)
    assert loss("Grad", {"scratch": AT0 + 128}) == L.E_PARA and loss("Combine", {"shards": 0}) == L.E_PARA and loss("Grad", tokens=0) == L.E_PARA
    assert loss("Grad", {"kind": 4}) == L.E_PARA and loss("Grad", {"kind": -1}) == L.E_PARA
    assert loss("Step", tokens=65537) == L.E_PARA and loss("Step", vocab=8) == L.E_PARA and loss("Step", tokens=0) == L.E_PARA
    for entry in ("Grad", "Step"):
        for kind in (1, 2, 3):
            assert loss(entry, {"kind": kind, "sum": None}) == L.E_PTR
        assert loss(entry, {"kind": 3, "dw": None}) == L.E_PTR and loss(entry, {"kind": 4}) == L.E_PARA and loss(entry, {"scratch": AT0 + 128}) == L.E_PARA
    assert loss("Scores", tokens=0, x=None, targets=None) == L.SUCCESS and loss("Combine", tokens=0, targets=None) == L.SUCCESS
    lib = L.lib()
    assert lib.HcclB200VocabLossScores(None, 0, AT, AT, None, AT0, None) == L.E_PTR
    assert lib.HcclB200VocabLossChunk(0, 1) == -1 and lib.HcclB200VocabLossChunk(1 << 31, 1) == -1
    for vocab in (1, 1000, 128256, 1 << 24):
        for grad in (0, 1):
            assert lib.HcclB200VocabLossChunk(vocab, grad) >= 256 and lib.HcclB200VocabLossChunk(vocab, grad) % 256 == 0
    assert lib.HcclB200VocabLossStepBytes(0, 16, 8) == -1 and lib.HcclB200VocabLossStepBytes(65537, 16, 8) == -1 and lib.HcclB200VocabLossStepBytes(4, 16, 12) == -1
    assert lib.HcclB200VocabLossScratchBytes(4, 16, 12, 1) == -1 and lib.HcclB200VocabLossScratchBytes((1 << 20) + 1, 16, 8, 1) == -1


def test_python_arguments():
    torch = pytest.importorskip("torch")
    from cann_hccl_b200.parallel import moe, vocab
    w, ids = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)        # host tensors are refused whatever they hold
    for call in (lambda: vocab.embedding(ids, w), lambda: vocab.embedding_grad(ids, torch.zeros(3, 8), 10), lambda: vocab.embedding_grad(ids, torch.zeros(4, 8), 10),
                 lambda: moe.gate(torch.zeros(4, 8), 2), lambda: moe.gate(None, 2),
                 lambda: vocab.linear_cross_entropy(torch.zeros(3, 8), w, ids), lambda: vocab.linear_cross_entropy_grad(torch.zeros(3, 8), w, ids)):
        with pytest.raises(ValueError):
            call()
