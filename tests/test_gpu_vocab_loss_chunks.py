"""The vocabulary loss over chunks of tokens of which the last, shorter one needs more scratch than the others."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import cann_hccl_b200 as H  # noqa: E402
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import vocab  # noqa: E402
from test_gpu_vocab_loss import Exact, problem  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(4)


def bytes_of(T, V, hidden, grad=1):
    return L.lib().HcclB200VocabLossScratchBytes(T, V, hidden, grad)


def test_calls_refuse_too_little_scratch():
    """Before anything is launched: results keep what they held."""
    T, V, hidden = 300, 1000, 64
    x, w, y = problem(T, V, hidden)
    need, step = bytes_of(T, V, hidden), L.lib().HcclB200VocabLossStepBytes(T, V, hidden)
    mem, words = torch.empty(step + 256, device="cuda", dtype=torch.uint8), torch.full((3, T), 7.0, device="cuda")
    dx, dw = torch.full((T, hidden), 7.0, device="cuda", dtype=torch.bfloat16), torch.full((V, hidden), 7.0, device="cuda", dtype=torch.bfloat16)
    lse, target, losses = [t.data_ptr() for t in words]
    lib, at, st = L.lib(), mem.data_ptr(), torch.cuda.current_stream().cuda_stream

    def call(scratch):
        return L.VocabLoss(x.data_ptr(), w.data_ptr(), hidden, hidden, y.data_ptr(), None, T, V, 0, V, -100, hidden, L.INT64, scratch)
    for entry, size in (("Scores", need), ("Grad", need), ("Step", step)):
        for scratch, want in ((size - 1, L.E_PARA), (1, L.E_PARA), (-1, L.E_PARA), (size, L.SUCCESS), (0, L.SUCCESS)):
            before = [t.clone() for t in (words, dx, dw)]
            p = call(scratch)
            rc = {"Scores": lambda: lib.HcclB200VocabLossScores(C.byref(p), 1, lse, target, losses, at, st),
                  "Grad": lambda: lib.HcclB200VocabLossGrad(C.byref(p), lse, target, None, 1.0, dx.data_ptr(), dw.data_ptr(), None, 0, at, st),
                  "Step": lambda: lib.HcclB200VocabLossStep(C.byref(p), 0, 1.0, losses, dx.data_ptr(), dw.data_ptr(), None, 0, at, st)}[entry]()
            assert rc == want, (entry, scratch)
            torch.cuda.synchronize()
            assert want == L.SUCCESS or all(torch.equal(a, b) for a, b in zip(before, (words, dx, dw)))
    # unequal answers of one rule: less tokens, more bytes
    assert bytes_of(388, 2000, 1024) > bytes_of(512, 2000, 1024)


@pytest.mark.parametrize("T,V,hidden,chunk", [(512 + 388, 2000, 1024, 512), (2 * 512 + 462, 2000, 1024, 512), (1024 + 795, 2000, 512, 1024), (2048 + 1905, 2000, 256, 2048)])
def test_short_chunks_of_more_shares(T, V, hidden, chunk, monkeypatch):
    assert bytes_of(T % chunk, V, hidden) > bytes_of(chunk, V, hidden)
    x, w, y = problem(T, V, hidden)
    weights = torch.rand(T, device="cuda")
    monkeypatch.setattr(L.lib(), "HcclB200VocabLossChunk", lambda v, g: chunk)
    e = Exact(x, w, y, weights)
    e.check(vocab.linear_cross_entropy_grad(x, w, y, weights))
    acc = torch.zeros(V, hidden, device="cuda")
    e.check(vocab.linear_cross_entropy_grad(x, w, y, weights, dw=acc), torch.float32)


def test_two_chunks_as_they_come(monkeypatch):
    """Chunks of the library's own size give what calls of their own give, to the bit (calls by parts: the whole step in one call adds a
    token's sums in another order)."""
    monkeypatch.setattr(vocab, "_STEP_MOST", 0)
    V, hidden = 50257, 768
    chunk = L.lib().HcclB200VocabLossChunk(V, 1)
    rest = max(range(chunk - 1, 0, -131), key=lambda t: bytes_of(t, V, hidden))
    assert bytes_of(rest, V, hidden) > bytes_of(chunk, V, hidden)
    x, w, y = problem(chunk + rest, V, hidden)
    guard = torch.full((1 << 26,), 3, device="cuda", dtype=torch.int32)       # memory that the allocator may place behind the scratch
    loss, dx, dw = vocab.linear_cross_entropy_grad(x, w, y, reduction="sum")
    acc, losses = torch.zeros(V, hidden, device="cuda"), []
    for a, b in ((0, chunk), (chunk, chunk + rest)):
        l, d, _ = vocab.linear_cross_entropy_grad(x[a:b], w, y[a:b], reduction="sum", dw=acc)
        assert torch.equal(d, dx[a:b])
        losses.append(float(l))
    assert torch.equal(acc.to(torch.bfloat16), dw) and bool((guard == 3).all())
    # the same fp32 sums of `chunk + rest` losses in another order
    assert abs(float(loss) - sum(losses)) <= 2.0 ** -24 * (2 * (chunk + rest) / 256 + 32) * sum(losses)


@pytest.mark.parametrize("p,chunk", [(2, 128), (3, 256)])
def test_chunks_over_shards(p, chunk, monkeypatch):
    """Several chunks of tokens, each exchanged between the ranks; the last one short."""
    cfg = L.CommConfig.default()
    cfg.hcclBufferSize = 2
    c = H.Communicator.init_local(p, device=True, device_id=0, config=cfg)
    T, V, hidden = 2 * chunk + 131, 700 * p, 1096
    x, w, y = problem(T, V, hidden)
    weights = torch.rand(T, device="cuda")
    weights[::7] = 0
    monkeypatch.setattr(L.lib(), "HcclB200VocabLossChunk", lambda v, g: chunk)
    e = Exact(x, w, y, weights)
    shards = [s.contiguous() for s in w.chunk(p)]
    args = (c, [x] * p, shards, [y] * p, [weights] * p)
    out = vocab.vocab_parallel_cross_entropy_grad(*args)
    acc = [torch.zeros(700, hidden, device="cuda") for _ in range(p)]
    added = vocab.vocab_parallel_cross_entropy_grad(*args, dw=acc)
    losses = vocab.vocab_parallel_cross_entropy(*args, reduction="none")
    assert c.sync() == 0, c.describe_status()
    e.check((out[0][0], out[0][1], torch.cat([o[2] for o in out])), parts=p)
    e.check((added[0][0], added[0][1], torch.cat(acc)), torch.float32, parts=p)
    for r in range(p):
        e.check_losses(losses[r])
        assert torch.equal(out[r][0], out[0][0]) and torch.equal(out[r][1], out[0][1])
    c.destroy()
