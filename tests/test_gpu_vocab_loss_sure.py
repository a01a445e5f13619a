"""Gradients of guesses that are all but sure, at logits of 20 to 40: the target's column of d is minus the probability of everything else,
which the sum of two fp32 numbers that size would lose."""
import pytest

torch = pytest.importorskip("torch")
import cann_hccl_b200 as H  # noqa: E402
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import vocab  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(9)


def problem(T, V):
    """Token t has a column t of its own, in which its target has weight 1 and one other id a weight below: two logits that count, a and a - gap,
    which any sum gives exactly; all others are below -4 a.  Returns x, w, targets, the other ids, a and the gaps."""
    hidden = (T + 7) // 8 * 8
    ids = torch.randperm(V, device="cuda")
    y, c = ids[:T], ids[T:2 * T]
    a = (torch.randint(80, 160, (T,), device="cuda") / 4).to(torch.bfloat16)
    want = 9.0 + 5.0 * torch.rand(T, device="cuda")                   # losses of e^-9 to e^-14
    b = (1 - want / a.float()).to(torch.bfloat16)
    t = torch.arange(T, device="cuda")
    x = torch.zeros(T, hidden, device="cuda", dtype=torch.bfloat16)
    w = torch.full((V, hidden), -4.0, device="cuda", dtype=torch.bfloat16)
    x[t, t], w[y, t], w[c, t] = a, 1.0, b
    return x, w, y, c, a.double(), a.double() * (1 - b.double())


def column(dw, y, a):
    """d of the targets, of an fp32 dw whose row y holds d a in the token's column and nothing else that counts."""
    t = torch.arange(len(y), device="cuda")
    return dw.double()[y, t] / a


def check(d, gap, more=0.0):
    """d = -e / (1 + e), e = exp(-gap).  e is off by 2^-18 of itself (exponent and its rounding); 1 + e is rounded to fp32, by 2^-24; its
    logarithm and expm1 by 2^-21 of themselves; d to bf16 by 2^-8 of itself.  more: of the logarithm of the sum, absolute."""
    e = torch.exp(-gap)
    want = -e / (1 + e)
    tol = (2.0 ** -18 + 2.0 ** -20) * want.abs() + 2.0 ** -24 + more
    tol = tol + (want.abs() + tol) * 2.0 ** -8
    assert bool(((d - want).abs() <= tol).all()), float(((d - want).abs() / tol).max())


# rows and d in one launch (short rows), in two (long ones, few tokens), single CTAs and pairs; by parts
@pytest.mark.parametrize("T,V", [(64, 1000), (64, 9001), (200, 1003), (200, 20000), (1100, 9000)])
@pytest.mark.parametrize("parts", [False, True])
def test_target_column(T, V, parts, monkeypatch):
    x, w, y, c, a, gap = problem(T, V)
    if parts:
        monkeypatch.setattr(vocab, "_STEP_MOST", 0)
    dw = torch.zeros(V, x.shape[1], device="cuda")
    loss, _, _ = vocab.linear_cross_entropy_grad(x, w, y, reduction="sum", dw=dw)
    check(column(dw, y, a), gap)
    assert bool(((vocab.linear_cross_entropy(x, w, y, reduction="none").double() - torch.log1p(torch.exp(-gap))).abs() <= 2.0 ** -18 * torch.exp(-gap) + 2.0 ** -23).all())


@pytest.mark.parametrize("p", [1, 2, 4])
def test_target_column_over_shards(p):
    cfg = L.CommConfig.default()
    cfg.hcclBufferSize = 2
    comm = H.Communicator.init_local(p, device=True, device_id=0, config=cfg)
    T, V = 200, 1000
    x, w, y, c, a, gap = problem(T, V)
    rows = V // p
    dws = [torch.zeros(rows, x.shape[1], device="cuda") for _ in range(p)]
    args = ([x] * p, [s.contiguous() for s in w.chunk(p)], [y] * p)
    vocab.vocab_parallel_cross_entropy_grad(comm, *args, reduction="sum", dw=dws)
    losses = vocab.vocab_parallel_cross_entropy(comm, *args, reduction="none")[0].double()
    assert comm.sync() == 0, comm.describe_status()
    d = column(torch.cat(dws), y, a)
    other = y // rows != c // rows
    # the shards' own logarithms are exchanged as fp32: half a step of a number up to 64 where both ids are in one of several
    check(d, gap, torch.where(other | (p == 1), 0.0, 2.0 ** -19).double())
    # and d is that of the losses
    assert bool(((d + -torch.expm1(-losses)).abs() <= (2.0 ** -8 + 2.0 ** -20) * losses.abs() + 1e-30).all())
    comm.destroy()
