"""Logits of the vocabulary loss whose depth is summed in parts: at the parts' edges, and sums that grow evenly, which the tensor cores'
running sum alone would leave too small."""
import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200.parallel import vocab  # noqa: E402
from test_gpu_vocab_loss import Exact, problem  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(10)


# single CTAs: parts of 8 to 15 steps of 64 elements, pairs: of 16 to 31; one part, two, a short last one; tiles of every width
@pytest.mark.parametrize("hidden", [960, 1024, 1032, 1536, 2040, 2048, 2056, 4160, 5000])
@pytest.mark.parametrize("T,V", [(7, 33), (7, 5000), (40, 130), (128, 1003), (129, 450), (300, 1003), (513, 70)])
def test_parts_of_the_depth(T, V, hidden):
    x, w, y = problem(T, V, hidden)
    e = Exact(x, w, y)
    e.check_losses(vocab.linear_cross_entropy(x, w, y, reduction="none"))
    e.check(vocab.linear_cross_entropy_grad(x, w, y))


@pytest.mark.parametrize("T,V", [(7, 300), (128, 2000), (200, 300), (300, 40000)])
def test_sums_that_grow_evenly(T, V):
    """All products positive.  A logit is summed 16 products at a time in parts of 16 steps of 64 at most: 66 additions in one, cut off by at most
    2^-23 of the part's sum each; its parts, 64 at most, are added, rounded by 2^-24 of the sum.  The target's logit is summed by at least 128
    threads in FMAs, hidden / 128 in a row, rounded by 2^-24 of the sum each.  (One running sum is off by about 275 x 2^-23 here.)"""
    hidden = 32768
    x = (0.5 + torch.rand(T, hidden, device="cuda")).to(torch.bfloat16)
    w = ((0.5 + torch.rand(V, hidden, device="cuda")) * (10 / hidden)).to(torch.bfloat16)
    y = torch.randint(0, V, (T,), device="cuda")
    s = torch.cat([x.double() @ part.double().T for part in w.split(4096)], 1)
    want = torch.logsumexp(s, 1) - s.gather(1, y[:, None])[:, 0]
    got = vocab.linear_cross_entropy(x, w, y, reduction="none").double()
    top = s.amax(1)
    err = top * (66 * 2.0 ** -23 + 64 * 2.0 ** -24 + (hidden / 128 + 12) * 2.0 ** -24) + 2.0 ** -18 * (1 + want)
    assert bool(((got - want).abs() <= err).all()), float(((got - want).abs() / err).max())
