"""What a Gate keeps of the call that made it: gate_grad() without mask and normalize is the gradient of that call."""
import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200.parallel import moe  # noqa: E402
from test_gpu_moe_gate import REL, gate64, grad64  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(8)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(40, 16, 3), (2371, 60, 4), (5000, 256, 8)])
def test_gradient_of_a_masked_batch(T, E, k, normalize):
    l, mask = torch.randn(T, E, device="cuda"), torch.rand(T, device="cuda") < 0.7
    d = torch.randn(T, k, device="cuda")
    g = moe.gate(l, k, mask, normalize)
    want = gate64(l, k, mask, normalize)
    for kind in (mask, mask.to(torch.uint8)):
        g = moe.gate(l, k, kind, normalize)
        got = moe.gate_grad(l, g, d, balance=0.9)
        assert bool((got[~mask] == 0).all())
        assert torch.equal(got, moe.gate_grad(l, g, d, 0.9, mask, normalize))
        d64 = grad64(l, want, k, d, 0.9, normalize)
        size = (want[6] * want[2].double()[None, :] * (0.9 * E / (k * want[4] ** 2))).amax() * 2 + d.abs().double().amax() * 2
        assert float((got.double() - d64).abs().max()) <= 8 * REL * float(size)


def test_gradient_without_normalised_gates():
    l, d = torch.randn(50, 24, device="cuda"), torch.randn(50, 5, device="cuda")
    g = moe.gate(l, 5, normalize=False)
    assert torch.equal(moe.gate_grad(l, g, d), moe.gate_grad(l, g, d, normalize=False))
    assert not torch.equal(moe.gate_grad(l, g, d), moe.gate_grad(l, g, d, normalize=True))
    # a Gate of other tensors: as it is told, normalised where nothing is said
    assert torch.equal(moe.gate_grad(l, moe.Gate(*g, normalize=False), d), moe.gate_grad(l, g, d))
    assert torch.equal(moe.gate_grad(l, moe.Gate(*g), d), moe.gate_grad(l, g, d, normalize=True))


def test_mask_that_was_written_to():
    """The Gate has the mask itself, not a copy: one that was written to since is refused, unless the caller gives one."""
    l, mask = torch.randn(64, 16, device="cuda"), torch.rand(64, device="cuda") < 0.5
    g, keep = moe.gate(l, 2, mask), mask.clone()
    want = moe.gate_grad(l, g, g.gates, 1.0)
    mask.logical_not_()
    with pytest.raises(RuntimeError, match="mask"):
        moe.gate_grad(l, g, g.gates, 1.0)
    assert torch.equal(moe.gate_grad(l, g, g.gates, 1.0, mask=keep), want)
    assert torch.equal(moe.gate_grad(l, moe.Gate(*g, mask=keep), g.gates, 1.0), want)
    with torch.inference_mode():                                    # tensors that do not count their writes
        m = keep.clone()
        assert torch.equal(moe.gate_grad(l, moe.gate(l, 2, m), g.gates, 1.0), want)


def test_captured_with_a_mask():
    l, mask = torch.randn(500, 64, device="cuda"), torch.rand(500, device="cuda") < 0.5
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = moe.gate(l, 4, mask)
        dl = moe.gate_grad(l, g, g.gates, 0.5)
    for _ in range(3):
        l.normal_()
        mask.copy_(torch.rand(500, device="cuda") < 0.5)
        graph.replay()
        want = moe.gate(l, 4, mask)
        assert torch.equal(dl, moe.gate_grad(l, want, want.gates, 0.5)) and bool((dl[~mask] == 0).all())


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("E", [16, 200])
def test_gate_by_hand_that_names_an_expert_twice(E, normalize):
    """Each slot passes its part on, whichever expert it names."""
    l, d = torch.randn(300, E, device="cuda"), torch.randn(300, 4, device="cuda")
    g = moe.gate(l, 4, normalize=normalize)
    idx = g.idx.clone()
    idx[::2, 1] = idx[::2, 0]
    idx[::4, 3] = idx[::4, 0]
    idx[1::4, 3] = idx[1::4, 2]
    p = torch.softmax(l.double(), 1)
    gates = p.gather(1, idx.long())
    if normalize:
        gates = gates / gates.sum(1, keepdim=True)
    counts = torch.bincount(idx.flatten(), minlength=E).int()
    hand = moe.Gate(idx, gates.float(), counts, p.sum(0).float(), g.routed, g.balance, normalize=normalize)
    want = grad64(l, (idx, gates, counts, None, 300, None, p), 4, d, 0.6, normalize)
    got = moe.gate_grad(l, hand, d, 0.6).double()
    # sums of at most nine terms of this size, each off by REL
    size = d.abs().double().amax() * 2 + 0.6 * E / (4 * 300 ** 2) * float(counts.max()) * 2
    assert float((got - want).abs().max()) <= 9 * REL * float(size)
    assert torch.equal(got, moe.gate_grad(l, hand, d, 0.6).double())


def test_slots_written_to_by_hand():
    """The same of a Gate of gate() whose experts were changed in place."""
    l, d = torch.randn(300, 40, device="cuda"), torch.randn(300, 4, device="cuda")
    g = moe.gate(l, 4)
    plain = moe.gate_grad(l, g, d, 0.6)
    assert torch.equal(plain, moe.gate_grad(l, moe.Gate(*g), d, 0.6))                # two variants, the same bits where experts differ
    g.idx[::3, 2] = g.idx[::3, 0]
    got = moe.gate_grad(l, g, d, 0.6)
    assert torch.equal(got, moe.gate_grad(l, moe.Gate(*[t.clone() for t in g]), d, 0.6))
    keep = torch.arange(300, device="cuda") % 3 != 0
    assert torch.equal(got[keep], plain[keep]) and not torch.equal(got, plain)
