"""Router (gates, counts, balance loss) and its gradient against plain statements in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import cann_hccl_b200 as H  # noqa: E402
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import moe  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(2)


def gate64(logits, k, mask=None, normalize=True):
    l = logits.double()
    T, E = l.shape
    on = (l > -math.inf).any(1)
    if mask is not None:
        on = on & mask.bool()
    p = torch.where(on[:, None], torch.softmax(l, 1), torch.zeros_like(l))
    vals, order = torch.sort(l, dim=1, descending=True, stable=True)
    idx = torch.where(on[:, None] & (vals[:, :k] > -math.inf), order[:, :k], -1)
    g = torch.where(idx >= 0, p.gather(1, idx.clamp(min=0)), 0.0)
    if normalize:
        g = torch.where(on[:, None], g / g.sum(1, keepdim=True), 0.0)
    counts = torch.bincount(idx[idx >= 0], minlength=E)
    n = int(on.sum())
    balance = float((counts * p.sum(0)).sum()) * E / (k * n * n) if n else 0.0
    return idx.int(), g, counts.int(), p.sum(0), n, balance, p


def grad64(logits, g, k, d_gates, coef, normalize):
    idx, gates, counts, _, n, _, p = g
    E = logits.shape[1]
    u = counts.double()[None, :] * (coef * E / (k * n * n) if n else 0.0)
    dl = torch.zeros_like(p)
    dg = torch.where(idx >= 0, d_gates.double(), 0.0)
    if normalize:
        part = gates * (dg - (gates * dg).sum(1, keepdim=True))
    else:
        part = gates * dg
        dl -= p * part.sum(1, keepdim=True)
    dl += p * (u - (p * u).sum(1, keepdim=True))
    return dl.scatter_add(1, idx.clamp(min=0).long(), torch.where(idx >= 0, part, 0.0))


# exp is off by a few units of 2^-23 and 2^-23 |x| through its argument (|x| < 16 here where it counts); sums of E terms
REL = 2.0 ** -18


def check(logits, k, mask=None, normalize=True):
    want = gate64(logits, k, mask, normalize)
    g = moe.gate(logits, k, mask, normalize)
    assert g.idx.dtype == torch.int32 and torch.equal(g.idx, want[0])
    assert torch.equal(g.counts, want[2]) and int(g.routed) == want[4]
    assert bool(((g.gates.double() - want[1]).abs() <= REL * want[1] + 1e-30).all())
    T, E = logits.shape
    # sums over the tokens in fp32: every addition is off by half a step of the sum at most
    assert bool(((g.prob_sum.double() - want[3]).abs() <= (REL + T * 2.0 ** -24) * want[3] + 1e-30).all())
    assert abs(float(g.balance) - want[5]) <= (REL + (T + E) * 2.0 ** -24) * want[5] + 1e-30
    d_gates = torch.randn(T, k, device="cuda")
    for dg, coef in ((d_gates, 0.7), (None, 1.3), (d_gates, 0.0)):
        d64 = grad64(logits, want, k, d_gates if dg is not None else torch.zeros_like(d_gates), coef, normalize)
        dl = moe.gate_grad(logits, g, dg, coef, mask, normalize)
        # differences of terms of this size, each off by REL
        size = want[6] * (want[2].double()[None, :] * (coef * E / (k * max(1, want[4]) ** 2)))
        size = size + want[6] * size.sum(1, keepdim=True)
        if dg is not None:
            both = (want[1] * d_gates.double().abs())
            size = size + (want[6] * both.sum(1, keepdim=True) if not normalize else 0.0)
            size = size.scatter_add(1, want[0].clamp(min=0).long(), both + want[1] * both.sum(1, keepdim=True))
        tol = REL * 4 * size + 1e-30
        if logits.dtype != torch.float32:
            f = torch.finfo(logits.dtype)
            tol = tol + d64.abs() * (f.eps / 2) + f.smallest_normal * f.eps
        assert dl.dtype == logits.dtype and bool(((dl.double() - d64).abs() <= tol).all())
    return g


# experts of a lane: 2 to 128 registers, whole and partly filled; k up to all experts and to 32; more tokens than warps
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 8, 8), (16, 64, 8), (129, 60, 4), (2371, 33, 2), (500, 128, 1), (8192, 256, 8), (77, 257, 17), (65, 512, 32),
                                   (40, 1000, 8), (33, 2048, 4), (19, 4096, 32)])
def test_gate(T, E, k, dtype, normalize):
    check((torch.randn(T, E, device="cuda") * 2).to(dtype), k, None, normalize)


def test_every_size_of_a_decode_batch():
    """Shared memory grows with tokens and experts: every size of it can be launched."""
    for T in [*range(1, 20), 40, 63, 64, 65, 66, 130]:
        for E in (60, 129, 257, 300, 400, 511, 700, 1000, 1300, 2000, 2500):
            l = torch.randn(T, E, device="cuda")
            g, want = moe.gate(l, 3), gate64(l, 3)
            assert torch.equal(g.idx, want[0]) and torch.equal(g.counts, want[2]), (T, E)
            assert moe.gate_grad(l, g, None, 1.0).shape == (T, E)


@pytest.mark.parametrize("E,k", [(7, 3), (64, 8), (300, 5)])
def test_ties_go_to_the_lowest_expert(E, k):
    l = torch.randint(-1, 2, (400, E), device="cuda").float()
    l[:50] = 0.0
    l[50:100, ::2] = -0.0                                             # equal to 0
    l[50:100, 1::2] = 0.0
    g = check(l, k)
    assert bool((g.idx[:100] == torch.arange(k, device="cuda")).all())


def test_masked_experts_and_tokens():
    inf = math.inf
    l = torch.randn(257, 96, device="cuda")
    l[:60, 5:] = -inf                                                 # fewer experts than slots
    l[60:64] = -inf                                                   # none at all
    l[70, :] = torch.finfo(torch.float32).min                         # the lowest value is a value
    l[71, 3] = 3.0e38
    mask = torch.rand(257, device="cuda") < 0.7
    for m in (None, mask, mask.to(torch.uint8)):
        g = check(l, 8, m)
        assert bool((g.idx[:60, 5:] == -1).all()) and bool((g.gates[:60, 5:] == 0).all()) and bool((g.idx[60:64] == -1).all())
    g = check(l, 8, torch.zeros_like(mask))
    assert int(g.routed) == 0 and float(g.balance) == 0 and bool((g.gates == 0).all()) and bool((g.counts == 0).all())


def test_more_equal_logits_than_a_list_holds():
    """Rows whose k-th largest logit is shared by many experts, among rows that have no such."""
    l = torch.randn(300, 200, device="cuda")
    l[::3] = (l[::3] > 0.5).float()                                   # about sixty experts share the largest
    l[1::7, 20:] = l[1::7, 20:21]
    for dtype in TYPES:
        check(l.to(dtype), 8)
        check((l * 3).round().to(dtype), 5)


def test_infinities_and_nan_stay_in_their_rows():
    l = torch.randn(64, 40, device="cuda")
    l[3, 7], l[9, 0], l[9, 30] = math.nan, math.inf, math.inf
    g = moe.gate(l, 4)
    assert int(g.idx[3, 0]) == 7 and g.idx[9, :2].tolist() == [0, 30]
    assert bool(((g.idx >= 0) & (g.idx < 40)).all()) and bool((g.idx.sort(1).values.diff(dim=1) > 0).all())
    rest = torch.ones(64, device="cuda", dtype=torch.bool)
    rest[3] = rest[9] = False
    want = gate64(l[rest], 4)
    assert torch.equal(g.idx[rest], want[0]) and bool(((g.gates[rest].double() - want[1]).abs() <= REL * want[1]).all())
    assert bool(g.gates[3].isnan().all()) and bool(g.gates[9].isnan().all())
    dl = moe.gate_grad(l, g, torch.randn(64, 4, device="cuda"))       # no balance loss: other rows are not reached
    assert bool(dl[rest].isfinite().all())


def test_strided_rows_and_no_tokens():
    base = torch.randn(50, 200, device="cuda")
    for l in (base[:, 4:132], base[:, 5:133], base[:, :100], base.to(torch.bfloat16)[:, 4:104], base.to(torch.float16)[:, 3:103]):
        assert torch.equal(check(l, 7).idx, moe.gate(l.contiguous(), 7).idx)
    assert torch.equal(check(base[:, 3:67], 6).idx, moe.gate(base[:, 3:67].contiguous(), 6).idx)
    g = moe.gate(base[:0], 6)
    assert g.idx.shape == (0, 6) and float(g.balance) == 0 and int(g.routed) == 0 and bool((g.counts == 0).all())
    assert moe.gate_grad(base[:0], g).shape == (0, 200)


def test_gradient_against_differences():
    """Change of sum(gates * d) + c * balance along a direction, the choice of experts and the counts held, in 64 bits."""
    l, k, c = torch.randn(40, 24, device="cuda"), 5, 0.9
    d, step = torch.randn(40, k, device="cuda"), torch.randn(40, 24, device="cuda")
    for normalize in (True, False):
        g = moe.gate(l, k, normalize=normalize)
        at = g.idx.long()

        def f(x):
            p = torch.softmax(x, 1)
            s = p.gather(1, at)
            s = s / s.sum(1, keepdim=True) if normalize else s
            return (s * d.double()).sum() + c * 24 / (k * 40 * 40) * (g.counts.double() * p.sum(0)).sum()
        h = 1e-5
        diff = (f(l.double() + h * step.double()) - f(l.double() - h * step.double())) / (2 * h)
        got = (moe.gate_grad(l, g, d, c, normalize=normalize).double() * step.double()).sum()
        # the difference leaves h^2 times a third derivative; the gradient REL of its terms' sizes
        assert abs(float(diff - got)) <= 1e-6 + REL * float((d.abs().sum() + 24) * step.abs().max())


def test_parts_of_a_gate():
    """Parts share memory with what later calls read; a Gate of other tensors (experts dropped by hand) is taken as well."""
    l = torch.randn(30, 16, device="cuda")
    g = moe.gate(l, 3)
    d = torch.randn(30, 3, device="cuda")
    assert [t.dtype for t in g] == [torch.int32, torch.float32, torch.int32, torch.float32, torch.int32, torch.float32]
    assert [tuple(t.shape) for t in g] == [(30, 3), (30, 3), (16,), (16,), (), ()] and all(t.is_contiguous() for t in g) and g.idx is g.idx
    want = moe.gate_grad(l, moe.Gate(*[t.clone() for t in g]), d, 0.3)
    assert torch.equal(moe.gate_grad(l, g, d, 0.3), want)
    with pytest.raises(AttributeError):
        g.idx = g.idx.clone()
    g.idx[4, 1] = -1                                                  # dropped: it passes nothing on, the other gates share its part
    dropped = moe.gate_grad(l, g, d)
    p = torch.softmax(l[4].double(), 0)
    at = g.idx[4, [0, 2]].long()
    q = p[at] / p[at].sum()
    part = q * (d[4, [0, 2]].double() - (q * d[4, [0, 2]].double()).sum())
    row = torch.zeros(16, device="cuda", dtype=torch.float64).scatter_add(0, at, part)
    assert bool(((dropped[4].double() - row).abs() <= 8 * REL * d[4].abs().max()).all())
    for bad in (g.idx[:, :2], g.idx.float(), g.idx[:7]):
        with pytest.raises(ValueError):
            moe.gate_grad(l, moe.Gate(bad, *list(g)[1:]))
    with pytest.raises(TypeError):
        moe.gate_grad(l, tuple(g))


def test_same_bits_again_and_captured():
    l = torch.randn(5000, 256, device="cuda")
    a, b = moe.gate(l, 8), moe.gate(l, 8)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g = moe.gate(l, 8)
        dl = moe.gate_grad(l, g, g.gates, 0.5)
    for _ in range(3):
        l.normal_()
        graph.replay()
        want = moe.gate(l, 8)
        assert all(torch.equal(x, y) for x, y in zip(g, want)) and torch.equal(dl, moe.gate_grad(l, want, want.gates, 0.5))


@pytest.mark.parametrize("p", [1, 3, 4])
def test_over_all_ranks(p):
    """Counts, sums and loss of all ranks' tokens; the gradient of a rank's logits is that of the joint loss."""
    cfg = L.CommConfig.default()
    cfg.hcclBufferSize = 2
    c = H.Communicator.init_local(p, device=True, device_id=0, config=cfg)
    ls = [torch.randn(100 + 7 * r, 60, device="cuda") for r in range(p)]
    ms = [torch.rand(len(l), device="cuda") < 0.8 for l in ls]
    gs = moe.gate(ls, 4, ms, comm=c)
    assert c.sync() == 0, c.describe_status()
    joint, mask = torch.cat(ls), torch.cat(ms)
    want = gate64(joint, 4, mask)
    d64 = grad64(joint, want, 4, torch.zeros(len(joint), 4, device="cuda"), 1.0, True).split([len(l) for l in ls])
    for r, g in enumerate(gs):
        assert torch.equal(g.counts, want[2]) and int(g.routed) == want[4]
        assert abs(float(g.balance) - want[5]) <= 2 * REL * want[5]
        dl = moe.gate_grad(ls[r], g, balance=1.0, mask=ms[r])
        assert bool(((dl.double() - d64[r]).abs() <= 16 * REL * d64[r].abs().max()).all())
    c.destroy()


def test_gate_feeds_the_exchange():
    """Router, dispatch, identity experts and combine: routed tokens come back, masked ones as zeros."""
    T, hidden, E, k = 300, 256, 32, 4
    c = H.Communicator.init_root(1, H.Communicator.get_root_info(), 0, device=True)
    ex = moe.MoEExchange(c, T, hidden, E, k)
    x = torch.randn(T, hidden, device="cuda").to(torch.bfloat16)
    mask = torch.rand(T, device="cuda") < 0.8
    g = moe.gate(torch.randn(T, E, device="cuda"), k, mask)
    ex.dispatch(x, g.idx)
    out = ex.combine(g.gates, source="recv")
    assert c.sync() == 0, c.describe_status()
    assert torch.equal(ex.expert_offsets[0].diff(), g.counts)
    want = x.float() * mask[:, None]
    # k products and sums in fp32 of gates that sum to one but for REL, one rounding to bf16
    assert bool(((out.float() - want).abs() <= (2.0 ** -8 + REL) * 1.01 * want.abs()).all())
    ex.close()
    c.destroy()
