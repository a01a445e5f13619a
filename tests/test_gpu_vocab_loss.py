"""Linear layer and softmax cross entropy over the vocabulary, with gradients, against a plain statement in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import cann_hccl_b200 as H  # noqa: E402
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import vocab  # noqa: E402

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8            # half a step of bf16
TINY = 2.0 ** -130          # below what bf16 and fp32 results resolve


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(3)


def problem(T, V, hidden, lean=6.0, dropped=0.1):
    w = (torch.randn(V, hidden, device="cuda") * (1.3 / math.sqrt(hidden))).to(torch.bfloat16)
    y = torch.randint(0, V, (T,), device="cuda")
    x = torch.randn(T, hidden, device="cuda") + torch.rand(T, 1, device="cuda") * lean * w[y].float()
    if T > 2:
        y[torch.rand(T, device="cuda") < dropped] = -100
    return x.to(torch.bfloat16), w, y


class Exact:
    """Losses, gradients and their error bounds.

    logits  a sum of `hidden` exact products, 16 at a time into an fp32 sum that may be cut off instead of rounded: each of the
            hidden / 16 + 2 additions is off by 2^-23 of the sum of absolute values at most
    p       exp of a difference of two such values and a logarithm, the fp16 exponential (half a step 2^-11, or 2^-40 of the half tile's
            largest probability where fp16 has no more digits), 2^-18 for exp, log and the factors
    d       one rounding to bf16
    dx, dw  products of d with the other operand summed as above, one rounding to bf16 (fp32 where it is summed there)"""

    def __init__(self, x, w, y, weights=None, reduction="mean", scale=1.0, whole=None, ignore=-100):
        x, w = x.double(), w.double()
        T, V, hidden = len(x), len(w), x.shape[1]
        on = (y != ignore) & (y >= 0) & (y < V)
        q = on.double() if weights is None else torch.where(on, weights.double(), 0.0)
        s = x @ w.T
        lse = torch.logsumexp(s, 1)
        at = torch.where(on, y, 0).long()
        self.losses = torch.where(on, lse - s.gather(1, at[:, None])[:, 0], 0.0)
        total = q.sum() if reduction == "mean" else 1.0
        g = torch.where(q != 0, q / total, 0.0) * scale if float(total) else q * 0
        self.loss = float((self.losses * torch.where(q != 0, q / total, 0.0)).sum()) if float(total) else 0.0
        step = (hidden / 16 + 2) * 2.0 ** -23 * (x.abs() @ w.abs().T)
        delta = step.amax(1, keepdim=True)
        self.losses_err = torch.where(on, 2 * delta[:, 0] + 2.0 ** -18 * (1 + self.losses.abs() * 2.0 ** -4), 0.0)
        self.loss_err = float((self.losses_err * (g.abs() / abs(scale) if scale else 0.0)).sum()) + abs(self.loss) * 2.0 ** -18 + 2.0 ** -24 * float((self.losses * (g.abs() / abs(scale))).sum()) * (T / 1024 + 10)
        p = torch.exp(s - lse[:, None])
        hit = torch.zeros_like(p)
        hit[on.nonzero()[:, 0], y[on].long()] = 1.0
        d = (p - hit) * g[:, None]
        err = (p * (2 * delta + 2.0 ** -11 + 2.0 ** -18) + 2.0 ** -40 * p.amax(1, keepdim=True)) * g.abs()[:, None]
        err = torch.where(hit > 0, g.abs()[:, None] * (p * 2 * delta + d.abs() / g.abs()[:, None].clamp(min=1e-300) * 2.0 ** -18), err)
        err = err + (d.abs() + err) * BF16
        self.dx, self.dw = d @ w, d.T @ x
        size_x, size_w = d.abs() @ w.abs(), d.abs().T @ x.abs()
        self.dx_err = err @ w.abs() + (V / 16 + 70) * 2.0 ** -23 * size_x
        self.dw_err = err.T @ x.abs() + (T / 16 + 70) * 2.0 ** -23 * size_w

    def check_losses(self, got):
        assert bool(((got.double() - self.losses).abs() <= self.losses_err).all())

    def check(self, got, dw_type=torch.bfloat16, parts=1):
        loss, dx, dw = got
        assert loss.dtype == torch.float32 and loss.dim() == 0 and abs(float(loss) - self.loss) <= self.loss_err
        assert dx.dtype == torch.bfloat16 and dw.dtype == dw_type
        # `parts` bf16 parts of dx are summed: each rounded, and the sum
        tol = self.dx_err * (1 + BF16) + (self.dx.abs() * BF16 if parts == 1 else self.dx_err * 0 + self.dx.abs().amax() * BF16 * (parts + 1)) + TINY
        assert bool(((dx.double() - self.dx).abs() <= tol).all())
        tol = self.dw_err * (1 + BF16) + (self.dw.abs() * (BF16 if dw_type == torch.bfloat16 else 2.0 ** -24)) + TINY
        assert bool(((dw.double() - self.dw).abs() <= tol).all())


# one row of a tile, single CTAs (128 rows) and pairs, one to several tiles of either side, depths of one step and partly filled ones,
# vocabularies below a tile, odd, and just beyond a multiple of it; dx cut along the vocabulary
SHAPES = [(1, 1, 8), (1, 100, 8), (2, 33, 16), (7, 1000, 72), (128, 257, 64), (129, 512, 136), (256, 130, 64), (300, 1003, 1000), (513, 4097, 520), (40, 20001, 264),
          (1000, 300, 2048), (640, 769, 24), (1531, 2050, 320), (60, 4000, 72), (129, 4000, 128), (70001, 100, 8)]


@pytest.mark.parametrize("T,V,hidden", SHAPES)
def test_losses(T, V, hidden):
    x, w, y = problem(T, V, hidden)
    e = Exact(x, w, y)
    got = vocab.linear_cross_entropy(x, w, y, reduction="none")
    assert got.shape == (T,) and got.dtype == torch.float32
    e.check_losses(got)
    assert torch.equal(vocab.linear_cross_entropy(x, w, y.int(), reduction="none"), got)
    assert abs(float(vocab.linear_cross_entropy(x, w, y)) - e.loss) <= e.loss_err


@pytest.mark.parametrize("T,V,hidden", SHAPES)
def test_gradients(T, V, hidden):
    x, w, y = problem(T, V, hidden)
    got = vocab.linear_cross_entropy_grad(x, w, y)
    Exact(x, w, y).check(got)
    again = vocab.linear_cross_entropy_grad(x, w, y)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    weights = torch.rand(T, device="cuda") * 3
    weights[::5] = 0
    Exact(x, w, y, weights, "sum", -2.5).check(vocab.linear_cross_entropy_grad(x, w, y, weights, "sum", scale=-2.5))
    acc = torch.randn(V, hidden, device="cuda")
    start = acc.double()
    loss, dx, dw = vocab.linear_cross_entropy_grad(x, w, y, weights, dw=acc)
    assert dw is acc
    e = Exact(x, w, y, weights)
    e.dw = e.dw + start
    e.dw_err = e.dw_err + start.abs() * 2.0 ** -24
    e.check((loss, dx, dw), torch.float32)


@pytest.mark.parametrize("V", [1, 33, 65, 97, 129, 161, 193, 220, 225, 289, 449, 673, 1345, 3137, 4480, 6657])
def test_gradients_at_the_end_of_the_vocabulary(V):
    """Tiles of every width whose last one ends near a multiple of 32 or 64: columns that no tile reaches are not read either (the scratch
    holds NaN before)."""
    for T in (5, 200):
        x, w, y = problem(T, V, 40)
        junk = torch.full((4 << 20,), 0x7fc0 * 0x10001, device="cuda", dtype=torch.int32)
        del junk                                    # the allocator hands this memory out again
        Exact(x, w, y).check(vocab.linear_cross_entropy_grad(x, w, y))


@pytest.mark.parametrize("T,V,hidden", [(40, 20001, 64), (1100, 9000, 64), (300, 500, 72), (1023, 9001, 40), (1024, 9001, 40)])
def test_one_call_and_its_parts(T, V, hidden, monkeypatch):
    """The whole step in one call, with rows and d in one launch and in two, gives what its parts give."""
    x, w, y = problem(T, V, hidden)
    weights = torch.rand(T, device="cuda")
    weights[::3] = 0
    for q, reduction in ((weights, "mean"), (None, "mean"), (weights, "sum")):
        whole = vocab.linear_cross_entropy_grad(x, w, y, q, reduction)
        monkeypatch.setattr(vocab, "_STEP_MOST", 0)
        parts = vocab.linear_cross_entropy_grad(x, w, y, q, reduction)
        monkeypatch.undo()
        e = Exact(x, w, y, q, reduction)
        e.check(whole)
        e.check(parts)
        # the same sums in another order
        assert abs(float(whole[0]) - float(parts[0])) <= 2.0 ** -20 * abs(float(parts[0])) + 1e-30
        for a, b in zip(whole[1:], parts[1:]):
            assert float((a.float() - b.float()).norm()) <= 2.0 ** -8 * float(b.float().norm())


def test_gradients_of_norm():
    """The errors are those of two roundings to bf16, not their bounds: 2-norm within one half step of the gradients'."""
    x, w, y = problem(700, 3000, 512)
    _, dx, dw = vocab.linear_cross_entropy_grad(x, w, y)
    e = Exact(x, w, y)
    for got, want in ((dx, e.dx), (dw, e.dw)):
        assert float((got.double() - want).norm()) <= BF16 * float(want.norm())


@pytest.mark.parametrize("T,V,hidden,chunk", [(700, 1003, 136, 256), (513, 400, 64, 512), (300, 5000, 72, 128), (1025, 130, 520, 256)])
def test_several_chunks(T, V, hidden, chunk, monkeypatch):
    x, w, y = problem(T, V, hidden)
    weights = torch.rand(T, device="cuda")
    monkeypatch.setattr(L.lib(), "HcclB200VocabLossChunk", lambda v, g: chunk)
    e = Exact(x, w, y, weights)
    e.check_losses(vocab.linear_cross_entropy(x, w, y, reduction="none"))
    e.check(vocab.linear_cross_entropy_grad(x, w, y, weights))
    acc = torch.zeros(V, hidden, device="cuda")
    e.check(vocab.linear_cross_entropy_grad(x, w, y, weights, dw=acc), torch.float32)


def test_strided_rows():
    x, w, y = problem(300, 600, 136)
    xs, ws = torch.zeros(300, 160, device="cuda", dtype=torch.bfloat16), torch.zeros(1200, 144, device="cuda", dtype=torch.bfloat16)
    xs[:, 8:144], ws[::2, :136] = x, w
    want = vocab.linear_cross_entropy_grad(x, w, y)
    got = vocab.linear_cross_entropy_grad(xs[:, 8:144], ws[::2, :136], y)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = vocab.linear_cross_entropy_grad(x[:1], w, y[:1])
    assert all(torch.equal(a, b) for a, b in zip(vocab.linear_cross_entropy_grad(xs[:1, 8:144], w, y[:1]), one))


def test_tokens_that_do_not_count():
    """Whatever stands in their rows, they reach nothing."""
    x, w, y = problem(260, 500, 72, dropped=0.0)
    out = torch.rand(260, device="cuda") < 0.4
    y[out] = torch.tensor([-100, -1, 500, 2 ** 40], device="cuda")[torch.randint(0, 4, (int(out.sum()),), device="cuda")]
    weights = torch.ones(260, device="cuda")
    zero = (torch.rand(260, device="cuda") < 0.3) & ~out
    weights[zero] = 0
    want = Exact(x, w, y, weights)
    dirty = x.clone()
    dirty[out] = math.nan
    dirty[zero, 3] = math.inf
    got = vocab.linear_cross_entropy_grad(dirty, w, y, weights)
    want.check(got)
    assert bool((got[1][out | zero] == 0).all())
    assert float(vocab.linear_cross_entropy(dirty, w, y, weights)) == float(got[0])
    losses = vocab.linear_cross_entropy(dirty, w, y, reduction="none")
    assert bool((losses[out] == 0).all())
    for bad in (torch.full_like(y, -100), y.clamp(min=500)):                       # none at all
        loss, dx, dw = vocab.linear_cross_entropy_grad(dirty, w, bad)
        assert float(loss) == 0 and bool((dx == 0).all()) and bool((dw == 0).all())
    e = Exact(x, w, y.clamp(0, 499), ignore=0)                                      # an id of the vocabulary may be the one to ignore
    e.check(vocab.linear_cross_entropy_grad(x, w, y.clamp(0, 499), ignore_index=0))


@pytest.mark.parametrize("T,hidden", [(7, 72), (300, 1000), (300, 128)])
def test_tokens_without_weight_have_losses(T, hidden):
    """reduction "none" gives every token's own loss; weights only matter to the sums."""
    x, w, y = problem(T, 500, hidden)
    weights = torch.rand(T, device="cuda")
    weights[::2] = 0
    got = vocab.linear_cross_entropy(x, w, y, weights, reduction="none")
    assert torch.equal(got, vocab.linear_cross_entropy(x, w, y, reduction="none"))
    e = Exact(x, w, y, weights)
    e.check_losses(got)
    assert abs(float(vocab.linear_cross_entropy(x, w, y, weights)) - e.loss) <= e.loss_err


def test_sure_and_wild_guesses():
    """Probabilities next to one, logits of thousands, and rows of equal logits."""
    x, w, y = problem(200, 900, 64, lean=0.0)
    x[:50] = (w[y.clamp(min=0)][:50].float() * 300).to(torch.bfloat16)              # logits of 300 times |w|^2: nothing but the target
    x[50:100] = (x[50:100].float() * 3000).to(torch.bfloat16)
    x[100:150] = 0
    got = vocab.linear_cross_entropy_grad(x, w, y)
    e = Exact(x, w, y)
    e.check(got)
    e.check_losses(vocab.linear_cross_entropy(x, w, y, reduction="none"))
    assert all(bool(t.isfinite().all()) for t in got)


def test_infinities_stay_in_their_rows():
    x, w, y = problem(130, 300, 64, dropped=0.0)
    clean = vocab.linear_cross_entropy(x, w, y, reduction="none")
    x[7, 0], x[9, 1] = math.inf, math.nan
    got = vocab.linear_cross_entropy(x, w, y, reduction="none")
    rest = torch.ones(130, device="cuda", dtype=torch.bool)
    rest[7] = rest[9] = False
    assert torch.equal(got[rest], clean[rest]) and bool(got[~rest].isnan().all())


def test_no_tokens():
    x, w, y = problem(4, 50, 16)
    assert vocab.linear_cross_entropy(x[:0], w, y[:0], reduction="none").shape == (0,)
    loss, dx, dw = vocab.linear_cross_entropy_grad(x[:0], w, y[:0])
    assert float(loss) == 0 and dx.shape == (0, 16) and bool((dw == 0).all())
    acc = torch.ones(50, 16, device="cuda")
    assert bool((vocab.linear_cross_entropy_grad(x[:0], w, y[:0], dw=acc)[2] == 1).all())


def test_against_differences():
    x, w, y = problem(60, 90, 40)
    loss, dx, dw = vocab.linear_cross_entropy_grad(x, w, y)
    on = y >= 0

    def f(xd, wd):
        s = xd @ wd.T
        return (torch.logsumexp(s, 1) - s.gather(1, y.clamp(min=0)[:, None])[:, 0])[on].mean()
    h = 1e-4
    for which in (0, 1):
        step = torch.randn_like((x, w)[which].double())
        pair = [(x.double() + s * h * step, w.double()) if which == 0 else (x.double(), w.double() + s * h * step) for s in (1, -1)]
        diff = float(f(*pair[0]) - f(*pair[1])) / (2 * h)
        got = (dx, dw)[which].double()
        # two roundings to bf16 of every term (sums of many: their 2-norms), and h^2 of the third derivative
        assert abs(diff - float((got * step).sum())) <= 1e-5 + 2 * BF16 * 6 * float(got.norm())


@pytest.mark.parametrize("p", [1, 2, 3, 4])
def test_vocab_parallel(p):
    cfg = L.CommConfig.default()
    cfg.hcclBufferSize = 2
    c = H.Communicator.init_local(p, device=True, device_id=0, config=cfg)
    T, V, hidden = 300, 131 * p, 136
    x, w, y = problem(T, V, hidden)
    y[5] = V                                                                         # no id, though the last shard's padding has room for it
    weights = torch.rand(T, device="cuda")
    shards = [s.contiguous() for s in w.chunk(p)]
    e = Exact(x, w, y, weights)
    out = vocab.vocab_parallel_cross_entropy_grad(c, [x] * p, shards, [y] * p, [weights] * p)
    losses = vocab.vocab_parallel_cross_entropy(c, [x] * p, shards, [y] * p, reduction="none")
    assert c.sync() == 0, c.describe_status()
    for r in range(p):
        assert torch.equal(out[r][0], out[0][0]) and torch.equal(out[r][1], out[0][1])
        e.check_losses(losses[r])
    e.check((out[0][0], out[0][1], torch.cat([o[2] for o in out])), parts=p)
    acc = [torch.zeros(131, hidden, device="cuda") for _ in range(p)]
    out = vocab.vocab_parallel_cross_entropy_grad(c, [x] * p, shards, [y] * p, [weights] * p, dw=acc)
    assert c.sync() == 0, c.describe_status()
    e.check((out[0][0], out[0][1], torch.cat(acc)), torch.float32, parts=p)
    c.destroy()


def test_table_beyond_32_bits_of_offset():
    """4.3 thousand million weights: targets on both sides of the border, rows of dw checked one by one."""
    hidden, V, T = 8192, (1 << 32) // 8192 + 300, 40
    w = torch.empty(V, hidden, device="cuda", dtype=torch.bfloat16).normal_(0, 0.01)
    x = torch.randn(T, hidden, device="cuda").to(torch.bfloat16)
    y = torch.cat([torch.randint(0, 100, (T // 2,), device="cuda"), torch.randint(V - 200, V, (T // 2,), device="cuda")])
    loss, dx, dw = vocab.linear_cross_entropy_grad(x, w, y)
    s = torch.cat([x.float() @ part.float().T for part in w.split(1 << 16)], 1).double()
    p = torch.softmax(s, 1)
    assert abs(float(loss) - float((torch.logsumexp(s, 1) - s.gather(1, y[:, None])[:, 0]).mean())) <= 1e-3
    d = p / T
    d[torch.arange(T), y] -= 1 / T
    for r in [0, 1, V // 2, V - 1] + y.tolist():
        want = d[:, r] @ x.double()
        assert float((dw[r].double() - want).norm()) <= 2 * BF16 * float(want.norm())
    want = sum((d[:, a:a + 65536].float() @ w[a:a + 65536].float()).double() for a in range(0, V, 65536))
    assert float((dx.double() - want).norm()) <= 2 * BF16 * float(want.norm())


def test_captured_and_replayed():
    x, w, y = problem(700, 2000, 264)
    vocab.linear_cross_entropy_grad(x, w, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = vocab.linear_cross_entropy_grad(x, w, y)
        losses = vocab.linear_cross_entropy(x, w, y, reduction="none")
    for _ in range(3):
        x2, w2, y2 = problem(700, 2000, 264)
        x.copy_(x2), w.copy_(w2), y.copy_(y2)
        graph.replay()
        want = vocab.linear_cross_entropy_grad(x, w, y)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(losses, vocab.linear_cross_entropy(x, w, y, reduction="none"))


@pytest.mark.parametrize("call", ["vocab.linear_cross_entropy_grad(x, w, y)", "vocab.linear_cross_entropy(x[:7], w, y[:7])", "vocab.embedding_grad(y, x, 5000)",
                                  "vocab.embedding_grad(y.repeat(40), x.repeat(40, 1), 5000)", "vocab.embedding(y, w)", "moe.gate_grad(x, moe.gate(x, 3), None, 1.0)"])
def test_first_call_of_a_program_is_captured(call):
    """Nothing has been loaded or asked for before the capture."""
    import os
    import subprocess
    import sys
    prog = """
import torch
from cann_hccl_b200.parallel import moe, vocab
torch.manual_seed(1)
x, w, y = torch.randn(300, 72, device="cuda").bfloat16(), torch.randn(5000, 72, device="cuda").bfloat16(), torch.randint(0, 5000, (300,), device="cuda")
side = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=side):
    got = %s
graph.replay()
torch.cuda.synchronize()
want = %s
for a, b in zip(*[t if isinstance(t, tuple) else (t,) for t in (got, want)]):
    assert torch.equal(a, b)
""" % (call, call)
    r = subprocess.run([sys.executable, "-c", prog], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_two_streams_at_once():
    data = [problem(300, 1500, 136) for _ in range(2)]
    want = [vocab.linear_cross_entropy_grad(*d) for d in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(vocab.linear_cross_entropy_grad(*data[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[k]))
