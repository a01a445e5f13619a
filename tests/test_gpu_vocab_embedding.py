"""Token embedding and its gradient against plain statements in 64 bits, at the edges of its vectors, tiles and sorts."""
import pytest

torch = pytest.importorskip("torch")
import cann_hccl_b200 as H  # noqa: E402
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import vocab  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(1)


def lookup64(ids, w, scale, first=0):
    inside = (ids >= first) & (ids < first + w.shape[0])
    rows = w.double()[(ids - first).long().clamp(0, w.shape[0] - 1)] * scale
    return torch.where(inside[..., None], rows, torch.zeros_like(rows))


def half_step(want, dtype):
    """Largest distance of a correctly rounded value: half a step of its size, or of the smallest numbers of the type."""
    f = torch.finfo(dtype)
    return want.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


# rows of whole 32-, 16- and 4-byte vectors, of single elements; one to several stretches of a row
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,hidden", [(1, 1, 1), (8, 50, 16), (7, 33, 8), (129, 1000, 258), (65, 777, 1001), (3, 100, 8192), (1000, 5000, 2056), (5, 9, 16400)])
def test_lookup(T, V, hidden, dtype):
    w = torch.randn(V, hidden, device="cuda").to(dtype)
    ids = torch.randint(-2, V + 3, (T,), device="cuda")
    ids[0] = V - 1
    got = vocab.embedding(ids, w)
    assert torch.equal(got.double(), lookup64(ids, w, 1.0))       # scale 1 copies the bits
    assert torch.equal(vocab.embedding(ids.int(), w), got)
    scale = 7.25
    want = lookup64(ids, w, scale)                                 # the fp32 product is rounded once to the type (fp32: is the product)
    assert bool(((vocab.embedding(ids, w, scale).double() - want).abs() <= half_step(want, dtype)
                 + (want.abs() * 2.0 ** -24 if dtype != torch.float32 else 0)).all())


def test_lookup_shapes_strides_and_shards():
    base = torch.randn(300, 96, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, 300, (4, 5), device="cuda")
    for w in (base[:, :64], base[:, 1:65], base[::2, 8:40]):
        assert torch.equal(vocab.embedding(ids, w).double(), lookup64(ids, w, 1.0))
    got = vocab.embedding(ids, base[100:200], first_id=100)
    assert got.shape == (4, 5, 96) and torch.equal(got.double(), lookup64(ids, base[100:200], 1.0, 100))
    assert vocab.embedding(ids[:0], base).shape == (0, 5, 96)
    out = torch.full((4, 5, 96), 9.0, device="cuda", dtype=torch.bfloat16)
    assert vocab.embedding(ids, base, out=out) is out and torch.equal(out.double(), lookup64(ids, base, 1.0))


def test_lookup_of_special_values():
    w = torch.tensor([[float("inf"), -0.0], [float("nan"), 1.0]], device="cuda")
    got = vocab.embedding(torch.tensor([1, 0, 5, -(2 ** 40)], device="cuda"), w, 2.0)
    assert bool(got[0, 0].isnan()) and got[1, 0] == float("inf") and bool((got[2:] == 0).all())


def test_lookup_beyond_32_bits_of_offset():
    rows, hidden = (1 << 32) // 8192 + 40, 8192                    # 4.3 thousand million elements, 8.6 GB
    w = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16)
    for r in (0, 1, rows // 2, rows - 1):
        w[r] = torch.randn(hidden, device="cuda").to(torch.bfloat16)
    ids = torch.tensor([rows - 1, 0, rows // 2, rows, 1], device="cuda")
    got = vocab.embedding(ids, w)
    for i, r in enumerate(ids.tolist()):
        assert torch.equal(got[i], w[r] if r < rows else torch.zeros_like(got[i]))


def grad64(ids, dy, V, scale, first=0):
    rows = dy.reshape(-1, dy.shape[-1]).double()
    at = (ids.reshape(-1) - first).long()
    ok = (at >= 0) & (at < V)
    want = torch.zeros(V, rows.shape[1], device="cuda", dtype=torch.float64).index_add_(0, at[ok], rows[ok])
    size = torch.zeros_like(want).index_add_(0, at[ok], rows[ok].abs())
    count = torch.zeros(V, device="cuda", dtype=torch.float64).index_add_(0, at[ok], torch.ones_like(at[ok], dtype=torch.float64))
    return want * scale, size * abs(scale), count[:, None]


def close(got, want, size, count, dtype):
    """n - 1 additions and one product in fp32, each off by half a step of at most the sum of the absolute values; one rounding to the
    type (of a value that is off by as much already: factor 1.01)."""
    err = (count + 1) * 2.0 ** -24 * size * 1.01
    if dtype != torch.float32:
        err = err + half_step(want, dtype) * 1.01
    return bool(((got.double() - want).abs() <= err).all())


def text(T, V, kind):
    if kind == "one":
        return torch.full((T,), V // 2, device="cuda")
    if kind == "zipf":
        return (float(V) ** torch.rand(T, device="cuda", dtype=torch.float64)).long().clamp_(1, V) - 1
    if kind == "outside":
        return torch.randint(-V, 2 * V, (T,), device="cuda")
    return torch.randint(0, V, (T,), device="cuda")


# one tile and several, runs of one id that cross tiles, one CTA's sort (8192 tokens) and the tiled one, vocabularies of one, two and
# three digits
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,hidden,kind", [(1, 1, 1, "even"), (31, 7, 24, "zipf"), (32, 100, 64, "one"), (33, 100, 64, "one"), (100, 1000, 33, "outside"),
                                             (1531, 50257, 1001, "zipf"), (1000, 40, 2056, "zipf"), (4097, 300, 512, "one"), (8192, 511, 128, "zipf"),
                                             (8193, 512, 96, "zipf"), (20000, 300000, 40, "outside"), (10001, 33, 8, "zipf"), (12345, 50000, 264, "one"),
                                             (40000, 9, 17, "even"), (7, 3, 9000, "zipf")])
def test_gradient(T, V, hidden, kind, dtype):
    ids, dy = text(T, V, kind), torch.randn(T, hidden, device="cuda").to(dtype)
    scale = 0.5 if hidden % 3 else 3.7
    want, size, count = grad64(ids, dy, V, scale)
    out = torch.full((V, hidden), 5.0, device="cuda", dtype=dtype)
    got = vocab.embedding_grad(ids, dy, V, scale, out=out)
    assert got is out and close(got, want, size, count, dtype)
    assert bool((got[(count[:, 0] == 0)] == 0).all())
    assert torch.equal(vocab.embedding_grad(ids.int(), dy, V, scale), got)   # and the same bits again
    acc = torch.randn(V, hidden, device="cuda")
    start = acc.clone()
    assert vocab.embedding_grad(ids, dy, V, scale, out=acc, add=True) is acc
    assert torch.equal(acc[count[:, 0] == 0], start[count[:, 0] == 0])       # rows without a token are left alone
    assert close(acc, want + start.double(), size + start.double().abs(), count + 1, torch.float32)


@pytest.mark.parametrize("T,V,hidden,dtype", [(300007, 2000, 8, torch.float32), (65536, 30000, 40, torch.bfloat16), (65537, 700, 33, torch.float16),
                                              (70000, 1 << 20, 5, torch.bfloat16)])
def test_gradient_of_a_large_batch(T, V, hidden, dtype):
    """Both sides of what one cluster sorts; long runs; three digits."""
    ids, dy = text(T, V, "zipf"), torch.randn(T, hidden, device="cuda").to(dtype)
    want, size, count = grad64(ids, dy, V, 1.0)
    out = torch.full((V, hidden), 5.0, device="cuda", dtype=dtype)
    assert close(vocab.embedding_grad(ids, dy, V, out=out), want, size, count, dtype)
    assert bool((out[(count[:, 0] == 0)] == 0).all())


def test_gradient_of_every_number_of_tokens():
    """Shared memory of the sort grows with the tokens: every size of it can be launched."""
    for T in [*range(1, 200, 7), *range(3500, 4400, 25), *range(7900, 8300, 33)]:
        ids, dy = text(T, 77, "zipf"), torch.randn(T, 4, device="cuda")
        for V in (77, 300000):
            want, size, count = grad64(ids, dy, V, 1.0)
            assert close(vocab.embedding_grad(ids, dy, V), want, size, count, torch.float32), T


def test_gradient_into_rows_off_a_boundary():
    """A table that starts between vectors, with something before and behind it."""
    for dtype, off in ((torch.bfloat16, 1), (torch.bfloat16, 3), (torch.float32, 1), (torch.float16, 17)):
        room = torch.full((1000 * 33 + 64,), 7.0, device="cuda", dtype=dtype)
        out = room[off:off + 33000].view(1000, 33)
        ids, dy = text(200, 1000, "zipf"), torch.randn(200, 33, device="cuda").to(dtype)
        vocab.embedding_grad(ids, dy, 1000, out=out)
        assert torch.equal(out, vocab.embedding_grad(ids, dy, 1000))
        assert bool((room[:off] == 7).all()) and bool((room[off + 33000:] == 7).all())


def test_gradient_strides_shards_and_empty():
    base = torch.randn(64, 200, device="cuda").to(torch.bfloat16)
    ids = text(64, 30, "even")
    for dy in (base[:, :128], base[:, 3:131]):
        want, size, count = grad64(ids, dy, 30, 1.0)
        assert close(vocab.embedding_grad(ids, dy, 30), want, size, count, torch.bfloat16)
    dy = base.view(4, 16, 200)
    whole = vocab.embedding_grad(ids.view(4, 16), dy, 30)
    halves = [vocab.embedding_grad(ids.view(4, 16), dy, 15, first_id=f) for f in (0, 15)]
    assert torch.equal(torch.cat(halves), whole)
    assert bool((vocab.embedding_grad(ids[:0], base[:0], 30) == 0).all())
    acc = torch.ones(30, 200, device="cuda")
    assert bool((vocab.embedding_grad(ids[:0], base[:0], 30, out=acc, add=True) == 1).all())


def test_gradient_passes_infinities_on():
    dy = torch.ones(6, 32, device="cuda")
    dy[1, 3], dy[2, 4] = float("inf"), float("nan")
    got = vocab.embedding_grad(torch.tensor([0, 1, 1, 2, 7, 0], device="cuda"), dy, 3)
    assert got[1, 3] == float("inf") and bool(got[1, 4].isnan()) and float(got[0, 0]) == 2 and bool((got[2] == 1).all())


def test_gradient_against_differences():
    """sum(embedding * dy) is linear in w: its change along a direction is the gradient's product with it, in 64 bits."""
    T, V, hidden = 50, 20, 12
    ids, dy, w, step = text(T, V, "zipf"), torch.randn(T, hidden, device="cuda"), torch.randn(V, hidden, device="cuda"), torch.randn(V, hidden, device="cuda")
    got = (vocab.embedding_grad(ids, dy, V, 1.5).double() * step.double()).sum()
    f = lambda x: (lookup64(ids, x, 1.5) * dy.double()).sum()  # noqa: E731
    diff = f(w.double() + step.double()) - f(w.double() - step.double())
    assert abs(float(diff / 2 - got)) <= T * hidden * 2.0 ** -22 * 30


@pytest.mark.parametrize("p", [1, 2, 4])
def test_vocab_parallel(p):
    cfg = L.CommConfig.default()
    cfg.hcclBufferSize = 2
    c = H.Communicator.init_local(p, device=True, device_id=0, config=cfg)
    V, hidden = 64 * p, 264
    whole = torch.randn(V, hidden, device="cuda").to(torch.bfloat16)
    ids = torch.randint(-1, V, (3, 37), device="cuda")
    shards = list(whole.chunk(p))
    outs = vocab.vocab_parallel_embedding(c, [ids] * p, shards, 2.0)
    assert c.sync() == 0, c.describe_status()
    want = vocab.embedding(ids, whole, 2.0)
    for o in outs:
        assert torch.equal(o, want)
    dy = torch.randn_like(want)
    parts = [vocab.embedding_grad(ids, dy, 64, 2.0, first_id=f) for f in vocab.first_ids(c, 64)]
    assert torch.equal(torch.cat(parts), vocab.embedding_grad(ids, dy, V, 2.0))
    c.destroy()


def test_captured_and_replayed():
    w, ids = torch.randn(500, 72, device="cuda"), torch.zeros(9000, device="cuda", dtype=torch.int64)
    dy = torch.randn(9000, 72, device="cuda")
    vocab.embedding(ids, w), vocab.embedding_grad(ids, dy, 500)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = vocab.embedding(ids, w, 3.0)
        dw = vocab.embedding_grad(ids, dy, 500)
    for kind in ("zipf", "even", "one"):
        ids.copy_(text(9000, 500, kind))
        dy.normal_()
        graph.replay()
        assert torch.equal(y, vocab.embedding(ids, w, 3.0)) and torch.equal(dw, vocab.embedding_grad(ids, dy, 500))


def test_two_streams_at_once():
    """Two calls in flight share nothing."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    data = [(text(6000, 900, "zipf"), torch.randn(6000, 256, device="cuda")) for _ in range(2)]
    want = [vocab.embedding_grad(i, d, 900) for i, d in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate((a, b)):
            with torch.cuda.stream(s):
                got[k].append(vocab.embedding_grad(*data[k], 900))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(g, want[k]) for g in got[k])


@pytest.mark.parametrize("call", ["vocab.embedding(i, w)", "vocab.embedding_grad(i, w[:3], 5)", "vocab.linear_cross_entropy(w[:3], w, i)", "moe.gate(w, 2)",
                                  "moe.gate_grad(w, moe.Gate(w[:, :2].int().contiguous(), None, w[0].int(), None, i[0].int(), None))"])
def test_first_call_of_a_program(call):
    """Whatever the first call into the package is, it loads the library."""
    import os
    import subprocess
    import sys
    prog = "import torch; from cann_hccl_b200.parallel import moe, vocab; w = torch.zeros(5, 8, device='cuda', dtype=torch.bfloat16); " \
           "i = torch.zeros(3, device='cuda', dtype=torch.int64); %s; torch.cuda.synchronize()" % call
    r = subprocess.run([sys.executable, "-c", prog], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
