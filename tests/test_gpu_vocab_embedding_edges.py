"""Embedding gradient on both sides of the edges of its sorts: by counting up to 4096 tokens, by small tiles up to 2^18, by large ones above;
bits of the rows in use made 2^18 rows at a time."""
import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200.parallel import vocab  # noqa: E402
from test_gpu_vocab_embedding import close, grad64, text  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,V", [(4095, 1000), (4096, 1000), (4097, 1000), (4096, (1 << 18) - 1), (4096, 1 << 18), (4096, (1 << 18) + 1), (1, (1 << 18) + 1),
                                 ((1 << 18) - 1, 30000), (1 << 18, 30000), ((1 << 18) + 1, 30000), ((1 << 18) + 1, (1 << 18) + 1), (1 << 18, 511), ((1 << 18) + 8192, 512)])
@pytest.mark.parametrize("kind", ["zipf", "outside", "one"])
def test_edges(T, V, kind):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(7)
    ids, dy = text(T, V, kind), torch.randn(T, 16, device="cuda")
    ids[0], ids[-1] = V - 1, 0
    want, size, count = grad64(ids, dy, V, 1.5)
    out = torch.full((V, 16), 5.0, device="cuda")
    got = vocab.embedding_grad(ids, dy, V, 1.5, out=out)
    assert close(got, want, size, count, torch.float32) and bool((got[count[:, 0] == 0] == 0).all())
    acc = torch.full((V, 16), 5.0, device="cuda")
    vocab.embedding_grad(ids, dy, V, 1.5, out=acc, add=True)
    assert close(acc, want + 5, size + 5, count + 1, torch.float32) and bool((acc[count[:, 0] == 0] == 5).all())
