"""A training step of a small model through the operators as they are used together: token embedding, router, expert exchange, loss
over the vocabulary, and back, the embedding's weight being the loss's too."""
import pytest

torch = pytest.importorskip("torch")
import cann_hccl_b200 as H  # noqa: E402
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import moe, vocab  # noqa: E402

pytestmark = pytest.mark.gpu
COEF = 0.05


def exact(ids, targets, w, wr, k, scale, idx):
    """Loss and gradients in 64 bits by automatic differentiation, the choice of experts given."""
    w, wr = w.double().requires_grad_(), wr.double().requires_grad_()
    e = w[ids] * scale
    p = torch.softmax(e @ wr, 1)
    g = p.gather(1, idx.long())                                     # gates as they are: the experts' share of a token is their sum
    x = e * (1 + g.sum(1, keepdim=True))
    s = x @ w.T
    on = targets >= 0
    ce = (torch.logsumexp(s, 1) - s.gather(1, targets.clamp(min=0)[:, None])[:, 0])[on].mean()
    T, E = p.shape
    counts = torch.bincount(idx.flatten().long(), minlength=E).double()
    balance = E / (k * T * T) * (counts * p.sum(0)).sum()
    (ce + COEF * balance).backward()
    return ce, balance, w.grad, wr.grad


@pytest.mark.parametrize("p", [1, 2])
def test_training_step(p):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.manual_seed(5)
    cfg = L.CommConfig.default()
    cfg.hcclBufferSize = 2
    c = H.Communicator.init_local(p, device=True, device_id=0, config=cfg)
    T, V, hidden, E, k, scale = 300, 512, 128, 16, 4, 4.0
    w = (torch.randn(V, hidden, device="cuda") * 0.1).to(torch.bfloat16)
    wr = (torch.randn(hidden, E, device="cuda") * 0.3).to(torch.bfloat16)
    ids = torch.randint(0, V, (T,), device="cuda")
    targets = torch.where(torch.rand(T, device="cuda") < 0.1, -100, torch.randint(0, V, (T,), device="cuda"))
    shards, firsts = list(w.chunk(p)), vocab.first_ids(c, V // p)
    ex = moe.MoEExchange(c, T, hidden, E, k, capacity_factor=float(p))
    many = (lambda t: [t] * p) if p > 1 else (lambda t: t)
    one = (lambda t: t[0]) if p > 1 else (lambda t: t)

    # forward: every rank has the same tokens, a shard of the vocabulary, and E / p of the experts (which leave rows as they are)
    e = vocab.vocab_parallel_embedding(c, [ids] * p, shards, scale)[0]
    logits = e.float() @ wr.float()
    g = moe.gate(logits, k, normalize=False)
    ex.dispatch(many(e), many(g.idx))
    x = (e.float() + one(ex.combine(many(g.gates), source="recv")).float()).to(torch.bfloat16)

    # backward
    grads = [torch.zeros(V // p, hidden, device="cuda") for _ in range(p)]
    out = vocab.vocab_parallel_cross_entropy_grad(c, [x] * p, shards, [targets] * p, dw=grads)
    assert c.sync() == 0, c.describe_status()
    loss, dx, _ = out[0]
    d_gates = (dx.float() * e.float()).sum(1, keepdim=True).expand(T, k).contiguous()
    d_logits = moe.gate_grad(logits, g, d_gates, balance=COEF, normalize=False)
    de = dx.float() * (1 + g.gates.sum(1, keepdim=True)) + d_logits @ wr.float().T
    for shard, first in zip(grads, firsts):
        vocab.embedding_grad(ids, de, V // p, scale, first_id=first, out=shard, add=True)
    ce, balance, dw, dwr = exact(ids, targets, w, wr, k, scale, g.idx)

    # roundings to bf16 on the way of any value: e, combine's, x, d, dx (and the sum of its shards): seven half steps at most
    seven = 7 * 2.0 ** -8
    ce, balance = float(ce.detach()), float(balance.detach())
    assert abs(float(loss) - ce) <= seven * ce and abs(float(g.balance) - balance) <= seven * balance
    assert float((torch.cat(grads).double() - dw).norm()) <= seven * float(dw.norm())
    assert float(((e.float().T @ d_logits).double() - dwr).norm()) <= seven * float(dwr.norm())
    ex.close()
    c.destroy()
