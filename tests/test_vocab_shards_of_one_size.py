"""The vocabulary-parallel operators want shards of one size: others are refused, in one process and over several."""
import os
import subprocess
import sys
import types

import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200.parallel import vocab  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))

# A rank of several on the CPU.  The operators' launches are stood in for; the exchange between the ranks is the communicator's own.
PROG = """
import sys
sys.path.insert(0, {here!r})
from _worker import make_comm
import contextlib
import torch
from cann_hccl_b200.parallel import vocab
p, rank = {p}, int(sys.argv[1])
c = make_comm(p, rank, {root!r})
launches, asked = [], []
exchange = c.exchange
c.exchange = lambda *a: (asked.append(a), exchange(*a))[1]
vocab._check_loss = lambda *a: None
vocab.on_device_of = lambda t: contextlib.nullcontext()
vocab.embedding = lambda ids, w, scale, first: launches.append(first) or torch.zeros(len(ids), w.shape[1])
vocab._run_loss = lambda shards, *a: launches.append((shards[0]._call.firstId, shards[0]._call.wholeVocab)) or [None]
c.all_reduce = lambda *a: None
x, y = torch.zeros(5, 16, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int64)
calls = (lambda w: vocab.vocab_parallel_embedding(c, y, w), lambda w: vocab.vocab_parallel_cross_entropy(c, x, w, y),
         lambda w: vocab.vocab_parallel_cross_entropy_grad(c, x, w, y))
odd = torch.zeros(12565 - 3 * (rank == p - 1), 16, dtype=torch.bfloat16)     # 50257 ids over four: the last rank has fewer
for call in calls:
    try:
        call(odd)
    except ValueError as e:
        assert "12562" in str(e) and "12565" in str(e), e
    else:
        raise AssertionError("taken")
assert not launches and len(asked) == 3
even = torch.zeros(12565, 16, dtype=torch.bfloat16)
for call in calls + calls:
    call(even)
assert launches == [12565 * rank, (12565 * rank, 12565 * p), (12565 * rank, 12565 * p)] * 2 and len(asked) == 4  # asked once for a size
c.destroy()
print("shards ok")
"""


@pytest.mark.parametrize("p", [2, 4])
def test_over_processes(p, tmp_path):
    prog = PROG.format(here=HERE, p=p, root=str(tmp_path / "root.bin"))
    env = dict(os.environ, HCCL_TRANSPORT="host", HCCL_CONNECT_TIMEOUT="30", PYTHONPATH=os.path.dirname(HERE))
    ranks = [subprocess.Popen([sys.executable, "-c", prog, str(r)], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for r in range(p)]
    outs = [r.communicate(timeout=90)[0] for r in ranks]
    assert all(r.returncode == 0 for r in ranks) and all("shards ok" in o for o in outs), "\n".join(outs)


def test_in_one_process(monkeypatch):
    monkeypatch.setattr(vocab, "_check_loss", lambda *a: None)
    monkeypatch.setattr(vocab, "embedding", lambda *a: pytest.fail("launched"))
    c = types.SimpleNamespace(nranks=2, nlocal=2, rank=0)
    x, y = torch.zeros(5, 16, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int64)
    ws = [torch.zeros(n, 16, dtype=torch.bfloat16) for n in (7, 6)]
    for call in (lambda: vocab.vocab_parallel_embedding(c, [y, y], ws), lambda: vocab.vocab_parallel_cross_entropy(c, [x, x], ws, [y, y]),
                 lambda: vocab.vocab_parallel_cross_entropy_grad(c, [x, x], ws, [y, y])):
        with pytest.raises(ValueError, match="one size"):
            call()
