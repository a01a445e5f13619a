"""The ends of a model that know the vocabulary: the token embedding, and the loss over the vocabulary, with their gradients.

    embedding(ids, w, scale)                          -> scale * w[ids]
    embedding_grad(ids, dy, vocab, scale)             -> gradient of w (rows of equal tokens summed, others zero)
    vocab_parallel_embedding(comm, ids, w)            -> the same where every rank holds vocab / p rows of w
    linear_cross_entropy(x, w, targets)               -> softmax cross entropy of the logits x @ w.T, which are never stored
    linear_cross_entropy_grad(x, w, targets)          -> (loss, dx, dw)
    vocab_parallel_cross_entropy(comm, x, w, targets) and vocab_parallel_cross_entropy_grad: w sharded over the ranks

Rows of a shard are ids first_id .. first_id + rows - 1; ids outside it (other ranks' rows, padding ids below zero) give zeros and have
no gradient.  On an all-local communicator w (and what is per rank) is a list with one tensor per virtual rank.
"""
import ctypes as C

import torch

from .. import _lib as L
from ..ops.comm import _raw_stream
from ..utils.dtypes import float_code
from ..utils.tensors import check_out, on_device_of

_IDS = {torch.int32: L.INT32, torch.int64: L.INT64}


def _check_ids(ids, device):
    if not (torch.is_tensor(ids) and ids.is_cuda and ids.dtype in _IDS and ids.device == device and ids.is_contiguous()):
        raise ValueError("ids must be a contiguous int32 or int64 CUDA tensor on the device of the rows")


def _check_rows(t, name):
    """[rows, hidden] whose rows lie in one piece each; returns the elements between rows."""
    if not (torch.is_tensor(t) and t.is_cuda and t.dim() == 2 and t.shape[1] > 0):
        raise ValueError("%s must be a CUDA tensor [rows, hidden]" % name)
    if float_code(t.dtype) is None:
        raise TypeError("%s must be fp32, fp16 or bf16, got %s" % (name, t.dtype))
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("rows of %s must lie in one piece each (strides %s)" % (name, tuple(t.stride())))
    return max(t.shape[1], t.stride(0))


def embedding(ids, w, scale=1.0, first_id=0, out=None):
    """scale * w[ids - first_id] -> [*ids.shape, hidden]; ids outside the rows of w give zeros.  The product is rounded once."""
    stride = _check_rows(w, "w")
    _check_ids(ids, w.device)
    with on_device_of(w):
        if out is None:
            out = torch.empty((*ids.shape, w.shape[1]), device=w.device, dtype=w.dtype)
        else:
            check_out(out, (*ids.shape, w.shape[1]), w.dtype, w.device)
        L.check(L.lib().HcclB200Embedding(ids.data_ptr(), _IDS[ids.dtype], ids.numel(), w.data_ptr(), stride, w.shape[0], first_id, w.shape[1],
                                          float_code(w.dtype), scale, out.data_ptr(), _raw_stream()), "HcclB200Embedding")
    return out


def embedding_grad(ids, dy, vocab, scale=1.0, first_id=0, out=None, add=False):
    """Gradient of embedding()'s w: [vocab, hidden] of dy's type, the fp32 sums of dy's rows by token, in token order (the same bits every
    time), times scale.  With `add` the sums are added to `out`, an fp32 tensor (gradients of several batches, or of a tied weight)."""
    if not (torch.is_tensor(dy) and dy.dim() >= 1) or tuple(dy.shape[:-1]) != tuple(ids.shape):
        raise ValueError("dy must be [*ids.shape, hidden]")
    rows = dy if dy.dim() == 2 else dy.reshape(-1, dy.shape[-1])
    stride, hidden = _check_rows(rows, "dy"), rows.shape[1]
    _check_ids(ids, rows.device)
    with on_device_of(rows):
        if out is None:
            if add:
                raise ValueError("add needs the fp32 tensor to add to")
            out = torch.empty(vocab, hidden, device=rows.device, dtype=rows.dtype)
        else:
            check_out(out, (vocab, hidden), torch.float32 if add else rows.dtype, rows.device)
        lib = L.lib()
        scratch = torch.empty(max(0, lib.HcclB200EmbeddingGradScratchBytes(ids.numel(), vocab, hidden)), device=rows.device, dtype=torch.uint8)
        L.check(lib.HcclB200EmbeddingGrad(ids.data_ptr(), _IDS[ids.dtype], ids.numel(), rows.data_ptr(), stride, vocab, first_id, hidden,
                                          float_code(rows.dtype), scale, out.data_ptr(), float_code(out.dtype), int(add), scratch.data_ptr(),
                                          _raw_stream()), "HcclB200EmbeddingGrad")
    return out


def _per_rank(comm, *xs):
    out = []
    for x in xs:
        x = list(x) if isinstance(x, (list, tuple)) else [x]
        if len(x) != comm.nlocal:
            raise ValueError("one tensor per local rank is needed")
        out.append(x)
    return out


def first_ids(comm, vocab_rows):
    """First token id of each local rank's shard, for shards of equal size."""
    return [r * vocab_rows for r in (range(comm.nranks) if comm.nlocal > 1 else [comm.rank])]


def vocab_parallel_embedding(comm, ids, w, scale=1.0):
    """Every rank holds vocab / p rows of the table (rank r the ids from r * rows on) and the same ids: the lookups are summed over the
    ranks (all but one are zero, so nothing is rounded twice).  Its gradient is embedding_grad() with the shard's first_id."""
    ids_l, ws = _per_rank(comm, ids, w)
    outs = [embedding(i, t, scale, first) for i, t, first in zip(ids_l, ws, first_ids(comm, ws[0].shape[0]))]
    if comm.nranks > 1 and outs[0].numel():
        comm.all_reduce(outs, outs)
    return outs if isinstance(w, (list, tuple)) else outs[0]


# ---------------------------------------------------------------------------------------------------------- loss
_BF16_OUT, _F32_OUT, _ADD, _ADD_BF16 = range(4)


def _check_loss(x, w, targets, weights, reduction):
    """[(x, w, strides)] of one shard; the rest of the arguments."""
    for t, name in ((x, "x"), (w, "w")):
        stride = _check_rows(t, name)
        if t.dtype != torch.bfloat16:
            raise TypeError("%s must be bf16, got %s" % (name, t.dtype))
        if t.shape[1] % 8 or stride % 8 or t.data_ptr() % 16:
            raise ValueError("rows of %s must be multiples of 8 elements that start on 16-byte boundaries" % name)
    if x.shape[1] != w.shape[1] or x.device != w.device or not w.shape[0]:
        raise ValueError("x %s and w %s must have the same hidden size and device" % (tuple(x.shape), tuple(w.shape)))
    _check_ids(targets, x.device)
    if targets.shape != x.shape[:1]:
        raise ValueError("targets must be [tokens]")
    if weights is not None and not (weights.device == x.device and weights.dtype == torch.float32 and weights.shape == x.shape[:1] and weights.is_contiguous()):
        raise ValueError("weights must be a contiguous fp32 tensor [tokens]")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be mean, sum or none")


class _Shard:
    """One shard's tensors, and the call structure of a stretch of its tokens."""

    def __init__(self, x, w, targets, weights, first, whole, ignore):
        self.x, self.w, self.targets, self.weights = x, w, targets, weights
        self.first, self.whole, self.ignore = first, whole, ignore
        self.T, self.V, self.H = x.shape[0], w.shape[0], w.shape[1]

    def part(self, a, b):
        x, w, y, q = self.x, self.w, self.targets, self.weights
        return C.byref(L.VocabLoss(x=x.data_ptr() + a * x.stride(0) * 2, w=w.data_ptr(), xStride=max(self.H, x.stride(0)), wStride=max(self.H, w.stride(0)),
                                   targets=y.data_ptr() + a * y.element_size(), weights=None if q is None else q.data_ptr() + a * 4, tokens=b - a,
                                   vocab=self.V, firstId=self.first, wholeVocab=self.whole, ignoreId=self.ignore, hidden=self.H, targetType=_IDS[y.dtype]))

    def new(self, shape, dtype=torch.float32):
        return torch.empty(shape, device=self.x.device, dtype=dtype)

    def scratch(self, tokens, grad):
        n = L.lib().HcclB200VocabLossScratchBytes(tokens, self.V, self.H, int(grad))
        if n < 0:
            raise RuntimeError("no scratch size for %d tokens, %d rows of %d" % (tokens, self.V, self.H))
        return self.new(n, torch.uint8)


def _at(t, a):
    return None if t is None else t.data_ptr() + a * t.element_size()


def _run_loss(shards, comm, reduction, scale=1.0, outs=None, grad=False):
    """The loss of shards that share their tokens (those of this process), chunk by chunk; with `grad` dx and dw of each."""
    lib, st, s0 = L.lib(), _raw_stream(), shards[0]
    T, alone = s0.T, comm is None or comm.nranks == 1
    chunk = min(max(T, 1), min(lib.HcclB200VocabLossChunk(s.V, int(grad)) for s in shards))
    losses = [s.new(T) for s in shards]
    total = None
    if reduction == "mean":
        total = [s.new(()) for s in shards]
        for s, t in zip(shards, total):
            L.check(lib.HcclB200VocabLossTotal(s.part(0, T), t.data_ptr(), st), "HcclB200VocabLossTotal")
    parts = [s.new((2, chunk)) for s in shards]                    # lse and target logits of a chunk
    joint = parts if alone else [s.new(chunk) for s in shards]
    scratch = [s.scratch(chunk, grad) for s in shards] if T else None
    if grad:
        dxs = [s.new((T, s.H), torch.bfloat16) for s in shards]
        several = T > chunk
        sums = [o if o is not None else s.new((s.V, s.H)) if several else None for s, o in zip(shards, outs)]
        dws = [o if o is not None else s.new((s.V, s.H), torch.bfloat16) for s, o in zip(shards, outs)]
    for a in range(0, T, chunk):
        b = min(T, a + chunk)
        n = b - a
        for s, p, mem, loss in zip(shards, parts, scratch, losses):
            L.check(lib.HcclB200VocabLossScores(s.part(a, b), int(grad), p.data_ptr(), p.data_ptr() + n * 4, _at(loss, a) if alone else None, mem.data_ptr(), st),
                    "HcclB200VocabLossScores")
        if not alone:
            every = [s.new((comm.nranks, 2, n)) for s in shards]
            mine = [p.view(-1)[:2 * n] for p in parts]
            comm.all_gather(mine, every)
            for s, e, lse, loss in zip(shards, every, joint, losses):
                L.check(lib.HcclB200VocabLossCombine(s.part(a, b), e.data_ptr(), comm.nranks, lse.data_ptr(), _at(loss, a), st), "HcclB200VocabLossCombine")
        if grad:
            for i, (s, p, lse, mem) in enumerate(zip(shards, parts, joint, scratch)):
                kind = _ADD if outs[i] is not None else _BF16_OUT if not several else _F32_OUT if a == 0 else _ADD if b < T else _ADD_BF16
                L.check(lib.HcclB200VocabLossGrad(s.part(a, b), lse.data_ptr(), p.data_ptr() + n * 4, _at(total and total[i], 0), scale,
                                                  dxs[i].data_ptr() + a * s.H * 2, dws[i].data_ptr(), _at(sums[i], 0), kind, mem.data_ptr(), st),
                        "HcclB200VocabLossGrad")
    if grad and not T:
        for o, d in zip(outs, dws):
            if o is None:
                d.zero_()
    if grad and not alone and T:
        comm.all_reduce(dxs, dxs)
    if reduction != "none":
        for i, (s, loss) in enumerate(zip(shards, losses)):
            out = s.new(())
            L.check(lib.HcclB200VocabLossSum(s.part(0, T), loss.data_ptr(), _at(total and total[i], 0), out.data_ptr(), st), "HcclB200VocabLossSum")
            losses[i] = out
    return list(zip(losses, dxs, dws)) if grad else losses


def linear_cross_entropy(x, w, targets, weights=None, reduction="mean", ignore_index=-100):
    """Softmax cross entropy of the logits x [tokens, hidden] @ w [vocab, hidden].T (bf16, fp32 sums) against `targets` (int32 or int64).
    Tokens whose target is ignore_index or no id of the vocabulary do not count.  `weights`: fp32 [tokens].  reduction: "none" gives
    the unweighted losses [tokens] (0 where a token does not count), "sum" their weighted sum, "mean" that divided by the sum of the
    weights that count (0 where there is none).  The logits are not stored: memory beyond the arguments is bounded by 128 MB."""
    _check_loss(x, w, targets, weights, reduction)
    with on_device_of(x):
        return _run_loss([_Shard(x, w, targets, weights, 0, w.shape[0], ignore_index)], None, reduction)[0]


def linear_cross_entropy_grad(x, w, targets, weights=None, reduction="mean", ignore_index=-100, scale=1.0, dw=None):
    """(loss, dx, dw): the loss as linear_cross_entropy() gives it ("mean" or "sum") and the gradients of scale * loss.  dx and dw are bf16;
    given an fp32 tensor `dw` [vocab, hidden], the weight's gradient is added to it (several batches, or a weight that the embedding
    shares) and it is returned.  Beyond the results it takes 2 GiB at most, for the exponentials of a chunk of tokens, and an fp32 sum of
    dw where the tokens are more than one chunk (16 thousand million logits)."""
    _check_loss(x, w, targets, weights, reduction)
    if reduction == "none":
        raise ValueError("gradients need a sum or mean over the tokens (weights scale each token)")
    if dw is not None:
        check_out(dw, w.shape, torch.float32, w.device)
    with on_device_of(x):
        return _run_loss([_Shard(x, w, targets, weights, 0, w.shape[0], ignore_index)], None, reduction, scale, [dw], True)[0]


def _sharded(comm, x, w, targets, weights, reduction, ignore_index):
    xs, ws, ys, qs = _per_rank(comm, x, w, targets, [None] * comm.nlocal if weights is None else weights)
    for a in zip(xs, ws, ys, qs):
        _check_loss(*a, reduction)
    if len({t.shape for t in xs}) > 1 or len({t.shape for t in ws}) > 1:
        raise ValueError("all ranks need the same tokens and shards of one size")
    whole = ws[0].shape[0] * comm.nranks
    return [_Shard(*a, f, whole, ignore_index) for a, f in zip(zip(xs, ws, ys, qs), first_ids(comm, ws[0].shape[0]))]


def vocab_parallel_cross_entropy(comm, x, w, targets, weights=None, reduction="mean", ignore_index=-100):
    """linear_cross_entropy() where every rank holds vocab / p rows of w (rank r the ids from r * rows on), and the same x, targets and
    weights.  The ranks exchange two numbers for each token."""
    shards = _sharded(comm, x, w, targets, weights, reduction, ignore_index)
    with on_device_of(shards[0].x):
        out = _run_loss(shards, comm, reduction)
    return out if isinstance(w, (list, tuple)) else out[0]


def vocab_parallel_cross_entropy_grad(comm, x, w, targets, weights=None, reduction="mean", ignore_index=-100, scale=1.0, dw=None):
    """linear_cross_entropy_grad() on shards: every rank gets the loss, the whole dx (bf16 parts summed over the ranks) and its shard's dw."""
    shards = _sharded(comm, x, w, targets, weights, reduction, ignore_index)
    if reduction == "none":
        raise ValueError("gradients need a sum or mean over the tokens (weights scale each token)")
    outs = _per_rank(comm, [None] * comm.nlocal if dw is None else dw)[0]
    for s, o in zip(shards, outs):
        if o is not None:
            check_out(o, s.w.shape, torch.float32, s.w.device)
    with on_device_of(shards[0].x):
        out = _run_loss(shards, comm, reduction, scale, outs, True)
    return out if isinstance(w, (list, tuple)) else out[0]
