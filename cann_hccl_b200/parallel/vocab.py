"""The ends of a model that know the vocabulary: the token embedding, and the loss over the vocabulary, with their gradients.

    embedding(ids, w, scale)                          -> scale * w[ids]
    embedding_grad(ids, dy, vocab, scale)             -> gradient of w (rows of equal tokens summed, others zero)
    vocab_parallel_embedding(comm, ids, w)            -> the same where every rank holds vocab / p rows of w
    linear_cross_entropy(x, w, targets)               -> softmax cross entropy of the logits x @ w.T, which are never stored
    linear_cross_entropy_grad(x, w, targets)          -> (loss, dx, dw)
    vocab_parallel_cross_entropy(comm, x, w, targets) and vocab_parallel_cross_entropy_grad: w sharded over the ranks

Rows of a shard are ids first_id .. first_id + rows - 1; ids outside it (other ranks' rows, padding ids below zero) give zeros and have
no gradient.  On an all-local communicator w (and what is per rank) is a list with one tensor per virtual rank.  Gradients are calls of
their own, as everywhere in this package: results carry no automatic differentiation.
"""
import ctypes as C
import struct

import torch

from .. import _lib as L
from ..ops.comm import _raw_stream
from ..utils.dtypes import float_codes
from ..utils.tensors import check_out, on_device_of

_IDS = {torch.int32: L.INT32, torch.int64: L.INT64}
_FLOAT = float_codes()


def _check_ids(ids, device):
    if not (torch.is_tensor(ids) and ids.is_cuda and ids.dtype in _IDS and ids.device == device and ids.is_contiguous()):
        raise ValueError("ids must be a contiguous int32 or int64 CUDA tensor on the device of the rows")


def _check_rows(t, name):
    """[rows, hidden] whose rows lie in one piece each; returns rows, hidden and the elements between rows."""
    if not (torch.is_tensor(t) and t.is_cuda and t.dim() == 2 and 0 < t.shape[1] < 1 << 31):
        raise ValueError("%s must be a CUDA tensor [rows, hidden]" % name)
    if t.dtype not in _FLOAT:
        raise TypeError("%s must be fp32, fp16 or bf16, got %s" % (name, t.dtype))
    (n, h), (a, b) = t.shape, t.stride()
    if h > 1 and b != 1 or n > 1 and a < h:
        raise ValueError("rows of %s must lie in one piece each (strides %s)" % (name, (a, b)))
    return n, h, a if n > 1 else h


def embedding(ids, w, scale=1.0, first_id=0, out=None):
    """scale * w[ids - first_id] -> [*ids.shape, hidden]; ids outside the rows of w give zeros.  The product is rounded once."""
    vocab, hidden, stride = _check_rows(w, "w")
    _check_ids(ids, w.device)
    with on_device_of(w):
        if out is None:
            out = w.new_empty((*ids.shape, hidden))
        else:
            check_out(out, (*ids.shape, hidden), w.dtype, w.device)
        L.lib()
        rc = L.fast.embedding(ids, _IDS[ids.dtype], ids.numel(), w, stride, vocab, first_id, hidden, _FLOAT[w.dtype], scale, out, _raw_stream())
        if rc:
            L.check(rc, "HcclB200Embedding")
    return out


def embedding_grad(ids, dy, vocab, scale=1.0, first_id=0, out=None, add=False):
    """Gradient of embedding()'s w: [vocab, hidden] of dy's type, the fp32 sums of dy's rows by token, in token order (the same bits every
    time), times scale.  With `add` the sums are added to `out`, an fp32 tensor (gradients of several batches, or of a tied weight)."""
    if not (torch.is_tensor(dy) and dy.dim() >= 1) or dy.shape[:-1] != ids.shape:
        raise ValueError("dy must be [*ids.shape, hidden]")
    rows = dy if dy.dim() == 2 else dy.reshape(-1, dy.shape[-1])
    _, hidden, stride = _check_rows(rows, "dy")
    _check_ids(ids, rows.device)
    with on_device_of(rows):
        if out is None:
            if add:
                raise ValueError("add needs the fp32 tensor to add to")
            out = rows.new_empty((vocab, hidden))
        else:
            check_out(out, (vocab, hidden), torch.float32 if add else rows.dtype, rows.device)
        n, lib = ids.numel(), L.lib()
        scratch = rows.new_empty(max(0, lib.HcclB200EmbeddingGradScratchBytes(n, vocab, hidden)), dtype=torch.uint8)
        rc = L.fast.embedding_grad(ids, _IDS[ids.dtype], n, rows, stride, vocab, first_id, hidden, _FLOAT[rows.dtype], scale, out, _FLOAT[out.dtype],
                                   int(add), scratch, _raw_stream())
        if rc:
            L.check(rc, "HcclB200EmbeddingGrad")
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


def _check_shards(comm, ws):
    """Refuses shards of several sizes: first ids follow from one.  Ranks of other processes are asked over the control plane, at the first
    call with a size (on every rank, since all of them have the same calls)."""
    rows = [t.shape[0] for t in ws]
    # a communicator without a control plane cannot be asked
    if comm.nlocal < comm.nranks and hasattr(comm, "exchange"):
        known = comm.__dict__.setdefault("_shard_rows", set())
        if rows[0] in known:
            return
        rows = [struct.unpack("<q", b)[0] for b in comm.exchange("vocab-rows", struct.pack("<q", rows[0]))]
        if len(set(rows)) == 1:
            known.add(rows[0])
    if len(set(rows)) > 1:
        raise ValueError("all ranks need shards of one size, they have %s rows: pad the vocabulary" % rows)


def vocab_parallel_embedding(comm, ids, w, scale=1.0):
    """Every rank holds vocab / p rows of the table (rank r the ids from r * rows on, the same number on all ranks) and the same ids: the
    lookups are summed over the ranks (all but one are zero, so nothing is rounded twice).  Its gradient is embedding_grad() with the shard's first_id."""
    ids_l, ws = _per_rank(comm, ids, w)
    _check_shards(comm, ws)
    outs = [embedding(i, t, scale, first) for i, t, first in zip(ids_l, ws, first_ids(comm, ws[0].shape[0]))]
    if comm.nranks > 1 and outs[0].numel():
        comm.all_reduce(outs, outs)
    return outs if isinstance(w, (list, tuple)) else outs[0]


# ---------------------------------------------------------------------------------------------------------- loss
_BF16_OUT, _F32_OUT, _ADD, _ADD_BF16 = range(4)


def _check_loss(x, w, targets, weights, reduction):
    for t, name in ((x, "x"), (w, "w")):
        _, h, stride = _check_rows(t, name)
        if t.dtype != torch.bfloat16:
            raise TypeError("%s must be bf16, got %s" % (name, t.dtype))
        if h % 8 or stride % 8 or t.data_ptr() % 16:
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
        (self.T, self.H), self.V = x.shape, w.shape[0]
        self._xs, ws = x.stride(0) if self.T > 1 else self.H, w.stride(0) if self.V > 1 else self.H
        self._x, self._y, self._ysize = x.data_ptr(), targets.data_ptr(), targets.element_size()
        self._q = None if weights is None else weights.data_ptr()
        self._call = L.VocabLoss(self._x, w.data_ptr(), self._xs, ws, self._y, self._q, self.T, self.V, first, whole, ignore,
                                 self.H, _IDS[targets.dtype])

    def part(self, a, b, losses=None):
        """The call for tokens a to b (the structure is the shard's: valid until the next one); losses: address of theirs."""
        c = self._call
        c.losses = losses
        c.x, c.targets, c.tokens = self._x + a * self._xs * 2, self._y + a * self._ysize, b - a
        if self._q is not None:
            c.weights = self._q + a * 4
        return C.byref(c)

    def scratch(self, n):
        """Bytes of the scratch that the calls of part() are given."""
        self._call.scratchBytes = n

    def new(self, shape, dtype=torch.float32):
        return self.x.new_empty(shape, dtype=dtype)


def _run_loss(shards, comm, reduction, scale=1.0, outs=None, grad=False):
    """The loss of shards that share their tokens (those of this process), chunk by chunk; with `grad` dx and dw of each."""
    lib, st, check, s0 = L.lib(), _raw_stream(), L.check, shards[0]
    T, alone, none = s0.T, comm is None or comm.nranks == 1, reduction == "none"
    chunk = min(max(T, 1), min(lib.HcclB200VocabLossChunk(s.V, int(grad)) for s in shards))
    losses = [s.new(T) for s in shards]
    sizes = {min(chunk, T), T % chunk}  # tokens of the chunks: a short last one may need more scratch than a whole one
    # fp32 words of each shard behind its scratch: lse and target logit of a chunk, the joint lse, the sum of the weights
    mem, words = [], []
    for s in shards:
        needs = [lib.HcclB200VocabLossScratchBytes(n, s.V, s.H, int(grad)) for n in sizes]
        if min(needs) < 0:
            raise RuntimeError("no scratch size for %d tokens, %d rows of %d" % (chunk, s.V, s.H))
        n = (max(needs) + 255) // 256 * 256
        s.scratch(n)
        m = s.new(n + (3 * chunk + 1) * 4, torch.uint8)
        mem.append(m)
        words.append(m.data_ptr() + n)
    totals = [p + 12 * chunk if reduction == "mean" else None for p in words]
    if reduction == "mean":
        for s, p in zip(shards, totals):
            check(lib.HcclB200VocabLossTotal(s.part(0, T), p, st), "HcclB200VocabLossTotal")
    if grad:
        dxs = [s.new((T, s.H), torch.bfloat16) for s in shards]
        several = T > chunk
        sums = [o if o is not None else s.new((s.V, s.H)) if several else None for s, o in zip(shards, outs)]
        dws = [o if o is not None else s.new((s.V, s.H), torch.bfloat16) for s, o in zip(shards, outs)]
    for a in range(0, T, chunk):
        b = min(T, a + chunk)
        n = b - a
        for s, m, p, loss in zip(shards, mem, words, losses):
            check(lib.HcclB200VocabLossScores(s.part(a, b), int(grad), p, p + n * 4, loss.data_ptr() + a * 4 if alone else None, m.data_ptr(), st), "HcclB200VocabLossScores")
        if not alone:
            every = [s.new((comm.nranks, 2, n)) for s in shards]
            mine = [m[p - m.data_ptr():p - m.data_ptr() + 8 * n].view(torch.float32) for m, p in zip(mem, words)]
            comm.all_gather(mine, every)
            for s, e, p, loss in zip(shards, every, words, losses):
                check(lib.HcclB200VocabLossCombine(s.part(a, b), e.data_ptr(), comm.nranks, p + 8 * chunk, loss.data_ptr() + a * 4, st), "HcclB200VocabLossCombine")
        if grad:
            for i, (s, m, p, loss) in enumerate(zip(shards, mem, words, losses)):
                kind = _ADD if outs[i] is not None else _BF16_OUT if not several else _F32_OUT if a == 0 else _ADD if b < T else _ADD_BF16
                check(lib.HcclB200VocabLossGrad(s.part(a, b, loss.data_ptr() + a * 4), p if alone else p + 8 * chunk, p + n * 4, totals[i], scale, dxs[i].data_ptr() + a * s.H * 2,
                                                dws[i].data_ptr(), None if sums[i] is None else sums[i].data_ptr(), kind, m.data_ptr(), st), "HcclB200VocabLossGrad")
    if grad and not T:
        for o, d in zip(outs, dws):
            if o is None:
                d.zero_()
    if grad and not alone and T:
        comm.all_reduce(dxs, dxs)
    if not none:
        for i, (s, loss) in enumerate(zip(shards, losses)):
            out = s.new(())
            check(lib.HcclB200VocabLossSum(s.part(0, T), loss.data_ptr(), totals[i], out.data_ptr(), st), "HcclB200VocabLossSum")
            losses[i] = out
    return list(zip(losses, dxs, dws)) if grad else losses


_STEP_MOST = 65536


def _step(s, reduction, scale, dw):
    """Loss and gradients of a lone shard whose tokens are one chunk: one call of the library."""
    n = L.lib().HcclB200VocabLossStepBytes(s.T, s.V, s.H)
    if n < 0:
        raise RuntimeError("no scratch size for %d tokens, %d rows of %d" % (s.T, s.V, s.H))
    s.scratch(n)
    mem, loss, dx = s.new(n, torch.uint8), s.new(()), s.new((s.T, s.H), torch.bfloat16)
    out = s.new((s.V, s.H), torch.bfloat16) if dw is None else dw
    at = out.data_ptr()
    rc = L.lib().HcclB200VocabLossStep(s.part(0, s.T), int(reduction == "mean"), scale, loss.data_ptr(), dx.data_ptr(), at, at if dw is not None else None,
                                       _BF16_OUT if dw is None else _ADD, mem.data_ptr(), _raw_stream())
    if rc:
        L.check(rc, "HcclB200VocabLossStep")
    return loss, dx, out


def linear_cross_entropy(x, w, targets, weights=None, reduction="mean", ignore_index=-100):
    """Softmax cross entropy of the logits x [tokens, hidden] @ w [vocab, hidden].T (bf16, fp32 sums) against `targets` (int32 or int64).
    Tokens whose target is ignore_index or no id of the vocabulary do not count.  `weights`: fp32 [tokens].  reduction: "none" gives
    the unweighted losses [tokens] (0 where a token does not count), "sum" their weighted sum, "mean" that divided by the sum of the
    weights that count (0 where there is none).  The logits are not stored: beyond arguments and results it takes about 130 MB at
    most (for 256 tokens at least) and, for more than 128 tokens whose hidden size is no multiple of 64, a copy of x (of a chunk of tokens,
    at most 2^20).
    The tensor cores' fp32 sums lean towards zero; they are taken in parts of about 1024 elements, whatever hidden is, and losses come out low by
    1e-7 of themselves at 10, 3e-6 at 0.1 (means of 256 tokens)."""
    _check_loss(x, w, targets, weights, reduction)
    with on_device_of(x):
        return _run_loss([_Shard(x, w, targets, weights, 0, w.shape[0], ignore_index)], None, reduction)[0]


def linear_cross_entropy_grad(x, w, targets, weights=None, reduction="mean", ignore_index=-100, scale=1.0, dw=None):
    """(loss, dx, dw): the loss as linear_cross_entropy() gives it ("mean" or "sum") and the gradients of scale * loss.  dx and dw are bf16;
    given an fp32 tensor `dw` [vocab, hidden], the weight's gradient is added to it (several batches, or a weight that the embedding
    shares) and it is returned.  Beyond the results it takes, for a chunk of tokens (a thousand million logits, 256 to 2^20 tokens), a copy of
    the chunk's x and about 3 GB at most up to hidden 16384 (exponentials, row sums, fp32 shares of dx); and an fp32 sum of dw where the
    tokens are more than one chunk."""
    _check_loss(x, w, targets, weights, reduction)
    if reduction == "none":
        raise ValueError("gradients need a sum or mean over the tokens (weights scale each token)")
    if dw is not None:
        check_out(dw, w.shape, torch.float32, w.device)
    with on_device_of(x):
        s = _Shard(x, w, targets, weights, 0, w.shape[0], ignore_index)
        if 0 < s.T <= min(_STEP_MOST, L.lib().HcclB200VocabLossChunk(s.V, 1)):
            return _step(s, reduction, scale, dw)
        return _run_loss([s], None, reduction, scale, [dw], True)[0]


def _sharded(comm, x, w, targets, weights, reduction, ignore_index):
    xs, ws, ys, qs = _per_rank(comm, x, w, targets, [None] * comm.nlocal if weights is None else weights)
    for a in zip(xs, ws, ys, qs):
        _check_loss(*a, reduction)
    if len({t.shape for t in xs}) > 1 or len({t.shape for t in ws}) > 1:
        raise ValueError("all ranks need the same tokens and shards of one size")
    _check_shards(comm, ws)
    whole = ws[0].shape[0] * comm.nranks
    return [_Shard(*a, f, whole, ignore_index) for a, f in zip(zip(xs, ws, ys, qs), first_ids(comm, ws[0].shape[0]))]


def vocab_parallel_cross_entropy(comm, x, w, targets, weights=None, reduction="mean", ignore_index=-100):
    """linear_cross_entropy() where every rank holds vocab / p rows of w (rank r the ids from r * rows on, the same number on all ranks), and
    the same x, targets and weights.  The ranks exchange two numbers for each token."""
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
