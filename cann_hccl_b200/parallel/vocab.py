"""The ends of a model that know the vocabulary: the token embedding and its gradient.

    embedding(ids, w, scale)                    -> scale * w[ids]
    embedding_grad(ids, dy, vocab, scale)       -> gradient of w (rows of equal tokens summed, others zero)
    vocab_parallel_embedding(comm, ids, w)      -> the same where every rank holds vocab / p rows of w

Rows of a shard are ids first_id .. first_id + rows - 1; ids outside it (other ranks' rows, padding ids below zero) give zeros and have
no gradient.  On an all-local communicator w (and what is per rank) is a list with one tensor per virtual rank.
"""
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
