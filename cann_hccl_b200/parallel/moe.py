"""MoE expert-parallel exchange on symmetric memory: dispatch (push rows to the expert owners) and combine (pull the
expert outputs and form the gate-weighted sum while receiving).

    ex = MoEExchange(comm, tokens, hidden, n_experts, topk)
    recv, expert_offsets, recv_rows = ex.dispatch(x, topk_idx)          # recv rows grouped by local expert
    ... run the local experts on recv[expert_offsets[e]:expert_offsets[e+1]] and write into ex.expert_out ...
    out = ex.combine(gates)                                              # [tokens, hidden]

The router in front of it, with the balance loss and the gradients of both:

    g = gate(logits, topk, mask=None)                                    # Gate(idx, gates, counts, prob_sum, routed, balance)
    recv, expert_offsets, recv_rows = ex.dispatch(x, g.idx)              # slots without an expert (-1) are skipped
    ...
    d_logits = gate_grad(logits, g, d_gates, balance=coefficient)        # of the routed tokens: g has the mask

Counts travel over the device (all-gather of the per-expert histogram); nothing synchronises with the host.  On an
all-local communicator every tensor argument is a list with one entry per virtual rank.
"""
import ctypes as C

import torch

from .. import _lib as L
from ..ops.comm import _raw_stream
from ..utils.dtypes import float_codes
from ..utils.tensors import check_out, on_device_of


class _DevPtr:
    """Exposes a raw device pointer to torch through the CUDA array interface (int16 elements)."""

    def __init__(self, ptr, nelem):
        self.__cuda_array_interface__ = {"shape": (nelem,), "typestr": "<i2", "data": (int(ptr), False), "version": 3}


def tensor_from_ptr(ptr, rows, cols, device):
    """bf16 [rows, cols] torch view of symmetric memory."""
    t = torch.as_tensor(_DevPtr(ptr, rows * cols), device=device)
    return t.view(torch.bfloat16).view(rows, cols)


class MoEExchange:
    def __init__(self, comm, tokens, hidden, n_experts, topk, capacity_factor=1.5, device="cuda"):
        assert n_experts % comm.nranks == 0 and hidden % 8 == 0
        self.comm, self.T, self.H, self.E, self.k = comm, tokens, hidden, n_experts, topk
        self.p, self.nl = comm.nranks, comm.nlocal
        self.El = n_experts // self.p
        self.cap = int(tokens * topk * capacity_factor + 127) // 128 * 128
        nbytes = self.cap * hidden * 2
        self.h_recv, recv_local = comm.mem_alloc(nbytes)
        self.h_out, out_local = comm.mem_alloc(nbytes)
        self.recv_tab, _, _ = comm.mem_query(self.h_recv)   # [local][rank]
        self.out_tab, _, _ = comm.mem_query(self.h_out)
        self.recv = [tensor_from_ptr(recv_local[l], self.cap, hidden, device) for l in range(self.nl)]
        self.expert_out = [tensor_from_ptr(out_local[l], self.cap, hidden, device) for l in range(self.nl)]
        mk = lambda n, dt=torch.int32: [torch.zeros(n, device=device, dtype=dt) for _ in range(self.nl)]
        self.hist, self.pos, self.counts = mk(n_experts), mk(tokens * topk), mk(self.p * n_experts)
        self.base, self.expert_offsets, self.recv_rows, self.overflow = mk(n_experts), mk(self.El + 1), mk(1), mk(1)
        self.dst_row = mk(tokens * topk)
        self._topk = None
        self._layer = self._local_layer(device)
        self.ranks = list(range(self.p)) if self.nl > 1 else [comm.rank]

    def _local_layer(self, device):
        """Tables of the launches that serve all ranks at once, where all of them are in this process on one GPU."""
        if not (self.comm.device and self.nl == self.p and self.E <= 4096):
            return None
        self._scratch = torch.zeros(L.lib().HcclB200MoeScratchBytes(self.p, self.T, self.k, self.E) // 4, device=device, dtype=torch.int32)
        y = L.MoeLayer(tokens=self.T, capacityRows=self.cap, topk=self.k, hidden=self.H, nExperts=self.E, scratch=self._scratch.data_ptr())
        for name, ts in (("rows", self.recv), ("pos", self.pos), ("dstRow", self.dst_row), ("expertOffsets", self.expert_offsets),
                         ("recvRows", self.recv_rows), ("overflow", self.overflow)):
            for r, t in enumerate(ts):
                getattr(y, name)[r] = t.data_ptr()
        self._out_rows = (C.c_void_p * 16)(*[t.data_ptr() for t in self.expert_out])
        self._layer_ptr, self._out_ptr = C.addressof(y), C.addressof(self._out_rows)
        torch.cuda.current_stream(device).synchronize()  # the scratch is zero whatever stream the first dispatch runs on
        return y

    def _l(self, x):
        return list(x) if isinstance(x, (list, tuple)) else [x]

    def dispatch(self, x, topk_idx, variant="mesh"):
        if self.recv is None:
            raise RuntimeError("dispatch() on a closed exchange")
        xs, idx = self._l(x), self._l(topk_idx)
        if self._layer is not None:  # no links between the ranks: the variants, which order the traffic on them, are one
            for t, i in zip(xs, idx):
                assert i.dtype == torch.int32 and i.is_contiguous() and t.dtype == torch.bfloat16 and t.is_contiguous()
            L.check(L.fast.moe_dispatch(self.comm.handle.value or 0, self.nl, self._layer_ptr, xs, idx, _raw_stream()), "HcclB200MoeDispatchLocal")
            self._topk = idx
            one = self.nl == 1
            return (self.recv[0] if one else self.recv, self.expert_offsets[0] if one else self.expert_offsets,
                    self.recv_rows[0] if one else self.recv_rows)
        lib, st = L.lib(), C.c_void_p(_raw_stream())
        pw = 1 if variant == "pairwise" else 0
        for l in range(self.nl):
            assert idx[l].dtype == torch.int32 and idx[l].is_contiguous() and xs[l].dtype == torch.bfloat16 and xs[l].is_contiguous()
            L.check(lib.HcclB200MoeCount(idx[l].data_ptr(), self.T * self.k, self.E, self.hist[l].data_ptr(), self.pos[l].data_ptr(), st), "HcclB200MoeCount")
        # device-side count exchange: all-gather of the histograms
        self.comm.all_gather(self.hist if self.nl > 1 else self.hist[0], self.counts if self.nl > 1 else self.counts[0])
        for l in range(self.nl):
            L.check(lib.HcclB200MoeOffsets(self.counts[l].data_ptr(), self.p, self.E, self.ranks[l], self.base[l].data_ptr(),
                                           self.expert_offsets[l].data_ptr(), self.recv_rows[l].data_ptr(), self.cap,
                                           self.overflow[l].data_ptr(), st), "HcclB200MoeOffsets")
        self.comm.barrier()  # every rank is done with the previous round's buffers
        for l in range(self.nl):
            peers = (C.c_void_p * self.p)(*self.recv_tab[l])
            L.check(lib.HcclB200MoeDispatch(xs[l].data_ptr(), idx[l].data_ptr(), self.pos[l].data_ptr(), self.base[l].data_ptr(), self.T, self.k,
                                            self.H, self.E, self.p, self.ranks[l], pw, peers, self.dst_row[l].data_ptr(), self.cap, st),
                    "HcclB200MoeDispatch")
        self.comm.barrier()  # all rows have landed everywhere
        self._topk = idx
        one = self.nl == 1
        return (self.recv[0] if one else self.recv, self.expert_offsets[0] if one else self.expert_offsets,
                self.recv_rows[0] if one else self.recv_rows)

    def combine(self, gates, variant="mesh", source="expert_out", out=None):
        """gates: fp32 [tokens, topk].  source: 'expert_out' (after the experts ran) or 'recv' (identity experts)."""
        if self._topk is None:
            raise RuntimeError("combine() needs the routing of a dispatch()")
        gs = self._l(gates)
        if self._layer is not None:
            outs = self._l(out) if out is not None else [torch.empty(self.T, self.H, device=g.device, dtype=torch.bfloat16) for g in gs]
            for g in gs:
                assert g.dtype == torch.float32 and g.is_contiguous()
            rows = self._out_ptr if source == "expert_out" else 0
            L.check(L.fast.moe_combine(self.comm.handle.value or 0, self.nl, self._layer_ptr, rows, self._topk, gs, outs, _raw_stream()),
                    "HcclB200MoeCombineLocal")
            return outs[0] if self.nl == 1 else outs
        lib, st = L.lib(), C.c_void_p(_raw_stream())
        tab = self.out_tab if source == "expert_out" else self.recv_tab
        outs = self._l(out) if out is not None else [torch.empty(self.T, self.H, device=gs[0].device, dtype=torch.bfloat16) for _ in range(self.nl)]
        pw = 1 if variant == "pairwise" else 0
        self.comm.barrier()  # the expert outputs of every rank are complete
        for l in range(self.nl):
            assert gs[l].dtype == torch.float32 and gs[l].is_contiguous()
            peers = (C.c_void_p * self.p)(*tab[l])
            L.check(lib.HcclB200MoeCombine(peers, self._topk[l].data_ptr(), gs[l].data_ptr(), self.dst_row[l].data_ptr(), self.T, self.k, self.H,
                                           self.E, self.p, self.ranks[l], pw, outs[l].data_ptr(), self.cap, st), "HcclB200MoeCombine")
        return outs[0] if self.nl == 1 else outs

    def close(self):
        self.recv = self.expert_out = self._topk = None  # nothing reaches the memory given back here
        self.comm.mem_free(self.h_recv)
        self.comm.mem_free(self.h_out)


class _Part:
    """A part of a Gate's memory, made a tensor at its first use (an instance attribute of the same name then takes over)."""

    def __init__(self, place, real):
        self.place, self.real = place, real  # place: number of the part; real: fp32

    def __set_name__(self, owner, name):
        self.name = name

    def __get__(self, g, owner=None):
        if g is None:
            return self
        words, i = g._words, self.place
        if self.real:
            words = words.view(torch.float32)
        if i < 2:
            t = words.as_strided((g._T, g._k), (g._k, 1), g._at[i])
        elif i < 4:
            t = words.as_strided((g._E,), (1,), g._at[i])
        else:
            t = words.as_strided((), (), g._at[i])
        g.__dict__[self.name] = t
        return t


def _writes(t):
    """Number of writes that torch has counted on a tensor."""
    return None if t.is_inference() else t._version


class Gate:
    """What gate() returns: tensors idx, gates, counts, prob_sum, routed, balance (in this order when it is iterated over).  gate() keeps
    them in one piece of memory and makes a tensor of a part when it is asked for: six allocations cost a decode step more than the
    kernel does.  Besides these it has the call's `mask` (the tensor itself, no copy) and `normalize`, which gate_grad() goes by."""
    _FIELDS = ("idx", "gates", "counts", "prob_sum", "routed", "balance")
    idx, gates, counts, prob_sum, routed, balance = (_Part(i, n in ("gates", "prob_sum", "balance")) for i, n in enumerate(_FIELDS))

    def __init__(self, idx, gates, counts, prob_sum, routed, balance, mask=None, normalize=True):
        self.__dict__.update(zip(self._FIELDS, (idx, gates, counts, prob_sum, routed, balance)), _words=None, mask=mask, normalize=normalize,
                             _written=None if mask is None else _writes(mask))

    def __setattr__(self, name, value):
        raise AttributeError("the parts of a Gate may be written to, not replaced: make a Gate of the tensors")

    @classmethod
    def _empty(cls, like, T, k, E, mask, normalize):
        g = object.__new__(cls)
        n, e = (T * k + 3) // 4 * 4, (E + 3) // 4 * 4
        g.__dict__.update(_T=T, _k=k, _E=E, _at=(0, n, 2 * n, 2 * n + e, 2 * n + 2 * e, 2 * n + 2 * e + 1),
                          _words=like.new_empty(2 * n + 2 * e + 2, dtype=torch.int32), mask=mask, normalize=normalize,
                          _written=None if mask is None else _writes(mask))
        return g

    def _touched(self):
        """Whether someone may have written to the parts: they are the caller's own, or torch has seen a write."""
        return self._words is None or _writes(self._words) != 0

    def __iter__(self):
        return (getattr(self, n) for n in self._FIELDS)

    def _addresses(self, *parts):
        """Of parts by number."""
        if self._words is None:
            return [getattr(self, self._FIELDS[i]).data_ptr() for i in parts]
        base, at = self._words.data_ptr(), self._at
        return [base + 4 * at[i] for i in parts]


_FLOAT = float_codes()
_REPEATED = 256  # of HcclB200MoeGateGrad's normalize


def _check_gate(logits, topk, mask):
    if not (torch.is_tensor(logits) and logits.is_cuda and logits.dim() == 2 and logits.shape[1] > 0):
        raise ValueError("logits must be a CUDA tensor [tokens, experts]")
    T, E = logits.shape
    a, b = logits.stride()
    code = _FLOAT.get(logits.dtype)
    if code is None:
        raise TypeError("logits must be fp32, fp16 or bf16, got %s" % logits.dtype)
    if b != 1 and E > 1 or a < E and T > 1:
        raise ValueError("the experts of a token must lie side by side (strides %s)" % ((a, b),))
    if not 1 <= topk <= E:
        raise ValueError("topk %d of %d experts" % (topk, E))
    if mask is not None and not (mask.device == logits.device and mask.dtype in (torch.bool, torch.uint8) and mask.shape == (T,) and mask.is_contiguous()):
        raise ValueError("mask must be a contiguous bool tensor [tokens] on the device of the logits")
    return T, E, max(E, a), code


def gate(logits, topk, mask=None, normalize=True, comm=None):
    """Router of a mixture-of-experts layer.  logits [tokens, experts] (fp32, fp16, bf16; rows may be strided); mask [tokens]: tokens that
    are routed, others (padding) get no expert and count nowhere.  Returns a Gate:

    idx       int32 [tokens, topk]: the experts with the largest logits, largest first, equal ones by number; a logit of -inf is never
              chosen, slots that stay empty have expert -1 (the exchange skips them) and gate 0
    gates     fp32 [tokens, topk]: softmax probabilities of the chosen experts, with `normalize` divided by their sum
    counts    int32 [experts], prob_sum fp32 [experts], routed int32 []: pairs, sums of probabilities and number of the routed tokens
    balance   fp32 []: experts / (topk * routed^2) * sum(counts * prob_sum), 1 for an even load

    The Gate has mask and normalize as well, for gate_grad().  The sums have a fixed order: the same inputs give the same bits.  With
    `comm` the three sums, and so the loss, are those of all ranks' tokens (on an all-local communicator logits and mask are lists with one tensor per rank, and a list of Gates returns)."""
    if comm is not None:
        ls = list(logits) if isinstance(logits, (list, tuple)) else [logits]
        ms = list(mask) if isinstance(mask, (list, tuple)) else [mask] * len(ls)
        if len(ls) != comm.nlocal or len(ms) != comm.nlocal:
            raise ValueError("one tensor per local rank is needed")
        gs = [gate(l, topk, m, normalize) for l, m in zip(ls, ms)]
        if comm.nranks > 1:
            for name in ("counts", "prob_sum", "routed"):
                ts = [getattr(g, name) for g in gs]
                comm.all_reduce(ts, ts)
            for l, g in zip(ls, gs):
                with on_device_of(l):
                    L.check(L.lib().HcclB200MoeBalance(g.counts.data_ptr(), g.prob_sum.data_ptr(), g.routed.data_ptr(), l.shape[1], topk,
                                                       g.balance.data_ptr(), _raw_stream()), "HcclB200MoeBalance")
        return gs if isinstance(logits, (list, tuple)) else gs[0]
    T, E, stride, code = _check_gate(logits, topk, mask)
    with on_device_of(logits):
        g = Gate._empty(logits, T, topk, E, mask, normalize)
        n = L.lib().HcclB200MoeGateScratchBytes(T, E)
        scratch = logits.new_empty(n, dtype=torch.uint8) if n > 0 else None
        rc = L.fast.gate(logits, code, T, E, stride, topk, int(normalize), mask, *g._addresses(0, 1, 2, 3, 4, 5), scratch, _raw_stream())
        if rc:
            L.check(rc, "HcclB200MoeGate")
    return g


def gate_grad(logits, g, d_gates=None, balance=0.0, mask=None, normalize=None, out=None):
    """Gradient of the logits: `d_gates` (fp32 [tokens, topk] or None) is the gates' gradient, the number `balance` that of the balance
    loss.  logits are those of the gate() call that returned `g`, and so are mask and normalize where they are not given; counts are constants
    of the loss.  A slot with expert -1 passes nothing on, rows that are not routed get zeros.  A mask that torch has seen written to since
    gate() is refused: give the one that gate() had."""
    if not isinstance(g, Gate):
        raise TypeError("g must be what gate() returned for these logits")
    if mask is None and g.mask is not None:
        mask = g.mask
        if _writes(mask) != g._written:
            raise RuntimeError("the mask has been written to since gate()")
    if normalize is None:
        normalize = g.normalize
    if g._words is not None:
        shape, experts, device = (g._T, g._k), (g._E,), g._words.device
    else:
        ts = (g.idx, g.counts, g.routed)
        if g.idx.dim() != 2 or g.routed.numel() != 1 or not all(t.dtype == torch.int32 and t.is_contiguous() and t.device == g.idx.device for t in ts):
            raise ValueError("g needs contiguous int32 tensors idx [tokens, topk], counts [experts] and routed []")
        shape, experts, device = tuple(g.idx.shape), tuple(g.counts.shape), g.idx.device
    T, E, stride, code = _check_gate(logits, shape[1], mask)
    dev, topk = logits.device, shape[1]
    if shape[0] != T or experts != (E,) or device != dev:
        raise ValueError("g must be what gate() returned for these logits")
    if d_gates is not None and not (d_gates.device == dev and d_gates.dtype == torch.float32 and d_gates.shape == shape and d_gates.is_contiguous()):
        raise ValueError("d_gates must be a contiguous fp32 tensor [tokens, topk] on the device of the logits")
    with on_device_of(logits):
        if out is None:
            out = logits.new_empty((T, E))
        else:
            check_out(out, (T, E), logits.dtype, dev)
        L.lib()
        idx, counts, routed = g._addresses(0, 2, 4)
        # slots that were written to may name an expert again
        rc = L.fast.gate_grad(logits, code, T, E, stride, topk, int(bool(normalize)) | (_REPEATED if g._touched() else 0), mask, idx, d_gates, counts, routed, balance, out, _raw_stream())
        if rc:
            L.check(rc, "HcclB200MoeGateGrad")
    return out


def route(tokens, n_experts, topk, seed, rank, device="cuda"):
    """Synthetic router of the benchmark config: N(0,1) logits, softmax, top-k; returns (int32 experts, fp32 gates)."""
    g = torch.Generator(device=device).manual_seed(seed * 1000 + rank)
    logits = torch.randn(tokens, n_experts, device=device, generator=g)
    probs = torch.softmax(logits, dim=-1)
    gates, idx = torch.topk(probs, topk, dim=-1)
    gates = gates / gates.sum(dim=-1, keepdim=True)
    return idx.to(torch.int32).contiguous(), gates.to(torch.float32).contiguous()


def bench(comm, world, rank, dist, max_over_ranks, sync, tokens=8192, hidden=7168, n_experts=256, topk=8, iters=5):
    """Dispatch + combine (identity experts) of the benchmark config, both variants, next to NCCL all-to-all."""
    if n_experts % world:
        return {"skipped": "experts do not divide over ranks"}
    out = {"config": {"tokens_per_rank": tokens, "hidden": hidden, "experts": n_experts, "topk": topk, "dtype": "bf16", "seed": 7}}
    g = torch.Generator(device="cuda").manual_seed(70 + rank)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).to(torch.bfloat16)
    idx, gates = route(tokens, n_experts, topk, 7, rank)
    ex = MoEExchange(comm, tokens, hidden, n_experts, topk)
    res = torch.empty(tokens, hidden, device="cuda", dtype=torch.bfloat16)

    def timed(fn):
        for _ in range(2):
            fn()
        sync()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(iters):
            fn()
        b.record()
        torch.cuda.synchronize()
        ms = a.elapsed_time(b) / iters
        sync()
        return max_over_ranks(ms)

    for variant in ("mesh", "pairwise"):
        def ours():
            ex.dispatch(x, idx, variant=variant)
            ex.combine(gates, variant=variant, source="recv", out=res)
        out[variant + "_ms"] = round(timed(ours), 4)
    assert comm.sync() == 0, comm.describe_status()
    assert int(ex.overflow[0].item()) == 0, "receive buffer overflow"
    # identity experts: combine returns sum_k gate * x = x (gates are normalised)
    err = float((res.float() - x.float()).abs().max())
    out["check_max_abs_err"] = round(err, 4)
    send_rows = tokens * topk
    out["bytes_per_rank_each_way"] = send_rows * hidden * 2
    # what crosses the links: a rank keeps 1/world of its rows; dispatch and combine each move the rest once per direction
    crossing = out["bytes_per_rank_each_way"] * (world - 1) / max(1, world)
    best = min(out["mesh_ms"], out["pairwise_ms"])
    out["link_GBps_per_direction"] = round(2 * crossing / best / 1e6, 1)
    out["fraction_of_900GBps"] = round(2 * crossing / best / 1e6 / 900.0, 3)
    # ---- baseline: NCCL all_to_all_single with the split lists, buffers and permutations prepared once outside the timed
    # loop (no host synchronisation and no allocation per step), combine as one gather and one batched product
    if dist is not None:
        El = n_experts // world
        flat = idx.flatten().long()
        order = torch.argsort(flat, stable=True)
        inv = torch.argsort(order)
        tok_of = order // topk
        send_counts = torch.bincount(flat // El, minlength=world)
        rc = torch.empty_like(send_counts)
        dist.all_to_all_single(rc, send_counts)
        s_l, r_l = send_counts.tolist(), rc.tolist()
        sbuf = torch.empty(send_rows, hidden, device="cuda", dtype=torch.bfloat16)
        rbuf = torch.empty(sum(r_l), hidden, device="cuda", dtype=torch.bfloat16)
        back = torch.empty_like(sbuf)
        perm = torch.empty_like(sbuf)
        gates_b = gates.to(torch.bfloat16).unsqueeze(1).contiguous()      # [tokens, 1, topk]
        res3 = res.view(tokens, 1, hidden)

        def base():
            torch.index_select(x, 0, tok_of, out=sbuf)                    # rows in destination order
            dist.all_to_all_single(rbuf, sbuf, r_l, s_l)                  # dispatch
            dist.all_to_all_single(back, rbuf, s_l, r_l)                  # combine transport (identity experts)
            torch.index_select(back, 0, inv, out=perm)                    # back to (token, k) order
            torch.bmm(gates_b, perm.view(tokens, topk, hidden), out=res3)  # gate-weighted sum over k
        out["nccl_a2a_ms"] = round(timed(base), 4)
        out["nccl_check_max_abs_err"] = round(float((res.float() - x.float()).abs().max()), 4)
        out["speedup_vs_nccl"] = round(out["nccl_a2a_ms"] / best, 3)
        # ---- the same schedule with this library's HcclAlltoAllV (parametric kernel: counts are launch arguments) as transport
        sc = [c * hidden for c in s_l]
        rcv = [c * hidden for c in r_l]
        sd = [sum(sc[:i]) for i in range(world)]
        rd = [sum(rcv[:i]) for i in range(world)]
        sflat, rflat, bflat = sbuf.view(-1), rbuf.view(-1), back.view(-1)

        def through_api():
            torch.index_select(x, 0, tok_of, out=sbuf)
            comm.all_to_all_v(sflat, sc, sd, rflat, rcv, rd)              # dispatch
            comm.all_to_all_v(rflat, rcv, rd, bflat, sc, sd)              # combine transport (identity experts)
            torch.index_select(back, 0, inv, out=perm)
            torch.bmm(gates_b, perm.view(tokens, topk, hidden), out=res3)
        res.zero_()
        out["alltoallv_api_ms"] = round(timed(through_api), 4)
        assert comm.sync() == 0, comm.describe_status()
        out["alltoallv_api_check_max_abs_err"] = round(float((res.float() - x.float()).abs().max()), 4)
        out["alltoallv_api_speedup_vs_nccl"] = round(out["nccl_a2a_ms"] / out["alltoallv_api_ms"], 3)
    ex.close()
    return out
