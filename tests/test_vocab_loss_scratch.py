"""Scratch of the vocabulary loss over several chunks of tokens: what is allocated covers every chunk's call.  The sizes are the library's own
for given numbers of multiprocessors and CTA pairs; launches are stood in for, tensors have no memory."""
import contextlib
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from cann_hccl_b200 import _lib as L  # noqa: E402
from cann_hccl_b200.parallel import vocab  # noqa: E402

REAL = L.lib()


class Comm:
    nranks, nlocal, rank = 4, 1, 2

    def all_gather(self, send, recv):
        pass

    all_reduce = all_gather


class Lib:
    """Sizes of a device with `pairs` concurrent clusters; writes down the tokens of every call that has scratch."""

    def __init__(self, pairs):
        self.pairs, self.calls = pairs, []

    def HcclB200VocabLossChunk(self, v, grad):
        return REAL.HcclB200VocabLossChunk(v, grad)

    def HcclB200VocabLossScratchBytes(self, tokens, v, h, grad):
        return REAL.HcclB200VocabLossScratchBytesOn(148, self.pairs, tokens, v, h, grad)

    def __getattr__(self, name):
        def call(p, *a):
            s = C.cast(p, C.POINTER(L.VocabLoss)).contents
            if name in ("HcclB200VocabLossScores", "HcclB200VocabLossGrad"):
                self.calls.append((s.tokens, s.scratchBytes))
            return 0
        return call


@pytest.fixture
def run(monkeypatch):
    """run(tokens, vocab, hidden, pairs, grad, sharded) -> chunk, [(tokens, bytes the call is told of)], bytes allocated before the fp32 words"""
    monkeypatch.setattr(vocab, "_check_loss", lambda *a: None)
    monkeypatch.setattr(vocab, "on_device_of", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(vocab, "_raw_stream", lambda: 0)
    new, sizes = vocab._Shard.new, []

    def record(self, shape, dtype=torch.float32):
        if dtype == torch.uint8:
            sizes.append(shape)
        return new(self, shape, dtype)
    monkeypatch.setattr(vocab._Shard, "new", record)

    def call(T, V, H, pairs, grad, sharded):
        lib = Lib(pairs)
        monkeypatch.setattr(vocab.L, "lib", lambda: lib)
        sizes.clear()
        x, w, y = [torch.empty(*s, dtype=d, device="meta") for s, d in (((T, H), torch.bfloat16), ((V, H), torch.bfloat16), ((T,), torch.int64))]
        if sharded:
            (vocab.vocab_parallel_cross_entropy_grad if grad else vocab.vocab_parallel_cross_entropy)(Comm(), x, w, y)
        else:
            (vocab.linear_cross_entropy_grad if grad else vocab.linear_cross_entropy)(x, w, y)
        chunk = lib.HcclB200VocabLossChunk(V, int(grad))
        assert len(sizes) == 1
        return chunk, lib.calls, sizes[0] - (3 * chunk + 1) * 4
    return call


# vocabularies and hidden sizes of language models and others; with gradients dx of a short last chunk is cut into more shares than a whole
# chunk's, without them its tiles may be narrower, which makes more row sums
@pytest.mark.parametrize("sharded", [False, True])
@pytest.mark.parametrize("V,H,grad", [(128256, 4096, True), (128256, 8192, True), (151936, 4096, True), (102400, 4096, True), (50257, 768, True), (32000, 1000, True),
                                      (8482, 512, False), (4116, 512, False), (128256, 4096, False), (50257, 1000, False)])
def test_allocation_covers_every_chunk(run, V, H, grad, sharded):
    for pairs in range(70, 75):
        need = lambda t: REAL.HcclB200VocabLossScratchBytesOn(148, pairs, t, V, H, int(grad))
        chunk = REAL.HcclB200VocabLossChunk(V, int(grad))
        step = max(1, chunk // 97)
        rests = [chunk - 1, 1, *range(chunk - step, 0, -step)]
        worst = max(rests, key=need)
        for rest in {worst, *rests[::9]}:
            at, calls, got = run(chunk + rest, V, H, pairs, grad, sharded)
            assert at == chunk and {t for t, _ in calls} == {chunk, rest}
            for t, told in calls:
                assert need(t) <= got, (pairs, t)
                assert need(t) <= told <= got, (pairs, t)          # and the library can refuse too little


def test_a_short_chunk_may_need_more():
    """The sizes do not grow with the tokens: this is what the allocation has to reckon with."""
    size = lambda t: REAL.HcclB200VocabLossScratchBytesOn(148, 74, t, 128256, 4096, 1)
    assert size(7424) > size(8192)


@pytest.mark.parametrize("grad", [False, True])
def test_one_chunk_and_less(run, grad):
    for T in (1, 5, 300, 7424):
        chunk, calls, got = run(T, 128256, 4096, 74, grad, True)
        assert {t for t, _ in calls} == {T} and all(REAL.HcclB200VocabLossScratchBytesOn(148, 74, T, 128256, 4096, int(grad)) <= told for _, told in calls)


def test_sizes_that_are_none():
    on = REAL.HcclB200VocabLossScratchBytesOn
    assert on(0, 74, 4, 16, 8, 1) == on(148, 0, 4, 16, 8, 1) == on(148, 74, -1, 16, 8, 1) == on(148, 74, 4, 16, 12, 1) == on(148, 74, 4, 0, 8, 1) == -1
    assert on(148, 74, 0, 16, 8, 1) > 0


def test_refused_before_anything_is_asked_for():
    mem = C.create_string_buffer(2048)
    at = (C.addressof(mem) + 255) // 256 * 256
    call = lambda **k: C.byref(L.VocabLoss(**{**dict(x=at, w=at, xStride=8, wStride=8, targets=at, tokens=4, vocab=16, wholeVocab=16, ignoreId=-100, hidden=8, targetType=L.INT64), **k}))
    assert REAL.HcclB200VocabLossScores(call(scratchBytes=-1), 1, at, at, at, at, None) == L.E_PARA
    assert REAL.HcclB200VocabLossStep(call(scratchBytes=-1), 1, 1.0, at, at, at, None, 0, at, None) == L.E_PARA
    assert REAL.HcclB200VocabLossGrad(call(scratchBytes=-1), at, at, at, 1.0, at, at, None, 0, at, None) == L.E_PARA
    assert REAL.HcclB200VocabLossGrad(call(losses=at + 2), at, at, at, 1.0, at, at, None, 0, at, None) == L.E_PARA


@pytest.mark.parametrize("grad", [0, 1])
@pytest.mark.parametrize("V", [256, 1000, 8000, 32000, 50257, 128256, 151936, 200064, 1 << 18, 1 << 19])
def test_scratch_stays_within_what_is_stated(V, grad):
    """Beside the copy of x (none without gradients where its rows start on 128-byte lines, or there is one row of tiles): 130 MB, or
    3 GB with the exponentials and shares of the gradients."""
    chunk = REAL.HcclB200VocabLossChunk(V, grad)
    for H in (64, 1000, 4096, 4104, 8192, 16384):
        for T in {1, 128, 129, 300, 700, 1500, 3000, 6000, *range(chunk - chunk // 4, chunk, max(1, chunk // 50)), chunk - 1, chunk}:
            if T > chunk:
                continue
            copy = T * ((H + 63) // 64 * 128) if grad or (T > 128 and H % 64) else 0
            for pairs in (70, 74):
                got = REAL.HcclB200VocabLossScratchBytesOn(148, pairs, T, V, H, grad) - copy
                assert got <= (3 * 10 ** 9 if grad else 130 * 10 ** 6), (H, T)
