"""The dense and the paged cache of one decoder used in turn: each gives what it gives alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decoder():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops
    from bladedisc_b200.decoder import DecoderConfig, QuantDecoder
    yield QuantDecoder(DecoderConfig.tiny(), None, seed=3)
    assert ops.kernel_status() == 0, "a kernel's bounded wait ran out"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ids(seed, *shape):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, 1000, shape, generator=gen).cuda()


def test_both_caches_in_turn(decoder):
    """Chunks of two requests far past the positions of a dense cache that is started between them."""
    chunks = [_ids(i, 48 + 31) for i in range(5)]
    dense_ids = _ids(9, 1, 20)

    def paged(between):
        decoder.start_paged(requests=2, num_blocks=40, max_seq=300, block_size=16)
        out = []
        for i, c in enumerate(chunks):
            out.append(decoder.forward_paged(c, i32([48, 31]), 48).clone())
            between(i)
        assert decoder.paged.lens.tolist() == [240, 155]
        return out

    def dense(i):
        decoder.start(1, 20 + i)
        got.append(decoder.forward(dense_ids).clone())

    got = []
    want = paged(lambda i: None)
    dense(0)
    mixed = paged(dense)
    assert all(torch.equal(a, b) for a, b in zip(mixed, want))
    assert all(torch.equal(g, got[0]) for g in got)


def test_captured_steps_of_both_caches_outlive_new_starts(decoder):
    """Graphs over a dense and a paged cache, replayed after other caches of the decoder were started."""
    prompt, ids = _ids(1, 40 + 17), _ids(2, 6, 2)
    one = i32([1, 1])

    def begin():
        cache = decoder.start_paged(requests=2, num_blocks=20, max_seq=130, block_size=16)
        decoder.forward_paged(prompt, i32([40, 17]), 40)
        return cache

    begin()
    want = [decoder.forward_paged(t, one, 1).clone() for t in ids]
    decoder.start(2, 33)
    prefill = ids.t().contiguous()
    want_dense = decoder.forward(prefill).clone()

    cache = begin()
    decoder.start(2, 33)
    buf = ids[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    paged, dense = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(paged, stream=side):
        y = decoder.forward_paged(buf, one, 1)
    with torch.cuda.graph(dense, stream=side):
        z = decoder.forward(prefill)
    kv = decoder.kv  # the caller keeps both caches
    other = decoder.start_paged(requests=1, num_blocks=70, max_seq=1000, block_size=16)
    hold = [torch.full((n, 32), float("nan"), device="cuda") for n in (33, 130, 144, 1008)]  # over what was given back
    for t, w in zip(ids, want):
        buf.copy_(t)
        paged.replay()
        assert torch.equal(y, w)
    dense.replay()
    assert torch.equal(z, want_dense)
    assert cache.lens.tolist() == [46, 23] and other.lens.tolist() == [0] and len(kv) == 2 and len(hold) == 4
    decoder.paged = None


class TwoRanks:
    """Collectives of two ranks that are two host threads and share a GPU and its default stream: a rank copies what it
    needs of the other's tensor, between two meetings of the threads."""

    def __init__(self, rank, box, gate):
        self.rank, self.world, self.box, self.gate = rank, 2, box, gate

    def _meet(self, t, copy):
        self.box[self.rank] = t
        self.gate.wait(60)
        copy(self.box[1 - self.rank])
        self.gate.wait(60)
        return t

    def all_gather_(self, buf):
        return self._meet(buf, lambda other: buf[1 - self.rank].copy_(other[1 - self.rank]))

    def all_reduce_max_(self, t):
        mine = t.clone()

        def copy(other):
            torch.maximum(mine, other, out=mine)
        self._meet(t, copy)
        return t.copy_(mine)


def test_two_ranks_have_half_of_the_heads_each(decoder):
    """Ragged prompts and steps over paged caches that hold two of four heads, against one rank."""
    import threading

    from bladedisc_b200.decoder import QuantDecoder
    steps = [[70, 5, 90], [1, 40, 1], [1, 1, 1]]

    def run(d, out):
        cache = d.start_paged(requests=3, num_blocks=30, max_seq=160, block_size=16)
        assert cache.k[0].shape[1] == d.cfg.heads // d.world
        for i, tokens in enumerate(steps):
            out.append(d.forward_paged(_ids(30 + i, sum(tokens)), i32(tokens), max(tokens)).clone())
        assert cache.lens.tolist() == [72, 46, 92]

    want, box, gate, got, errors = [], [None, None], threading.Barrier(2), [[], []], []
    run(decoder, want)

    def rank(r):
        try:
            run(QuantDecoder(decoder.cfg, TwoRanks(r, box, gate), seed=3), got[r])
        except Exception as e:  # raised below, in the thread that waits
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b, w in zip(*got, want):
        assert torch.equal(a, b)
        # the same integers, scales and heads; sums over a row of the norms may be added in another order, which can turn
        # an int8 rounding: as far as two runs of a quantized net differ
        assert (a.float() - w.float()).abs().mean() < 0.01 * w.float().abs().mean()


def test_steps_without_tokens(decoder):
    """Rows of no request, a batch of such rows only, and an empty batch."""
    cache = decoder.start_paged(requests=2, num_blocks=20, max_seq=100, block_size=16)
    for rows, tokens, lens in ((7, [3, 0], [3, 0]), (4, [0, 0], [3, 0]), (0, [0, 0], [3, 0]), (0, [1, 0], [3, 0])):
        y = decoder.forward_paged(_ids(5, rows), i32(tokens), max(tokens))
        assert y.shape == (rows, decoder.cfg.hidden) and torch.isfinite(y).all()
        assert cache.lens.tolist() == lens
    decoder.paged = None
