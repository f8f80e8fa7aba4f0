"""The dense and the paged cache of one decoder, side by side, on the host: which rotation tables a paged step gets."""
import gc
import weakref

import pytest
import torch

from bladedisc_b200.decoder import DecoderConfig, QuantDecoder


class Recorder:
    """Stands for the calls of a paged cache that need a GPU and notes the tables that the append is given."""

    def __init__(self, cache):
        self.cache, self.tables = cache, None

    def __getattr__(self, name):
        return getattr(self.cache, name)

    def extend(self, tokens, max_tokens):
        return None

    def append(self, layer, qkv, plan, cos, sin):
        self.tables = cos, sin
        return qkv

    def attend(self, layer, q, plan, max_q, max_kv=None, out=None):
        return out


@pytest.fixture
def decoder(monkeypatch):
    d = object.__new__(QuantDecoder)  # no weights: those are made on a GPU
    d.cfg, d.world, d.device = DecoderConfig.tiny(), 1, torch.device("cpu")
    d.kv, d.pos, d.paged, d.embed = None, 0, None, torch.zeros(1, 1)
    d._cos = d._sin = None
    monkeypatch.setattr(d, "_run_layers", lambda ids, attention: attention(None, 0, torch.zeros(ids.numel(), 4)))
    return d


def tables_of_a_step(decoder, cache):
    decoder.paged = rec = Recorder(cache)
    decoder.forward_paged(torch.zeros(3, dtype=torch.int64), None, 3)
    decoder.paged = cache
    return rec.tables


def angles(rows, half):
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float32) / half)
    return torch.arange(rows, dtype=torch.float32)[:, None] * inv[None, :]


def test_a_dense_start_leaves_a_paged_cache_its_positions(decoder):
    cache = decoder.start_paged(requests=2, num_blocks=30, max_seq=800)
    decoder.start(1, 128)
    cos, sin = tables_of_a_step(decoder, cache)
    room = cache.table.shape[1] * cache.block_size
    want = angles(room, decoder.cfg.head_dim // 2)
    assert room >= 800 and torch.equal(cos, want.cos()) and torch.equal(sin, want.sin())


def test_neither_start_replaces_the_tables_of_the_other_cache(decoder):
    """A graph captured from a step holds their addresses."""
    decoder.start(1, 300)
    dense = decoder._cos, decoder._sin
    cache = decoder.start_paged(requests=2, num_blocks=30, max_seq=800)
    assert decoder._cos is dense[0] and decoder._sin is dense[1]
    before = tables_of_a_step(decoder, cache)
    decoder.start(1, 100)
    decoder.start(2, 4000)
    after = tables_of_a_step(decoder, cache)
    assert all(a is b for a, b in zip(before, after))


def test_tables_live_as_long_as_the_cache_that_uses_them(decoder):
    first = decoder.start_paged(requests=1, num_blocks=3, max_seq=50)
    cos, sin = tables_of_a_step(decoder, first)
    held = weakref.ref(cos), weakref.ref(sin)
    second = decoder.start_paged(requests=1, num_blocks=30, max_seq=1000)
    decoder.start(1, 60)
    del cos, sin
    gc.collect()
    assert held[0]() is not None and held[1]() is not None  # `first` is still in use, by a captured step for instance
    assert tables_of_a_step(decoder, first)[0] is held[0]()
    assert tables_of_a_step(decoder, second)[0].shape[0] >= 1000


def test_a_cache_without_tables_is_refused(decoder):
    cache = decoder.start_paged(requests=1, num_blocks=3, max_seq=50)
    cache.rope = None
    with pytest.raises(RuntimeError, match="start_paged"):
        tables_of_a_step(decoder, cache)


def test_a_step_without_tokens_touches_nothing(decoder):
    cache = decoder.start_paged(requests=1, num_blocks=3, max_seq=50)
    decoder.paged = rec = Recorder(cache)
    y = decoder.forward_paged(torch.zeros(0, dtype=torch.int64), None, 0)
    assert y.shape == (0, decoder.cfg.hidden) and rec.tables is None
