"""The decoder over the paged 8-bit cache: every append and every attention of every layer and step is checked
against the plain statements of oracle/kv8_ref.py on what that layer was given."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decoder():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops
    from bladedisc_b200.decoder import DecoderConfig, QuantDecoder
    yield QuantDecoder(DecoderConfig.tiny(), None, seed=3)
    assert ops.kernel_status() == 0, "a kernel's bounded wait ran out"


class Checked:
    """Wraps a cache: runs its calls and verifies them."""

    def __init__(self, cache, cos, sin):
        self.cache, self.cos, self.sin, self.checks = cache, cos.cpu().numpy(), sin.cpu().numpy(), 0

    def __getattr__(self, name):
        return getattr(self.cache, name)

    def append(self, layer, qkv, plan, cos, sin):
        c = self.cache
        before = [t[layer].cpu().numpy() for t in (c.k, c.v, c.k_scale, c.v_scale)]
        heads, dim = before[0].shape[1], before[0].shape[3]
        x = qkv.float().cpu().numpy().reshape(qkv.shape[0], -1, dim)
        q_heads = x.shape[1] - 2 * heads
        at = np.clip(plan.positions.cpu().numpy(), 0, len(self.cos) - 1)
        rot = kv8_ref.rotate(x[:, :q_heads + heads], self.cos[at], self.sin[at])
        q = c.append(layer, qkv, plan, cos, sin)
        assert torch.equal(q.cpu(), torch.from_numpy(rot[:, :q_heads]).half())
        slots = plan.slots.cpu().numpy()
        for new, i in ((rot[:, q_heads:], 0), (x[:, q_heads + heads:], 1)):
            levels, scales = kv8_ref.append(new, before[i], before[2 + i], slots)
            assert np.array_equal((c.k, c.v)[i][layer].cpu().numpy(), levels)
            assert np.array_equal((c.k_scale, c.v_scale)[i][layer].cpu().numpy(), scales)
        self.checks += 1
        return q

    def attend(self, layer, q, plan, max_q, max_kv, out):
        c = self.cache
        start = out.double().cpu().numpy()
        got = c.attend(layer, q, plan, max_q, max_kv, out=out).double().cpu().numpy()
        want, slack = kv8_ref.attention(q.double().cpu().numpy(),
                                        *[t[layer].cpu().numpy() for t in (c.k, c.v, c.k_scale, c.v_scale)],
                                        c.table.cpu().numpy(), plan.q_start.cpu().numpy(), plan.q_lens.tolist(),
                                        plan.kv_lens.tolist(), q.shape[2] ** -0.5, start)
        assert (np.abs(got - want) <= slack * 1.001 + 2.0 ** -11 * np.abs(want) + 2.0 ** -24).all()
        self.checks += 1
        return torch.from_numpy(got).to(q.dtype).cuda().view_as(q)


def test_prompts_chunks_and_single_tokens(decoder):
    """Ragged prompts, a chunk behind one of them, single tokens, a request that ends and one that finds no room."""
    cache = decoder.start_paged(requests=4, num_blocks=24, max_seq=200, block_size=16)
    decoder.paged = checked = Checked(cache, decoder._cos, decoder._sin)
    gen = torch.Generator().manual_seed(1)

    def step(tokens, max_kv=None):
        ids = torch.randint(0, 1000, (sum(tokens),), generator=gen).cuda()
        return decoder.forward_paged(ids, torch.tensor(tokens, dtype=torch.int32, device="cuda"),
                                     max(tokens), max_kv)

    for tokens in ([70, 5, 0, 133], [1, 40, 3, 1], [1, 1, 1, 1], [1, 1, 1, 1]):
        y = step(tokens)
        assert y.shape == (sum(tokens), 256) and torch.isfinite(y).all()
    assert cache.lens.tolist() == [73, 47, 5, 136]
    # 24 blocks, 5 + 3 + 1 + 9 used: 8 more blocks are not there, the request behind still gets its slot in its own
    y = step([0, 0, 128, 1])
    assert cache.lens.tolist() == [73, 47, 5, 137] and torch.isfinite(y).all()
    cache.trim(torch.tensor([1000, 0, 1000, 120], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [73, 0, 5, 120] and int(cache.free_count) == 24 - 5 - 1 - 8
    step([1, 12, 1, 1], max_kv=130)
    assert cache.lens.tolist() == [74, 12, 6, 121]
    assert checked.checks == 2 * 2 * 6
    decoder.paged = None


def test_a_captured_step_equals_an_eager_one(decoder):
    """Single tokens replayed from a graph while the lengths grow, against the same steps run eagerly."""
    gen = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, 1000, (30 + 17,), generator=gen).cuda()
    tokens = torch.randint(0, 1000, (25, 2), generator=gen).cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, one = i32([30, 17]), i32([1, 1])

    def begin():
        decoder.start_paged(requests=2, num_blocks=12, max_seq=96, block_size=16)
        return decoder.forward_paged(prompt, lens, 30)

    begin()
    eager = [decoder.forward_paged(t, one, 1).clone() for t in tokens]
    begin()
    ids = tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = decoder.forward_paged(ids, one, 1)
    for t, want in zip(tokens, eager):
        ids.copy_(t)
        graph.replay()
        assert torch.equal(y, want)
    assert decoder.paged.lens.tolist() == [55, 42]
    decoder.paged = None


def test_refusals(decoder):
    from bladedisc_b200.kv_cache import PagedKVCache8
    decoder.paged = None
    with pytest.raises(RuntimeError, match="start_paged"):
        decoder.forward_paged(torch.zeros(1, dtype=torch.int64, device="cuda"), None, 1)
    for kw in (dict(block_size=8), dict(head_dim=80), dict(num_blocks=0)):
        with pytest.raises(ValueError):
            PagedKVCache8(**{**dict(layers=1, requests=1, num_blocks=1, kv_heads=1, head_dim=64, max_seq=1), **kw})
