"""Drafted tokens that are taken back inside a block and appended over: what of the cache is as before, and what is not."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops as o
    return o


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def state(cache):
    return [t.cpu().numpy() for t in (cache.lens, cache.table, cache.free_list, cache.free_count)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,size", [(64, 16), (128, 64)])
@pytest.mark.parametrize("loud", [0.25, 30.0, float("inf")])
def test_a_rejected_draft(ops, loud, dim, size, dtype):
    """Tables, lengths and stack return to what they were.  Levels and scales of blocks that keep tokens do not: the
    scale stays that of the largest value ever stored since the block was begun, kept tokens at its levels, and later
    tokens use it; NaN if a draft held a value that is not finite.  A block that is begun anew starts over."""
    from bladedisc_b200.kv_cache import PagedKVCache8
    rng = np.random.default_rng(6)
    heads, requests = 2, 3
    cache = PagedKVCache8(1, requests, 40, heads, dim, 6 * size, size)
    levels = [t[0].cpu().numpy() for t in (cache.k, cache.v)]
    scales = [t[0].cpu().numpy() for t in (cache.k_scale, cache.v_scale)]

    def step(tokens, by=1.0):
        plan = cache.extend(i32(tokens), sum(tokens))
        x = torch.from_numpy(by * rng.uniform(0.5, 1, (sum(tokens), 2 * heads, dim)).astype(np.float32)).to(dtype)
        assert cache.append(0, x.reshape(sum(tokens), -1).cuda(), plan) is None
        slots, x = plan.slots.cpu().numpy(), x.float().numpy()
        for i in range(2):
            levels[i], scales[i] = kv8_ref.append(x[:, i * heads:(i + 1) * heads], levels[i], scales[i], slots)
        for got, want in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), levels + scales):
            assert np.array_equal(got[0].cpu().numpy(), want, equal_nan=True)

    kept = [size + 3, 2 * size, size - 1]  # inside a block, at its end, before it
    step(kept)
    before, old = state(cache), [s.copy() for s in scales]
    step([5, 4, 3], loud)
    cache.trim(i32(kept))
    assert all(np.array_equal(a, b) for a, b in zip(state(cache), before))
    table = before[1]
    inside = [table[0, 1], table[2, 0]]  # keep tokens beside the draft's
    whole = [table[0, 0], table[1, 0], table[1, 1]]
    for was, now in zip(old, scales):
        assert np.array_equal(was[whole], now[whole])
        if np.isinf(loud):
            assert np.isnan(now[inside]).all()
        else:
            assert (now[inside] >= was[inside]).all() and (loud < 1 or (now[inside] > 10 * was[inside]).all())
    step([1, 1, 1])  # over the draft's places
    step([size, size, size])
    for now in scales:  # the second request's block behind its full ones was begun anew
        assert (now[table_of(cache)[1, 2]] < 1.01 / 127).all()


def table_of(cache):
    return cache.table.cpu().numpy()
