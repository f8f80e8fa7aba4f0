"""Attention over the 8-bit cache for values at the ends of their ranges, against kv8_ref in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops as o
    yield o
    assert o.kernel_status() == 0, "a kernel's bounded wait ran out"


def cache_of(rng, kv, size, heads, dim):
    """Levels, scales and table of one request of kv tokens."""
    blocks = -(-kv // size)
    k, v = (rng.integers(-127, 128, (blocks, heads, size, dim)).astype(np.int8) for _ in range(2))
    ks, vs = ((np.exp(0.3 * rng.standard_normal((blocks, heads))) / 127).astype(np.float32) for _ in range(2))
    return k, v, ks, vs, rng.permutation(blocks).astype(np.int32)[None]


def by_position(t, table):
    """View [heads, tokens, dim] (a copy) of levels, by the token's position."""
    return t[table[0]].transpose(1, 0, 2, 3).reshape(t.shape[1], -1, t.shape[3])


def put_positions(t, table, x):
    """The other way round: levels by position into the cache."""
    b = t[table[0]].shape
    t[table[0]] = x.reshape(x.shape[0], b[0], b[2], b[3]).transpose(1, 0, 2, 3)


def attend(ops, q, cache, q_len, kv, scale):
    k, v, ks, vs, table = cache
    gpu = [torch.from_numpy(a).cuda() for a in (k, v, ks, vs, table)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return ops.kv8_attention(q, *gpu, i32([0, q_len]), i32([q_len]), i32([kv]), max_q=q_len, scale=scale)


def reference(q, cache, q_len, kv, scale):
    k, v, ks, vs, table = cache
    q64 = q.double().cpu().numpy()
    return kv8_ref.attention(q64, k, v, ks, vs, table, np.array([0, q_len]), [q_len], [kv], scale, np.zeros(q64.shape))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("level", [1, 0])
@pytest.mark.parametrize("q_len,kv", [(3, 700), (100, 700), (70, 9000), (300, 2000)])
def test_infinite_queries_show(ops, q_len, kv, level, dim, dtype):
    """A query with an infinity, over keys that bring it to -infinity but for some that make it +infinity or NaN (0 times
    infinity): those lie at every place of a group of 16 in turn, in the part of the cache that all rows see whole."""
    size, heads, group = 32, 16, 2
    rng = np.random.default_rng(1)
    cache = cache_of(rng, kv, size, heads, dim)
    keys = by_position(cache[0], cache[4])
    keys[:, :, 0] = rng.integers(-127, 0, keys.shape[:2])
    for h in range(heads):  # head h: place h of the groups
        keys[h, h:256:16, 0] = level
    put_positions(cache[0], cache[4], keys)
    q = torch.from_numpy(rng.standard_normal((q_len, heads * group, dim)).astype(np.float32)).to(dtype)
    q[::2, :, 0] = float("inf")
    q = q.cuda()
    got = attend(ops, q, cache, q_len, kv, dim ** -0.5).double().cpu().numpy()
    assert np.isnan(got[::2]).all()
    assert np.isfinite(got[1::2]).all()
    if kv < 1000:
        finite = torch.where(torch.isinf(q), 0, q)
        want, slack = reference(finite, cache, q_len, kv, dim ** -0.5)
        err = np.abs(got - want)[1::2]
        assert (err <= 1.001 * slack[1::2] + HALF_STEP[dtype] * np.abs(want[1::2]) + SMALLEST[dtype]).all()
