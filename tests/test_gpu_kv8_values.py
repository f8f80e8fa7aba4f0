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


def plain(q, cache, q_len, kv, scale):
    """One request in 64 bits: outputs, and what a kernel may be off by before it rounds its result.

    Probabilities times value scales enter the second product as f16, half a step 2^-11 relative to each, and 2^-25
    absolute where they are subnormal, in units that bring a row's largest one to 2^8 at least: 2^-33 of that for each key.
    Scores: (d + 4) 2^-23 of the magnitudes they are summed from, twice that in a probability; 2^-19 for exp2 and the rest."""
    k, v, ks, vs, table = cache
    g, d = q.shape[1] // k.shape[1], q.shape[2]
    q = q.double().cpu().numpy()
    want, allowed = np.zeros(q.shape), np.zeros(q.shape)
    hidden = np.arange(kv)[None] > (kv - q_len + np.arange(q_len))[:, None]
    each = np.repeat
    for h in range(q.shape[1]):
        kk, vv = (by_position(t, table)[h // g, :kv].astype(np.float64) for t in (k, v))
        ksh, vsh = (each(s[table[0], h // g].astype(np.float64), k.shape[2])[:kv] for s in (ks, vs))
        s = np.where(hidden, -np.inf, (q[:, h] @ kk.T) * ksh * scale)
        mag = np.where(hidden, 0, (np.abs(q[:, h]) @ np.abs(kk).T) * ksh * scale).max(axis=1, keepdims=True)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        want[:, h] = p @ (vv * vsh[:, None])
        largest = (p * vsh).max(axis=1, keepdims=True)
        allowed[:, h] = (p @ np.abs(vv * vsh[:, None])) * (2.0 ** -11 + 2 * mag * (d + 4) * 2.0 ** -23 + 2.0 ** -19) \
            + kv * 2.0 ** -33 * largest * 127
    return want, allowed


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,size", [(64, 16), (128, 64)])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("ratio,gap", [(20, 60), (30, 60), (20, 14), (-20, 0), (-30, 0)])
def test_a_block_of_other_magnitude(ops, ratio, gap, where, dim, size, dtype):
    """Values of one block 2^ratio times those of the others, its scores `gap` lower: with a large gap it has no part in
    the result, which has to keep its bits all the same; with 14 its part is like that of all others together."""
    rng = np.random.default_rng(2)
    for q_len, kv in ((1, 700), (5, 3000), (100, 700), (70, 5000)):
        cache = k, v, ks, vs, table = cache_of(rng, kv, size, 1, dim)
        blocks = k.shape[0]
        odd = table[0, {"first": 0, "middle": blocks // 2, "last": blocks - 1}[where]]
        ks[:] = 1 / 127
        k[:, :, :, 0] = 0
        k[odd, :, :, 0] = -127
        vs[odd] *= 2.0 ** ratio
        q = rng.standard_normal((q_len, 2, dim)).astype(np.float32) * 1.5
        q[:, :, 0] = gap * dim ** 0.5
        q = torch.from_numpy(q).to(dtype).cuda()
        got = attend(ops, q, cache, q_len, kv, dim ** -0.5).double().cpu().numpy()
        want, allowed = plain(q, cache, q_len, kv, dim ** -0.5)
        assert (np.abs(want) < 2.0 ** 15).all() and np.isfinite(want).all()
        bad = np.abs(got - want) > allowed * 1.001 + HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]
        assert not bad.any(), (q_len, kv, np.abs(got - want)[bad].max(), np.abs(want[bad]).max(), bad.mean())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_len,kv", [(2, 400), (3, 2500), (90, 400), (70, 5000)])
def test_value_scales_over_the_whole_range(ops, q_len, kv, dtype):
    """Blocks without values (scale 0) before, between and behind blocks of scales from 2^-60 to 2^8, in every order, and
    rows that see nothing but zeros."""
    rng = np.random.default_rng(3)
    dim, size, heads = 64, 16, 6
    cache = k, v, ks, vs, table = cache_of(rng, kv, size, heads, dim)
    blocks = k.shape[0]
    j = np.arange(blocks)
    by_head = [np.where(j % 2, 2.0 ** -8, 0), np.where(j < blocks // 2, 0, 2.0 ** -7), np.where(j < 3, 2.0 ** -6, 0),
               2.0 ** (-60 + 68 * j / blocks), 2.0 ** (8 - 68 * j / blocks), np.zeros(blocks)]
    vs[table[0]] = np.stack(by_head, axis=1).astype(np.float32)
    q = torch.from_numpy(rng.standard_normal((q_len, heads, dim)).astype(np.float32)).to(dtype).cuda()
    got = attend(ops, q, cache, q_len, kv, dim ** -0.5).double().cpu().numpy()
    want, allowed = plain(q, cache, q_len, kv, dim ** -0.5)
    assert not got[:, 5].any()
    bad = np.abs(got - want) > allowed * 1.001 + HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]
    assert not bad.any(), (np.abs(got - want)[bad].max(), np.argwhere(bad)[:5])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,size", [(64, 16), (128, 64)])
@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("q_len,kv,gap", [(1, 480, 9), (1, 8192, 13), (7, 8192, 13), (100, 1124, 10), (70, 16400, 14),
                                          (300, 2300, 11)])
def test_one_large_probability_beside_thousands(ops, q_len, kv, gap, where, dim, size, dtype):
    """One key 2^gap above 2^gap others, which together weigh as much as it does: half of the result comes from
    probabilities of 2^-gap of the largest, with the largest met first or last."""
    rng = np.random.default_rng(4)
    cache = k, v, ks, vs, table = cache_of(rng, kv, size, 1, dim)
    keys = by_position(k, table)
    keys[:, :, 0] = 0
    keys[0, 0 if where == "first" else kv - q_len, 0] = 127  # the last key that every row sees
    put_positions(k, table, keys)
    ks[:] = 1 / 127
    q = 0.2 * rng.standard_normal((q_len, 2, dim)).astype(np.float32)
    q[:, :, 0] = gap * np.log(2) * dim ** 0.5
    q = torch.from_numpy(q).to(dtype).cuda()
    s = (q.double().cpu().numpy() @ by_position(k, table)[0, :kv - q_len + 1].T) / 127 * dim ** -0.5
    p = np.exp(s - s.max(axis=-1, keepdims=True))
    largest = 1 / p.sum(axis=-1)
    # scores vary by 0.2 times the spread of a level, 0.58: twelve times that is the factor of four allowed here
    assert ((largest > 0.25) & (largest < 0.75)).all() and (np.sort(p, axis=-1)[..., -2] < 2.0 ** (2 - gap)).all()
    got = attend(ops, q, cache, q_len, kv, dim ** -0.5).double().cpu().numpy()
    want, allowed = plain(q, cache, q_len, kv, dim ** -0.5)
    bad = np.abs(got - want) > allowed * 1.001 + HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]
    assert not bad.any(), (np.abs(got - want)[bad].max(), np.argwhere(bad)[:5])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,group,dim,q_lens,kv_lens", [
    (1, 16, 64, [1, 120, 1, 1], [900, 333, 3000, 15]),        # single tokens of 16 rows
    (2, 4, 128, [4, 3, 100, 16, 1], [700, 1500, 100, 33, 64]),  # drafts of 4 to 64 rows
    (1, 33, 64, [1, 2, 70], [2000, 600, 70]),
])
def test_requests_of_a_few_rows_beside_prompts(ops, heads, group, dim, q_lens, kv_lens, dtype):
    """Between one tile of eight rows and a prompt: 9 to 66 rows per request and kv head, in one batch with prompts."""
    rng = np.random.default_rng(5)
    size, n = 16, len(q_lens)
    width = -(-max(kv_lens) // size)
    k, v, ks, vs, order = cache_of(rng, n * width * size, size, heads, dim)
    table = order.reshape(n, width)
    start = np.cumsum([0] + q_lens)
    q = torch.from_numpy(rng.standard_normal((start[-1], heads * group, dim)).astype(np.float32)).to(dtype).cuda()
    i32 = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    gpu = [torch.from_numpy(a).cuda() for a in (k, v, ks, vs, table)]
    got = ops.kv8_attention(q, *gpu, i32(start), i32(q_lens), i32(kv_lens), max_q=max(q_lens)).double().cpu().numpy()
    for r in range(n):
        rows = slice(start[r], start[r + 1])
        want, allowed = plain(q[rows], (k, v, ks, vs, table[r:r + 1]), q_lens[r], kv_lens[r], dim ** -0.5)
        bad = np.abs(got[rows] - want) > allowed * 1.001 + HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]
        assert not bad.any(), (r, np.abs(got[rows] - want)[bad].max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [20, 80, 150, 1000])
@pytest.mark.parametrize("where", ["first", "middle"])
def test_the_largest_probabilities_belong_to_a_block_without_values(ops, where, gap, dtype):
    """Keys of a block whose values are all zeros are e^gap times as probable as the others: what is left of those."""
    rng = np.random.default_rng(7)
    dim, size = 64, 16
    for q_len, kv in ((1, 400), (9, 3000), (80, 700), (70, 5000)):
        cache = k, v, ks, vs, table = cache_of(rng, kv, size, 1, dim)
        k[:, :, :, 0] = 0
        block = table[0, {"first": 0, "middle": k.shape[0] // 2}[where]]
        k[block, :, :, 0] = 127
        ks[:] = 1 / 127
        v[block], vs[block] = 0, 0
        q = rng.standard_normal((q_len, 2, dim)).astype(np.float32)
        q[:, :, 0] = gap * dim ** 0.5
        q = torch.from_numpy(q).to(dtype).cuda()
        got = attend(ops, q, cache, q_len, kv, dim ** -0.5).double().cpu().numpy()
        want, allowed = plain(q, cache, q_len, kv, dim ** -0.5)
        # below 2^-126 of the row's largest a probability is nothing
        allowed += 2.0 ** -126 * kv * vs.max() * 127
        bad = np.abs(got - want) > allowed * 1.001 + HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]
        assert np.isfinite(got).all() and not bad.any(), (q_len, kv, np.abs(got - want)[bad].max(), np.abs(want).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["first", "last", "all"])
def test_value_scales_that_are_not_finite_show(ops, which, bad, dtype):
    """In every value of the rows that see such a block, and in no other."""
    rng = np.random.default_rng(8)
    dim, size = 64, 16
    for q_len, kv in ((1, 400), (20, 3000), (80, 700), (300, 2000), (70, 5000)):
        cache = k, v, ks, vs, table = cache_of(rng, kv, size, 1, dim)
        blocks = k.shape[0]
        begin = {"first": 0, "last": blocks - 1, "all": 0}[which]
        vs[table[0, begin:] if which == "all" else table[0, begin]] = bad
        q = torch.from_numpy(rng.standard_normal((q_len, 2, dim)).astype(np.float32)).to(dtype).cuda()
        got = attend(ops, q, cache, q_len, kv, dim ** -0.5).double().cpu().numpy()
        see = kv - q_len + np.arange(q_len) >= begin * size
        assert see.any() and not np.isfinite(got[see]).any() and np.isfinite(got[~see]).all(), (q_len, kv)
