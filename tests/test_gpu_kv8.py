"""The paged 8-bit cache on the GPU against the plain numpy statements of oracle/kv8_ref.py.

Tables, slots, levels and scales are compared for equality: the statements do the kernels' float32 operations one
rounding at a time.  Attention is compared with float64 arithmetic; the allowance per value is derived in
kv8_ref.attention, plus half a step of the output's type (f16 2^-11, bf16 2^-8 relative)."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops as o
    yield o
    assert o.kernel_status() == 0, "a kernel's bounded wait ran out"


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a)).to(dtype).cuda()


# ------------------------------------------------------------------------------------------------ tables
def _tables(rng, requests, block, width, spare, most):
    lens = rng.integers(0, most + 1, requests)
    held = -(-lens // block)
    order = rng.permutation(int(held.sum()) + spare + 2)
    table = np.full((requests, width), -1, np.int32)
    at = 0
    for r in range(requests):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    free = np.full(len(order), -1, np.int32)
    free[:spare] = order[at:at + spare]
    return lens.astype(np.int32), table, free


@pytest.mark.parametrize("requests,block,width,spare,most,new,cap", [
    (1, 16, 1, 1, 0, 1, 1), (1, 16, 4, 0, 16, 5, 8), (3, 16, 8, 100, 100, 9, 64), (7, 64, 3, 4, 150, 60, 1000),
    (64, 64, 40, 20, 2000, 1, 64), (64, 16, 200, 5000, 2000, 900, 20000), (33, 32, 16, 40, 400, 200, 2500),
    (1025, 16, 6, 700, 60, 30, 20000), (8192, 16, 3, 9000, 20, 20, 100000), (5, 128, 0, 3, 0, 4, 10),
    (2500, 16, 2, 100, 3, 1, 2000), (4, 16, 3, 50, 48, 0, 0),
])
def test_extend_and_trim(ops, requests, block, width, spare, most, new, cap):
    rng = np.random.default_rng(requests * 1000 + block + new)
    lens, table, free = _tables(rng, requests, block, width, spare, min(most, width * block))
    tokens = rng.integers(-2, new + 1, requests).astype(np.int32)
    want = kv8_ref.extend(tokens, lens, table, free, spare, block, cap)
    d = [dev(v) for v in (tokens, lens, table, free, [spare])]
    p = ops.kv_blocks_extend(*d, block, cap)
    got = [t.cpu().numpy() for t in p] + [d[1].cpu().numpy(), d[2].cpu().numpy()]
    for name, g, w in zip(("slots", "positions", "q_start", "q_lens", "kv_lens", "lens", "table"), got, want):
        assert np.array_equal(g, w), name
    assert int(d[4]) == want[7] and np.array_equal(d[3].cpu().numpy(), free)
    # some requests shrink, some are released, some keep more than they have
    keep = rng.integers(-1, most + new + 2, requests).astype(np.int32)
    back = kv8_ref.trim(keep, want[5], want[6], free, want[7], block)
    e = [d[0].clone()] + [t.clone() for t in d[1:]]
    ops.kv_blocks_trim(dev(keep), *e[1:], block)
    assert np.array_equal(e[1].cpu().numpy(), back[0]) and np.array_equal(e[2].cpu().numpy(), back[1])
    assert np.array_equal(e[3].cpu().numpy(), back[2]) and int(e[4]) == back[3]
    # trim to the old lengths undoes the extend
    ops.kv_blocks_trim(dev(lens), *d[1:], block)
    assert np.array_equal(d[1].cpu().numpy(), lens) and np.array_equal(d[2].cpu().numpy(), table)
    assert np.array_equal(d[3].cpu().numpy(), free) and int(d[4]) == spare


def test_no_requests(ops):
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    p = ops.kv_blocks_extend(z, z, z.view(0, 4), dev([1, 2]), dev([2]), 16, 3)
    assert p.slots.tolist() == [-1] * 3 and p.positions.tolist() == [-1] * 3 and p.q_start.tolist() == [0]
    ops.kv_blocks_trim(z, z, z.view(0, 4), dev([1, 2]), dev([2]), 16)


def test_state_that_makes_no_sense_stays_in_bounds(ops):
    """Lengths beyond the table, a count beyond the stack, ids that are no blocks: no access outside the tensors."""
    table = np.array([[99, -7], [0, 1]], np.int32)
    d = [dev(v) for v in ([5, 3], [1000, 20], table, [50, -3, 2, 1], [77])]
    p = ops.kv_blocks_extend(*d, 16, 12)
    want = kv8_ref.extend(np.array([5, 3]), np.array([1000, 20]), table, np.array([50, -3, 2, 1]), 4, 16, 12)
    assert np.array_equal(p.q_lens.cpu().numpy(), want[3]) and np.array_equal(p.slots.cpu().numpy(), want[0])
    d = [dev(v) for v in ([3], [0], [[-1]], [-3], [1])]
    p = ops.kv_blocks_extend(*d, 16, 3)  # hands out an id that is no block
    assert p.slots.tolist() == [-1] * 3
    ops.kv_blocks_trim(dev([0]), *d[1:], 16)
    d = [dev(v) for v in ([0], [16], [[0]], [0], [1])]  # a stack that is full already
    ops.kv_blocks_trim(d[0], *d[1:], 16)
    assert int(d[4]) == 1 and d[1].tolist() == [0]


# ------------------------------------------------------------------------------------------------ append, read
def _cache(rng, blocks, heads, size, dim):
    k = rng.integers(-127, 128, (blocks, heads, size, dim)).astype(np.int8)
    v = rng.integers(-127, 128, (blocks, heads, size, dim)).astype(np.int8)
    ks = np.exp(rng.standard_normal((blocks, heads)) * 0.7).astype(np.float32) / 40
    vs = np.exp(rng.standard_normal((blocks, heads)) * 0.7).astype(np.float32) / 40
    return k, v, ks, vs


def _dev_cache(c):
    return [dev(c[0], torch.int8), dev(c[1], torch.int8), dev(c[2], torch.float32), dev(c[3], torch.float32)]


def _slots(rng, runs, size, blocks, pads):
    """Runs of consecutive tokens of different requests, each through fresh blocks from some offset on."""
    ids = rng.permutation(blocks).tolist()
    slots, pos = [], []
    for n in runs:
        start = int(rng.integers(0, 3 * size))
        b = None
        for i in range(n):
            p = start + i
            if b is None or p % size == 0:
                b = ids.pop()
            slots.append(b * size + p % size)
            pos.append(p)
        for _ in range(pads):
            slots.append(-1)
            pos.append(-1)
    return np.array(slots, np.int32), np.array(pos, np.int32)


def _check_append(ops, x, dtype, cache, slots, pos, q_heads, cos, sin, pad_cols=0):
    heads, dim = cache[0].shape[1], cache[0].shape[3]
    t = len(slots)
    wide = torch.full((t, x.shape[1] + pad_cols), 7.0, dtype=dtype, device="cuda")
    qkv = wide[:, :x.shape[1]]
    qkv.copy_(torch.from_numpy(x).cuda())
    seen = qkv.float().cpu().numpy().reshape(t, -1, dim)
    d = _dev_cache(cache)
    if cos is None:
        q = ops.kv8_append(qkv, *d, dev(slots))
        rot = seen
    else:
        q = ops.kv8_append(qkv, *d, dev(slots), dev(pos), dev(cos, torch.float32), dev(sin, torch.float32))
        at = np.clip(pos, 0, len(cos) - 1)
        rot = np.concatenate([kv8_ref.rotate(seen[:, :q_heads + heads], cos[at], sin[at]),
                              seen[:, q_heads + heads:]], axis=1)
    if q_heads:
        assert torch.equal(q, torch.from_numpy(rot[:, :q_heads]).to(dtype).cuda())
    else:
        assert q is None
    k, ks = kv8_ref.append(rot[:, q_heads:q_heads + heads], cache[0], cache[2], slots)
    v, vs = kv8_ref.append(rot[:, q_heads + heads:], cache[1], cache[3], slots)
    for name, got, want in (("k_scale", d[2], ks), ("v_scale", d[3], vs), ("k", d[0], k), ("v", d[1], v)):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=name.endswith("scale")), name
    # the input is not touched
    assert np.array_equal(qkv.float().cpu().numpy(), seen.reshape(t, -1), equal_nan=True)
    return d


@pytest.mark.parametrize("runs,size,heads,q_heads,dim,dtype,rope,pads,pad_cols", [
    ([1], 16, 1, 1, 64, torch.float16, True, 0, 0),
    ([1, 1, 1, 1, 1], 16, 4, 4, 64, torch.bfloat16, True, 1, 8),
    ([3, 40, 1, 17], 16, 2, 6, 128, torch.float16, True, 0, 0),
    ([129, 65, 5], 64, 3, 0, 128, torch.bfloat16, True, 2, 24),
    ([300], 128, 2, 5, 64, torch.float16, False, 0, 0),
    ([200, 333, 60], 32, 2, 2, 128, torch.float16, True, 0, 0),
    ([700, 1, 1500, 33], 16, 1, 8, 64, torch.bfloat16, True, 3, 0),
    ([1] * 70, 64, 8, 32, 128, torch.float16, True, 0, 0),
])
def test_append(ops, runs, size, heads, q_heads, dim, dtype, rope, pads, pad_cols):
    rng = np.random.default_rng(sum(runs) * 7 + size + dim)
    blocks = sum(-(-n // size) + 2 for n in runs) + 2
    slots, pos = _slots(rng, runs, size, blocks, pads)
    x = rng.standard_normal((len(slots), (q_heads + 2 * heads) * dim)).astype(np.float32)
    x *= np.exp(rng.standard_normal((len(slots), 1))).astype(np.float32)  # tokens of different size: scales grow
    ang = np.arange(pos.max() + 1)[:, None] * (10000.0 ** (-np.arange(dim // 2) / (dim // 2)))[None]
    cos, sin = (np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)) if rope else (None, None)
    _check_append(ops, x, dtype, _cache(rng, blocks, heads, size, dim), slots, pos, q_heads, cos, sin, pad_cols)


def test_append_of_zeros_and_of_values_that_are_not_finite(ops):
    rng = np.random.default_rng(3)
    cache = _cache(rng, 8, 2, 16, 64)
    cache[2][3] = 0.0      # a block of zeros that gets its first values at offset 4
    cache[0][3] = 0
    cache[3][5] = np.nan   # poisoned and reused from offset 0
    slots = np.array([3 * 16 + 4, 3 * 16 + 5, 0, 1, 5 * 16, 2 * 16 + 9, 6 * 16 + 15, 7 * 16], np.int32)
    x = rng.standard_normal((8, 4 * 64)).astype(np.float32)
    x[2:4] = 0.0           # a whole block of zeros
    x[5, 3] = np.inf
    x[6, 130] = np.nan
    x[7, 64:128] = 6e-8    # subnormal f16: scales near the smallest
    d = _check_append(ops, x, torch.float16, cache, slots, np.zeros(8, np.int32), 0, None, None)
    assert torch.isnan(d[2][2, 0]) and torch.isnan(d[3][6, 0]) and not torch.isnan(d[3][5]).any()


def test_append_step_by_step_reads_back_as_the_values(ops):
    """Fifty tokens one at a time: every value is within one level for each time the scale has grown, plus its own half."""
    rng = np.random.default_rng(11)
    size, dim, dtype = 16, 64, torch.float16
    cache = [torch.zeros(6, 1, size, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    cache += [torch.full((6, 1), float("nan"), device="cuda") for _ in range(2)]
    x = torch.from_numpy(rng.standard_normal((50, 128)).astype(np.float32)).to(dtype).cuda()
    growths = torch.zeros(6, dtype=torch.int64)
    for i in range(50):  # blocks 2, 3, 4 and two tokens of block 5
        was = cache[2][:, 0].clone()
        assert ops.kv8_append(x[i:i + 1], *cache, dev([2 * size + i])) is None
        growths += (cache[2][:, 0] > was).cpu()
    k, v = ops.kv8_read(*cache, dev([2, 3, 4, -1, 6]), dtype)
    assert not k[3:].any() and not v[3:].any()
    for j in range(3):
        # its own rounding and one for each growth, each half a level of at most the last scale; then the f16 result
        tol = float(cache[2][2 + j, 0]) * 0.501 * (1 + int(growths[2 + j])) + 2.0 ** -11 * float(x.abs().max())
        assert (k[j, 0].float() - x[j * size:(j + 1) * size, :64].float()).abs().max() <= tol
    assert torch.isnan(cache[2][:2]).all() and torch.isfinite(cache[2][2:]).all()


# ------------------------------------------------------------------------------------------------ attention
def _attend(ops, rng, q_lens, kv_lens, size, heads, q_heads, dim, dtype, *, cache=None, table=None, q_scale=1.0,
            max_q=None, max_kv=None, gap=0, ld=0, blocks=None, width=None):
    n = len(q_lens)
    held = [-(-max(k, 0) // size) for k in kv_lens]
    width = max(held + [1]) if width is None else width
    blocks = sum(held) + 2 if blocks is None else blocks
    if cache is None:
        cache = _cache(rng, blocks, heads, size, dim)
    if table is None:
        order = rng.permutation(blocks)
        table = np.full((n, width), -1, np.int32)
        at = 0
        for r in range(n):
            table[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
    start = np.cumsum([0] + [q + gap for q in q_lens]).astype(np.int32)
    tokens = int(start[-1])
    x = (rng.standard_normal((tokens, q_heads * dim)) * q_scale).astype(np.float32)
    wide = torch.zeros(tokens, q_heads * dim + ld, dtype=dtype, device="cuda")
    wide[:, :q_heads * dim] = torch.from_numpy(x).cuda()
    q = wide[:, :q_heads * dim].unflatten(1, (q_heads, dim))
    scale = dim ** -0.5
    out0 = torch.full((tokens, q_heads, dim), 3.0, dtype=dtype, device="cuda")
    d = _dev_cache(cache)
    args = [dev(v) for v in (table, start, q_lens, kv_lens)]
    mq = max(list(q_lens) + [0]) if max_q is None else max_q
    got = ops.kv8_attention(q, *d, *args, max_q=mq, max_kv=max_kv, out=out0.clone())
    want, slack = kv8_ref.attention(q.double().cpu().numpy(), *cache, table, start, q_lens, kv_lens, scale,
                                    out0.double().cpu().numpy(), mq)
    return got, want, slack, (q, d, args, mq)


def _check(got, want, slack):
    half = HALF_STEP[got.dtype]
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(want)), "NaN in other places"
    ok = ~np.isnan(want)
    over = np.abs(g - want)[ok] - (slack[ok] * (1 + half) + half * np.abs(want[ok]) + 2.0 ** -24)
    assert over.max(initial=-1) <= 0, f"{(over > 0).sum()} values off, the worst by {over.max():.3e} too much"


SHAPES = [
    # q_lens, kv_lens, block, kv heads, q heads, dim
    ([1], [1], 16, 1, 1, 64), ([1], [129], 16, 4, 4, 64), ([1], [2], 128, 2, 2, 128),
    ([1, 1, 1], [16, 17, 15], 16, 2, 8, 128), ([1] * 9, [1, 63, 64, 65, 127, 128, 129, 500, 1000], 64, 2, 2, 128),
    ([1, 1], [3000, 7], 16, 1, 16, 64), ([1], [5000], 32, 2, 14, 128), ([1, 1], [700, 900], 32, 1, 33, 64),
    ([7, 3, 1, 5], [300, 3, 90, 1111], 32, 2, 6, 64), ([2, 4], [400, 257], 128, 3, 3, 128),
    ([16, 9], [16, 640], 16, 2, 16, 128), ([24], [1000], 64, 5, 5, 64),
    ([128], [128], 16, 1, 1, 128), ([129, 1], [129, 1], 64, 2, 2, 64), ([300, 257], [300, 1000], 32, 2, 4, 128),
    ([1, 500, 1, 77, 1], [600, 500, 33, 200, 1025], 16, 2, 6, 128), ([640], [1500], 128, 1, 7, 64),
    # many rows over long caches: the keys in shares
    ([150], [6000], 16, 1, 2, 64), ([70, 1, 300], [4000, 9, 2500], 32, 2, 4, 128), ([200], [5003], 64, 1, 1, 128),
    ([255], [511], 16, 1, 3, 64), ([65, 190], [129, 190], 16, 2, 10, 128), ([1030], [1030], 64, 1, 2, 128),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"q{s[0][0]}x{len(s[0])}-kv{s[1][0]}-b{s[2]}-{s[4]}over{s[3]}-d{s[5]}")
def test_attention_matches_the_formula(ops, shape, dtype):
    q_lens, kv_lens, size, heads, q_heads, dim = shape
    rng = np.random.default_rng(sum(kv_lens) + size + dim + q_heads)
    got, want, slack, _ = _attend(ops, rng, q_lens, kv_lens, size, heads, q_heads, dim, dtype)
    _check(got, want, slack)


@pytest.mark.parametrize("big", [1, 40, 300])
def test_rows_without_keys_and_requests_without_rows(ops, big):
    """Empty requests, more rows than keys (the first rows see nothing), empty caches, rows of no request."""
    rng = np.random.default_rng(5)
    got, want, slack, _ = _attend(ops, rng, [0, big, 4, big, 3, 0], [50, 0, 2, big + 20, 3, 0], 16, 2, 4, 64,
                                  torch.float16, gap=3)
    _check(got, want, slack)
    start = [0, 3, big + 6, big + 13, 2 * big + 16, 2 * big + 22]
    assert not got[start[1]:start[1] + big].any() and not got[start[2]:start[2] + 2].any()
    assert (got[start[1] + big:start[2]] == 3).all() and (got[-3:] == 3).all()


@pytest.mark.parametrize("q_len", [1, 6, 200])
def test_bad_table_entries_are_left_out(ops, q_len):
    rng = np.random.default_rng(6)
    cache = _cache(rng, 12, 2, 16, 64)
    table = np.array([[3, -1, 5, 12, 1, 99, 7, -(2 ** 31), 2, 0, 11, 4, 6, 2 ** 31 - 1, 8]], np.int32)
    got, want, slack, _ = _attend(ops, rng, [q_len], [230], 16, 2, 4, 64, torch.float16, cache=cache, table=table)
    _check(got, want, slack)
    table = np.full((1, 15), -1, np.int32)
    got, want, slack, _ = _attend(ops, rng, [q_len], [230], 16, 2, 4, 64, torch.float16, cache=cache, table=table)
    assert not got.any()


@pytest.mark.parametrize("q_len,kv", [(1, 150), (5, 150), (140, 150)])
def test_what_lies_behind_the_last_key_does_not_count(ops, q_len, kv):
    """Levels of -128 and 127 behind the last token, scales of NaN in blocks no row or not every row sees."""
    rng = np.random.default_rng(7)
    k, v, ks, vs = _cache(rng, 14, 1, 16, 64)
    table = np.arange(13, dtype=np.int32)[None]
    k[9, :, 6:], v[9, :, 6:] = 127, -128       # token 150 sits at offset 6 of block 9
    ks[10:], vs[10:] = np.nan, np.inf          # blocks of no token
    got, want, slack, _ = _attend(ops, rng, [q_len], [kv], 16, 1, 2, 64, torch.float16, cache=(k, v, ks, vs),
                                  table=table)
    assert torch.isfinite(got).all()
    _check(got, want, slack)
    # the last block is poisoned: the rows that see none of it must not be
    for bad in (ks, vs):
        bad[9] = np.nan
        got, want, slack, _ = _attend(ops, rng, [q_len], [kv], 16, 1, 2, 64, torch.float16, cache=(k, v, ks, vs),
                                      table=table)
        _check(got, want, slack)
        assert torch.isnan(got[-6:]).all() and torch.isfinite(got[:-6]).all()
        bad[9] = 0.02


@pytest.mark.parametrize("q_len", [1, 150])
def test_scales_of_very_different_size(ops, q_len):
    """Value scales from 1e-30 to 1e3, whole blocks of zeros, scores that differ by hundreds."""
    rng = np.random.default_rng(8)
    k, v, ks, vs = _cache(rng, 20, 1, 16, 128)
    vs[:, 0] = 10.0 ** rng.uniform(-30, 3, 20)
    vs[5], vs[11] = 0.0, 0.0
    ks[3], ks[7] = 0.0, 3.0
    for order in (np.arange(20), np.argsort(vs[:, 0]), np.argsort(-vs[:, 0])):
        got, want, slack, _ = _attend(ops, rng, [q_len], [311], 16, 1, 1, 128, torch.bfloat16, cache=(k, v, ks, vs),
                                      table=order[None].astype(np.int32), q_scale=2.0)
        _check(got, want, slack)


def test_many_small_probabilities_beside_a_large_one(ops):
    """One key far above thousands of others that together weigh as much."""
    rng = np.random.default_rng(9)
    k, v, ks, vs = _cache(rng, 260, 1, 16, 64)
    k[:] = rng.integers(-3, 4, k.shape)
    k[100, 0, 3] = 0
    ks[:] = 0.01
    q_dir = np.zeros(64)
    q_dir[:8] = 40
    k[100, 0, 3, :8] = 90
    ks[100] = 0.0032
    got, want, slack, st = _attend(ops, rng, [1], [4000], 16, 1, 1, 64, torch.float16, cache=(k, v, ks, vs),
                                   table=np.arange(260, dtype=np.int32)[None])
    _check(got, want, slack)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [400, 33, 1]), ([7, 2], [70, 400]), ([200, 1], [400, 90])])
def test_strides_bounds_and_run_to_run(ops, q_lens, kv_lens):
    """Rows with a stride, a bound on the lengths that is too small or much too large, a table that is wider than
    needed: the same bits every time."""
    rng = np.random.default_rng(10)
    got, want, slack, (q, d, args, mq) = _attend(ops, rng, q_lens, kv_lens, 16, 2, 4, 64, torch.float16, ld=64,
                                                 width=40)
    _check(got, want, slack)
    again = ops.kv8_attention(q, *d, *args, max_q=mq, out=torch.full_like(got, 3.0))
    assert torch.equal(got, again)
    for max_kv in (0, 1, 100, 10 ** 6):
        other = ops.kv8_attention(q, *d, *args, max_q=mq, max_kv=max_kv, out=torch.full_like(got, 3.0))
        _check(other, want, slack)
    wide = ops.kv8_attention(q, *d, *args, max_q=4 * mq + 300, out=torch.full_like(got, 3.0))
    _check(wide, want, slack)


def test_rows_behind_max_q_are_left(ops):
    rng = np.random.default_rng(12)
    for q_len, mq in ((5, 2), (300, 140), (40, 1)):
        got, want, slack, _ = _attend(ops, rng, [q_len], [q_len + 9], 16, 1, 2, 64, torch.float16, max_q=mq)
        _check(got, want, slack)
        assert (got[mq:] == 3).all()


def test_a_request_whose_rows_are_not_in_q(ops):
    """q_start beyond the tensor or negative: nothing is read or written there."""
    rng = np.random.default_rng(13)
    for q_len in (3, 200):
        got, want, slack, (q, d, args, mq) = _attend(ops, rng, [q_len], [q_len], 16, 1, 1, 64, torch.float16)
        for start in (-2, q_len - 1, 10 ** 6, -(2 ** 31), 2 ** 31 - 1):
            s = dev([start, start + 1 if start < 2 ** 31 - 1 else start])
            o = ops.kv8_attention(q, *d, args[0], s, args[2], args[3], max_q=mq, out=torch.full_like(got, 3.0))
            w, sl = kv8_ref.attention(q.double().cpu().numpy(), *[t.cpu().numpy() for t in d],
                                      args[0].cpu().numpy(), np.array([start]), [q_len], [q_len], 0.125,
                                      np.full(got.shape, 3.0), mq)
            _check(o, w, sl)


@pytest.mark.parametrize("q_len", [1, 6, 180])
def test_a_row_of_nan_stays_alone(ops, q_len):
    """Infinities and NaN in one query row leave every other row as it is."""
    rng = np.random.default_rng(14)
    got, _, _, (q, d, args, mq) = _attend(ops, rng, [q_len, 3], [700, 40], 16, 2, 4, 64, torch.bfloat16)
    bad = q.clone()
    bad[0, 1, 5], bad[0, 2, 7] = float("nan"), float("inf")
    again = ops.kv8_attention(bad, *d, *args, max_q=mq, out=torch.full_like(got, 3.0))
    same = torch.ones(got.shape[:2], dtype=torch.bool)
    same[0, 1:3] = False
    assert torch.equal(again[same.cuda()], got[same.cuda()]) and torch.isnan(again[0, 1]).all()


def test_offsets_past_32_bits(ops):
    """Blocks that lie behind the first four gigabytes of levels: append, read and both attention kernels."""
    rng = np.random.default_rng(15)
    blocks, heads, size, dim = 34000, 8, 128, 128  # 4.46 GB of keys, as much of values
    k, v = (torch.zeros(blocks, heads, size, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(blocks, heads, device="cuda") for _ in range(2))
    ids = np.array([33999, 33990, 17, 33998, 33000], np.int32)
    small = _cache(rng, 5, heads, size, dim)
    at = dev(ids, torch.int64)
    for big, part, kind in ((k, small[0], torch.int8), (v, small[1], torch.int8), (ks, small[2], torch.float32),
                            (vs, small[3], torch.float32)):
        big[at] = dev(part, kind)
    for q_len, kv in ((1, 600), (300, 600), (5, 333)):
        q = torch.from_numpy(rng.standard_normal((q_len, heads, dim))).half().cuda()
        args = [dev([[0, 1, 2, 3, 4]]), dev([0, q_len]), dev([q_len]), dev([kv])]
        want = ops.kv8_attention(q, *_dev_cache(small), *args, max_q=q_len)
        got = ops.kv8_attention(q, k, v, ks, vs, dev(ids[None]), *args[1:], max_q=q_len)
        assert torch.equal(got, want)
    slots = np.array([33998 * size + 7, 33998 * size + 8, 33000 * size + 127], np.int64).astype(np.int32)
    x = rng.standard_normal((3, 2 * heads * dim)).astype(np.float32)
    xt = torch.from_numpy(x).half().cuda()
    ops.kv8_append(xt, k, v, ks, vs, dev(slots))
    local = np.array([3 * size + 7, 3 * size + 8, 4 * size + 127], np.int32)
    rows = xt.float().cpu().numpy().reshape(3, -1, dim)
    for big, scale, i, part in ((k, ks, 0, rows[:, :heads]), (v, vs, 1, rows[:, heads:])):
        levels, scales = kv8_ref.append(part, small[i], small[2 + i], local)
        assert np.array_equal(big[at].cpu().numpy(), levels) and np.array_equal(scale[at].cpu().numpy(), scales)
    a, b = ops.kv8_read(k, v, ks, vs, dev(ids), torch.float16)
    assert torch.equal(a, (k[at].float() * ks[at][..., None, None]).half())
    assert torch.equal(b, (v[at].float() * vs[at][..., None, None]).half())


@pytest.mark.parametrize("requests", [5, 33, 70])
@pytest.mark.parametrize("kv", [200, 3000])
def test_rows_behind_the_batch(ops, requests, kv):
    """q ends before the rows of its requests do; prompts of many lengths among requests of a few rows."""
    rng = np.random.default_rng(19)
    q_lens = [300 if i == 2 else 90 if i % 7 == 4 else 10 * (i % 3) + 1 for i in range(requests)]
    kv_lens = [max(q, kv - 13 * i) if i % 2 else q for i, q in enumerate(q_lens)]
    got, want, slack, (q, d, args, mq) = _attend(ops, rng, q_lens, kv_lens, 32, 1, 2, 64, torch.float16, gap=1)
    _check(got, want, slack)
    for cut in (311, q.shape[0] - 3, 17):
        part = ops.kv8_attention(q[:cut], *d, *args, max_q=mq, out=torch.full_like(got[:cut], 3.0))
        _check(part, want[:cut], slack[:cut])


def test_shares_without_keys(ops):
    """A bound on the lengths that promises a long cache, requests that are short or empty: shares of nothing."""
    rng = np.random.default_rng(18)
    got, want, slack, (q, d, args, mq) = _attend(ops, rng, [100, 80, 90], [130, 3, 90], 16, 1, 2, 64, torch.float16,
                                                 width=2000, gap=2)
    _check(got, want, slack)
    assert (got[100:102] == 3).all() and not got[102:179].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_lens, kv_lens, width", [
    ([330], [1100], 100),              # a whole round of items, and a few whose keys are in shares
    ([200, 1, 131], [900, 40, 700], 100),
    ([331] + [1] * 40, [1000] + [20] * 40, 120),   # room for more items than there are
])
def test_last_round_in_shares(ops, q_lens, kv_lens, width, dtype):
    """Up to 33 row blocks of 8 kv heads with 24 query heads each: more than one CTA per SM, the rest in shares."""
    rng = np.random.default_rng(21)
    got, want, slack, (q, d, args, mq) = _attend(ops, rng, q_lens, kv_lens, 16, 8, 192, 64, dtype, width=width)
    _check(got, want, slack)
    again = ops.kv8_attention(q, *d, *args, max_q=mq)
    assert torch.equal(got, again)


@pytest.mark.parametrize("kv", [300, 3000])
def test_steps_that_follow_at_once_read_what_was_appended(ops, kv):
    """Appends over the same slots and attention of prompts beside single tokens, waited for and not."""
    size, heads, q_heads, dim = 32, 2, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(20)
    q_lens = [1] * 40 + [130, 200] + [1] * 3
    kv_lens = [kv - i if q == 1 else kv for i, q in enumerate(q_lens)]
    n, width, tokens = len(q_lens), -(-kv // size), sum(q_lens)
    table = torch.randperm(n * width, generator=gen, device="cuda").to(torch.int32).view(n, width)
    start = dev(np.cumsum([0] + q_lens))
    ql, kl = dev(q_lens), dev(kv_lens)
    at = [(r, kv_lens[r] - q + i) for r, q in enumerate(q_lens) for i in range(q)]
    slots = torch.stack([table[r, pos // size] * size + pos % size for r, pos in at]).to(torch.int32)
    first = [torch.randint(-127, 128, (n * width, heads, size, dim), dtype=torch.int8, generator=gen, device="cuda")
             for _ in range(2)] + [torch.full((n * width, heads), 0.01, device="cuda") for _ in range(2)]
    rows = [torch.randn(tokens, (q_heads + 2 * heads) * dim, generator=gen, device="cuda").half() for _ in range(12)]
    outs = []
    for waits in (True, False):
        cache = [t.clone() for t in first]
        got = []
        for x in rows:
            q = ops.kv8_append(x, *cache, slots)
            if waits:
                torch.cuda.synchronize()
            got.append(ops.kv8_attention(q, *cache, table, start, ql, kl, max_q=200))
            got.append(got[-1] + 1)  # a reader of all rows
            if waits:
                torch.cuda.synchronize()
        outs.append(torch.stack(got).cpu())
    assert torch.equal(*outs)


@pytest.mark.parametrize("captured", [False, True])
def test_two_streams_at_once(ops, captured):
    """Calls that need a workspace on two streams, and two captured graphs of them, run side by side."""
    rng = np.random.default_rng(16)
    cases = []
    for i in range(2):
        got, _, _, (q, d, args, mq) = _attend(ops, rng, [1, 2], [9000, 5000 + i], 16, 2, 8, 128, torch.float16)
        cases.append((got, lambda q=q, d=d, args=args, mq=mq, got=got: ops.kv8_attention(
            q, *d, *args, max_q=mq, out=torch.full_like(got, 3.0))))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    runs, results = [], []
    for s, (_, call) in zip(streams, cases):
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                results.append(call())
            runs.append(g.replay)
        else:
            results.append(None)
            runs.append(call)
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                r = runs[i]()
                results[i] = results[i] if captured else r
    torch.cuda.synchronize()
    for (want, _), r in zip(cases, results):
        assert torch.equal(r, want)


def test_many_requests_with_few_prompts_among_them(ops):
    """More requests than a warp, prompts scattered between single tokens and empty ones."""
    rng = np.random.default_rng(17)
    n = 70
    q_lens = [1] * n
    for i, v in ((3, 150), (33, 90), (40, 0), (69, 200)):
        q_lens[i] = v
    kv_lens = [max(v, int(rng.integers(1, 120))) for v in q_lens]
    got, want, slack, _ = _attend(ops, rng, q_lens, kv_lens, 16, 2, 4, 64, torch.float16)
    _check(got, want, slack)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("captured", [False, True])
def test_decode_steps_together(ops, captured):
    """Prompts, then single tokens, with a request that ends and one that comes: tables, append and attention one
    after the other on their own stream; the step of single tokens also replayed from a CUDA graph."""
    rng = np.random.default_rng(21)
    R, size, heads, q_heads, dim, blocks, width = 4, 16, 2, 4, 64, 40, 12
    cols = (q_heads + 2 * heads) * dim
    lens, table = dev([0] * R), torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    free, count = dev(rng.permutation(blocks)), dev([blocks])
    cache = [torch.zeros(blocks, heads, size, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    cache += [torch.zeros(blocks, heads, device="cuda") for _ in range(2)]
    ang = np.arange(width * size)[:, None] * (10000.0 ** (-np.arange(dim // 2) / (dim // 2)))[None]
    cos, sin = dev(np.cos(ang), torch.float32), dev(np.sin(ang), torch.float32)

    def step(tokens, qkv, max_q):
        p = ops.kv_blocks_extend(tokens, lens, table, free, count, size, qkv.shape[0])
        q = ops.kv8_append(qkv, *cache, p.slots, p.positions, cos, sin)
        return p, q, ops.kv8_attention(q, *cache, table, p.q_start, p.q_lens, p.kv_lens, max_q=max_q)

    def verify(p, q, got):
        c = [t.cpu().numpy() for t in cache]
        want, slack = kv8_ref.attention(q.double().cpu().numpy(), *c, table.cpu().numpy(), p.q_start.cpu().numpy(),
                                        p.q_lens.tolist(), p.kv_lens.tolist(), dim ** -0.5,
                                        np.zeros(got.shape))
        served = np.zeros(got.shape[0], bool)
        for a, n in zip(p.q_start.tolist(), p.q_lens.tolist()):
            served[a:a + n] = True
        _check(got[torch.from_numpy(served).cuda()], want[served], slack[served])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = dev(rng.standard_normal((33 + 70 + 5, cols)), torch.float16)
        verify(*step(dev([33, 70, 0, 5]), x, 70))
        one = dev([1, 1, 0, 1])
        buf = torch.zeros(3, cols, dtype=torch.float16, device="cuda")
        if captured:
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = step(one, buf, 1)
        for i in range(20):
            if i == 8:  # the second request ends, the third one begins
                ops.kv_blocks_trim(dev([10 ** 6, 0, 10 ** 6, 10 ** 6]), lens, table, free, count, size)
                one.copy_(dev([1, 0, 1, 1]))
            buf.copy_(dev(rng.standard_normal((3, cols)), torch.float16))
            if captured:
                graph.replay()
                verify(*held)
            else:
                verify(*step(one, buf, 1))
    side.synchronize()
    assert lens.tolist() == [53, 0, 12, 25]
    used = [int(b) for b in table[table >= 0].tolist()]
    assert len(set(used)) == len(used) and sorted(used + free[:int(count)].tolist()) == list(range(blocks))


def test_refusals(ops):
    rng = np.random.default_rng(1)
    c = _dev_cache(_cache(rng, 4, 2, 16, 64))
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    i = dev([0, 1, 2])
    table = dev([[0, 1]] * 3)
    good = dict(max_q=1)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.kv8_attention(q.float(), *c, table, i, i, i, **good)
    with pytest.raises(ValueError, match="multiple of 2 heads"):
        ops.kv8_attention(q[:, :3], *c, table, i, i, i, **good)
    with pytest.raises(ValueError, match="one after the other"):
        ops.kv8_attention(q.transpose(0, 1).contiguous().transpose(0, 1), *c, table, i, i, i, **good)
    with pytest.raises(ValueError, match="one entry"):
        ops.kv8_attention(q, *c, table, i, i[:2], i, **good)
    with pytest.raises(ValueError, match="contiguous torch.int32"):
        ops.kv8_attention(q, *c, table, i, i, i.long(), **good)
    with pytest.raises(ValueError, match="contiguous torch.int8"):
        ops.kv8_attention(q, c[0].float(), *c[1:], table, i, i, i, **good)
    with pytest.raises(ValueError, match="scales"):
        ops.kv8_attention(q, c[0], c[1], c[2][:2].contiguous(), c[3], table, i, i, i, **good)
    with pytest.raises(ValueError, match="not on cuda"):
        ops.kv8_attention(q, *c, table, i, i, i.cpu(), **good)
    with pytest.raises(ValueError, match="q's shape"):
        ops.kv8_attention(q, *c, table, i, i, i, out=q[:2].clone(), **good)
    with pytest.raises(RuntimeError, match="score scale"):
        ops.kv8_attention(q, *c, table, i, i, i, scale=-1.0, **good)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="whole heads"):
        ops.kv8_append(qkv[:, :100], *c, i)
    with pytest.raises(ValueError, match="one slot"):
        ops.kv8_append(qkv, *c, i[:2])
    with pytest.raises(ValueError, match="needs cos"):
        ops.kv8_append(qkv, *c, i, i, torch.zeros(4, 32, device="cuda"))
    with pytest.raises(ValueError, match="cos / sin"):
        ops.kv8_append(qkv, *c, i, i, torch.zeros(4, 16, device="cuda"), torch.zeros(4, 16, device="cuda"))
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.kv8_append(torch.zeros(3 * 8 * 64 + 4, dtype=torch.float16, device="cuda")[4:].view(3, -1), *c, i)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.kv8_read(*c, i, torch.float32)
    with pytest.raises(ValueError, match="one entry"):
        ops.kv_blocks_trim(i[:2], i, table, i, dev([0]), 16)
    with pytest.raises(ValueError, match="must not be negative"):
        ops.kv_blocks_extend(i, i, table, i, dev([0]), 16, -1)
