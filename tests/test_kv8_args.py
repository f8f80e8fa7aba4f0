"""Refusals of the paged 8-bit cache that are answered before anything touches a GPU, and the plain statements
the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

from bladedisc_b200 import lib as L
from oracle import kv8_ref


@pytest.fixture(scope="module")
def lib(built_lib):
    return L.load()


def _err(lib):
    return lib.disc_b200_last_error_string().decode()


def _refused(lib, fn, args, text):
    assert fn(ctypes.byref(args), None) != 0 and text in _err(lib), _err(lib)


def _cache():
    return L.Kv8Cache(0x1000, 0x1000, 0x1000, 0x1000, 4, 2, 16, 64)  # never dereferenced on these paths


def test_null_args(lib):
    for name in ("kv_blocks_extend", "kv_blocks_trim", "kv8_append", "kv8_read", "kv8_attention"):
        assert getattr(lib, "disc_b200_" + name)(None, None) != 0 and "null args" in _err(lib)


@pytest.mark.parametrize("call", ["kv_blocks_extend", "kv_blocks_trim"])
def test_blocks(lib, call):
    fn = getattr(lib, "disc_b200_" + call)

    def args(**kw):
        a = L.KvBlocksArgs(*[0x1000] * 5, 3, 4, 10, 16, 8, *[0x1000] * 5)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    _refused(lib, fn, args(requests=8193), "requests must be")
    _refused(lib, fn, args(requests=-1), "requests must be")
    _refused(lib, fn, args(block_size=0), "negative size")
    _refused(lib, fn, args(num_blocks=1 << 30), "32-bit")
    _refused(lib, fn, args(table_width=1 << 30), "32-bit")
    for name in ("tokens", "lens", "table", "free_list", "free_count"):
        _refused(lib, fn, args(**{name: None}), "null operand")
    if call == "kv_blocks_extend":
        _refused(lib, fn, args(max_tokens=-1), "negative size")
        for name in ("slots", "positions", "q_start", "q_lens", "kv_lens"):
            _refused(lib, fn, args(**{name: None}), "null operand")
    else:
        assert fn(ctypes.byref(args(requests=0)), None) == 0  # nothing to do


def _cache_refusals(lib, fn, args):
    for field, value, text in (("kv_heads", 0, "positive"), ("num_blocks", -1, "positive"), ("dim", 96, "head size"),
                               ("block_size", 24, "block size"), ("block_size", 8, "block size"),
                               ("num_blocks", 1 << 28, "32-bit"), ("k", None, "null operand"),
                               ("v_scale", None, "null operand"), ("v", 0x1008, "aligned")):
        a = args()
        setattr(a.cache, field, value)
        _refused(lib, fn, a, text)


def test_append(lib):
    fn = lib.disc_b200_kv8_append

    def args(**kw):
        a = L.Kv8AppendArgs(0x1000, 5, 8 * 64, 4, L.F16, 0x1000, 0x1000, 0x1000, 0x1000, 0x1000, 9, _cache())
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    _cache_refusals(lib, fn, args)
    _refused(lib, fn, args(type=L.F32), "element type")
    _refused(lib, fn, args(tokens=-1), "out of range")
    _refused(lib, fn, args(q_heads=-1), "out of range")
    _refused(lib, fn, args(ld_qkv=8 * 64 - 8), "16-byte")
    _refused(lib, fn, args(ld_qkv=8 * 64 + 4), "16-byte")
    _refused(lib, fn, args(qkv=0x1008), "16-byte")
    _refused(lib, fn, args(q_out=0x1008), "16-byte")
    _refused(lib, fn, args(table_rows=0), "not empty")
    _refused(lib, fn, args(tokens=1 << 30, q_heads=1 << 20, ld_qkv=1 << 30), "too many tokens and heads")
    for name in ("qkv", "slots", "positions", "sin_table", "q_out"):
        _refused(lib, fn, args(**{name: None}), "null operand")
    assert fn(ctypes.byref(args(tokens=0)), None) == 0


def test_read(lib):
    fn = lib.disc_b200_kv8_read

    def args(**kw):
        a = L.Kv8ReadArgs(_cache(), 0x1000, 3, L.BF16, 0x1000, 0x1000)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    _cache_refusals(lib, fn, args)
    _refused(lib, fn, args(type=L.F32), "element type")
    _refused(lib, fn, args(count=-1), "negative")
    _refused(lib, fn, args(v_out=0x1004), "aligned")
    for name in ("blocks", "k_out", "v_out"):
        _refused(lib, fn, args(**{name: None}), "null operand")
    assert fn(ctypes.byref(args(count=0)), None) == 0


def test_attention(lib):
    fn = lib.disc_b200_kv8_attention

    def args(**kw):
        a = L.Kv8AttentionArgs(0x1000, 0x1000, 7, 4 * 64, 4 * 64, 4, L.F16, _cache(), 0x1000, 0x1000, 0x1000, 0x1000,
                               3, 5, 2, 80, 0.125)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    _cache_refusals(lib, fn, args)
    _refused(lib, fn, args(type=L.F32), "element type")
    _refused(lib, fn, args(q_heads=3), "multiple of the kv heads")
    _refused(lib, fn, args(q_heads=0), "multiple of the kv heads")
    _refused(lib, fn, args(requests=65536), "out of range")
    _refused(lib, fn, args(tokens=-1), "out of range")
    _refused(lib, fn, args(max_q=-1), "out of range")
    _refused(lib, fn, args(table_width=1 << 28), "32-bit")
    _refused(lib, fn, args(ld_q=4 * 64 - 8), "16-byte")
    _refused(lib, fn, args(ld_out=4 * 64 + 4), "16-byte")
    _refused(lib, fn, args(out=0x1008), "16-byte")
    _refused(lib, fn, args(scale=0.0), "positive")
    # a long cache wants its workspace, whole and aligned; a short one none
    need_of = lambda **kw: lib.disc_b200_kv8_attention_workspace_bytes(ctypes.byref(args(**kw)))  # noqa: E731
    need = need_of(max_kv=513)
    assert need > 0 and need_of(max_kv=L.KV8_DIRECT_KEYS) == 0 and lib.disc_b200_kv8_attention_workspace_bytes(None) == -1
    for kw in (dict(), dict(workspace=0x1000, workspace_bytes=need - 1), dict(workspace=0x1008, workspace_bytes=need)):
        _refused(lib, fn, args(max_kv=513, **kw), "workspace")
    # many rows of one request over a long cache: their keys are cut into shares
    big = dict(tokens=300, max_q=300, max_kv=100000, requests=1)
    assert need_of(**big) >= 2 * 300 * 4 * (64 * 4 + 8) and need_of(**{**big, "max_kv": 600}) == 0
    _refused(lib, fn, args(workspace=0x1000, workspace_bytes=need_of(**big) - 1, **big), "workspace")
    a = args()
    a.cache.num_blocks = 0
    _refused(lib, fn, a, "without blocks")
    _refused(lib, fn, args(scale=float("nan")), "positive")
    for name in ("q", "out", "table", "q_start", "q_lens", "kv_lens"):
        _refused(lib, fn, args(**{name: None}), "null operand")
    for name in ("tokens", "requests", "max_q"):
        assert fn(ctypes.byref(args(**{name: 0})), None) == 0


def test_cpu_tensors_are_refused():
    from bladedisc_b200 import ops
    i = torch.zeros(2, dtype=torch.int32)
    c = (torch.zeros(3, 1, 16, 64, dtype=torch.int8),) * 2 + (torch.zeros(3, 1),) * 2
    with pytest.raises(ValueError, match="no CPU"):
        ops.kv_blocks_extend(i, i, i[:, None], i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="no CPU"):
        ops.kv_blocks_trim(i, i, i[:, None], i, i[:1], 16)
    with pytest.raises(ValueError, match="no CPU"):
        ops.kv8_append(torch.zeros(2, 192).half(), *c, i)
    with pytest.raises(ValueError, match="no CPU"):
        ops.kv8_read(*c, i)
    with pytest.raises(ValueError, match="no CPU"):
        ops.kv8_attention(torch.zeros(2, 1, 64).half(), *c, i[:, None], i, i, i, max_q=1)


def test_the_statements_agree_with_a_small_example():
    """Two requests, blocks of 4 from a stack of 3; the second does not fit."""
    table = np.full((2, 3), -1, np.int32)
    free = np.array([7, 5, 6], np.int32)
    lens = np.zeros(2, np.int32)
    got = kv8_ref.extend(np.array([6, 5]), lens, table, free, 3, 4, 16)
    slots, positions, q_start, q_lens, kv, new_lens, new_table, count = got
    assert q_start.tolist() == [0, 6, 11] and q_lens.tolist() == [6, 0] and kv.tolist() == [6, 0] and count == 1
    assert new_table.tolist() == [[6, 5, -1], [-1, -1, -1]]
    assert slots[:6].tolist() == [24, 25, 26, 27, 20, 21] and (slots[6:] == -1).all()
    back = kv8_ref.trim(np.zeros(2), new_lens, new_table, free, count, 4)
    assert back[0].tolist() == [0, 0] and (back[1] == -1).all() and back[2].tolist() == [7, 5, 6] and back[3] == 3


def test_the_append_statement_keeps_values():
    rng = np.random.default_rng(0)
    levels, scales = np.zeros((2, 1, 4, 8), np.int8), np.full((2, 1), np.nan, np.float32)
    x = rng.standard_normal((3, 1, 8)).astype(np.float32)
    x[2] *= 10  # the third token moves the first two to a larger scale
    for i in range(3):
        levels, scales = kv8_ref.append(x[i:i + 1], levels, scales, np.array([4 + i]))
    assert np.isnan(scales[0, 0]) and scales[1, 0] == np.float32(np.abs(x[2]).max()) / np.float32(127)
    # each of the two roundings of an old token is off by at most half a level of its scale
    assert np.abs(levels[1, 0, :3] * scales[1, 0] - x[:, 0]).max() <= scales[1, 0] * 1.01
