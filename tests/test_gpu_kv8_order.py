"""Attention of mixed batches right behind what it reads, with other kernels of the library between its launches."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops as o
    yield o
    assert o.kernel_status() == 0, "a kernel's bounded wait ran out"


@pytest.mark.parametrize("kv", [300, 3000])
def test_another_thread_launches_on_the_same_stream(ops, kv):
    """Single tokens beside prompts, appended and attended in turn, while a second thread normalizes rows."""
    size, heads, q_heads, dim = 32, 2, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(21)
    q_lens = [1] * 20 + [130, 200] + [1] * 3
    kv_lens = [kv - i if q == 1 else kv for i, q in enumerate(q_lens)]
    n, width, tokens = len(q_lens), -(-kv // size), sum(q_lens)
    table = torch.randperm(n * width, generator=gen, device="cuda").to(torch.int32).view(n, width)
    i32 = lambda v: torch.as_tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    start, ql, kl = i32(np.cumsum([0] + q_lens)), i32(q_lens), i32(kv_lens)
    at = [(r, kv_lens[r] - q + i) for r, q in enumerate(q_lens) for i in range(q)]
    slots = torch.stack([table[r, pos // size] * size + pos % size for r, pos in at]).to(torch.int32)
    first = [torch.randint(-127, 128, (n * width, heads, size, dim), dtype=torch.int8, generator=gen, device="cuda")
             for _ in range(2)] + [torch.full((n * width, heads), 0.01, device="cuda") for _ in range(2)]
    rows = [torch.randn(tokens, (q_heads + 2 * heads) * dim, generator=gen, device="cuda").half() for _ in range(24)]
    h, gain = torch.randn(64, 1024, generator=gen, device="cuda").half(), torch.ones(1024, device="cuda").half()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()

    def steps():
        cache = [t.clone() for t in first]
        got = []
        for x in rows:
            q = ops.kv8_append(x, *cache, slots)
            got.append(ops.kv8_attention(q, *cache, table, start, ql, kl, max_q=200))
        return torch.stack(got)

    with torch.cuda.stream(stream):
        want = steps()
    stream.synchronize()
    done, others, launched = threading.Event(), [], [0]

    def other():
        try:
            with torch.cuda.stream(stream):
                while not done.is_set():
                    ops.rmsnorm_dynamic_quant(h, gain, 1e-5)
                    launched[0] += 1
        except Exception as e:  # shown by the thread that waits
            others.append(e)

    thread = threading.Thread(target=other)
    thread.start()
    try:
        with torch.cuda.stream(stream):
            got = [steps() for _ in range(3)]
    finally:
        done.set()
        thread.join()
    stream.synchronize()
    assert not others and launched[0] > 0
    assert all(torch.equal(g, want) for g in got)
