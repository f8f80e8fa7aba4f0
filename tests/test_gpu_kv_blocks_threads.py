"""Block tables of large batches built by several host threads at once, each with its own cache and stream."""
import ctypes
import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from bladedisc_b200 import ops as o
    return o


@pytest.mark.parametrize("sizes", [(8192, 5000), (8192, 6200, 4100, 100)])
def test_batches_of_different_sizes_at_once(ops, sizes):
    """The bookkeeping of more than 4096 (trim: 6144) requests takes more shared memory than a kernel has unasked."""
    calls, errors, results = 400, [], {}
    gate = threading.Barrier(len(sizes))

    def work(requests):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                i32 = dict(dtype=torch.int32, device="cuda")
                lens, table = torch.zeros(requests, **i32), torch.full((requests, 2), -1, **i32)
                free = torch.arange(2 * requests, **i32)
                count = torch.full((1,), 2 * requests, **i32)
                new, none = torch.full((requests,), 3, **i32), torch.zeros(requests, **i32)
                stream.synchronize()
                gate.wait()
                for _ in range(calls):
                    plan = ops.kv_blocks_extend(new, lens, table, free, count, 16, 3 * requests)
                    ops.kv_blocks_trim(none, lens, table, free, count, 16)
                stream.synchronize()
                results[requests] = (plan.slots.cpu(), plan.q_lens.cpu(), lens.cpu(), free.cpu(), int(count), table.cpu())
        except Exception as e:  # raised below, in the thread that waits
            errors.append((requests, e))

    threads = [threading.Thread(target=work, args=(n,)) for n in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for n in sizes:
        slots, q_lens, lens, free, count, table = results[n]
        block = 2 * n - 1 - torch.arange(n)  # taken from the top of the stack
        want = (block[:, None] * 16 + torch.arange(3)).reshape(-1)
        assert torch.equal(slots, want.int()) and (q_lens == 3).all() and not lens.any()
        assert torch.equal(free, torch.arange(2 * n).int()) and count == 2 * n and (table == -1).all()


@pytest.mark.parametrize("call,sizes", [("kv_blocks_trim", (8192, 6200)), ("kv_blocks_extend", (8192, 4200))])
def test_calls_in_close_succession(ops, call, sizes):
    """The same through the C entry points, so that the calls of two threads overlap as often as they can."""
    from bladedisc_b200 import lib as L
    lib = L.load()
    fn = getattr(lib, "disc_b200_" + call)
    gate, codes, held = threading.Barrier(len(sizes)), {}, []

    def arguments(n):
        i32 = dict(dtype=torch.int32, device="cuda")
        t = [torch.zeros(n, **i32), torch.zeros(n, **i32), torch.full((n, 1), -1, **i32), torch.arange(n, **i32),
             torch.full((1,), n, **i32), torch.empty(1, **i32), torch.empty(1, **i32), torch.empty(n + 1, **i32),
             torch.empty(n, **i32), torch.empty(n, **i32)]
        held.append(t)
        a = [x.data_ptr() for x in t]
        return ctypes.byref(L.KvBlocksArgs(*a[:5], n, 1, n, 16, 1, *a[5:]))

    def work(n, args, stream):
        gate.wait()
        bad = 0
        for _ in range(6000):
            bad += fn(args, stream.cuda_stream) != 0
        codes[n] = bad

    jobs = [(n, arguments(n), torch.cuda.Stream()) for n in sizes]
    torch.cuda.synchronize()
    switch = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=j) for j in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(switch)
    torch.cuda.synchronize()
    assert codes == {n: 0 for n in sizes}
