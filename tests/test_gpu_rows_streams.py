"""The 8-bit row table on several streams."""
import pytest
import torch

from instascene_amd.rows import QuantizedRows

pytestmark = pytest.mark.gpu


def test_a_second_stream_writes_right_behind_the_first_large_write():
    """A table without its helper table: the write that makes it comes behind long work on one stream, another stream writes disjoint rows
    without waiting for it."""
    P, F, n = 40000, 32, 9000
    order = torch.randperm(P, device="cuda")
    a, b = order[:n].contiguous(), order[n:2 * n].contiguous()
    base, xa, xb = (torch.randn(k, F, device="cuda") for k in (P, n, n))
    busy = torch.randn(4096, 4096, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for k in range(4):
        t = QuantizedRows.from_rows(base, dtype=torch.int8)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            old = torch.full((P,), 2 ** 30, dtype=torch.int32, device="cuda")       # what the helper table's memory holds before it is filled
            s1.synchronize()
            del old
            for _ in range(20):
                busy = torch.tanh(busy @ busy)
            t.write(xa, a)
        with torch.cuda.stream(s2):
            t.write(xb, b)
        torch.cuda.synchronize()
        want = QuantizedRows.from_rows(base, dtype=torch.int8).read()
        want[a], want[b] = QuantizedRows.from_rows(xa, dtype=torch.int8).read(), QuantizedRows.from_rows(xb, dtype=torch.int8).read()
        assert torch.equal(t.read(), want), k
        assert bool((t._owner == -1).all())


def test_a_dropped_table_stays_until_the_other_stream_is_done():
    P, F = 300_000, 32
    x, index = torch.randn(1000, F, device="cuda"), torch.arange(1000, device="cuda")
    t = QuantizedRows(P, F, dtype=torch.int8)
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = torch.tanh(busy @ busy)
        t.write(x, index)
    t.record_stream(side)
    held = {m.data_ptr() for m in (t.codes, t.scales, t._owner)}
    done = torch.cuda.Event()
    done.record(side)
    del t
    fresh = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (P * F, 4 * P, 4 * P)]
    if done.query():
        pytest.skip("the other stream was done too early to tell")
    assert not held & {m.data_ptr() for m in fresh}
    torch.cuda.synchronize()
