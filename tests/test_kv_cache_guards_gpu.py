"""4-bit key/value cache on the GPU at the edge of what is allowed.  Bounds as
in test_kv_cache_gpu.py, whose cases these use."""
import threading

import pytest
import torch

from test_kv_cache_gpu import Case, _device, device_error  # noqa: F401 (_device: a fixture)

pytestmark = pytest.mark.gpu


def test_threads_share_a_batch_and_a_stream():
    """Calls of several host threads on their common default stream, each with
    parts to join: every thread gets the bits of its own call."""
    case = Case([2100, 900], [1, 1], 2, 128, page=32, junk=True)
    queries = [case.queries(8, 128, torch.float16) for _ in range(4)]
    want = [case.cache.attention(q, case.batch) for q in queries]
    for q, y in zip(queries, want):
        case.check(q, y)
    got = [[] for _ in queries]
    go = threading.Barrier(len(queries))

    def calls(i):
        go.wait(30)
        got[i] += [case.cache.attention(queries[i], case.batch) for _ in range(50)]

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(queries))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert len(ys) == 50 and all(torch.equal(x, y) for x in ys)
    assert device_error() == 0


def test_two_streams_in_flight_at_once():
    case = Case([3000, 500, 1200], [1, 1, 1], 2, 64, page=16, junk=True)
    q = [case.queries(16, 64, torch.bfloat16) for _ in range(2)]
    want = [case.cache.attention(x, case.batch) for x in q]
    case.check(q[0], want[0])
    case.check(q[1], want[1])
    streams = [torch.cuda.Stream() for _ in q]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(40):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(case.cache.attention(q[i], case.batch))
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert all(torch.equal(x, y) for x in ys)
