"""4-bit key/value cache: calls at the edge of what is allowed, as far as that
needs no GPU."""
import math
import threading

import pytest
import torch


def test_threads_on_one_stream_have_workspaces_of_their_own(monkeypatch):
    """A call is several kernels that hand results on through the workspace,
    and two threads on one stream may launch theirs in turn."""
    from openquant_b200 import kv_cache as kc

    monkeypatch.setattr(kc, "_stream_handle", lambda dev: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    batch = kc.KVBatch.__new__(kc.KVBatch)
    batch._dev, batch._buffers = 0, {}
    held, both = [], threading.Barrier(2)

    def call():
        ws = batch._workspace(4096, "cpu")
        both.wait(10)  # both threads are between the kernels of their calls
        held.append(ws)
        assert batch._workspace(4096, "cpu") is ws  # the next call of this thread

    threads = [threading.Thread(target=call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(held) == 2 and held[0].data_ptr() != held[1].data_ptr()


def test_workspaces_of_many_threads_are_not_all_kept(monkeypatch):
    from openquant_b200 import kv_cache as kc

    monkeypatch.setattr(kc, "_stream_handle", lambda dev: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    batch = kc.KVBatch.__new__(kc.KVBatch)
    batch._dev, batch._buffers = 0, {}
    for i in range(9):
        monkeypatch.setattr(threading, "get_ident", lambda i=i: i)
        assert batch._workspace(64, "cpu").numel() == 64
    assert len(batch._buffers) <= 4


@pytest.mark.parametrize("dim, base, original, factor", [
    (128, 1e4, 4096, 8.0),     # both turning points among the pairs
    (128, 1e4, 131072, 4.0),   # even the slowest pair turns more than once
    (32, 1e4, 131072, 8.0),
    (64, 500.0, 65536, 2.0),
    (128, 1e4, 150, 4.0),      # even the fastest pair turns less than 32 times
    (64, 1e4, 5, 4.0),         # no pair turns once
])
def test_rotary_scaling_by_parts_is_a_line_between_the_turning_points(dim, base, original, factor):
    from openquant_b200.kv_cache import _frequencies

    plain, _ = _frequencies(dim, base, None)
    got, _ = _frequencies(dim, base, {"type": "parts", "factor": factor, "original_positions": original})
    turns = original / (2 * math.pi) * base ** (-2.0 * torch.arange(-8 * dim, 9 * dim, dtype=torch.float64) / dim)
    index = range(-8 * dim, 9 * dim)
    first = max(i for i, t in zip(index, turns) if t >= 32)
    last = min(i for i, t in zip(index, turns) if t <= 1)
    for i in range(dim // 2):
        share = min(max((i - first) / (last - first), 0.0), 1.0)  # of the divided angle
        want = plain[i] * (1 - share) + plain[i] / factor * share
        assert math.isclose(float(got[i]), float(want), rel_tol=1e-12), i
        t = original * plain[i] / (2 * math.pi)
        if t >= 32 * base ** (2 / dim):
            assert got[i] == plain[i]
        if t <= base ** (-2 / dim):
            assert math.isclose(float(got[i]), float(plain[i]) / factor, rel_tol=1e-12)


def test_too_many_key_heads_are_refused_before_anything_is_launched():
    import ctypes

    from openquant_b200 import _native as nat, build, kv_cache as kc

    build.build()
    lib, p = nat.load(), 1 << 20
    cache = kc._Cache(p, p, p, p, 4, 16, 40000, 128, 32)
    batch = kc._Batch(p, p, None, 2, 2, 1)
    heads = 32 * 40000  # two blocks of 16 rows a key head: 80000 items
    st = lib.oq_kv4_attention(ctypes.byref(cache), ctypes.byref(batch), p, nat.OQ_F16, heads, heads * 128, 128, p, None,
                              2, 1.0, 0, 0, p, 1 << 40, None)
    assert st == nat.OQ_ERR_INVALID and "key heads" in nat.last_error()


def test_scales_whose_log2_factor_is_not_finite_are_refused():
    import ctypes

    from openquant_b200 import _native as nat, build, kv_cache as kc

    build.build()
    lib, p = nat.load(), 1 << 20
    cache, batch = kc._Cache(p, p, p, p, 4, 16, 2, 128, 32), kc._Batch(p, p, None, 2, 2, 1)
    for scale in (2.5e38, -3e38, math.inf, math.nan):
        st = lib.oq_kv4_attention(ctypes.byref(cache), ctypes.byref(batch), p, nat.OQ_F16, 4, 512, 128, p, None, 2, scale,
                                  0, 0, p, 1 << 30, None)
        assert st == nat.OQ_ERR_INVALID and "finite" in nat.last_error()
