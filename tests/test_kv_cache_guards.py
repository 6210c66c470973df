"""4-bit key/value cache: calls at the edge of what is allowed, as far as that
needs no GPU."""
import threading

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
