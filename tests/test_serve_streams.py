"""Which stream the calls of bpd_substrate_amd.serve name (no kernel is launched; no GPU)."""
import threading

import torch

from bpd_substrate_amd import gpu, serve


def test_the_stream_goes_with_the_call(monkeypatch):
    """Threads with streams of their own: each call carries its thread's, and the process-wide one, which the helpers of
    gpu set for themselves, is never touched."""
    current = threading.local()
    dev = torch.device("cuda", 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: current.stream, raising=False)
    set_, got = [], []

    def entry(stream, mine):
        got.append((stream, mine))

    monkeypatch.setitem(gpu._fns, "bpd_gpu_set_stream", set_.append)

    def work(i):
        current.stream = 1000 + i
        for _ in range(200):
            serve._launch(dev, entry, 1000 + i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert len(got) == 800 and all(a == b for a, b in got)
    assert set_ == []
