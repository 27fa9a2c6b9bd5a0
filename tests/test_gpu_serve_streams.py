"""Which stream the operators of include/bpdq_serve.h launch on, beside the library's other calls."""
import threading

import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import gpu, serve, synth

pytestmark = pytest.mark.gpu


def test_serving_calls_leave_the_launch_stream_alone(dev):
    """bpd_gpu_set_stream()'s stream stays the program's own: a call after serve's still waits for it."""
    b = O.Batch(31, [1] * 4, [70, 20, 33, 1], 40, 8, 2, 64, "f16", "f16", 16, decode=True)
    cache, batch, q = b.device(dev)
    rope = serve.Rope(64, device=dev)
    logits, u = torch.randn(4, 1000, device=dev), torch.rand(4, device=dev)
    x, y = torch.zeros(64, device=dev), torch.zeros(64, device=dev)
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    step = (lambda: serve.attention(cache, batch, q), lambda: serve.sample(logits, u),
            lambda: serve.rope_append(cache, batch, q, None, None, rope=rope))
    for call in step:
        call()
        y.zero_()
        torch.cuda.synchronize()
        gpu.call("bpd_gpu_set_stream", mine.cuda_stream)
        try:
            with torch.cuda.stream(mine):
                torch.cuda._sleep(500_000_000)
            call()
            gpu.call("bpd_expf_gpu", x, y, 64)     # on `mine`, behind the sleep
            with torch.cuda.stream(other):
                seen = y.clone()
            other.synchronize()
            assert not mine.query(), "the sleep was over too early to tell"
            assert (seen == 0).all()
            mine.synchronize()
            assert (y == 1).all()
        finally:
            gpu.call("bpd_gpu_set_stream", 0)


def test_serving_beside_the_helpers_of_gpu_on_streams_of_their_own(dev):
    """A thread that serves and a thread that dequantizes: neither launches on the other's stream."""
    b = O.Batch(32, [1] * 6, [900, 20, 333, 1, 64, 500], 300, 8, 2, 64, "f16", "f16", 16, decode=True)
    cache, batch, q = b.device(dev)
    w = torch.from_numpy(synth.q4k(64, 4096, synth.key(42, 7))).to(dev)
    want = serve.attention(cache, batch, q), gpu.dequant_q4k(w)
    torch.cuda.synchronize()
    wrong, ready = [], threading.Barrier(2)

    def work(i, call):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            ready.wait()
            for _ in range(100):
                got = call()
                st.synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    ts = [threading.Thread(target=work, args=a) for a in ((0, lambda: serve.attention(cache, batch, q)),
                                                          (1, lambda: gpu.dequant_q4k(w)))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not wrong
