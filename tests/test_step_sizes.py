"""Numbers that do not fit the C interface's 32 bits: bpd_substrate_amd.serve clamps them where that means the same, and
refuses them elsewhere.  No GPU."""
import pytest
import torch

from bpd_substrate_amd import gpu, serve

from test_serve_host import make
from test_step_host import i32

TOP = 2 ** 31 - 1


def pool():
    return serve.PagePool.empty(10, 16, 4, 5, windowed=True, device="cpu")


@pytest.fixture
def sent(monkeypatch):
    """What a call hands to the library."""
    got = []
    monkeypatch.setattr(serve, "_launch", lambda device, fn, *args: got.append(args))
    return got


@pytest.mark.parametrize("window,sinks,prefix_len,want", [
    (2 ** 32 + 5, 0, 0, (TOP, 0)), (64, 2 ** 32, 0, (64, TOP)), (64, 2 ** 32 + 7, 7, (64, TOP)), (2 ** 31, 2 ** 31, 0, (TOP, TOP)),
    (TOP, TOP, 0, (TOP, TOP)), (64, 2 ** 33 + 4, 2 ** 33, (64, 4)), (64, 4, 2 ** 33, (64, 0))])
def test_release_keeps_what_the_attention_sees(sent, window, sinks, prefix_len, want):
    """Every row of a pool is below 2^31: a window or sinks of as much keep all of them."""
    pool().release(window=window, sinks=sinks, prefix_len=prefix_len)
    assert sent[0][-2:] == want


def test_the_attention_clamps_alike(sent):
    c, b, q = make()
    serve.attention(c, b, q, window=2 ** 32 + 5, sinks=2 ** 32 + 1)
    assert sent[0][-4:-2] == (TOP, TOP)
    for window, sinks, text in ((5 - 2 ** 32, 0, "window"), (0, 0, "window"), (5, 1 - 2 ** 32, "sinks")):
        with pytest.raises(gpu.BpdqError, match=text):
            serve.attention(c, b, q, window=window, sinks=sinks)


def test_what_has_no_such_meaning_is_refused(sent):
    p, t = pool(), dict(table=i32(4, 5), lens=i32(4), free=i32(10), n_free=i32(2))
    c, b, q = make()
    far = torch.empty(0, dtype=torch.int32).expand(2 ** 32 + 3, 0)   # no memory behind it
    for f, text in ((lambda: p.extend(i32(2), 4, prefix_len=2 ** 32), "prefix_len"),
                    (lambda: p.extend(i32(2), 4, prefix_len=3 - 2 ** 32), "prefix_len"),
                    (lambda: p.extend(i32(2), 2 ** 32 + 4), "n_tokens"),
                    (lambda: serve.PagePool(page_size=2 ** 32 + 16, **t), "page_size"),
                    (lambda: serve.PagePool(page_size=16 - 2 ** 32, **t), "page_size"),
                    (lambda: serve.PagedBatch(i32(2, 5), i32(2), q_start=i32(3), n_tokens=2 ** 32 + 1), "n_tokens"),
                    (lambda: serve.PagedBatch(i32(2, 5), i32(2), prefix=i32(4), prefix_len=2 ** 32 + 1), "prefix_len"),
                    (lambda: serve.adjust_logits(torch.zeros(2, 0), mask=far), "masks")):
        with pytest.raises(gpu.BpdqError, match=text):
            f()
    assert not sent
