"""The score operators from threads of a program."""
import threading

import pytest
import torch

from coral_b200 import capi
from tests.test_gpu_scores import BF16, F32, check_scores, rows8

pytestmark = pytest.mark.gpu


@pytest.fixture
def ix():
    with capi.Index(1, 4, 32, "ip") as h:
        yield h
        torch.cuda.synchronize()


def in_a_thread(f):
    got = []

    def work():
        try:
            got.append(f())
        except BaseException as e:
            got.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(got[0], BaseException):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("Q,n,dim,dtype", [(3, 5000, 200, F32), (3, 700, 2100, F32), (200, 40_000, 200, BF16)])
def test_first_call_of_a_thread(ix, Q, n, dim, dtype):
    """A thread whose first use of the GPU is the product: its device is current, its context not yet."""
    q, base = rows8(ix, Q, dim, 1, 2), rows8(ix, n, dim, 2, 2)
    out = torch.zeros(Q, n, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    in_a_thread(lambda: ix.fp8_scores(q, base, dim, 2.0 ** -9, out=out))
    torch.cuda.synchronize()
    check_scores(out, q, base, dim, 2.0 ** -9, None)


def test_threads_that_are_refused_at_once(ix):
    """Two threads with different refusals on one handle: each reads its own text, whole; launches are counted."""
    x = torch.randn(4, 64, device="cuda")
    before = ix.launch_count
    turns, wrong = 2000, []
    start = threading.Barrier(3)
    lib, h, d = ix._lib, ix._h, x.data_ptr()
    texts = {}

    def work(i, call):
        try:
            start.wait()
            for _ in range(turns):
                assert call() == capi.ERR_ARG
                got = lib.coral_last_error(h)
                assert texts.setdefault(i, got) == got and len(got) > 20, (texts[i], got)
        except BaseException as e:
            wrong.append(e)

    def count():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(turns):
                    ix.fp8_quantize(x)
            stream.synchronize()
        except BaseException as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(0, lambda: lib.coral_fp8_quantize(h, d, 0, 4, 64, 63, d, d, 1))),
               threading.Thread(target=work, args=(1, lambda: lib.coral_fp8_scores(h, d, d, 4, d, d, 4, 0, 1.0, None, d, 0, 4, 1))),
               threading.Thread(target=count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    assert texts[0].startswith(b"ld must be") and texts[1].startswith(b"dim must be")
    assert ix.launch_count - before == turns


def test_the_error_text_of_another_thread(ix):
    """A thread without a failure of its own on the handle reads the last of any thread's."""
    with capi.Index(1, 4, 32, "ip") as other:
        for h, name in ((ix, "no such one"), (other, "nor this")):
            with pytest.raises(capi.CoralError):
                in_a_thread(lambda h=h, name=name: h.set_option(name, 1))
        read = lambda h: h._lib.coral_last_error(h._h)
        assert read(ix).endswith(b"no such one") and read(other).endswith(b"nor this")
        with pytest.raises(capi.CoralError):
            ix.set_option("mine", 1)
        in_a_thread(lambda: read(ix))
        assert read(ix).endswith(b"mine") and read(other).endswith(b"nor this") and read(ix).endswith(b"mine")
