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


def test_a_later_error_of_another_thread(ix):
    """A thread that had its own failure, and asked for it, reads what another thread left since."""
    with pytest.raises(capi.CoralError):
        ix.set_option("mine", 1)
    with pytest.raises(capi.CoralError):
        in_a_thread(lambda: ix.set_option("theirs", 1))
    assert ix._lib.coral_last_error(ix._h).endswith(b"theirs")


def test_a_handle_that_outlives_its_thread(tmp_path):
    """A C++ program whose static object destroys its handle: the main thread's own state is gone by then."""
    import os
    import subprocess
    src, exe = tmp_path / "late.cpp", str(tmp_path / "late")
    src.write_text("""
#include <cstdio>
#include "coral_b200.h"
struct Holder {
    coral_index_t* h = nullptr;
    ~Holder() {
        coral_set_option(h, "none", 1);
        const bool text = coral_last_error(h) != nullptr;
        std::printf("destroyed %d %d\\n", coral_index_destroy(h), text);
        std::fflush(stdout);
    }
} holder;
int main() {
    if (coral_index_create(&holder.h, 0, 1, 4, 32, CORAL_IP) != CORAL_OK) return 2;
    coral_index_t* more[8];
    for (auto& h : more)
        if (coral_index_create(&h, 0, 1, 4, 32, CORAL_IP) != CORAL_OK || coral_scores_check(h) != CORAL_OK) return 3;
    return coral_scores_check(holder.h);
}
""")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.dirname(capi.lib_path())
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(root, "include"), str(src), "-o", exe, "-L" + lib, "-lcoral_b200",
                    "-Wl,-rpath," + lib], check=True, capture_output=True, timeout=120)
    # freed memory is overwritten, so that a use of it shows
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120, env=dict(os.environ, MALLOC_PERTURB_="165"))
    assert r.returncode == 0 and r.stdout == "destroyed 0 1\n", (r.returncode, r.stdout, r.stderr)
