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
