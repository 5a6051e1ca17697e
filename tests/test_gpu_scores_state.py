"""What a handle keeps for the score operators: the limit of bounded waits and the failures they leave."""
from concurrent.futures import ThreadPoolExecutor

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


# A call of every kernel and way of storing: up to 16 and 32 queries, tiles shared by clusters, query tiles
# with tensor stores, with an odd end and with plain stores.
CALLS = [(3, 40_000, 200, F32, 0), (20, 40_000, 200, BF16, 0), (3, 700, 2100, F32, 0), (200, 60_000, 700, BF16, 0),
         (200, 40_001, 200, F32, 0), (200, 40_001, 200, BF16, 1)]


@pytest.mark.parametrize("Q,n,dim,dtype,lead", CALLS)
def test_a_wait_that_runs_out_is_reported(ix, Q, n, dim, dtype, lead):
    """With a limit of 0 the wait for the first codes runs out: the call ends, the check reports it once, and
    the next call is right."""
    q, base = rows8(ix, Q, dim, 1, 2), rows8(ix, n, dim, 2, 2)
    out = torch.zeros(Q, n + 8, dtype=dtype, device="cuda")[:, lead:lead + n]
    for _ in range(2):
        ix.set_option("score_wait_us", 0)
        ix.fp8_scores(q, base, dim, 2.0 ** -9, out=out)
        torch.cuda.synchronize()
        with pytest.raises(capi.CoralError) as e:
            ix.scores_check()
        assert e.value.code == capi.ERR_KERNEL and "wait" in str(e.value)
        ix.scores_check()
        ix.set_option("score_wait_us", 2_000_000)
        ix.fp8_scores(q, base, dim, 2.0 ** -9, out=out)
        torch.cuda.synchronize()
        ix.scores_check()
        check_scores(out, q, base, dim, 2.0 ** -9, None)


def test_the_limit_of_waits(ix):
    assert ix.get_option("score_wait_us") == 2_000_000
    for v in (-1, 2_000_001):
        with pytest.raises(capi.CoralError) as e:
            ix.set_option("score_wait_us", v)
        assert e.value.code == capi.ERR_ARG
    ix.set_option("score_wait_us", 7)
    assert ix.get_option("score_wait_us") == 7


class Worker:
    """A thread that does what it is told, one thing after the other."""

    def __init__(self):
        self.pool = ThreadPoolExecutor(1)

    def __call__(self, f, *args):
        return self.pool.submit(f, *args).result()


def failed(ix):
    try:
        ix.scores_check()
        return False
    except capi.CoralError as e:
        assert e.code == capi.ERR_KERNEL
        return True


def test_every_thread_is_told_of_a_failed_wait(ix):
    q, base = rows8(ix, 3, 200, 1, 2), rows8(ix, 5000, 200, 2, 2)

    def call(limit):
        ix.set_option("score_wait_us", limit)
        ix.fp8_scores(q, base, 200)
        torch.cuda.synchronize()
        ix.set_option("score_wait_us", 2_000_000)
    first, second, late, watcher = (Worker() for _ in range(4))
    first(call, 2_000_000)
    second(call, 2_000_000)
    assert not first(failed, ix) and not second(failed, ix)
    first(call, 0)
    assert second(failed, ix) and first(failed, ix)           # one's check leaves the other's
    assert not second(failed, ix) and not first(failed, ix)   # once
    late(call, 2_000_000)
    assert not late(failed, ix)                               # what was found before it came is not its own
    assert watcher(failed, ix) and not watcher(failed, ix)    # no call of its own: all since the handle's creation
    second(call, 0)
    first(call, 2_000_000)
    assert [w(failed, ix) for w in (first, late, second, watcher)] == [True] * 4
    with capi.Index(1, 4, 32, "ip") as other:
        assert not first(failed, other) and not watcher(failed, other)


@pytest.mark.parametrize("Q,n,dim,dtype,lead", CALLS + [(3, 40_000, 20_000, F32, 0), (128, 512, 65536, F32, 0), (200, 20_000, 5000, BF16, 0)])
def test_a_wait_that_runs_out_on_the_way(ix, Q, n, dim, dtype, lead):
    """Short limits, which some waits keep: the call ends whichever runs out, and the next one is right."""
    q, base = rows8(ix, Q, dim, 1, 2), rows8(ix, n, dim, 2, 2)
    out = torch.zeros(Q, n + 8, dtype=dtype, device="cuda")[:, lead:lead + n]
    want = ix.fp8_scores(q, base, dim, 2.0 ** -9, dtype=dtype)
    for limit in (1, 3, 10, 30):
        for _ in range(3):
            ix.set_option("score_wait_us", limit)
            ix.fp8_scores(q, base, dim, 2.0 ** -9, out=out)
            torch.cuda.synchronize()
            if not failed(ix):
                assert torch.equal(out, want)
        ix.set_option("score_wait_us", 2_000_000)
        ix.fp8_scores(q, base, dim, 2.0 ** -9, out=out)
        torch.cuda.synchronize()
        assert not failed(ix) and torch.equal(out, want)
