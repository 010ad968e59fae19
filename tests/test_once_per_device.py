"""What a call site sets up once per device before its first launch, with first calls on several threads: none may go on before it
is set up, and a failure is reported and tried again.  Host logic, checked without a GPU."""
import ctypes as C

import pytest

import clusternet_amd as cn


def _first_calls(threads, failures):
    out = [C.c_int(-1) for _ in range(3)]
    cn.lib().cn_host_once_per_device(threads, failures, *(C.byref(x) for x in out))
    return tuple(x.value for x in out)  # attempts, failed calls, calls that went on too early


@pytest.mark.parametrize("threads", [1, 2, 8])
def test_others_wait_for_the_first(threads):
    assert _first_calls(threads, 0) == (1, 0, 0)


@pytest.mark.parametrize("threads,failures", [(1, 1), (3, 1), (8, 3), (4, 4)])
def test_failures_are_reported_and_tried_again(threads, failures):
    assert _first_calls(threads, failures) == (min(threads, failures + 1), failures, 0)
