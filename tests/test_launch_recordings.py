"""When a program of several kernels is recorded as a CUDA graph (fake driver: calls are counted, nothing runs)."""
import pytest

from accy_b200 import tensor
from accy_b200._native import lib


@pytest.fixture
def launches():
    """A program of two kernels or more on the fake driver; call(k) launches it on the k-th set of device buffers and returns
    (kernels launched, graphs launched, graphs recorded) by that call."""
    lib.accy_b200_test_use_fake_driver(1)
    session = tensor.Session(device=0)
    compiled = session.compile(tensor.define("two_stage", [tensor.spec("f32", a=50, b=70)], lambda b, a: a[0].sum("b").max("a")))
    kernels = compiled.work()["launches"]
    assert kernels >= 2
    names = (b"cuLaunchKernel", b"cuGraphLaunch", b"cuGraphInstantiateWithFlags")

    def call(k):
        before = [lib.accy_b200_test_fake_call_count(n) for n in names]
        session.invoke_device(compiled, [(2 * k + 1) << 20], [(2 * k + 2) << 20], 1)
        return tuple(lib.accy_b200_test_fake_call_count(n) - b for n, b in zip(names, before))
    yield call, (kernels, 0, 0), (kernels, 1, 1), (0, 1, 0)
    session.deinit()
    lib.accy_b200_test_use_fake_driver(0)


def test_new_buffers_are_launched_directly(launches):
    call, direct, _, _ = launches
    assert all(call(k) == direct for k in range(20))


def test_buffers_that_come_again_are_recorded_and_replayed(launches):
    call, direct, recorded, replayed = launches
    assert [call(0) for _ in range(4)] == [direct, recorded, replayed, replayed]


def test_two_buffer_sets_in_turn_and_then_one(launches):
    """The graph that is there is replayed whenever its buffers come; once the buffers settle on others these are recorded too."""
    call, direct, recorded, replayed = launches
    assert [call(0), call(0)] == [direct, recorded]
    for _ in range(10):
        assert [call(1), call(0)] == [direct, replayed]
    settled = [call(1) for _ in range(6)]
    assert settled == [direct] * 3 + [recorded] + [replayed] * 2
    # recordings get rarer, but a caller that settles always gets one
    for k in range(2, 8):
        calls = [call(k) for _ in range(2 << k)]
        assert calls.count(recorded) == 1 and calls[-1] in (recorded, replayed)


def test_buffers_in_turn_are_never_recorded_at_first_sight(launches):
    call, direct, _, _ = launches
    assert all(call(k % 3) == direct for k in range(30))
