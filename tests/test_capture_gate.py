"""A step capture that begins in one thread while another thread's call synchronizes the device, on the CPU: over the HIP
runtime that runs nothing (tests/cpp/fake_hip.cpp), which counts the synchronizations that meet a capture; on a GPU one
would end that capture."""
import ctypes
import threading

import pytest

from test_serving_refusals import Fake
from tmac_attn import TMAC_OK


@pytest.fixture
def two():
    pair = Fake(), Fake()
    pair[0].lib.fake_set_capture_us(300)
    yield pair
    pair[0].lib.fake_set_capture_us(0)
    for f in pair:
        f.lib.tmac_shutdown(f.handle)


def test_no_synchronize_meets_a_capture(two):
    a, b = two
    met = a.lib.fake_syncs_in_capture()
    begun, stop, errors = [0], threading.Event(), []

    def capture():
        try:
            for _ in range(60):
                graph = ctypes.c_void_p()
                assert a.lib.tmac_step_begin(a.handle, 0x1000) == TMAC_OK
                assert a.lib.tmac_step_end(a.handle, 0x1000, ctypes.byref(graph)) == TMAC_OK
                assert a.lib.tmac_graph_destroy(a.handle, graph) == TMAC_OK
                begun[0] += 1
        except BaseException as e:  # reported below
            errors.append(e)
        finally:
            stop.set()

    def check():
        while not stop.is_set():
            if b.lib.tmac_check_device_error(b.handle) != TMAC_OK:
                errors.append("check_device_error")

    threads = [threading.Thread(target=capture), threading.Thread(target=check)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors and begun == [60]
    assert a.lib.fake_syncs_in_capture() == met
