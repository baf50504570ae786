"""The forced cut of Muon's products (a tool of the tests) belongs to the thread that asks for it."""
import ctypes as C
import threading

from distributed_tensorflow_amd.ops import hip_backend as hb


def test_a_forced_cut_is_the_calling_threads_own():
    lib = hb.require()
    rows, cols = (C.c_int32 * 1)(1024), (C.c_int32 * 1)(1024)
    size = lambda: lib.dtf_muon_workspace(1, rows, cols)  # noqa: E731
    plain, seen = size(), []
    forced, look = threading.Event(), threading.Event()

    def other():
        lib.dtf_debug_set_muon_cut(256, 8)
        seen.append(size())
        forced.set()
        look.wait(20)

    t = threading.Thread(target=other)
    t.start()
    try:
        assert forced.wait(20)
        assert size() == plain
    finally:
        look.set()
        t.join()
    assert seen[0] > plain          # eight parts of k, their sums kept between two launches
