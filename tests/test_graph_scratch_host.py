"""rdna_graph_scratch_stats without a GPU."""
import ctypes

from tests.test_paged_host import lib  # noqa: F401


def test_stats_of_a_device_that_was_never_used(lib):  # noqa: F811
    nbytes, blocks = ctypes.c_uint64(7), ctypes.c_int64(7)
    assert lib.rdna_graph_scratch_stats(0, ctypes.byref(nbytes), ctypes.byref(blocks)) == 0
    assert (nbytes.value, blocks.value) == (0, 0)
    assert lib.rdna_graph_scratch_stats(0, None, ctypes.byref(blocks)) == -3
    assert lib.rdna_graph_scratch_stats(0, ctypes.byref(nbytes), None) == -3
    assert "null output pointer" in lib.rdna_get_error().decode()
