"""The library's workspaces where the GPU has no memory left: context.cc and attend_split.cc over a HIP runtime of host memory
(tests/cpp/lib/scratch_host.cc), so these tests need no GPU."""

from __future__ import annotations

import ctypes as C
import shutil
import threading
from pathlib import Path

import pytest

HOST_SO = Path(__file__).resolve().parent / "cpp" / "bin" / "libscratch_host.so"
OK, BAD_ALLOC, RUNTIME_ERROR, TEMP_ATTEND = 0, 4, 5, 7


@pytest.fixture
def host(tmp_path):
    """The library anew: a copy of the file has state of its own."""
    at = tmp_path / "libscratch_host.so"
    shutil.copy(HOST_SO, at)
    lib = C.CDLL(str(at))
    lib.scratch_host_refuse_from.argtypes = [C.c_size_t]
    lib.scratch_host_generation.restype = C.c_uint64
    lib.scratch_host_block.argtypes, lib.scratch_host_block.restype = [C.c_void_p], C.c_size_t
    return lib


def temp(host, size):
    out = C.c_void_p()
    return host.scratch_host_temp(TEMP_ATTEND, C.c_size_t(size), C.byref(out)), out.value


def workspace(host, size):
    out = C.c_void_p()
    return host.scratch_host_workspace(C.c_size_t(size), C.byref(out)), out.value


@pytest.mark.parametrize("get", [temp, workspace])
def test_a_workspace_that_cannot_grow_stays_as_it_was(host, get):
    rc, first = get(host, 1000)
    assert rc == OK and host.scratch_host_block(first) >= 1000
    generation = host.scratch_host_generation()
    host.scratch_host_refuse_from(1500)
    assert get(host, 5000)[0] == BAD_ALLOC
    for size in (1000, 10):  # what fits is served from memory that is there
        rc, again = get(host, size)
        assert rc == OK and again == first and host.scratch_host_block(again) >= size
    assert host.scratch_host_generation() == generation  # captured graphs still point to it
    host.scratch_host_refuse_from(1 << 62)
    rc, grown = get(host, 5000)
    assert rc == OK and host.scratch_host_block(grown) >= 5000 and host.scratch_host_generation() > generation


@pytest.mark.parametrize("get", [temp, workspace])
def test_a_first_workspace_that_there_is_no_memory_for(host, get):
    host.scratch_host_refuse_from(1)
    assert get(host, 1000)[0] == BAD_ALLOC
    assert get(host, 10)[0] == BAD_ALLOC
    host.scratch_host_refuse_from(1 << 62)
    rc, p = get(host, 10)
    assert rc == OK and host.scratch_host_block(p) >= 10


@pytest.mark.parametrize("get", [temp, workspace])
def test_a_failed_allocation_is_reported_once(host, get):
    """Kernel launches ask HIP for the thread's last error: a reported one may not be there any more."""
    host.scratch_host_refuse_from(1)
    assert get(host, 1000)[0] == BAD_ALLOC
    assert host.scratch_host_last_error() == 0


def test_a_failed_device_allocation_is_reported_once(host):
    out = (C.c_uint64 * 3)()
    host.scratch_host_refuse_from(1)
    assert host.accel_hip_allocate(C.c_size_t(1000), out) == BAD_ALLOC
    assert host.scratch_host_last_error() == 0


def split(host, most, heads=32, dim=128):
    count = C.c_int()
    return host.scratch_host_split(heads, dim, C.c_int64(most), C.byref(count)), count.value


def test_a_key_range_whose_parts_have_no_memory_stays_whole(host):
    assert split(host, 8) == (OK, 8)
    host.scratch_host_refuse_from(1)
    assert split(host, 4) == (OK, 4)  # room that is there
    assert split(host, 200) == (OK, 1)
    assert split(host, 8) == (OK, 8)
    assert host.scratch_host_last_error() == 0
    host.scratch_host_refuse_from(1 << 62)
    assert split(host, 200) == (OK, 200)


def test_a_graph_waits_for_the_parts_that_another_thread_uses(host):
    """A captured attention call writes its parts to the same memory: a replay may not come between another thread's
    two launches."""
    graph = C.c_void_p()
    assert host.scratch_host_hold_parts() == OK
    host.scratch_host_release_parts()
    assert host.accel_hip_capture_begin() == OK and host.accel_hip_capture_end(C.byref(graph)) == OK
    launched = []
    other = threading.Thread(target=lambda: launched.append(host.accel_hip_graph_launch(graph, 2)))
    assert host.scratch_host_hold_parts() == OK
    other.start()
    other.join(0.3)
    waited = not launched
    host.scratch_host_release_parts()
    other.join(10)
    assert waited and launched == [OK]
    assert host.accel_hip_graph_destroy(graph) == OK


def test_a_graph_is_refused_once_the_parts_moved(host):
    """Also where they move while the replay waits for them."""
    graph = C.c_void_p()
    assert split(host, 8) == (OK, 8)
    assert host.accel_hip_capture_begin() == OK and host.accel_hip_capture_end(C.byref(graph)) == OK
    assert host.accel_hip_graph_launch(graph, 1) == OK
    launched = []
    other = threading.Thread(target=lambda: launched.append(host.accel_hip_graph_launch(graph, 1)))
    assert host.scratch_host_hold_parts() == OK
    other.start()
    other.join(0.3)
    rc = temp(host, 1 << 24)[0]
    host.scratch_host_release_parts()
    other.join(10)
    assert rc == OK and launched == [RUNTIME_ERROR]
    assert host.accel_hip_graph_destroy(graph) == OK
