"""Sources that map files: never page-locked in place, whatever route is asked for (a window copies them); other memory is."""
import mmap
import os

import numpy as np
import pytest
import torch

import emel_cpp_b200 as eb
from emel_cpp_b200 import window as ew
from tests.test_gpu_layer_window import LAYERS, STREAMING_BUDGET, slot_content_matches, stream_image

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = eb.Backend(0)
    yield b
    b.close()


@pytest.mark.parametrize("how", ["path", "memmap", "anonymous", "array"])
def test_a_window_page_locks_memory_but_not_files(be, how, tmp_path):
    image, layers = stream_image()
    path = os.path.join(tmp_path, "window.bin")
    image.tofile(path)
    source = path if how == "path" else image
    if how == "memmap":
        source = np.memmap(path, dtype=np.uint8, mode="c")
    elif how == "anonymous":
        source = np.frombuffer(mmap.mmap(-1, image.nbytes, flags=mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS), dtype=np.uint8)
        source[:] = image
    win = ew.LayerWindow(be)
    try:
        assert win.bind(source, layers, STREAMING_BUDGET, 4, 2), win.last_error
        assert win.bound["source_page_locked"]
        if how != "path":
            first = np.asarray(source)[layers[0][0][1]:]          # the header in front of the layers stays as it is
            assert torch.frombuffer(first, dtype=torch.uint8).is_pinned() == (how != "memmap")
        for l in range(LAYERS):
            got = win.acquire(l)
            assert got is not None and slot_content_matches(be, got, l)
        assert win.unbind()
    finally:
        win.close()


@pytest.mark.parametrize("route", ["ring", "plain", "register"])
def test_uploads_of_a_mapped_file(be, route, tmp_path):
    """A span of a file's mapping, from a place inside of a page, right behind its writing."""
    data = np.random.default_rng(3).integers(0, 256, (9 << 20) + 77, dtype=np.uint8)
    path = os.path.join(tmp_path, "span.bin")
    data.tofile(path)
    span = np.memmap(path, dtype=np.uint8, mode="r")[1111:]
    assert be.set_upload_route(route)
    try:
        be.upload(5, span, tensor_type=24)
        got = np.empty(len(span), np.uint8)
        assert be.to_host(got, be.state(5).buffer, len(got)) and np.array_equal(got, span)
        be.evict(5)
    finally:
        assert be.set_upload_route("ring")
