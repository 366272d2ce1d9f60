"""Uploads that wait for the device longer than the context's limit: an error on the host, in time, and a context that goes on."""
import time

import numpy as np
import pytest
import torch

import emel_cpp_b200 as eb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("route,pinned", [("plain", True), ("register", False), ("ring", True)])
def test_upload_behind_a_busy_stream_ends_at_the_limit(route, pinned):
    be = eb.Backend(0)
    rng = np.random.default_rng(2)
    host = torch.from_numpy(rng.integers(0, 256, 6 << 20, dtype=np.uint8))
    host = host.pin_memory() if pinned else host
    try:
        be.upload(1, host.numpy(), tensor_type=24)                # first of all without anything in front
        assert be.set_upload_route(route) and be.set_upload_wait_ms(60) and not be.set_upload_wait_ms(0)
        with torch.cuda.stream(torch.cuda.ExternalStream(be.stream())):
            torch.cuda._sleep(int(1.2e9))                         # 0.6 s of the context's stream
        t0 = time.perf_counter()
        with pytest.raises(eb.BackendError):
            be.upload(2, host.numpy(), tensor_type=24)
        assert time.perf_counter() - t0 < 2.0 and be.last_error == eb.INTERNAL_ERROR
        assert eb.LIFECYCLE[be.state(2).lifecycle_state] != "resident"
        assert be.sync()
        assert be.set_upload_wait_ms(60000)
        be.upload(3, host.numpy(), tensor_type=24)
        for t in (1, 3):
            got = np.empty(host.numel(), np.uint8)
            assert be.to_host(got, be.state(t).buffer, len(got)) and np.array_equal(got, host.numpy())
    finally:
        be.close()
