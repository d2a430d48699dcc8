"""A bad index (device code 108) is a report on one call's arguments: until the
host reads it, the kernels that follow run as ever, their waits included, and
an error of theirs is reported in its place."""

import pytest
import torch

from transformer_optimization_b200 import _abi, kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    assert _abi.device_status() == 0
    yield
    _abi.device_status()


def report_bad_slot():
    x = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    cache = torch.zeros(1, 16, 1, 64, dtype=torch.float16, device="cuda")
    freqs, _ = K.rotary_freqs(64, device="cuda")
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    K.rotary_append(x, x, x, zero, freqs, cache, cache.clone(), zero + 16)


@pytest.mark.parametrize("m,k,n", [(16384, 1024, 1024), (1000, 4096, 1024)])
def test_overlapped_pair_behind_a_bad_index(m, k, n):
    """The LayerNorm that waits for a GEMM's rows waits for them all the same."""
    g = torch.Generator().manual_seed(m)
    a = (torch.randn(m, k, generator=g) * 0.5).half().cuda()
    w = (torch.randn(n, k, generator=g) * k ** -0.5).half().cuda()
    bias, lnw, lnb = (torch.randn(n, generator=g).cuda() for _ in range(3))
    x = torch.randn(m, n, generator=g).cuda()
    want_x = K.linear_residual(a, w, bias, x, None)
    want = K.ln_residual(want_x, None, lnw, lnb, 1e-5)[1]
    ready = K.ready_counters(m, x.device)
    got_x = [torch.empty_like(want_x) for _ in range(5)]
    normed = [torch.zeros_like(want) for _ in range(5)]
    graph = torch.cuda.CUDAGraph()  # as the models run it: no gap between the two
    with torch.cuda.graph(graph):
        for y, z in zip(got_x, normed):
            K.linear_residual(a, w, bias, x, y, ready=ready)
            K.ln_ready(y, lnw, lnb, 1e-5, ready, normed=z)
    report_bad_slot()
    for _ in range(3):
        for t in got_x + normed:
            t.zero_()
        graph.replay()
        assert all(torch.equal(y, want_x) for y in got_x)
        assert all(torch.equal(z, want) for z in normed)
        assert not ready.any()
    assert _abi.device_status() == 108


def test_wait_runs_out_behind_a_bad_index():
    """A wait lasts its whole time, and its code takes the place of the index error."""
    src = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    report_bad_slot()
    start.record()
    out = K.wait_timeout_probe(src, 20_000_000)
    end.record()
    torch.cuda.synchronize()
    assert out.tolist()[:2] == [1, 1]
    assert start.elapsed_time(end) >= 20.0
    assert _abi.device_status() == 106 and _abi.device_status() == 0


def test_index_error_behind_a_wait():
    """The other way round the wait's code stays."""
    K.wait_timeout_probe(torch.zeros(4096, dtype=torch.uint8, device="cuda"), 20_000)
    report_bad_slot()
    assert _abi.device_status() == 106


def test_status_message_says_what_it_was():
    report_bad_slot()
    assert _abi.device_status() == 108
    message = _abi.load().tf_last_error().decode()
    assert "index" in message and "108" in message and "wait" not in message
