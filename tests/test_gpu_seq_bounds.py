"""Bounds of "any number": the largest 64-bit max_q, max_k and max_kv give what
bounds the size of the arrays give."""

import pytest
import torch

from test_gpu_seq_attention import BF16, F16, check_packed, check_paged, packed_case, paged_case
from transformer_optimization_b200 import _abi, kernels as K

pytestmark = pytest.mark.gpu

ANY = 2 ** 63 - 1


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _abi.device_status() == 0


@pytest.mark.parametrize("most", [ANY, ANY - 254, 2 ** 62, 2 ** 30 + 1])
@pytest.mark.parametrize("sizes", [(8, 2, 4, 2, 64), (4096, 300, 32, 8, 128), (40, 1, 8, 8, 64)])
def test_workspace_of_any_bound(sizes, most):
    """A workspace for any bound is that for the largest bound there is."""
    t, b, h, g, hd = sizes
    for fn in ("tf_flash_packed_workspace", "tf_flash_paged_workspace"):
        want = _abi.call_value(fn, t, b, h, g, hd, 2 ** 30, 2 ** 31 - 1)
        assert want > 0
        assert _abi.call_value(fn, t, b, h, g, hd, most, max(most, 2 ** 31)) == want


@pytest.mark.parametrize("most", [ANY, 2 ** 62])
@pytest.mark.parametrize("q_lens,k_lens,h,g", [([40, 0, 300], [50, 20, 2500], 8, 2), ([1], [700], 4, 1),
                                               ([500] * 30, [500] * 30, 8, 4)])
def test_packed_any_bound(q_lens, k_lens, h, g, most):
    q, k, v, cu_q, cu_k = packed_case(q_lens, k_lens, h, g, 64, F16)
    out, lse = K.flash_attention_packed(q, k, v, cu_q, cu_k, most, 0.125, max_k=most, causal=True, want_lse=True)
    check_packed(q, k, v, cu_q, cu_k, 0.125, True, out, lse)


@pytest.mark.parametrize("most", [ANY, 2 ** 62])
@pytest.mark.parametrize("q_lens,k_lens,h,g", [([40, 1, 300], [50, 900, 2500], 8, 2), ([1, 1], [700, 0], 4, 1),
                                               ([1] * 60, [100 + 9 * i for i in range(60)], 16, 4)])
def test_paged_any_bound(q_lens, k_lens, h, g, most):
    q, kc, vc, table, cu, lens, rows = paged_case(q_lens, k_lens, h, g, 128, 16, BF16)
    for max_q in (most, max(q_lens)):
        out, lse = K.flash_attention_paged(q, kc, vc, table, cu, lens, max_q, 0.1, max_kv=most, want_lse=True)
        check_paged(q, rows, q_lens, 0.1, True, out, lse)
