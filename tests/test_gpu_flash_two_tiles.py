"""The padded flash kernel, causal, where both query tiles of a CTA run and the
first ends a key block before the second, so that the second's products go on
while the first reads its result."""

import pytest
import torch

from test_gpu_seq_attention import check, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from transformer_optimization_b200 import _abi, kernels
    _abi.load()
    yield kernels
    assert _abi.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seq", [129, 256, 300, 1500])
def test_flash_unequal_tiles(K, seq, hd, dtype):
    """Against 64 bits, with the bounds of the packed kernel (the same
    arithmetic), and the same bits on every run; the keys grow along the
    sequence, so that O is rescaled at most blocks."""
    b, h = 3, 5
    g = torch.Generator().manual_seed(seq + hd)
    q = torch.randn(b, seq, h * hd, generator=g).to(dtype).cuda()
    k = (torch.randn(b, seq, h * hd, generator=g) * torch.linspace(0.1, 6, seq)[None, :, None]).to(dtype).cuda()
    v = torch.randn(b, seq, h * hd, generator=g).to(dtype).cuda()
    out, lse = K.flash_attention(q, k, v, h, hd ** -0.5, causal=True, want_lse=True)
    for i in range(b):
        qi, ki, vi = (x[i].view(seq, h, hd) for x in (q, k, v))
        check(out[i].view(seq, h, hd), lse[i], *reference(qi, ki, vi, hd ** -0.5, True, None, None))
    for _ in range(100):
        again, lse2 = K.flash_attention(q, k, v, h, hd ** -0.5, causal=True, want_lse=True)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


def test_flash_unequal_tiles_split_positions(K):
    """Key blocks at other positions than the queries' (a context-parallel
    rank): the first tile without keys, or with one block fewer."""
    h, hd, seq = 2, 128, 256
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, seq, h * hd, generator=g).half().cuda() for _ in range(3))
    qi, ki, vi = (x[0].view(seq, h, hd) for x in (q, k, v))
    for shift in (0, 100, 128, 200):  # the first key stands `shift` positions behind the first query
        out, lse = K.flash_attention(q, k, v, h, hd ** -0.5, causal=True, want_lse=True, k_pos0=shift)
        assert not out[0, :shift].any() and (lse[0, :, :shift] == -float("inf")).all()
        n = seq - shift  # queries from `shift` on see the first n keys, each up to its own position
        want = reference(qi[shift:], ki[:n], vi[:n], hd ** -0.5, True, None, None)
        check(out[0, shift:].view(n, h, hd), lse[0, :, shift:], *want)
