"""Rotary positions of keys without queries: a head count of 0, with null
pointers and no strides for what is not there."""

import pytest
import torch

from transformer_optimization_b200 import _abi

# a tf_rotary call of 2 key heads of 64, 4 tokens, no query heads; addresses that are never read here
KEYS = [None, 0, 0, None, 0, 0, 64, 128, 64, 64, 128, 64, 64, 64, 4, 0, 2, 64, 32, 1.0, 0, None]


def test_keys_alone_pass_the_checks():
    """On a host without a device the checks are passed and the device is what is missing."""
    if torch.cuda.is_available():
        pytest.skip("would launch")
    lib = _abi.load()
    assert lib.tf_rotary(*KEYS) not in (0, 1, 2), lib.tf_last_error()
    assert b"overlap" not in lib.tf_last_error()
    bad = list(KEYS)
    bad[10] = 64  # the keys' own rows still have to lie apart
    assert lib.tf_rotary(*bad) == 1 and b"overlap" in lib.tf_last_error()
    bad = list(KEYS)
    bad[16] = 0  # neither queries nor keys
    assert lib.tf_rotary(*bad) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [0, 1])
def test_keys_alone(interleaved):
    from transformer_optimization_b200 import kernels as K
    lib = _abi.load()
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(37, 3, 64, generator=gen).half().cuda() for _ in range(2))
    pos = torch.arange(37, device="cuda") * 11
    freqs, _ = K.rotary_freqs(48, device="cuda")
    _, want = K.rotary(k, k, pos, freqs, interleaved=bool(interleaved))
    got = torch.empty_like(k)
    stream = torch.cuda.current_stream().cuda_stream
    rc = lib.tf_rotary(None, 0, 0, None, 0, 0, k.data_ptr(), 192, 64, got.data_ptr(), 192, 64, pos.data_ptr(),
                       freqs.data_ptr(), 37, 0, 3, 64, 48, 1.0, interleaved, stream)
    assert rc == 0, lib.tf_last_error()
    assert torch.equal(got, want)
    kc, vc = (torch.zeros(3, 16, 3, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    slots = torch.arange(37, device="cuda")
    rc = lib.tf_rotary_append(None, 0, 0, None, 0, 0, k.data_ptr(), 192, 64, v.data_ptr(), 192, 64, pos.data_ptr(),
                              freqs.data_ptr(), kc.data_ptr(), vc.data_ptr(), 16 * 192, 192, 64, 3, 16, slots.data_ptr(),
                              37, 0, 3, 64, 48, 1.0, interleaved, stream)
    assert rc == 0, lib.tf_last_error()
    assert torch.equal(kc.flatten(0, 1)[:37], want) and torch.equal(vc.flatten(0, 1)[:37], v)
    none = k[:, :0]  # and through the wrapper
    q2, k2 = K.rotary(none, k, pos, freqs, interleaved=bool(interleaved))
    assert q2.shape == (37, 0, 64) and torch.equal(k2, want)
    assert _abi.device_status() == 0
