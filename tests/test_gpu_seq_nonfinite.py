"""A NaN or an infinity among a sequence's own keys and queries, in packed and
paged attention, with the keys in one piece and in several that are joined:
what the formula makes NaN comes out as NaN, in the result and in the
log-sum-exp, and nothing else changes.

A score of NaN or +inf makes its row NaN (inf - inf); one of -inf has weight
0. The other rows keep the bounds of the finite case: their scores, and so the
terms of the bound, are those of the finite keys.
"""

import math

import pytest
import torch

from test_gpu_seq_attention import BF16, F16, packed_case, paged_case, spread
from transformer_optimization_b200 import _abi, kernels as K

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _abi.device_status() == 0


def check(q, k, v, scale, causal, out, lse):
    """One sequence against 64 bits; returns how many rows are NaN and how many are not."""
    (nq, h, hd), (nk, g, _) = q.shape, k.shape
    u = torch.finfo(q.dtype).eps / 2
    hidden = torch.arange(nk, device=q.device)[None] > torch.arange(nq, device=q.device)[:, None] + (nk - nq)
    lost = kept = 0
    for i in range(h):
        qi, ki, vi = q[:, i].double(), k[:, i // (h // g)].double(), v[:, i // (h // g)].double()
        s = (qi[:, None] * ki[None]).sum(-1) * scale
        if causal:
            s = s.masked_fill(hidden, -INF)
        bad = (s.isnan() | (s == INF)).any(1)
        assert out[bad, i].isnan().all() and lse[i, bad].isnan().all()
        lost, kept = lost + int(bad.sum()), kept + int((~bad).sum())
        none = (s == -INF).all(1)  # a query without keys
        assert not out[none, i].any() and (lse[i, none] == -INF).all()
        fine = ~bad & ~none
        s, qi = s[fine], qi[fine]
        if s.shape[0] == 0:
            continue
        mag = (qi.abs() @ ki.abs().nan_to_num(0, posinf=0).T).amax(1) * scale
        top = s.abs().masked_fill(s == -INF, 0).amax(1)
        d = (hd * 2.0 ** -23 * mag + 2.0 ** -22 * (1 + top))[:, None]
        rl = torch.logsumexp(s, 1)
        p = torch.exp(s - rl[:, None])
        want, a = p @ vi, p @ vi.abs()
        bound = u * want.abs() + (u + 2 * d + nk * 2.0 ** -23) * a + nk * 2.0 ** -25 * vi.abs().amax()
        assert ((out[fine, i].double() - want).abs() <= bound).all()
        assert ((lse[i, fine].double() - rl).abs() <= d[:, 0] + nk * 2.0 ** -23 + 2.0 ** -22 * rl.abs() + 2.0 ** -20).all()
    return lost, kept


def plant(kind, q, k):
    """In place: one element of one key (of key head 0) or of one query."""
    if kind == "nan query":
        q[q.shape[0] // 2, 0, 5] = NAN
    else:
        k[k.shape[0] // 3, 0, 3] = NAN if kind == "nan key" else INF


def slices(lens):
    at = 0
    for n in lens:
        yield slice(at, at + n)
        at += n


KINDS = ["nan key", "inf key", "nan query"]
LONG = [  # q_lens, k_lens, heads, kv_heads, the sequence that gets it
    ([40], [300], 4, 2, 0),  # one key range
    ([40], [6000], 4, 2, 0),  # few items: keys split
    (spread(60, 20, 500, 1), spread(60, 30, 700, 2), 8, 4, 3),  # listed items
    ([3] * 30 + [5], [100] * 30 + [9000], 16, 8, 30),  # a long one cut into key ranges
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hd,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("q_lens,k_lens,h,g,at", LONG)
def test_packed_nonfinite(q_lens, k_lens, h, g, at, hd, dtype, causal, kind):
    q, k, v, cu_q, cu_k = packed_case(q_lens, k_lens, h, g, hd, dtype)
    parts = list(zip(slices(q_lens), slices(k_lens)))
    plant(kind, q[parts[at][0]], k[parts[at][1]])
    for out_dtype in (dtype, torch.float32):
        out, lse = K.flash_attention_packed(q, k, v, cu_q, cu_k, max(q_lens), hd ** -0.5, max_k=max(k_lens), causal=causal,
                                            out_dtype=out_dtype, want_lse=True)
        for i, (a, b) in enumerate(parts):
            if i == at or i % 7 == 0:
                lost, kept = check(q[a], k[b], v[b], hd ** -0.5, causal, out[a], lse[:, a])
                assert kept > 0 and (lost > 0) == (i == at) or kind == "inf key" and lost == 0  # (every score -inf)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("q_lens,k_lens,h,g,at", LONG)
def test_paged_nonfinite(q_lens, k_lens, h, g, at, hd, dtype, kind):
    paged_nonfinite(q_lens, k_lens, h, g, at, hd, dtype, kind, max(max(q_lens), 17))


DECODE = [  # at most 16 rows to a key head
    ([1, 1, 1], [40, 9000, 700], 8, 2, 1), ([1, 1, 1], [40, 9000, 700], 8, 2, 0), ([4, 1, 3], [50, 20, 3000], 8, 2, 2),
    ([1] * 120, [1 + 53 * i % 900 for i in range(120)], 16, 4, 77), ([2, 1] * 150, [11 * i % 257 + 2 for i in range(300)], 16, 2, 10),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("q_lens,k_lens,h,g,at", DECODE)
def test_decode_nonfinite(q_lens, k_lens, h, g, at, hd, dtype, kind):
    paged_nonfinite(q_lens, k_lens, h, g, at, hd, dtype, kind, max(q_lens))


def paged_nonfinite(q_lens, k_lens, h, g, at, hd, dtype, kind, max_q):
    page = 16
    q, kc, vc, table, cu, lens, rows = paged_case(q_lens, k_lens, h, g, hd, page, dtype, peak=1.0)
    parts = list(slices(q_lens))
    plant(kind, q[parts[at]], rows[at][0])
    j = torch.arange(k_lens[at], device="cuda")
    kc[table[at, j // page].long(), j % page] = rows[at][0]
    for out_dtype in (dtype, torch.float32):
        out, lse = K.flash_attention_paged(q, kc, vc, table, cu, lens, max_q, hd ** -0.5, max_kv=max(k_lens),
                                           out_dtype=out_dtype, want_lse=True)
        for i, (a, (k, v)) in enumerate(zip(parts, rows)):
            if i == at or i % 7 == 0:
                lost, kept = check(q[a], k, v, hd ** -0.5, True, out[a], lse[:, a])
                assert kept > 0 and (lost > 0) == (i == at) or kind == "inf key" and lost == 0  # (every score -inf)
