"""Packed and paged attention on a B200, against softmax attention in 64 bits.

Tolerance. With u = eps / 2 of the 16-bit type, A_i = sum_j p_j |v_j| and n
keys, a result is off by at most
  u |out|              its rounding
  u A                  the rounding of each probability for the second product
  n 2^-25 max|v|       fp16 probabilities below 2^-14 (absolute step 2^-24; the
                       reference maximum's own key contributes 1 to the sum)
  (2 d + n 2^-23) A    d: error of a score, hd fp32 additions of the products
                       (2^-23 each, which allows a truncating adder), 2^-22 for
                       exp2 and the shift; n fp32 additions of the second product
and the log-sum-exp by d + n 2^-23 + 2^-22 |lse| + 2^-20.
Joining key ranges adds one fp32 rounding per range, inside the n 2^-23.
"""

import math

import pytest
import torch

from transformer_optimization_b200 import _abi, kernels as K

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def no_device_error(request):
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        assert _abi.device_status() == 0


def reference(q, k, v, scale, causal, out, lse):
    """One sequence in 64 bits: results and their tolerances."""
    (nq, h, hd), (nk, g, _) = q.shape, k.shape
    res = torch.zeros(nq, h, hd, dtype=torch.float64, device=q.device)
    rl = torch.full((h, nq), -math.inf, dtype=torch.float64, device=q.device)
    bound, bl = torch.zeros_like(res), torch.zeros_like(rl)
    u = torch.finfo(q.dtype).eps / 2
    if nk == 0 or nq == 0:
        return res, rl, bound, bl
    kd, vd = k.double(), v.double()
    admit = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (nk - nq)
    for i in range(h):
        qi, ki, vi = q[:, i].double(), kd[:, i // (h // g)], vd[:, i // (h // g)]
        s = qi @ ki.T * scale
        d = (hd * 2.0 ** -23 * (qi.abs() @ ki.abs().T).amax(1) * scale + 2.0 ** -22 * (1 + s.abs().amax(1)))[:, None]
        if causal:
            s = s.masked_fill(~admit, -math.inf)
        rl[i] = torch.logsumexp(s, 1)
        p = torch.nan_to_num(torch.exp(s - rl[i][:, None]))
        res[:, i] = p @ vi
        a = p @ vi.abs()
        bound[:, i] = u * res[:, i].abs() + (u + 2 * d + nk * 2.0 ** -23) * a + nk * 2.0 ** -25 * vi.abs().amax()
        bl[i] = d[:, 0] + nk * 2.0 ** -23 + 2.0 ** -22 * rl[i].abs().nan_to_num(posinf=0) + 2.0 ** -20
    return res, rl, bound, bl


def check(got, lse, want, want_lse, bound, bl):
    got = got.double()
    assert bool(got.isfinite().all())
    off = (got - want).abs()
    over = off > bound
    at = over.nonzero()
    assert at.numel() == 0, f"{len(at)} of {off.numel()} off, first {at[0].tolist()}, by {(off - bound).max():.3g}"
    if lse is not None:
        none = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        assert ((lse.double() - want_lse).abs()[~none] <= bl[~none]).all()


def offsets(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)


def packed_case(q_lens, k_lens, h, g, hd, dtype, seed=0, peak=1.0):
    gen = torch.Generator().manual_seed(seed + sum(q_lens) + 7 * sum(k_lens) + h)
    q = (torch.randn(sum(q_lens), h, hd, generator=gen) * peak).to(dtype).cuda()
    kv = torch.randn(sum(k_lens), 2 * g, hd, generator=gen).to(dtype).cuda()
    return q, kv[:, :g], kv[:, g:], offsets(q_lens).cuda(), offsets(k_lens).cuda()


def check_packed(q, k, v, cu_q, cu_k, scale, causal, out, lse):
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cq) - 1):
        rq, rk = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        check(out[rq], None if lse is None else lse[:, rq], *reference(q[rq], k[rk], v[rk], scale, causal, out, lse))


PACKED = [  # q_lens, k_lens (None: the same), heads, kv_heads, hd, causal
    ([1], None, 1, 1, 64, True), ([2, 1, 3], None, 4, 2, 64, False), ([127, 128, 129], None, 2, 2, 64, True),
    ([255, 0, 257, 1], None, 4, 1, 128, True), ([64, 65, 63, 300], None, 8, 2, 64, True),
    ([33, 500], None, 3, 1, 128, False), ([1, 700, 31], None, 5, 1, 64, True), ([130] * 40, None, 2, 1, 64, True),
    ([17, 3], [0, 200], 4, 4, 64, False), ([17, 3, 40], [0, 200, 39], 4, 4, 128, True),  # queries without keys
    ([5, 90, 1], [700, 1000, 129], 7, 1, 64, True), ([300], [10], 4, 2, 64, True), ([1, 1], [3000, 1], 16, 2, 128, True),
    ([20], [2500], 128, 1, 64, True), ([9], [5000], 6, 2, 128, False), ([1500], None, 2, 2, 128, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_lens,k_lens,h,g,hd,causal", PACKED)
def test_packed(q_lens, k_lens, h, g, hd, causal, dtype):
    k_lens = q_lens if k_lens is None else k_lens
    q, k, v, cu_q, cu_k = packed_case(q_lens, k_lens, h, g, hd, dtype, peak=3.0)
    out, lse = K.flash_attention_packed(q, k, v, cu_q, cu_k, max(q_lens), hd ** -0.5, causal=causal, want_lse=True,
                                        max_k=max(k_lens))
    assert out.dtype == dtype and lse.shape == (h, sum(q_lens))
    check_packed(q, k, v, cu_q, cu_k, hd ** -0.5, causal, out, lse)
    # fp32 results are those rounded; loose bounds change the grid and the split, not the answer
    out32, none = K.flash_attention_packed(q, k, v, cu_q, cu_k, sum(q_lens), hd ** -0.5, causal=causal,
                                           out_dtype=torch.float32)
    assert none is None and out32.dtype == torch.float32
    check_packed(q, k, v, cu_q, cu_k, hd ** -0.5, causal, out32, None)


def spread(n, lo, hi, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi, (n,), generator=gen).tolist()


LISTED = [  # more items than SMs: listed tiles, the last with long keys cut into ranges
    (spread(60, 1, 700, 1), None, 8, 4, 64, True), (spread(70, 0, 300, 2), spread(70, 0, 500, 3), 12, 4, 128, False),
    ([40, 3000, 500, 2900], [3500, 3000, 2600, 4000], 16, 4, 64, True),
    ([900, 1, 1, 1, 700], [2500, 5000, 4000, 17, 3000], 24, 8, 128, True),
    ([1000, 0, 600], [4100, 3, 6000], 10, 5, 64, False), (spread(1100, 0, 71, 4), None, 8, 1, 64, True),
    (spread(1300, 1, 4, 5), spread(1300, 0, 300, 6), 4, 4, 64, True),
    ([2500, 2400], None, 16, 16, 64, True),  # asks for more ranges than there are places for
]


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,k_lens,h,g,hd,causal", LISTED)
def test_packed_listed(q_lens, k_lens, h, g, hd, causal):
    k_lens = q_lens if k_lens is None else k_lens
    q, k, v, cu_q, cu_k = packed_case(q_lens, k_lens, h, g, hd, BF16, peak=2.0)
    args = (q, k, v, cu_q, cu_k, max(q_lens), hd ** -0.5)
    out, lse = K.flash_attention_packed(*args, causal=causal, want_lse=True, max_k=max(k_lens))
    check_packed(q, k, v, cu_q, cu_k, hd ** -0.5, causal, out, lse)
    for _ in range(10):  # the draw of items depends on timing, results do not
        again, lse2 = K.flash_attention_packed(*args, causal=causal, want_lse=True, max_k=max(k_lens))
        assert torch.equal(again, out) and torch.equal(lse2, lse)


CUT = [  # more items than SMs, a few so long that their keys are cut into ranges
    ([3] * 30 + [5], [100] * 30 + [9000], 16, 8, 64), ([130, 40, 2, 7] * 11, [9001, 60, 300, 7] + [150] * 40, 12, 4, 128),
    ([300] * 6, [10000, 5, 300, 100, 8300, 0], 25, 25, 64), ([1, 2] * 600, [20, 1] * 599 + [12000, 6000], 4, 1, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens,k_lens,h,g,hd", CUT)
def test_long_among_short(q_lens, k_lens, h, g, hd, causal):
    q, k, v, cu_q, cu_k = packed_case(q_lens, k_lens, h, g, hd, F16, peak=2.0)
    args = (q, k, v, cu_q, cu_k, max(q_lens), hd ** -0.5)
    out, lse = K.flash_attention_packed(*args, causal=causal, want_lse=True, max_k=max(k_lens))
    check_packed(q, k, v, cu_q, cu_k, hd ** -0.5, causal, out, lse)
    for _ in range(3):
        again, lse2 = K.flash_attention_packed(*args, causal=causal, want_lse=True, max_k=max(k_lens))
        assert torch.equal(again, out) and torch.equal(lse2, lse)
    q, kc, vc, table, cu, lens, rows = paged_case(q_lens, k_lens, h, g, hd, 32, F16)
    out, lse = K.flash_attention_paged(q, kc, vc, table, cu, lens, max(max(q_lens), 17), hd ** -0.5, causal=causal,
                                       want_lse=True, max_kv=max(k_lens))
    check_paged(q, rows, q_lens, hd ** -0.5, causal, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_rows_outside_and_other_sequences(hd, causal):
    """Tokens before the first and behind the last sequence are left as they
    were; what other sequences and unused tokens hold never reaches a result."""
    q, k, v, _, _ = packed_case([400], [600], 4, 2, hd, F16)
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([7, 140, 311], [50, 190, 470]))
    want, wl = K.flash_attention_packed(q, k, v, cu_q, cu_k, 200, 0.1, causal=causal, want_lse=True, max_k=280)
    bad_q, bad_k, bad_v = q.clone(), k.clone(), v.clone()
    for t, keep in ((bad_q, (7, 140)), (bad_k, (50, 190)), (bad_v, (50, 190))):
        t[:keep[0]] = float("nan")
        t[keep[1]:] = float("inf")
    out = torch.full_like(want, 7.0)
    lse = torch.full_like(wl, 9.0)
    one_q, one_k = (torch.stack([c[0], c[1]]) for c in (cu_q, cu_k))
    K.flash_attention_packed(bad_q, bad_k, bad_v, one_q, one_k, 133, 0.1, causal=causal, out=out, lse=lse, max_k=280)
    assert torch.equal(out[7:140], want[7:140]) and torch.equal(lse[:, 7:140], wl[:, 7:140])
    assert (out[:7] == 7).all() and (out[140:] == 7).all()
    assert (lse[:, :7] == 9).all() and (lse[:, 140:] == 9).all()


@pytest.mark.gpu
def test_packed_split_rows_outside():
    """The same where the keys are split and joined."""
    q, k, v, _, _ = packed_case([40], [6000], 4, 2, 64, BF16)
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3, 20, 20], [100, 5900, 5900]))
    out, lse = torch.full_like(q, 7.0), torch.full((4, 40), 9.0, device="cuda")
    K.flash_attention_packed(q, k, v, cu_q, cu_k, 17, 0.1, out=out, lse=lse, causal=True)
    check_packed(q, k, v, cu_q, cu_k, 0.1, True, out, lse)
    assert (out[:3] == 7).all() and (out[20:] == 7).all() and (lse[:, :3] == 9).all() and (lse[:, 20:] == 9).all()


@pytest.mark.gpu
def test_packed_equals_padded_kernel():
    """One full-length sequence per batch entry: the padded kernel's bits."""
    b, s, h, hd = 2, 384, 4, 64
    q, k, v, cu, _ = packed_case([s] * b, [s] * b, h, h, hd, F16)
    out, lse = K.flash_attention_packed(q, k, v, cu, cu, s, hd ** -0.5, causal=True, want_lse=True)
    flat = [x.reshape(b, s, h * hd).contiguous() for x in (q, k, v)]
    ref, ref_lse = K.flash_attention(*flat, h, hd ** -0.5, causal=True, want_lse=True)
    assert torch.equal(out.view(b, s, h * hd), ref)
    assert torch.equal(lse.view(h, b, s).transpose(0, 1), ref_lse)


@pytest.mark.gpu
def test_packed_key_ranges_merge():
    """fp32 results over two halves of the keys, merged by attn_merge."""
    q, k, v, cu_q, _ = packed_case([70, 5], [600, 600], 4, 2, 64, F16)
    parts = []
    for r in (slice(0, 250), slice(250, 600)):
        n = r.stop - r.start
        kk, vv = (torch.cat([x[r], x[600:][r]]) for x in (k, v))
        cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        parts.append(K.flash_attention_packed(q, kk, vv, cu_q, cu, 70, 0.125, out_dtype=torch.float32, want_lse=True))
    (o, l), (o2, l2) = parts
    K.attn_merge(o.view(1, 75, 256), l[None], o2.view(1, 75, 256), l2[None], 4)
    cu = torch.tensor([0, 600, 1200], dtype=torch.int32, device="cuda")
    check_packed(q, k, v, cu_q, cu, 0.125, False, o, l)


# ----------------------------------------------------------------- paged
def paged_case(q_lens, kv_lens, h, g, hd, page, dtype, swapped=False, peak=3.0, fill=float("nan")):
    """Caches whose unused rows and pages hold `fill`, and a table whose unused entries are out of range."""
    gen = torch.Generator().manual_seed(sum(q_lens) + 3 * sum(kv_lens) + page + h)
    q = (torch.randn(sum(q_lens), h, hd, generator=gen) * peak).to(dtype).cuda()
    need = [-(-n // page) for n in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(kv_lens), max(need + [0]) + 2), -7, dtype=torch.int32)
    shape = (pages, g, page, hd) if swapped else (pages, page, g, hd)
    kc, vc = (torch.full(shape, fill, dtype=dtype, device="cuda") for _ in range(2))
    if swapped:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    rows, at = [], 0
    for b, n in enumerate(kv_lens):
        table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        k, v = (torch.randn(n, g, hd, generator=gen).to(dtype).cuda() for _ in range(2))
        j = torch.arange(n)
        where = table[b, j // page].long()
        kc[where, j % page], vc[where, j % page] = k, v
        rows.append((k, v))
    return q, kc, vc, table.cuda(), offsets(q_lens).cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), rows


def check_paged(q, rows, q_lens, scale, causal, out, lse):
    at = 0
    for n, (k, v) in zip(q_lens, rows):
        r = slice(at, at + n)
        check(out[r], None if lse is None else lse[:, r], *reference(q[r], k, v, scale, causal, out, lse))
        at += n


PAGED = [  # q_lens, kv_lens, heads, kv_heads, hd, page
    ([1], [1], 1, 1, 64, 16), ([1, 1, 1], [15, 16, 17], 8, 2, 64, 16), ([1] * 5, [63, 64, 65, 0, 1000], 16, 4, 128, 32),
    ([1] * 70, list(range(1, 71)), 4, 1, 64, 16), ([1, 0, 1], [300, 50, 2000], 14, 2, 128, 64),
    ([2, 3, 1, 4], [2, 300, 1, 77], 4, 1, 64, 16), ([4, 1], [3, 900], 12, 4, 128, 128),  # a token without keys
    ([1, 1], [20000, 3], 3, 3, 64, 256), ([1], [9000], 16, 1, 128, 16), ([16], [500], 3, 3, 64, 16),
    ([40, 1, 300], [40, 700, 1000], 8, 2, 64, 16), ([129, 5], [640, 5], 4, 4, 128, 32),
    ([17, 1, 1, 64], [17, 129, 5000, 200], 5, 1, 64, 64), ([300, 2], [300, 100], 14, 2, 128, 128),
    ([33, 20], [32, 4000], 8, 8, 128, 512), ([1] * 30 + [300, 170], [1 + 61 * i for i in range(30)] + [2000, 4000], 32, 8, 64, 32), ([5], [7000], 32, 4, 64, 16), ([200, 0, 1], [0, 0, 333], 6, 2, 64, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,kv_lens,h,g,hd,page", PAGED)
def test_paged(q_lens, kv_lens, h, g, hd, page, causal, dtype):
    q, kc, vc, table, cu, lens, rows = paged_case(q_lens, kv_lens, h, g, hd, page, dtype, swapped=h % 3 == 0)
    out, lse = K.flash_attention_paged(q, kc, vc, table, cu, lens, max(q_lens), hd ** -0.5, causal=causal,
                                       want_lse=True, max_kv=max(kv_lens))
    check_paged(q, rows, q_lens, hd ** -0.5, causal, out, lse)
    # looser bounds take another kernel, grid or split; the answer stays
    out32, _ = K.flash_attention_paged(q, kc, vc, table, cu, lens, max(max(q_lens), 17), hd ** -0.5, causal=causal,
                                       out_dtype=torch.float32)
    check_paged(q, rows, q_lens, hd ** -0.5, causal, out32, None)


MANY = [  # more (sequence, key head, row)s than blocks of the join fit on the card
    ([1] * 120, [1 + 53 * i % 900 for i in range(120)], 16, 4, 128), ([1, 0, 1] * 50, [7 * i % 300 for i in range(150)], 16, 4, 64),
    ([2, 1] * 150, [11 * i % 257 for i in range(300)], 16, 2, 64), ([3] * 150, [5 + 2 * i for i in range(150)], 20, 4, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens,h,g,hd", MANY)
def test_paged_many_sequences(q_lens, kv_lens, h, g, hd):
    q, kc, vc, table, cu, lens, rows = paged_case(q_lens, kv_lens, h, g, hd, 16, BF16)
    args = (q, kc, vc, table, cu, lens, max(q_lens), hd ** -0.5)
    out, lse = K.flash_attention_paged(*args, want_lse=True, max_kv=max(kv_lens))
    check_paged(q, rows, q_lens, hd ** -0.5, True, out, lse)
    again, lse2 = K.flash_attention_paged(*args, want_lse=True, max_kv=max(kv_lens))
    assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 100])
def test_paged_rows_outside(max_q):
    q, kc, vc, table, _, lens, rows = paged_case([1, 1, 1], [100, 3000, 0], 4, 2, 64, 16, F16)
    wide = torch.zeros(9, 4, 64, dtype=F16, device="cuda")
    wide[4:7] = q
    out, lse = torch.full_like(wide, 7.0), torch.full((4, 9), 9.0, device="cuda")
    cu = torch.tensor([4, 5, 6, 7], dtype=torch.int32, device="cuda")
    K.flash_attention_paged(wide, kc, vc, table, cu, lens, max_q, 0.125, out=out, lse=lse)
    check_paged(q, rows, [1, 1, 1], 0.125, True, out[4:7], lse[:, 4:7])
    for t in (out[:4], out[7:]):
        assert (t == 7).all()
    assert (lse[:, :4] == 9).all() and (lse[:, 7:] == 9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 100])
def test_paged_bad_indices_are_reported(max_q):
    """A page outside the cache reads as zeros, lengths are cut to the arrays;
    both set the device status and leave other sequences alone."""
    q, kc, vc, table, cu, lens, rows = paged_case([1, 1], [100, 200], 4, 2, 64, 16, F16)
    want, _ = K.flash_attention_paged(q, kc, vc, table, cu, lens, max_q, 0.125)
    for bad in (-1, kc.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 2] = bad
        out, _ = K.flash_attention_paged(q, kc, vc, t, cu, lens, max_q, 0.125)
        assert _abi.device_status() == 108
        k, v = (x.clone() for x in rows[0])
        k[32:48] = v[32:48] = 0
        check_paged(q, [(k, v), rows[1]], [1, 1], 0.125, True, out, None)
        assert torch.equal(out[1], want[1])
    for bad in ([-5, 200], [100, 10 ** 6]):
        n = torch.tensor(bad, dtype=torch.int32, device="cuda")
        t = table.clamp(0, kc.shape[0] - 1)
        out, _ = K.flash_attention_paged(q, kc, vc, t, cu, n, max_q, 0.125)
        assert _abi.device_status() == 108
        i = 0 if bad[0] == 100 else 1
        check_paged(q[i:i + 1], rows[i:i + 1], [1], 0.125, True, out[i:i + 1], None)
    for bad in ([-3, 1, 2], [0, 1, 9], [1, 0, 2], [0, 0, 200000]):
        c = torch.tensor(bad, dtype=torch.int32, device="cuda")
        K.flash_attention_paged(q, kc, vc, table, c, lens, max_q, 0.125)
        assert _abi.device_status() == 108


@pytest.mark.gpu
def test_packed_bad_offsets_are_reported():
    q, k, v, cu, _ = packed_case([100, 60], [100, 60], 4, 2, 64, F16)
    want, _ = K.flash_attention_packed(q, k, v, cu, cu, 100, 0.125)
    for bad_q, bad_k, max_q in (([0, 100, 161], cu, 100), (cu, [0, 100, 161], 100), ([-9, 100, 160], cu, 110),
                                (cu, [-1, 100, 160], 100), (cu, [0, 100, 90], 100), (cu, cu, 99),
                                (cu, [2 ** 31 - 1, 100, 160], 100)):
        c, d = (torch.tensor(x, dtype=torch.int32, device="cuda") if isinstance(x, list) else x for x in (bad_q, bad_k))
        K.flash_attention_packed(q, k, v, c, d, max_q, 0.125)
        assert _abi.device_status() == 108
    out, _ = K.flash_attention_packed(q, k, v, cu, cu, 100, 0.125)
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_sequences_over_one_another_are_reported():
    """More tiles than the tokens can hold, with a list, and with tiles cut into key ranges: reported, and in bounds."""
    k_lens = [9000] + [100] * 79
    q, k, v, _, cu_k = packed_case([2000], k_lens, 2, 2, 64, F16)
    cu_q = torch.tensor([0, 2000] * 40 + [0], dtype=torch.int32, device="cuda")
    for max_k in (1000, 9000):
        args = (q, k, v, cu_q, cu_k, 2000, 0.125)
        need = _abi.call_value("tf_flash_packed_workspace", 2000, 80, 2, 2, 64, 2000, max_k)
        space = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
        K.flash_attention_packed(*args, max_k=max_k, workspace=space[:need])
        assert _abi.device_status() == 108
        assert (space[need:] == 0x5a).all()
    again = torch.tensor([0, 2000], dtype=torch.int32, device="cuda"), torch.tensor([0, 9000], dtype=torch.int32, device="cuda")
    out, lse = K.flash_attention_packed(q, k[:9000], v[:9000], *again, 2000, 0.125, want_lse=True, max_k=9000)
    check_packed(q, k[:9000], v[:9000], *again, 0.125, False, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 64])
def test_paged_past_32_bits(max_q):
    """A cache whose pages start past 2^31 elements."""
    pages, page, g, hd = 2 ** 31 // (256 * 8 * 128) + 40, 256, 8, 128
    kc, vc = (torch.empty(pages, page, g, hd, dtype=BF16, device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(3)
    ids = [pages - 1, 0, pages - 20]
    k, v = (torch.randn(700, g, hd, generator=gen).to(BF16).cuda() for _ in range(2))
    pad = torch.zeros(768 - 700, g, hd, dtype=BF16, device="cuda")
    for c, x in ((kc, k), (vc, v)):
        c[ids] = torch.cat([x, pad]).view(3, page, g, hd)
    q = torch.randn(1, 16, hd, generator=gen).to(BF16).cuda()
    t = torch.tensor([ids], dtype=torch.int32, device="cuda")
    cu, n = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [700]))
    out, lse = K.flash_attention_paged(q, kc, vc, t, cu, n, max_q, hd ** -0.5, want_lse=True)
    check_paged(q, [(k, v)], [1], hd ** -0.5, True, out, lse)
    # and written there: the last row of the last page
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    freqs, _ = K.rotary_freqs(hd, device="cuda")
    K.rotary_append(q, k[:1], v[:1], pos, freqs, kc, vc, torch.tensor([pages * page - 1], device="cuda"))
    assert torch.equal(kc[-1, -1], k[0]) and torch.equal(vc[-1, -1], v[0])


@pytest.mark.gpu
@pytest.mark.parametrize("most", [0, 100])
def test_key_bound_only_sizes_the_split(most):
    """A bound on the keys that is too small costs time, not results."""
    q, k, v, cu, cu_k = packed_case([40, 90], [3000, 200], 4, 2, 64, F16)
    out, lse = K.flash_attention_packed(q, k, v, cu, cu_k, 90, 0.125, causal=True, want_lse=True, max_k=most)
    check_packed(q, k, v, cu, cu_k, 0.125, True, out, lse)
    for q_lens in ([1, 1], [40, 9]):
        q, kc, vc, table, cu, lens, rows = paged_case(q_lens, [3000, 200], 4, 2, 64, 16, F16)
        out, lse = K.flash_attention_paged(q, kc, vc, table, cu, lens, max(q_lens), 0.125, want_lse=True, max_kv=most)
        check_paged(q, rows, q_lens, 0.125, True, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_scores_that_grow_from_block_to_block(hd, causal):
    """Every block outgrows the reference of the one before (for half of the rows; for the others none does)."""
    q, k, v, cu, _ = packed_case([310], [1000], 4, 2, hd, F16)
    ramp = torch.arange(1000, device="cuda")[:, None, None] * (0.02 * 64 / hd)
    k = (0.1 * k.float() + ramp).to(F16)
    q = (0.1 * q.float() + torch.where(torch.arange(310, device="cuda") % 2 == 0, 1.0, -1.0)[:, None, None]).to(F16)
    cu_k = torch.tensor([0, 1000], dtype=torch.int32, device="cuda")
    out, lse = K.flash_attention_packed(q, k, v, cu, cu_k, 310, 0.125, causal=causal, want_lse=True, max_k=1000)
    check_packed(q, k, v, cu, cu_k, 0.125, causal, out, lse)


@pytest.mark.gpu
def test_large_scores_and_lowest_values():
    """Scores far apart (the running maximum moves by more than 2^8 in later
    blocks), and values at fp16's ends; in bf16 2^20 below them, since the fp32
    sum before its division holds up to 2^8 n |v|."""
    for dtype in (F16, BF16):
        q, k, v, cu, _ = packed_case([300], [900], 4, 2, 64, dtype, peak=20.0)
        ramp = torch.linspace(0.1, 8, 900, device="cuda")[:, None, None]
        k = (k.float() * ramp).to(dtype)
        v = v.clone()
        most = torch.finfo(dtype).max * (1 if dtype == F16 else 2.0 ** -20)
        v[100], v[200] = most, -most
        cu_k = torch.tensor([0, 900], dtype=torch.int32, device="cuda")
        out, lse = K.flash_attention_packed(q, k, v, cu, cu_k, 300, 0.125, causal=True, want_lse=True)
        want, wl, bound, bl = reference(q, k, v, 0.125, True, out, lse)
        fits = (want.abs() + bound < torch.finfo(dtype).max)
        assert ((out.double() - want).abs() <= bound)[fits].all()
        assert ((lse.double() - wl).abs() <= bl).all()
        # the same through the cache, one token
        kc, vc = (torch.cat([x, x[:124]]).view(64, 16, 2, 64) for x in (k, v))
        t = torch.arange(64, dtype=torch.int32, device="cuda")[None]
        one, n = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [900]))
        out1, lse1 = K.flash_attention_paged(q[-1:], kc, vc, t, one, n, 1, 0.125, want_lse=True)
        assert ((out1.double() - want[-1:]).abs() <= bound[-1:])[fits[-1:]].all()
        assert ((lse1.double() - wl[:, -1:]).abs() <= bl[:, -1:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_q,page", [(1, 16), (64, 32)])
def test_paged_graph_streams_and_repeats(max_q, page):
    """Captured and replayed with new lengths; on another stream; two graphs
    that share a workspace, replayed in turn; the same bits every time."""
    q_lens, kv_lens = [1, 1, 1], [5000, 90, 0]
    q, kc, vc, table, cu, lens, rows = paged_case(q_lens, kv_lens, 8, 2, 64, page, F16)
    args = (q, kc, vc, table, cu, lens, max_q, 0.125)
    want, _ = K.flash_attention_paged(*args)
    for _ in range(20):
        assert torch.equal(K.flash_attention_paged(*args)[0], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = K.flash_attention_paged(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    ws = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, _ = K.flash_attention_paged(*args, workspace=ws)
        graphs.append((g, o))
    ws.fill_(0xFF)  # NaN: nothing is read that the call has not written
    for g, o in graphs * 2:
        o.fill_(0)
        g.replay()
        assert torch.equal(o, want)
    lens.copy_(torch.tensor([700, 90, 0], dtype=torch.int32))
    graphs[0][0].replay()
    rows[0] = (rows[0][0][:700], rows[0][1][:700])
    check_paged(q, rows, q_lens, 0.125, True, graphs[0][1], None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_then_decode(dtype):
    """The operators together: prompts rotated into the cache, attended packed
    and, in chunks, through the cache; then decode steps. All against 64-bit
    attention over the rotated keys that the cache holds."""
    h, g, hd, page = 8, 2, 64, 16
    lens = [70, 1, 133]
    steps = 3
    gen = torch.Generator().manual_seed(11)
    freqs, m = K.rotary_freqs(hd, scaling="parts", factor=4.0, device="cuda")
    pages = 40
    kc, vc = (torch.full((pages, page, g, hd), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.randperm(pages, generator=gen)[:36].view(3, 12).int().cuda()

    def project(n):
        return torch.randn(n, (h + 2 * g) * hd, generator=gen).to(dtype).cuda().view(n, h + 2 * g, hd)

    def slots_of(b, first, n):
        j = torch.arange(first, first + n, device="cuda")
        return table[b, j // page].long() * page + j % page

    def held(b, n):  # what the cache holds of sequence b
        j = torch.arange(n, device="cuda")
        where = table[b, j // page].long()
        return kc[where, j % page], vc[where, j % page]

    qkv = project(sum(lens))
    q, k, v = qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    slots = torch.cat([slots_of(b, 0, n) for b, n in enumerate(lens)])
    qr = K.rotary_append(q, k, v, pos, freqs, kc, vc, slots, mscale=m)
    q2, kr = K.rotary(q, k, pos, freqs, mscale=m)
    assert torch.equal(qr, q2)
    cu = offsets(lens).cuda()
    out, lse = K.flash_attention_packed(qr, kr, v, cu, cu, max(lens), hd ** -0.5, causal=True, want_lse=True)
    rows = [held(b, n) for b, n in enumerate(lens)]
    check_paged(qr, rows, lens, hd ** -0.5, True, out, lse)
    n_kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = K.flash_attention_paged(qr, kc, vc, table, cu, n_kv, max(lens), hd ** -0.5, want_lse=True)
    check_paged(qr, rows, lens, hd ** -0.5, True, out, lse)
    one = torch.arange(4, dtype=torch.int32, device="cuda")
    for s in range(steps):
        now = [n + s for n in lens]
        qkv = project(3)
        slots = torch.cat([slots_of(b, n, 1) for b, n in enumerate(now)])
        qr = K.rotary_append(qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:], torch.tensor(now).cuda(), freqs, kc, vc, slots,
                             mscale=m)
        n_kv = torch.tensor([n + 1 for n in now], dtype=torch.int32, device="cuda")
        out, lse = K.flash_attention_paged(qr, kc, vc, table, one, n_kv, 1, hd ** -0.5, want_lse=True)
        check_paged(qr, [held(b, n + 1) for b, n in enumerate(now)], [1, 1, 1], hd ** -0.5, True, out, lse)


@pytest.mark.gpu
def test_empty_calls():
    q, k, v, cu, _ = packed_case([5], [5], 4, 2, 64, F16)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    K.flash_attention_packed(q, k, v, none, none, 5, 0.125, out=out)
    assert (out == 3).all()
    o, _ = K.flash_attention_packed(q[:0], k, v, torch.zeros_like(cu), cu, 0, 0.125)
    assert o.shape == (0, 4, 64)
    o, l = K.flash_attention_packed(q, k[:0], v[:0], cu, torch.zeros_like(cu), 5, 0.125, want_lse=True)
    assert (o == 0).all() and (l == -math.inf).all()
    cache = torch.zeros(0, 16, 2, 64, dtype=F16, device="cuda")
    for max_q in (5, 2):
        cu = torch.tensor([0, max_q], dtype=torch.int32, device="cuda")
        o, l = K.flash_attention_paged(q[:max_q], cache, cache, torch.zeros(1, 0, dtype=torch.int32, device="cuda"), cu,
                                       torch.zeros(1, dtype=torch.int32, device="cuda"), max_q, 0.125, want_lse=True)
        assert (o == 0).all() and (l == -math.inf).all()


# ----------------------------------------------------------------- refusals (any host)
def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _packed_args():
    return dict(q=torch.zeros(8, 4, 64).half(), k=torch.zeros(9, 2, 64).half(), v=torch.zeros(9, 2, 64).half(),
                cu_q=_i32(3), cu_k=_i32(3), max_q=4, scale=0.125)


def _paged_args():
    return dict(q=torch.zeros(8, 4, 64).half(), k_cache=torch.zeros(3, 16, 2, 64).half(),
                v_cache=torch.zeros(3, 16, 2, 64).half(), page_table=_i32(2, 4), cu_q=_i32(3), kv_lens=_i32(2), max_q=4,
                scale=0.125)


COMMON_REFUSALS = [
    ("q", torch.zeros(8, 4, 64), "fp16 or bf16|of the queries|float32"), ("q", torch.zeros(8, 256).half(), "tokens, heads"),
    ("q", torch.zeros(8, 3, 64).half(), "3 query heads"), ("q", torch.zeros(8, 4, 128).half()[..., ::2], "unit inner"),
    ("cu_q", torch.zeros(3, dtype=torch.int64), "int32"), ("cu_q", _i32(0), "offsets|entries"),
    ("max_q", -1, "negative"), ("scale", 0.0, "scale"), ("scale", -1.0, "scale"), ("scale", math.nan, "scale"),
    ("scale", math.inf, "scale"), ("out", torch.zeros(8, 4, 32).half(), "shape"),
    ("out", torch.zeros(8, 4, 64).double(), "out_dtype"), ("out_dtype", torch.bfloat16, "out_dtype"),
    ("lse", torch.zeros(8, 4), "lse"),
]


@pytest.mark.parametrize("name,value,match", COMMON_REFUSALS + [
    ("k", torch.zeros(9, 2, 32).half(), "one shape"), ("k", torch.zeros(9, 2, 64), "float16"),
    ("v", torch.zeros(8, 2, 64).half(), "one shape"), ("cu_k", _i32(4), "3 entries"), ("max_k", -1, "max_k"),
])
def test_packed_refuses(name, value, match):
    with pytest.raises(ValueError, match=match):
        K.flash_attention_packed(**{**_packed_args(), name: value})


@pytest.mark.parametrize("name,value,match", COMMON_REFUSALS + [
    ("k_cache", torch.zeros(3, 24, 2, 64).half(), "24|matching"), ("k_cache", torch.zeros(3, 16, 2, 64), "k_cache"),
    ("v_cache", torch.zeros(4, 16, 2, 64).half(), "matching"), ("page_table", _i32(3, 4), "page_table"),
    ("page_table", torch.zeros(2, 4, dtype=torch.int64), "page_table"), ("page_table", _i32(2, 8)[:, ::2], "page_table"),
    ("kv_lens", _i32(3), "kv_lens"), ("max_kv", -1, "max_kv"),
])
def test_paged_refuses(name, value, match):
    with pytest.raises(ValueError, match=match):
        K.flash_attention_paged(**{**_paged_args(), name: value})


@pytest.mark.parametrize("page", [8, 24, 17])
def test_paged_refuses_page_sizes(page):
    c = torch.zeros(3, page, 2, 64).half()
    with pytest.raises(ValueError, match="page_size"):
        K.flash_attention_paged(**{**_paged_args(), "k_cache": c, "v_cache": c})


def test_refuse_other_head_dims_and_cpu():
    q = torch.zeros(8, 4, 96).half()
    with pytest.raises(ValueError, match="head_dim"):
        K.flash_attention_packed(**{**_packed_args(), "q": q, "k": q, "v": q})
    with pytest.raises(RuntimeError, match="CUDA"):
        K.flash_attention_packed(**_packed_args())
    with pytest.raises(RuntimeError, match="CUDA"):
        K.flash_attention_paged(**_paged_args())


def test_seq_abi_refuses_without_device():
    """The C entries refuse malformed arguments with a status, device or not."""
    lib = _abi.load()
    ok = [64, 256, 64, 64, 128, 64, 64, 128, 64, 64, 64, 64, 256, 64, None, 8, 9, 2, 4, 2, 64, 4, 9, 0.125, 0, None, 0,
          None]
    for at, value, code in [(0, None, 1), (3, None, 1), (6, None, 1), (9, None, 1), (10, None, 1), (11, None, 1),
                            (0, 72, 2), (11, 72, 2), (25, 8, 2), (1, 257, 2), (5, 4, 2), (15, -1, 1), (15, 1 << 40, 1),
                            (16, -1, 1), (17, -1, 1), (18, 3, 1), (18, 1 << 40, 1), (19, 0, 1), (20, 96, 1), (21, -1, 1),
                            (22, -1, 1), (23, 0.0, 1), (23, math.nan, 1), (24, 4, 1)]:
        args = list(ok)
        args[at] = value
        assert lib.tf_flash_packed(*args) == code, (at, value)
        assert lib.tf_last_error()
    ok = [64, 256, 64, 64, 64, 2048, 128, 64, 3, 16, 64, 4, 4, 64, 64, 64, 256, 64, None, 8, 2, 4, 2, 64, 4, 64, 0.125, 0,
          None, 0, None]
    for at, value, code in [(0, None, 1), (3, None, 1), (4, None, 1), (10, None, 1), (13, None, 1), (14, None, 1),
                            (15, None, 1), (3, 72, 2), (5, 2049, 2), (8, -1, 1), (9, 0, 1), (9, 8, 1), (9, 24, 1),
                            (12, -1, 1), (12, 1 << 40, 1), (23, 32, 1), (26, -0.5, 1), (27, 16, 1)]:
        args = list(ok)
        args[at] = value
        assert lib.tf_flash_paged(*args) == code, (at, value)
    assert lib.tf_flash_packed_workspace(8, 2, 4, 3, 64, 4, 9) == -1
    assert lib.tf_flash_paged_workspace(8, -2, 4, 2, 64, 4, 9) == -1


@pytest.mark.parametrize("at,value", [(11, 0), (11, 192), (12, 0), (12, 56), (11, 64)])
def test_seq_abi_refuses_overlapping_results(at, value):
    """Rows of out in one place would be written in any order."""
    lib = _abi.load()
    args = [64, 256, 64, 64, 128, 64, 64, 128, 64, 64, 64, 64, 256, 64, None, 8, 9, 2, 4, 2, 64, 4, 9, 0.125, 0, None, 0,
            None]
    args[at + 1] = value
    assert lib.tf_flash_packed(*args) == 1
    assert b"overlap" in lib.tf_last_error()


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_workspace_needs_sizes_alone(hd):
    """(on a host without a device the size cannot be known: -1, with the device's message, not a refusal of sizes)"""
    lib = _abi.load()
    need = lib.tf_flash_paged_workspace(8, 2, 4, 2, hd, 4, 9)
    assert need > 0 or (not torch.cuda.is_available() and b"overlap" not in lib.tf_last_error())
