"""The serving operators beside the framework's flash attention, as they are measured.

    rotary / rotary_append     rotary positions of queries and keys, and the same with the new
                               keys and values written into a paged cache
    flash_attention_packed     attention over prompts of different lengths laid end to end, with
                               grouped heads
    flash_attention_paged      attention of each sequence's new tokens (one, a few, or a chunk)
                               over its paged cache

With `own` false, `run` computes them with elementary torch operations in 32 bits (rotary angles
in 64: the position times the frequency loses its fraction in 32), rounded once at the end. With
`own` true it calls the framework. Widths come from the framework's configurations (head widths 64
and 128, 4 to 16 heads, 100 000 tokens) and from grouped-head forms of them.
"""

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 24 sequences: positions and cache write, where launch latency counts
        dict(name="rotary_step", op="rotary", tokens=24, heads=16, kv_heads=4, hd=64, rot=64, interleaved=False,
             scaling="none", factor=1.0, far=8000, append=True, page=16, dtype="fp16"),
        # a prompt of 8 x 2048 tokens, half of each head rotated in the interleaved layout
        dict(name="rotary_prompt", op="rotary", tokens=16384, heads=16, kv_heads=16, hd=64, rot=32, interleaved=True,
             scaling="none", factor=1.0, far=2048, append=False, page=0, dtype="bf16"),
        # a 100 000-token prompt at a length eight times the trained one, written into the cache
        dict(name="rotary_long", op="rotary", tokens=100000, heads=32, kv_heads=8, hd=128, rot=128, interleaved=False,
             scaling="parts", factor=8.0, far=100000, append=True, page=64, dtype="bf16"),
        # two short prompts, the smallest attention call
        dict(name="packed_short", op="packed", seqs=2, shortest=100, longest=128, prefix=0, heads=4, kv_heads=4, hd=64,
             causal=True, lse=False, dtype="fp16"),
        # a batch of ragged prompts with four query heads to each key head
        dict(name="packed_ragged", op="packed", seqs=16, shortest=33, longest=2048, prefix=0, heads=16, kv_heads=4,
             hd=64, causal=True, lse=True, dtype="bf16"),
        # encoder batch: every token sees its whole sequence
        dict(name="packed_full", op="packed", seqs=8, shortest=1025, longest=2047, prefix=0, heads=16, kv_heads=16,
             hd=64, causal=False, lse=False, dtype="fp16"),
        # one long prompt
        dict(name="packed_long", op="packed", seqs=1, shortest=16384, longest=16384, prefix=0, heads=16, kv_heads=2,
             hd=128, causal=True, lse=False, dtype="bf16"),
        # one token of one sequence over a short cache: latency
        dict(name="paged_one", op="paged", seqs=1, kv_min=1000, kv_max=1000, chunks=0, chunk=1, few=1, heads=16,
             kv_heads=4, hd=64, page=16, lse=False, dtype="fp16"),
        # one token each of 64 sequences of very different lengths
        dict(name="paged_batch", op="paged", seqs=64, kv_min=100, kv_max=8192, chunks=0, chunk=1, few=1, heads=32,
             kv_heads=8, hd=128, page=16, lse=False, dtype="bf16"),
        # one token over a very long cache: only the split over its keys fills the card
        dict(name="paged_long", op="paged", seqs=1, kv_min=100000, kv_max=100000, chunks=0, chunk=1, few=1, heads=16,
             kv_heads=4, hd=64, page=64, lse=True, dtype="fp16"),
        # a chunk of a new prompt beside decoding sequences
        dict(name="paged_mixed", op="paged", seqs=24, kv_min=300, kv_max=6000, chunks=2, chunk=512, few=1, heads=32,
             kv_heads=8, hd=128, page=32, lse=False, dtype="bf16"),
        # chunks of long prompts over what is cached already
        dict(name="paged_chunk", op="paged", seqs=2, kv_min=12000, kv_max=16000, chunks=2, chunk=2000, few=1, heads=16,
             kv_heads=4, hd=64, page=128, lse=False, dtype="fp16"),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1.6e15)


def draw(rng):
    """One more case of the same ranges, no larger than the largest listed one."""
    most = max(map(_cost, listed()))
    case = _draw(rng)
    while _cost(case) > most:
        case = _draw(rng)
    return case


def _draw(rng):
    op = rng.choice(["rotary", "packed", "packed", "paged", "paged", "paged"])
    hd = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rotary":
        # an even part of the head, odd multiples of two among them
        rot = rng.choice([hd, hd // 2, 2 * rng.randint(1, hd // 2)])
        scaling = rng.choice(["none", "linear", "ntk", "parts"])
        append = rng.random() < 0.5
        return dict(op=op, tokens=_between(rng, 1, 60000), heads=heads, kv_heads=kv_heads, hd=hd, rot=rot,
                    interleaved=rng.random() < 0.5, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 32.0]), far=_between(rng, 100, 1000000),
                    append=append, page=rng.choice([16, 32, 64, 128]) if append else 0, dtype=dtype)
    if op == "packed":
        longest = _between(rng, 1, 4096)
        return dict(op=op, seqs=_between(rng, 1, 24), shortest=max(1, longest // rng.choice([1, 4, 50])),
                    longest=longest, prefix=rng.choice([0, 0, 0, _between(rng, 1, 2000)]), heads=heads,
                    kv_heads=kv_heads, hd=hd, causal=rng.random() < 0.75, lse=rng.random() < 0.5, dtype=dtype)
    seqs = _between(rng, 1, 64)
    kv_max = _between(rng, 1, 100000 if seqs <= 4 else 8192)
    chunks = rng.choice([0, 0, rng.randint(0, min(seqs, 3)), min(seqs, 2)])
    return dict(op=op, seqs=seqs, kv_min=max(1, kv_max // rng.choice([1, 3, 80])), kv_max=kv_max, chunks=chunks,
                chunk=_between(rng, 2, 1500), few=rng.choice([1, 1, 1, 2, 5]), heads=heads, kv_heads=kv_heads, hd=hd,
                page=rng.choice([16, 32, 64, 128, 256]), lse=rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """Query and key lengths of a case's sequences, from the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "packed":
        q = [_between(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]
        return q, [n + case["prefix"] for n in q]
    kv = [_between(rng, case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    q = [min(n, case["chunk"] if i < case["chunks"] else case["few"]) for i, n in enumerate(kv)]
    return q, kv


def _pairs(case):
    """Admitted (query, key) pairs, one head."""
    total = 0
    for q, k in zip(*_lengths(case)):
        total += q * k - (q * (q - 1) // 2 if case["op"] == "paged" or case["causal"] else 0)
    return total


def work(case):
    h, g, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["op"] == "rotary":
        t, heads = case["tokens"], h + g
        values = 2 * t * hd * (heads + (g if case["append"] else 0))  # read once, written once
        return {"bytes": 2 * values + 8 * t * (2 if case["append"] else 1), "flops": 3 * t * heads * case["rot"]}
    q, k = _lengths(case)
    nbytes = 2 * hd * (2 * h * sum(q) + 2 * g * sum(k)) + (4 * h * sum(q) if case["lse"] else 0)
    if case["op"] == "paged":
        nbytes += 4 * sum(-(-n // case["page"]) for n in k)
    return {"bytes": nbytes, "flops": 4 * hd * h * _pairs(case)}


# ------------------------------------------------------------------ inputs
def _freqs(case):
    """Angles per position (64 bits) and the factor on the rotated values."""
    rot, factor = case["rot"], case["factor"]
    base = 10000.0
    if case["scaling"] == "ntk" and rot > 2:
        base *= factor ** (rot / (rot - 2))
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "parts":
        turns = 4096 * f / (2 * math.pi)  # within the trained length
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return f, 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    h, g, hd = case["heads"], case["kv_heads"], case["hd"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dt)

    st = {"case": case}
    if case["op"] == "rotary":
        t = case["tokens"]
        qkv = normal(t, (h + 2 * g) * hd).view(t, h + 2 * g, hd)  # the packed projection's output
        st.update(q=qkv[:, :h], k=qkv[:, h:h + g], v=qkv[:, h + g:])
        st["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device=dev)
        f, st["mscale"] = _freqs(case)
        st["freqs"] = f.to(dev)
        if case["append"]:
            pages = -(-t // case["page"]) + 3
            st["k_cache"] = torch.zeros(pages, case["page"], g, hd, dtype=dt, device=dev)
            st["v_cache"] = torch.zeros_like(st["k_cache"])
            order = torch.randperm(pages, generator=gen, device=dev)
            at = torch.arange(t, device=dev)
            st["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        return st
    ql, kl = _lengths(case)
    st["scale"] = hd ** -0.5
    st["q_lens"], st["k_lens"] = ql, kl
    st["max_q"], st["max_k"] = max(ql), max(kl)
    cu = [0]
    for n in ql:
        cu.append(cu[-1] + n)
    st["cu_q"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    if case["op"] == "packed":
        cu = [0]
        for n in kl:
            cu.append(cu[-1] + n)
        st["cu_k"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        if case["prefix"]:
            kv = normal(sum(kl), 2 * g * hd).view(-1, 2 * g, hd)
            st.update(q=normal(sum(ql), h, hd), k=kv[:, :g], v=kv[:, g:])
        else:  # the packed projection's output
            qkv = normal(sum(ql), (h + 2 * g) * hd).view(-1, h + 2 * g, hd)
            st.update(q=qkv[:, :h], k=qkv[:, h:h + g], v=qkv[:, h + g:])
        return st
    page = case["page"]
    need = [-(-n // page) for n in kl]
    st["q"] = normal(sum(ql), h, hd)
    st["k_cache"] = normal(sum(need) + 2, page, g, hd)
    st["v_cache"] = normal(sum(need) + 2, page, g, hd)
    order = torch.randperm(sum(need) + 2, generator=gen, device=dev).tolist()
    table = torch.full((len(kl), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    st["page_table"] = table.to(dev)
    st["kv_lens"] = torch.tensor(kl, dtype=torch.int32, device=dev)
    return st


# ------------------------------------------------------------------ the operators
def run(state):
    case = state["case"]
    if own:
        from transformer_optimization_b200 import kernels

        if case["op"] == "rotary":
            if case["append"]:
                q = kernels.rotary_append(state["q"], state["k"], state["v"], state["positions"], state["freqs"],
                                          state["k_cache"], state["v_cache"], state["slots"],
                                          interleaved=case["interleaved"], mscale=state["mscale"])
                return q, state["k_cache"], state["v_cache"]
            return kernels.rotary(state["q"], state["k"], state["positions"], state["freqs"],
                                  interleaved=case["interleaved"], mscale=state["mscale"])
        if case["op"] == "packed":
            out, lse = kernels.flash_attention_packed(
                state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], state["max_q"], state["scale"],
                max_k=state["max_k"], causal=case["causal"], want_lse=case["lse"])
        else:
            out, lse = kernels.flash_attention_paged(
                state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["cu_q"],
                state["kv_lens"], state["max_q"], state["scale"], max_kv=state["max_k"], want_lse=case["lse"])
        return (out, lse) if case["lse"] else out

    if case["op"] == "rotary":
        angle = state["positions"].double()[:, None] * state["freqs"]
        cos = (angle.cos() * state["mscale"]).float()[:, None]
        sin = (angle.sin() * state["mscale"]).float()[:, None]
        q, k = (_turn(state[n], cos, sin, case) for n in ("q", "k"))
        if not case["append"]:
            return q, k
        g, hd = case["kv_heads"], case["hd"]
        state["k_cache"].view(-1, g, hd)[state["slots"]] = k
        state["v_cache"].view(-1, g, hd)[state["slots"]] = state["v"]
        return q, state["k_cache"], state["v_cache"]

    q = state["q"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
    q0 = k0 = 0
    for i, (nq, nk) in enumerate(zip(state["q_lens"], state["k_lens"])):
        if case["op"] == "packed":
            k, v = state["k"][k0:k0 + nk], state["v"][k0:k0 + nk]
        else:
            rows = state["page_table"][i, :-(-nk // case["page"])].long()
            k, v = (state[n][rows].flatten(0, 1)[:nk] for n in ("k_cache", "v_cache"))
        _attend(q[q0:q0 + nq], k, v, state["scale"], case["op"] == "paged" or case["causal"], out[q0:q0 + nq],
                lse[:, q0:q0 + nq])
        q0, k0 = q0 + nq, k0 + nk
    return (out, lse) if case["lse"] else out


def _turn(x, cos, sin, case):
    rot, xf = case["rot"], x.float()
    part, rest = xf[..., :rot], xf[..., rot:]
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([part, rest], -1).to(x.dtype)


def _attend(q, k, v, scale, causal, out, lse):
    """One sequence: q [nq, H, hd], k and v [nk, G, hd]; the last query stands at the last key."""
    (nq, h, hd), (nk, g, _) = q.shape, k.shape
    step = g if nq * nk * h <= 1 << 29 else 1  # key heads at a time
    for j in range(0, g, step):
        n = min(step, g - j)
        qf = q[:, j * (h // g):(j + n) * (h // g)].float().reshape(nq, n, h // g, hd).permute(1, 2, 0, 3)
        kf = k[:, j:j + n].float().permute(1, 2, 0)
        vf = v[:, j:j + n].float().transpose(0, 1)
        s = torch.matmul(qf, kf[:, None]) * scale
        if causal and nq > 1:
            i = torch.arange(nq, device=q.device)[:, None] + (nk - nq)
            s = s.masked_fill(torch.arange(nk, device=q.device) > i, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, vf[:, None]) / total
        hs = slice(j * (h // g), (j + n) * (h // g))
        out[:, hs] = o.permute(2, 0, 1, 3).reshape(nq, n * (h // g), hd).to(out.dtype)
        lse[hs] = (top + total.log()).reshape(n * (h // g), nq)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, st)
    if 4 * case["hd"] * case["heads"] * sum(a * b for a, b in zip(st["q_lens"], st["k_lens"])) > 6e12:
        return None
    h, g = case["heads"], case["kv_heads"]
    q = st["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(h, q.shape[0], dtype=torch.float64, device=q.device)
    qs, ks = 0, 0
    for i, (nq, nk) in enumerate(zip(st["q_lens"], st["k_lens"])):
        if case["op"] == "packed":
            k, v = st["k"][ks:ks + nk].double(), st["v"][ks:ks + nk].double()
        else:
            where = torch.arange(nk, device=q.device)
            pages = st["page_table"][i].long()[where // case["page"]]
            k = st["k_cache"][pages, where % case["page"]].double()
            v = st["v_cache"][pages, where % case["page"]].double()
        masked = case["op"] == "paged" or case["causal"]
        for head in range(h):
            kk, vv = k[:, head // (h // g)], v[:, head // (h // g)]
            for a in range(0, nq, 4096):  # rows at a time
                b = min(nq, a + 4096)
                logit = st["scale"] * (q[qs + a:qs + b, head] @ kk.T)
                if masked:
                    last = torch.arange(a, b, device=q.device) + nk - nq
                    logit[last[:, None] < torch.arange(nk, device=q.device)[None]] = -math.inf
                lse[head, qs + a:qs + b] = torch.logsumexp(logit, 1)
                out[qs + a:qs + b, head] = torch.softmax(logit, 1) @ vv
        qs, ks = qs + nq, ks + nk
    return (out, lse) if case["lse"] else out


def _exact_rotary(case, st):
    rot, m = case["rot"], st["mscale"]
    turn = torch.polar(torch.full((), m, dtype=torch.float64, device=st["q"].device),
                       torch.outer(st["positions"].double(), st["freqs"]))[:, None]

    def go(x):
        y = x.double().clone()
        first, second = ((slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"]
                         else (slice(0, rot // 2), slice(rot // 2, rot)))
        z = torch.complex(y[..., first].clone(), y[..., second].clone()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = go(st["q"]), go(st["k"])
    if not case["append"]:
        return q, k
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    where = st["slots"]
    kc[where // case["page"], where % case["page"]] = k
    vc[where // case["page"], where % case["page"]] = st["v"].double()
    return q, kc, vc
