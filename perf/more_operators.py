"""The operators of a block that generates chunk by chunk from a cache of keys and values, in their plain form and as the package's kernels.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before
the call, ``run`` is one pass - forward, or forward and backward - and ``work`` counts the bytes and operations a pass
cannot do without.  ``exact`` is the operator's definition in 64 bits.  Where ``own`` is false ``run`` computes the plain form
with elementary torch operations, angles in 64 bits and the rest in 32, rounded once at the end; where it is true it calls the package.

* ``rotary``     rotary positions of q and k ``[B, L, H, D]``: channels 2 i and 2 i + 1 (interleaved) or i and i + R / 2 (halves) of the first R
                 turn by position times frequency i, the position one of several axes' where the pairs are divided into sections;
                 its backward pass turns the gradients back.
* ``append``     new keys and values go into the pages of a cache ``[pages, Hkv, page size, D]`` of the tensors' type or of 8 bits with a
                 scale for every head; q and the keys are given their rotary positions on the way.
* ``attention``  softmax(sm_scale q k^T) v of the last tokens of every sequence on all its keys in the cache, causal or not.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
DEVICE = "cuda"
#: what the scales of an 8-bit cache let its largest code stand for
LARGEST = 5.0


def listed():
    return [
        # One new token in each of a few sequences, far into them: launches and host work.
        _rotary("rotary_few_tokens", "fwd", B=8, L=1, H=40, Hkv=8, D=128, R=128, interleaved=False, sections=0, far=131072, dtype="bf16"),
        # The 14B video model's q and k at 480p, positions of frame, row and column; forward and backward.
        _rotary("rotary_video_train", "train", B=1, L=32760, H=40, Hkv=40, D=128, R=128, interleaved=True, sections=3, far=0, dtype="bf16"),
        # A part of an unusual head, few key heads, an odd length, positions far out, fp32.
        _rotary("rotary_part_fp32_train", "train", B=3, L=2777, H=12, Hkv=4, D=80, R=32, interleaved=False, sections=0, far=1000003, dtype="fp32"),
        # A decoding step of a batch: a token of each sequence goes into small pages.
        _append("append_tokens", B=64, L=1, Lk=1024, H=32, Hkv=8, D=128, page=16, interleaved=False, sections=0, dtype="bf16", cache="bf16", ragged=True),
        # Long prompts of two lengths.
        _append("append_prompt", B=2, L=16384, Lk=16384, H=32, Hkv=8, D=128, page=64, interleaved=False, sections=0, dtype="bf16", cache="bf16", ragged=True),
        # One latent frame of a 480p video (30 x 52 tokens) goes into an 8-bit cache with a page for each frame.
        _append("append_frame_fp8", B=1, L=1560, Lk=6 * 1560, H=40, Hkv=40, D=128, page=1560, interleaved=True, sections=3, dtype="bf16", cache="fp8", ragged=False),
        # Five new tokens on a few cached ones, one sequence without any: nothing but latency.
        _attention("attention_short_fp16", B=3, Lq=5, Lk=67, H=12, Hkv=12, D=64, page=16, causal=True, dtype="fp16", cache="fp16", ragged=True),
        # One token of one long sequence, key heads shared by five.
        _attention("attention_token_32760", B=1, Lq=1, Lk=32760, H=40, Hkv=8, D=128, page=64, causal=True, dtype="bf16", cache="bf16", ragged=False),
        # A decoding step of a batch of sequences of all lengths in small pages.
        _attention("attention_tokens_ragged", B=64, Lq=1, Lk=8192, H=32, Hkv=8, D=128, page=16, causal=True, dtype="bf16", cache="bf16", ragged=True),
        # The same on 8-bit caches of longer sequences.
        _attention("attention_tokens_fp8", B=16, Lq=1, Lk=32760, H=40, Hkv=8, D=128, page=64, causal=True, dtype="bf16", cache="fp8", ragged=True),
        # A latent frame attends to itself and twenty before it.
        _attention("attention_frame", B=1, Lq=1560, Lk=32760, H=40, Hkv=40, D=128, page=1560, causal=False, dtype="bf16", cache="bf16", ragged=False),
        # A chunk of a long prompt, causal: the largest.
        _attention("attention_chunk_4096", B=1, Lq=4096, Lk=32768, H=40, Hkv=8, D=128, page=64, causal=True, dtype="bf16", cache="bf16", ragged=False),
    ]


def _rotary(name, mode, **sizes):
    return dict(name=name, op="rotary", mode=mode, **sizes)


def _append(name, **sizes):
    return dict(name=name, op="append", **sizes)


def _attention(name, **sizes):
    return dict(name=name, op="attention", **sizes)


def _log_int(rng, lo, hi):
    """An integer spread evenly over its logarithm; odd as often as even."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "attention", "attention", "attention"))
    if op == "rotary":
        D = rng.choice((64, 128, 128, 80, 96, 256))
        case = dict(op=op, mode=rng.choice(("train", "fwd")), B=rng.choice((1, 1, 2, 3, 8)), L=_log_int(rng, 1, 32760), H=rng.choice((1, 8, 12, 32, 40)), Hkv=0,
                    D=D, R=rng.choice((D, D, D // 2, 32)), interleaved=rng.random() < 0.5, sections=rng.choice((0, 0, 3)), far=rng.choice((0, 131072, 1000003)),
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
        case["Hkv"] = case["H"] // rng.choice([g for g in (1, 1, 4, 5) if case["H"] % g == 0])
        while work(case)["bytes"] > 5.3e9 / (2 if case["mode"] == "train" else 4):
            case["L"] = max(1, case["L"] * 9 // 10)
        return case
    H = rng.choice((1, 8, 12, 16, 32, 40))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    case = dict(op=op, B=0, H=H, Hkv=H // rng.choice([g for g in (1, 1, 2, 4, 5, 8) if H % g == 0]), D=rng.choice((128, 128, 64)),
                page=rng.choice((16, 16, 32, 64, 64, 128, 256, 20, 100, 1560)), dtype=dtype, cache=rng.choice((dtype, dtype, "fp8")), ragged=rng.random() < 0.6)
    if op == "append":
        case.update(B=_log_int(rng, 1, 64), L=1 if rng.random() < 0.4 else _log_int(rng, 2, 16384), interleaved=rng.random() < 0.5, sections=rng.choice((0, 0, 3)))
        case["Lk"] = case["L"] + _log_int(rng, 1, 2048)
        while work(case)["bytes"] > 5e8 or case["B"] * case["Lk"] * case["Hkv"] * case["D"] > 1 << 27:
            case["L"], case["Lk"], case["B"] = max(1, case["L"] * 4 // 5), max(2, case["Lk"] * 4 // 5), max(1, case["B"] * 9 // 10)
        return case
    kind = rng.choice(("token", "token", "few", "chunk", "chunk"))
    case.update(B=_log_int(rng, 1, 64) if kind == "token" else rng.choice((1, 1, 2, 3)), Lq={"token": 1, "few": _log_int(rng, 2, 64), "chunk": _log_int(rng, 64, 4096)}[kind],
                causal=kind == "token" or rng.random() < 0.7)
    case["Lk"] = case["Lq"] + _log_int(rng, 1, 32760)
    while work(case)["flops"] > 2.5e12 or work(case)["bytes"] > 1e9 or case["B"] * case["Lk"] * case["H"] * case["Lq"] > 1 << 32:
        case["Lk"] = max(case["Lq"], case["Lk"] * 9 // 10)
        case["Lq"], case["B"] = min(case["Lk"], max(1, case["Lq"] * 19 // 20)), max(1, case["B"] * 19 // 20)
    return case


def _counts(case):
    """(tokens of each sequence with the new ones, new ones) of a padded batch: the first is the longest, of three the third has none."""
    B, new, all_ = case["B"], case.get("Lq", case.get("L")), case["Lk"]
    share = [1.0 - 0.9 * b / B for b in range(B)] if case["ragged"] else [1.0] * B
    n = [max(1, int(new * s)) for s in share]
    total = [max(m, int(all_ * s)) for m, s in zip(n, share)]
    if case["ragged"] and B == 3:
        n[2] = total[2] = 0
    return total, n


def _values(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std).to(dtype)


def _sections(case):
    """Pairs of each axis: frame, row and column of a video; one axis otherwise."""
    pairs = case.get("R", case["D"]) // 2
    return (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3) if case["sections"] else None


def _frequencies(case):
    """Radians that a pair turns by from one position to the next, in 64 bits: 10000^(-i / pairs), of every axis anew; far positions on a scale of their own."""
    pairs, base = case.get("R", case["D"]) // 2, 1e6 if case.get("far") else 1e4
    parts = [torch.arange(n, dtype=torch.float64, device=DEVICE) / n for n in (_sections(case) or (pairs,))]
    return torch.pow(base, -torch.cat(parts)) * (0.25 if case.get("far") == 1000003 else 1.0)


def _grid(g, case, B, L):
    """Positions of a video's tokens: 30 rows of 52, frame after frame, each sequence starting at a frame of its own."""
    at = torch.arange(L, device=DEVICE)
    first = torch.randint(0, 21, (B, 1), generator=g, device=DEVICE)
    return torch.stack(torch.broadcast_tensors(first + at // 1560, at // 52 % 30, at % 52), -1).int()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, B, H, Hkv, D, dtype = (case[n] for n in ("op", "B", "H", "Hkv", "D", "dtype"))
    dtype = DTYPES[dtype]
    state = dict(op=op)
    if op in ("rotary", "append"):
        L = case["L"]
        state.update(interleaved=case["interleaved"], sections=_sections(case), frequencies=_frequencies(case), positions=None)
        if case["sections"]:
            state["positions"] = _grid(g, case, B, L)
    if op == "rotary":
        train = case["mode"] == "train"
        state["train"] = train
        if case["far"] and not case["sections"]:
            state["positions"] = (torch.randint(0, case["far"], (B, 1), generator=g, device=DEVICE) + torch.arange(L, device=DEVICE)).int()
        state["q"], state["k"] = (_values(g, (B, L, h, D), dtype).requires_grad_(train) for h in (H, Hkv))
        if train:
            state["dq"], state["dk"] = (_values(g, (B, L, h, D), dtype) for h in (H, Hkv))
        return state
    total, new = _counts(case)
    page, kind = case["page"], DTYPES[case["cache"]]
    needed = [(n + page - 1) // page for n in total]
    # pages of all sequences in no order, some of nobody; entries behind a sequence's last page are -1
    pages = sum(needed) + 2
    order = torch.randperm(pages, generator=g, device=DEVICE).int().tolist()
    table, used = [], 0
    for n in needed:
        table.append(order[used : used + n] + [-1] * (max(needed) + 1 - n))
        used += n
    state["pages"] = torch.tensor(table, dtype=torch.int32, device=DEVICE)
    state["k_lens"] = torch.tensor(total, dtype=torch.int32, device=DEVICE)
    state["q_lens"] = torch.tensor(new, dtype=torch.int32, device=DEVICE) if case["ragged"] else None
    state["k_scale"] = state["v_scale"] = None
    spread = 1.0
    if kind == DTYPES["fp8"]:
        state["k_scale"], state["v_scale"] = (LARGEST / 448 * (0.8 + 0.4 * torch.rand(Hkv, generator=g, device=DEVICE)) for _ in range(2))
        spread = 448 / LARGEST
    # keys as a model has them, off zero by an amount of each head's channel
    offset = torch.randn((Hkv, 1, D), generator=g, device=DEVICE)
    state["k_pages"] = (_values(g, (pages, Hkv, page, D), torch.float32, 0.8) + 0.5 * offset).mul_(spread).clamp_(-448, 448).to(kind)
    state["v_pages"] = _values(g, (pages, Hkv, page, D), torch.float32, spread).clamp_(-448, 448).to(kind)
    L = case["L"] if op == "append" else case["Lq"]
    state["q"] = _values(g, (B, L, H, D), dtype)
    if op == "append":
        state["k"], state["v"] = _values(g, (B, L, Hkv, D), dtype), _values(g, (B, L, Hkv, D), dtype)
    else:
        state["causal"] = case["causal"]
    return state


# ------------------------------------------------------------------------------------------------ the calls

def run(state):
    if state["op"] == "rotary":
        return _rotary_own(state) if own else _rotary_plain(state)
    if state["op"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attention_own(state) if own else _attention_plain(state)


def _rotary_own(state):
    from ksanadit_amd import train_ops

    q, k = train_ops.rotary(state["q"], state["k"], frequencies=state["frequencies"], positions=state["positions"], sections=state["sections"],
                            interleaved=state["interleaved"])
    if not state["train"]:
        return q, k
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"])))


def _cache(state):
    from ksanadit_amd import cache_ops

    return cache_ops.PagedCache(state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"])


def _append_own(state):
    from ksanadit_amd import cache_ops

    q = cache_ops.append(state["k"], state["v"], _cache(state), state["pages"], state["k_lens"], state["q_lens"], q=state["q"], frequencies=state["frequencies"],
                         positions=state["positions"], sections=state["sections"], interleaved=state["interleaved"])
    return q, state["k_pages"], state["v_pages"]


def _attention_own(state):
    from ksanadit_amd import cache_ops

    return cache_ops.attention(state["q"], _cache(state), state["pages"], state["k_lens"], state["q_lens"], is_causal=state["causal"])


# ------------------------------------------------------------------------------------------------ the plain forms

def _turns(state, positions, bits):
    """Cosines and sines ``[B or 1, L, 1, pairs]`` of tokens at ``positions`` ([B or 1, L], or with an axis behind for every section)."""
    if state["sections"] is not None:
        axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device=positions.device), torch.tensor(state["sections"], device=positions.device))
        at = positions.index_select(-1, axis)
    else:
        at = positions.unsqueeze(-1)
    angle = (at.double() * state["frequencies"]).unsqueeze(-2)
    return angle.cos().to(bits), angle.sin().to(bits)


def _turned(x, cos, sin, interleaved):
    """x's first channels turned, the others as they are."""
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2 : R])
    c, d = a * cos - b * sin, a * sin + b * cos
    return torch.cat((torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1), x[..., R:]), -1)


def _rotary_positions(state):
    if state["positions"] is None:
        return torch.arange(state["q"].shape[1], device=state["q"].device).unsqueeze(0)
    return state["positions"]


def _rotary_plain(state):
    cos, sin = _turns(state, _rotary_positions(state), torch.float32)
    q, k = state["q"].detach(), state["k"].detach()
    out = tuple(_turned(t.float(), cos, sin, state["interleaved"]).to(t.dtype) for t in (q, k))
    if not state["train"]:
        return out
    return out + tuple(_turned(state[n].float(), cos, -sin, state["interleaved"]).to(q.dtype) for n in ("dq", "dk"))


def _new_tokens(state):
    """(position of every new token, whether there is one) ``[B, L]``"""
    L = state["q"].shape[1]
    at = torch.arange(L, device=state["q"].device).unsqueeze(0)
    n = torch.full_like(state["k_lens"], L) if state["q_lens"] is None else state["q_lens"]
    return (state["k_lens"] - n).unsqueeze(1) + at, at < n.unsqueeze(1)


def _append_plain(state):
    place, there = _new_tokens(state)
    cos, sin = _turns(state, place if state["positions"] is None else state["positions"], torch.float32)
    q = _turned(state["q"].float(), cos, sin, state["interleaved"]).to(state["q"].dtype) * there[:, :, None, None]
    b, i = there.nonzero(as_tuple=True)
    at = place[b, i]
    size = state["k_pages"].shape[2]
    page, slot = state["pages"][b, at // size].long(), at % size
    k = _turned(state["k"].float(), cos, sin, state["interleaved"])[b, i]
    v = state["v"].float()[b, i]
    if state["k_scale"] is not None:
        k, v = (k / state["k_scale"][:, None]).clamp(-448, 448), (v / state["v_scale"][:, None]).clamp(-448, 448)
    raw = torch.uint8 if state["k_scale"] is not None else state["k_pages"].dtype  # (torch writes 8-bit floats by index as bytes only)
    state["k_pages"].view(raw)[page, :, slot] = k.to(state["k_pages"].dtype).view(raw)
    state["v_pages"].view(raw)[page, :, slot] = v.to(state["v_pages"].dtype).view(raw)
    return q, state["k_pages"], state["v_pages"]


def _attention_plain(state):
    q = state["q"]
    B, L, H, D = q.shape
    Hkv, size = state["k_pages"].shape[1:3]
    table = state["pages"].clamp(min=0).long()
    raw = torch.uint8 if state["k_scale"] is not None else q.dtype
    # a sequence's pages side by side: [B, Hkv, keys, D]
    k, v = (state[n].view(raw)[table].view(state[n].dtype).float().transpose(1, 2).reshape(B, Hkv, -1, D) for n in ("k_pages", "v_pages"))
    place, there = _new_tokens(state)
    key = torch.arange(k.shape[2], device=q.device)
    seen = (key < state["k_lens"][:, None, None]) & there[:, :, None]
    if state["causal"]:
        seen = seen & (key <= place[:, :, None])
    # rows of the heads that share a key head stand below each other
    group = H // Hkv
    rows = q.float().reshape(B, L, Hkv, group, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, group * L, D)
    p = torch.matmul(rows, k.transpose(2, 3).contiguous()).mul_(D ** -0.5)
    if state["k_scale"] is not None:
        p.mul_(state["k_scale"][:, None, None])
    p.view(B, Hkv, group, L, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total.masked_fill_(total == 0, 1.0)
    if state["v_scale"] is not None:
        o = o * state["v_scale"][:, None, None]
    return o.reshape(B, Hkv, group, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H, D).to(q.dtype)


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _attention_exact(case, state)
    if case["op"] == "append":
        return _append_exact(case, state)
    names = ("q", "k", "dq", "dk") if state["train"] else ("q", "k")
    B, L = state["q"].shape[:2]
    positions = [None] * B if state["positions"] is None else [state["positions"][b if state["positions"].shape[0] > 1 else 0] for b in range(B)]
    return tuple(torch.stack([_complex_turn(state, state[n].detach()[b], torch.arange(L, device=DEVICE) if positions[b] is None else positions[b],
                                            1.0 if n in ("q", "k") else -1.0) for b in range(B)]) for n in names)


def _complex_turn(state, x, positions, sign):
    """``[L, H, D]``: each pair a complex number, multiplied with exp(i sign position frequency)."""
    pairs = state["frequencies"].shape[0]
    columns, first = [], 0
    for axis, n in enumerate(state["sections"] or (pairs,)):
        at = positions[:, axis] if state["sections"] else positions
        columns.append(at.double()[:, None] * state["frequencies"][first : first + n])
        first += n
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), sign * torch.cat(columns, 1))[:, None]
    x = x.double()
    if state["interleaved"]:
        pair = torch.view_as_real(torch.view_as_complex(x[..., : 2 * pairs].reshape(*x.shape[:2], pairs, 2)) * turn).reshape(*x.shape[:2], 2 * pairs)
    else:
        z = torch.complex(x[..., :pairs], x[..., pairs : 2 * pairs]) * turn
        pair = torch.cat((z.real, z.imag), -1)
    return torch.cat((pair, x[..., 2 * pairs :]), -1)


def _append_exact(case, state):
    total, new = _counts(case)
    size = case["page"]
    q = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    pages = [state[n].float().double() for n in ("k_pages", "v_pages")]
    for b, (n, m) in enumerate(zip(total, new)):
        if m == 0:
            continue
        place = torch.arange(n - m, n, device=DEVICE)
        positions = place if state["positions"] is None else state["positions"][b, :m]
        q[b, :m] = _complex_turn(state, state["q"][b, :m], positions, 1.0)
        for out, rows, scale in zip(pages, (_complex_turn(state, state["k"][b, :m], positions, 1.0), state["v"][b, :m].double()), (state["k_scale"], state["v_scale"])):
            if scale is not None:
                rows = (rows / scale.double()[:, None]).clamp(-448, 448)
            out[state["pages"][b].long()[place // size], :, place % size] = rows
    return q, *pages


def _attention_exact(case, state):
    """Sequence by sequence, head by head."""
    total, new = _counts(case)
    q, size = state["q"], case["page"]
    H, D = q.shape[2:]
    group = H // case["Hkv"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (n, m) in enumerate(zip(total, new)):
        at = torch.arange(n, device=q.device)
        page, slot = state["pages"][b].long()[at // size], at % size
        hidden = at[None] > at[n - m :, None] if case["causal"] else None
        for h in range(case["Hkv"] if m else 0):
            k, v = (state[name][:, h].float()[page, slot].double() for name in ("k_pages", "v_pages"))
            if state["k_scale"] is not None:
                k, v = k * state["k_scale"][h].double(), v * state["v_scale"][h].double()
            for j in range(h * group, (h + 1) * group):
                scores = torch.mm(q[b, :m, j].double(), k.t()) / math.sqrt(D)
                if hidden is not None:
                    scores = scores.masked_fill(hidden, -math.inf)
                o[b, :m, j] = torch.mm(torch.softmax(scores, 1), v)
    return o


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    """Operations: a multiply-add counts as 2.  Bytes: every input that exists read once and every output written once; of a cache, the tokens that are seen or written."""
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
    B, H, Hkv, D, t = case["B"], case["H"], case["Hkv"], case["D"], size[case["dtype"]]
    if case["op"] == "rotary":
        n = B * case["L"] * (H + Hkv) * (2.0 if case["mode"] == "train" else 1.0)
        return {"bytes": 2 * n * D * t, "flops": 3 * n * case["R"]}
    total, new = _counts(case)
    c = size[case["cache"]]
    if case["op"] == "append":
        rows, all_ = sum(new), B * case["L"]
        return {"bytes": float((rows * H + all_ * H + 2 * rows * Hkv) * D * t + 2 * rows * Hkv * D * c), "flops": 3.0 * rows * (H + Hkv) * D}
    pairs = sum(m * n - (m * (m - 1) // 2 if case["causal"] else 0) for n, m in zip(total, new))
    return {"bytes": float((sum(new) + B * case["Lq"]) * H * D * t + 2 * sum(n for n, m in zip(total, new) if m) * Hkv * D * c), "flops": 4.0 * pairs * H * D}
