"""The differentiable operators of a transformer block's attention half, in their plain form and as the package's kernels.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before
the call, ``run`` is one pass - forward, or forward and backward - and ``work`` counts the bytes and operations a pass
cannot do without.  ``exact`` is the operator's definition in 64 bits.  Where ``own`` is false ``run`` computes the plain form
with elementary torch operations in fp32, rounded once at the end; where it is true it calls the package.

* ``attention``      softmax(sm_scale q k^T) v on 16-bit tensors ``[B, L, H, D]``, with the key and query counts of padded
                     batches, causal masking and shared key heads; its backward pass gives dq, dk, dv.
* ``residual_norm``  what stands between two parts of a block: h = r x + gate * post_norm(y), n = norm(h) * (1 + scale) +
                     shift, x the residual stream, y the part's output; its backward pass gives the gradients of both
                     tensors and of every vector.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"
EPS = 1e-6


def listed():
    return [
        # A unit-test-sized step: nothing but latency (launches and host work).
        _attention("unit_train_fp16", "train", B=2, H=64, Hkv=64, Lq=32, Lk=32, D=128, dtype="fp16"),
        # One new token attends to a long sequence of shared key heads: the form of a call that generates.
        _attention("one_token_32760", "fwd", B=1, H=40, Hkv=8, Lq=1, Lk=32760, D=128, dtype="bf16"),
        # One latent frame of a 480p video (30 x 52 tokens), a small fine-tuning step.
        _attention("one_frame_train", "train", B=1, H=40, Hkv=40, Lq=1560, Lk=1560, D=128, dtype="bf16"),
        # Video tokens attend to text tokens: few keys under very many rows.
        _attention("cross_train", "train", B=1, H=40, Hkv=40, Lq=32760, Lk=512, D=128, dtype="bf16"),
        # A causal generator over frames, key heads shared by four.
        _attention("causal_train", "train", B=1, H=16, Hkv=4, Lq=8192, Lk=8192, D=128, dtype="bf16", causal=True),
        # A padded batch of joint text and image sequences, one entry shorter than the other, and one without any key.
        _attention("padded_train_fp16", "train", B=3, H=24, Hkv=24, Lq=4352, Lk=4352, D=128, dtype="fp16", lens=True),
        # Head size 64, odd lengths, queries and keys of different sequences; evaluation without gradients.
        _attention("d64_odd_fwd", "fwd", B=2, H=12, Hkv=12, Lq=5003, Lk=7001, D=64, dtype="fp16"),
        # 14B video model at 480p, half of its heads: the largest step.
        _attention("video_480p_train", "train", B=1, H=20, Hkv=20, Lq=32760, Lk=32760, D=128, dtype="bf16"),
        # A few tokens of a wide model, no gradients: latency.
        _norm("few_tokens_fwd", "fwd", B=2, L=32, C=8192, x="bf16", y="bf16", norm="rms", post="rms", vectors="fp32"),
        # The 14B video model's rows at 480p: gate, layer norm and modulation of a diffusion block, forward and backward.
        _norm("video_rows_train", "train", B=1, L=32760, C=5120, x="bf16", y="bf16", norm="layer", post=None, vectors="fp32"),
        # The residual stream kept in fp32, two samples, no gradients.
        _norm("fp32_stream_fwd", "fwd", B=2, L=4352, C=5120, x="fp32", y="bf16", norm="layer", post=None, vectors="fp32"),
        # Norms before and after the part, rows of an odd width, 16-bit vectors.
        _norm("sandwich_odd_train", "train", B=3, L=2777, C=1153, x="fp16", y="fp16", norm="rms", post="rms", vectors="fp16"),
    ]


def _attention(name, mode, **sizes):
    return dict(name=name, op="attention", mode=mode, **{"causal": False, "lens": False, **sizes})


def _norm(name, mode, **sizes):
    return dict(name=name, op="residual_norm", mode=mode, **sizes)


def _log_int(rng, lo, hi):
    """An integer spread evenly over its logarithm; odd as often as even."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    mode = rng.choice(("train", "train", "fwd"))
    if rng.random() < 0.4:
        narrow = rng.random() < 0.5
        case = dict(op="residual_norm", mode=mode, B=rng.choice((1, 1, 2, 3, 5)), L=_log_int(rng, 1, 32760),
                    C=_log_int(rng, 64, 1024) * (1 if narrow else 8), x=rng.choice(("bf16", "bf16", "fp16", "fp32")), y="",
                    norm=rng.choice(("layer", "rms")), post=rng.choice((None, None, "rms", "layer")), vectors="")
        case["y"] = case["x"] if case["x"] != "fp32" else rng.choice(("bf16", "fp32"))
        case["vectors"] = rng.choice(("fp32", case["y"]))
        while case["B"] * case["L"] * case["C"] > 32760 * 5120:
            case["L"] = max(1, case["L"] * 9 // 10)
        return case
    hq = rng.choice((1, 8, 12, 16, 24, 32, 40, 64))
    kind = rng.choice(("self", "self", "cross", "few"))
    lq = {"self": _log_int(rng, 32, 32760), "cross": _log_int(rng, 64, 32760), "few": _log_int(rng, 1, 200)}[kind]
    lk = {"self": lq, "cross": _log_int(rng, 33, 1024), "few": _log_int(rng, 100, 75600)}[kind]
    case = dict(op="attention", mode=mode, B=rng.choice((1, 1, 2, 3)), H=hq, Hkv=hq // rng.choice([g for g in (1, 1, 2, 4, 5) if hq % g == 0]),
                Lq=lq, Lk=lk, D=rng.choice((128, 128, 64)), dtype=rng.choice(("bf16", "bf16", "fp16")),
                causal=kind == "self" and rng.random() < 0.4, lens=rng.random() < 0.3)
    while work(case)["flops"] > 3e13:
        case["Lq"], case["Lk"] = (max(1, n * 9 // 10) for n in (case["Lq"], case["Lk"]))
    return case


def _batch_lens(case):
    """Key and query counts of a padded batch: the first entry is full, the others shorter, the third has no keys at all."""
    share = (1.0, 0.62, 0.35)
    lens = [[max(1, int(n * share[b])) for b in range(case["B"])] for n in (case["Lk"], case["Lq"])]
    if case["B"] == 3:
        lens[0][2] = 0
    return lens


def _values(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    train = case["mode"] == "train"
    state = dict(op=case["op"], train=train)
    if case["op"] == "attention":
        B, H, Hkv, Lq, Lk, D, dtype = (case[n] for n in ("B", "H", "Hkv", "Lq", "Lk", "D", "dtype"))
        dtype = DTYPES[dtype]
        state["q"] = _values(g, (B, Lq, H, D), dtype).requires_grad_(train)
        # keys as a model has them, off zero by an amount of each head's channel
        k = _values(g, (B, Lk, Hkv, D), torch.float32) + torch.randn((Hkv, D), generator=g, device=DEVICE)
        state["k"] = k.to(dtype).requires_grad_(train)
        state["v"] = _values(g, (B, Lk, Hkv, D), dtype).requires_grad_(train)
        if train:
            state["do"] = _values(g, (B, Lq, H, D), dtype)
        state["causal"], state["k_lens"], state["q_lens"] = case["causal"], None, None
        if case["lens"]:
            state["k_lens"], state["q_lens"] = (torch.tensor(n, dtype=torch.int32, device=DEVICE) for n in _batch_lens(case))
        return state
    B, L, C = case["B"], case["L"], case["C"]
    xt, yt, vt = DTYPES[case["x"]], DTYPES[case["y"]], DTYPES[case["vectors"]]
    state["norm"], state["post"] = case["norm"], case["post"]
    state["residual_scale"] = 1.0 if case["post"] is None else 0.5 ** 0.5

    def vector(shape, std, mean=0.0):
        return (mean + std * torch.randn(shape, generator=g, device=DEVICE)).to(vt).requires_grad_(train)

    leaves = {"x": _values(g, (B, L, C), xt, 3.0).requires_grad_(train), "y": _values(g, (B, L, C), yt).requires_grad_(train),
              "gate": vector((B, 1, C), 0.3, 0.5), "scale": vector((B, 1, C), 0.3), "shift": vector((B, 1, C), 0.3)}
    if case["post"] is not None:
        leaves["post_weight"] = vector((C,), 0.2, 1.0)
    if case["norm"] == "rms":
        leaves["weight"] = vector((C,), 0.2, 1.0)
    state["leaves"] = leaves
    if train:
        state["dh"], state["dn"] = _values(g, (B, L, C), xt), _values(g, (B, L, C), yt)
    return state


# ------------------------------------------------------------------------------------------------ the calls

def run(state):
    if state["op"] == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    return _norm_own(state) if own else _norm_plain(state)


def _attention_own(state):
    from ksanadit_amd import train_ops

    q, k, v = state["q"], state["k"], state["v"]
    o = train_ops.attention(q, k, v, is_causal=state["causal"], k_lens=state["k_lens"], q_lens=state["q_lens"])
    if not state["train"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), state["do"]))


def _norm_own(state):
    from ksanadit_amd import train_ops

    leaves = state["leaves"]
    h, n = train_ops.residual_norm(**leaves, norm=state["norm"], post_norm=state["post"], residual_scale=state["residual_scale"],
                                   eps=EPS)
    if not state["train"]:
        return h, n
    grads = torch.autograd.grad((h, n), list(leaves.values()), (state["dh"], state["dn"]))
    return {"h": h.detach(), "n": n.detach(), **dict(zip(leaves, grads))}


# ------------------------------------------------------------------------------------------------ the plain forms

#: scores that the plain form holds at a time
_SCORES = 1 << 28


def _attention_plain(state):
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    group, scale, train = H // Hkv, D ** -0.5, state["train"]
    heads = max(1, min(Hkv, _SCORES // (group * Lq * Lk)))
    rows = max(1, min(Lq, _SCORES // (heads * group * Lk)))
    o = torch.empty_like(q)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v)) if train else (None, None, None)
    key = torch.arange(Lk, device=q.device)
    for b in range(B):
        for h in range(0, Hkv, heads):
            n = min(heads, Hkv - h)
            own_heads = slice(h * group, (h + n) * group)
            kf = k[b, :, h : h + n].float().permute(1, 2, 0).contiguous()  # [n, D, Lk]
            vf = v[b, :, h : h + n].float().transpose(0, 1).contiguous()  # [n, Lk, D]
            if train:
                kt, vt = kf.transpose(1, 2).contiguous(), vf.transpose(1, 2).contiguous()
                gk, gv = torch.zeros_like(kt), torch.zeros_like(vf)
            for r in range(0, Lq, rows):
                m = min(rows, Lq - r)

                def heads_first(t):  # rows of the heads that share a key head stand below each other
                    return t[b, r : r + m, own_heads].float().transpose(0, 1).reshape(n, group * m, D)

                def rows_first(t):
                    return t.reshape(n * group, m, D).transpose(0, 1).to(q.dtype)

                qf = heads_first(q)
                row = torch.arange(r, r + m, device=q.device).repeat(group).unsqueeze(1)
                seen = key.unsqueeze(0) <= row if state["causal"] else None
                if state["k_lens"] is not None:
                    within = (key.unsqueeze(0) < state["k_lens"][b]) & (row < state["q_lens"][b])
                    seen = within if seen is None else seen & within
                p = torch.matmul(qf, kf).mul_(scale)
                if seen is not None:
                    p.masked_fill_(~seen, -math.inf)
                top = p.amax(-1, keepdim=True)
                top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                p = p.sub_(top).exp_()
                total = p.sum(-1, keepdim=True)
                p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
                of = torch.matmul(p, vf)
                o[b, r : r + m, own_heads] = rows_first(of)
                if train:
                    do = heads_first(state["do"])
                    gv += torch.matmul(p.transpose(1, 2), do)
                    ds = torch.matmul(do, vt)
                    ds = ds.sub_((do * of).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                    dq[b, r : r + m, own_heads] = rows_first(torch.matmul(ds, kt))
                    gk += torch.matmul(ds.transpose(1, 2), qf)
            if train:
                dk[b, :, h : h + n] = gk.transpose(0, 1).to(k.dtype)
                dv[b, :, h : h + n] = gv.transpose(0, 1).to(v.dtype)
    return (o, dq, dk, dv) if train else o


def _normed(t, kind):
    """(t's rows normalised, what they were multiplied with)"""
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    inv = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    return t * inv, inv


def _normed_backward(g, hat, inv, kind):
    out = g - hat * (g * hat).mean(-1, keepdim=True)
    if kind == "layer":
        out = out - g.mean(-1, keepdim=True)
    return out * inv


def _norm_plain(state):
    leaves = {name: t.detach() for name, t in state["leaves"].items()}
    x, y = leaves["x"].float(), leaves["y"].float()
    gate, scale, shift = (leaves[n].float() for n in ("gate", "scale", "shift"))
    weight = leaves["weight"].float() if "weight" in leaves else 1.0
    r = state["residual_scale"]
    u = y
    if state["post"] is not None:
        y_hat, y_inv = _normed(y, state["post"])
        u = y_hat * leaves["post_weight"].float()
    h = x * r + gate * u
    hat, inv = _normed(h, state["norm"])
    n = hat * weight * (1.0 + scale) + shift
    out = {"h": h.to(leaves["x"].dtype), "n": n.to(leaves["y"].dtype)}
    if not state["train"]:
        return out["h"], out["n"]
    dn = state["dn"].float()
    dh = state["dh"].float() + _normed_backward(dn * weight * (1.0 + scale), hat, inv, state["norm"])
    grads = {"x": dh * r, "gate": (dh * u).sum(1, keepdim=True), "scale": (dn * hat * weight).sum(1, keepdim=True),
             "shift": dn.sum(1, keepdim=True)}
    du = dh * gate
    if state["post"] is not None:
        grads["post_weight"] = (du * y_hat).sum((0, 1))
        du = _normed_backward(du * leaves["post_weight"].float(), y_hat, y_inv, state["post"])
    grads["y"] = du
    if "weight" in leaves:
        grads["weight"] = (dn * (1.0 + scale) * hat).sum((0, 1))
    return {**out, **{name: grads[name].to(t.dtype) for name, t in leaves.items()}}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return _attention_exact(state) if case["op"] == "attention" else _norm_exact(state)


def _attention_exact(state):
    """Row block by row block of one head, differentiated by torch."""
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    train, group, (B, Lq, H, D) = state["train"], q.shape[2] // k.shape[2], q.shape
    Lk = k.shape[1]
    out = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in ((q, q, k, v) if train else (q,))]
    counts = [[Lk] * B, [Lq] * B] if state["k_lens"] is None else [state[n].tolist() for n in ("k_lens", "q_lens")]
    step = max(1, (1 << 27) // Lk)
    for b in range(B):
        keys, rows = counts[0][b], counts[1][b]
        for h in range(H if keys else 0):
            kd, vd = (t[b, :keys, h // group].double().requires_grad_(train) for t in (k, v))
            for r in range(0, rows, step):
                e = min(rows, r + step)
                qd = q[b, r:e, h].double().requires_grad_(train)
                with torch.set_grad_enabled(train):
                    scores = torch.mm(qd, kd.t()) / math.sqrt(D)
                    if state["causal"]:
                        hidden = torch.ones((e - r, keys), dtype=torch.bool, device=q.device).triu(r + 1)
                        scores = scores.masked_fill(hidden, -math.inf)
                    weights = (scores - scores.logsumexp(1, keepdim=True)).exp()
                    result = torch.mm(weights, vd)
                out[0][b, r:e, h] = result.detach()
                if train:
                    gq, gk, gv = torch.autograd.grad(result, (qd, kd, vd), state["do"][b, r:e, h].double())
                    out[1][b, r:e, h] = gq
                    out[2][b, :keys, h // group] += gk
                    out[3][b, :keys, h // group] += gv
    return tuple(out) if train else out[0]


def _norm_exact(state):
    """Batch entry by batch entry, differentiated by torch."""
    train = state["train"]
    leaves = {name: t.detach().double().requires_grad_(train) for name, t in state["leaves"].items()}

    def normed(t, kind):
        if kind == "layer":
            return (t - t.mean(-1, keepdim=True)) / (t.var(-1, keepdim=True, unbiased=False) + EPS).sqrt()
        return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt()

    results, sums = [], {name: torch.zeros_like(t) for name, t in leaves.items()} if train else None
    for b in range(leaves["x"].shape[0]):
        one = {name: t.detach()[b : b + 1].requires_grad_(train) if t.dim() == 3 else t for name, t in leaves.items()}
        with torch.set_grad_enabled(train):
            u = one["y"] if state["post"] is None else normed(one["y"], state["post"]) * one["post_weight"]
            h = one["x"] * state["residual_scale"] + one["gate"] * u
            n = normed(h, state["norm"]) * one.get("weight", 1.0) * (1 + one["scale"]) + one["shift"]
        results.append((h.detach(), n.detach()))
        if train:
            grads = torch.autograd.grad((h, n), list(one.values()), (state["dh"][b : b + 1].double(), state["dn"][b : b + 1].double()))
            for name, grad in zip(one, grads):
                if leaves[name].dim() == 3:
                    sums[name][b : b + 1] = grad
                else:
                    sums[name] += grad
    h, n = (torch.cat(t) for t in zip(*results))
    return {"h": h, "n": n, **sums} if train else (h, n)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    """Operations: a multiply-add counts as 2.  Attention: two products over the pairs of tokens that take part, five more in
    its backward pass.  Bytes: every input read once and every output written once, of padded batches the rows that exist."""
    train = case["mode"] == "train"
    if case["op"] == "attention":
        B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
        k_lens, q_lens = _batch_lens(case) if case["lens"] else ([case["Lk"]] * B, [case["Lq"]] * B)
        pairs = 0
        for nk, nq in zip(k_lens, q_lens):
            below = min(nk, nq)
            pairs += below * (below + 1) // 2 + max(0, nq - nk) * nk if case["causal"] else nk * nq
        rows_q, rows_k = sum(n for n, m in zip(q_lens, k_lens) if m) * H * D, sum(k_lens) * Hkv * D
        written = B * case["Lq"] * H * D
        nbytes = 2.0 * (rows_q + 2 * rows_k + written)
        if train:
            nbytes += 2.0 * (rows_q + written + 2 * B * case["Lk"] * Hkv * D)
        return {"bytes": nbytes, "flops": (14.0 if train else 4.0) * pairs * H * D}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    n, sx, sy, sv = case["B"] * case["L"] * case["C"], size[case["x"]], size[case["y"]], size[case["vectors"]]
    vectors = (3 * case["B"] + (case["norm"] == "rms") + (case["post"] is not None)) * case["C"] * sv
    # forward: x, y in, h, n out; backward besides: dh, dn in, dx, dy out, the vectors' gradients
    return {"bytes": float((4 if train else 2) * n * (sx + sy) + (2 if train else 1) * vectors), "flops": (50.0 if train else 16.0) * n}
