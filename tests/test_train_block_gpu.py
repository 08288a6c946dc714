"""The operators with gradients as a block uses them: a diffusion block's attention half from its residual stream and back - norm and
modulation, projections, attention, projection, gate and the next norm - against the same block written with torch in 64 bits."""

import pytest
import torch

from ksanadit_amd import train_ops

gpu = pytest.mark.gpu


def block(p, x, ops):
    B, L, C = x.shape
    h, n = ops.norm(x, None, scale=p["s1"], shift=p["t1"])
    q, k, v = (torch.nn.functional.linear(n, p[w]).view(B, L, -1, 64) for w in ("wq", "wk", "wv"))
    a = ops.attention(q, k, v).reshape(B, L, -1)
    y = torch.nn.functional.linear(a, p["wo"])
    return ops.norm(h, y, gate=p["g1"], scale=p["s2"], shift=p["t2"])


class Ours:
    def __init__(self, lens):
        self.lens = lens

    def norm(self, x, y, **vectors):
        return train_ops.residual_norm(x, y, norm="layer", **vectors)

    def attention(self, q, k, v):
        return train_ops.attention(q, k, v, k_lens=self.lens)


class Plain:
    def __init__(self, lens):
        self.lens = lens

    def norm(self, x, y, scale, shift, gate=1.0):
        h = x if y is None else x + gate * y
        mean, var = h.mean(-1, keepdim=True), h.var(-1, keepdim=True, unbiased=False)
        return h, (h - mean) / (var + 1e-6).sqrt() * (1 + scale) + shift

    def attention(self, q, k, v):
        rep = q.shape[2] // k.shape[2]
        q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(rep, 1), v.transpose(1, 2).repeat_interleave(rep, 1)
        hidden = torch.arange(k.shape[2]) >= torch.tensor(self.lens).view(-1, 1)
        s = (q @ k.transpose(2, 3) / 8).masked_fill(hidden.view(len(self.lens), 1, 1, -1), -torch.inf)
        return (s.softmax(-1) @ v).transpose(1, 2)


@gpu
def test_a_blocks_attention_half_forward_and_backward(hip_device):
    B, L, C, lens = 2, 150, 256, [150, 90]
    g = torch.Generator().manual_seed(1)

    def n(*shape, std=1.0):
        return (std * torch.randn(shape, generator=g)).bfloat16()

    p = {"wq": n(256, C, std=C**-0.5), "wk": n(128, C, std=C**-0.5), "wv": n(128, C, std=C**-0.5), "wo": n(C, 256, std=1 / 16),
         **{name: n(B, 1, C, std=0.3) for name in ("s1", "t1", "g1", "s2", "t2")}}
    x, dh, dn = n(B, L, C), n(B, L, C), n(B, L, C)

    def run(move, ops):
        leaves = {k: move(v).requires_grad_() for k, v in {"x": x, **p}.items()}
        outs = block({k: v for k, v in leaves.items() if k != "x"}, leaves["x"], ops)
        return [*outs, *torch.autograd.grad(outs, list(leaves.values()), [move(dh), move(dn)])]

    want = run(lambda t: t.double(), Plain(lens))
    got = run(lambda t: t.to(hip_device), Ours(lens))
    # Every tensor between two operators is rounded to bf16, up to 2^-9 of itself in the mean square (2^-8 / sqrt 3 at most): about ten
    # on the way there and twenty on the way back, their errors independent - the square root of thirty times 2^-8 / sqrt 3, doubled
    # for what a gradient's sums cancel.
    most = 2 * 30**0.5 * 2.0**-8 / 3**0.5
    for a, b in zip(got, want):
        a = a.detach().cpu().double()
        assert (a - b).norm() <= most * b.detach().norm()
