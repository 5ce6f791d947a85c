"""The new ops together, as a layer over an image's tokens uses them in training: group norm and SiLU over (N, H, W, C)
features, projections, rotary positions of two axes on q and k, attention, dropout onto the residual; forward and
gradients against the same layer in 64 bits on the CPU, differentiated by torch.

Tolerance: fp32 throughout.  The longest chain from an input to a gradient passes three products with inner sizes of 64
channels or 48 tokens each way, and about forty further operations: fewer than 500 roundings of u = 2^-24, relative to
the magnitudes of what is added.  The scores lie below 8 in magnitude, and the softmax turns an error of a score into that
share of its result, so an error relative to the scores counts eight times: 500 * 8 u = 2.4e-4 of the largest magnitude in
each tensor."""
import numpy as np
import pytest
import torch

import stream_ops_oracle as S

pytestmark = pytest.mark.gpu

N, H, W, C, HEADS, GROUPS, P = 2, 6, 8, 64, 4, 8, 0.2
SECTIONS = (4, 4)
BOUND = 500 * 8 * 2.0 ** -24


def plain(x, w, b, wq, wk, wv, table, pos, keep):
    """The layer in elementary operations of the type of its inputs."""
    T, d = H * W, C // HEADS
    v = x.view(N, T, GROUPS, C // GROUPS)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(N, T, C) * w + b
    y = z * torch.sigmoid(z)
    axis = torch.tensor(S.pair_axes(SECTIONS, "blocks"))
    row = pos.long()[..., axis]
    cs = table.view(-1, d // 2, 2)[row, torch.arange(d // 2)][:, :, None]

    def rotate(t):
        t = t.view(N, T, HEADS, d // 2, 2)
        return torch.stack([t[..., 0] * cs[..., 0] - t[..., 1] * cs[..., 1], t[..., 1] * cs[..., 0] + t[..., 0] * cs[..., 1]], -1).flatten(-2)

    q, k, vals = rotate(y @ wq), rotate(y @ wk), (y @ wv).view(N, T, HEADS, d)
    return y, q, k, vals, attend(q, k, vals), keep


def attend(q, k, v):
    d = q.shape[-1]
    scores = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1)) / d ** 0.5
    return (scores.softmax(-1) @ v.transpose(1, 2)).transpose(1, 2).reshape(N, H * W, C)


def near(got, want):
    got, want = got.detach().cpu().double(), want.detach().double().reshape(got.shape)
    assert float((got - want).abs().max()) <= BOUND * max(1.0, float(want.abs().max()))


def test_layer(sa):
    from l2_torch_alloc_amd import ops
    g = torch.Generator().manual_seed(0)
    T, d = H * W, C // HEADS
    x, w, b = torch.randn(N, H, W, C, generator=g), 1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
    wq, wk, wv = (torch.randn(C, C, generator=g) / C ** 0.5 for _ in range(3))
    table = ops.freqs_cis_axes_table(SECTIONS, max(H, W), 100.0)
    pos = torch.stack(torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij"), -1).view(1, T, 2).expand(N, T, 2).contiguous().int()
    seed = torch.tensor([17, 4])
    dout = torch.randn(N, T, C, generator=g)

    # 64 bits on the CPU, gradients by torch
    leaves = [t.double().requires_grad_() for t in (x, w, b, wq, wk, wv)]
    threshold = ops.dropout_threshold(P)
    keep = torch.from_numpy((S.dropout_bits(N * T * C, 17, 4) >= threshold).astype(np.float64)).view(N, T, C)
    xt, wt, bt, qt, kt, vt = leaves
    want_y, want_q, want_k, _, want_a, _ = plain(xt.view(N, T, C), wt, bt, qt, kt, vt, table.double(), pos, keep)
    want = xt.view(N, T, C) + want_a * keep * (65536.0 / (65536 - threshold))
    assert float((want_q.detach().transpose(1, 2) @ want_k.detach().permute(0, 2, 3, 1)).abs().max()) / d ** 0.5 < 8.0
    want.backward(dout.double())

    # the layer on the GPU
    X, Wt, Bt, Wq, Wk, Wv, F, Pos, Seed, G = (t.cuda() for t in (x, w, b, wq, wk, wv, table, pos, seed, dout))
    y, stats = ops.group_norm_forward(X, Wt, Bt, GROUPS, activation="silu")
    tokens = y.view(N, T, C)
    q, k, v = ((tokens @ m).view(N, T, HEADS, d) for m in (Wq, Wk, Wv))
    rq, rk = ops.rope_axes_forward_many([q, k], F, Pos, SECTIONS, outs=[torch.empty_like(q), torch.empty_like(k)])
    ql, kl, vl = (t.detach().requires_grad_() for t in (rq, rk, v))
    a = attend(ql, kl, vl)
    out = ops.dropout_forward(a.detach(), P, Seed, residual=X.view(N, T, C))
    near(y, want_y)
    near(rq, want_q)
    near(rk, want_k)
    near(out, want)

    # and back
    a.backward(ops.dropout_backward(G, P, Seed))
    dq, dk = ops.rope_axes_backward_many([ql.grad.contiguous(), kl.grad.contiguous()], F, Pos, SECTIONS)
    grads = [t.reshape(N * T, C) for t in (dq, dk, vl.grad)]
    flat = tokens.reshape(N * T, C)
    dy = sum(gr @ m.t().contiguous() for gr, m in zip(grads, (Wq, Wk, Wv)))
    dx, dw, db = ops.group_norm_backward(dy.view(N, H, W, C), X, Wt, Bt, stats, GROUPS, activation="silu")
    near(dx + G.view(N, H, W, C), xt.grad)
    near(dw, wt.grad)
    near(db, bt.grad)
    for gr, leaf in zip(grads, (qt, kt, vt)):
        near(flat.t().contiguous() @ gr, leaf.grad)
    assert sa.sideaware_last_error() == ""
