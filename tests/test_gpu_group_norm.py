"""Group norm with an activation on an MI355X, forward and backward, against 64-bit statements, with tolerances
that follow the arithmetic: u = 2^-24 is half a step of fp32; a lane adds at most 256 values in fp32 before
its sums become doubles."""
import numpy as np
import pytest
import torch

import stream_ops_oracle as S

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # of a 16-bit result's storage
HALF_STEP_SUBNORMAL = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def f64(t):
    return t.detach().cpu().double().numpy()


def no_error(sa):
    assert sa.sideaware_last_error() == "", sa.sideaware_last_error()


def make(N, P, C, dtype, wtype, seed=0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, P, C, generator=g) * 1.5 + torch.randn(C, generator=g) + offset).to(dtype)
    w, b = (1 + 0.3 * torch.randn(C, generator=g)).to(wtype), (0.3 * torch.randn(C, generator=g)).to(wtype)
    return x, w, b, torch.randn(N, P, C, generator=g).to(dtype)


def grouped(a, G):
    N, P, C = a.shape
    return a.reshape(N, P, G, C // G)


def check_forward(y, stats, x, w, b, G, eps, activation):
    """Tolerances.  A lane's sums of d = x - pivot and d^2 over at most 256 pixels and then the 8 channels of a vector,
    L = 264 at most, are off by L u of the sums of the magnitudes, and |d| <= 2 D where D is the largest |x - mean| of the group; the mean is off by that and by its
    rounding, the variance by (L + 4) u (2 D)^2 / var of itself, 1/sqrt of it by half as much."""
    X, W, B = f64(x), 1.0 if w is None else f64(w), 0.0 if b is None else f64(b)
    N, P, C = X.shape
    want, want_stats = S.group_norm(X, W, B, G, float(np.float32(eps)), activation)
    mean, rstd = want_stats[..., 0], want_stats[..., 1]
    L = min(P, 256) + 8
    D = np.abs(grouped(X, G) - mean[:, None, :, None]).max((1, 3))
    e_mean = U * np.abs(mean) + L * U * 2 * D
    e_rstd = rstd * ((L / 2 + 4) * U * (2 * D * rstd) ** 2 + 4 * U)
    got = f64(stats)
    assert np.all(np.abs(got[..., 0] - mean) <= e_mean)
    assert np.all(np.abs(got[..., 1] - rstd) <= e_rstd)
    h = (grouped(X, G) - mean[:, None, :, None]) * rstd[:, None, :, None]
    e_h = (np.abs(h) * (e_rstd / rstd)[:, None, :, None] + (rstd * e_mean)[:, None, :, None] + 3 * U * np.abs(h)).reshape(N, P, C)
    z = h.reshape(N, P, C) * W + B
    e_z = np.abs(W) * e_h + 3 * U * (np.abs(h.reshape(N, P, C) * W) + np.abs(B))
    # silu's slope is at most 1.1; its own exponential, sum, reciprocal and product: (|z| + 8) u of the result
    e = e_z if activation == "none" else 1.1 * e_z + (np.abs(z) + 8) * U * np.abs(want)
    tol = e + HALF_STEP[x.dtype] * 1.01 * np.abs(want) + HALF_STEP_SUBNORMAL[x.dtype] + U * np.abs(want)
    off = np.abs(f64(y) - want)
    worst = np.unravel_index(int((off - tol).argmax()), off.shape)
    assert np.all(off <= tol), (worst, off[worst], tol[worst], want[worst])


def check_backward(got, dout, x, w, b, stats, G, activation):
    """Tolerances: h takes three roundings, z two more; silu's derivative s (1 + z (1 - s)) has the error of s,
    (|z| + 8) u, in both places and a slope of at most 0.5 in z; sums of at most 256 values in fp32, then doubles."""
    X, GR, ST = f64(x), f64(dout), f64(stats)
    W, B = 1.0 if w is None else f64(w), 0.0 if b is None else f64(b)
    N, P, C = X.shape
    dx, dw, db = S.group_norm_backward(GR, X, W, B, ST, G, activation)
    mean, rstd = ST[:, None, :, None, 0], ST[:, None, :, None, 1]
    h = ((grouped(X, G) - mean) * rstd).reshape(N, P, C)
    e_h = 3 * U * np.abs(h)
    z = h * W + B
    if activation == "silu":
        e_z = np.abs(W) * e_h + 2 * U * (np.abs(h * W) + np.abs(B))
        f = S.sigmoid(z) * (1 + z * S.sigmoid(-z))
        e_dz = np.abs(GR) * (0.5 * e_z + 2 * U * (np.abs(z) + 10) * (1 + np.abs(z)) + 2 * U)
        dz = GR * f
    else:
        e_dz, dz = np.zeros_like(X), GR
    L = min(P, 256)
    e_p = (e_dz + L * U * np.abs(dz)).sum(1)                              # (N, C)
    e_q = (e_dz * np.abs(h) + np.abs(dz) * e_h + (L + 1) * U * np.abs(dz * h)).sum(1)
    M = P * (C // G)
    c1 = grouped(dz * W, G).sum((1, 3)) / M
    c2 = grouped(dz * W * h, G).sum((1, 3)) / M
    aw = np.abs(W) * np.ones(C)
    spread = lambda t: np.repeat(t, C // G, axis=-1)[:, None, :]          # noqa: E731
    e_c1 = (e_p * aw).reshape(N, G, -1).sum(-1) / M + 2 * U * np.abs(c1)
    e_c2 = (e_q * aw).reshape(N, G, -1).sum(-1) / M + 2 * U * np.abs(c2)
    r = spread(ST[..., 1])
    e = r * (aw * e_dz + 4 * U * (np.abs(W * dz) + np.abs(spread(c1)) + np.abs(h * spread(c2))) + spread(e_c1) + np.abs(h) * spread(e_c2)
             + e_h * np.abs(spread(c2)))
    tol = e + (HALF_STEP[x.dtype] * 1.01 + U) * np.abs(dx) + HALF_STEP_SUBNORMAL[x.dtype]
    off = np.abs(f64(got[0]) - dx)
    worst = np.unravel_index(int((off - tol).argmax()), off.shape)
    assert np.all(off <= tol), (worst, off[worst], tol[worst], dx[worst])
    for grad, param, want, err in ((got[1], w, dw, e_q.sum(0)), (got[2], b, db, e_p.sum(0))):
        if param is None:
            assert grad is None
            continue
        assert grad.dtype == param.dtype
        # the channels' sums of each row of the workspace are rounded to fp32 once more (and added up there, for a
        # workgroup with several samples)
        err = err + 4 * U * np.abs(want) + (N + 1) * U * (np.abs(dz).sum((0, 1)) if want is db else np.abs(dz * h).sum((0, 1)))
        tol = err + (HALF_STEP[param.dtype] * 1.01 + U) * np.abs(want) + HALF_STEP_SUBNORMAL[param.dtype]
        assert np.all(np.abs(f64(grad) - want) <= tol)


SHAPES = [
    # N, pixels, C, G: one launch (small) and two (chunks), groups that split vectors, odd rows, one group, one
    # channel per group, several samples per workgroup, wide rows cut into slabs and slices
    (1, 1, 8, 1), (2, 1, 64, 8), (3, 5, 30, 10), (2, 64, 1280, 32), (1, 7, 33, 11), (2, 100, 7, 1), (4, 9, 48, 48), (3, 1024, 24, 4),
    (1, 4096, 320, 32), (2, 5003, 96, 8), (1, 3000, 1029, 3), (2, 333, 8200, 1), (1, 2, 20000, 4), (1, 40000, 1, 1), (700, 3, 16, 2),
    (1, 30011, 40, 4), (2, 2048, 2560, 32), (5000, 1, 8, 2), (1, 70000, 12, 3),
    (2, 6001, 128, 32), (1, 20000, 64, 64), (3, 1369, 1152, 24), (20, 1024, 64, 4)]


@pytest.mark.parametrize("N,P,C,G", SHAPES)
def test_group_norm(sa, N, P, C, G):
    from l2_torch_alloc_amd import ops
    for at, dtype in enumerate((torch.bfloat16, torch.float16, torch.float32)):
        if P * (C // G) < 4 and dtype != torch.float32:
            continue
        activation = ("silu", "none", "silu")[at] if (N + P) % 2 else ("none", "silu", "silu")[at]
        wtype = dtype if at == 1 else torch.float32
        x, w, b, dout = make(N, P, C, dtype, wtype, seed=P + C)
        xd, wd, bd, gd = x.cuda(), w.cuda(), b.cuda(), dout.cuda()
        y, stats = ops.group_norm_forward(xd, wd, bd, G, activation=activation)
        check_forward(y, stats, x, w, b, G, 1e-5, activation)
        got = ops.group_norm_backward(gd, xd, wd, bd, stats, G, activation=activation)
        check_backward(got, dout, x, w, b, stats, G, activation)
        # the same call gives the same bits, in place too
        y2, stats2 = ops.group_norm_forward(xd.clone(), wd, bd, G, activation=activation)
        assert torch.equal(y, y2) and torch.equal(stats, stats2)
        x3 = xd.clone()
        assert ops.group_norm_forward(x3, wd, bd, G, activation=activation, out=x3)[0] is x3 and torch.equal(x3, y)
        g3 = gd.clone()
        again = ops.group_norm_backward(g3, xd, wd, bd, stats, G, activation=activation, out=g3)
        assert again[0] is g3 and all(torch.equal(p, q) for p, q in zip(got, again))
        x4 = xd.clone()
        again = ops.group_norm_backward(gd, x4, wd, bd, stats, G, activation=activation, out=x4)
        assert again[0] is x4 and all(torch.equal(p, q) for p, q in zip(got, again))
    no_error(sa)


@pytest.mark.parametrize("P", [20, 6000])
def test_without_weight_or_bias(sa, P):
    from l2_torch_alloc_amd import ops
    x, w, b, dout = make(2, P, 48, torch.float32, torch.float32, seed=3)
    for ww, bb in ((None, None), (w, None), (None, b)):
        dev = lambda t: None if t is None else t.cuda()              # noqa: E731
        y, stats = ops.group_norm_forward(x.cuda(), dev(ww), dev(bb), 6, activation="silu")
        check_forward(y, stats, x, ww, bb, 6, 1e-5, "silu")
        check_backward(ops.group_norm_backward(dout.cuda(), x.cuda(), dev(ww), dev(bb), stats, 6, activation="silu"), dout, x, ww, bb, stats, 6, "silu")
    no_error(sa)


@pytest.mark.parametrize("P", [50, 9000])
def test_mean_far_from_zero(sa, P):
    from l2_torch_alloc_amd import ops
    for dtype, offset in ((torch.float32, 3000.0), (torch.bfloat16, 100.0), (torch.float16, -300.0)):
        x, w, b, dout = make(2, P, 64, dtype, torch.float32, seed=4, offset=offset)
        y, stats = ops.group_norm_forward(x.cuda(), w.cuda(), b.cuda(), 8)
        check_forward(y, stats, x, w, b, 8, 1e-5, "none")
        check_backward(ops.group_norm_backward(dout.cuda(), x.cuda(), w.cuda(), b.cuda(), stats, 8), dout, x, w, b, stats, 8, "none")
    no_error(sa)


def test_constant_group_and_outlier(sa):
    from l2_torch_alloc_amd import ops
    for P in (30, 8000):
        x, w, b, _ = make(1, P, 16, torch.float32, torch.float32, seed=6)
        x[..., :4] = 2.5                                                  # no spread: 1/sqrt(eps)
        x[0, 0, 5] = 3e4                                                  # the first pixel far from all others
        y, stats = ops.group_norm_forward(x.cuda(), w.cuda(), b.cuda(), 4)
        check_forward(y, stats, x, w, b, 4, 1e-5, "none")
        assert float(stats[0, 0, 0]) == 2.5 and torch.equal(y[..., :4].cpu(), b[:4].expand(1, P, 4))
    no_error(sa)


def test_nonfinite_values_stay_in_their_group(sa):
    from l2_torch_alloc_amd import ops
    for P in (30, 8000):
        x, w, b, dout = make(2, P, 24, torch.bfloat16, torch.float32, seed=7)
        x[0, 3, 7] = float("inf")
        x[1, P - 1, 20] = float("nan")
        y, stats = ops.group_norm_forward(x.cuda(), w.cuda(), b.cuda(), 4, activation="silu")
        bad = torch.zeros(2, 4, dtype=torch.bool)
        bad[0, 1] = bad[1, 3] = True
        fine = torch.isfinite(y.cpu().float()).view(2, P, 4, 6).all(3).all(1)
        assert torch.equal(fine, ~bad)
        assert not bool(torch.isfinite(stats[..., 1].cpu())[bad].any() and torch.isfinite(stats[..., 0].cpu())[bad].any())
        dx, dw, db = ops.group_norm_backward(dout.cuda(), x.cuda(), w.cuda(), b.cuda(), stats, 4, activation="silu")
        assert torch.equal(torch.isfinite(dx.cpu().float()).view(2, P, 4, 6).all(3).all(1), ~bad)
    no_error(sa)


def test_writes_nothing_outside(sa):
    from l2_torch_alloc_amd import ops
    for N, P, C, G in ((1, 5, 33, 11), (2, 3001, 31, 1), (3, 100, 40, 4)):
        n = N * P * C
        x, w, b, dout = (t.cuda() for t in make(N, P, C, torch.bfloat16, torch.bfloat16))
        out = torch.full((n + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
        stats = torch.full((N * G * 2 + 16,), 9.0, device="cuda")
        for backward in (False, True):
            need = ops.group_norm_workspace(x, G, backward)
            ws = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
            if not backward:
                ops.group_norm_forward(x, w, b, G, out=out[:n].view(N, P, C), stats=stats[:N * G * 2].view(N, G, 2), workspace=ws[:need])
            else:
                par = torch.full((2, C + 16), 9.0, dtype=torch.bfloat16, device="cuda")
                ops.group_norm_backward(dout, x, w, b, stats[:N * G * 2].view(N, G, 2), G, out=out[:n].view(N, P, C), dweight=par[0, :C], dbias=par[1, :C],
                                        workspace=ws[:need])
                assert bool((par[:, C:] == 9).all()) and bool(torch.isfinite(par.float()).all())
            assert bool((ws[need:] == 77).all()) and bool((out[n:] == 9).all()) and bool((stats[N * G * 2:] == 9).all())
    no_error(sa)


def test_graphs_with_workspaces_of_their_own(sa):
    """Forward and backward captured into two graphs, replayed in turn with eager calls between, each replay
    against the eager result."""
    from l2_torch_alloc_amd import ops
    jobs = []
    for seed, (N, P, C, G) in enumerate(((2, 64, 320, 32), (2, 4096, 320, 32))):
        x, w, b, dout = (t.cuda() for t in make(N, P, C, torch.bfloat16, torch.float32, seed=seed))
        kept = dict(out=torch.empty_like(x), stats=torch.empty(N, G, 2, device="cuda"),
                    workspace=torch.empty(max(1, ops.group_norm_workspace(x, G)), dtype=torch.uint8, device="cuda"))
        kept_b = dict(out=torch.empty_like(x), dweight=torch.empty_like(w), dbias=torch.empty_like(b),
                      workspace=torch.empty(max(1, ops.group_norm_workspace(x, G, True)), dtype=torch.uint8, device="cuda"))

        def step(x=x, w=w, b=b, dout=dout, G=G, kept=kept, kept_b=kept_b):
            ops.group_norm_forward(x, w, b, G, activation="silu", **kept)
            ops.group_norm_backward(dout, x, w, b, kept["stats"], G, activation="silu", **kept_b)
        step()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            step()
        jobs.append((graph, x, w, b, dout, G, kept, kept_b))
    for turn in range(3):
        for graph, x, w, b, dout, G, kept, kept_b in jobs:
            x.mul_(1.1).add_(0.1)
            graph.replay()
            torch.cuda.synchronize()
            y, stats = ops.group_norm_forward(x, w, b, G, activation="silu")
            grads = ops.group_norm_backward(dout, x, w, b, stats, G, activation="silu")
            assert torch.equal(kept["out"], y) and torch.equal(kept["stats"], stats)
            assert all(torch.equal(p, q) for p, q in zip(grads, (kept_b["out"], kept_b["dweight"], kept_b["dbias"])))
    no_error(sa)


def test_streams_side_by_side(sa):
    from l2_torch_alloc_amd import ops
    inputs = [[t.cuda() for t in make(1, 20000 + 8 * i, 64, torch.bfloat16, torch.float32, seed=i)] for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    results = []
    for (x, w, b, dout), stream in zip(inputs, streams):
        with torch.cuda.stream(stream):
            y, stats = ops.group_norm_forward(x, w, b, 8, activation="silu")
            results.append((y, stats) + ops.group_norm_backward(dout, x, w, b, stats, 8, activation="silu"))
    torch.cuda.synchronize()
    for (x, w, b, dout), result in zip(inputs, results):
        y, stats = ops.group_norm_forward(x, w, b, 8, activation="silu")
        want = (y, stats) + ops.group_norm_backward(dout, x, w, b, stats, 8, activation="silu")
        assert all(torch.equal(p, q) for p, q in zip(result, want))
    no_error(sa)


def test_array_past_four_gib(sa):
    """Offsets past 32 bits: the last sample's rows lie behind 4 GiB."""
    from l2_torch_alloc_amd import ops
    N, P, C, G = 3, 1 << 20, 768, 32
    x = torch.zeros(N, P, C, dtype=torch.bfloat16, device="cuda")
    x[2] = torch.randn(P, C, device="cuda").to(torch.bfloat16) + 1
    y, stats = ops.group_norm_forward(x, None, None, G)
    v = x[2].float().view(P, G, C // G)
    mean = v.double().mean((0, 2))
    var = ((v - mean.float()[None, :, None]).square()).double().mean((0, 2))
    assert float((stats[2, :, 0].double() - mean).abs().max()) <= 1e-5
    assert float((stats[2, :, 1].double() * (var + 1e-5).sqrt() - 1).abs().max()) <= 1e-5
    tail = ((x[2, -100:].double().view(100, G, -1) - mean[None, :, None]) / (var + 1e-5).sqrt()[None, :, None]).view(100, C)
    # bf16 storage, and 1e-5 of the values for the statistics
    assert float((y[2, -100:].double() - tail).abs().max()) <= float(tail.abs().max()) * (2.0 ** -8 + 3e-5)
    assert bool((y[0] == 0).all()) and float(stats[0].abs()[:, 0].max()) == 0
    del x, y, v
    no_error(sa)


def test_refused(sa):
    from l2_torch_alloc_amd import ops
    lib = sa.library()
    x, w, b, dout = (t.cuda() for t in make(1, 9000, 16, torch.float32, torch.float32))
    with pytest.raises(AssertionError):
        ops.group_norm_forward(x.transpose(1, 2), None, None, 4)
    with pytest.raises(AssertionError):
        ops.group_norm_forward(x.view(-1)[1:-15].view(1, -1, 16), None, None, 4)
    no_error(sa)
    assert ops.group_norm_workspace(x, 4) > 0
    with pytest.raises(RuntimeError, match="workspace"):
        ops.group_norm_forward(x, w, b, 4, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    lib.sideaware_clear_error()
    y = torch.full_like(x, 5.0)
    args = (y.data_ptr(), y.data_ptr(), x.data_ptr(), None, None, 1, 9000, 16, 4, 1e-5)
    for tail in ((9, 0, 1, 0, 0), (0, 9, 1, 0, 0), (0, 0, 1, 0, 0)):     # activation, type, weight type, no workspace
        assert lib.sideaware_group_norm_forward(*args, *tail, -1, None) == -1
        assert sa.sideaware_last_error() != ""
        lib.sideaware_clear_error()
    assert lib.sideaware_group_norm_forward(None, *args[1:], 0, 0, 1, 0, 0, -1, None) == -1
    lib.sideaware_clear_error()
    torch.cuda.synchronize()
    assert bool((y == 5).all())


def test_overlapping_arrays_are_refused(sa):
    """An output may be x or dout, but no other arrays of a call may share memory with what it writes."""
    from l2_torch_alloc_amd import ops
    lib = sa.library()
    n, pixels, channels = 1, 9000, 16
    count = n * pixels * channels
    buf = torch.ones(2 * count + 64, device="cuda")
    shape = (n, pixels, channels)
    x, behind, dout = buf[:count].view(shape), buf[32:count + 32].view(shape), buf[count + 64:].view(shape)
    w, b = torch.ones(channels, device="cuda"), torch.zeros(channels, device="cuda")
    stats = torch.ones(n, 4, 2, device="cuda")
    other = torch.empty_like(x)
    need = ops.group_norm_workspace(x, 4, backward=True)
    assert need > 0
    inside = x.view(-1)[:(need + 3) // 4]
    for call in (lambda: ops.group_norm_forward(x, w, b, 4, out=behind, stats=stats),
                 lambda: ops.group_norm_forward(x, w, b, 4, out=other, stats=x.view(-1)[:8].view(1, 4, 2)),
                 lambda: ops.group_norm_forward(x, w, b, 4, out=other, stats=stats, workspace=inside),
                 lambda: ops.group_norm_forward(x, x.view(-1)[:16], b, 4, out=x, stats=stats),
                 lambda: ops.group_norm_backward(dout, x, w, b, stats, 4, out=behind),
                 lambda: ops.group_norm_backward(dout, x, w, b, stats, 4, out=other, dweight=w),
                 lambda: ops.group_norm_backward(dout, x, w, b, stats, 4, out=other, dweight=b),
                 lambda: ops.group_norm_backward(dout, x, w, b, stats, 4, out=other, dweight=other.view(-1)[:16]),
                 lambda: ops.group_norm_backward(dout, x, w, b, stats, 4, out=other, dweight=buf[-16:], dbias=buf[-16:]),
                 lambda: ops.group_norm_backward(dout, x, w, b, stats, 4, out=other, workspace=inside)):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
        lib.sideaware_clear_error()
    torch.cuda.synchronize()
    assert bool((buf == 1).all()) and bool((w == 1).all()) and bool((b == 0).all()) and bool((stats == 1).all())
    # one tensor as input, gradient and weight and bias of another call is all right
    want = ops.group_norm_backward(x, x, w, w, stats, 4)
    have = ops.group_norm_backward(x, x, w, w, stats, 4, out=x)
    assert all(torch.equal(h, t) for h, t in zip(have, want))
    no_error(sa)


@pytest.mark.parametrize("N,P,C,G,dtype", [(16, 900, 640, 32, torch.bfloat16), (16, 700, 640, 32, torch.float32), (128, 700, 66, 3, torch.float16),
                                           (33, 401, 512, 32, torch.bfloat16), (40, 1024, 640, 32, torch.float16)])
def test_many_samples_in_pieces_of_rows(sa, N, P, C, G, dtype):
    """Workgroups that share memory lines: their numbering over the XCDs, and stores that the L2 puts together."""
    from l2_torch_alloc_amd import ops
    x, w, b, dout = make(N, P, C, dtype, torch.float32, seed=N + P)
    xd, wd, bd, gd = x.cuda(), w.cuda(), b.cuda(), dout.cuda()
    y, stats = ops.group_norm_forward(xd, wd, bd, G, activation="silu")
    check_forward(y, stats, x, w, b, G, 1e-5, "silu")
    check_backward(ops.group_norm_backward(gd, xd, wd, bd, stats, G, activation="silu"), dout, x, w, b, stats, G, "silu")
    again, _ = ops.group_norm_forward(xd, wd, bd, G, activation="silu", out=xd, stats=stats)
    assert torch.equal(again, y)
    no_error(sa)


def test_workspace_does_not_depend_on_tuning(sa):
    from l2_torch_alloc_amd import ops
    lib = sa.library()
    x, w, b, dout = (t.cuda() for t in make(16, 900, 640, torch.bfloat16, torch.float32))
    want, stats = ops.group_norm_forward(x, w, b, 32, activation="silu")
    grads = ops.group_norm_backward(dout, x, w, b, stats, 32, activation="silu")
    before = lib.sideaware_tune_get(b"cache_bytes")
    try:
        for cache in (1 << 16, 1 << 40):
            assert lib.sideaware_tune(b"cache_bytes", cache) == 0
            assert torch.equal(ops.group_norm_forward(x, w, b, 32, activation="silu")[0], want)
            got = ops.group_norm_backward(dout, x, w, b, stats, 32, activation="silu")
            assert all(torch.equal(g, t) for g, t in zip(got, grads))
    finally:
        lib.sideaware_tune(b"cache_bytes", before)
    no_error(sa)
