"""The multi-axis rotary and dropout ops on an MI355X: against plain 64-bit statements, bit for bit against
the ops with one position where all axes agree, in place and out of place, in graphs, on another stream,
past 2 GiB, and what they refuse."""
import numpy as np
import pytest
import torch

import stream_ops_oracle as S

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half a step below the smallest normal number (a step there no longer shrinks with the value)
HALF_STEP_SUBNORMAL = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def f64(t):
    return t.detach().cpu().double().numpy()


def no_error(sa):
    assert sa.sideaware_last_error() == "", sa.sideaware_last_error()


def rope_inputs(B, T, heads, d, sections, dtype, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    xs = [torch.randn(B, T, h, d, generator=g).to(dtype).cuda() for h in heads]
    table = torch.randn(rows, d, generator=g)
    pos = torch.randint(0, rows, (B, T, len(sections)), generator=g, dtype=torch.int32)
    return xs, table.cuda(), pos.cuda()


def check_rope(got, x, table, pos, sections, half, order, backward):
    B, T, H, d = x.shape
    want = S.rope_axes(f64(x).reshape(B * T, H, d), f64(table), pos.cpu().numpy().reshape(B * T, -1), sections, half, order, backward).reshape(B, T, H, d)
    # two products and a sum in fp32, each off by half a step of at most |x1 c| + |x2 s|; then the storage
    finite = f64(x)[np.isfinite(f64(x))]
    scale = 2 * np.abs(finite).max() * np.abs(f64(table)).max()
    tol = 3 * 2.0 ** -24 * scale + (0 if x.dtype == torch.float32 else HALF_STEP[x.dtype]) * 1.01 * np.abs(want) + HALF_STEP_SUBNORMAL[x.dtype]
    got = f64(got)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.all(np.isnan(want) | (np.abs(got - want) <= tol))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,sections,order,half", [
    (128, (16, 24, 24), "blocks", False), (128, (16, 24, 24), "blocks", True), (128, (24, 20, 20), "turns", False),
    (128, (24, 20, 20), "turns", True), (64, (13, 19), "blocks", True), (64, (16, 16), "turns", False), (72, (12, 24), "blocks", False),
    (256, (50, 50, 28), "turns", True), (512, (200, 56), "blocks", False), (32, (16,), "blocks", True), (16, (3, 4, 1), "turns", True)])
def test_rope_axes(sa, dtype, d, sections, order, half):
    from l2_torch_alloc_amd import ops
    for B, T in ((1, 1), (3, 37)):
        (q, k), table, pos = rope_inputs(B, T, (6, 2), d, sections, dtype, 50, seed=d + T)
        pos[0, 0, -1] = 50                                           # outside the table
        for forward in (True, False):
            f = ops.rope_axes_forward_many if forward else ops.rope_axes_backward_many
            q0, k0 = q.clone(), k.clone()
            outs = f([q, k], table, pos, sections, half=half, order=order, outs=[torch.empty_like(q), torch.empty_like(k)])
            assert torch.equal(q, q0) and torch.equal(k, k0)
            check_rope(outs[0], q, table, pos, sections, half, order, not forward)
            check_rope(outs[1], k, table, pos, sections, half, order, not forward)
            # in place, one tensor at a time: the same bits
            one = ops.rope_axes_forward if forward else ops.rope_axes_backward
            assert one(q0, table, pos, sections, half=half, order=order) is q0
            assert torch.equal(q0.view(torch.uint8), outs[0].view(torch.uint8))
    no_error(sa)


@pytest.mark.parametrize("half", [False, True])
def test_rope_axes_equals_one_position_where_axes_agree(sa, half):
    from l2_torch_alloc_amd import ops
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for sections, order in (((16, 24, 24), "blocks"), ((21, 43), "blocks"), ((24, 20, 20), "turns")):
            (q, k), table, pos = rope_inputs(2, 65, (8, 3), 128, sections, dtype, 200, seed=1)
            same = pos[..., :1].contiguous()
            spread = same.expand(-1, -1, len(sections)).contiguous()
            for backward in (False, True):
                got = (ops.rope_axes_backward if backward else ops.rope_axes_forward)(q, table, spread, sections, out=torch.empty_like(q), half=half, order=order)
                if half:
                    f = ops.rope_half_backward if backward else ops.rope_half_forward
                else:
                    f = ops.rope_backward_heads if backward else ops.rope_forward_heads
                want = f(q, table, out=torch.empty_like(q), positions=same.view(-1))
                assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    no_error(sa)


def test_rope_axes_backward_is_the_gradient(sa):
    """<dout, R x'> - <dout, R x> against <R^T dout, x' - x>: the op is linear, so differences are exact up to
    rounding (products of 64-bit sums of fp32 outputs, each output off by at most 3 * 2^-24 * scale)."""
    from l2_torch_alloc_amd import ops
    sections = (24, 20, 20)
    (x, dx_in), table, pos = rope_inputs(2, 30, (4, 4), 128, sections, torch.float32, 64, seed=4)
    dout = torch.randn_like(x)
    for half, order in ((False, "blocks"), (True, "turns")):
        kw = dict(half=half, order=order)
        y0 = ops.rope_axes_forward(x, table, pos, sections, out=torch.empty_like(x), **kw)
        y1 = ops.rope_axes_forward(x + dx_in, table, pos, sections, out=torch.empty_like(x), **kw)
        grad = ops.rope_axes_backward(dout, table, pos, sections, out=torch.empty_like(x), **kw)
        left = float((dout.double() * (y1.double() - y0.double())).sum())
        right = float((grad.double() * ((x + dx_in).double() - x.double())).sum())
        scale = 2 * float((x + dx_in).abs().max()) * float(table.abs().max())
        bound = 3 * 2.0 ** -24 * scale * (2 * float(dout.abs().sum()) + float((dx_in).abs().sum()) * float(dout.abs().max()))
        assert abs(left - right) <= bound
    no_error(sa)


def test_rope_axes_nonfinite_values_stay_in_their_pair(sa):
    from l2_torch_alloc_amd import ops
    sections = (16, 24, 24)
    for half in (False, True):
        (x, _), table, pos = rope_inputs(1, 5, (3, 1), 128, sections, torch.bfloat16, 20, seed=9)
        x[0, 2, 1, 7] = float("inf")
        x[0, 3, 0, 100] = float("nan")
        got = ops.rope_axes_forward(x, table, pos, sections, out=torch.empty_like(x), half=half)
        bad = torch.zeros_like(x, dtype=torch.bool)
        for t, h, e in ((2, 1, 7), (3, 0, 100)):
            bad[0, t, h, e] = True
            bad[0, t, h, (e + 64) % 128 if half else e ^ 1] = True
        assert bool(torch.isfinite(got)[~bad].all())
        assert not bool(torch.isfinite(got)[bad].any())
    no_error(sa)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(sa, dtype, residual):
    from l2_torch_alloc_amd import ops
    g = torch.Generator().manual_seed(11)
    for n, p in ((1, 0.5), (7, 0.25), (8, 0.1), (4093, 0.1), (65536, 0.9), (65536 + 5, 0.0), (1000003, 0.3), (100, 1.0)):
        x = torch.randn(n, generator=g).to(dtype)
        r = torch.randn(n, generator=g).to(dtype) if residual else None
        if p == 1.0:
            x[3], x[5] = float("nan"), float("-inf")
        seed = torch.tensor([n * 7919 - 2 ** 62, 2 ** 61 + n])
        y = ops.dropout_forward(x.cuda(), p, seed.cuda(), residual=None if r is None else r.cuda())
        t = ops.dropout_threshold(p)
        with np.errstate(invalid="ignore"):
            want = S.dropout(f64(x), t, int(seed[0]), int(seed[1]), None if r is None else f64(r))
        # the scale, the product and the sum in fp32, then the storage
        mag = np.abs(want) + (0 if r is None else np.abs(want - f64(r)) + np.abs(f64(r)))
        tol = (3 * 2.0 ** -24 + (0 if dtype == torch.float32 else HALF_STEP[dtype])) * mag + HALF_STEP_SUBNORMAL[dtype]
        assert np.all(np.abs(f64(y) - want) <= tol), (n, p)
    no_error(sa)


def test_dropout_backward_has_the_forwards_mask(sa):
    from l2_torch_alloc_amd import ops
    n = 100001
    seed = torch.tensor([5, 9]).cuda()
    ones = torch.ones(n, device="cuda")
    masks = [ops.dropout_backward(ones.to(t), 0.25, seed).float() for t in (torch.float32, torch.bfloat16, torch.float16)]
    forward = ops.dropout_forward(ones, 0.25, seed)
    assert torch.equal(masks[0], forward)
    for m in masks[1:]:
        assert torch.equal(m != 0, forward != 0)                     # the mask does not depend on the type
    share = float((forward != 0).double().mean())
    assert abs(share - 0.75) <= 5 * (0.25 * 0.75 / n) ** 0.5         # five standard deviations
    other = ops.dropout_forward(ones, 0.25, torch.tensor([5, 10]).cuda())
    differ = float(((other != 0) != (forward != 0)).double().mean())
    assert abs(differ - 2 * 0.25 * 0.75) <= 5 * (0.375 * 0.625 / n) ** 0.5
    no_error(sa)


def test_dropout_in_place_and_onto_the_residual(sa):
    from l2_torch_alloc_amd import ops
    x, r = torch.randn(3, 1001, device="cuda"), torch.randn(3, 1001, device="cuda")
    seed = torch.tensor([1, 2]).cuda()
    y, z = ops.dropout_forward(x, 0.4, seed), ops.dropout_forward(x, 0.4, seed, residual=r)
    r2 = r.clone()
    assert ops.dropout_forward(x, 0.4, seed, residual=r2, out=r2) is r2 and torch.equal(r2, z)
    x2 = x.clone()
    assert ops.dropout_forward(x2, 0.4, seed, out=x2) is x2 and torch.equal(x2, y)
    no_error(sa)


def test_dropout_writes_nothing_behind_its_end(sa):
    from l2_torch_alloc_amd import ops
    for n in (1, 5, 8 * 256 + 3, 8 * 256 * 9 + 7, 100003):
        buf = torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.dropout_forward(torch.ones(n, dtype=torch.bfloat16, device="cuda"), 0.5, torch.tensor([3, 4]).cuda(), out=buf[:n])
        assert bool((buf[n:] == 7.0).all()) and bool(((buf[:n] == 0) | (buf[:n] == 2)).all())
    no_error(sa)


def test_dropout_in_a_graph_reads_the_seed_at_every_replay(sa):
    from l2_torch_alloc_amd import ops
    for n in (4099, 1 << 23):                                        # striped and sided launches
        x = torch.randn(n, device="cuda")
        seed = torch.tensor([77, 0]).cuda()
        out = torch.empty_like(x)
        ops.dropout_forward(x, 0.3, seed, out=out)                   # compiles
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ops.dropout_forward(x, 0.3, seed, out=out)
        last = None
        for step in range(4):
            seed[1] = step
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            want = ops.dropout_forward(x, 0.3, torch.tensor([77, step]).cuda())
            assert torch.equal(got, want)
            assert last is None or not torch.equal(got, last)
            last = got
    no_error(sa)


def test_rope_axes_in_a_graph(sa):
    from l2_torch_alloc_amd import ops
    sections = (24, 20, 20)
    (q, k), table, pos = rope_inputs(4, 9, (8, 2), 128, sections, torch.bfloat16, 64, seed=2)
    outs = [torch.empty_like(q), torch.empty_like(k)]
    ops.rope_axes_forward_many([q, k], table, pos, sections, half=True, outs=outs)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        ops.rope_axes_forward_many([q, k], table, pos, sections, half=True, outs=outs)
    for step in range(3):
        pos.copy_((pos + 5) % 64)
        q.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.rope_axes_forward_many([q, k], table, pos, sections, half=True, outs=[torch.empty_like(q), torch.empty_like(k)])
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    no_error(sa)


def test_on_another_stream(sa):
    from l2_torch_alloc_amd import ops
    x = torch.randn(1 << 20, device="cuda").to(torch.bfloat16)
    seed = torch.tensor([1, 1]).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = ops.dropout_forward(x, 0.5, seed)
        b = ops.dropout_backward(a, 0.5, seed)
    side.synchronize()
    want = ops.dropout_forward(x, 0.5, seed)
    assert torch.equal(a, want) and torch.equal(b, ops.dropout_backward(want, 0.5, seed))
    no_error(sa)


def test_dropout_past_two_gib(sa):
    """64-bit indices: the block counters and addresses behind 2^31 bytes, and a ragged end there."""
    from l2_torch_alloc_amd import ops
    n = (1 << 30) + 8 * 1000 + 5                                     # elements of 2 bytes
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout_forward(x, 0.5, torch.tensor([123, 456]).cuda(), out=x)
    for first, count in ((0, 1000), ((1 << 30) - 4096, 9000), (n - n % 8 - 800, 800 + n % 8)):
        want = (S.dropout_bits(count, 123, 456, first) >= 32768) * 2.0
        have = y[first:first + count].cpu().double().numpy()
        assert np.array_equal(have, want[:have.size])
    del x, y
    no_error(sa)


def test_empty_and_refused(sa):
    from l2_torch_alloc_amd import ops
    seed = torch.tensor([1, 1]).cuda()
    assert ops.dropout_forward(torch.empty(0, 5, device="cuda"), 0.5, seed).shape == (0, 5)
    sections = (16, 16)
    table, pos = torch.zeros(4, 64, device="cuda"), torch.zeros(0, 3, 2, dtype=torch.int32, device="cuda")
    assert ops.rope_axes_forward(torch.empty(0, 3, 2, 64, device="cuda"), table, pos, sections).numel() == 0
    x = torch.ones(64, 64, device="cuda")
    with pytest.raises(AssertionError):
        ops.dropout_forward(x.t(), 0.5, seed)                        # a view that is not contiguous
    with pytest.raises(AssertionError):
        ops.dropout_forward(x.view(-1)[1:], 0.5, seed)               # off a 16-byte boundary
    with pytest.raises(AssertionError):
        ops.dropout_forward(x, 0.5, seed.cpu())
    no_error(sa)
    lib = sa.library()
    # whole elements only, and only ops that say so take a ragged end
    kid = ops._kernel("dropout", ("fp32", False))
    lib.sideaware_elementwise(kid, 4 * 64 + 2, x.data_ptr(), 0, 0, 0, x.data_ptr(), 0, 0, 0, seed.data_ptr(), 0, 0, 0, 0, None)
    assert "whole number" in sa.sideaware_last_error()
    lib.sideaware_clear_error()
    kid = ops._kernel("fill")
    lib.sideaware_elementwise(kid, 1000, x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None)
    assert "multiples of 16" in sa.sideaware_last_error()
    lib.sideaware_clear_error()
    torch.cuda.synchronize()
    assert bool((x == 1).all())


def test_dropout_under_torch_compile(sa):
    from l2_torch_alloc_amd import ops

    @torch.compile(fullgraph=True)
    def step(x, seed, residual):
        return ops.dropout_forward(x * 2, 0.25, seed, residual=residual) + 1

    x, r = torch.randn(64, 96, device="cuda"), torch.randn(64, 96, device="cuda")
    seed = torch.tensor([3, 1]).cuda()
    want = ops.dropout_forward(x * 2, 0.25, seed, residual=r) + 1
    assert torch.equal(step(x, seed, r), want)
    no_error(sa)


def test_overlapping_arrays_are_refused(sa):
    """An output may be its own input, but not share memory with another array of the launch."""
    from l2_torch_alloc_amd import ops
    seed, sections = torch.tensor([3, 1]).cuda(), (16, 16)
    table = ops.freqs_cis_axes_table(sections, 8, 10000.0).cuda()
    pos = torch.zeros(2, 5, 2, dtype=torch.int32, device="cuda") + 3
    shape, n = (2, 5, 3, 64), 2 * 5 * 3 * 64
    buf = torch.ones(4 * n, device="cuda")
    x, behind, apart = buf[:n].view(shape), buf[16:n + 16].view(shape), buf[2 * n:3 * n].view(shape)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope_axes_forward(x, table, pos, sections, out=behind)
    for tensors, outs in (([x, x], None), ([x, behind], None), ([x, x], [apart, apart]), ([x, apart], [apart, x]),
                          ([x, apart], [buf[n:2 * n].view(shape), x]), ([apart, x], [x, buf[n:2 * n].view(shape)])):
        with pytest.raises(ValueError, match="overlap"):
            ops.rope_axes_forward_many(tensors, table, pos, sections, outs=outs)
    for kw in ({"out": behind}, {"residual": apart, "out": behind}, {"residual": behind, "out": x}):
        with pytest.raises(ValueError, match="overlap"):
            ops.dropout_forward(x, 0.5, seed, **kw)
    torch.cuda.synchronize()
    assert bool((buf == 1).all())
    # neighbours in one allocation, the same input twice, and an input as the output are all right
    twice = [buf[n:2 * n].view(shape), buf[3 * n:].view(shape)]
    a, b = ops.rope_axes_forward_many([x, x], table, pos, sections, outs=twice)
    assert torch.equal(a, b) and bool((x == 1).all())
    ops.rope_axes_forward_many([x, apart], table, pos, sections)
    assert torch.equal(x, a) and torch.equal(apart, a)
    want = ops.dropout_forward(x, 0.5, seed, residual=x)
    assert torch.equal(ops.dropout_forward(x, 0.5, seed, residual=x, out=x), want)
    no_error(sa)


def test_rope_axes_under_torch_compile(sa):
    from l2_torch_alloc_amd import ops
    sections = (16, 24, 24)
    table = ops.freqs_cis_axes_table(sections, 50, 10000.0).cuda()
    pos = (torch.arange(2 * 7 * 3, dtype=torch.int32) % 50).view(2, 7, 3).cuda()
    torch.manual_seed(3)
    q, k = (torch.randn(2, 7, heads, 128, device="cuda", dtype=torch.bfloat16) for heads in (4, 2))

    def rotate(q, k):
        a, b = ops.rope_axes_forward_many([q * 2, k + 1], table, pos, sections)
        return a + 1, ops.rope_axes_backward(b, table, pos, sections, out=torch.empty_like(b), half=True, order="turns")

    want = rotate(q, k)
    for fullgraph in (False, True):
        compiled = torch.compile(rotate, fullgraph=fullgraph)
        for _ in range(2):
            assert all(torch.equal(h, w) for h, w in zip(compiled(q, k), want))
    no_error(sa)


def test_group_norm_under_torch_compile(sa):
    """Its calls stand between the compiled parts of a function."""
    from l2_torch_alloc_amd import ops
    torch.manual_seed(3)
    x, w, b = torch.randn(2, 30, 64, device="cuda"), torch.randn(64, device="cuda"), torch.randn(64, device="cuda")

    def layer(x):
        y, stats = ops.group_norm_forward(x * 2, w, b, 8, activation="silu")
        return ops.group_norm_backward(y + 1, x * 2, w, b, stats, 8, activation="silu")

    want = layer(x)
    compiled = torch.compile(layer)
    for _ in range(2):
        assert all(torch.equal(h, t) for h, t in zip(compiled(x), want))
    no_error(sa)
