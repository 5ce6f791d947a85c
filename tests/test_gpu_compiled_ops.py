"""The multi-axis RoPE and dropout ops inside compiled graphs on an MI355X: the eager call's results for lengths and
probabilities that change, and its refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SECTIONS = (16, 16)
SHAPE, COUNT = (2, 5, 3, 64), 2 * 5 * 3 * 64


def test_lengths_and_probabilities_that_change(sa):
    from l2_torch_alloc_amd import ops
    table, seed = ops.freqs_cis_axes_table(SECTIONS, 40, 10000.0).cuda(), torch.tensor([3, 1]).cuda()

    def step(q, k, positions, p):
        a, b = ops.rope_axes_forward_many([q * 2, k + 1], table, positions, SECTIONS, half=True)
        return ops.dropout_forward(a, p, seed, residual=q), b - 1

    compiled = torch.compile(step, fullgraph=True)
    for T, p in ((5, 0.5), (7, 0.25), (31, 0.125), (5, 0.0)):
        q, k = torch.randn(2, T, 3, 64, device="cuda"), torch.randn(2, T, 1, 64, device="cuda")
        positions = (torch.arange(2 * T * 2, dtype=torch.int32, device="cuda") % 41).view(2, T, 2)       # 40: outside the table
        for have, want in zip(compiled(q, k, positions, p), step(q, k, positions, p)):
            assert torch.equal(have.view(torch.int32), want.view(torch.int32))
    assert sa.sideaware_last_error() == "", sa.sideaware_last_error()


def test_overlaps_are_refused(sa):
    from l2_torch_alloc_amd import ops
    table, seed = ops.freqs_cis_axes_table(SECTIONS, 8, 10000.0).cuda(), torch.tensor([3, 1]).cuda()
    positions = torch.zeros(2, 5, 2, dtype=torch.int32, device="cuda")
    for call in (lambda b: ops.rope_axes_forward_many([b[:COUNT].view(SHAPE)] * 2, table, positions, SECTIONS),
                 lambda b: ops.rope_axes_forward(b[:COUNT].view(SHAPE), table, positions, SECTIONS, out=b[16:COUNT + 16].view(SHAPE)),
                 lambda b: ops.dropout_forward(b[:COUNT], 0.5, seed, out=b[16:COUNT + 16])):
        buf = torch.ones(4096, device="cuda")
        with pytest.raises(ValueError, match="overlap"):
            torch.compile(call, fullgraph=True)(buf)
        torch.cuda.synchronize()
        assert bool((buf == 1).all())
    assert sa.sideaware_last_error() == "", sa.sideaware_last_error()
