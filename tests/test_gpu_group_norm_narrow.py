"""Group norm on an MI355X where groups are narrower than a vector of channels and vectors are full: every number of
channels per group that a 16-byte vector may hold parts of, in one launch, in chunks and with several samples to a
workgroup."""
import pytest
import torch

import test_gpu_group_norm as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,P,C,G", [
    (2, 100, 40, 8), (2, 4096, 160, 32), (2, 64, 160, 32), (1, 30000, 40, 8), (1300, 3, 40, 8), (2, 64, 320, 64), (3, 50, 80, 16),
    (2, 100, 16, 8), (1, 9000, 64, 32), (2, 100, 24, 8), (1, 9000, 96, 32), (2, 100, 56, 8), (1, 9000, 224, 32), (2, 100, 48, 8), (2, 100, 32, 8),
    (2, 100, 72, 8), (1, 9000, 88, 8), (2, 300, 104, 8), (1300, 20, 56, 8)])
def test_narrow_groups(sa, N, P, C, G, dtype):
    from l2_torch_alloc_amd import ops
    for activation, wtype in (("none", torch.float32), ("silu", dtype)):
        x, w, b, dout = T.make(N, P, C, dtype, wtype, seed=P + C)
        xd, wd, bd = x.cuda(), w.cuda(), b.cuda()
        y, stats = ops.group_norm_forward(xd, wd, bd, G, activation=activation)
        T.check_forward(y, stats, x, w, b, G, 1e-5, activation)
        T.check_backward(ops.group_norm_backward(dout.cuda(), xd, wd, bd, stats, G, activation=activation), dout, x, w, b, stats, G, activation)
    T.no_error(sa)
