"""The sideband value of a segment of a batched launch takes whatever that of a single launch takes: any integer, of which
the low 32 bits are passed on."""
import ctypes

import pytest
import torch

from l2_torch_alloc_amd import ops, wrapper

VALUES = (0, 1, -1, 2 ** 31 - 1, 2 ** 31, 0xDEADBEEF, 2 ** 32 - 1, -2 ** 31, 2 ** 32 + 5)


def test_values_reach_the_library_as_a_single_launch_passes_them(monkeypatch):
    seen = []

    class Library:
        @staticmethod
        def sideaware_elementwise_batch(kernel_id, count, packed, device, stream):
            seen.extend((ops._Segment * count).from_buffer_copy(packed))

    monkeypatch.setattr(wrapper, "library", lambda: Library)
    monkeypatch.setattr(wrapper, "_check", lambda t, name: 0 if t is None else t.data_ptr())
    monkeypatch.setattr(wrapper, "_device_and_stream", lambda t=None: (0, 0))
    x, side = torch.zeros(4, dtype=torch.int32), torch.zeros(2)
    ops.elementwise_batch(3, [(16, [x], [None, x], side, v) for v in VALUES])
    assert [s.sideband_value for s in seen] == [ctypes.c_int(v).value for v in VALUES]
    for s in seen:
        assert (s.num_bytes, s.out[0], s.inp[0], s.inp[1], s.sideband_memory) == (16, x.data_ptr(), None, x.data_ptr(), side.data_ptr())


@pytest.mark.gpu
def test_fill_patterns_in_one_launch(sa):
    outs = [torch.zeros(64 + 4 * i, dtype=torch.int32, device="cuda") for i in range(len(VALUES))]
    ops.elementwise_batch(ops._kernel("fill"), [(t.numel() * 4, [t], [], None, v) for t, v in zip(outs, VALUES)])
    for t, v in zip(outs, VALUES):
        single = torch.empty_like(t)
        ops.fill_int32(single, v)
        assert torch.equal(t, single) and int(t[0]) == ctypes.c_int(v).value
    assert sa.sideaware_last_error() == "", sa.sideaware_last_error()
