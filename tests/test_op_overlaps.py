"""An output of the multi-axis RoPE or dropout ops may be the input that it belongs to, element for element, and shares no
memory with any other array of the call: workgroups finish in any order, and what one of them reads another may have
overwritten.  On the CPU, with the library's entry points in the place of recorders and tensors that claim to be on a GPU."""
import pytest
import torch

from l2_torch_alloc_amd import ops, wrapper


@pytest.fixture
def calls(monkeypatch):
    seen = []

    class Library:
        @staticmethod
        def sideaware_elementwise_batch(*args):
            seen.append(args)

        @staticmethod
        def sideaware_elementwise(*args):
            seen.append(args)

    monkeypatch.setattr(wrapper, "library", lambda: Library)
    monkeypatch.setattr(wrapper, "_device_and_stream", lambda t=None: (0, 0))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(ops, "_kernel", lambda *args: 7)
    monkeypatch.setattr(ops, "_plans", {})
    return seen


SECTIONS = (16, 16)
SHAPE, COUNT = (2, 5, 3, 64), 2 * 5 * 3 * 64


def rope(*args, **kw):
    return lambda: ops.rope_axes_forward(*args, **kw)


def test_rope_axes(calls):
    buf = torch.zeros(4096 + 2 * COUNT)
    table, positions = torch.zeros(8, 64), torch.zeros(2, 5, 2, dtype=torch.int32)
    x, apart = buf[:COUNT].view(SHAPE), buf[COUNT:2 * COUNT].view(SHAPE)
    here = lambda at, *shape: buf[at:at + torch.Size(shape).numel()].view(shape)          # noqa: E731
    where = lambda at: here(at, 2, 5, 2).view(torch.int32)                                # noqa: E731
    refused = [rope(x, here(0, 8, 64), positions, SECTIONS),                              # the table at the start of what is written,
               rope(x, here(COUNT - 64, 8, 64), positions, SECTIONS),                     # at its end,
               rope(x, buf.view(-1, 64)[:-1], positions, SECTIONS, out=apart),            # around it
               rope(x, table, where(0), SECTIONS), rope(x, table, where(COUNT - 1), SECTIONS), rope(x, table, where(COUNT + 40), SECTIONS, out=apart),
               lambda: ops.rope_axes_backward_many([x, apart], table, where(COUNT + 4), SECTIONS),
               lambda: ops.rope_axes_forward_many([x, apart], here(2 * COUNT - 4, 8, 64), positions, SECTIONS)]
    for call in refused:
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert not calls
    # neighbours, and reading what the table or the positions lie in, are all right
    accepted = [rope(x, here(COUNT, 8, 64), positions, SECTIONS), rope(x, table, where(COUNT), SECTIONS),
                rope(apart, here(COUNT - 512, 8, 64), positions, SECTIONS), rope(apart, table, where(COUNT - 20), SECTIONS),
                rope(x, here(0, 8, 64), where(4), SECTIONS, out=apart)]
    for call in accepted:
        call()
    assert len(calls) == len(accepted)


def test_dropout(calls):
    buf = torch.zeros(3 * COUNT)
    x, apart = buf[:COUNT], buf[COUNT:2 * COUNT]
    seed = lambda at: buf[at:at + 4].view(torch.int64)                                    # noqa: E731
    for at, out in ((0, x), (COUNT - 2, x), (COUNT - 2, apart), (2 * COUNT - 2, apart), (COUNT + 64, apart)):
        with pytest.raises(ValueError, match="overlap"):
            ops.dropout_forward(x, 0.5, seed(at), out=out)
        with pytest.raises(ValueError, match="overlap"):
            ops.dropout_forward(x, 0.5, seed(at), residual=buf[2 * COUNT:], out=out)
    assert not calls
    ops.dropout_forward(x, 0.5, seed(COUNT), out=x)
    ops.dropout_forward(x, 0.5, seed(0), out=apart)
    ops.dropout_backward(x, 0.5, seed(2 * COUNT), out=apart)
    assert len(calls) == 3
