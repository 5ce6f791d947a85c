"""An output of the multi-axis RoPE or dropout ops may be the input that it belongs to, element for element, and shares no
memory with any other array of the call: workgroups finish in any order, and what one of them reads another may have
overwritten.  On the CPU, with the library's entry points in the place of recorders and tensors that claim to be on a GPU."""
import contextlib

import pytest
import torch

from l2_torch_alloc_amd import ops, wrapper


@contextlib.contextmanager
def recorded():
    """The list of the library's calls while tensors claim to be on a GPU."""
    seen = []

    class Library:
        @staticmethod
        def sideaware_elementwise_batch(*args):
            seen.append(args)

        @staticmethod
        def sideaware_elementwise(*args):
            seen.append(args)

    with pytest.MonkeyPatch.context() as monkeypatch:
        monkeypatch.setattr(wrapper, "library", lambda: Library)
        monkeypatch.setattr(wrapper, "_device_and_stream", lambda t=None: (0, 0))
        monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
        monkeypatch.setattr(torch.Tensor, "is_cuda", True)
        monkeypatch.setattr(ops, "_kernel", lambda *args: 7)
        monkeypatch.setattr(ops, "_plans", {})
        yield seen


@pytest.fixture
def calls():
    with recorded() as seen:
        yield seen


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


@pytest.fixture(scope="module")
def compiled():
    """The ops' nodes in compiled graphs run their implementation on the CPU, too."""
    library = torch.library.Library("sideaware", "IMPL")

    def on_cpu(implementation, name):
        def run(*args):
            with recorded() as seen:
                implementation(*args)
            nodes.append((name, len(seen), args))
        library.impl(name, run, "CPU")
    nodes = []
    on_cpu(ops._rope_axes_launch, "rope_axes")
    on_cpu(ops._dropout_node, "dropout")
    yield nodes
    library._destroy()


def test_compiled_calls_are_one_node_with_the_same_refusals(compiled):
    table, positions, seed = torch.zeros(8, 64), torch.zeros(2, 5, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    compile = lambda f: torch.compile(f, fullgraph=True)                                 # noqa: E731
    rotate = compile(lambda q, k: ops.rope_axes_forward_many([q, k], table, positions, SECTIONS))
    x, y = torch.zeros(SHAPE), torch.zeros(2, 5, 1, 64)
    rotate(x, y)
    (name, launches, args), = compiled
    assert (name, launches) == ("rope_axes", 1) and [t.data_ptr() for t in args[-1]] == [x.data_ptr(), y.data_ptr()]
    compiled.clear()
    drop = compile(lambda x, p: ops.dropout_forward(x + 1, p, seed, residual=x))
    for n, p in ((5, 0.5), (7, 0.25), (9, 0.125)):                                       # lengths and probabilities that change
        assert drop(torch.zeros(n), p).shape == (n,)
    assert [(name, launches, args[1]) for name, launches, args in compiled] == [("dropout", 1, p) for p in (0.5, 0.25, 0.125)]
    compiled.clear()

    # the same tensor twice, and a view that is shifted inside its input: in place, as the compiler leaves them
    with pytest.raises(ValueError, match="overlap"):
        compile(lambda x: ops.rope_axes_forward_many([x, x], table, positions, SECTIONS))(torch.zeros(SHAPE))
    with pytest.raises(ValueError, match="overlap"):
        compile(lambda b: ops.rope_axes_forward(b[:COUNT].view(SHAPE), table, positions, SECTIONS, out=b[16:COUNT + 16].view(SHAPE)))(torch.zeros(4096))
    with pytest.raises(ValueError, match="overlap"):
        compile(lambda b: ops.dropout_forward(b[:COUNT], 0.5, seed, out=b[16:COUNT + 16]))(torch.zeros(4096))
    assert not compiled
    for call in (lambda x: ops.rope_axes_forward(x, table[:, :32], positions, SECTIONS), lambda x: ops.dropout_forward(x, 0.5, seed[:1])):
        with pytest.raises(AssertionError):
            compile(call)(torch.zeros(SHAPE))
