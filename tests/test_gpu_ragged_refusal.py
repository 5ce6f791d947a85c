"""A launch whose length is no multiple of 16 bytes, of an op that does not take such arrays, is refused before anything
is compiled for it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_refused_before_compiling(sa):
    lib = sa.library()
    x = torch.ones(512, device="cuda")
    kid = sa.sideaware_create_kernel(b"#define KERNEL_NAME never_compiled\nthis text is no op header\n")
    lib.sideaware_elementwise(kid, 1000, x.data_ptr(), 0, 0, 0, x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, None)
    assert "multiples of 16" in sa.sideaware_last_error()
    lib.sideaware_clear_error()
    # the built-in copy, and an id that was never given out
    for kernel in (0, 1 << 20, -1):
        lib.sideaware_elementwise(kernel, 1000, x.data_ptr(), 0, 0, 0, x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, None)
        assert "multiples of 16" in sa.sideaware_last_error()
        lib.sideaware_clear_error()
    # an op that only mentions the hook is looked at by the compiler, and refused then
    kid = sa.sideaware_create_kernel(b"// no RAGGED_TAIL\n" + b"\n".join([
        b"typedef int o0;", b"struct unused {};", b"typedef unused o1, o2, o3, i0, i1, i2, i3;", b"constexpr bool reverse_order = false;",
        b"constexpr bool input_evict[4] = {false, false, false, false};",
        b"__device__ void elementwise_op(size_t i, int v, o0 &a, o1 &, o2 &, o3 &, const i0 &, const i1 &, const i2 &, const i3 &) { a = v; }", b""]))
    lib.sideaware_elementwise(kid, 1000, x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None)
    assert "multiples of 16" in sa.sideaware_last_error()
    lib.sideaware_clear_error()
    torch.cuda.synchronize()
    assert bool((x == 1).all())
