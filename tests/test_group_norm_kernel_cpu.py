"""The shipped group norm file (kernels and launch code) on the CPU, under sanitizers: a workgroup's threads are threads of
the host, LDS and every array are exactly as long as they are, and every access is on its type's boundary.  Results against the 64-bit statements, with the
tolerances of the tests on the GPU (a reciprocal and an exponential of the host are no further off than the device's)."""
import os
import re
import subprocess

import pytest
import torch

import test_gpu_group_norm as T
from l2_torch_alloc_amd import build as sa_build

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")
CLANG = os.path.join(sa_build.rocm_root(), "lib", "llvm", "bin", "clang++")
pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="ROCm clang++ not found")


def cpu_text():
    """group_norm.hip with the few statements that only the device's compiler takes written for the host's."""
    text = open(os.path.join(sa_build.CSRC, "group_norm.hip")).read()

    def swap(pattern, by, count):
        nonlocal text
        text, n = re.subn(pattern, by, text)
        assert n == count if count else n > 0, (pattern, n)

    swap(r"#include <hip/hip_runtime.h>\n", "", 1)
    swap(r'asm volatile\("" : "\+v"\(here\)\);', "", 1)
    swap(r'asm volatile\("global_store_dwordx4[^;]*;', "*(W*)to = words;", 2)
    swap(r"extern __shared__ [^;]*double lds\[\];", "double* lds = (double*)cpu_lds;", 2)
    swap(r"(group_norm_\w+<[^;{}]*?>)<<<(.*?)>>>\(a\);", r"cpu_launch([](const GnArgs& args) { \1(args); }, a, \2);", 0)
    return text[:text.index("hipError_t launch_type(")] + "}\n}\n"        # of its types, fp32 and bf16


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    where = tmp_path_factory.mktemp("group_norm")
    src, exe = str(where / "tu.cpp"), str(where / "tu")
    with open(src, "w") as f:
        f.write('#include "%s/group_norm_cpu_prelude.h"\n' % NATIVE + cpu_text() + '#include "%s/group_norm_cpu_driver.h"\n' % NATIVE)
    proc = subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-g1", "-pthread", "-ffp-contract=off", "-fsanitize=address,undefined",
                           "-fno-sanitize-recover=undefined", "-Wno-unused-value", "-Wno-unknown-pragmas", "-I", sa_build.CSRC, src, "-o", exe],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-4000:]
    return exe


def run(driver, tmp_path, backward, x, w, b, G, activation, more=(), cus=8):
    """The outputs of one call and how many of its launches had chunks."""
    N, P, C = x.shape
    fp32 = x.dtype == torch.float32
    raw = lambda t: t.contiguous().view(-1).view(torch.uint8).numpy().tobytes()          # noqa: E731
    (tmp_path / "in").write_bytes(b"".join(raw(t) for t in (x, w, b) + tuple(more)))
    line = "%d %d %d %d %d %d %d %d %d %s %s\n" % (backward, N, P, C, G, fp32, {"none": 0, "silu": 1}[activation], w.dtype == torch.float32, cus,
                                                 tmp_path / "in", tmp_path / "out")
    proc = subprocess.run([driver], input=line, capture_output=True, text=True, timeout=300, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert proc.returncode == 0, proc.stderr[-3000:]
    data, outs = (tmp_path / "out").read_bytes(), []
    for like in ((x, w, b) if backward else (x, torch.empty(N, G, 2))):
        size = like.numel() * like.element_size()
        outs.append(torch.frombuffer(bytearray(data[:size]), dtype=like.dtype).view(like.shape))
        data = data[size:]
    assert not data
    return outs, int(re.search(r"chunked=(\d+)", proc.stdout)[1])


def check(driver, tmp_path, N, P, C, G, dtype, activation, wtype=torch.float32, cus=8):
    x, w, b, dout = T.make(N, P, C, dtype, wtype, seed=P + C)
    (y, stats), chunked = run(driver, tmp_path, 0, x, w, b, G, activation, cus=cus)
    T.check_forward(y, stats, x, w, b, G, 1e-5, activation)
    grads, _ = run(driver, tmp_path, 1, x, w, b, G, activation, (dout, stats), cus=cus)
    T.check_backward(grads, dout, x, w, b, stats, G, activation)
    return chunked


@pytest.mark.parametrize("gc", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 13, 15, 16])
def test_every_channel_reaches_its_group(driver, tmp_path, gc):
    """Groups of every width against vectors of 8 and 4 channels (eight groups: whole vectors), 2 and 1."""
    for G, P in ((8, 9), (16, 3)):
        check(driver, tmp_path, 2, P, gc * G, G, torch.bfloat16, "none")
    check(driver, tmp_path, 1, 7, gc * 4, 4, torch.float32, "silu")
    check(driver, tmp_path, 1, 5, gc * 3, 3, torch.bfloat16, "silu", torch.bfloat16)


@pytest.mark.parametrize("N,P,C,G,dtype,cus", [
    (1, 4096, 40, 8, torch.bfloat16, 4), (2, 700, 160, 32, torch.bfloat16, 1), (9, 3, 40, 8, torch.bfloat16, 1), (1, 6000, 24, 8, torch.float32, 4),
    (1, 900, 33, 11, torch.bfloat16, 2), (1, 5, 2056, 1, torch.bfloat16, 2), (2, 80, 1285, 257, torch.bfloat16, 1), (3, 257, 24, 4, torch.float32, 1)])
def test_chunks_and_loops(driver, tmp_path, N, P, C, G, dtype, cus):
    """Several launches, several samples per workgroup, slabs of several slices."""
    check(driver, tmp_path, N, P, C, G, dtype, "silu", cus=cus)


def test_groups_that_a_vector_touches(tmp_path):
    exe = str(tmp_path / "vector")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", os.path.join(NATIVE, "group_norm_vector_main.cpp"), "-o", exe],
                   check=True, capture_output=True, text=True)
    proc = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert proc.returncode == 0 and "cases=320 ok" in proc.stdout, proc.stdout + proc.stderr


@pytest.mark.parametrize("N,P,C,G,dtype", [(2, 100, 7, 1, torch.bfloat16), (1, 40, 21, 3, torch.float32), (1, 3000, 7, 7, torch.bfloat16)])
def test_odd_rows_of_odd_channels(driver, tmp_path, N, P, C, G, dtype):
    """What comes before the pairs of doubles in LDS is an odd number of doubles."""
    check(driver, tmp_path, N, P, C, G, dtype, "silu")
