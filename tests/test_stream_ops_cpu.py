"""The multi-axis rotary and dropout op headers without a GPU: the shipped template and headers run lane by
lane on the CPU under AddressSanitizer (every array exactly as long as it is), the generator against
known values, and the refusals of the Python layer that need no device."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

import stream_ops_oracle as S
from l2_torch_alloc_amd import build as sa_build
from l2_torch_alloc_amd import headers, ops, wrapper

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")
CLANG = os.path.join(sa_build.rocm_root(), "lib", "llvm", "bin", "clang++")
needs_clang = pytest.mark.skipif(not os.path.exists(CLANG), reason="ROCm clang++ not found")
TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
# Below a type's smallest normal number its step no longer shrinks with the value: fp16's is 2^-24 under
# 2^-14, so a rounding there is off by up to 2^-25, whatever the value (bf16 and fp32: 2^-134, 2^-150).
HALF_STEP_SUBNORMAL = {"fp32": 2.0 ** -150, "bf16": 2.0 ** -134, "fp16": 2.0 ** -25}


@pytest.fixture(scope="module")
def lib():
    return wrapper.bind(sa_build.build_library(force=False))


def build_driver(lib, tmp_path, header, variant):
    tu = "\n".join(['#include "%s"' % os.path.join(NATIVE, "kernel_cpu_prelude.h"), lib.sideaware_config_block(variant).decode(),
                    header.decode(), lib.sideaware_kernel_source().decode(),
                    '#include "%s"' % os.path.join(NATIVE, "stream_ops_cpu_driver.h")])
    src = tmp_path / "tu.cpp"
    src.write_text(tu)
    exe = str(tmp_path / "tu")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-g", "-ffp-contract=off", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=undefined", "-Wno-unused-value", str(src), "-o", exe], check=True, capture_output=True, text=True)
    return exe


def run(exe, tmp_path, x, ins, mem, val, grid=0, off=0, stripe=14):
    """One launch; x and ins are torch tensors, mem a torch tensor; returns the output, shaped like x."""
    paths = []
    for i, t in enumerate([x] + list(ins) + [None] * (3 - len(ins)) + [mem]):
        if t is None:
            paths.append("-")
        else:
            path = str(tmp_path / ("in%d" % i))
            t.contiguous().view(torch.uint8).numpy().tofile(path)
            paths.append(path)
    out = str(tmp_path / "out")
    proc = subprocess.run([exe, str(grid), str(x.numel() * x.element_size()), str(off), str(stripe), str(val)] + paths + [out],
                          capture_output=True, text=True, timeout=300, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert proc.returncode == 0, proc.stderr[-3000:]
    return torch.from_numpy(np.fromfile(out, dtype=np.uint8)).view(x.dtype).view(x.shape)


def test_generator_matches_published_values():
    # Philox4x32 with 10 and with 7 rounds on the all-zero and all-ones inputs
    ones = 0xFFFFFFFF
    zero10 = [int(w) for w in S.philox4x32((0, 0, 0, 0), (0, 0), 10)]
    assert zero10 == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones10 = [int(w) for w in S.philox4x32((ones, ones, ones, ones), (ones, ones), 10)]
    assert ones10 == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    zero7 = [int(w) for w in S.philox4x32((0, 0, 0, 0), (0, 0), 7)]
    assert zero7 == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]


@needs_clang
@pytest.mark.parametrize("dtype,residual,variant", [("bf16", False, 0), ("bf16", True, 1), ("fp32", False, 1), ("fp32", True, 0), ("fp16", False, 32),
                                                    ("fp32", False, 33)])
def test_dropout_header_on_cpu(lib, tmp_path, dtype, residual, variant):
    exe = build_driver(lib, tmp_path, headers.dropout_header(dtype, residual), variant)
    g = torch.Generator().manual_seed(3)
    vec = 4 if dtype == "fp32" else 8
    seed, offset = -0x123456789ABCDEF, (1 << 40) + 17
    mem = torch.tensor([seed, offset])
    # shorter than a vector, ragged, whole vectors, whole tiles, whole tiles and a ragged end
    for n in (1, vec - 1, vec, vec + 1, 255 * vec, 256 * vec, 256 * vec + 3, 8 * 256 * vec + vec - 1, 5000 * vec + 5):
        for grid, off, threshold in ((0, 0, 6554), (16, 48, 0), (0, 4096 + 16, 65536), (8, 0, 1)):
            x = torch.randn(n, generator=g).to(TORCH[dtype])
            if threshold == 65536:
                x[0] = float("nan")                             # dropped: contributes 0 all the same
                x[n // 2] = float("inf")
            r = torch.randn(n, generator=g).to(TORCH[dtype]) if residual else None
            got = run(exe, tmp_path, x, [r] if residual else [], mem, threshold, grid, off)
            with np.errstate(invalid="ignore"):
                want = S.dropout(x.double().numpy(), threshold, seed, offset, None if r is None else r.double().numpy())
            # fp32 roundings: the scale, the product, the sum; then the storage
            mag = np.abs(want) + (0 if r is None else np.abs(want - r.double().numpy()) + np.abs(r.double().numpy()))
            tol = (3 * 2.0 ** -24 + (0 if dtype == "fp32" else HALF_STEP[dtype])) * mag + HALF_STEP_SUBNORMAL[dtype]
            assert np.all(np.abs(got.double().numpy() - want) <= tol), (n, grid, off, threshold)


@needs_clang
@pytest.mark.parametrize("dtype,d,sections,order,variant", [
    ("bf16", 128, (16, 24, 24), "blocks", 0), ("bf16", 128, (24, 20, 20), "turns", 1), ("fp32", 72, (13, 23), "blocks", 0),
    ("fp16", 64, (1, 30, 1), "turns", 32), ("fp32", 8, (1, 1, 2), "blocks", 33), ("bf16", 80, (40,), "blocks", 0), ("bf16", 512, (100, 100, 56), "blocks", 0)])
def test_rope_axes_header_on_cpu(lib, tmp_path, dtype, d, sections, order, variant):
    """Interleaved pairs (half-split pairs exchange lanes).  The table is exactly as long as its rows, so a
    position outside that was followed would trip the sanitizer."""
    for backward in (False, True):
        exe = build_driver(lib, tmp_path, headers.rope_axes_header(d, sections, dtype, False, order, backward), variant)
        g = torch.Generator().manual_seed(d)
        rows = 9
        table = torch.randn(rows, d, generator=g)
        for tokens, heads, grid, off in ((1, 1, 0, 0), (3, 5, 16, 32), (37, 3, 0, 4096), (70, 8, 8, 0)):
            x = torch.randn(tokens, heads, d, generator=g).to(TORCH[dtype])
            pos = torch.randint(0, rows, (tokens, len(sections)), generator=g, dtype=torch.int32)
            pos[tokens // 2, -1] = rows                          # outside: just behind, far behind, negative
            pos[0, 0] = 2 ** 31 - 1
            if tokens > 2:
                pos[2, 0] = -1
            got = run(exe, tmp_path, x, [table], pos, headers.rope_axes_sideband(heads, rows), grid, off).double().numpy()
            want = S.rope_axes(x.double().numpy(), table.double().numpy(), pos.numpy(), sections, False, order, backward)
            assert np.array_equal(np.isnan(got), np.isnan(want))
            # two products and a sum in fp32, then the storage; |x1 c| + |x2 s| <= |x| |table| maxima
            scale = 2 * float(x.float().abs().max()) * float(table.abs().max())
            tol = 3 * 2.0 ** -24 * scale + (0 if dtype == "fp32" else HALF_STEP[dtype]) * np.abs(want) * 1.01 + HALF_STEP_SUBNORMAL[dtype]
            assert np.all(np.isnan(want) | (np.abs(got - want) <= tol))


def test_pair_axes():
    for sections, order in (((16, 24, 24), "blocks"), ((24, 20, 20), "turns"), ((1, 30, 1), "turns"), ((3, 5), "turns"), ((7,), "blocks")):
        assert headers.rope_pair_axes(sections, order) == S.pair_axes(sections, order)
    assert headers.rope_pair_axes((3, 1, 2), "turns") == [0, 1, 2, 0, 2, 0]


def test_axes_table():
    table = ops.freqs_cis_axes_table((2, 2), 5, 100.0)
    want = np.array([[[np.cos(t * f), np.sin(t * f)] for f in (1.0, 0.1, 1.0, 0.1)] for t in range(5)])
    assert np.abs(table.double().numpy() - want.reshape(5, 8)).max() <= 2.0 ** -24
    turns = ops.freqs_cis_axes_table((2, 2), 5, 100.0, order="turns")
    assert torch.equal(turns[:, 2:4], table[:, 0:2]) and torch.equal(turns[:, 4:6], table[:, 2:4])


def test_header_refusals():
    for bad in (dict(head_dim=64, sections=(16, 17)), dict(head_dim=64, sections=(8, 8, 8, 8)), dict(head_dim=64, sections=(33, -1)),
                dict(head_dim=64, sections=(16, 16), order="rows"), dict(head_dim=64, sections=(16, 16), dtype="fp64"),
                dict(head_dim=80, sections=(20, 20), half=True), dict(head_dim=36, sections=(9, 9)), dict(head_dim=1024, sections=(256, 256))):
        with pytest.raises(ValueError):
            headers.rope_axes_header(**bad)
    for heads, rows in ((0, 4), (1024, 4), (4, 0), (4, 1 << 22)):
        with pytest.raises(ValueError):
            headers.rope_axes_sideband(heads, rows)
    word = headers.rope_axes_sideband(1023, (1 << 22) - 1)
    assert -2 ** 31 <= word < 2 ** 31 and word & 0xFFFFFFFF == 0xFFFFFFFF
    with pytest.raises(ValueError):
        headers.dropout_header("fp64")
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout_threshold(p)
    assert [ops.dropout_threshold(p) for p in (0.0, 0.1, 0.5, 1.0)] == [0, 6554, 32768, 65536]


def test_op_refusals_need_no_device():
    x = torch.zeros(2, 3, 4, 64)
    freqs, pos = torch.zeros(10, 64), torch.zeros(2, 3, 2, dtype=torch.int32)
    for args in ((x, freqs[:, :32], pos, (16, 16)), (x, freqs.double(), pos, (16, 16)), (x, freqs, pos.long(), (16, 16)),
                 (x, freqs, pos[:1], (16, 16)), (x, freqs, pos, (16, 8, 8)), (x[0], freqs, pos, (16, 16)),
                 (x, freqs, torch.zeros(2, 3, 4, dtype=torch.int32)[..., ::2], (16, 16))):
        with pytest.raises(AssertionError):
            ops.rope_axes_forward(*args)
    with pytest.raises(TypeError):
        ops.rope_axes_forward(x.double(), freqs, pos, (16, 16))
    with pytest.raises(AssertionError):
        ops.rope_axes_forward_many([x, x.half()], freqs, pos, (16, 16))
    with pytest.raises(AssertionError):
        ops.rope_axes_forward(x, freqs, pos, (16, 16), out=x.half())
    seed = torch.zeros(2, dtype=torch.int64)
    for args, kw in (((x, 0.1, seed.int()), {}), ((x, 0.1, seed[:1]), {}), ((x, 0.1, seed), {"residual": x[:1]}),
                     ((x, 0.1, seed), {"out": x.half()}), ((x, 0.1, torch.zeros(4, dtype=torch.int64)[::2]), {})):
        with pytest.raises(AssertionError):
            ops.dropout_forward(*args, **kw)
    with pytest.raises(TypeError):
        ops.dropout_forward(x.int(), 0.1, seed)
    with pytest.raises(ValueError):
        ops.dropout_forward(x, 1.5, seed)


@pytest.mark.parametrize("variant", [0, 1, 2, 4, 16, 33])
def test_headers_compile_for_gfx950(lib, variant):
    log = ctypes.create_string_buffer(1 << 16)
    for header in (headers.dropout_header("bf16", True), headers.dropout_header("fp32"), headers.rope_axes_header(128, (16, 24, 24)),
                   headers.rope_axes_header(128, (24, 20, 20), "fp32", True, "turns", True),
                   headers.rope_axes_header(72, (13, 23), "fp16", False)):
        assert lib.sideaware_compile_check(header, variant, log, len(log)) == 0, log.value.decode()
        assert log.value == b""
