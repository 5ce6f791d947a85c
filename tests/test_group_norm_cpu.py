"""Group norm without a GPU: the plan that cuts the work (every size it may be given stays inside LDS,
workspace and grid), the oracle's gradients against differences, and refusals."""
import os
import random
import re
import subprocess

import numpy as np
import pytest
import torch

import stream_ops_oracle as S
from l2_torch_alloc_amd import build as sa_build
from l2_torch_alloc_amd import ops, wrapper

HERE = os.path.dirname(os.path.abspath(__file__))


def check_plans(tmp_path, text, cases):
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", os.path.join(HERE, "native", "group_norm_plan_main.cpp"),
                    "-o", exe], check=True, capture_output=True, text=True)
    proc = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and "ok" in proc.stdout, proc.stdout + proc.stderr
    assert "cases=%d " % cases in proc.stdout
    return int(re.search(r"one_launch=(\d+)", proc.stdout)[1])


def test_plan(tmp_path):
    rng = random.Random(5)
    cases = [(1, 1, 1, 1), (1, 1, 8192, 1), (1, 7, 8191, 1), (65536, 1, 320, 32), (1, 1 << 20, 512, 32), (2, 64, 1280, 32), (1, 3, 65536, 65536),
             (1, 5, 65536, 1), (16, 1024, 640, 32), (1, 1 << 26, 1, 1), (3, 999, 33, 33), (1 << 20, 1, 8, 2), (1, 262144, 256, 32), (4, 100, 30000, 3)]
    for _ in range(3000):
        groups = rng.choice([1, 2, 3, 4, 7, 8, 16, 32, 64, 100, 257, 512])
        channels = groups * rng.choice([1, 1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 33, 40, 64, 129, 1024])
        cases.append((int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 20)), channels, groups))
    text = "".join("%d %d %d %d %d %d\n" % (c + (rng.choice([2, 4]), rng.choice([0, 1]))) for c in cases)
    check_plans(tmp_path, text, len(cases))


def test_plan_of_many_samples(tmp_path):
    """Where one launch takes pieces of rows that do not fit a workgroup's own caches: vectors of every width, pixels up to
    what a lane may add."""
    rng = random.Random(6)
    cases = []
    for _ in range(3000):
        groups = rng.choice([1, 2, 3, 8, 32])
        channels = groups * rng.choice([1, 2, 3, 8, 10, 20, 33, 40, 65])
        cases.append((int(2 ** rng.uniform(3, 9)), int(2 ** rng.uniform(5, 13)), channels, groups))
    cases += [(16, 1024, 640, 32), (256, 3971, 33, 1), (256, 4096, 32, 1), (512, 1985, 33, 1), (128, 700, 66, 3)]
    text = "".join("%d %d %d %d %d %d\n" % (c + (rng.choice([2, 4]), rng.choice([0, 1]))) for c in cases)
    assert check_plans(tmp_path, text, len(cases)) > 500


@pytest.mark.parametrize("activation", ["none", "silu"])
def test_oracle_gradients_against_differences(activation):
    rng = np.random.default_rng(1)
    N, P, C, G, eps, step = 2, 5, 12, 3, 1e-5, 1e-6
    x, w, b = rng.normal(size=(N, P, C)) + 0.5, rng.normal(size=C), rng.normal(size=C)
    dout = rng.normal(size=(N, P, C))
    y, stats = S.group_norm(x, w, b, G, eps, activation)
    grads = S.group_norm_backward(dout, x, w, b, stats, G, activation)
    for at, (value, grad) in enumerate(zip((x, w, b), grads)):
        for _ in range(20):
            v = rng.normal(size=value.shape)
            args_up, args_down = [x, w, b], [x, w, b]
            args_up[at], args_down[at] = value + step * v, value - step * v
            up, down = (float((S.group_norm(*a, G, eps, activation)[0] * dout).sum()) for a in (args_up, args_down))
            # central differences: a third derivative times step^2 (about 1e-12 of it), and 2^-53 of the sums over step
            assert abs((up - down) / (2 * step) - float((grad * v).sum())) <= 1e-7 * (1 + abs(float((grad * v).sum())))


def test_refusals_need_no_device(monkeypatch):
    x, w = torch.zeros(2, 3, 3, 8), torch.ones(8)
    for args, kw, error in (((x, w, w, 3), {}, ValueError), ((x, w, w, 0), {}, ValueError), ((x.double(), w, w, 2), {}, TypeError),
                            ((x, w, w, 2), {"activation": "tanh"}, ValueError), ((x, w[:4], w, 2), {}, AssertionError),
                            ((x, w.half(), w, 2), {}, AssertionError), ((x.half(), w.bfloat16(), None, 2), {}, AssertionError),
                            ((x[0, 0, 0], w, w, 2), {}, AssertionError), ((x[:, :0], w, w, 2), {}, ValueError),
                            ((x, w, w, 2), {"out": x[:1]}, AssertionError), ((x, w, w, 2), {"stats": torch.zeros(2, 3, 2)}, AssertionError)):
        with pytest.raises(error):
            ops.group_norm_forward(*args, **kw)
    stats = torch.zeros(2, 2, 2)
    for args, kw in (((x[:1], x, w, w, stats, 2), {}), ((x, x, w, w, stats[:1], 2), {}), ((x, x, w, w, stats.double(), 2), {}),
                     ((x, x, None, w, stats, 2), {"dweight": w}), ((x, x, w, w, stats, 2), {"dbias": w.half()})):
        with pytest.raises(AssertionError):
            ops.group_norm_backward(*args, **kw)
    # a tensor of a type, shape or place that does not fit is found before the library is asked
    with pytest.raises(AssertionError):
        ops.group_norm_forward(x.transpose(0, 1), w, w, 2)          # not on a GPU
    # under capture with this library's allocator nothing is allocated behind the caller's back
    monkeypatch.setattr(wrapper, "_allocator_installed", True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        ops.group_norm_forward(x, w, w, 2)
    with pytest.raises(RuntimeError, match="capture"):
        ops.dropout_forward(x, 0.5, torch.zeros(2, dtype=torch.int64))


def test_empty_batch():
    x, w = torch.zeros(0, 4, 8), torch.ones(8)
    y, stats = ops.group_norm_forward(x, w, w, 2)
    assert y.shape == x.shape and stats.shape == (0, 2, 2)
    dx, dw, db = ops.group_norm_backward(x, x, w, None, stats, 2)
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros(8)) and db is None


def test_built_library_has_the_entry_points():
    lib = wrapper.bind(sa_build.build_library(force=False))
    assert lib.sideaware_group_norm_workspace(1, 1, 8, 3, 0, 0, -1) == 0
    assert b"groups divide" in lib.sideaware_last_error()
    assert lib.sideaware_group_norm_workspace(1, 1, 8, 2, 7, 0, -1) == 0
    assert b"unknown type" in lib.sideaware_last_error()
    lib.sideaware_clear_error()
