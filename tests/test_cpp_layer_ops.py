"""The layer operators through the C++ mirror (include/larql_backend.hpp): it compiles without warnings, links, and gives the
formula's results on a GPU."""
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import larql_b200
from larql_b200 import build as lqbuild
from test_layer_ops import fp8_tolerance, fp8_want, fp8_weight, gen, quantized

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    lqbuild.build()
    out = tmp_path_factory.mktemp("cpp") / "layer_ops_check"
    lib_dir = Path(larql_b200.LIB_PATH).parent
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(ROOT / "tests/cpp/layer_ops_check.cpp"),
                    "-L", str(lib_dir), "-llarql_b200", f"-Wl,-rpath,{lib_dir}", "-o", str(out)], check=True, capture_output=True, text=True)
    return out


def test_the_mirror_compiles_and_has_no_cpu_fallback(exe):
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == (0 if torch.cuda.is_available() else 3)


@pytest.mark.gpu
def test_fp8_product_through_the_mirror(exe, tmp_path):
    rows, cols, t = 200, 320, 9
    wq, ws = fp8_weight(gen(3), rows, cols)
    x = torch.randn(t, cols, generator=gen(4))
    (tmp_path / "in.bin").write_bytes(np.array([rows, cols, t, 0], np.int32).tobytes() + wq.view(torch.uint8).numpy().tobytes() +
                                      ws.numpy().tobytes() + x.numpy().tobytes())
    r = subprocess.run([str(exe), str(tmp_path / "in.bin"), str(tmp_path / "out.bin")], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)
    got = torch.from_numpy(np.fromfile(tmp_path / "out.bin", np.float32).reshape(t, rows)).double()
    want, mag = fp8_want(*quantized(x), wq, ws)
    assert ((got - want).abs() <= fp8_tolerance("f32", want, mag, cols)).all()
