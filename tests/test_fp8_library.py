"""The library of the 8-bit rows is loaded by what needs it: layer calls of 16 and 32 bits work without it, 8-bit ones say what is missing."""
import os
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def run(code, **env):
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, **env}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout


def test_other_calls_do_not_load_it():
    out = run("from jacobiforcing_amd import _native as N, layer_ops as LO\n"
              "h = LO._host()\n"
              "print(isinstance(h, N._NoHost), 'layers_fp8' in N.layers()._libs)\n"
              "N.host_fp8(h)\n"
              "print('layers_fp8' in N.layers()._libs)\n")
    assert out.split() == ["False", "False", "True"]


def test_without_it_only_its_own_calls_fail(tmp_path):
    out = run("import torch\n"
              "from jacobiforcing_amd import _native as N, layer_ops as LO\n"
              "print(isinstance(LO._host(), N._NoHost))\n"
              "x = torch.zeros(2, 128)\n"
              "print(LO._H.quantize_fp8(x, torch.float32) is NotImplemented)\n"
              "for call in (lambda: LO.quantize_fp8(x), lambda: N.layers().jl_linear_fp8_floats(None)):\n"
              "    try:\n"
              "        call()\n"
              "    except N.NativeLibraryError as e:\n"
              "        print('missing.so' in str(e))\n", JF_LAYERS_FP8_LIB=str(tmp_path / "missing.so"))
    assert out.split() == ["False", "True", "True", "True"]
