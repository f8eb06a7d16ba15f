"""CPU: the assembly checks of the convolution kernels on the code that ships.  The library is compiled with flags of its makefile
that the checks' own compile lines do not name; here the same checks run with them."""
import importlib.util
import os
import re
import subprocess
import types

from test_kloop_asm import CSRC, HIPCC

HERE = os.path.dirname(os.path.abspath(__file__))
FLAGS = re.search(r"^NO_PACKED_FP32 = (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()


def _run(cmd, **kw):
    return subprocess.run([cmd[0]] + FLAGS + cmd[1:] if cmd[0] == HIPCC else cmd, **kw)


def _shipped(name):
    spec = importlib.util.spec_from_file_location("shipped_" + name, os.path.join(HERE, name + ".py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.subprocess = types.SimpleNamespace(run=_run, PIPE=subprocess.PIPE, CalledProcessError=subprocess.CalledProcessError)
    return module


_kloop, _stem, _block = _shipped("test_kloop_asm"), _shipped("test_stem_asm"), _shipped("test_block_asm")
tmp, asm = _kloop.tmp, _stem.asm
test_stem3d_k_loop, test_large_tile_k_loop = _kloop.test_stem3d_k_loop, _kloop.test_large_tile_k_loop
test_stem_strip_vector_memory_stream = _stem.test_stem_strip_vector_memory_stream
test_block_kernel_k_loops = _block.test_block_kernel_k_loops


def test_every_source_is_compiled_with_them():
    lines = subprocess.run(["make", "-n", "-B", "-C", CSRC], check=True, capture_output=True, text=True).stdout.splitlines()
    compiles = [line for line in lines if " -c " in line]
    assert len(compiles) == len([f for f in os.listdir(CSRC) if f.endswith(".hip")]) and all(" ".join(FLAGS) in line for line in compiles)
