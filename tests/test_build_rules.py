"""CPU: objects are compiled anew when what they were compiled with changes, the makefile's own flags among it."""
import os
import subprocess

import pytest

from test_kloop_asm import CSRC, HIPCC


@pytest.mark.parametrize("changed", ["Makefile", "xent_args.h", "train_common.h", "common.h"])
def test_objects_depend_on(changed):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not present")
    out = subprocess.run(["make", "-n", "-C", CSRC, "-W", changed], check=True, capture_output=True, text=True).stdout
    sources = [f for f in os.listdir(CSRC) if f.endswith(".hip")]
    assert all(f" -c {f} " in out for f in sources)
