"""CPU: the forms of the cross entropy operator's kernels for few rows that the library holds are those that a call can reach.
Rows of bf16 come there up to 16 at a time, one half of a 32-row tile; rows of fp32 up to 32."""
import os
import re

import pytest

from test_kloop_asm import CSRC

LIB = os.path.join(CSRC, "libaslhip.so")


@pytest.mark.parametrize("kernel", ["logits", "rest", "grad"])
def test_forms_for_few_rows(kernel):
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    name = f"xent_few_{kernel}_kernel"
    with open(LIB, "rb") as f:
        forms = set(re.findall(rb"_ZN10asl_detail%d%sI([sf])Li(\d)EE" % (len(name), name.encode()), f.read()))
    assert forms == {(b"s", b"1"), (b"f", b"1"), (b"f", b"2")}
