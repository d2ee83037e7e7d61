"""A kernel's limit of shared memory, where threads may launch it in other sizes at the same time."""

import os
import re

from lily_b200.csrc import build


def test_the_weighed_decode_raises_its_limit_to_one_number():
    """A limit that follows the call's size can be lowered by another thread between being raised and the launch."""
    with open(os.path.join(build.HERE, "attention_weighed.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    raised = re.findall(r"cudaFuncAttributeMaxDynamicSharedMemorySize,\s*([^;]*?)\)\s*(?:!=|;)", text)
    assert len(raised) == 3
    for size in raised:
        assert re.fullmatch(r"\(int\)most_smem<D, CLUSTER>\(\)|most", size.strip()), size
    assert re.search(r"const int most = \(int\)\(weighed::simt_floats\(256\) \* sizeof\(float\)\);", text)
