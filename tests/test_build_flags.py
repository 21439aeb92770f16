"""What every kernel of the two libraries is compiled with, from the compile lines that make would run."""
import os
import re
import subprocess

import pytest

PACKAGE = os.path.abspath(os.path.join(os.path.dirname(__file__), "..", "chatterbox_vllm_amd"))


@pytest.mark.parametrize("sub", ["csrc", "csrc_s3gen"])
@pytest.mark.parametrize("given", [[], ["EXTRA=-DONE"], ["EXTRA=-DONE", "PRELOAD=", "BUILD=build_x"]])
def test_no_kernel_has_packed_fp32_instructions(sub, given):
    lines = subprocess.run(["make", "-n", "-B", "-C", os.path.join(PACKAGE, sub), *given], capture_output=True, text=True, check=True).stdout.splitlines()
    lines = [x for x in lines if re.search(r" -c \w+\.hip ", x)]
    assert {re.search(r" -c (\w+\.hip) ", x)[1] for x in lines} == {x for x in os.listdir(os.path.join(PACKAGE, sub)) if x.endswith(".hip")}
    for x in lines:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in x and "--offload-arch=gfx950" in x, x
        assert ("-DONE" in x) == (len(given) > 0) and ("-fno-slp-vectorize" in x) == ("cfm_split.hip" in x), x
