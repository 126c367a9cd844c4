"""The build's check of the registers that kernels must be launched with (CPU only)."""
import pytest

from loom_skills_b200 import build as B

LINES = """ptxas info    : 0 bytes gmem
ptxas info    : Compiling entry function '_ZN2lk5k_mvxILi2EEEvi' for 'sm_100a'
ptxas info    : Function properties for _ZN2lk5k_mvxILi2EEEvi
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used {} registers, used 2 barriers, 480 bytes cumulative stack size
ptxas info    : Compiling entry function '_ZN2lk5otherEvi' for 'sm_100a'
ptxas info    : Function properties for _ZN2lk5otherEvi
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used 8 registers, used 0 barriers
"""


def test_enough():
    B.check_registers("lk_mvx.cu", LINES.format(96))


@pytest.mark.parametrize("text", [LINES.format(95), "", LINES.format(96).replace("k_mvx", "k_new"),
                                  LINES.format(96).replace("Used 8 registers", "")])
def test_too_few_or_none_reported(text):
    with pytest.raises(RuntimeError):
        B.check_registers("lk_mvx.cu", text)


def test_the_limit_is_the_kernels():
    import os
    import re
    text = open(os.path.join(B.CSRC, "lk_mvx.cu")).read()
    assert int(re.search(r"kLaunchRegs = (\d+)", text).group(1)) == B.LAUNCH_REGISTERS["lk_mvx.cu"][1]
    assert set(B.LAUNCH_REGISTERS) <= set(B.SOURCES)
