"""The build refuses a kernel whose split of the registers would not add up: a compiler that gives it another number of them."""
import os
import re

import pytest

from flashck_b200 import build


def _log(*counts, kernel="_ZN3fck19splitkv_int4_kernelI6__halfLi128ELi1ELi2EEEv14CUtensorMap_st"):
    return "".join(f"ptxas info    : Compiling entry function '{kernel}{i}' for 'sm_100a'\nptxas info    : Function properties for {kernel}{i}\n"
                   f"    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\nptxas info    : Used {n} registers, used 2 barriers\n"
                   f"ptxas info    : Compile time = 900.0 ms\n" for i, n in enumerate(counts))


def test_counts_that_add_up():
    build.check_registers("splitkv_int4.cu", _log(96) + _log(40, kernel="another") + _log(96, 96))
    build.check_registers("combine.cu", "anything")


@pytest.mark.parametrize("log", [_log(96, 88), _log(128), _log(96) + _log(255), _log(96, kernel="another"), ""])
def test_others_are_refused(log):
    with pytest.raises(RuntimeError, match="96 registers"):
        build.check_registers("splitkv_int4.cu", log)


def test_the_source_counts_on_the_same_number():
    with open(os.path.join(build.CSRC, "splitkv_int4.cu")) as f:
        text = f.read()
    consumers, = re.findall(r"kConsumers = (\d+)", text)
    assert "kThreads = (kConsumers + 4) * 32, kLaunch = 65536 / kThreads / 8 * 8" in text
    assert build._REGISTERS["splitkv_int4.cu"] == ("splitkv_int4_kernel", 65536 // ((int(consumers) + 4) * 32) // 8 * 8)
