"""Non-coherent loads (__ldg, ld.global.nc) are for memory that nothing writes while the kernel lives.  A grid of the W8A8 chain starts while the kernel
in front writes its rows, so only weights may be read that way.  (No run can show a load that the compiler moved in front of the wait: the source is looked at.)"""
import os
import re

from chimere_b200 import build


def test_only_weights_are_read_by_non_coherent_loads():
    with open(os.path.join(build.CSRC, "w8a8.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    found = [m.start() for m in re.finditer(r"__ldg\(|ld\.global\.nc|__ldlu\(|tex1Dfetch", code)]
    assert len(found) == 1
    statement = code[found[0]:code.index(";", code.index('"l"(', found[0]))]
    assert '"l"(wr[' in statement          # (wr: a lane's rows of the weights)
    assert not re.search(r"__restrict__", code)     # (with const __restrict__ the compiler chooses such loads itself)
