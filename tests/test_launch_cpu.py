"""The launches' host side and order, without a GPU."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "libnrn_b200", "csrc")


@pytest.mark.parametrize("name", ["linattn.cu", "scaled.cu", "gatednorm.cu"])
def test_no_kernel_lets_the_next_in_before_it_has_its_tmem(name):
    """tcgen05.alloc waits for columns without a limit: a block of the next kernel, on the same SM, could take them and wait
    for this one."""
    src = open(os.path.join(CSRC, name)).read()
    for kernel in re.split(r"\n(?=__global__)", src)[1:]:
        alloc = kernel.find("tcgen05.alloc")
        if alloc < 0:
            continue
        body = kernel[:alloc]
        for at in (m.start() for m in re.finditer(r"\blet_next\(\)", body)):
            # only where the block ends without any
            assert re.match(r"let_next\(\);\s*previous_done\(\);\s*return;", body[at:]), f"{name}: let_next before tcgen05.alloc"
        assert re.search(r"\blet_next\(\)", kernel[alloc:])
