"""What the kernels' sources have to say to the compiler: without a GPU."""
import glob
import os
import re

import bitween_amd as bw


def test_assembly_names_the_registers_that_it_writes():
    """The compiler keeps an address of LDS in M0 where it likes to: assembly that writes it says so."""
    found = 0
    for path in glob.glob(os.path.join(os.path.dirname(bw.__file__), "csrc", "*.h*")):
        with open(path) as f:
            for statement in re.findall(r"asm volatile\((.*?)\);", f.read(), re.S):
                if "m0," in statement.split(":")[0]:
                    found += 1
                    assert '"m0"' in statement.split(":")[-1], (path, statement)
    assert found
