"""Loads from tensor memory, checked in the sources."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparseconvnet_b200", "csrc")


def test_what_reads_tensor_memory_stays_behind_the_wait():
    """The registers of a tcgen05.ld hold nothing before tcgen05.wait::ld, and the compiler orders what reads them by the statements that
    name them only: a wait stands in the load's own statement, or it is told the registers of every load before it."""
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        text = re.sub(r"//.*", "", open(path).read())
        if "tcgen05.ld" in text:
            for m in re.finditer(r"tcgen05\.ld\.", text):
                function = re.findall(r"\bvoid (\w+)\(", text[:m.start()])[-1]
                statement = text[text.rindex("asm volatile(", 0, m.start()):text.index(";\n", text.index('"r"(', m.start()))]
                assert ("tcgen05.wait::ld" in statement) != function.endswith("_nowait"), (path, function)
        if not path.endswith("tc_ptx.cuh"):
            loaded = {r.strip() for r in re.findall(r"\btmem_ld\d+_nowait\([^;]*,([^;,]*)\);", text)}
            told = [{r.strip() for r in call.split(",")} for call in re.findall(r"\btmem_wait_ld\(([^;]*)\);", text)]
            assert {""} not in told and loaded == set().union(*told), path
