"""What the kernels' sources have to say to the compiler."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "artdeco_amd", "csrc")


def test_inline_assembly_that_writes_m0_says_so():
    """The compiler otherwise takes m0 as kept across the statement."""
    writes = re.compile(r"\bs_\w+ m0,")
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        for statement in re.findall(r"\basm\b(?: volatile)?\s*\((.*?)\);", open(path).read(), flags=re.S):
            if writes.search(statement):
                found += 1
                assert '"m0"' in statement, (path, statement)
    assert found
