"""The device status word names one kernel: (kernel id << 16) | site."""
import collections
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "torchpairwise_b200" / "csrc"


def test_no_two_kernels_report_the_same_code():
    codes, owners = collections.Counter(), collections.defaultdict(set)
    for path in sorted(CSRC.glob("*.cu*")):
        for found, site in re.findall(r"atomicCAS\([^;]*?\(([^;]*?) << 16\) \| (\w+)\)", path.read_text()):
            for number in re.findall(r"\d+", found):   # `(A ? 20 : 21)` has two
                codes[int(number), site] += 1
                owners[int(number)].add((path.name, site == "site"))
    assert len(owners) >= 12
    assert all(n == 1 for n in codes.values()), {c: n for c, n in codes.items() if n > 1}
    # where the site is a variable, the id is that kernel's alone
    for number, where in owners.items():
        assert len(where) == 1 or not any(variable for _, variable in where), (number, where)
