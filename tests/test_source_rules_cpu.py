"""Rules of the kernels' sources that no run can show broken for certain; no GPU needed."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crispasr_b200", "csrc")


def test_no_wait_is_taken_as_over_because_another_lane_saw_it():
    """A lane reads what an asynchronous copy brought only behind its own successful wait on the copy's barrier: a vote that any lane's wait
    succeeded hands none of that lane's order to the others."""
    waits = 0
    for f in sorted(os.listdir(CSRC)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, f)).read())
        waits += text.count("mbar_try_wait(")
        for m in re.finditer(r"__any_sync\(([^;]*);", text):
            assert "mbar_try_wait" not in m.group(1), f"{f}: {m.group(0)}"
    assert waits
