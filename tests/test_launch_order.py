"""The kernels' programmatic launches, read from their sources: every kernel lets its dependents start after its own wait, in
each of its roles. What a kernel reads before its wait rests on that: it then has to be untouched by the kernel launched just
before it only, not by those before that one."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "whisper-trt_b200" / "csrc"


def test_kernels_trigger_after_their_wait():
    seen = 0
    for path in sorted(CSRC.glob("*.cu")):
        for body in path.read_text().split("__global__")[1:]:
            calls = re.findall(r"\b(pdl_wait|pdl_launch_dependents)\(\)", body)
            waited = False
            for call in calls:
                if call == "pdl_wait":
                    waited = True
                else:
                    assert waited, f"{path.name}: {body.split('{')[0].strip()[:120]} triggers before it waits"
                    waited, seen = False, seen + 1
    assert seen > 20
