"""CPU: no kernel touches another CTA's shared memory before the cluster has met.

CUDA asks that every CTA of a cluster is known to have started before its
shared memory is accessed by another. A run cannot show the lack of it (a late
CTA's start is a matter of luck), so the sources are read: in each function the
first access through map_shared_rank comes after a cluster barrier."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "sepia_b200" / "csrc"
MEET = re.compile(r"\bcl\.(?:sync|barrier_wait)\(\)")
# a store or load through the mapped pointer, on the spot or by a name that was given to it
ON_THE_SPOT = re.compile(r"\*\s*cl\.map_shared_rank\(|map_shared_rank\([^;]*?\)\s*->|map_shared_rank\([^;]*?\)\s*\[")
NAMED = re.compile(r"\*\s*(?:const\s+)?(\w+)\s*=\s*cl\.map_shared_rank\(")


def functions(text):
    """(name, body) of the functions at the top level of a file."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/|__launch_bounds__\([^)]*\)", "", text, flags=re.S)
    for m in re.finditer(r"(\w+)\s*\([^;{}]*\)\s*(?:const\s*)?\{", text):
        if m.group(1) in ("if", "for", "while", "switch"):
            continue
        depth, i = 1, m.end()
        while depth and i < len(text):
            depth += (text[i] == "{") - (text[i] == "}")
            i += 1
        if "map_shared_rank" in text[m.end():i]:
            yield m.group(1), text[m.end():i]


CASES = [(p.name, name, body) for p in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]) for name, body in functions(p.read_text())]


def test_there_are_cluster_kernels():
    assert {"sample.cu", "model.cu"} <= {file for file, _, _ in CASES}


@pytest.mark.parametrize("file,name,body", CASES, ids=[f"{file}-{name}" for file, name, _ in CASES])
def test_cluster_meets_before_remote_access(file, name, body):
    uses = [m.start() for m in ON_THE_SPOT.finditer(body)]
    for m in NAMED.finditer(body):
        uses += [m.end() + u.start() for u in re.finditer(rf"\b{m.group(1)}\s*(?:->|\[)", body[m.end():])]
    met = MEET.search(body)
    assert uses and met and met.start() < min(uses), (file, name)
