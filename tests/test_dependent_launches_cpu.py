"""Kernels that are launched as programmatic dependents run beside the kernel before them until their
``griddepcontrol.wait``.  The read-only path (``__ldg``) is for memory that nothing writes while a kernel lives, so such a
kernel may take by it what was complete before the chain began, the caller's tensors, and nothing that the chain
itself writes."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "neural_scaling_weather_b200" / "ops" / "csrc"

# operands of the waiting kernels that are the caller's: tokens (p, x, the attention's base), residual, weights, and in the
# gather the experts' outputs (read in the backward alone, whose launch is an ordinary one)
CALLERS = {"p", "x", "base", "res", "wg", "wu", "w", "w0", "w1", "other"}


def kernels(text):
    """(name, body) of the kernels of a source file."""
    for m in re.finditer(r"__global__\s+void\s+(?:__\w+__\([^()]*(?:\([^()]*\))?[^()]*\)\s*)*(\w+)\(", text):
        at = text.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        yield m.group(1), text[at:end]


WAITING = [(f.name, name, body) for f in sorted(CSRC.glob("*.cu")) for name, body in kernels(f.read_text())
           if "griddepcontrol.wait" in body]


def test_the_waiting_kernels_are_found():
    assert {name for _, name, _ in WAITING} >= {"gather_kernel", "combine_kernel", "few_down_kernel", "split_kernel",
                                                "skinny_kernel"}


@pytest.mark.parametrize("file,name,body", WAITING, ids=[f"{f}:{n}" for f, n, _ in WAITING])
def test_the_chain_is_read_by_ordinary_loads(file, name, body):
    read_only = re.findall(r"__ldg\((?:reinterpret_cast<[^>]*>\()?\s*(\w+)", body)
    read_only += re.findall(r"(?:row8|load8)<\w+, true>\(\s*(\w+)", body)
    assert set(read_only) <= CALLERS, f"{file}: {name}"
    # a helper without the second argument would take the read-only path unsaid
    assert not re.search(r"row8<\w+>\(", body), f"{file}: {name}"
