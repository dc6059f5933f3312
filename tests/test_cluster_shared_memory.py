"""A CTA may touch the shared memory of another one of its cluster when it knows that that one has started: behind a cluster barrier.  Read from
the sources, since a CTA that starts late enough to show it cannot be arranged."""
import os
import re

import pytest
from conftest import ROOT

CSRC = os.path.join(ROOT, "mytorch_b200", "csrc")
WAIT = re.compile(r"cluster\.sync\(\)|cluster_wait\(\)|barrier_wait\(")
REMOTE = re.compile(r"map_shared_rank\(")


def _functions(text):
    """(name, body) of what a source file defines at a line's beginning, without its comments."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/|__launch_bounds__\([^)]*\)", "", text, flags=re.S)
    for m in re.finditer(r"^(?:template [^\n]*\n)?(?:__global__|__device__)[^;{]*?(\w+)\(", text, flags=re.M):
        begin = text.index("{", m.end())
        depth, at = 0, begin
        while True:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            if depth == 0:
                break
            at += 1
        yield m.group(1), text[begin:at]


def _remote_functions():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            for function, body in _functions(open(os.path.join(CSRC, name)).read()):
                if REMOTE.search(body):
                    yield pytest.param(body, id=f"{name}-{function}")


@pytest.mark.parametrize("body", list(_remote_functions()))
def test_no_remote_access_before_a_cluster_barrier(body):
    waits = [m.start() for m in WAIT.finditer(body)]
    assert waits and waits[0] < REMOTE.search(body).start()


def test_the_kernels_are_found():
    assert len(list(_remote_functions())) >= 3
