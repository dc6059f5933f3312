"""A word of shared memory that all warps of a CTA read, to decide by, is written again only behind a barrier that follows the read: a warp that comes late would
read the new value, take another branch than the others and miss their barriers.  Read from the sources, since a warp that is late enough to show it cannot be arranged."""
import os
import re

import pytest
from conftest import ROOT
from test_cluster_shared_memory import _functions

CSRC = os.path.join(ROOT, "mytorch_b200", "csrc")
BARRIER = re.compile(r"\bmeet<\w+>\(\)|__syncthreads\(\)|cluster\.sync\(\)")
READ = re.compile(r"=\s*shared\.(\w+);")


def _reads():
    """(source file, function, word, what stands between a read of it and the next plain store to it)"""
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            text = open(os.path.join(CSRC, name)).read()
            text = re.sub(r"^template <int W, class F>\n", "", text, flags=re.M)
            for function, body in _functions(text):
                for k, m in enumerate(READ.finditer(body)):
                    store = re.compile(rf"shared\.{m.group(1)} = ").search(body, m.end())
                    if store:
                        yield pytest.param(body[m.end() : store.start()], id=f"{name}-{function}-{m.group(1)}-{k}")


@pytest.mark.parametrize("between", list(_reads()))
def test_a_barrier_lies_between_a_read_and_the_next_store(between):
    assert BARRIER.search(between)


def test_the_reads_are_found():
    assert any("token_log_probs.cu-look-candidates" in p.id for p in _reads())
