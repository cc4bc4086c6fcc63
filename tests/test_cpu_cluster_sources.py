"""Kernels that write into the shared memory of another block of their cluster.  That block has to have started: each arrives at a cluster
barrier on entry and waits for the others before its first access.  A missing barrier shows on a GPU only now and then, and then as a fault,
so this reads the sources."""
import glob
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "haste_b200", "csrc")


def _functions_with(text, word):
    """The bodies of the functions in which `word` stands (a function starts at a line that opens a brace in the first column's scope)."""
    for m in re.finditer(r"^[A-Za-z_].*?\{\n(.*?)^\}", text, re.M | re.S):
        if word in m.group(1):
            yield m.group(1)


def unguarded(text):
    """Functions that map a remote block's shared memory before they have arrived at a cluster barrier and waited there."""
    bad = []
    for body in _functions_with(text, "map_shared_rank"):
        before = body[:body.index("map_shared_rank")]
        arrive, wait = before.find("cluster_started_arrive()"), before.find("cluster_started_wait()")
        if not 0 <= arrive < wait:
            bad.append(body)
    return bad


def test_remote_shared_memory_is_touched_after_a_barrier():
    found = 0
    for path in glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")):
        text = open(path).read()
        assert not unguarded(text), f"{os.path.basename(path)}: {unguarded(text)[0][:300]}"
        maps = text.count("map_shared_rank(")
        assert maps == sum(b.count("map_shared_rank(") for b in _functions_with(text, "map_shared_rank")), path      # none is outside what is looked at
        found += maps
    assert found >= 2


def test_what_it_looks_for():
    kernel = "__global__ void k(int* out) {\n%s  *this_cluster().map_shared_rank(&x, 0) = 1;\n  this_cluster().sync();\n}\n"
    assert unguarded(kernel % "") and unguarded(kernel % "  cluster_started_arrive();\n") and unguarded(kernel % "  cluster_started_wait();\n  cluster_started_arrive();\n")
    assert not unguarded(kernel % "  cluster_started_arrive();\n  work();\n  cluster_started_wait();\n")
