"""A CTA's shared memory may be stored to by another CTA of its cluster only once it is known to have started: in every kernel the first
remote store or arrival comes behind a wait at the cluster's barrier.  Checked on the sources, since a violation shows only when one CTA
of a cluster starts late."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bamboo_b200", "csrc")
REMOTE = re.compile(r"\b(?:st_shared_cluster_\w+|mbar_arrive_cluster\w*)\s*\(")
WAIT = re.compile(r"\bcluster_(?:sync|wait)\s*\(")


def kernels(text):
    text = re.sub(r"//[^\n]*", "", text)
    starts = [m.start() for m in re.finditer(r"__global__|\n(?:template[^\n]*\n)?(?:static |inline )*__device__|\nextern \"C\"|\nnamespace", text)]
    return [b for b in (text[a:z] for a, z in zip(starts, starts[1:] + [len(text)])) if b.startswith("__global__")]


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu"))), ids=os.path.basename)
def test_remote_stores_come_behind_a_cluster_barrier(path):
    with open(path) as f:
        text = f.read()
    for body in kernels(text):
        remote = REMOTE.search(body)
        if remote:
            name = re.search(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", body)).group(1)
            wait = WAIT.search(body)
            assert wait and wait.start() < remote.start(), f"{os.path.basename(path)}: {name}"


def test_the_check_sees_a_store_without_a_wait():
    good = "__global__ void k() {\n  cluster_arrive_relaxed();\n  cluster_wait();\n  st_shared_cluster_u32(a, b);\n  cluster_sync();\n}\n"
    for text, ok in ((good, True), (good.replace("  cluster_wait();\n", ""), False)):
        (body,) = kernels(text)
        assert (WAIT.search(body).start() < REMOTE.search(body).start()) == ok
