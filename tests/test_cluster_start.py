"""Shared memory of another block of a cluster may be touched only once that block is known to have started, which a barrier of the cluster says and nothing
else does.  Read from the sources: a kernel without it seldom fails, and must not be run to see whether it does."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "vllm_omni_b200" / "csrc"
REMOTE = re.compile(r"\b(at_rank|mapa_shared)\(|mapa\.")
BARRIER = re.compile(r"\b(cluster_sync_all|cluster_barrier|cluster_wait)\(\)")


def kernels(path):
    """Texts from one kernel's head to the next one's, without comments; the device functions that follow a kernel stay with it."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)
    return re.split(r"\b__global__\b", text)[1:]


def reaches_first(kernel):
    far, barrier = REMOTE.search(kernel), BARRIER.search(kernel)
    return far is not None and (barrier is None or far.start() < barrier.start())


FILES = sorted(p for p in CSRC.glob("*.cu*") if REMOTE.search(p.read_text()))


def test_files_are_found():
    assert {"sample_given.cu", "gemm_sm100.cu", "moe.cu"} <= {p.name for p in FILES}


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_a_barrier_comes_before_other_blocks_memory(path):
    late = [re.search(r"\w+_kernel\b|$", k).group() for k in kernels(path) if reaches_first(k)]
    assert late == []


def test_a_wait_has_its_arrival():
    """The barrier in two halves: every thread arrives before it waits."""
    for path in FILES:
        for kernel in kernels(path):
            for wait in re.finditer(r"\bcluster_wait\(\)", kernel):
                assert len(re.findall(r"\bcluster_arrive\(\)", kernel[:wait.start()])) > len(re.findall(r"\bcluster_wait\(\)", kernel[:wait.start()])), path.name
