"""CPU check of the CUDA sources: shared memory of another CTA of a cluster may be accessed only once that CTA
is known to have started, and for that a cluster barrier has to lie before the access.  (A missing one need
not show on a GPU: it is looked for in the text.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensorplay_b200", "csrc")
BARRIER = re.compile(r"barrier\.cluster\.wait|\bcluster_wait\(\)|\bcluster\.sync\(\)")
REMOTE = re.compile(r"\bmap_shared_rank\s*\(|\bmapa\.")


def kernels(text):
    """The texts from one __global__ to the next, without comments."""
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    text = re.sub(r"//[^\n]*", "", text)
    return re.split(r"\b__global__\b", text)[1:]


def unguarded(text):
    bad = []
    for k in kernels(text):
        access = REMOTE.search(k)
        if access and not BARRIER.search(k[:access.start()]):
            bad.append(k[:300].split("(")[-2].split()[-1] if "(" in k else k[:60])
    return bad


def test_the_check_itself():
    body = "__global__ void %s(int* p) { %s *cluster.map_shared_rank(p, 0u) = 1; cluster.sync(); }"
    assert len(unguarded(body % ("k", "") + body % ("l", "cluster_wait(); "))) == 1
    assert len(unguarded(body % ("k", "// cluster.sync()\n"))) == 1
    assert unguarded(body % ("k", 'asm volatile("barrier.cluster.wait.acquire;");')) == []


@pytest.mark.parametrize("name", ["logprob.cu", "softmax.cu", "topk_select.cuh"])
def test_remote_shared_memory_lies_behind_a_cluster_barrier(name):
    text = open(os.path.join(CSRC, name)).read()
    assert any(REMOTE.search(k) for k in kernels(text))
    assert unguarded(text) == []


def test_every_source_with_remote_shared_memory_is_listed():
    files = [f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))]
    found = {f for f in files if any(REMOTE.search(k) for k in kernels(open(os.path.join(CSRC, f)).read()))}
    assert found == {"logprob.cu", "softmax.cu", "topk_select.cuh"}
