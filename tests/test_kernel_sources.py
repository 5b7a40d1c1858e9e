"""Rules of the kernels that a run does not show, checked on their sources."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "ncas_b200" / "csrc"


def kernels():
    """(file:kernel, body) of every __global__ function."""
    out = []
    for path in sorted(CSRC.glob("*.cu*")):
        text = path.read_text()
        for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^)]*\) )?(\w+)\(", text):
            at = text.index("{\n", m.end())
            end = text.find("\n}\n", at)
            out.append((f"{path.name}:{m.group(1)}", text[at:end]))
    return out


REMOTE_WRITE = re.compile(r"put_remote\(|st\.shared::cluster")


def test_kernels_are_found():
    names = [n.split(":")[1] for n, _ in kernels()]
    for name in ("gemm_kernel", "gemm_rows_kernel", "norm_held_forward_kernel", "norm_held_backward_kernel",
                 "distill_row_kernel", "distill_held_kernel"):
        assert name in names


@pytest.mark.parametrize("name,body", [pytest.param(n, b, id=n) for n, b in kernels() if REMOTE_WRITE.search(b)])
def test_remote_shared_memory_is_written_after_the_cluster_has_started(name, body):
    # a block of a cluster may not have started yet when another one already runs: every write into
    # another block's shared memory comes after a barrier of the cluster
    first = REMOTE_WRITE.search(body).start()
    arrive, wait = body.find("cluster_started_arrive()"), body.find("cluster_started_wait()")
    assert 0 <= arrive < wait < first, name
