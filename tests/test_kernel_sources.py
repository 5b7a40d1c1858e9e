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


def test_epilogue_warps_meet_at_the_named_barriers_after_a_failure():
    # warps that leave the loop over tiles early would leave the others waiting at a barrier without a limit:
    # after a wait that ran out, the loop goes on to the next tile's barriers
    body = dict(kernels())["gemm.cuh:gemm_kernel"]
    loop = body[body.index("} else if (warp >= 4) {") :]
    barrier = loop.rindex('"bar.sync 1, 256;"')
    tile = loop[loop.index("for (int t = first; t < tiles; t += step) {") : loop.index("cp.async.bulk.wait_group 0")]
    leaves = [line for line in tile.splitlines() if "break;" in line]
    assert [line.strip() for line in leaves] == ["if (!ok) break;"]  # of the pieces of a tile
    assert "if (!ok) continue;" in loop[barrier:] and "return" not in tile


def test_tensor_memory_is_read_by_whole_warps():
    # tcgen05.ld takes all lanes: a wait before it may not let some lanes pass and others give up
    for name in ("gemm.cuh:gemm_kernel", "gemm_rows.cuh:gemm_rows_kernel"):
        body = dict(kernels())[name]
        epilogue = body[body.index("    const int q = ") :]
        assert "tmem_take" in epilogue and "mbar_wait_warp(" in epilogue and "mbar_wait(" not in epilogue, name


def test_accumulators_are_loaded_and_waited_for_in_one_statement():
    # the registers of a load from tensor memory are its own until the wait: code between two statements can move them
    files = {f: (CSRC / f).read_text() for f in ("gemm.cuh", "gemm_rows.cuh")}
    statements = re.findall(r"asm volatile\((.*?)\);", files["gemm.cuh"], re.S)
    loads = [s for s in statements if "tcgen05.ld." in s]
    assert len(loads) == 3 and all(s.rindex("tcgen05.ld.") < s.index("tcgen05.wait::ld") for s in loads)
    for text in files.values():
        assert "tmem_ld" not in text and "tc_wait_ld" not in text


def test_planes_are_read_before_they_are_asked_for_again():
    body = dict(kernels())["gemm.cuh:gemm_kernel"]
    read, fence = body.rindex("take_row("), body.index("fence_async_proxy();", body.rindex("take_row("))
    assert read < fence < body.index("__syncwarp();", fence) < body.index("ask(c + 64);")
    assert "put_row" not in body[read:fence] and "ask(" not in body[read:fence]


def test_copies_and_products_in_flight_end_before_a_block_leaves():
    # whichever warp gave up: the loads, and the MMAs before the tensor memory is freed
    body = dict(kernels())["gemm.cuh:gemm_kernel"]
    assert "\n      if (rank == 0) {  // loads in flight land" in body
    assert "\n      umma_commit_local<CG>(drained);\n" in body
    body = dict(kernels())["gemm_rows.cuh:gemm_rows_kernel"]
    assert "\n      for (int j = i > S::kStages ? i - S::kStages : 0; j < i; ++j)" in body
    assert body.count("mbar_try_wait(done, 0)") == 1
