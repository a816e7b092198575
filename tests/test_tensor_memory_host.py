"""Every kernel that holds tensor memory, by name: what each has to do before the next kernel starts and before its memory is freed. (Read,
not run: nothing makes a wait run out on a healthy GPU.) A kernel that is new shows as a name that is not listed here."""

from __future__ import annotations

import re

import pytest

from fastforks_b200 import _lib

KERNELS = {"attn_fwd_kernel", "gemm_pair_kernel", "gemm_split_kernel", "sam_rel_lines_kernel", "kv4_tiles_kernel"}


def bodies() -> dict[str, str]:
    got = {}
    for path in (*_lib.SOURCES, *_lib.HEADERS):
        for body in path.read_text().split("__global__")[1:]:
            if "tmem_alloc" in body or "tmem_dealloc" in body:
                name = body[: body.index("(", body.index("_kernel"))].split()[-1]
                assert name not in got
                got[name] = body
    return got


def test_the_kernels_that_hold_tensor_memory() -> None:
    assert set(bodies()) == KERNELS


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_tensor_memory_is_held_before_the_next_kernel_starts(name: str) -> None:
    body = bodies()[name]
    assert body.index("tmem_alloc") < body.index("grid_launch_dependents();")


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_products_end_before_tensor_memory_is_freed(name: str) -> None:
    """A last commit, and behind it a wait for what it commits."""
    body = bodies()[name]
    last = re.search(r"umma_commit(_pair)?\(&(sm\.)?(drain(\[t\])?|acc_full)\);", body)
    assert last
    free = body.index("tmem_dealloc")
    assert last.start() < free
    assert re.search(r"mbar_wait(_\w+)?\(&(sm\.)?(drain|acc_full)", body[last.end() : free])


def test_terms_by_lines_leave_their_loop_where_all_warps_see_the_flag() -> None:
    lines = bodies()["sam_rel_lines_kernel"]
    gives_up = lines.index("if (abort != 0)")
    assert lines.rindex("__syncthreads();", 0, gives_up) > lines.index("mbar_wait(&done")
    assert "break;" in lines[gives_up : lines.index("tmem_dealloc")]
