"""Kernels that may start before the one ahead of them in the stream has ended.

What they read can still change while their grid runs, up to the wait; the read-only path (ld.global.nc,
__ldg) is for memory that does not change during the kernel. So such sources do not use it.
"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).parents[1] / "h3_flash_b200" / "csrc"
DEPENDENT = sorted(p.name for p in CSRC.glob("*.cu") if "launch_after(" in p.read_text())


def test_there_are_such_sources():
    assert {"block_select.cu", "sparse_attention.cu"} <= set(DEPENDENT)


@pytest.mark.parametrize("name", DEPENDENT)
def test_no_read_only_loads(name):
    code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.search(r"\bld_cached\b|__ldg\b|\.nc\b", code)


@pytest.mark.parametrize("name", DEPENDENT)
def test_every_dependent_kernel_waits(name):
    code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    for kernel in set(re.findall(r"launch_after\((\w+)", code)):
        body = code[re.search(r"__global__[^;{]*\b%s\(" % kernel, code).end():]
        body = body[: body.index("__global__") if "__global__" in body else len(body)]
        assert "grid_wait();" in body, kernel
