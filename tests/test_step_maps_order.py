"""Kernels start beside the ones before them: what reads a step's maps must not do so before they are made (no GPU)."""

import re

import pytest

from kernel_rush_kawk_b200.csrc.build import SRC_DIR

# what a step's kernel makes, and the helpers that read it
MADE = re.compile(r"\b(cu_q|row_seq|row_pos|row_place|prefix_unit|own_unit|add_rows)\b")


def kernels():
    """(file, name, body) of every kernel, comments left out."""
    for path in sorted([*SRC_DIR.glob("*.cu"), *SRC_DIR.glob("*.cuh")]):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for match in re.finditer(r"__global__", text):
            depth, at = 0, match.end()
            while text[at] != ";" and not (text[at] == "{" and depth == 0):
                depth += {"(": 1, ")": -1}.get(text[at], 0)
                at += 1
            if text[at] == ";":
                continue
            first, depth = at, 0
            while True:
                depth += {"{": 1, "}": -1}.get(text[at], 0)
                at += 1
                if depth == 0:
                    break
            names = [n for n in re.findall(r"(\w+)\s*\(", text[match.end():first]) if n not in ("__launch_bounds__", "__cluster_dims__")]
            yield path.name, names[0], text[first:at]


ALL = list(kernels())


@pytest.mark.parametrize("file,name,body", [k for k in ALL if "grid_dependency_wait" in k[2]], ids=lambda v: v if len(v) < 60 else "")
def test_nothing_is_read_before_the_wait(file, name, body):
    """A kernel that starts beside the ones before it reads a step's maps behind its wait."""
    before = body[:body.index("grid_dependency_wait")]
    assert not MADE.search(before), f"{file}: {name} reads '{MADE.search(before).group()}' before it waits"


@pytest.mark.parametrize("name", ["first_factor_tiles_kernel", "first_factor_few_kernel", "first_factor_kernel"])
def test_the_first_factor_waits_before_it_lets_the_product_in(name):
    """The products read a step's maps and rows before they wait: by then all that was before the first factor is over."""
    (body,) = [body for _, n, body in ALL if n == name]
    assert body.index("grid_dependency_wait") < body.index("grid_launch_dependents")


def test_no_kernel_overtakes_the_maps():
    """The attention of single tokens reads positions, slots and the page table before it waits, as copies leave them: the kernel that makes maps and enters
    pages lets none in, like those that select tokens and move a step on."""
    (body,) = [body for _, n, body in ALL if n == "step_maps_kernel"]
    assert "grid_launch_dependents" not in body
    (select,) = [body for _, n, body in ALL if n == "select_finish_kernel"]
    assert "grid_launch_dependents" not in select


def test_there_are_kernels():
    assert len(ALL) > 90 and {"step_maps_kernel", "prefix_tcgen05_kernel", "few_rows_kernel", "qk_norm_rope_write_kernel"} <= {n for _, n, _ in ALL}
