"""How a product with adapters is dealt to the pairs of SMs: every block of k of a tile and every adapter of its rows comes exactly once (no GPU)."""

import shutil
import subprocess
from pathlib import Path

import pytest

from kernel_rush_kawk_b200.csrc import build
from kernel_rush_kawk_b200.csrc.adapter_ops import AdapterOps, AdapterRows


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    compiler = shutil.which("g++")
    assert compiler, "the shares' arithmetic is compiled for the host"
    program = tmp_path_factory.mktemp("walk") / "walk"
    subprocess.run([compiler, "-O2", "-std=c++17", "-I", str(build.SRC_DIR), str(Path(__file__).parent / "adapted_walk.cpp"), "-o", str(program)], check=True)

    def run(products):
        lines = "\n".join(" ".join(map(str, p)) for p in products)
        r = subprocess.run([str(program)], input=lines, capture_output=True, text=True)
        assert r.returncode == 0 and r.stdout.startswith(f"{len(products)} products"), r.stdout[:2000]

    return run


def dealt(M, K, N, adapters):
    """The product as the host deals it: (row tiles, column tiles, tiles taken whole, blocks of k, adapters)."""
    heights = AdapterRows.HEIGHTS if M > 256 else (max(32, -(-M // 32) * 32),)
    which, shared = AdapterOps._tiling(heights, M, K, N)
    return -(-M // heights[which]), -(-N // 256), shared, -(-K // 64), adapters


def in_empty_parts(product):
    """Whether tiles have several rows of tiles, are dealt in equal parts of k, and some of these are empty."""
    row_tiles, column_tiles, shared, k_blocks, _ = product
    rest = row_tiles * column_tiles - shared
    each = 74 // rest if rest else 0
    return row_tiles > 1 and rest > 0 and rest * each * 10 >= 74 * 9 and 1 < each and (min(each, k_blocks) - 1) * -(-k_blocks // min(each, k_blocks)) >= k_blocks


# parts of k that are empty, behind the last block
EMPTY = [(300, 13888, 256), (384, 14336, 256), (257, 17408, 256), (500, 17408, 256), (513, 9920, 256), (3457, 36864, 4096), (8200, 36864, 4608), (3585, 18496, 5120),
         (3649, 23104, 3840)]


@pytest.mark.parametrize("M,K,N", EMPTY)
def test_parts_of_k_without_any(walk, M, K, N):
    product = dealt(M, K, N, 3)
    assert in_empty_parts(product)
    walk([product])


def test_every_product_is_dealt_once(walk):
    products = [dealt(M, K, N, adapters) for M in (17, 64, 129, 250, 257, 300, 513, 900, 1921, 2103, 4096)
                for K in (64, 320, 576, 2560, 4096, 9728, 11008, 13888, 17408) for N in (64, 256, 520, 1536, 2560, 6144, 19456) for adapters in (1, 7)]
    walk(products)


def test_every_number_of_tiles_and_blocks(walk):
    """Beyond what the choice of tiles comes to."""
    walk([(rows, tiles, shared, k_blocks, adapters) for rows in (1, 3) for tiles in (1, 2, 3, 5, 8, 13, 37, 74, 75) for shared in (0, 74)
          if shared <= rows * tiles for k_blocks in (1, 2, 5, 17, 36, 40, 73, 217, 272) for adapters in (0, 1, 5, 40)])
