"""What the C entries of attention over shared prefixes refuse before they launch anything (no GPU: the addresses are numbers)."""

from __future__ import annotations

import pytest

from rapid_llm_b200.ops import kernels

INVALID = 1       # cudaErrorInvalidValue
BASE = 1 << 20    # an address on every boundary


def call(dtype, dim, tile_rows=64, num_pages=10, **moved):
    at = {name: BASE + moved.get(name, 0) for name in ("q", "cache", "out", "part_out", "part_lse")}
    lists = dict(members=BASE, positions=BASE, part_first=BASE)
    tail = (BASE, BASE, 3, 8, 2, dim, 16, num_pages, 4, 5, 0.125, None, None, 8 * dim, None, 0, BASE, 0, None)
    if dtype == "f32":
        return kernels.core().rl_attention_shared_f32(*at.values(), BASE, 1, *lists.values(), *tail)
    return kernels.attention_lib(dim).rl_attention_shared(*at.values(), BASE, 1, tile_rows, BASE, 1, 4, BASE, BASE, BASE, 6, *tail)


KINDS = [("f32", 64, 64), ("bf16", 64, 64), ("bf16", 128, 128), ("bf16", 128, 256)]


@pytest.mark.parametrize("dtype,dim,tile_rows", KINDS)
@pytest.mark.parametrize("name,off", [("q", 2), ("q", 4), ("q", 8), ("cache", 4), ("cache", 8), ("part_out", 4), ("part_out", 8)])
def test_operands_that_are_read_sixteen_bytes_at_a_time(dtype, dim, tile_rows, name, off):
    assert call(dtype, dim, tile_rows, **{name: off}) == INVALID


@pytest.mark.parametrize("dtype,dim,tile_rows", KINDS)
def test_a_cache_without_pages(dtype, dim, tile_rows):
    """A bad page id reads page 0 in its place, so there has to be one."""
    assert call(dtype, dim, tile_rows, num_pages=0) == INVALID
