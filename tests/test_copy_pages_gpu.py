"""Copies of cache pages, and what the call refuses."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from rapid_llm_b200.ops import kernels

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shape", [
    (torch.bfloat16, (3, 40, 2, 2, 16, 64)), (torch.float32, (2, 9, 2, 1, 16, 80)), (torch.bfloat16, (1, 12, 5, 3)),
    (torch.float32, (1, 7, 3)), (torch.int32, (1, 33, 1)), (torch.uint8, (2, 11, 13)), (torch.bfloat16, (36, 30, 2, 8, 16, 128)),
], ids=str)
def test_targets_become_their_sources_and_nothing_else_changes(dtype, shape):
    gen = torch.Generator(device=DEV).manual_seed(1)
    pages = (torch.randn(shape, generator=gen, device=DEV) * 50).to(dtype)
    if pages.is_floating_point():
        pages[0, 0].view(-1)[0] = float("nan")
    before = pages.clone()
    ids = np.random.RandomState(2).permutation(shape[1])
    half = shape[1] // 2
    for pairs in ([(int(ids[0]), int(ids[1]))],                                       # one page
                  [(int(ids[0]), int(t)) for t in ids[1 : half + 1]],                 # a fork: one source
                  np.stack([ids[:half], ids[half : 2 * half]], 1)):                    # as many as can be
        pages.copy_(before)
        assert kernels.copy_pages(pages, pairs) is pages
        want = before.clone()
        for source, target in pairs:
            want[:, target] = before[:, source]
        bits = lambda t: t.contiguous().view(torch.uint8)
        assert torch.equal(bits(pages), bits(want))


@pytest.mark.gpu
def test_more_pairs_than_a_launch_takes():
    pages = torch.arange(9001, device=DEV, dtype=torch.int32).view(1, -1, 1).repeat(2, 1, 4).contiguous()
    pages[1] += 100000
    before = pages.clone()
    ids = np.random.RandomState(3).permutation(9001)
    pairs = np.stack([ids[:4500], ids[4500:9000]], 1)
    launches = kernels.LAUNCHES.count
    kernels.copy_pages(pages, pairs)
    assert kernels.LAUNCHES.count - launches == 2
    before[:, torch.from_numpy(pairs[:, 1]).to(DEV)] = before[:, torch.from_numpy(pairs[:, 0]).to(DEV)]
    assert torch.equal(pages, before)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    pages = torch.zeros((2, 70000, 32768), dtype=torch.int8, device=DEV)         # 4.6 GB
    pages[0, 69999] = 5
    pages[1, 69998] = 7
    kernels.copy_pages(pages, [(69999, 1), (69998, 69997)])
    assert int(pages[0, 1].min()) == 5 and int(pages[1, 1].max()) == 0
    assert int(pages[1, 69997].min()) == 7 and int(pages[0, 69997].max()) == 0 and int(pages.count_nonzero()) == 4 * 32768


@pytest.mark.gpu
def test_a_captured_call_keeps_its_pairs():
    pages = torch.randn((2, 6, 32), device=DEV)
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    pairs = np.array([[0, 1], [2, 3]])
    with torch.cuda.graph(graph, stream=other):
        kernels.copy_pages(pages, pairs)
    pairs[:] = 0                                       # the caller's list may change
    pages.copy_(torch.randn_like(pages))
    before = pages.clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(pages[:, 1], before[:, 0]) and torch.equal(pages[:, 3], before[:, 2])
    assert torch.equal(pages[:, [0, 2, 4, 5]], before[:, [0, 2, 4, 5]])


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [[(0, 9)], [(-1, 0)], [(9, 0)], [(0, -2)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)],
                                   [(0, 1, 2)], [(0.5, 1.0)], [0, 1], [(2**32, 1)], [(2**40, 2**33 + 1)]], ids=str)
def test_refused(pairs):
    pages = torch.randn((2, 9, 32), device=DEV)
    before = pages.clone()
    with pytest.raises(kernels.KernelError):
        kernels.copy_pages(pages, pairs)
    assert torch.equal(pages, before)
    assert kernels.copy_pages(pages, []) is pages


@pytest.mark.gpu
def test_long_lists_are_looked_over_too():
    pages = torch.randn((1, 300, 4), device=DEV)
    before = pages.clone()
    good = [(i, 150 + i) for i in range(140)]
    for wrong in ((3, 160), (160, 299), (299, 5), (0, 300), (-1, 299), (298, 298)):
        with pytest.raises(kernels.KernelError):
            kernels.copy_pages(pages, good + [wrong])
    assert torch.equal(pages, before)
    kernels.copy_pages(pages, good + [(149, 299), (0, 298)])
    assert torch.equal(pages[0, 150:290], before[0, :140]) and torch.equal(pages[0, 298], before[0, 0])


@pytest.mark.gpu
def test_strided_pages_are_refused():
    with pytest.raises(kernels.KernelError):
        kernels.copy_pages(torch.randn((4, 4, 32), device=DEV).transpose(0, 1), [(0, 1)])
    with pytest.raises(kernels.KernelError):
        kernels.copy_pages(torch.randn((32,), device=DEV), [(0, 1)])


def test_there_is_no_cpu_path():
    with pytest.raises(kernels.KernelError):
        kernels.copy_pages(torch.zeros((1, 4, 16)), [(0, 1)])
