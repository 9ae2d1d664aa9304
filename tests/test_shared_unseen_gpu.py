"""Several new tokens a request in 32 bits: what only a later token sees does not reach the earlier ones, finite or not."""

from __future__ import annotations

import pytest
import torch
from test_attention_shared_gpu import DEV, Step, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spoil", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min], ids=str)
@pytest.mark.parametrize("plane", [0, 1], ids=["key", "value"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 2, 64), (4, 1, 128), (3, 3, 16), (10, 2, 256)])
def test_a_later_tokens_key_and_value(heads, kv_heads, dim, plane, spoil):
    step = Step([96, 33], [(0, 9, 5), (0, 70, 3), (1, 1, 1), (0, 4, 4), (-1, 66, 7), (1, 130, 2)], heads=heads, kv_heads=kv_heads, dim=dim,
                page=16, dtype=torch.float32, seed=dim)
    clean = step.run()
    check(clean, step.want(), torch.float32, dim)
    last = torch.zeros(len(step.positions), dtype=torch.bool, device=DEV)
    for entry, (start, new) in enumerate(zip(step.starts, step.new)):
        position = start + new - 1
        page = int(step.table[step.slots[entry], position // step.page])
        if new > 1:                       # the last of several tokens: the ones before it must not notice
            step.cache[page, plane, :, position % step.page] = spoil
            last[int(sum(step.new[:entry])) + new - 1] = True
    got = step.run()
    assert torch.equal(got[~last], clean[~last])
    if plane == 1 and spoil != torch.finfo(torch.float32).min:
        assert not bool(torch.isfinite(got[last]).any())
