"""Adapters whose rank is not a multiple of 16 are padded inside the kernel: an infinity in x
must not meet the padding (inf * 0 is NaN)."""
import math

import pytest
import torch

import b200attn


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 72, 104])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 64), (3, 4096, 1024), (130, 64, 64), (300, 200, 520)])
def test_an_infinity_in_x_stays_one(cuda, rank, rows, k, n):
    """Positive A and B: rows with a +infinity in x give +infinity in every column, -infinity
    likewise, NaN gives NaN, and the other rows are as without them."""
    g = torch.Generator().manual_seed(rank + rows)
    x = torch.randn(rows, k, generator=g).bfloat16()
    y = torch.randn(rows, n, generator=g).bfloat16()
    a = (torch.rand(1, rank, k, generator=g) * 0.1 + 0.01).bfloat16()
    b = (torch.rand(1, n, rank, generator=g) + 0.1).bfloat16()
    seg, who = torch.tensor([0, rows], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)
    add = lambda x: b200attn.lora_add(*(t.to(cuda) for t in (x, a, b, y, seg, who)),
                                      out=torch.empty(rows, n, dtype=torch.bfloat16, device=cuda)).cpu()
    plain, bad = add(x), x.clone()
    want = {0: math.inf, 1: -math.inf, 2: math.nan, rows - 1: math.inf}
    want = {r: v for r, v in want.items() if r < rows}
    for r, v in want.items():
        bad[r, (7 * r + k - 1) % k] = v
    got = add(bad)
    for r in range(rows):
        if r in want:
            assert torch.equal(got[r].nan_to_num(5.0, math.inf, -math.inf),
                               torch.full((n,), 5.0 if math.isnan(want[r]) else want[r]).bfloat16()), r
        else:
            assert torch.equal(got[r], plain[r])
