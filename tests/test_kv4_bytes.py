"""The bytes of a group that is not finite: a NaN step and the number 0 for every channel."""
import math

import pytest
import torch

import b200attn
from test_kv4 import D, k_nibble, paged, step_at, v_nibble


@pytest.mark.gpu
def test_numbers_of_a_group_that_is_not_finite_are_zero(cuda):
    pool, table, g = paged(cuda, [8], 1)
    x = torch.randn(1, 1, 8, D, generator=g).bfloat16()
    bad = {0: math.inf, 1: -math.inf, 2: math.nan, 3: 2.0 ** 126, 5: -2.0 ** 127}
    for tok, value in bad.items():
        x[0, 0, tok, 32 + 9 * (tok % 3)] = value  # group 1
    b200attn.kv4_store(x.to(cuda), x.to(cuda), pool, table)
    block = pool[table[0, 0].item(), 0].cpu().numpy()
    for part, where in enumerate((k_nibble, v_nibble)):
        for tok in bad:
            at = step_at(tok, 1, part)
            assert int(block[at]) | int(block[at + 1]) << 8 == 0x7fc0
            for ch in range(32, 64):
                byte, high = where(tok, ch)
                assert int(block[byte]) >> (4 * high) & 15 == 8, (part, tok, ch)
