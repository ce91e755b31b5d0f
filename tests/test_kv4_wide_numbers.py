"""Numbers that do not fit the library's 32 bits are refused, not cut off."""
import pytest
import torch

import b200attn

D, BLOCK = 128, 9216
WIDE = [2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 32 + 64, -2 ** 32 + 1, 2 ** 63]


@pytest.mark.parametrize("wide", WIDE)
def test_wide_numbers_are_refused(wide):
    pool = torch.zeros(3, 2, BLOCK, dtype=torch.uint8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    q = torch.zeros(1, 2, 5, D, dtype=torch.bfloat16)
    v = torch.zeros(1, 5, 2, D, dtype=torch.bfloat16)
    w, pe = torch.ones(D), torch.zeros(5, D)
    for call in (lambda: b200attn.kv4_copy_pages(pool, [wide], [1]),
                 lambda: b200attn.kv4_copy_pages(pool, [0, 1], [2, wide]),
                 lambda: b200attn.kv4_load(pool, table, None, wide),
                 lambda: b200attn.kv4_workspace_bytes(1, 2, 200, wide),
                 lambda: b200attn.kv4_workspace_bytes(1, 2, wide, 64),
                 lambda: b200attn.kv4_workspace_bytes(1, wide, 200, 64),
                 lambda: b200attn.kv4_workspace_bytes(wide, 2, 200, 64),
                 lambda: b200attn.kv4_joint_attention(q, q, v, pool, table, wide),
                 lambda: b200attn.kv4_attention_forward(v, v, v, pool, table, wide, w, w, pe)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def test_page_ids_may_be_any_integers():
    """numpy's integers and tensors' elements as well as ints: what they reach is the check of
    the device."""
    import numpy as np
    pool = torch.zeros(3, 2, BLOCK, dtype=torch.uint8)
    for src in (np.array([0]), torch.tensor([0]), [np.int64(0)], (0,)):
        with pytest.raises(ValueError, match="CUDA"):
            b200attn.kv4_copy_pages(pool, src, [1])
