"""Attention over prefixes so long that one CTA walks more than 32 and more than 64 pages: the
page ids come in groups of 32, fetched one group ahead."""
import pytest
import torch

import b200attn
from test_kv4 import D, check, i32, paged, values


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 20, 50, 200])
@pytest.mark.parametrize("prefix", [16384 + 65, 17000, 40001])
def test_long_prefixes(cuda, prefix, tokens):
    lengths = [prefix, prefix // 2 + 1]
    pool, table, g = paged(cuda, lengths, 1, seed=prefix % 1000 + tokens)
    dense = torch.randn(2, 2, 1, prefix, D, generator=g).bfloat16()
    # every page of its own scale: a page read in another's place shows in the output
    scale = torch.exp(torch.randn(2, 1, -(-prefix // 64), 1, generator=g)).repeat_interleave(64, 2)[:, :, :prefix]
    dense[1] = (dense[1].float() * scale).bfloat16()
    b200attn.kv4_store(dense[0].to(cuda), dense[1].to(cuda), pool, table, count=i32(cuda, *lengths))
    q, ko = (torch.randn(2, 1, tokens, D, generator=g).bfloat16() for _ in range(2))
    vo = torch.randn(2, tokens, 1, D, generator=g).bfloat16()
    q = (q.float() * 3).bfloat16()  # peaked: few keys carry a row
    desc = torch.tensor([[n, tokens] for n in lengths], dtype=torch.int32, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = b200attn.kv4_joint_attention(q.to(cuda), ko.to(cuda), vo.to(cuda), pool, table, prefix, desc=desc,
                                       status=status)
    assert status.item() == 0
    check(got, q, ko, vo, values(dense[0]), values(dense[1]), [(n, tokens) for n in lengths])
