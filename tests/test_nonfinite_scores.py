"""Scores that are not finite: a row of an attention with a NaN or a +infinity among its valid
scores is NaN throughout (exp(inf - inf) = NaN, and a NaN stays one), in every form and
wherever in a tile the key lies; a score of -infinity has the weight 0."""
import math

import pytest
import torch

import b200attn
from test_kv4 import D, check, paged, values

TILE = 128  # keys of one step of the tensor-core kernel; its exp2 differs by the key's place


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 20, 40, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_stored_key_that_is_not_finite(cuda, tokens, bad):
    """Head r has the key at place r (mod 8) of a full tile in a group that is not finite,
    which reads as NaN: all of its rows are NaN, and the head without one is not touched."""
    heads, n = 9, 2 * TILE
    pool, table, g = paged(cuda, [n], heads, seed=tokens)
    k, v = torch.randn(2, 1, heads, n, D, generator=g).bfloat16()
    for r in range(8):
        k[0, r, TILE + 8 * (r + 3) + r, 37] = bad
    b200attn.kv4_store(k.to(cuda), v.to(cuda), pool, table)
    q, ko = (torch.randn(1, heads, tokens, D, generator=g).bfloat16() for _ in range(2))
    vo = torch.randn(1, tokens, heads, D, generator=g).bfloat16()
    got = b200attn.kv4_joint_attention(q.to(cuda), ko.to(cuda), vo.to(cuda), pool, table, n)
    nan = torch.isnan(got.cpu()).reshape(tokens, heads, D)
    assert nan[:, :8].all(), [r for r in range(8) if not nan[:, r].all()]
    assert not nan[:, 8].any()
    check(got, q, ko, vo, values(k), values(v), [(n, tokens)])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("prefix", [0, 300])
def test_dense_keys_that_are_not_finite(cuda, bad, prefix):
    """The same for the dense joint attention, at each place of the prefix's full tiles and of
    the call's own: q is positive in the channel concerned for even rows and negative for odd
    ones, so an infinity gives scores of either sign."""
    heads, t = 17, 260
    g = torch.Generator().manual_seed(prefix + 1)
    q, k = (torch.randn(1, heads, t, D, generator=g).bfloat16() for _ in range(2))
    v = torch.randn(1, t, heads, D, generator=g).bfloat16()
    pk, pv = (torch.randn(1, heads, prefix, D, generator=g).bfloat16() for _ in range(2))
    q[..., 5] = (1 - 2 * (torch.arange(t) % 2)).bfloat16()
    for r in range(8):
        if prefix:
            pk[0, r, TILE * (r % 2) + 8 * r + r, 5] = bad
        k[0, 8 + r, TILE * (r % 2) + 8 * (15 - r) + r, 5] = bad
    own = [x.to(cuda) for x in (q, k, v)]
    got = b200attn.joint_attention(*own, *((pk.to(cuda), pv.to(cuda)) if prefix else (None, None)))
    check(got, q, k, v, pk.double(), pv.double(), [(prefix, t)])


@pytest.mark.gpu
def test_a_split_row_keeps_its_nan(cuda):
    """Few blocks over many keys are cut into pieces that are merged: a NaN in one of them
    reaches the row, even where that piece has nothing else."""
    heads, t, prefix = 1, 256, 4096
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(1, heads, t, D, generator=g).bfloat16() for _ in range(2))
    v = torch.randn(1, t, heads, D, generator=g).bfloat16()
    pk, pv = (torch.randn(1, heads, prefix, D, generator=g).bfloat16() for _ in range(2))
    ws = torch.empty(b200attn.SPLIT_WORKSPACE_BYTES, dtype=torch.uint8, device=cuda)
    attend = lambda keys: b200attn.joint_attention(*(x.to(cuda) for x in (q, k, v, keys, pv)), workspace=ws)
    for place in (6, 7, 1030, 4095):
        bad = pk.clone()
        bad[0, 0, place] = math.nan
        assert torch.isnan(attend(bad)).all(), place
    assert torch.isnan(attend(torch.full_like(pk, math.nan))).all()
    check(attend(pk), q, k, v, pk.double(), pv.double(), [(prefix, t)])
