"""Outputs that lie on inputs which are still to be read are refused; columns of one buffer
that keep apart, and a row's own x, are not."""
import pytest
import torch

import b200attn
from test_lora import check, make

BASE = 1 << 20  # an address for calls that are refused before anything is read


def lib_call(x, y, out, rows=200, n=64, k=64, ldx=64, ldy=64, ldo=64):
    return b200attn.lib().b200_lora_add(x, ldx, 16, 16, y, ldy, out, ldo, 16, 16, None, rows, 2, 3, n, k, 16,
                                        None, None)


@pytest.mark.parametrize("where", [
    dict(x=0, y=128 * 64 * 8, out=64 * 2),                       # out is x, one row later
    dict(x=64 * 2 * 199, y=128 * 64 * 8, out=0),                 # out's last row is x's first
    dict(x=0, y=64 * 2, out=64 * 2),                             # in place, x one row before
    dict(x=0, y=1 << 18, out=16, ldx=72, ldo=64),                # other strides
    dict(x=0, y=1 << 18, out=136 * 2 - 16, ldx=136, ldo=136),    # across a row's end
    dict(x=1 << 18, y=0, out=16),                                # y, 8 columns later
    dict(x=1 << 18, y=0, out=64 * 2),
    dict(x=1 << 18, y=16, out=0, rows=1),
    dict(x=1 << 18, y=0, out=56 * 2, ldy=128, ldo=128),          # the last 8 columns of y
    dict(x=1 << 18, y=0, out=128 * 2 - 16, ldy=128, ldo=128),    # the first 8 of its next row
])
def test_overlaps_are_refused(where):
    at = {name: BASE + v if name in ("x", "y", "out") else v for name, v in where.items()}
    assert lib_call(**at) == b200attn.ERR_INVALID


@pytest.mark.gpu
def test_columns_that_keep_apart_and_own_rows(cuda):
    """y and out as columns of one buffer, x, y and out as columns of one buffer, and x as y
    in place."""
    g = torch.Generator().manual_seed(4)
    lens, who, k, n, rank = [130, 3, 200], [0, -1, 1], 512, 512, 24
    x, y, a, b, scale, seg, w = make(g, lens, who, k, n, rank, 2)
    rest = [t.to(cuda) for t in (seg, w)]
    a_dev, b_dev, s_dev = a.to(cuda), b.to(cuda), scale.to(cuda)
    both = torch.zeros(333, 3 * n, dtype=torch.bfloat16, device=cuda)
    both[:, :k], both[:, k:k + n] = x.to(cuda), y.to(cuda)
    out = b200attn.lora_add(both[:, :k], a_dev, b_dev, both[:, k:k + n], *rest, scale=s_dev, out=both[:, k + n:])
    check(out, x, y, a, b, scale, seg, w)
    assert torch.equal(both[:, :k].cpu(), x) and torch.equal(both[:, k:k + n].cpu(), y)
    own = x.to(cuda)
    check(b200attn.lora_add(own, a_dev, b_dev, own, *rest, scale=s_dev), x, x, a, b, scale, seg, w)
    with pytest.raises(b200attn.B200Error):
        b200attn.lora_add(both[:-1, :k], a_dev, b_dev, both[1:, :n], *[
            torch.tensor([0, 130, 133, 332], dtype=torch.int32, device=cuda), rest[1]], scale=s_dev)
