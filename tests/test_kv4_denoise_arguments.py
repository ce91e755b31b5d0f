"""Arguments of the denoising loop that do not go together, or not with the batch."""
from types import SimpleNamespace

import pytest
import torch

from b200attn import mmdit
from b200attn.kv4 import KV4Cache

CFG = mmdit.MMDiTConfig(layers=2, heads=2, text_dim=256)


def refused(embs, **kwargs):
    """denoise with a model that must not get as far as computing anything."""
    def computed(*args, **kw):
        raise AssertionError("the call was not refused")
    model = SimpleNamespace(cfg=CFG, device=torch.device("cpu"), text_embed=computed)
    model.prefix_fill = lambda *a, **kw: mmdit.MMDiT.prefix_fill(model, *a, **kw)
    with pytest.raises(ValueError):
        mmdit.denoise(model, embs, None, (2, 2), 2, 1.0, torch.zeros(len(embs), 4, 64), **kwargs)


def test_a_4bit_cache_is_not_offloaded():
    embs = [torch.zeros(70, 256, dtype=torch.bfloat16)]
    cache = KV4Cache(2, 2, 6, device="cpu")
    refused(embs, kv4=cache, offload_cache=True)
    assert cache.tables.free_pages == 6
    refused(embs, kv4=KV4Cache(2, 2, 6, device="cpu"), offload_cache=True)


@pytest.mark.parametrize("ids", [[], [0], [0, 1, 0], [None], [-1, None, None]])
@pytest.mark.parametrize("kv4", [None, True])
def test_one_adapter_id_per_prompt(ids, kv4):
    embs = [torch.zeros(70, 256, dtype=torch.bfloat16), torch.zeros(3, 256, dtype=torch.bfloat16)]
    cache = KV4Cache(2, 2, 6, device="cpu") if kv4 else None
    refused(embs, adapters=ids, kv4=cache)
    assert cache is None or cache.tables.free_pages == 6


@pytest.mark.parametrize("ids", [[], [0], [None], [-1, None, None]])
def test_a_step_takes_one_adapter_id_per_sequence(ids):
    model = SimpleNamespace(adapters=object())
    with pytest.raises(ValueError, match="adapter ids"):
        mmdit.MMDiT._batch_adapters(model, ids, 2, 4)
    assert mmdit.MMDiT._batch_adapters(model, [None, -1], 2, 4) is None
