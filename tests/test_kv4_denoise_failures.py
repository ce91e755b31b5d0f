"""A prefix fill or a denoising run that fails leaves a caller's 4-bit cache as it found it."""
from types import SimpleNamespace

import pytest
import torch

from b200attn import mmdit
from b200attn.kv4 import KV4Cache, KV4View

CFG = mmdit.MMDiTConfig(layers=2, heads=2, text_dim=256)
FAIL = RuntimeError("no memory")


def stub_model(**fails):
    """Just enough of an MMDiT for prefix_fill on the CPU; the named parts raise."""
    def part(name, result):
        def call(*args, **kwargs):
            if name in fails:
                raise FAIL
            return result
        return call
    return SimpleNamespace(cfg=CFG, device=torch.device("cpu"),
                           text_embed=lambda e: torch.zeros(e.shape[0], CFG.hidden),
                           zero_time_embed=part("zero_time_embed", None), modulation=part("modulation", None),
                           _run_blocks=part("_run_blocks", None))


@pytest.mark.parametrize("part", ["modulation", "zero_time_embed", "_run_blocks"])
def test_prefix_fill_gives_its_pages_back(part):
    cache = KV4Cache(2, 2, 6, device="cpu")
    embs = [torch.zeros(70, 256, dtype=torch.bfloat16), torch.zeros(3, 256, dtype=torch.bfloat16)]
    with pytest.raises(RuntimeError):
        mmdit.MMDiT.prefix_fill(stub_model(**{part: True}), embs, kv4=cache)
    assert cache.tables.free_pages == 6 and not cache.tables._pages
    view = mmdit.MMDiT.prefix_fill(stub_model(), embs, kv4=cache)
    assert view.lengths == [70, 3] and cache.tables.free_pages == 3


def test_prefix_fill_gives_its_pages_back_when_the_view_fails(monkeypatch):
    cache = KV4Cache(2, 2, 6, device="cpu")

    def view(seqs):
        raise FAIL
    monkeypatch.setattr(cache, "view", view)
    with pytest.raises(RuntimeError):
        mmdit.MMDiT.prefix_fill(stub_model(), [torch.zeros(70, 256, dtype=torch.bfloat16)], kv4=cache)
    assert cache.tables.free_pages == 6 and not cache.tables._pages


@pytest.mark.parametrize("part", ["fork", "second fork", "view", "target_pe", "step"])
def test_denoise_gives_its_pages_back(monkeypatch, part):
    """The negative prompt is shared (two forks of it); each part after the fill fails once."""
    cache = KV4Cache(2, 2, 8, device="cpu")
    fork, calls = cache.fork, []

    def forks(seqs):
        calls.append(seqs)
        if part == "fork" or (part == "second fork" and len(calls) == 2):
            raise FAIL
        return fork(seqs)

    def raising(*args, **kwargs):
        raise FAIL
    monkeypatch.setattr(cache, "fork", forks)
    if part == "view":
        monkeypatch.setattr(cache, "view", raising)
    model = SimpleNamespace(
        cfg=CFG, device=torch.device("cpu"), step=raising,
        prefix_fill=lambda embs, kv4=None, **kw: KV4View(kv4, kv4.add([int(e.shape[0]) for e in embs])),
        target_pe=raising if part == "target_pe" else (lambda *a: None))
    pos = [torch.zeros(n, 256) for n in (65, 10, 3)]
    neg = torch.zeros(64, 256)
    with pytest.raises(RuntimeError):
        mmdit.denoise(model, pos, [neg] * 3, (2, 2), 2, 2.0, torch.zeros(3, 4, 64), kv4=cache)
    assert cache.tables.free_pages == 8 and not cache.tables._pages
