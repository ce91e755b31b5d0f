"""The denoising loop with an adapter per prompt, over the bf16 cache and over 4-bit pages,
against the float32 oracle with each adapter merged into its weights.

Every step of the loop is recorded and compared for itself, from the loop's own latents: the
velocity of each sequence with the oracle's, within the bound of a single step (rel L2 1.5e-2;
bf16 GEMM operands put the model about 1e-2 from float32), and the next step's latents with the
Euler update of the recorded velocities, exactly.  (From the noise on, the distance of the two
trajectories is no measure of the adapters: with 8 steps and this CFG scale the model without
any is 2.0e-2 from the oracle's, each step's error being carried and amplified by the rest.)"""
import pytest
import torch

from b200attn import mmdit
from b200attn.kv4 import KV4Cache
from b200attn.lora import AdapterBank
from oracle import mmdit_ref as M
from test_lora import GRID, TINY, _adapter, _names

STEPS, CFG_SCALE, IDS = 8, 2.5, [0, 1, None, 0]


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.fixture(scope="module")
def job(cuda):
    """A model with two adapters of different ranks on different linears, four prompts with
    one negative prompt for all, and the oracle of each adapter."""
    w = mmdit.random_weights(TINY, 0, std=0.1)
    model = mmdit.MMDiT(TINY, w, device=cuda)
    g = torch.Generator().manual_seed(21)
    adapters = [_adapter(g, 8, _names(0) + _names(1)), _adapter(g, 20, _names(1))]
    scales = [0.7, 1.3]
    model.set_adapters(AdapterBank(adapters, scales, cuda))
    pos = [torch.randn(n, 256, generator=g).to(torch.bfloat16) for n in (40, 72, 65, 40)]
    neg = torch.randn(70, 256, generator=g).to(torch.bfloat16)
    noise = mmdit.pack_latents(torch.randn(4, 64, 1, *GRID, generator=g))
    base, oracles = model.effective_weights(w), {}
    for e in (0, 1, None):
        merged = dict(base)
        for name, (A, B) in (adapters[e] if e is not None else {}).items():
            merged[name + ".weight"] = base[name + ".weight"].float() + scales[e] * (
                B.bfloat16().float() @ A.bfloat16().float())
        oracles[e] = M.Reference(merged, TINY.layers, TINY.heads)
    return model, pos, neg, noise, oracles


def recorded(model, *args, **kwargs):
    """denoise's result, and (latents, t, velocity) of every step, on the CPU."""
    steps, step = [], model.step

    def recording(lat, t, *rest, **kw):
        out = step(lat, t, *rest, **kw)
        steps.append((lat.cpu(), t, out.cpu()))
        return out
    model.step = recording
    try:
        return mmdit.denoise(model, *args, **kwargs).cpu(), steps
    finally:
        del model.step


def check_loop(result, steps, noise, oracles, prefixes, ids, with_neg):
    """prefixes: the oracle's (cache, length) of each sequence of the batch; ids: the adapter
    of each."""
    assert len(steps) == STEPS
    sig = M.sigmas(STEPS, GRID[0] * GRID[1])
    for i, (lat, t, pred) in enumerate(steps):
        assert abs(t - float(sig[i])) <= 2e-7
        for row, e in enumerate(ids):
            cache, n = prefixes[row]
            want = oracles[e].forward_cached(lat[row], t, cache, n, GRID)
            assert _rel(pred[row], want) <= 1.5e-2, (i, row, _rel(pred[row], want))
        now = lat[0::2] if with_neg else lat
        if i == 0:
            assert torch.equal(now, noise.float())
        if with_neg:
            assert torch.equal(lat[0::2], lat[1::2])
            pred = pred[1::2] + (pred[0::2] - pred[1::2]) * CFG_SCALE
        after = now.double() + pred.double() * mmdit.euler_dt(mmdit.flow_match_sigmas(STEPS, 256), i)
        got = result if i + 1 == STEPS else steps[i + 1][0][0::2] if with_neg else steps[i + 1][0]
        # a product, a sum and (with the guidance) three more operations in f32
        assert (got.double() - after).abs().max() <= 8 * 2 ** -24 * (now.abs().max() + 8 * pred.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("with_neg", [False, True])
def test_denoise_with_an_adapter_per_prompt(job, with_neg):
    """Without and with a negative prompt, which takes its prompt's adapter."""
    model, pos, neg, noise, oracles = job
    negs = [neg] * 4 if with_neg else None
    got, steps = recorded(model, pos, negs, GRID, STEPS, CFG_SCALE, noise, adapters=IDS)
    rows = [(e, a) for p, a in zip(pos, IDS) for e in ((p, neg) if with_neg else (p,))]
    prefixes = [(oracles[a].prefix_kv(e.float(), GRID), len(e)) for e, a in rows]
    check_loop(got, steps, noise, oracles, prefixes, [a for _, a in rows], with_neg)


@pytest.mark.gpu
def test_adapters_move_the_latents_of_their_prompts(job):
    model, pos, neg, noise, _ = job
    run = lambda ids: mmdit.denoise(model, pos, [neg] * 4, GRID, STEPS, CFG_SCALE, noise, adapters=ids).cpu()
    got, plain = run(IDS), run(None)
    for p, e in enumerate(IDS):
        assert torch.equal(got[p], plain[p]) if e is None else _rel(got[p], plain[p]) > 0.05
    assert torch.equal(run([None] * 4), plain)


@pytest.mark.gpu
def test_denoise_with_adapters_over_the_4bit_cache(job, cuda):
    """The negative prompt is filled once for each adapter and its pages are shared; the oracle
    takes the prefixes that the cache holds (a value next to a border may fall on either side
    of it in another precision)."""
    model, pos, neg, noise, oracles = job
    filled, fill = [], model.prefix_fill
    model.prefix_fill = lambda embs, **kw: filled.append((list(embs), kw["adapters"])) or fill(embs, **kw)
    pages = KV4Cache.pages_for([40, 72, 65, 40, 70, 70, 70])
    cache = KV4Cache(TINY.layers, TINY.heads, pages, cuda)
    try:
        got, steps = recorded(model, pos, [neg] * 4, GRID, STEPS, CFG_SCALE, noise, kv4=cache, adapters=IDS)
    finally:
        del model.prefix_fill
    assert cache.tables.free_pages == pages
    (embs, ids), = filled  # p0, its negative (adapter 0), p1, negative (1), p2, negative (none), p3
    assert [len(e) for e in embs] == [40, 70, 72, 70, 65, 70, 40] and ids == [0, 0, 1, 1, None, None, 0]
    view = model.prefix_fill(embs, kv4=cache, adapters=ids)
    held = [[t.float().cpu() for t in view.load(i)] for i in range(TINY.layers)]
    rows = [0, 1, 2, 3, 4, 5, 6, 1]
    prefixes = [([(k[r, :, :view.lengths[r]], v[r, :, :view.lengths[r]]) for k, v in held], view.lengths[r])
                for r in rows]
    check_loop(got, steps, noise, oracles, prefixes, [ids[r] for r in rows], True)
    cache.free(view.seqs)


@pytest.mark.gpu
def test_a_failing_run_with_adapters_leaves_the_cache(job, cuda):
    model, pos, neg, noise, _ = job
    cache = KV4Cache(TINY.layers, TINY.heads, 20, cuda)
    for wrong in ([0, 1, 2, None], [0, 1]):
        with pytest.raises(ValueError):
            mmdit.denoise(model, pos, None, GRID, 2, 1.0, noise, kv4=cache, adapters=wrong)
        assert cache.tables.free_pages == 20

    def stop(i):
        raise KeyboardInterrupt
    with pytest.raises(KeyboardInterrupt):
        mmdit.denoise(model, pos, None, GRID, 2, 1.0, noise, step_callback=stop, kv4=cache, adapters=IDS)
    assert cache.tables.free_pages == 20
