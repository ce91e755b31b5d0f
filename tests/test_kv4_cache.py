"""Page accounting of the 4-bit prefix cache, its page moves on the GPU, and the denoising
loop over it."""
import random

import pytest
import torch

import b200attn
from b200attn import mmdit
from b200attn.kv4 import KV4Cache, OutOfPages, PAGE, PageTables
from oracle import mmdit_ref as M
from test_kv4 import check, i32, values

D = 128


# ----------------------------------------------------------------- accounting (CPU)
class Naive:
    """Every sequence as the list of its tokens; a pool as page -> 64 slots."""

    def __init__(self, pages):
        self.slots = [[None] * PAGE for _ in range(pages)]
        self.tokens = {}
        self.fresh = 0

    def write(self, tables, seq, start):
        for i in range(start, tables.length(seq)):
            self.slots[tables.pages(seq)[i // PAGE]][i % PAGE] = self.fresh
            self.tokens.setdefault(seq, []).append(self.fresh)
            self.fresh += 1

    def move(self, copies):
        src, dst = [c[0] for c in copies], [c[1] for c in copies]
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for s, d in copies:
            self.slots[d] = list(self.slots[s])

    def check(self, tables):
        held = set()
        for seq, tokens in self.tokens.items():
            pages = tables.pages(seq)
            assert tables.length(seq) == len(tokens) and len(pages) == -(-len(tokens) // PAGE)
            assert [self.slots[pages[i // PAGE]][i % PAGE] for i in range(len(tokens))] == tokens
            held |= set(pages)
        assert tables.free_pages == tables.num_pages - len(held)


@pytest.mark.parametrize("seed", range(8))
def test_any_sequence_of_calls_keeps_every_token(seed):
    rng = random.Random(seed)
    tables, naive = PageTables(40), Naive(40)
    refused = 0
    for _ in range(300):
        live = list(naive.tokens)
        op = rng.choice(("add", "fork", "extend", "extend", "free", "compact"))
        try:
            if op == "add" or not live:
                seq = tables.add(rng.choice((0, 1, 63, 64, 65, 200)))
                naive.tokens[seq] = []
                naive.write(tables, seq, 0)
            elif op == "fork":
                seq = rng.choice(live)
                new = tables.fork(seq)
                naive.tokens[new] = list(naive.tokens[seq])
            elif op == "extend":
                some = rng.sample(live, rng.randint(1, len(live)))
                old = [tables.length(s) for s in some]
                naive.move(tables.extend(some, [rng.choice((0, 1, 5, 64, 70)) for _ in some]))
                for s, n in zip(some, old):
                    naive.write(tables, s, n)
            elif op == "free":
                seq = rng.choice(live)
                tables.free(seq)
                del naive.tokens[seq]
            else:
                naive.move(tables.compact())
                used = {p for s in naive.tokens for p in tables.pages(s)}
                assert used == set(range(len(used)))
        except OutOfPages:
            refused += 1
        naive.check(tables)
    assert refused > 0


def test_accounting_refuses():
    tables = PageTables(2)
    seq = tables.add(64)
    with pytest.raises(OutOfPages):
        tables.add(65)
    with pytest.raises(OutOfPages):
        tables.extend([seq], [65])
    assert tables.length(seq) == 64 and tables.free_pages == 1
    for bad in (lambda: tables.add(-1), lambda: tables.extend([seq, seq], [1, 1]),
                lambda: tables.extend([seq], [-1]), lambda: tables.extend([seq], []), lambda: PageTables(-1)):
        with pytest.raises(ValueError):
            bad()
    tables.free(seq)
    with pytest.raises(KeyError):
        tables.free(seq)
    assert tables.free_pages == 2


# ----------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("layers,pages,heads,moves", [(1, 2, 1, 1), (3, 9, 5, 4), (2, 700, 2, 350), (40, 8, 1, 3)])
def test_copy_pages(cuda, layers, pages, heads, moves):
    """Every byte of the copied pages, and no other; more copies than one launch takes."""
    g = torch.Generator().manual_seed(moves)
    pool = torch.randint(0, 256, (layers, pages, heads, 9216), generator=g).to(torch.uint8)
    order = torch.randperm(pages, generator=g).tolist()
    src = [order[i % max(1, moves // 2)] for i in range(moves)]  # a page may be copied twice
    dst = order[moves:2 * moves]
    dev = pool.to(cuda)
    b200attn.kv4_copy_pages(dev, src, dst)
    pool[:, dst] = pool[:, src]
    assert torch.equal(dev.cpu(), pool)
    one = dev[0].clone()                                         # one layer's pool
    b200attn.kv4_copy_pages(one, src[:1], dst[:1])
    assert torch.equal(one, dev[0])


def attend(view, layer, g, t=3, desc_lengths=None):
    b, h = len(view.seqs), view.cache.heads
    dev = view.page_table.device
    q, k = (torch.randn(b, h, t, D, generator=g).bfloat16().to(dev) for _ in range(2))
    v = torch.randn(b, t, h, D, generator=g).bfloat16().to(dev)
    desc = torch.tensor([[n, t] for n in view.lengths], dtype=torch.int32, device=dev)
    out = b200attn.kv4_joint_attention(q, k, v, view.pool(layer), view.page_table, view.max_len, desc=desc)
    return out, (q, k, v)


@pytest.mark.gpu
def test_fork_extend_free_compact_and_attend(cuda):
    """A cache as an engine uses it: prompts, forks of them, each fork extended by other
    tokens, some requests done, the pool made dense, attention after each."""
    g = torch.Generator().manual_seed(1)
    heads, layers = 3, 2
    cache = KV4Cache(layers, heads, 24, cuda)
    lengths = [100, 64, 1]
    seqs = cache.add(lengths)
    toks = [torch.randn(layers, 2, heads, n, D, generator=g).bfloat16() for n in lengths]

    def dense(parts, most):
        out = torch.zeros(layers, 2, len(parts), heads, most, D, dtype=torch.bfloat16)
        for b, p in enumerate(parts):
            out[:, :, b, :, :p.shape[3]] = p
        return out

    def verify(ids, parts):
        view = cache.view(ids)
        assert view.lengths == [p.shape[3] for p in parts]
        want = dense(parts, view.max_len)
        for layer in range(layers):
            k, v = view.load(layer)
            assert torch.equal(k.cpu().double(), values(want[layer, 0]))
            assert torch.equal(v.cpu().double(), values(want[layer, 1]))
            out, (q, ko, vo) = attend(view, layer, g)
            check(out, q, ko, vo, values(want[layer, 0]), values(want[layer, 1]), [(n, 3) for n in view.lengths])

    view = cache.view(seqs)
    put = dense(toks, 100).to(cuda)
    for layer in range(layers):
        view.store(layer, put[layer, 0], put[layer, 1], count=i32(cuda, *lengths))
    verify(seqs, toks)
    before = cache.tables.free_pages
    forks = cache.fork(seqs)
    assert cache.tables.free_pages == before                     # a fork takes no page
    new = [torch.randn(layers, 2, heads, n, D, generator=g).bfloat16() for n in (30, 5, 64)]
    cache.extend(forks, [30, 5, 64])
    view, put = cache.view(forks), dense(new, 64).to(cuda)
    for layer in range(layers):
        view.store(layer, put[layer, 0], put[layer, 1], start=i32(cuda, *lengths), count=i32(cuda, 30, 5, 64))
    grown = [torch.cat([a, b], 3) for a, b in zip(toks, new)]
    verify(seqs, toks)                                           # the originals are untouched
    verify(forks, grown)
    cache.free([seqs[0], forks[1]])
    assert cache.compact() > 0
    verify([seqs[1], seqs[2], forks[0], forks[2]], [toks[1], toks[2], grown[0], grown[2]])
    again = cache.add([64 * cache.tables.free_pages])
    with pytest.raises(OutOfPages):
        cache.add([1])
    cache.free(again + seqs[1:] + [forks[0], forks[2]])
    assert cache.tables.free_pages == 24


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [4, 150])
def test_captured_and_on_another_stream(cuda, tokens):
    """A captured store and attention replayed on new inputs and a new page table, and the
    same calls on a stream of their own, equal the plain calls."""
    g = torch.Generator().manual_seed(tokens)
    heads, n = 2, 150
    cache = KV4Cache(1, heads, 12, cuda)
    a, b = cache.add([n, n])
    new = lambda: torch.randn(1, heads, n, D, generator=g).bfloat16().to(cuda)
    rows = lambda: torch.randn(1, heads, tokens, D, generator=g).bfloat16().to(cuda)
    k, v, q, ko = new(), new(), rows(), rows()
    vo = rows().transpose(1, 2).contiguous()
    table = cache.view([a]).page_table.clone()
    out = torch.empty(1, tokens, heads * D, dtype=torch.bfloat16, device=cuda)
    ws = torch.empty(max(1, b200attn.kv4_workspace_bytes(1, heads, tokens, n)), dtype=torch.uint8, device=cuda)

    def calls(stream=None):
        b200attn.kv4_store(k, v, cache.pool[0], table, stream=stream)
        b200attn.kv4_joint_attention(q, ko, vo, cache.pool[0], table, n, out=out, workspace=ws, stream=stream)

    calls()
    plain = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out.zero_()
    torch.cuda.synchronize()
    calls(side)
    side.synchronize()
    assert torch.equal(out, plain)
    own = b200attn.kv4_joint_attention(q, ko, vo, cache.pool[0], table, n, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(own, plain)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for t in (k, v, q, ko):
        t.copy_(torch.randn(t.shape, generator=g))
    table.copy_(cache.view([b]).page_table)
    graph.replay()
    replayed = out.clone()
    out.zero_()
    calls()
    assert torch.equal(replayed, out) and not torch.equal(replayed, plain)


TINY = mmdit.MMDiTConfig(layers=2, heads=2, text_dim=256)
GRID = (16, 16)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _embs(lengths, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, TINY.text_dim, generator=g).to(torch.bfloat16) for n in lengths]


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_cached_step_over_the_4bit_cache(cuda, fused):
    """One denoising step of ragged prompts over 4-bit pages against the float32 oracle whose
    prefix K/V carry the same quantisation, and over the pages read back as a dense cache."""
    w = mmdit.random_weights(TINY, 0, std=0.1)
    model = mmdit.MMDiT(TINY, w, device=cuda, fused_qkv=fused)
    lengths = [40, 72, 130]
    embs = _embs(lengths, 5)
    lat = torch.randn(3, 256, 64, generator=torch.Generator().manual_seed(6))
    cache = KV4Cache(TINY.layers, TINY.heads, KV4Cache.pages_for(lengths) + 1, cuda)
    view = model.prefix_fill(embs, kv4=cache)
    assert view.lengths == lengths and cache.tables.free_pages == 1
    pe, desc = model.target_pe(lengths, GRID), mmdit.cached_desc(view, 256, cuda)
    got = model.step(lat.to(cuda), 0.5, view, pe, desc).cpu()
    dense = [view.load(i) for i in range(TINY.layers)]
    plain = mmdit.PrefixCache(k=[k for k, _ in dense], v=[v for _, v in dense], lengths=lengths)
    assert torch.equal(got, model.step(lat.to(cuda), 0.5, plain, pe, desc).cpu())
    R = M.Reference(w, TINY.layers, TINY.heads)
    for b, n in enumerate(lengths):
        # the model's own stored prefix: a value next to a border may fall on either side of
        # it in another precision, so the oracle reads what the cache holds
        prefix = [(k[b, :, :n].float().cpu(), v[b, :, :n].float().cpu()) for k, v in dense]
        assert _rel(got[b], R.forward_cached(lat[b], 0.5, prefix, n, GRID)) <= 1.5e-2
        for (k, v), (kw, vw) in zip(prefix, R.prefix_kv(embs[b].float(), GRID)):
            # each within half a step (1/14 of its group's largest, 1/16 cut) and rounding
            for have, want in ((k, kw), (v, vw)):
                top = want.reshape(*want.shape[:-1], 4, 32).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32)
                off = (have - want).reshape(*want.shape[:-1], 4, 32).abs()
                assert (off <= top * (0.5 / 7 + 0.05)).all()


@pytest.mark.gpu
def test_denoise_shares_the_negative_prompt(cuda):
    """denoise over a 4-bit cache: one negative prompt for all requests is filled once, and
    the result is that of negatives filled one by one."""
    w = mmdit.random_weights(TINY, 0, std=0.1)
    model = mmdit.MMDiT(TINY, w, device=cuda)
    pos, neg = _embs((40, 72, 65), 31), _embs((70,), 32)[0]
    noise = mmdit.pack_latents(torch.randn(3, 64, 1, *GRID, generator=torch.Generator().manual_seed(3)))
    pages = KV4Cache.pages_for([40, 72, 65])
    cache = KV4Cache(TINY.layers, TINY.heads, pages + 2, cuda)
    shared = mmdit.denoise(model, pos, [neg] * 3, GRID, 4, 2.5, noise, kv4=cache)
    assert cache.tables.free_pages == pages + 2
    apart = mmdit.denoise(model, pos, [neg.clone() for _ in range(3)], GRID, 4, 2.5, noise, kv4=True)
    assert torch.equal(shared, apart)
    with pytest.raises(OutOfPages):
        mmdit.denoise(model, pos, [neg.clone() for _ in range(3)], GRID, 4, 2.5, noise, kv4=cache)
    assert cache.tables.free_pages == pages + 2
    with pytest.raises(ValueError):
        model.prefix_fill(pos, offload=True, kv4=cache)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 150])
def test_attention_forward_is_norm_rope_and_attention(cuda, tokens):
    g = torch.Generator().manual_seed(tokens)
    heads, n, b = 4, 90, 2
    cache = KV4Cache(1, heads, 8, cuda)
    view = cache.view(cache.add([n, 20]))
    kv = torch.randn(2, b, heads, n, D, generator=g).bfloat16().to(cuda)
    view.store(0, kv[0], kv[1], count=i32(cuda, n, 20))
    q, k, v = (torch.randn(b, tokens, heads, D, generator=g).bfloat16().to(cuda) for _ in range(3))
    wq, wk = (1 + 0.1 * torch.randn(2, D, generator=g)).to(cuda)
    ang = torch.rand(tokens, D // 2, generator=g) * 6
    pe = torch.stack([ang.cos(), ang.sin()], -1).reshape(tokens, D).to(cuda)
    desc = torch.tensor([[n, tokens], [20, tokens - 1]], dtype=torch.int32, device=cuda)
    k_rot = torch.empty(b, heads, tokens, D, dtype=torch.bfloat16, device=cuda)
    v_out = torch.empty_like(k_rot)
    got = b200attn.kv4_attention_forward(q, k, v, view.pool(0), view.page_table, n, wq, wk, pe, desc=desc,
                                         k_rot_out=k_rot, v_out=v_out)
    qr, kr = b200attn.qk_norm_rope(q, k, wq, wk, 1e-6, pe)
    want = b200attn.kv4_joint_attention(qr, kr, v, view.pool(0), view.page_table, n, desc=desc)
    assert torch.equal(got, want) and torch.equal(k_rot, kr) and torch.equal(v_out, v.transpose(1, 2))
    assert torch.equal(got, b200attn.kv4_attention_forward(q, k, v, view.pool(0), view.page_table, n, wq, wk,
                                                           pe.expand(b, -1, -1).contiguous(), desc=desc))
