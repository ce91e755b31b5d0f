"""Low-rank adapters of many requests beside a shared projection, against a plain 64-bit
implementation.

Tolerance per element: u = scale x A^T is summed in f32 (K terms, at most K 2^-24 of the sum
of magnitudes), rounded to bf16 (2^-8), multiplied with B in f32, and the sum with y is
rounded to bf16 (2^-8):
|got - want| <= 2^-8 |want| + (2^-8 + 2^-10) * |scale| sum_r |u_r B_r|, where 2^-10 covers the
f32 sums (K <= 12288: 12288 * 2^-24 = 2^-10.4 at the very most) and the second order."""
import pytest
import torch

import b200attn
from b200attn import mmdit
from b200attn.lora import TARGETS, AdapterBank, BatchAdapters
from oracle import mmdit_ref as M


def lib_call(rows=4, segments=2, adapters=3, n=64, k=64, rank=16, ldx=None, ldy=None, ldo=None, x=16, y=16,
             out=32, a=16, b=16, seg=16, who=16):
    return b200attn.lib().b200_lora_add(x, ldx or k, a, b, y, ldy or n, out, ldo or n, seg, who, None, rows,
                                        segments, adapters, n, k, rank, None, None)


def test_refuses_bad_arguments():
    bad = b200attn.ERR_INVALID
    for name in ("rows", "segments", "adapters", "n"):
        assert lib_call(**{name: -1}) == bad
    assert lib_call(k=0) == bad and lib_call(k=60) == bad and lib_call(n=60) == bad
    assert lib_call(rank=0) == bad and lib_call(rank=12) == bad and lib_call(rank=136) == bad
    assert lib_call(ldx=56) == bad and lib_call(ldy=56) == bad and lib_call(ldo=56) == bad
    assert lib_call(ldx=68) == bad and lib_call(ldy=68) == bad and lib_call(ldo=68) == bad
    for name in ("x", "y", "out", "a", "b", "seg", "who"):
        assert lib_call(**{name: None}) == bad
    for name in ("x", "y", "out", "a", "b"):
        assert lib_call(**{name: 24}) == bad                  # not 16-byte aligned
    assert lib_call(y=16, out=16, ldo=72) == bad              # in place with another stride
    for name in ("rows", "segments", "n"):
        assert lib_call(**{name: 0}) == b200attn.OK           # nothing to do, nothing launched


def test_python_refuses_wrong_tensors():
    bf = torch.bfloat16
    x, y = torch.zeros(4, 64, dtype=bf), torch.zeros(4, 32, dtype=bf)
    a, b = torch.zeros(2, 16, 64, dtype=bf), torch.zeros(2, 32, 16, dtype=bf)
    seg, who = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        b200attn.lora_add(x, a, b, y, seg, who)
    with pytest.raises(ValueError, match="x must be"):
        b200attn.lora_add(x.float(), a, b, y, seg, who)
    with pytest.raises(ValueError, match="b must have"):
        b200attn.lora_add(x, a, b[:, :16], y, seg, who)
    with pytest.raises(ValueError, match="seg_start"):
        b200attn.lora_add(x, a, b, y, seg[:1], who)
    with pytest.raises(ValueError, match="seg_adapter"):
        b200attn.lora_add(x, a, b, y, seg, who.long())
    with pytest.raises(ValueError, match="scale"):
        b200attn.lora_add(x, a, b, y, seg, who, scale=torch.zeros(3))
    with pytest.raises(ValueError, match="rows of y"):
        b200attn.lora_add(x, a, b, y.t().contiguous().t(), seg, who)
    with pytest.raises(ValueError, match="out must"):
        b200attn.lora_add(x, a, b, y, seg, who, out=y[:3])


def make(g, lens, who, k, n, rank, adapters, pad=0):
    rows = sum(lens)
    x = torch.randn(rows, k + pad, generator=g).bfloat16()[:, :k]
    y = torch.randn(rows, n + pad, generator=g).bfloat16()[:, :n]
    a = (torch.randn(adapters, rank, k, generator=g) * k ** -0.5).bfloat16()
    b = torch.randn(adapters, n, rank, generator=g).bfloat16()
    scale = torch.rand(adapters, generator=g) * 2 - 1
    seg = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)
    return x, y, a, b, scale, seg, torch.tensor(who, dtype=torch.int32)


def check(got, x, y, a, b, scale, seg, who, before=None):
    got = got.cpu().double()
    want = (y if before is None else before).double().clone()
    size = torch.zeros_like(want)
    for s, e in enumerate(who.tolist()):
        r = slice(int(seg[s]), int(seg[s + 1]))
        if e < 0:
            want[r] = y[r].double()
            continue
        f = 1.0 if scale is None else float(scale[e])
        u = x[r].double() @ a[e].double().T
        want[r] = y[r].double() + f * (u @ b[e].double().T)
        size[r] = abs(f) * (u.abs() @ b[e].double().abs().T)
    off = (got - want).abs()
    assert (off <= 2 ** -8 * want.abs() + (2 ** -8 + 2 ** -10) * size).all(), off.max().item()


CASES = [  # (rows of each request, adapters of them, K, N, rank, adapters)
    ([1], [0], 64, 64, 16, 1),
    ([1], [0], 8, 8, 8, 1),
    ([1, 1, 1, 1], [2, 0, -1, 2], 4096, 4096, 16, 3),
    ([3, 0, 128, 129, 1], [0, 1, 1, 0, 1], 200, 136, 8, 2),
    ([127, 1, 128, 300], [1, -1, 0, 3], 1000, 520, 24, 4),
    ([64] * 40, [i % 3 - 1 for i in range(40)], 512, 256, 64, 2),
    ([1000], [0], 4096, 1024, 32, 1),
    ([700, 5], [1, 0], 768, 4096, 128, 2),
    ([2, 2], [0, 1], 136, 64, 72, 2),
    ([2500, 2600, 17], [0, 1, 0], 256, 640, 48, 2),
    ([40000], [0], 64, 72, 64, 1),
    *[([128] * tiles + [67], [i % 2 for i in range(tiles)] + [0], 1032, 1160, rank, 2)
      for tiles, rank in ((4, 16), (7, 64), (12, 32), (18, 128), (26, 48), (40, 16), (57, 64), (100, 8))],
    ([20000, 1], [0, 1], 72, 64, 128, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,who,k,n,rank,adapters", CASES)
def test_lora_add(cuda, lens, who, k, n, rank, adapters):
    g = torch.Generator().manual_seed(len(lens) * 1000 + k)
    x, y, a, b, scale, seg, w = make(g, lens, who, k, n, rank, adapters)
    dev = [t.to(cuda) for t in (x, a, b, y, seg, w)]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((sum(lens), n), 7.0, dtype=torch.bfloat16, device=cuda)
    got = b200attn.lora_add(*dev, scale=scale.to(cuda), out=out, status=status)
    assert got is out and status.item() == 0
    check(got, x, y, a, b, scale, seg, w)
    assert torch.equal(dev[3].cpu(), y)
    again = b200attn.lora_add(*dev, scale=scale.to(cuda), out=torch.empty_like(out))
    assert torch.equal(out, again)                            # sums in a fixed order
    inplace = b200attn.lora_add(*dev, scale=scale.to(cuda))   # in place: the same bits
    assert inplace is dev[3] and torch.equal(inplace, out)
    assert status.item() == 0


@pytest.mark.gpu
def test_row_strides_gaps_and_foreign_rows(cuda):
    """Rows wider than the operands, requests that leave rows out, NaN in the rows of others,
    no scale, and the bytes around the rows left as they were."""
    g = torch.Generator().manual_seed(5)
    k, n, pad = 320, 200, 24
    xf, yf = torch.randn(300, k + pad, generator=g).bfloat16(), torch.randn(300, n + pad, generator=g).bfloat16()
    xf[100:110] = float("nan")
    yf[100:110] = float("nan")
    _, _, a, b, _, _, _ = make(g, [1], [0], k, n, 40, 2)
    seg = torch.tensor([5, 100, 100, 110, 290], dtype=torch.int32)
    who = torch.tensor([1, 0, -1, 0], dtype=torch.int32)
    y_dev = yf.to(cuda)
    b200attn.lora_add(xf.to(cuda)[:, :k], a.to(cuda), b.to(cuda), y_dev[:, :n], seg.to(cuda), who.to(cuda))
    got = y_dev.cpu()
    assert torch.equal(got[:, n:].nan_to_num(9), yf[:, n:].nan_to_num(9))
    for r in (slice(0, 5), slice(290, 300), slice(100, 110)):
        assert torch.equal(got[r].nan_to_num(9), yf[r].nan_to_num(9))
    keep = [r for r in range(300) if not 100 <= r < 110]
    ident = torch.tensor([5, 100, 280], dtype=torch.int32)
    check(got[keep, :n], xf[keep, :k], yf[keep, :n], a, b, None, ident, torch.tensor([1, 0]), before=yf[keep, :n])


@pytest.mark.gpu
def test_bad_adapters_and_segments_stay_in_bounds(cuda):
    """An adapter that is not there counts as none and is reported; starts outside the rows
    are limited to them."""
    g = torch.Generator().manual_seed(6)
    x, y, a, b, scale, _, _ = make(g, [50], [0], 128, 64, 16, 2)
    seg = torch.tensor([-20, 10, 30, 4000], dtype=torch.int32)
    who = torch.tensor([0, 2, 1], dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = b200attn.lora_add(*(t.to(cuda) for t in (x, a, b, y, seg, who)), scale=scale.to(cuda),
                            out=torch.zeros(50, 64, dtype=torch.bfloat16, device=cuda), status=status)
    assert status.item() == b200attn.LORA_STATUS_BAD_ADAPTER
    check(got, x, y, a, b, scale, torch.tensor([0, 10, 30, 50]), torch.tensor([0, -1, 1]))


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda):
    """A captured call replayed with other adapters, rows and inputs, and a call on a stream
    of its own, equal the plain call."""
    g = torch.Generator().manual_seed(8)
    x, y, a, b, scale, seg, who = (t.to(cuda) for t in make(g, [70, 130, 1], [0, 1, -1], 512, 384, 16, 2))
    out = torch.empty_like(y)
    call = lambda stream=None: b200attn.lora_add(x, a, b, y, seg, who, scale=scale, out=out, stream=stream)
    plain = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out.zero_()
    torch.cuda.synchronize()
    call(side)
    side.synchronize()
    assert torch.equal(out, plain)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    x.copy_(torch.randn(x.shape, generator=g))
    seg.copy_(torch.tensor([0, 1, 200, 201]))
    who.copy_(torch.tensor([1, -1, 0]))
    graph.replay()
    replayed = out.clone()
    out.zero_()
    assert torch.equal(replayed, call()) and not torch.equal(replayed, plain)


# ----------------------------------------------------------------- the model's adapters
TINY = mmdit.MMDiTConfig(layers=2, heads=2, text_dim=256)
GRID = (16, 16)


def _adapter(g, rank, names):
    shapes = {k[:-len(".weight")]: v for k, v in mmdit.weight_shapes(TINY).items()}
    return {n: (torch.randn(rank, shapes[n][1], generator=g) * shapes[n][1] ** -0.5,
                torch.randn(shapes[n][0], rank, generator=g) * 0.1) for n in names}


def _names(layer, targets=TARGETS):
    return [f"transformer_blocks.{layer}.{t}" for t in targets]


def test_bank_refuses_what_does_not_fit():
    g = torch.Generator().manual_seed(0)
    good = _adapter(g, 4, _names(0))
    bank = AdapterBank([good], device="cpu")
    assert bank.linears["transformer_blocks.0.attn.to_q"][0].shape == (1, 8, 256)  # ranks in eights
    with pytest.raises(ValueError):
        AdapterBank([], device="cpu")
    with pytest.raises(ValueError, match="scale"):
        AdapterBank([good], scales=[1.0, 2.0], device="cpu")
    with pytest.raises(ValueError, match="block linear"):
        AdapterBank([{"proj_out": (torch.zeros(4, 8), torch.zeros(8, 4))}], device="cpu")
    with pytest.raises(ValueError, match="block linear"):
        AdapterBank([{"transformer_blocks.0": (torch.zeros(4, 8), torch.zeros(8, 4))}], device="cpu")
    n = "transformer_blocks.0.attn.to_q"
    with pytest.raises(ValueError, match="fit together"):
        AdapterBank([{n: (torch.zeros(4, 8), torch.zeros(8, 5))}], device="cpu")
    with pytest.raises(ValueError, match="fit together"):
        AdapterBank([{n: (torch.zeros(4, 8), torch.zeros(8, 4))}, {n: (torch.zeros(4, 16), torch.zeros(8, 4))}],
                    device="cpu")
    with pytest.raises(ValueError, match="rank"):
        AdapterBank([{n: (torch.zeros(130, 8), torch.zeros(8, 130))}], device="cpu")
    with pytest.raises(ValueError, match="adapters"):
        BatchAdapters(bank, [1], 4)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "q4_k_m"])
def test_every_sequence_with_its_own_adapter(cuda, fmt):
    """A batched prefix fill and step whose sequences carry different adapters (of different
    ranks, on different linears, or none) against the float32 oracle with each adapter merged
    into the weights, sequence by sequence; the MLP in chunks that cut sequences."""
    w = mmdit.random_weights(TINY, 0, std=0.1)
    model = mmdit.MMDiT(TINY, w, device=cuda, weight_format=fmt, mlp_chunk_rows=200)
    g = torch.Generator().manual_seed(11)
    adapters = [_adapter(g, 8, _names(0) + _names(1)), _adapter(g, 20, _names(1, TARGETS[2:5]))]
    scales = [0.7, 1.3]
    model.set_adapters(AdapterBank(adapters, scales, cuda))
    lengths, ids = [40, 72, 65], [1, None, 0]
    embs = [torch.randn(n, 256, generator=g).to(torch.bfloat16) for n in lengths]
    lat = torch.randn(3, 256, 64, generator=g)
    cache = model.prefix_fill(embs, adapters=ids)
    got = model.step(lat.to(cuda), 0.5, cache, model.target_pe(lengths, GRID),
                     mmdit.cached_desc(cache, 256, cuda), adapters=ids).cpu()
    base = model.effective_weights(w)
    for b, e in enumerate(ids):
        merged = dict(base)
        if e is not None:
            for name, (A, B) in adapters[e].items():
                merged[name + ".weight"] = base[name + ".weight"].float() + scales[e] * (
                    B.bfloat16().float() @ A.bfloat16().float())
        R = M.Reference(merged, TINY.layers, TINY.heads)
        want = R.forward_cached(lat[b], 0.5, R.prefix_kv(embs[b].float(), GRID), lengths[b], GRID)
        rel = float((got[b].double() - want.double()).norm() / want.double().norm())
        assert rel <= 1.5e-2, (b, rel)
    with pytest.raises(ValueError, match="adapter ids"):
        model.prefix_fill(embs, adapters=[0])
    for wrong in ({"transformer_blocks.2.attn.to_q": (torch.zeros(8, 256), torch.zeros(256, 8))},
                  {"transformer_blocks.0.attn.to_q": (torch.zeros(8, 128), torch.zeros(256, 8))}):
        with pytest.raises(ValueError, match="shape"):
            model.set_adapters(AdapterBank([wrong], device=cuda))
    model.set_adapters(None)
    with pytest.raises(ValueError, match="no adapters"):
        model.prefix_fill(embs, adapters=ids)


@pytest.mark.gpu
def test_rows_behind_32_bit_offsets(cuda):
    """y of more than 2^32 elements: requests at its start and end."""
    rows, n, k, rank = 350000, 12296, 64, 8
    g = torch.Generator().manual_seed(2)
    x = torch.randn(rows, k, device=cuda, dtype=torch.bfloat16)
    y = torch.zeros(rows, n, device=cuda, dtype=torch.bfloat16)
    a = (torch.randn(2, rank, k, generator=g) * k ** -0.5).bfloat16()
    b = torch.randn(2, n, rank, generator=g).bfloat16()
    seg = torch.tensor([0, 3, rows - 130, rows], dtype=torch.int32)
    who = torch.tensor([1, -1, 0], dtype=torch.int32)
    b200attn.lora_add(x, a.to(cuda), b.to(cuda), y, seg.to(cuda), who.to(cuda))
    assert not y[3:rows - 130].any()
    for r, e in ((slice(0, 3), 1), (slice(rows - 130, rows), 0)):
        ident = torch.tensor([0, r.stop - r.start])
        check(y[r], x[r].cpu(), torch.zeros(r.stop - r.start, n), a, b, None, ident, torch.tensor([e]))


@pytest.mark.gpu
def test_calls_at_once_on_two_streams(cuda):
    g = torch.Generator().manual_seed(12)
    args = []
    for lens, k, n, rank in (([300, 5], 1024, 2048, 16), ([1000], 512, 768, 128)):
        x, y, a, b, scale, seg, who = make(g, lens, [0] * len(lens), k, n, rank, 1)
        args.append((torch.cuda.Stream(), [t.to(cuda) for t in (x, a, b, y, seg, who)], [], (x, y, a, b, None, seg, who)))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, dev, outs, _ in args:
            with torch.cuda.stream(s):
                outs.append(b200attn.lora_add(*dev, out=torch.empty_like(dev[3])))
    torch.cuda.synchronize()
    for s, dev, outs, (x, y, a, b, scale, seg, who) in args:
        assert all(torch.equal(o, outs[0]) for o in outs)
        check(outs[0], x, y, a, b, scale, seg, who)


@pytest.mark.gpu
def test_a_status_word_elsewhere_is_refused(cuda):
    g = torch.Generator().manual_seed(1)
    x, y, a, b, scale, seg, who = (t.to(cuda) for t in make(g, [4], [0], 64, 64, 8, 1))
    for status in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device=cuda),
                   torch.zeros(0, dtype=torch.int32, device=cuda)):
        with pytest.raises(ValueError, match="status"):
            b200attn.lora_add(x, a, b, y, seg, who, status=status)


@pytest.mark.gpu
def test_ranks_from_several_threads(cuda):
    """Host threads that launch with different ranks (and so different shared memory)."""
    import threading
    g = torch.Generator().manual_seed(3)
    jobs = [make(g, [200], [0], 256, 512, r, 1) for r in (16, 128, 64, 72)]
    outs, failed = {}, []

    def run(i):
        try:
            x, y, a, b, scale, seg, who = (t.to(cuda) for t in jobs[i])
            for _ in range(50):
                outs[i] = b200attn.lora_add(x, a, b, y, seg, who, scale=scale, out=torch.empty_like(y))
        except Exception as e:  # reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for i, (x, y, a, b, scale, seg, who) in enumerate(jobs):
        check(outs[i], x, y, a, b, scale, seg, who)
