"""The paged 4-bit prefix cache: its bytes, refusals and page copies, and joint attention
over it, against a plain 64-bit implementation.

Tolerances.  Reading the cache is exact, so stored values are compared bit for bit.
Attention: P enters the P.V product rounded to bf16 (after its V step, or as it is), at most
2^-8 of each term, and the output is rounded to bf16, at most 2^-8 of it; scores are f32 sums
of 128 products of |q.k| up to ~60, at most 128 * 2^-24 * 60 ~ 5e-4 off, which moves p by as
much.  Per element: |got - want| <= 2^-8 |want| + (2^-8 + 2e-3) * sum_j p_j |v_j|, and
2e-3 covers the scores' and exp2's errors four times over."""
import ctypes
import math

import numpy as np
import pytest
import torch

import b200attn

D, PAGE, BLOCK = 128, 64, 9216
TINY, HUGE = 2.0 ** -100, 2.0 ** 126


# ----------------------------------------------------------------- plain definition
def quantise(x):
    """[..., 128] -> numbers int [..., 128] and steps f64 [..., 4], in 64 bits."""
    g = x.double().reshape(*x.shape[:-1], 4, 32)
    top = g.abs().amax(-1)
    frac, power = torch.frexp(top / 7)
    step = torch.ldexp(torch.floor(frac * 32) / 32, power)
    step = torch.where(top < TINY, 0.0, step)
    step = torch.where(top < HUGE, step, math.nan)
    use = (step > 0)[..., None]
    num = torch.where(use, torch.sign(g) * torch.floor(g.abs() / step[..., None] + 0.5), 0.0)
    return num.reshape(x.shape), step


def values(x):
    num, step = quantise(x)
    return (num.reshape(*x.shape[:-1], 4, 32) * step[..., None]).reshape(x.shape)


def k_nibble(tok, ch):
    """(byte of the block, high nibble?) of K's number of token tok, channel ch."""
    a, g, c, t, j = tok // 8, tok % 8, ch // 32, ch % 32 // 8, ch % 8
    return a * 512 + (4 * g + t) * 16 + c * 4 + j // 2, j % 2


def v_nibble(tok, ch):
    a, t, p, c, g, i = tok // 8, tok % 8 // 2, tok % 2, ch // 32, ch % 32 // 4, ch % 4
    return 4096 + a * 512 + (4 * g + t) * 16 + c * 4 + p * 2 + i // 2, i % 2


def step_at(tok, c, part):
    a, t, p = tok // 8, tok % 8 // 2, tok % 2
    return 8192 + 512 * part + 2 * (a * 32 + t * 8 + 2 * c + p)


def decode(block, part):
    """One block (uint8 numpy [9216]) -> f64 [64, 128] of K (part 0) or V (part 1)."""
    out = np.zeros((PAGE, D))
    where = k_nibble if part == 0 else v_nibble
    for tok in range(PAGE):
        steps = [np.uint32(int(block[step_at(tok, c, part)]) | int(block[step_at(tok, c, part) + 1]) << 8)
                 for c in range(4)]
        steps = [(s << np.uint32(16)).view(np.float32) for s in steps]
        for ch in range(D):
            byte, high = where(tok, ch)
            out[tok, ch] = ((int(block[byte]) >> (4 * high) & 15) - 8) * float(steps[ch // 32])
    return out


def test_block_layout_is_a_bijection():
    for where, lo in ((k_nibble, 0), (v_nibble, 4096)):
        seen = {where(t, c) for t in range(PAGE) for c in range(D)}
        assert len(seen) == PAGE * D and {b for b, _ in seen} == set(range(lo, lo + 4096))
    seen = {step_at(t, c, p) for t in range(PAGE) for c in range(4) for p in range(2)}
    assert seen == set(range(8192, BLOCK, 2))


def test_every_value_is_a_bf16_number():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(4000, D, generator=g) * torch.exp(8 * torch.randn(4000, 1, generator=g))).bfloat16()
    x[0, :32] = 8.4e37  # next to the largest magnitude that a group may have
    v = values(x)
    assert torch.equal(v, v.to(torch.bfloat16).double())
    num, step = quantise(x)
    assert num.abs().max() == 7
    off = (v - x.double()).abs().reshape(-1, 4, 32)
    assert (off <= step[..., None] * 0.5).all()


# ----------------------------------------------------------------- refusals (CPU)
def view(pool=16, table=16, num_pages=4, max_pages=2):
    return ctypes.byref(b200attn.Kv4View(pool, table, num_pages, max_pages))


def test_store_and_load_refuse_bad_arguments():
    L, bad = b200attn.lib(), b200attn.ERR_INVALID

    def store(v=None, k=16, d=128, b=1, h=2, t=3, st=(128 * 6, 128 * 3, 128)):
        return L.b200_kv4_store(v or view(), k, *st, 16, *st, b, h, t, d, None, None, None, None)

    assert store(d=64) == b200attn.ERR_UNSUPPORTED
    assert store(b=-1) == bad and store(h=-1) == bad and store(t=-1) == bad
    assert store(b=70000) == bad and store(h=70000) == bad
    assert store(k=None) == bad and store(k=8) == bad
    assert store(st=(768, 384, 4)) == bad                    # rows not 16-byte aligned
    assert store(view(pool=None)) == bad and store(view(pool=8)) == bad
    assert store(view(table=None)) == bad and store(view(table=18)) == bad
    assert store(view(num_pages=-1)) == bad and store(view(max_pages=-1)) == bad
    assert L.b200_kv4_store(None, 16, 0, 0, 0, 16, 0, 0, 0, 1, 1, 1, 128, None, None, None, None) == bad
    for zero in ("b", "h", "t"):
        assert store(**{zero: 0}) == b200attn.OK             # nothing to do, nothing launched

    def load(v=None, k=16, out_v=16, d=128, b=1, h=2, n=128, stride=1):
        return L.b200_kv4_load(v or view(), None, stride, k, out_v, b, h, n, d, None, None)

    assert load(d=64) == b200attn.ERR_UNSUPPORTED
    assert load(n=129) == bad                                # behind the page table
    assert load(n=2**31 - 1, v=view(max_pages=2**30)) == bad
    assert load(n=-1) == bad and load(b=-1) == bad and load(stride=-1) == bad
    assert load(k=None) == bad and load(out_v=8) == bad
    assert load(n=0) == b200attn.OK and load(b=0) == b200attn.OK


def test_attention_refuses_bad_arguments():
    L, bad = b200attn.lib(), b200attn.ERR_INVALID

    def attend(v=None, q=16, out=16, b=1, h=2, t=3, p=128, d=128, scale=0.1, ws=None, n=0):
        return L.b200_kv4_joint_attention(v or view(), q, 16, 16, b, h, t, p, d, None, None, scale, out,
                                          ws, n, None, None)

    assert attend(d=64) == b200attn.ERR_UNSUPPORTED
    assert attend(b=0) == bad and attend(h=0) == bad and attend(t=-1) == bad and attend(p=-1) == bad
    assert attend(p=129) == bad                              # more tokens than the table has room for
    assert attend(q=None) == bad and attend(q=8) == bad and attend(out=None) == bad and attend(ws=8) == bad
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert attend(scale=scale) == bad
    assert attend(view(pool=None)) == bad
    assert attend(t=0) == b200attn.OK
    # many rows expand the pages into a workspace
    need = b200attn.kv4_workspace_bytes(1, 2, 200, 128)
    assert need >= 2 * 2 * 128 * D * 2 and b200attn.kv4_workspace_bytes(4, 32, 65, 128) > need
    assert b200attn.kv4_workspace_bytes(4, 32, 64, 128) == b200attn.kv4_workspace_bytes(1, 2, 128, 512) == 0
    assert b200attn.kv4_workspace_bytes(1, 2, 128, 511) > 0
    assert attend(t=200) == b200attn.ERR_WORKSPACE
    assert attend(t=200, ws=256, n=need - 1) == b200attn.ERR_WORKSPACE

    a = b200attn.AttnArgs()
    a.batch, a.heads, a.head_dim, a.target_len, a.prefix_len, a.scale = 1, 2, 128, 4, 128, 0.1
    for f in ("q", "k", "v", "out", "norm_q_w", "norm_k_w", "pe"):
        setattr(a, f, 16)
    fwd = lambda: L.b200_kv4_attn_fwd(ctypes.byref(a), view(), None)
    assert fwd() == b200attn.ERR_WORKSPACE
    a.prefix_k = 16
    assert fwd() == bad                                      # the prefix is in the cache
    a.prefix_k, a.prefix_len = None, 129
    assert fwd() == bad
    a.prefix_len, a.pe = 128, None
    assert fwd() == bad


def test_copy_pages_refuses_bad_pages():
    L, bad = b200attn.lib(), b200attn.ERR_INVALID

    def copy(src, dst, pages=8, layers=2, stride=8 * 4 * BLOCK, pool=16):
        n = len(src)
        return L.b200_kv4_copy_pages(pool, layers, stride, pages, 4, (ctypes.c_int32 * n)(*src),
                                     (ctypes.c_int32 * n)(*dst), n, None)

    assert copy([8], [0]) == bad and copy([0], [8]) == bad
    assert copy([-1], [0]) == bad and copy([0], [-1]) == bad
    assert copy([0, 1], [2, 2]) == bad                       # written twice
    assert copy([0, 1], [1, 2]) == bad                       # 1 is read and written
    assert copy([3], [3]) == bad
    assert copy([0], [1], stride=8 * 4 * BLOCK - 16) == bad  # layers overlap
    assert copy([0], [1], stride=8 * 4 * BLOCK + 8) == bad
    assert copy([0], [1], pool=None) == bad and copy([0], [1], pool=8) == bad
    assert L.b200_kv4_copy_pages(16, 1, 0, 8, 4, None, None, 1, None) == bad
    assert copy([], []) == b200attn.OK


def test_python_refuses_wrong_tensors():
    pool = torch.zeros(3, 2, BLOCK, dtype=torch.uint8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    k = torch.zeros(1, 2, 5, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        b200attn.kv4_store(k, k, pool, table)
    with pytest.raises(ValueError, match="pool"):
        b200attn.kv4_store(k, k, pool[:, :1], table)
    with pytest.raises(ValueError, match="page_table"):
        b200attn.kv4_store(k, k, pool, table.long())
    with pytest.raises(ValueError, match="page_table"):
        b200attn.kv4_store(k, k, pool, table.expand(2, 2))
    with pytest.raises(ValueError, match="k must be"):
        b200attn.kv4_store(k.float(), k, pool, table)
    with pytest.raises(ValueError, match="dense"):
        b200attn.kv4_store(k.transpose(2, 3).contiguous().transpose(2, 3), k, pool, table)
    with pytest.raises(ValueError, match="start"):
        b200attn.kv4_store(k, k, pool, table, start=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="k_rot"):
        b200attn.kv4_joint_attention(k, k[:, :, :4], k.transpose(1, 2).contiguous(), pool, table, 5)
    with pytest.raises(ValueError, match="desc"):
        b200attn.kv4_joint_attention(k, k, k.transpose(1, 2).contiguous(), pool, table, 5,
                                     desc=torch.zeros(1, 2))
    with pytest.raises(ValueError, match="same length"):
        b200attn.kv4_copy_pages(pool, [0], [])
    with pytest.raises(ValueError, match="CUDA"):
        b200attn.kv4_copy_pages(pool, [0], [1])


# ----------------------------------------------------------------- GPU
def paged(cuda, lengths, heads, spare=2, seed=0):
    """Random bytes everywhere, and a table of pages in random order, -1 behind each row's."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g).int()
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pool = torch.randint(0, 256, (len(order), heads, BLOCK), generator=g).to(torch.uint8)
    return pool.to(cuda), table.to(cuda), g


def i32(cuda, *v):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


@pytest.mark.gpu
def test_stored_bytes_follow_the_layout(cuda):
    """Every byte of a block, decoded one by one; values with exact halves, zeros, one tiny
    and one enormous group among them."""
    pool, table, g = paged(cuda, [64], 2)
    x = torch.randn(2, 1, 2, 64, D, generator=g).bfloat16()
    x[0, 0, 0, 0] = (torch.arange(D) % 29 - 14) * 0.25   # halves of the step 1/2
    x[0, 0, 0, 1, :32] = 0
    x[0, 0, 0, 2, 32:64] = 2.0 ** -110
    x[1, 0, 1, 3, 64:96] = 8.4e37
    b200attn.kv4_store(x[0].to(cuda), x[1].to(cuda), pool, table)
    blocks = pool[table[0, 0].item()].cpu().numpy()
    for part in range(2):
        for h in range(2):
            want = values(x[part, 0, h]).numpy()
            assert np.array_equal(decode(blocks[h], part), want)


@pytest.mark.gpu
def test_numbers_at_every_border(cuda):
    """Every 8-bit largest magnitude of a group (all 128 mantissas) with every mantissa of the
    other values at the exponents where a number can be 1 to 7, both signs: the halves that
    are exact and the values next to a border get the definition's numbers."""
    mant = 1 + torch.arange(128).double() / 128
    other = torch.cat([mant * 2.0 ** e for e in range(-5, 1)])           # 768 values up to 2
    other = torch.cat([other, -other])
    rows = []
    for top in mant:
        use = other[other.abs() <= top]
        use = torch.nn.functional.pad(use, (0, -len(use) % 31))
        part = use.reshape(-1, 31)
        rows.append(torch.cat([torch.full((len(part), 1), float(top)), part.float()], 1))
    x = torch.cat(rows)
    x = torch.nn.functional.pad(x, (0, 0, 0, -len(x) % 4)).reshape(-1, D).bfloat16()
    assert torch.equal(x.double().reshape(-1, 32)[:len(rows[0])], rows[0].double())
    x = x.reshape(1, 1, -1, D)
    n = x.shape[2]
    pool, table, _ = paged(cuda, [n], 1)
    b200attn.kv4_store(x.to(cuda), -x.to(cuda), pool, table)
    k, v = b200attn.kv4_load(pool, table, None, n)
    assert torch.equal(k.cpu().double(), values(x)) and torch.equal(v.cpu().double(), values(-x))


@pytest.mark.gpu
@pytest.mark.parametrize("starts,counts,tokens,heads", [
    ([0], [1], 1, 1), ([63], [2], 2, 3), ([0, 5, 64], [130, 1, 0], 130, 2),
    ([7, 200], [64, 3], 64, 4), ([15, 16, 17], [16, 15, 33], 33, 1), ([1], [511], 600, 5),
])
def test_store_then_load(cuda, starts, counts, tokens, heads):
    """Appending leaves what the pages held before, to the byte, and pages of no row."""
    ends = [s + min(c, tokens) for s, c in zip(starts, counts)]
    pool, table, g = paged(cuda, ends, heads)
    b = len(starts)
    old = torch.randn(2, b, heads, max(max(starts), 1), D, generator=g).bfloat16().to(cuda)
    b200attn.kv4_store(old[0], old[1], pool, table, count=i32(cuda, *starts))
    before = pool.clone()
    k = torch.randn(b, heads, tokens, D, generator=g).bfloat16().to(cuda)
    v = torch.randn(b, tokens, heads, D, generator=g).bfloat16().to(cuda).transpose(1, 2)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    b200attn.kv4_store(k, v, pool, table, i32(cuda, *starts), i32(cuda, *counts), status=status)
    most = max(ends) + 3 if max(ends) % PAGE < PAGE - 3 and max(ends) % PAGE else max(ends)
    got = b200attn.kv4_load(pool, table, i32(cuda, *ends), most, status=status)
    assert status.item() == 0
    for part, (new, was) in enumerate(((k, old[0]), (v, old[1]))):
        want = torch.zeros(b, heads, most, D, dtype=torch.float64)
        for i in range(b):
            want[i, :, :starts[i]] = values(was[i, :, :starts[i]].cpu())
            want[i, :, starts[i]:ends[i]] = values(new[i, :, :ends[i] - starts[i]].cpu())
        assert torch.equal(got[part].cpu().double(), want)
    used = {int(x) for x in table.flatten() if x >= 0}
    rest = [i for i in range(pool.shape[0]) if i not in used]
    assert torch.equal(pool[rest], before[rest])
    # storing the same again changes no byte; bytes behind the last token stay random
    again = pool.clone()
    b200attn.kv4_store(k, v, pool, table, i32(cuda, *starts), i32(cuda, *counts))
    assert torch.equal(pool, again)
    i = int(np.argmax(ends))
    if ends[i] % PAGE:
        page = int(table[i, ends[i] // PAGE])
        for tok in range(ends[i] % PAGE, PAGE):
            for ch in (0, 31, 77, 127):
                for byte, _ in (k_nibble(tok, ch), v_nibble(tok, ch)):
                    assert torch.equal(pool[page, :, byte], before[page, :, byte])


@pytest.mark.gpu
def test_non_finite_groups_read_as_nan(cuda):
    pool, table, g = paged(cuda, [4], 1)
    x = torch.randn(1, 1, 4, D, generator=g).bfloat16()
    x[0, 0, 0, 5], x[0, 0, 1, 40], x[0, 0, 2, 127], x[0, 0, 3, 0] = math.inf, -math.inf, math.nan, 2.0 ** 126
    b200attn.kv4_store(x.to(cuda), x.to(cuda), pool, table)
    for got in b200attn.kv4_load(pool, table, None, 4):
        nan = torch.isnan(got.cpu()).reshape(4, 4, 32)
        assert nan[0, 0].all() and nan[1, 1].all() and nan[2, 3].all() and nan[3, 0].all()
        assert nan.sum() == 128


@pytest.mark.gpu
def test_bad_pages_are_left_out_and_reported(cuda):
    """Ids outside the pool and positions outside the table: not stored, read as zeros."""
    pool, table, g = paged(cuda, [200], 2)
    before = pool.clone()
    k = torch.randn(1, 2, 200, D, generator=g).bfloat16().to(cuda)
    broken = table.clone()
    broken[0, 1], broken[0, 2] = pool.shape[0], -7
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    b200attn.kv4_store(k, k, pool, broken, status=status)
    assert status.item() == b200attn.KV4_STATUS_BAD_PAGE
    assert torch.equal(pool[table[0, 1:3].long()], before[table[0, 1:3].long()])
    status.zero_()
    b200attn.kv4_store(k, k, pool, table, start=i32(cuda, 256 - 10), status=status)
    assert status.item() == b200attn.KV4_STATUS_BAD_PAGE
    status.zero_()
    kk, _ = b200attn.kv4_load(pool, broken, None, 200, status=status)
    assert status.item() == b200attn.KV4_STATUS_BAD_PAGE
    assert torch.equal(kk[0, :, 64:192], torch.zeros_like(kk[0, :, 64:192]))
    for t in (5, 40, 150):  # the three forms of the attention: such tokens count as keys of zeros
        q, ko = (torch.randn(1, 2, t, D, generator=g).bfloat16().to(cuda) for _ in range(2))
        vo = torch.randn(1, t, 2, D, generator=g).bfloat16().to(cuda)
        status.zero_()
        got = b200attn.kv4_joint_attention(q, ko, vo, pool, broken, 200, status=status)
        assert status.item() == b200attn.KV4_STATUS_BAD_PAGE
        dense = b200attn.kv4_load(pool, broken, None, 200)
        check(got, q, ko, vo, dense[0], dense[1], [(200, t)])


def check(got, q, ko, vo, pk, pv, desc, limit=None):
    """got against 64-bit attention over [pk, pv (cache values) ; ko, vo], see the tolerances
    above."""
    b, h, t, _ = q.shape
    got = got.cpu().double().reshape(b, t, h, D)
    for i, (n, m) in enumerate(desc):
        keys = torch.cat([pk[i, :, :n].cpu().double(), ko[i, :, :m].cpu().double()], 1)
        vals = torch.cat([pv[i, :, :n].cpu().double(), vo[i, :m].transpose(0, 1).cpu().double()], 1)
        x = q[i].cpu().double() @ keys.transpose(1, 2) / math.sqrt(D)
        if limit is not None:
            hide = torch.arange(m).view(1, -1) >= limit.view(-1, 1)
            x[:, :, n:] = x[:, :, n:].masked_fill(hide, -math.inf)
        p = torch.softmax(x, -1)
        want, size = (p @ vals).transpose(0, 1), (p @ vals.abs()).transpose(0, 1)
        if n + m == 0:  # an empty softmax: torch's empty product would say 0
            want = torch.full_like(want, math.nan)
        none = torch.isnan(want)
        assert torch.equal(none, torch.isnan(got[i])), i
        off = (got[i] - want).abs()
        ok = off <= 2 ** -8 * want.abs() + (2 ** -8 + 2e-3) * size
        assert (ok | none).all(), (i, off[~none].max().item())


ATTEND = [  # (prefix lengths, tokens, target_valid, heads, causal)
    ([1], 1, [1], 1, False), ([0], 1, [1], 2, False), ([64], 1, [1], 32, False),
    ([65, 0, 63], 1, [1, 1, 0], 3, False), ([513], 2, [2], 4, True),
    ([17, 1000, 300], 16, [16, 9, 1], 2, True), ([2000], 17, [17], 3, False),
    ([100, 7], 37, [37, 20], 5, True), ([5000], 64, [64], 1, True),
    ([129, 30], 65, [65, 40], 2, True), ([700, 0], 300, [300, 299], 3, False),
    ([33], 33, [33], 2, True), ([520, 3, 0], 48, [48, 1, 0], 3, False), ([600, 2], 100, [100, 99], 2, True),
    ([3000], 50, [50], 1, False), ([1500, 1500], 128, [128, 60], 1, True),
    ([300, 64, 1], 129, [129, 70, 0], 2, True), ([70] * 5, 66, [66, 65, 3, 1, 0], 16, True),
    ([0, 0], 5, [5, 0], 2, True), ([0, 64], 130, [0, 130], 1, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,tokens,valid,heads,causal", ATTEND)
def test_joint_attention(cuda, lengths, tokens, valid, heads, causal):
    """Ragged prefixes and targets, empty ones, rows without any key (NaN), every byte that
    no valid token owns random (steps that are NaN among them), and infinities and NaN behind
    target_valid in K and V."""
    pool, table, g = paged(cuda, lengths, heads, seed=tokens)
    b, most = len(lengths), max(lengths)
    dense = torch.randn(2, b, heads, max(most, 1), D, generator=g).bfloat16()
    b200attn.kv4_store(dense[0].to(cuda), dense[1].to(cuda), pool, table, count=i32(cuda, *lengths))
    q, ko = (torch.randn(b, heads, tokens, D, generator=g).bfloat16() for _ in range(2))
    vo = torch.randn(b, tokens, heads, D, generator=g).bfloat16()
    for i, m in enumerate(valid):
        ko[i, :, m:] = math.nan
        vo[i, m:] = math.inf if i % 2 else math.nan
    desc = torch.tensor(list(zip(lengths, valid)), dtype=torch.int32, device=cuda)
    limit = torch.arange(1, tokens + 1, dtype=torch.int32) if causal else None
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = b200attn.kv4_joint_attention(q.to(cuda), ko.to(cuda), vo.to(cuda), pool, table, most, desc=desc,
                                       row_limit=None if limit is None else limit.to(cuda), status=status)
    assert status.item() == 0
    check(got, q, ko, vo, values(dense[0]), values(dense[1]), list(zip(lengths, valid)), limit)


@pytest.mark.gpu
def test_pages_behind_32_bit_offsets(cuda):
    """A pool of more than 4 GiB: its last pages are stored, read, copied and attended to."""
    heads, pages = 32, 15000
    pool = torch.zeros(pages, heads, BLOCK, dtype=torch.uint8, device=cuda)
    table = i32(cuda, pages - 1, 0, pages - 2).view(1, 3)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, heads, 150, D, generator=g).bfloat16() for _ in range(2))
    b200attn.kv4_store(k.to(cuda), v.to(cuda), pool, table)
    b200attn.kv4_copy_pages(pool, [pages - 1], [pages - 3])
    assert torch.equal(pool[pages - 1], pool[pages - 3])
    table[0, 0] = pages - 3
    pool[pages - 1].zero_()
    got = b200attn.kv4_load(pool, table, None, 150)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.cpu().double(), values(y))
    for t in (3, 40, 129):
        q, ko = (torch.randn(1, heads, t, D, generator=g).bfloat16().to(cuda) for _ in range(2))
        vo = torch.randn(1, t, heads, D, generator=g).bfloat16().to(cuda)
        check(b200attn.kv4_joint_attention(q, ko, vo, pool, table, 150), q, ko, vo, values(k), values(v), [(150, t)])


@pytest.mark.gpu
def test_dense_attention_ignores_values_behind_the_valid_keys(cuda):
    """The dense joint attention: infinities and NaN in K and V behind the valid keys of the
    prefix and of the call do not reach the output."""
    g = torch.Generator().manual_seed(9)
    b, h, t, p = 2, 2, 200, 300
    q, k = (torch.randn(b, h, t, D, generator=g).bfloat16() for _ in range(2))
    v = torch.randn(b, t, h, D, generator=g).bfloat16()
    pk, pv = (torch.randn(b, h, p, D, generator=g).bfloat16() for _ in range(2))
    desc = [(300, 130), (37, 200)]
    for i, (n, m) in enumerate(desc):
        pk[i, :, n:], pv[i, :, n:] = math.nan, math.inf
        k[i, :, m:], v[i, m:] = math.inf, math.nan
    got = b200attn.joint_attention(*(x.to(cuda) for x in (q, k, v, pk, pv)),
                                   desc=torch.tensor(desc, dtype=torch.int32, device=cuda))
    check(got, q, k, v, pk.double(), pv.double(), desc)


@pytest.mark.gpu
def test_calls_at_once_on_two_streams(cuda):
    """Two streams that attend over and extend the same pool at the same time, each with its
    own sequences and workspace."""
    pool, table, g = paged(cuda, [1200, 900], 4)
    dense = torch.randn(2, 2, 4, 1200, D, generator=g).bfloat16()
    b200attn.kv4_store(dense[0].to(cuda), dense[1].to(cuda), pool, table, count=i32(cuda, 1200, 900))
    work = []
    for i, t in ((0, 6), (1, 150)):
        q, ko = (torch.randn(1, 4, t, D, generator=g).bfloat16().to(cuda) for _ in range(2))
        vo = torch.randn(1, t, 4, D, generator=g).bfloat16().to(cuda)
        work.append((torch.cuda.Stream(), q, ko, vo, table[i:i + 1].contiguous(), (1200, 900)[i], []))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, q, ko, vo, tab, n, outs in work:
            outs.append(b200attn.kv4_joint_attention(q, ko, vo, pool, tab, n, stream=s))
    torch.cuda.synchronize()
    for i, (s, q, ko, vo, tab, n, outs) in enumerate(work):
        assert all(torch.equal(o, outs[0]) for o in outs)
        check(outs[0], q, ko, vo, values(dense[0, i:i + 1]), values(dense[1, i:i + 1]), [(n, q.shape[2])])


@pytest.mark.gpu
def test_status_and_workspace_elsewhere_are_refused(cuda):
    pool, table, g = paged(cuda, [64], 1)
    q = torch.zeros(1, 1, 200, D, dtype=torch.bfloat16, device=cuda)
    v = q.transpose(1, 2).contiguous()
    with pytest.raises(ValueError, match="status"):
        b200attn.kv4_joint_attention(q, q, v, pool, table, 64, status=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="workspace"):
        b200attn.kv4_joint_attention(q, q, v, pool, table, 64, workspace=torch.zeros(1 << 26, dtype=torch.uint8))
    with pytest.raises(b200attn.B200Error):
        b200attn.kv4_joint_attention(q, q, v, pool, table, 64,
                                     workspace=torch.zeros(64, dtype=torch.uint8, device=cuda))
    with pytest.raises(b200attn.B200Error):
        b200attn.kv4_joint_attention(q, q, v, pool, table, 65)
    with pytest.raises(ValueError, match="status"):
        b200attn.kv4_load(pool, table, None, 64, status=torch.zeros(1, dtype=torch.int64, device=cuda))


@pytest.mark.gpu
def test_an_empty_pool_reads_as_zeros(cuda):
    pool = torch.empty(0, 2, BLOCK, dtype=torch.uint8, device=cuda)
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    k, v = b200attn.kv4_load(pool, table, None, 64, status=status)
    assert not k.any() and not v.any() and status.item() == b200attn.KV4_STATUS_BAD_PAGE
    q = torch.randn(1, 2, 3, D, device=cuda).bfloat16()
    vo = torch.randn(1, 3, 2, D, device=cuda).bfloat16()
    none = torch.zeros(1, 0, dtype=torch.int32, device=cuda)     # no table at all: own keys only
    check(b200attn.kv4_joint_attention(q, q, vo, pool, none, 0), q, q, vo, k, v, [(0, 3)])
    status.zero_()
    b200attn.kv4_store(q, q, pool, none, status=status)
    assert status.item() == b200attn.KV4_STATUS_BAD_PAGE
