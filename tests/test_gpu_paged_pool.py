"""The page pool's operators on the GPU against plain implementations in 64 bits.

Tolerances are bounds, not fits.  With u = 2^-24 (fp32) and h the half unit of the output's type (u,
2^-11 for fp16, 2^-8 for bf16, plus fp16's smallest step):

* rotary: two products and a sum, each rounded: 3 u (|a c| + |b s|), plus h of the result;
* append: the rows and scales are the ones the paged store writes, bit for bit, so no tolerance;
* attention: out = sum w v / sum w.  A score is off by at most ds = (D u + e) sum |q k| scale plus its
  own rounding, 4 u |s|; a weight by the factor 1 + 2 ds; the sums over n tokens add n u, and splitting
  an operand for the tensor cores e: |out - exact| <= (2 ds + n u + e) sum w |v| + h |out|.
  e = 2^-19 for 32-bit queries, which are computed as 32-bit products; for 16-bit queries
  2^-17 in the scores and 2^-11 in the weights (weights of 11 bits).
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}
PAGE_TYPE = {"fp32": torch.float32, "fp16": torch.float16, "int8": torch.int8, "int4": torch.uint8}


@pytest.fixture(scope="module")
def skv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import shadow_infer_b200.shadowkv as m
    return m


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(gen, B, H, S, D, dtype, layout="bhsd"):
    """[B, H, S, D] rows: contiguous, a slice of a projection [B, S, 3H, D], or rows 16-byte vectors cannot read."""
    if layout == "bhsd":
        return torch.randn(B, H, S, D, generator=gen, device="cuda").to(dtype)
    if layout == "projection":
        return torch.randn(B, S, 3 * H, D, generator=gen, device="cuda").to(dtype).transpose(1, 2)[:, H:2 * H]
    flat = torch.randn(B * H * S * (D + 1) + 1, generator=gen, device="cuda").to(dtype)
    return flat[1:].view(B, H, S, D + 1)[..., :D]


# --------------------------------------------------------------------------------------------- rotary
def _turn64(x, cos, sin, interleaved, inverse=False):
    """x [B, H, S, D] in 64 bits by cos / sin [B, S, rot / 2]; the bound on a 32-bit result too."""
    x = x.double()
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos.double()[:, None], (-sin if inverse else sin).double()[:, None]
    y, size = x.clone(), x.abs() * 0
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a], size[..., b] = (x[..., a] * c).abs() + (x[..., b] * s).abs(), (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, 3 * U * size


@pytest.mark.parametrize("B,Hq,Hk,S,D,rot", [
    (1, 1, 1, 1, 2, 2), (2, 8, 2, 1, 128, 128), (3, 5, 3, 33, 64, 64), (1, 32, 8, 257, 128, 64), (2, 3, 1, 17, 80, 32),
    (2, 2, 2, 9, 33, 22), (1, 4, 4, 40, 256, 256), (2, 6, 3, 21, 96, 24), (1, 2, 1, 5, 40, 40), (1, 40, 0, 3, 128, 128),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(skv, B, Hq, Hk, S, D, rot, dtype, interleaved):
    gen = _gen(B * 1000 + S)
    cos, sin = skv.rotary_tables(rot, 4096)
    positions = torch.randint(0, 4096, (B, S), generator=gen, device="cuda")
    for layout, inverse in (("bhsd", False), ("projection", True), ("odd", False)):
        q = _rows(gen, B, Hq, S, D, dtype, layout)
        k = _rows(gen, B, Hk, S, D, dtype, layout) if Hk else None
        got = skv.apply_rotary(q, cos, sin, k=k, positions=positions, interleaved=interleaved, inverse=inverse)
        got = got if Hk else (got,)
        for x, y in zip((q, k), got):
            want, bound = _turn64(x, cos[positions], sin[positions], interleaved, inverse)
            assert y.dtype == dtype and y.shape == x.shape
            off = (y.double() - want).abs() - (bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype])
            assert off.max() <= 0, (layout, off.max())


def test_rotary_positions(skv):
    """Default positions are the rows' indexes; int32, broadcast and host positions mean the same as int64 ones."""
    cos, sin = skv.rotary_tables(64, 100)
    x = _rows(_gen(1), 2, 4, 7, 64, torch.float32)
    p = torch.arange(7, device="cuda")
    want = skv.apply_rotary(x, cos, sin, positions=p.expand(2, 7).contiguous())
    for at in (None, p, p.int(), p.cpu(), p[None].int()):
        assert torch.equal(skv.apply_rotary(x, cos, sin, positions=at), want)
    one = skv.apply_rotary(x, cos, sin, positions=torch.tensor([[3], [90]], device="cuda"))
    assert torch.equal(one[0, :, 3], want[0, :, 3])


def test_rotary_unknown_positions_are_nan(skv):
    cos, sin = skv.rotary_tables(32, 10)
    x = _rows(_gen(2), 1, 2, 4, 64, torch.float16)
    y = skv.apply_rotary(x, cos, sin, positions=torch.tensor([0, 9, 10, -1], device="cuda"))
    assert torch.isfinite(y[:, :, :2]).all() and torch.isnan(y[:, :, 2:, :32]).all()
    assert torch.equal(y[..., 32:], x[..., 32:])


def test_rotary_host_tensors_and_empty(skv):
    cos, sin = skv.rotary_tables(16, 10)
    x = torch.randn(1, 2, 4, 16)
    y = skv.apply_rotary(x, cos, sin)
    assert y.device.type == "cpu" and torch.equal(y, skv.apply_rotary(x.cuda(), cos, sin).cpu())
    assert skv.apply_rotary(x[:, :, :0], cos, sin).shape == (1, 2, 0, 16)
    assert skv.apply_rotary(x[:0].cuda(), cos, sin).shape == (0, 2, 4, 16)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(skv, interleaved):
    """The inverse turn of a gradient is the gradient: against the formula's (64-bit autograd) and against differences."""
    B, H, S, D, rot = 1, 2, 5, 48, 32
    cos, sin = skv.rotary_tables(rot, 64)
    pos = torch.tensor([[0, 63, 7, 7, 21]], device="cuda")
    gen = _gen(3)
    x, g = (_rows(gen, B, H, S, D, torch.float32) for _ in range(2))
    got = skv.apply_rotary(g, cos, sin, positions=pos, interleaved=interleaved, inverse=True)
    x64 = x.double().requires_grad_()
    (_turn64(x64, cos[pos], sin[pos], interleaved)[0] * g.double()).sum().backward()
    _, bound = _turn64(g, cos[pos], sin[pos], interleaved, True)
    assert ((got.double() - x64.grad).abs() <= bound + U * x64.grad.abs() + 1e-38).all()
    for at in ((0, 0, 1, 0), (0, 1, 4, 17), (0, 1, 0, 31), (0, 0, 2, 40)):
        e = torch.zeros_like(x)
        e[at] = 0.5
        f = [(skv.apply_rotary(x + s * e, cos, sin, positions=pos, interleaved=interleaved).double() * g.double()).sum()
             for s in (1, -1)]
        # f is linear: its difference is off by the roundings of x + e and of the turn, of the two rows' values
        assert abs(float(f[0] - f[1]) - float(got[at])) <= 16 * U * float((x[at[:3]].abs().sum() + 1) * g[at[:3]].abs().max()) * 2


def test_rotary_refusals(skv):
    cos, sin = skv.rotary_tables(64, 10)
    x = torch.zeros(1, 2, 3, 64, device="cuda")
    with pytest.raises(ValueError, match="4-D"):
        skv.apply_rotary(x[0], cos, sin)
    with pytest.raises(ValueError, match="q/k shapes"):
        skv.apply_rotary(x, cos, sin, k=x[:, :, :2])
    with pytest.raises(ValueError, match="rotate 64 values of a head of 32"):
        skv.apply_rotary(x[..., :32], cos, sin)
    with pytest.raises(ValueError, match="cos/sin shapes"):
        skv.apply_rotary(x, cos, sin[:5])
    with pytest.raises(ValueError, match="cos must be"):
        skv.apply_rotary(x, cos[0], sin)
    with pytest.raises(ValueError, match="positions must be int"):
        skv.apply_rotary(x, cos, sin, positions=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError, match="broadcast"):
        skv.apply_rotary(x, cos, sin, positions=torch.zeros(4, dtype=torch.int32, device="cuda"))


# --------------------------------------------------------------------------------------------- a pool
def _pool(kv, N, H, P, D, G=16):
    group = G if D % G == 0 else D
    row = (D + 1) // 2 if kv == "int4" else D
    pages = [torch.zeros(N, H, P, row, dtype=PAGE_TYPE[kv], device="cuda") for _ in range(2)]
    tail = {"int8": (1,), "int4": (D // group, 1)}.get(kv)
    scales = [None if tail is None else torch.ones(N, H, P, *tail, device="cuda") for _ in range(2)]
    return pages, scales


def _table(counts, P, seed, spare=2):
    """Shuffled pages for sequences of `counts` tokens; -1 past their end."""
    per = [-(-c // P) for c in counts]
    order = torch.randperm(sum(per) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = torch.full((len(counts), max(per) + 1), -1, dtype=torch.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda(), sum(per) + spare


def _values64(pages, scale, D):
    if pages.dtype == torch.uint8:
        x = (torch.stack((pages >> 4, pages & 15), -1).flatten(-2)[..., :D].double() - 8)
        return (x.unflatten(-1, (scale.shape[-2], -1)) * scale.double()).flatten(-2)
    return pages.double() if scale is None else pages.double() * scale.double()


def _dense64(pages, scale, table, b, n, D):
    """Tokens [H, n, D] of sequence b in 64 bits."""
    P = pages.shape[2]
    ids = table[b, :-(-n // P)].long()
    x = _values64(pages[ids], None if scale is None else scale[ids], D)
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


# --------------------------------------------------------------------------------------------- append
def _turn32(x, cos, sin, interleaved):
    """The turn in torch's 32-bit operations, each rounded: what the cache is given to quantise."""
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos[:, None], sin[:, None]
    y = x.float().clone()
    y[..., a], y[..., b] = x[..., a].float() * c - x[..., b].float() * s, x[..., b].float() * c + x[..., a].float() * s
    return y


APPEND = [  # B, Hq, Hk, S, D, rot, P, G, layout
    (2, 8, 2, 1, 128, 128, 32, 16, "projection"),
    (3, 3, 3, 37, 64, 64, 16, 16, "projection"),
    (1, 4, 1, 70, 128, 64, 7, 32, "bhsd"),
    (2, 2, 2, 19, 96, 24, 17, 16, "bhsd"),
    (2, 0, 3, 11, 33, 0, 5, 16, "bhsd"),       # odd head: padded int4 rows, one group
    (1, 2, 2, 9, 40, 40, 8, 16, "odd"),        # rows that vectors cannot read; the group falls back to 40
    (2, 4, 4, 13, 256, 256, 32, 64, "projection"),
    (2, 2, 1, 6, 80, 16, 64, 4, "projection"),
    (1, 0, 2, 5, 48, 0, 9, 24, "bhsd"),
]


@pytest.mark.parametrize("B,Hq,Hk,S,D,rot,P,G,layout", APPEND)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_writes_the_paged_stores_rows(skv, B, Hq, Hk, S, D, rot, P, G, layout, kv, dtype):
    gen = _gen(S * 100 + D)
    interleaved = S % 2 == 0
    first = [(5 * b + 3) % (2 * P) for b in range(B)]
    new = [S] + [max(0, S - 1 - 3 * b) for b in range(1, B)]
    table, N = _table([a + S for a in first], P, S)
    (kp, vp), (sk, sv) = _pool(kv, N, Hk, P, D, G)
    before = [None if t is None else t.clone() for t in (kp, vp, sk, sv)]
    k, v = (_rows(gen, B, Hk, S, D, dtype, layout) for _ in range(2))
    q = _rows(gen, B, Hq, S, D, dtype, layout) if Hq else None
    if S > 3:
        v[0, 0, 2] = 0     # a row of zeros has a scale of one
    cos, sin = skv.rotary_tables(rot, 4096) if rot else (None, None)
    lens, new_d = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (first, new))
    q_out = skv.paged_append(k, v, kp, vp, table, lens, sk, sv, new_d, q, cos, sin, interleaved=interleaved, check=True)
    at = lens.long()[:, None] + torch.arange(S, device="cuda")
    turned = _turn32(k, cos[at], sin[at], interleaved) if rot else k.float()
    if Hq:
        assert torch.equal(q_out, _turn32(q, cos[at], sin[at], interleaved).to(dtype))
    else:
        assert q_out is None
    # the same rows through the paged store, sequence by sequence
    for b in range(B):
        if new[b] == 0:
            continue
        store = skv.PagedKVStore(1, Hk, D, page_size=S, device="cuda", int4_group_size=G)
        store.append(turned[b:b + 1, :, :new[b]].contiguous(), v[b:b + 1, :, :new[b]].float().contiguous(), kv)
        page = store.pages[0]
        where = torch.arange(first[b], first[b] + new[b], device="cuda")
        ids, row = table[b].long()[where // P], where % P
        for mine, theirs in ((kp, page.k), (vp, page.v), (sk, page.scale_k), (sv, page.scale_v)):
            if mine is not None:
                assert torch.equal(mine[ids, :, row].transpose(0, 1), theirs[0])
                mine[ids, :, row] = 0
    # nothing else was written
    for b in range(B):
        where = torch.arange(first[b], first[b] + new[b], device="cuda")
        for t in before:
            if t is not None:
                t[table[b].long()[where // P], :, where % P] = 0
    for mine, was in zip((kp, vp, sk, sv), before):
        assert mine is None or torch.equal(mine, was)


@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("D,P,G", [(64, 16, 16), (33, 5, 16), (128, 32, 32), (40, 7, 8)])
def test_read_gives_the_values(skv, kv, D, P, G):
    H, counts = 3, [0, 1, P, 4 * P + 3]
    table, N = _table(counts, P, D)
    (kp, vp), (sk, sv) = _pool(kv, N, H, P, D, G)
    gen = _gen(D)
    k, v = (_rows(gen, 4, H, max(counts), D, torch.float32) for _ in range(2))
    lens = torch.tensor(counts, dtype=torch.int32, device="cuda")
    skv.paged_append(k, v, kp, vp, table, torch.zeros_like(lens), sk, sv, lens, check=True)
    n = max(counts) + 2
    start = torch.tensor([0, 0, 2, P + 1], dtype=torch.int32, device="cuda")
    for first in (None, start):
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            got = skv.paged_read(kp, vp, table, lens, n, sk, sv, first, D, dtype, check=True)
            for y, pages, scale in zip(got, (kp, vp), (sk, sv)):
                want = torch.zeros(4, H, n, D, dtype=torch.float64, device="cuda")
                for b, c in enumerate(counts):
                    a = 0 if first is None else int(first[b])
                    if c > a:
                        want[b, :, :c - a] = _dense64(pages, scale, table, b, c, D)[:, a:]
                # int8 and int4 products of 32 bits, rounded; then the output's type
                assert torch.equal(y, want.float().to(dtype))


# ------------------------------------------------------------------------------------------ attention
def _attention64(q, pages, scales, table, counts, new, causal):
    """In 64 bits, and the bound of the module's docstring."""
    B, Hq, Sq, D = q.shape
    H = pages[0].shape[1]
    out, bound = (torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device="cuda") for _ in range(2))
    wide = q.dtype == torch.float32
    es, ep = (2.0 ** -19, 2.0 ** -19) if wide else (2.0 ** -17, 2.0 ** -11)
    for b, n in enumerate(counts):
        if n == 0:
            continue
        k, v = (_dense64(p, s, table, b, n, D) for p, s in zip(pages, scales))
        qb = q[b].double().unflatten(0, (H, -1))
        s = torch.einsum("grsd,gtd->grst", qb, k) / math.sqrt(D)
        size = torch.einsum("grsd,gtd->grst", qb.abs(), k.abs()) / math.sqrt(D)
        i, t = torch.arange(Sq, device="cuda")[:, None], torch.arange(n, device="cuda")
        seen = (i < new[b]) & ((t <= n - new[b] + i) if causal else (t >= 0))
        s = s.masked_fill(~seen, -math.inf)
        w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        ds = ((D * U + es) * size + 4 * U * s.abs().nan_to_num(posinf=0.0)).masked_fill(~seen, 0).amax(-1, keepdim=True)
        out[b] = torch.einsum("grst,gtd->grsd", w, v).flatten(0, 1)
        bound[b] = ((2 * ds + n * U + ep) * torch.einsum("grst,gtd->grsd", w, v.abs())).flatten(0, 1)
    return out, bound + HALF[q.dtype] * (out.abs() + bound) + TINY[q.dtype]


def _filled(skv, kv, counts, H, P, D, G, seed, channels=1.0):
    """A pool that holds random tokens; every row and page that no sequence holds is NaN (or garbage with NaN scales)."""
    table, N = _table(counts, P, seed)
    (kp, vp), (sk, sv) = _pool(kv, N, H, P, D, G)
    gen = _gen(seed)
    for t in (kp, vp, sk, sv):
        if t is not None:
            t.fill_(math.nan) if t.dtype.is_floating_point else t.random_(0, 100, generator=gen)
    n = max(max(counts), 1)
    k, v = (_rows(gen, len(counts), H, n, D, torch.float32) for _ in range(2))
    k[..., :: max(1, D // 4)] *= channels
    lens = torch.tensor(counts, dtype=torch.int32, device="cuda")
    skv.paged_append(k, v, kp, vp, table, torch.zeros_like(lens), sk, sv, lens, check=True)
    return (kp, vp), (sk, sv), table, lens


ATTENTION = [  # counts, H, rep, Sq, D, P, G, causal
    ([1], 1, 1, 1, 64, 16, 16, False),
    ([512], 4, 1, 1, 128, 32, 16, False),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129], 2, 4, 1, 128, 32, 16, False),
    ([5000, 1, 0, 700], 2, 8, 1, 128, 32, 16, False),       # parts that are joined
    ([300, 40], 3, 3, 1, 64, 16, 32, False),
    ([257, 3, 96], 2, 2, 4, 128, 64, 16, True),
    ([200, 5], 1, 5, 7, 64, 32, 16, True),                  # 35 rows a key head; queries before the first token
    ([90, 33], 2, 1, 31, 128, 32, 128, False),
    ([130, 0, 77], 3, 3, 3, 80, 7, 16, True),               # page and head that divide nothing
    ([61, 20], 2, 2, 1, 33, 5, 16, False),                  # odd head
    ([100], 2, 6, 2, 256, 32, 16, True),
    ([75, 12], 1, 2, 1, 96, 24, 48, False),
    ([40], 1, 1, 1, 300, 8, 16, False),
    ([333, 1000], 1, 12, 1, 128, 128, 64, False),
    ([2100], 1, 16, 2, 64, 16, 16, False),                  # 32 rows a key head
    ([300, 17, 0, 1000], 2, 3, 1, 256, 32, 16, False),
    ([70, 260], 1, 8, 3, 256, 16, 64, True),
    ([129, 5], 3, 2, 1, 160, 32, 32, False),                # heads between the sizes that the kernels are cut to
    ([66, 190], 1, 4, 1, 192, 11, 16, False),
    ([95], 2, 1, 5, 112, 48, 16, True),
    ([50, 31], 2, 2, 1, 32, 16, 16, False),
    ([77], 1, 3, 1, 16, 64, 16, False),
    ([210, 33], 2, 2, 1, 80, 32, 16, False),                # int4 rows of 40 bytes
    ([64, 19], 1, 4, 2, 72, 5, 8, True),                    # int8 rows of 72
]


@pytest.mark.parametrize("counts,H,rep,Sq,D,P,G,causal", ATTENTION)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_attention(skv, counts, H, rep, Sq, D, P, G, causal, kv, dtype):
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, G, sum(counts) + D, channels=3.0)
    gen = _gen(7)
    for layout in ("bhsd", "projection", "odd"):
        q = _rows(gen, len(counts), H * rep, Sq, D, dtype, layout)
        got = skv.paged_attention(q, *pages, table, lens, *scales, causal=causal, check=True)
        assert got.dtype == dtype and got.shape == q.shape
        want, bound = _attention64(q, pages, scales, table, counts, [Sq] * len(counts), causal)
        off = (got.double() - want).abs() - bound
        assert off.max() <= 0, (layout, float(off.max()))
        assert torch.equal(got, skv.paged_attention(q, *pages, table, lens, *scales, causal=causal))   # the same bits


@pytest.mark.parametrize("kv", ["fp16", "int8", "int4"])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_ragged_prompt(skv, kv, causal):
    """Padding queries give zeros, and the causal limit counts a sequence's own new tokens."""
    counts, new, Sq = [40, 9, 64, 3], [5, 9, 1, 0], 9
    pages, scales, table, lens = _filled(skv, kv, counts, 2, 16, 128, 16, 5)
    q = _rows(_gen(9), 4, 8, Sq, 128, torch.float16)
    got = skv.paged_attention(q, *pages, table, lens, *scales, causal=causal,
                              new_lengths=torch.tensor(new, dtype=torch.int32, device="cuda"))
    want, bound = _attention64(q, pages, scales, table, counts, new, causal)
    assert ((got.double() - want).abs() <= bound).all()
    for b, n in enumerate(new):
        assert (got[b, :, n:] == 0).all()


MANY_ROWS = [  # counts, H, rep, Sq, D, P, new, causal: 48 query rows a key head and more, from 1 to some hundred units of 128
    ([300, 0, 1, 127, 128, 129] * 5, 4, 4, 16, 128, 32, None, False),
    ([300, 0, 1, 127, 128, 129] * 5, 4, 4, 16, 128, 32, None, True),
    ([9000, 16, 2500], 2, 4, 31, 128, 16, None, True),       # parts that are joined
    ([3000, 20] * 10, 8, 2, 33, 128, 16, None, True),
    ([5000], 1, 3, 33, 64, 64, None, False),
    ([700, 130, 64], 19, 2, 130, 64, 7, None, True),         # blocks of one head's tokens, the last of two
    ([700, 130, 64], 19, 2, 130, 64, 7, [130, 60, 0], True), # and padding of a ragged prompt
    ([1000, 400], 15, 1, 400, 128, 32, [400, 257], True),
    ([515], 24, 1, 515, 128, 128, None, True),               # a whole prompt
    ([515], 1, 1, 515, 128, 128, None, True),
    ([515, 200], 14, 2, 200, 96, 24, None, False),
    ([140], 38, 3, 128, 80, 16, None, True),
    ([333, 90] * 16, 4, 8, 9, 112, 11, [9, 4] * 16, True),
    ([260, 33] * 16, 4, 64, 1, 32, 16, None, False),         # many heads, one token
    ([77, 12], 1, 50, 1, 16, 64, None, False),
    ([300, 77, 0] * 6, 8, 2, 33, 256, 32, None, True),       # heads of more than 128 values
    ([900, 140], 3, 2, 140, 160, 17, None, True),
    ([2500], 1, 8, 31, 192, 16, None, False),
]


@pytest.mark.parametrize("counts,H,rep,Sq,D,P,new,causal", MANY_ROWS)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_attention_of_many_rows(skv, counts, H, rep, Sq, D, P, new, causal, kv, dtype):
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, sum(counts) + D, channels=3.0)
    gen = _gen(17)
    fresh = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    for layout in ("bhsd", "projection", "odd"):
        q = _rows(gen, len(counts), H * rep, Sq, D, dtype, layout)
        got = skv.paged_attention(q, *pages, table, lens, *scales, causal=causal, new_lengths=fresh, check=True)
        want, bound = _attention64(q, pages, scales, table, counts, new or [Sq] * len(counts), causal)
        off = (got.double() - want).abs() - bound
        assert off.max() <= 0, (layout, float(off.max()))
        assert torch.equal(got, skv.paged_attention(q, *pages, table, lens, *scales, causal=causal, new_lengths=fresh))


@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_attention_of_many_rows_extremes(skv, kv):
    """A NaN row, rows of very different size and a page outside the pool, for a prompt."""
    counts, H, D, P, Sq = [600, 300], 15, 128, 32, 140
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, 8)
    q = _rows(_gen(5), 2, 2 * H, Sq, D, torch.float16)
    q *= 10.0 ** torch.linspace(-4, 2, Sq, device="cuda").half()[:, None]
    clean = skv.paged_attention(q, *pages, table, lens, *scales, causal=True)
    want, bound = _attention64(q, pages, scales, table, counts, [Sq] * 2, True)
    assert ((clean.double() - want).abs() <= bound).all()
    p = q.clone()
    p[0, 1, 3, 5] = math.nan
    got = skv.paged_attention(p, *pages, table, lens, *scales, causal=True)
    assert torch.isnan(got[0, 1, 3]).all()
    got[0, 1, 3] = clean[0, 1, 3]
    assert torch.equal(got, clean)
    bad = table.clone()
    bad[0, 3] = -5
    with pytest.raises(ValueError, match="outside"):
        skv.paged_attention(q, *pages, bad, lens, *scales, causal=True, check=True)
    # the tokens of that page count as absent
    got = skv.paged_attention(q, *pages, bad, lens, *scales)
    keep = torch.ones(600, dtype=torch.bool, device="cuda")
    keep[3 * P:4 * P] = False
    k, v = (_dense64(x, y, table, 0, 600, D)[:, keep] for x, y in zip(pages, scales))
    w = torch.softmax(torch.einsum("grsd,gtd->grst", q[0].double().unflatten(0, (H, -1)), k) / math.sqrt(D), -1)
    exact = torch.einsum("grst,gtd->grsd", w, v).flatten(0, 1)
    _, bound = _attention64(q, pages, scales, table, counts, [Sq] * 2, False)
    # (the bound of all tokens' weights, at least half of which are these)
    assert ((got[0].double() - exact).abs() <= 2 * bound[0] + 2.0 ** -11 * exact.abs()).float().mean() > 0.999


@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_attention_of_extreme_values(skv, kv, dtype):
    """Rows of very different size: a token of tiny values that takes nearly all the weight, large values next to
    small ones, and scores far apart."""
    counts, H, D, P = [150, 40], 1, 128, 32
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, 31)
    gen = _gen(11)
    k, v = (_rows(gen, 2, H, 150, D, torch.float32) for _ in range(2))
    size = 10.0 ** torch.linspace(-3, 3, 150, device="cuda")
    v *= size[torch.randperm(150, generator=torch.Generator().manual_seed(1)).cuda()][:, None]
    q = _rows(gen, 2, 4, 1, D, dtype) * 4
    k[:, :, 17] = 3.0 * q[:, :1, 0].float()       # this token wins for head 0
    v[:, :, 17] *= 1e-3
    skv.paged_append(k, v, *pages, table, torch.zeros_like(lens), *scales, lens, check=True)
    got = skv.paged_attention(q, *pages, table, lens, *scales, check=True)
    want, bound = _attention64(q, pages, scales, table, counts, [1, 1], False)
    assert ((got.double() - want).abs() <= bound).all()


def test_attention_large_scores(skv):
    """Scores of thousands, whose exponentials only the running maximum keeps in range."""
    pages, scales, table, lens = _filled(skv, "fp16", [700], 2, 32, 128, 16, 3)
    q = _rows(_gen(4), 1, 4, 1, 128, torch.float32)
    for scale in (100.0, 0.0, -1.0):
        got = skv.paged_attention(q, *pages, table, lens, scale=scale)
        want, bound = _attention64(q * (scale * math.sqrt(128)), pages, scales, table, [700], [1], False)
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_attention_nan_and_infinity_reach_only_their_rows(skv, kv):
    """A NaN query row gives NaN in its row alone; an infinite score likewise, as the formula says."""
    pages, scales, table, lens = _filled(skv, kv, [100, 50], 2, 32, 128, 16, 8)
    q = _rows(_gen(5), 2, 4, 1, 128, torch.float16)
    clean = skv.paged_attention(q, *pages, table, lens, *scales)
    q[0, 1, 0, 5] = math.nan
    got = skv.paged_attention(q, *pages, table, lens, *scales)
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = clean[0, 1]
    assert torch.equal(got, clean)


def test_attention_beyond_32_bit_offsets(skv):
    """Pages whose byte and element offsets do not fit 32 bits."""
    H, P, D = 8, 32, 128
    N = 2 ** 32 // (H * P * D) + 40               # more than 2^32 values in each of K and V
    kp, vp = (torch.empty(N, H, P, D, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[N - 1, 3, N - 7, N // 2], [N - 2, N - 3, 0, 1]], dtype=torch.int32, device="cuda")
    counts = [P * 4 - 5, P * 2 + 1]
    lens = torch.tensor(counts, dtype=torch.int32, device="cuda")
    gen = _gen(6)
    k, v = (_rows(gen, 2, H, P * 4, D, torch.float16) for _ in range(2))
    skv.paged_append(k, v, kp, vp, table, torch.zeros_like(lens), new_lengths=lens, check=True)
    q = _rows(gen, 2, 2 * H, 1, D, torch.float16)
    got = skv.paged_attention(q, kp, vp, table, lens, check=True)
    want, bound = _attention64(q, (kp, vp), (None, None), table, counts, [1, 1], False)
    assert ((got.double() - want).abs() <= bound).all()
    rk, _ = skv.paged_read(kp, vp, table, lens, P * 4, dtype=torch.float16)
    assert torch.equal(rk[0, :, :counts[0]], k[0, :, :counts[0]])


def test_attention_over_another_stream_and_a_graph(skv):
    """The caller's stream is used; a captured step replays with the lengths and tables of the moment."""
    pages, scales, table, lens = _filled(skv, "int8", [200, 300], 2, 32, 128, 16, 21)
    q = _rows(_gen(2), 2, 8, 1, 128, torch.bfloat16)
    want = skv.paged_attention(q, *pages, table, lens, *scales)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = skv.paged_attention(q, *pages, table, lens, *scales)
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = skv.paged_attention(q, *pages, table, lens, *scales)
    for counts in ([200, 300], [1, 0], [64, 299]):
        lens.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, skv.paged_attention(q, *pages, table, lens, *scales))


def test_pages_outside_the_pool(skv):
    """Page numbers that name nothing are not followed; check=True says so."""
    pages, scales, table, lens = _filled(skv, "int8", [100], 2, 32, 128, 16, 2)
    q = _rows(_gen(3), 1, 2, 1, 128, torch.float16)
    bad = table.clone()
    bad[0, 1] = pages[0].shape[0]
    bad[0, 2] = -5
    with pytest.raises(ValueError, match="outside the pool"):
        skv.paged_attention(q, *pages, bad, lens, *scales, check=True)
    got = skv.paged_attention(q, *pages, bad, lens, *scales)
    k, v = (torch.cat([_dense64(p, s, table, 0, 100, 128)[:, a:b] for a, b in ((0, 32), (96, 100))], 1)
            for p, s in zip(pages, scales))
    w = torch.softmax(torch.einsum("hd,htd->ht", q[0, :, 0].double(), k) / math.sqrt(128), -1)
    want = torch.einsum("ht,htd->hd", w, v)
    assert float((got[0, :, 0].double() - want).abs().max()) < 1e-2 * float(want.abs().max())
    with pytest.raises(ValueError, match="outside the pool"):
        skv.paged_read(*pages, bad, lens, 100, *scales, check=True)
    assert (skv.paged_read(*pages, bad, lens, 100, *scales)[0][:, :, 32:96] == 0).all()
    rows = torch.ones(1, 2, 100, 128, device="cuda")
    with pytest.raises(ValueError, match="outside the pool"):
        skv.paged_append(rows, rows, *pages, bad, torch.zeros_like(lens), *scales, check=True)
    with pytest.raises(ValueError, match="outside the pool"):   # behind the table's last page
        skv.paged_append(rows, rows, *pages, table, lens, *scales, check=True)
    with pytest.raises(ValueError, match="outside the pool"):   # more tokens than the table holds
        skv.paged_attention(q, *pages, table[:, :2].contiguous(), lens, *scales, check=True)


def test_pool_refusals(skv):
    pages, scales, table, lens = _filled(skv, "int4", [10], 2, 16, 64, 16, 2)
    q = torch.zeros(1, 4, 1, 64, device="cuda")
    k = torch.zeros(1, 2, 3, 64, device="cuda")
    ok = (*pages, table, lens)
    for match, call in [
        ("4-D", lambda: skv.paged_attention(q[0], *ok, *scales)),
        ("need scale_k", lambda: skv.paged_attention(q, *ok)),
        ("3 query heads do not share 2", lambda: skv.paged_attention(q[:, :3], *ok, *scales)),
        ("do not hold a head_dim of 32", lambda: skv.paged_attention(q[..., :32], *ok, *scales)),
        ("block_table must be", lambda: skv.paged_attention(q.expand(2, 4, 1, 64), *ok, *scales)),
        ("lengths must have shape", lambda: skv.paged_attention(q, *pages, table, lens.expand(2), *scales)),
        ("lengths must be int32", lambda: skv.paged_attention(q, *pages, table, lens.float(), *scales)),
        ("must be alike", lambda: skv.paged_attention(q, pages[0], pages[1][:1], table, lens, *scales)),
        ("must be alike", lambda: skv.paged_attention(q, pages[0], pages[1].float(), table, lens, *scales)),
        ("Unsupported page precision", lambda: skv.paged_attention(q, *(p.double() for p in pages), table, lens)),
        ("must be CUDA", lambda: skv.paged_attention(q, *(p.cpu() for p in pages), table, lens, *scales)),
        ("contiguous", lambda: skv.paged_attention(q, *(p.transpose(1, 2) for p in pages), table, lens, *scales)),
        ("scales must be", lambda: skv.paged_attention(q, *ok, scales[0].half(), scales[1])),
        ("scales must be", lambda: skv.paged_attention(q, *ok, scales[0][..., 0], scales[1])),
        ("groups do not divide", lambda: skv.paged_attention(q, *ok, scales[0], scales[1][..., :2, :].contiguous())),
        ("k/v shapes disagree", lambda: skv.paged_append(k, k[:, :1], *ok, *scales)),
        ("k/v must be 4-D", lambda: skv.paged_append(k[0], k[0], *ok, *scales)),
        ("1 heads, the pool has 2", lambda: skv.paged_append(k[:, :1], k[:, :1], *ok, *scales)),
        ("given together", lambda: skv.paged_append(k, k, *ok, *scales, cos=q[0, 0])),
        ("nothing to be rotated by", lambda: skv.paged_append(k, k, *ok, *scales, q=k)),
        ("tokens must be", lambda: skv.paged_read(*ok, -1, *scales)),
        ("dtype must be", lambda: skv.paged_read(*ok, 1, *scales, dtype=torch.int8)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    big = torch.zeros(1, 1, 1, 520, device="cuda")
    wide = torch.zeros(1, 1, 16, 520, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim 520 above"):
        skv.paged_attention(big, wide, wide, table, lens)
    # nothing to do
    assert skv.paged_attention(q[:0], *pages, table[:0], lens[:0], *scales).shape == (0, 4, 1, 64)
    assert skv.paged_attention(q[:, :, :0], *ok, *scales).shape == (1, 4, 0, 64)
    assert skv.paged_append(k[:, :, :0], k[:, :, :0], *ok, *scales) is None
    assert skv.paged_read(*ok, 0, *scales)[0].shape == (1, 2, 0, 64)


# ------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
def test_pool_serves_ragged_sequences(skv, kv):
    """A prompt, then single tokens, a sequence that ends and one that takes its pages: each step's attention against
    the formula over what the pool holds, and every row held where the sequence's own tokens put it."""
    B, H, rep, D, P = 3, 2, 2, 64, 8
    pool = skv.PagedKVPool(24, B, H, D, max_tokens=96, page_size=P, precision=kv)
    cos, sin = skv.rotary_tables(D, 128)
    gen = _gen(17)
    counts = [0] * B
    for step, new in enumerate([[13, 1, 30], None, None, [1, 0, 1], "release", [20, 3, 1], None]):
        if new == "release":
            assert pool.release(2) == -(-counts[2] // P)
            counts[2] = 0
            continue
        S = 1 if new is None else max(new)
        x = torch.randn(B, S, H * (rep + 2), D, generator=gen, device="cuda").transpose(1, 2)
        q, k, v = x[:, :H * rep], x[:, H * rep:-H], x[:, -H:]
        qr = pool.append(k, v, q=q, cos=cos, sin=sin, new_lengths=new)
        had, new = counts, [S] * B if new is None else new
        counts = [c + n for c, n in zip(counts, new)]
        assert pool.token_counts == counts and pool.lengths.tolist() == counts
        assert pool.free_pages == 24 - sum(-(-c // P) for c in counts)
        fresh = torch.tensor(new, dtype=torch.int32, device="cuda")
        got = pool.attention(qr, causal=True, new_lengths=fresh)
        want, bound = _attention64(qr, (pool.k_pages, pool.v_pages), (pool.scale_k, pool.scale_v), pool.block_table,
                                   counts, new, True)
        assert ((got.double() - want).abs() <= bound).all(), step
        k_held, v_held = pool.read()
        for b in range(B):
            at = torch.arange(had[b], counts[b], device="cuda")
            kt = _turn32(k[b:b + 1], cos[had[b]:had[b] + S][None], sin[had[b]:had[b] + S][None], False)
            ref = skv.PagedKVStore(1, H, D, page_size=64, device="cuda")
            if new[b]:
                ref.append(kt[:, :, :new[b]].contiguous(), v[b:b + 1, :, :new[b]].contiguous(), kv)
                kd, vd = ref.gather()
                assert torch.equal(k_held[b, :, at], kd[0]) and torch.equal(v_held[b, :, at], vd[0])
    with pytest.raises(RuntimeError, match="pages wanted"):
        pool.append(torch.zeros(B, H, 55, D, device="cuda"), torch.zeros(B, H, 55, D, device="cuda"))
    with pytest.raises(RuntimeError, match="does not fit"):
        pool.append(torch.zeros(B, H, 96, D, device="cuda"), torch.zeros(B, H, 96, D, device="cuda"))
    with pytest.raises(ValueError, match="new_lengths must be"):
        pool.append(x[:, :H], x[:, :H], new_lengths=[0, 0, x.shape[2] + 1])
    assert pool.token_counts == counts


def test_block_forward_over_the_pool(skv):
    """A transformer block fed token by token over a pool gives what it gives over the whole prompt at once, and what
    torch computes in 32 bits without a cache (the cache is fp32)."""
    torch.manual_seed(3)
    nh, nkv, hd, S, B = 4, 2, 32, 11, 2

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            hidden = nh * hd
            self.hidden_dim, self.num_heads, self.num_kv_heads, self.head_dim = hidden, nh, nkv, hd
            self.ln1, self.ln2 = torch.nn.LayerNorm(hidden), torch.nn.LayerNorm(hidden)
            self.q_proj, self.o_proj = torch.nn.Linear(hidden, hidden), torch.nn.Linear(hidden, hidden)
            self.k_proj, self.v_proj = (torch.nn.Linear(hidden, nkv * hd) for _ in range(2))
            self.up_proj, self.down_proj = torch.nn.Linear(hidden, 2 * hidden), torch.nn.Linear(2 * hidden, hidden)

    block = Block().cuda()
    x = torch.randn(B, S, nh * hd, device="cuda")
    cos, sin = skv.rotary_tables(hd, 64)

    def pool():
        return skv.PagedKVPool(8, B, nkv, hd, max_tokens=32, page_size=8, precision="fp32")

    with torch.no_grad():
        whole = skv.paged_block_forward(block, x, pool(), cos, sin, causal=True)
        p = pool()
        steps = [skv.paged_block_forward(block, x[:, i:i + 1], p, cos, sin) for i in range(S)]
        n = block.ln1(x)
        heads = lambda y: y.view(B, S, -1, hd).transpose(1, 2)  # noqa: E731
        at = torch.arange(S, device="cuda").expand(B, S)
        q, k = (_turn32(heads(f(n)), cos[at], sin[at], False) for f in (block.q_proj, block.k_proj))
        k, v = (y.repeat_interleave(nh // nkv, 1) for y in (k, heads(block.v_proj(n))))
        s = (q @ k.transpose(2, 3) / math.sqrt(hd)).masked_fill(torch.ones(S, S, device="cuda").triu(1).bool(), -math.inf)
        h = x + block.o_proj((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, S, -1))
        want = h + block.down_proj(torch.nn.functional.gelu(block.up_proj(block.ln2(h))))
    # hidden states of size ~1 through fp32 products of up to 256 terms on both sides
    assert float((whole - want).abs().max()) < 512 * U * float(want.abs().max())
    assert float((torch.cat(steps, 1) - want).abs().max()) < 512 * U * float(want.abs().max())
