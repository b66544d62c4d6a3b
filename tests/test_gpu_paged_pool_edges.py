"""The page pool's operators where they could go wrong: the largest and oddest calls, values that are not finite, and what
a call may and may not write.  Bounds are those of test_gpu_paged_pool, whose helpers these tests use."""

import math

import pytest
import torch
from test_gpu_paged_pool import (  # noqa: F401  (skv is a fixture)
    HALF, TINY, U, _attention64, _dense64, _filled, _gen, _pool, _rows, _table, _turn32, _turn64, skv)

pytestmark = pytest.mark.gpu


def _one64(q, pages, scales, table, b, n, D):
    """Queries q [H_q, D] of sequence b over its first n tokens: in 64 bits, and the bound of test_gpu_paged_pool."""
    wide = q.dtype == torch.float32
    es, ep = (2.0 ** -19, 2.0 ** -19) if wide else (2.0 ** -17, 2.0 ** -11)
    k, v = (_dense64(p, s, table, b, n, D) for p, s in zip(pages, scales))
    qb = q.double().unflatten(0, (k.shape[0], -1))
    s, size = (torch.einsum("grd,gtd->grt", x, y) / math.sqrt(D) for x, y in ((qb, k), (qb.abs(), k.abs())))
    w = torch.softmax(s, -1)
    out, spread = (torch.einsum("grt,gtd->grd", w, x).flatten(0, 1) for x in (v, v.abs()))
    ds = ((D * U + es) * size + 4 * U * s.abs()).amax(-1).flatten()[:, None]
    bound = (2 * ds + n * U + ep) * spread
    return out, bound + HALF[q.dtype] * (out.abs() + bound) + TINY[q.dtype]


def _widened(table, width):
    """The same table with room for `width` pages."""
    wide = torch.full((table.shape[0], width), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return wide


# ------------------------------------------------------------------------------------- how large a call may be
WIDE = [(1, 16384, 131072), (8, 8192, 32768), (32, 2048, 32768), (64, 1024, 32768), (64, 4096, 8192)]   # sequences, tokens, room


@pytest.mark.parametrize("B,S,room,kv,dtype", [(*w, *t) for w in WIDE for t in (("fp16", torch.bfloat16), ("int8", torch.float16))] +
                         [(*WIDE[0], "fp16", torch.float32)])
def test_prompts_behind_wide_tables(skv, B, S, room, kv, dtype):
    """Whole prompts of 32 query heads, in pools whose tables have room for much longer sequences."""
    H, rep, D, P = 4, 8, 64, 32
    counts = [S - 7 * b for b in range(B)]
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, 3)
    q = torch.randn(B, S, H * rep, D, generator=_gen(4), device="cuda", dtype=dtype).transpose(1, 2)
    got = skv.paged_attention(q, *pages, _widened(table, room // P), lens, *scales, causal=True, new_lengths=lens, check=True)
    for b in {0, B // 2, B - 1}:
        for i in (0, 130, counts[b] // 2, counts[b] - 1):
            want, bound = _one64(q[b, :, i], pages, scales, table, b, i + 1, D)
            assert ((got[b, :, i].double() - want).abs() <= bound).all(), (b, i)
        assert (got[b, :, counts[b]:] == 0).all()


@pytest.mark.parametrize("D,rep,Sq,dtype", [(64, 2, 64, torch.float32), (300, 2, 24, torch.float16), (64, 4, 256, torch.bfloat16)])
def test_calls_in_parts_of_their_sequences(skv, D, rep, Sq, dtype):
    """Tables so wide that one launch's tile numbers could not count all sequences."""
    H, P, B = 2, 512, 40
    counts = [Sq + 11 * (b % 5) for b in range(B)]
    pages, scales, table, lens = _filled(skv, "fp16", counts, H, P, D, 16, 5)
    q = _rows(_gen(6), B, H * rep, Sq, D, dtype)
    wide = _widened(table, 2 ** 19 if D == 64 else 2 ** 18)
    got = skv.paged_attention(q, *pages, wide, lens, causal=True, check=True)
    assert torch.equal(got, skv.paged_attention(q, *pages, wide, lens, causal=True, new_lengths=torch.full_like(lens, Sq)))
    want, bound = _attention64(q, pages, scales, table, counts, [Sq] * B, True)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("B,S,H,D,kv,dtype", [
    (64, 1200, 2, 32, "fp16", torch.bfloat16), (40, 2000, 4, 32, "int8", torch.float16), (64, 1300, 1, 16, "int4", torch.float32),
    (160, 1000, 1, 16, "fp32", torch.float16),
])
def test_append_of_many_small_rows(skv, B, S, H, D, kv, dtype):
    """So many tokens of so few values that a block could take more than 64 of them."""
    P = 100
    table, N = _table([S] * B, P, 1)
    (kp, vp), (sk, sv) = _pool(kv, N, H, P, D)
    gen = _gen(3)
    k, v = (_rows(gen, B, H, S, D, dtype) for _ in range(2))
    cos, sin = skv.rotary_tables(D, S)
    skv.paged_append(k, v, kp, vp, table, torch.zeros(B, dtype=torch.int32, device="cuda"), sk, sv, cos=cos, sin=sin, check=True)
    store = skv.PagedKVStore(B, H, D, page_size=S, device="cuda")
    store.append(_turn32(k, cos[None], sin[None], False).contiguous(), v.float().contiguous(), kv)
    page, ids = store.pages[0], table[:, :S // P].long()
    for mine, theirs in ((kp, page.k), (vp, page.v), (sk, page.scale_k), (sv, page.scale_v)):
        if mine is not None:
            assert torch.equal(mine[ids].transpose(1, 2).flatten(2, 3), theirs)


# -------------------------------------------------------------------------------------- what an append leaves
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("D,interleaved,layout", [(64, False, "bhsd"), (64, True, "bhsd"), (40, False, "bhsd"), (64, False, "odd")])
def test_append_of_unknown_positions_writes_nothing(skv, kv, D, interleaved, layout):
    """A token whose position the tables do not hold: neither its key nor its value, nor their scales; the others' are."""
    B, H, S, P = 2, 3, 5, 4
    table, N = _table([S] * B, P, 1)
    pages, scales = _pool(kv, N, H, P, D, 8)
    gen = _gen(2)
    for t in (*pages, *scales):
        if t is not None:
            t.copy_(torch.randint(1, 100, t.shape, generator=gen, device="cuda"))
    before = [None if t is None else t.clone() for t in (*pages, *scales)]
    k, v = (_rows(gen, B, H, S, D, torch.float32, layout) for _ in range(2))
    cos, sin = skv.rotary_tables(16, 10)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    good = [(0, 0), (0, 2), (1, 1), (1, 4)]
    for dtype in (torch.int32, torch.int64):
        at = torch.tensor([[0, 10, 9, -1, 1000], [-7, 3, 10, 11, 9]], dtype=dtype, device="cuda")
        now = [None if t is None else t.clone() for t in before]
        args = (k, v, *now[:2], table, zero, *now[2:], None, None, cos, sin)
        skv.paged_append(*args, positions=at, interleaved=interleaved)
        want = [None if t is None else t.clone() for t in before]
        inside = at.clamp(0, 9)
        skv.paged_append(k, v, *want[:2], table, zero, *want[2:], None, None, cos, sin, positions=inside, interleaved=interleaved)
        for mine, same, old in zip(now, want, before):
            if mine is None:
                continue
            for b in range(B):
                for s in range(S):
                    where = (int(table[b, s // P]), slice(None), s % P)
                    assert torch.equal(mine[where], (same if (b, s) in good else old)[where]), (b, s)
        with pytest.raises(ValueError, match="position"):
            skv.paged_append(*args, positions=at, interleaved=interleaved, check=True)


def test_pool_refuses_positions_behind_the_tables(skv):
    """The pool's lengths never pass what was written: positions that the tables do not hold are refused."""
    pool = skv.PagedKVPool(8, 2, 2, 32, max_tokens=64, page_size=16, precision="fp16")
    cos, sin = skv.rotary_tables(32, 20)
    x = torch.ones(2, 2, 15, 32, device="cuda")
    pool.append(x, x, cos=cos, sin=sin, new_lengths=[15, 2])
    held = [t.clone() for t in (pool.k_pages, pool.v_pages, pool.block_table, pool.lengths)]
    free = pool.free_pages
    with pytest.raises(ValueError, match="position"):
        pool.append(x, x, cos=cos, sin=sin, new_lengths=[6, 1])
    with pytest.raises(ValueError, match="position"):
        pool.append(x, x, cos=cos, sin=sin, new_lengths=[1, 6], positions=torch.full((2, 15), 20, device="cuda"), check=True)
    assert pool.token_counts == [15, 2] and pool.free_pages == free
    for t, old in zip((pool.k_pages, pool.v_pages, pool.block_table, pool.lengths), held):
        assert torch.equal(t, old)
    pool.append(x, x, cos=cos, sin=sin, new_lengths=[5, 1])                                  # up to the last position
    pool.append(x, x, cos=cos, sin=sin, new_lengths=[1, 6], positions=torch.full((2, 15), 19, device="cuda"), check=True)
    pool.append(x, x, new_lengths=[1, 1])                                                    # no rotation, no limit
    assert pool.token_counts == [22, 10] == pool.lengths.tolist()


def test_tables_of_64_bit_numbers(skv):
    """int64 tables and lengths mean what int32 ones do, and numbers beyond 32 bits name nothing."""
    pages, scales, table, lens = _filled(skv, "fp16", [100, 40], 2, 32, 64, 16, 2)
    q = _rows(_gen(3), 2, 4, 1, 64, torch.float16)
    want = skv.paged_attention(q, *pages, table, lens)
    for where in ("cuda", "cpu"):
        assert torch.equal(skv.paged_attention(q, *pages, table.long().to(where), lens.long().to(where)), want)
    far = table.long()
    far[0, 1] += 2 ** 32
    far[1, 0] -= 2 ** 33
    with pytest.raises(ValueError, match="outside the pool"):
        skv.paged_attention(q, *pages, far, lens, check=True)
    k, _ = skv.paged_read(*pages, far, lens, 100)
    assert (k[0, :, 32:64] == 0).all() and (k[1, :, :32] == 0).all() and (k[0, :, :32] != 0).any()
    rows = torch.ones(2, 2, 1, 64, device="cuda")
    held = [t.clone() for t in pages]
    with pytest.raises(ValueError, match="outside the pool"):
        skv.paged_append(rows, rows, *pages, table, torch.tensor([2 ** 32, -2 ** 32], device="cuda"), check=True)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(pages, held))


@pytest.mark.parametrize("kt,vt,qt", [(torch.bfloat16, torch.float32, torch.float16), (torch.float16, torch.bfloat16, torch.bfloat16),
                                      (torch.float32, torch.float16, torch.float64)])
def test_rows_of_different_types(skv, kt, vt, qt):
    """Keys, values and queries of different types: each row as it is, not rounded to another's type."""
    B, H, S, D = 2, 2, 9, 64
    gen = _gen(6)
    k, v, q = (torch.randn(B, H, S, D, generator=gen, device="cuda").to(t) for t in (kt, vt, qt))
    cos, sin = skv.rotary_tables(D, 64)
    at = torch.arange(S, device="cuda").expand(B, S)
    for kv in ("fp32", "int8"):
        (kp, vp), (sk, sv) = _pool(kv, 2, H, 16, D)
        table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
        out = skv.paged_append(k, v, kp, vp, table, torch.zeros(B, dtype=torch.int32, device="cuda"), sk, sv, q=q, cos=cos, sin=sin)
        assert out.dtype == qt and torch.equal(out, _turn32(q, cos[at], sin[at], False).to(qt))
        store = skv.PagedKVStore(B, H, D, page_size=S, device="cuda")
        store.append(_turn32(k, cos[at], sin[at], False), v.float(), kv)
        page = store.pages[0]
        for mine, theirs in ((kp, page.k), (vp, page.v), (sk, page.scale_k), (sv, page.scale_v)):
            assert mine is None or torch.equal(mine[:, :, :S], theirs)
        got = skv.paged_attention(q, kp, vp, table, torch.full((B,), S, dtype=torch.int32, device="cuda"), sk, sv)
        assert got.dtype == qt
    for x, y in ((q, k), (k, v)):
        turned = skv.apply_rotary(x, cos, sin, k=y)
        for a, b in zip((x, y), turned):
            assert b.dtype == a.dtype and torch.equal(b, skv.apply_rotary(a, cos, sin))


@pytest.mark.parametrize("Sq,D", [(1, 64), (60, 64), (1, 33)])
def test_negative_lengths_hold_nothing_and_are_named(skv, Sq, D):
    pages, scales, table, lens = _filled(skv, "fp16", [100, 40], 2, 32, D, 16, 2)
    q = _rows(_gen(3), 2, 4, Sq, D, torch.float16)
    lens[1] = -1
    got = skv.paged_attention(q, *pages, table, lens)
    assert (got[1] == 0).all() and (got[0] != 0).any() and (skv.paged_read(*pages, table, lens, 40)[0][1] == 0).all()
    with pytest.raises(ValueError, match="length"):
        skv.paged_attention(q, *pages, table, lens, check=True)
    with pytest.raises(ValueError, match="length"):
        skv.paged_read(*pages, table, lens, 40, head_dim=D, check=True)


def _alike(a, b, but=None):
    """Equal, NaN where the other is, apart from `but`."""
    same = (a == b) | (a.isnan() & b.isnan()) if a.dtype.is_floating_point else a == b
    return bool((same if but is None else same | but).all())


PROMPTS = [  # B, Hq, Hk, S, D, rot, P, G: enough tokens that a thread takes several rows, and a block several tokens
    (2, 8, 5, 400, 128, 128, 32, 16), (3, 0, 7, 900, 64, 32, 16, 16), (2, 6, 9, 500, 96, 96, 17, 8), (1, 4, 3, 2000, 256, 128, 64, 32),
    (8, 4, 1, 1200, 128, 64, 32, 16), (4, 2, 2, 4000, 64, 64, 128, 32), (2, 5, 6, 600, 80, 0, 32, 16),
]


@pytest.mark.parametrize("B,Hq,Hk,S,D,rot,P,G", PROMPTS)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_prompts(skv, B, Hq, Hk, S, D, rot, P, G, kv, dtype, interleaved):
    """Ragged prompts: the paged store's rows, those with infinite, NaN, very large and very small values too."""
    gen = _gen(S)
    first, new = [5 * b for b in range(B)], [S - 13 * b for b in range(B)]
    table, N = _table([a + n for a, n in zip(first, new)], P, S)
    (kp, vp), (sk, sv) = _pool(kv, N, Hk, P, D, G)
    k, v = (_rows(gen, B, Hk, S, D, dtype, "projection") for _ in range(2))
    for x in (k, v):
        x[0, 0, 3::50, 2], x[0, -1, 7::50, 5], x[0, 0, 11::50, 1] = math.inf, math.nan, -math.inf
        x[:, :, 17::40] *= 1e-6
        x[:, 0, 23::40] *= 1e4
        x[:, :, 29::60] = 0
        x[0, :, 31::60] = math.nan
    q = _rows(gen, B, Hq, S, D, dtype, "projection") if Hq and rot else None
    cos, sin = skv.rotary_tables(rot, S + 100) if rot else (None, None)
    lens, fresh = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (first, new))
    out = skv.paged_append(k, v, kp, vp, table, lens, sk, sv, fresh, q, cos, sin, interleaved=interleaved, check=True)
    at = lens.long()[:, None] + torch.arange(S, device="cuda")
    turned = _turn32(k, cos[at], sin[at], interleaved) if rot else k.float()
    if q is not None:
        assert _alike(out, _turn32(q, cos[at], sin[at], interleaved).to(dtype))
    store = skv.PagedKVStore(B, Hk, D, page_size=S, device="cuda", int4_group_size=G)
    store.append(turned.contiguous(), v.float().contiguous(), kv)
    for b in range(B):
        where = torch.arange(first[b], first[b] + new[b], device="cuda")
        ids, row = table[b].long()[where // P], where % P
        for pages, scale, rows, theirs in ((kp, sk, turned, (store.pages[0].k, store.pages[0].scale_k)),
                                           (vp, sv, v.float(), (store.pages[0].v, store.pages[0].scale_v))):
            mine, nan = pages[ids, :, row].transpose(0, 1), None
            if scale is not None:   # a row or group that holds a NaN has a scale of NaN, and integers that mean nothing
                kept = scale[ids, :, row].transpose(0, 1)
                groups = kept.shape[2] if kv == "int4" else 1
                nan = rows[b, :, :new[b]].unflatten(-1, (groups, -1)).isnan().any(-1)
                assert torch.equal(kept.isnan().view(nan.shape), nan)
                assert _alike(kept, theirs[1][b, :, :new[b]], nan.view(kept.shape))
                scale[ids, :, row] = 1
                nan = nan[..., None].expand(*nan.shape, mine.shape[-1] // groups).flatten(-2)
            assert _alike(mine, theirs[0][b, :, :new[b]], nan), b
            pages[ids, :, row] = 0
    assert all((t == 0).all() for t in (kp, vp)) and all(t is None or (t == 1).all() for t in (sk, sv))   # nothing else was written


@pytest.mark.parametrize("D,G,layout", [(64, 16, "bhsd"), (64, 32, "projection"), (40, 8, "bhsd"), (33, 33, "bhsd"), (96, 16, "odd")])
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
def test_a_nan_is_read_as_one(skv, D, G, layout, kv):
    """A NaN among the values of a row: what its scale is shared by is NaN when read, everything else is as without it."""
    (kp, vp), (sk, sv) = _pool(kv, 2, 2, 8, D, G)
    table, zero = torch.tensor([[1]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = (_rows(_gen(i), 1, 2, 8, D, torch.float32, layout) for i in range(2))
    seen = torch.full((1,), 8, dtype=torch.int32, device="cuda")

    def held():
        skv.paged_append(k, v, kp, vp, table, zero, sk, sv, check=True)
        return skv.paged_read(kp, vp, table, seen, 8, sk, sv, head_dim=D, check=True)

    clean = held()
    k[0, 0, 3, 5] = v[0, 1, 6, D - 1] = math.nan
    odd = held()
    wide = {"int8": D, "int4": G if D % G == 0 else D}.get(kv, 1)
    for t, (h, s, d), before, now in ((k, (0, 3, 5), clean[0], odd[0]), (v, (1, 6, D - 1), clean[1], odd[1])):
        nan = torch.zeros(1, 2, 8, D, dtype=torch.bool, device="cuda")
        nan[0, h, s, d // wide * wide:d // wide * wide + wide] = True
        assert torch.equal(now.isnan(), nan) and torch.equal(now[~nan], before[~nan])


def test_append_of_more_rows_than_31_bits_number(skv):
    """2^31 rows and more, nearly all of them padding: the tokens are written all the same."""
    S, D = 2 ** 30 + 100, 16
    pages, _ = _pool("fp32", 2, 1, 8, D)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device="cuda")
    k, v = (_rows(_gen(i), 2, 1, 1, D, torch.float32) for i in range(2))
    new = torch.tensor([5, 8], dtype=torch.int32, device="cuda")
    skv.paged_append(k.expand(2, 1, S, D), v.expand(2, 1, S, D), *pages, table, torch.zeros_like(new), new_lengths=new, check=True)
    for mine, rows in zip(pages, (k, v)):
        want = torch.zeros_like(mine)
        want[1, 0, :5], want[0, 0] = rows[0, 0], rows[1, 0]
        assert torch.equal(mine, want)


# ------------------------------------------------------------------------------------ values that are not finite
ODD = [  # counts, H, rep, Sq, D, P, new: kernels for few rows, for many, and for any size
    ([200, 37], 2, 2, 9, 128, 16, None),
    ([70, 260, 7], 1, 5, 7, 64, 32, [7, 3, 0]),
    ([130, 77], 3, 3, 3, 80, 7, None),
    ([5000], 2, 2, 5, 128, 32, None),              # parts that are joined
    ([300, 70], 2, 1, 30, 256, 32, None),
    ([700, 150], 15, 2, 130, 128, 32, None),       # a prompt: blocks of one head's tokens
    ([700, 150], 2, 2, 130, 64, 7, [130, 60]),
    ([300, 90], 2, 8, 16, 128, 32, None),          # rows of several heads
    ([9000, 20], 2, 4, 31, 96, 16, None),
    ([260], 2, 2, 140, 256, 16, None),
    ([60, 33], 2, 2, 5, 300, 8, None),
    ([3000, 33], 1, 2, 6, 35, 8, None),
]


@pytest.mark.parametrize("counts,H,rep,Sq,D,P,new", ODD)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_attention_of_values_that_are_not_finite(skv, counts, H, rep, Sq, D, P, new, kv, dtype):
    """Infinite and NaN values among the newest tokens, and in one value or int4 group of an old one, reach the queries that
    see them, in their own values, and nothing else."""
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, sum(counts) + D)
    q = _rows(_gen(5), len(counts), H * rep, Sq, D, dtype)
    at = [(b, n - 1 - (i * Sq // 3), i % H, i) for b, n in enumerate(counts) for i in range(3) if n > i * Sq // 3]
    if kv != "int8":
        at.append((0, 3, 0, 1))
    for b, t, h, i in at:
        page, x = int(table[b, t // P]), (math.inf, math.nan, -math.inf)[i]
        if scales[1] is None:
            pages[1][page, h, t % P, (7 * i + 3) % D] = x
        else:
            scales[1][page, h, t % P, ((i + 1) % scales[1].shape[3]) if kv == "int4" else 0] = x
    fresh = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    got = skv.paged_attention(q, *pages, table, lens, *scales, causal=True, new_lengths=fresh, check=True)
    es, ep = (2.0 ** -19, 2.0 ** -19) if dtype == torch.float32 else (2.0 ** -17, 2.0 ** -11)
    for b, n in enumerate(counts):
        k, v = (_dense64(p, s, table, b, n, D) for p, s in zip(pages, scales))
        odd = ~torch.isfinite(v)
        v = v.masked_fill(odd, 0)
        qb = q[b].double().unflatten(0, (H, rep))
        s = torch.einsum("grsd,gtd->grst", qb, k) / math.sqrt(D)
        size = torch.einsum("grsd,gtd->grst", qb.abs(), k.abs()) / math.sqrt(D)
        i, t = torch.arange(Sq, device="cuda")[:, None], torch.arange(n, device="cuda")
        m = Sq if new is None else new[b]
        seen = (i < m) & (t <= n - m + i)
        w = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1), nan=0.0)
        ds = ((D * U + es) * size + 4 * U * s.abs()).masked_fill(~seen, 0).amax(-1, keepdim=True)
        want = torch.einsum("grst,gtd->grsd", w, v)
        bound = (2 * ds + n * U + ep) * torch.einsum("grst,gtd->grsd", w, v.abs())
        bound = bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype]
        hit = (torch.einsum("st,gtd->gsd", seen.double(), odd.double()) > 0)[:, None].expand(H, rep, Sq, D)
        mine = got[b].double().unflatten(0, (H, rep))
        assert torch.equal(~torch.isfinite(mine), hit)
        off = torch.where(hit, -1.0, (mine - want).abs() - bound)
        assert off.max() <= 0, float(off.max())


@pytest.mark.parametrize("counts,H,rep,Sq,D,P,new", ODD)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_keys_that_are_nan(skv, counts, H, rep, Sq, D, P, new, kv, dtype):
    """A NaN among the newest keys: the queries of its head that see it are NaN, the others are what they were."""
    pages, scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, sum(counts) + D)
    q = _rows(_gen(5), len(counts), H * rep, Sq, D, dtype)
    new = new or [Sq] * len(counts)
    want, bound = _attention64(q, pages, scales, table, counts, new, True)
    hit = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    for b, n in enumerate(counts):
        t, h = n - 1 - Sq // 3, b % H
        if t < 0:
            continue
        page = int(table[b, t // P])
        if scales[0] is None:
            pages[0][page, h, t % P, 3] = math.nan
        else:
            scales[0][page, h, t % P, 0] = math.nan
        i = torch.arange(Sq, device="cuda")
        hit[b, h * rep:(h + 1) * rep] |= (i < new[b]) & (t <= n - new[b] + i)
    got = skv.paged_attention(q, *pages, table, lens, *scales, causal=True, new_lengths=torch.tensor(new, dtype=torch.int32, device="cuda"))
    assert got[hit].isnan().all() and not got[~hit].isnan().any()
    off = (got[~hit].double() - want[~hit]).abs() - bound[~hit]
    assert off.max() <= 0, float(off.max())


@pytest.mark.parametrize("B,Hq,Hk,S,D,rot", [(2, 1, 0, 8000, 128, 128), (3, 2, 1, 6000, 64, 32), (1, 5, 3, 20000, 64, 64), (1, 40, 8, 3000, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_prompts(skv, B, Hq, Hk, S, D, rot, dtype, interleaved):
    """Enough tokens that a block takes several."""
    gen = _gen(S)
    cos, sin = skv.rotary_tables(rot, S)
    q, k = (_rows(gen, B, max(H, 1), S, D, dtype, "projection") for H in (Hq, Hk))
    got = skv.apply_rotary(q, cos, sin, k=k if Hk else None, interleaved=interleaved)
    at = torch.arange(S, device="cuda").expand(B, S)
    for x, y in zip((q, k), got if Hk else (got,)):
        assert torch.equal(y, _turn32(x, cos[at], sin[at], interleaved).to(dtype))


# ------------------------------------------------------------------------------------------------ gradients
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_backward(skv, dtype, interleaved):
    """Rows that require a gradient get the formula's: queries and keys, slices of one projection, a key head that all
    share, turned either way, one of the two results unused."""
    B, H, S, D, rot = 2, 3, 7, 48, 32
    cos, sin = skv.rotary_tables(rot, 64, scaling="ntk_parts", factor=4.0, original_positions=8)
    pos = torch.randint(0, 64, (B, S), generator=_gen(1), device="cuda")
    gen = _gen(2)
    x = torch.randn(B, S, H + 1, D, generator=gen, device="cuda").to(dtype).requires_grad_()
    for inverse in (False, True):
        for used in ("qk", "q", "k"):
            rows = x.transpose(1, 2)
            q, k = rows[:, :H], rows[:, H:].expand(B, H, S, D)
            yq, yk = skv.apply_rotary(q, cos, sin, k, pos, interleaved, inverse)
            gq, gk = (torch.randn(B, H, S, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
            x.grad = None
            torch.autograd.backward([y for n, y in (("q", yq), ("k", yk)) if n in used], [g for n, g in (("q", gq), ("k", gk)) if n in used])
            want, bound = torch.zeros(2, B, S, H + 1, D, dtype=torch.float64, device="cuda")
            for n, g, to in (("q", gq, slice(0, H)), ("k", gk, None)):
                if n in used:
                    turned, off = (t.transpose(1, 2) for t in _turn64(g, cos[pos], sin[pos], interleaved, not inverse))
                    off = off + HALF[dtype] * (turned.abs() + off) + TINY[dtype]
                    if to is not None:
                        want[:, :, to] += turned
                        bound[:, :, to] += off
                    else:   # the sum over the heads that share the key, rounded H - 1 times, and added to the rest
                        want[:, :, H] += turned.sum(2)
                        bound[:, :, H] += off.sum(2) + H * HALF[dtype] * (turned.abs() + off).sum(2)
            assert ((x.grad.double() - want).abs() <= bound + HALF[dtype] * want.abs() + TINY[dtype]).all(), (inverse, used)
    one = x.detach().transpose(1, 2).contiguous().requires_grad_()
    y = skv.apply_rotary(one, cos, sin, positions=pos, interleaved=interleaved)
    assert torch.equal(y, skv.apply_rotary(one.detach(), cos, sin, positions=pos, interleaved=interleaved)) and y.requires_grad
    (g,) = torch.autograd.grad(y, one, torch.ones_like(y), create_graph=True)   # linear: the second turn is the first one's inverse's inverse
    assert torch.equal(g, skv.apply_rotary(torch.ones_like(y), cos, sin, positions=pos, interleaved=interleaved, inverse=True))
    with torch.no_grad():
        assert not skv.apply_rotary(one, cos, sin, positions=pos).requires_grad


def test_pool_does_not_wait_for_the_gpu(skv):
    """Taking pages, ragged appends, the block's forward and the end of a sequence put work on the stream and return."""
    pool = skv.PagedKVPool(64, 2, 2, 32, max_tokens=128, page_size=8, precision="int8")
    cos, sin = skv.rotary_tables(32, 128)

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.hidden_dim, self.num_heads, self.head_dim = 64, 2, 32
            self.ln1, self.ln2 = torch.nn.LayerNorm(64), torch.nn.LayerNorm(64)
            self.q_proj, self.k_proj, self.v_proj, self.o_proj, self.up_proj, self.down_proj = (torch.nn.Linear(64, 64) for _ in range(6))

    block = Block().cuda()
    x = torch.randn(2, 2, 20, 32, generator=_gen(1), device="cuda")
    hidden = torch.randn(2, 9, 64, generator=_gen(2), device="cuda")

    def steps():
        pool.append(x, x, q=x, cos=cos, sin=sin, new_lengths=[20, 3])
        pool.append(x[:, :, :5], x[:, :, :5])
        y = skv.paged_block_forward(block, hidden, pool, cos, sin, causal=True, new_lengths=[9, 4])
        pool.read(10)
        pool.release(1)
        return y

    with torch.no_grad():
        steps()
        pool.release(0)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            steps()
        finally:
            torch.cuda.set_sync_debug_mode("default")
    assert pool.lengths.tolist() == pool.token_counts == [34, 0]
    assert pool.block_table[0, :5].tolist() == pool._table[0, :5].tolist() and (pool.block_table[1] == -1).all()


# ----------------------------------------------------------------------------------------- threads and scratch
def test_attention_from_two_threads_on_one_stream(skv):
    """Calls whose parts are joined by a second launch, from two host threads on one stream, which share their scratch."""
    import threading

    calls = []
    for seed, (counts, H, rep, Sq) in enumerate((([9000, 16], 2, 4, 31), ([7000, 3000, 5], 1, 3, 33))):
        pages, scales, table, lens = _filled(skv, "fp16", counts, H, 32, 128, 16, seed)
        q = _rows(_gen(seed), len(counts), H * rep, Sq, 128, torch.bfloat16)
        calls.append(lambda q=q, pages=pages, table=table, lens=lens: skv.paged_attention(q, *pages, table, lens))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(2)

    def work(i):
        go.wait()
        for _ in range(300):
            if not torch.equal(calls[i](), want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
