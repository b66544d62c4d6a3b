"""Page bounds, page selection and attention of the selected pages on the GPU, against plain implementations in 64 bits.

Bounds and selections are whole numbers and are compared exactly.  Attention of listed pages is bounded like that of whole
sequences (see test_gpu_paged_pool.py), over the tokens of the listed pages.
"""

import math

import pytest
import torch

from test_gpu_paged_pool import HALF, TINY, U, _dense64, _filled, _gen, _pool, _rows, _table, skv  # noqa: F401

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def _power64(top):
    """The least power of two, 2^-126 and up, of which 127 reach `top`; one for zero, +inf for what is not finite."""
    out = torch.ones_like(top)
    for i, x in enumerate(top.flatten().tolist()):
        if not x < math.inf:
            out.view(-1)[i] = math.inf
        elif x > 0:
            e = -126
            while 127.0 * 2.0 ** e < x:
                e += 1
            out.view(-1)[i] = 2.0 ** e
    return out


def _bounds64(x):
    """Bounds and steps of a page's tokens [H, n, D] in 64 bits."""
    low, high = x.amin(1), x.amax(1)
    step = _power64(x.abs().amax((1, 2)))
    scale = torch.where(step < math.inf, step, torch.ones_like(step))[:, None]
    pair = torch.stack((torch.floor(low / scale), torch.ceil(high / scale)), 1)
    return torch.where((step < math.inf)[:, None, None], pair, torch.zeros_like(pair)).to(torch.int8), step.float()


def _lens(counts):
    return torch.tensor(counts, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------------------------- bounds
BOUNDS = [  # counts, H, D, P, G
    ([0, 1, 2, 31, 32, 33, 100], 2, 128, 32, 16),
    ([77, 0, 5], 3, 80, 7, 16),          # 10 lanes a row, 2 left over
    ([300, 40], 1, 64, 16, 64),
    ([129, 17], 2, 256, 64, 32),
    ([50], 5, 96, 17, 48),
    ([61, 20], 2, 33, 5, 16),            # an odd head, one int4 group
    ([40, 3], 1, 300, 8, 16),            # a head above 256 values
    ([9], 2, 8, 1, 8),
    ([10, 3], 2, 24, 4, 4),              # int4 groups of half a lane
]


@pytest.mark.parametrize("counts,H,D,P,G", BOUNDS)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
def test_bounds_are_those_of_the_tokens(skv, counts, H, D, P, G, kv):
    (kp, _), (sk, _), table, lens = _filled(skv, kv, counts, H, P, D, G, sum(counts), channels=4.0)
    N = kp.shape[0]
    for first in (None, [max(0, c - 1) for c in counts], [c // 2 for c in counts], list(counts), [c + 5 for c in counts]):
        bounds = torch.full((N, H, 2, D), 99, dtype=torch.int8, device="cuda")
        steps = torch.full((N, H), 3.0, device="cuda")
        want, want_steps = bounds.clone(), steps.clone()
        got = skv.page_bounds(kp, table, lens, sk, None if first is None else _lens(first), bounds, steps, head_dim=D, check=True)
        assert got[0] is bounds and got[1] is steps
        for b, n in enumerate(counts):
            if n == 0:
                continue
            # a cache's values are products of 32 bits
            x = _dense64((kp), sk, table, b, n, D).float().double()
            f = 0 if first is None else first[b]
            for j in range(f // P if f < n else 1 << 30, -(-n // P)):
                page = int(table[b, j])
                want[page], want_steps[page] = _bounds64(x[:, j * P:(j + 1) * P])
        assert torch.equal(bounds, want) and torch.equal(steps, want_steps)
    made = skv.page_bounds(kp, table, lens, sk, head_dim=D)
    assert made[0].shape == (N, H, 2, D) and made[1].shape == (N, H)


def test_bounds_of_extreme_values(skv):
    """Values at the ends of the format, and values that are not finite."""
    rows = [
        [1e-45, -1e-45], [-1e-45, 0.0], [0.0, -0.0], [3.4028234663852886e38, -1.0], [-3.4028234663852886e38, 1e-45],
        [127.0, -127.0], [127.00001, -1.0], [254.0, 1.0], [63.5, 0.25], [1.1754943508222875e-38, 2.0 ** -149],
        [math.inf, 1.0], [-math.inf, 1.0], [math.nan, 1.0], [2.0 ** -120, -1e-44], [1.0, -1e-30], [2.0 ** 127, 2.0 ** -126],
    ]
    D, N = 8, len(rows)
    kp = torch.zeros(N, 1, 2, D, device="cuda")
    for i, (x, y) in enumerate(rows):
        kp[i, 0, 0, 3], kp[i, 0, 1, 3] = x, y
        kp[i, 0, 0, 5] = y
    table = torch.arange(N, dtype=torch.int32, device="cuda")[None]
    bounds, steps = skv.page_bounds(kp, table, _lens([2 * N]))
    for i in range(N):
        want, step = _bounds64(kp[i].double())
        assert torch.equal(steps[i], step), rows[i]
        assert torch.equal(bounds[i], want), rows[i]
    # every page's bounds hold its keys (in 64 bits)
    finite = steps[:, 0] < math.inf
    s = steps.double()[:, :, None]
    assert (kp.double().amin(2) >= bounds[:, :, 0].double() * s)[finite].all() and (kp.double().amax(2) <= bounds[:, :, 1].double() * s)[finite].all()


def test_bounds_name_bad_pages_and_lengths(skv):
    kp, table, lens = torch.randn(4, 1, 8, 16, device="cuda"), torch.tensor([[0, 9, -1]], dtype=torch.int32, device="cuda"), _lens([20])
    with pytest.raises(ValueError, match="outside"):
        skv.page_bounds(kp, table, lens, check=True)
    skv.page_bounds(kp, table, lens)                    # the other page's are written
    for n in (-1, 25):
        with pytest.raises(ValueError, match="outside"):
            skv.page_bounds(kp, table[:, :1].repeat(1, 3), _lens([n]), check=True)
    for kw in (dict(bounds=torch.zeros(4, 1, 2, 16, dtype=torch.int8, device="cuda")), dict(start=_lens([1, 2])),
               dict(bounds=torch.zeros(4, 1, 2, 8, dtype=torch.int8, device="cuda"), steps=torch.ones(4, 1, device="cuda")),
               dict(bounds=torch.zeros(4, 1, 2, 16, device="cuda"), steps=torch.ones(4, 1, device="cuda")),
               dict(bounds=torch.zeros(4, 1, 2, 16, dtype=torch.int8, device="cuda"), steps=torch.ones(4, 1))):
        with pytest.raises(ValueError):
            skv.page_bounds(kp, table, lens, **kw)


# ------------------------------------------------------------------------------------------ selection
def _select64(q, bounds, steps, table, counts, P, keep, first, recent, causal, new):
    """The definition in 64-bit whole numbers."""
    B, Hq, Sq, D = q.shape
    N, H = steps.shape
    out = torch.full((B, H, Sq, keep), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        if n <= 0:
            continue
        qb = q[b].double().unflatten(0, (H, -1))
        top = qb.abs().amax(-1)
        t = _power64(top.masked_fill(~(top < math.inf), 0.0))
        whole = torch.where((top < math.inf)[..., None], torch.round(qb / t[..., None]), torch.zeros_like(qb))
        ids = table[b, :-(-n // P)].long()
        named = (ids >= 0) & (ids < N)
        low, high = (bounds[ids.clamp(0, N - 1), :, i].double() for i in (0, 1))
        dot = torch.einsum("hrsd,phd->hsrp", whole.clamp_min(0), high) + torch.einsum("hrsd,phd->hsrp", whole.clamp_max(0), low)
        score = (dot * t.transpose(1, 2)[..., None]).amax(2)
        step = steps[ids.clamp(0, N - 1)].double().T[:, None]
        score = torch.where(step < math.inf, score * torch.where(step < math.inf, step, torch.ones_like(step)), torch.full_like(score, math.inf))
        score = score.float().double().masked_fill(~named, -math.inf).cpu()
        for i in range(Sq):
            seen = 0 if i >= new[b] else max(0, n - new[b] + 1 + i) if causal else n
            total = -(-seen // P)
            for h in range(H):
                if total <= keep:
                    chosen = list(range(total))
                else:
                    middle = torch.sort(score[h, i, first:total - recent], descending=True, stable=True).indices[:keep - first - recent]
                    chosen = sorted(list(range(first)) + (middle + first).tolist() + list(range(total - recent, total)))
                out[b, h, i, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out.cuda()


SELECT = [  # counts, H, rep, Sq, D, P, keep, first, recent, causal
    ([1], 1, 1, 1, 64, 16, 3, 1, 1, False),
    ([5000], 2, 4, 1, 128, 16, 32, 1, 2, False),
    ([0, 1, 16, 17, 200, 3000], 3, 3, 1, 128, 16, 8, 0, 1, False),
    ([1000, 37, 512], 2, 1, 5, 80, 7, 11, 2, 3, True),
    ([900], 1, 8, 13, 96, 8, 20, 1, 1, True),
    ([400, 40], 2, 12, 3, 64, 4, 9, 1, 1, True),          # two tiles of heads
    ([400, 333], 1, 40, 2, 32, 4, 9, 1, 1, False),        # more than four
    ([700], 3, 2, 40, 128, 16, 7, 1, 1, True),            # more columns than a block takes
    ([300, 80], 2, 3, 3, 33, 5, 6, 1, 1, True),           # an odd head
    ([200], 1, 2, 2, 300, 4, 5, 1, 1, False),             # a head above 256 values
    ([2000], 1, 5, 2, 256, 16, 100, 1, 1, False),
    ([9000], 1, 2, 1, 16, 4, 50, 1, 1, False),            # more pages than a block keeps in registers
    ([640], 2, 2, 1, 64, 16, 3, 1, 2, False),             # nothing to choose
    ([20], 2, 2, 1, 64, 16, 5, 1, 1, False),              # the table is narrower than the list
]


@pytest.mark.parametrize("counts,H,rep,Sq,D,P,keep,first,recent,causal", SELECT)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("layout", ["bhsd", "projection", "odd"])
def test_selection_is_the_definitions(skv, counts, H, rep, Sq, D, P, keep, first, recent, causal, dtype, layout):
    gen = _gen(sum(counts) + D)
    table, N = _table(counts, P, D)
    bounds = torch.randint(-127, 128, (N, H, 2, D), generator=gen, device="cuda", dtype=torch.int8).sort(2).values
    steps = 2.0 ** torch.randint(-3, 2, (N, H), generator=gen, device="cuda").float()
    q = _rows(gen, len(counts), H * rep, Sq, D, dtype, layout)
    for new in ([Sq] * len(counts), [max(0, Sq - b) for b in range(len(counts))]):
        got = skv.page_select(q, bounds, steps, table, _lens(counts), P, keep, first, recent, causal, _lens(new), check=True)
        assert torch.equal(got, _select64(q, bounds, steps, table, counts, P, keep, first, recent, causal, new))
    if not causal or Sq == 1:
        got = skv.page_select(q, bounds, steps, table, _lens(counts), P, keep, first, recent)
        assert torch.equal(got, _select64(q, bounds, steps, table, counts, P, keep, first, recent, False, [Sq] * len(counts)))


@pytest.mark.parametrize("B", [1, 5, 20, 40])
def test_selection_of_heads_above_128_values(skv, B):
    """However many blocks share a sequence's pages."""
    counts = [16 * (1 + 37 * b % 190) for b in range(B - 1)] + [16 * 300]
    test_selection_is_the_definitions(skv, counts, 8, 2, 1, 256, 16, 20, 1, 1, False, torch.bfloat16, "bhsd")


@pytest.mark.parametrize("rep", [1, 4, 9])
@pytest.mark.parametrize("size", [5e33, 1e30, 1e-30, 4e-36])
def test_selection_of_very_large_and_small_queries(skv, size, rep):
    """Scores are whole numbers below 2^24 times powers of two: exact as long as the score itself fits a float."""
    gen = _gen(rep)
    kp = torch.randn(90, 2, 8, 64, generator=gen, device="cuda")
    table = torch.randperm(90, generator=gen, device="cuda").int()[None, :88]
    lens = _lens([700])
    bounds, steps = skv.page_bounds(kp, table, lens)
    q = torch.randn(1, 2 * rep, 3, 64, generator=gen, device="cuda") * size
    want = _select64(q, bounds, steps, table, [700], 8, 11, 1, 2, False, [3])
    assert torch.equal(skv.page_select(q, bounds, steps, table, lens, 8, 11, 1, 2, check=True), want)


def test_selection_ties_and_pages_that_nothing_bounds(skv):
    """Equal scores go to the lowest page, pages without a finite step come first, unnamed ones last."""
    H, D, P, n = 2, 64, 4, 400
    gen = _gen(5)
    counts = [n, n - 3]
    table, N = _table(counts, P, 3)
    bounds = torch.randint(-2, 3, (N, H, 2, D), generator=gen, device="cuda", dtype=torch.int8).sort(2).values
    steps = torch.ones(N, H, device="cuda")
    bounds[::2] = bounds[0]                                # half of the pages score alike
    q = torch.randint(-1, 2, (2, 2 * H, 3, D), generator=gen, device="cuda").float()
    for case in range(4):
        if case == 1:
            steps[torch.randperm(N, generator=torch.Generator().manual_seed(1))[:9].cuda()] = math.inf
        if case == 2:
            q[0, 1, 2, 7], q[1, 0, 0, 0] = math.nan, math.inf
        if case == 3:
            q.zero_()
        for keep in (2, 7, 60, 98, 99):
            got = skv.page_select(q, bounds, steps, table, _lens(counts), P, keep, 1, 1, True, check=True)
            assert torch.equal(got, _select64(q, bounds, steps, table, counts, P, keep, 1, 1, True, [3, 3]))
    table[0, 5], table[0, 50], table[1, 7] = -1, N, -7
    with pytest.raises(ValueError, match="outside"):
        skv.page_select(q, bounds, steps, table, _lens(counts), P, 97, check=True)
    q.normal_(generator=gen)
    for keep in (7, 96, 97, 98):
        got = skv.page_select(q, bounds, steps, table, _lens(counts), P, keep)
        assert torch.equal(got, _select64(q, bounds, steps, table, counts, P, keep, 1, 1, False, [3, 3]))


@pytest.mark.parametrize("D,rep", [(16, 1), (128, 4), (64, 12), (33, 2)])
def test_pages_that_are_not_finite_go_before_scores_that_overflow(skv, D, rep):
    k = torch.ones(1, 1, 24, D, device="cuda")
    k[:, :, 4:8], k[:, :, 17, 3] = 2.0 ** 60, math.nan       # pages 1 and 4 of 6
    table = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    bounds, steps = skv.page_bounds(k.view(6, 4, 1, D).transpose(1, 2).contiguous(), table, _lens([24]))
    assert steps[4] == math.inf
    q = torch.full((1, rep, 1, D), 2.0 ** 90, device="cuda")
    for keep, want in ((1, [5]), (2, [4, 5]), (3, [1, 4, 5]), (4, [0, 1, 4, 5])):
        assert skv.page_select(q, bounds, steps, table, _lens([24]), 4, keep, first=0)[0, 0, 0].tolist() == want


@pytest.mark.parametrize("n", [-3, 41])
def test_selection_names_bad_lengths(skv, n):
    bounds, steps = torch.zeros(4, 1, 2, 16, dtype=torch.int8, device="cuda"), torch.ones(4, 1, device="cuda")
    q, table = torch.randn(1, 1, 1, 16, device="cuda"), torch.zeros(1, 5, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="outside"):
        skv.page_select(q, bounds, steps, table, _lens([n]), 8, 2, check=True)
    got = skv.page_select(q, bounds, steps, table, _lens([n]), 8, 2)
    assert got.flatten().tolist() == ([-1, -1] if n < 0 else [0, 4])


def test_selection_over_a_pool_without_pages(skv):
    """No table entry can name a page: the pages that are always read, then the lowest, and no memory of the pool is looked at."""
    bounds, steps = torch.zeros(0, 2, 2, 64, dtype=torch.int8, device="cuda"), torch.ones(0, 2, device="cuda")
    q, table = torch.randn(1, 4, 3, 64, device="cuda"), torch.zeros(1, 50, dtype=torch.int32, device="cuda")
    got = skv.page_select(q, bounds, steps, table, _lens([400]), 8, 5)
    assert (got == torch.tensor([0, 1, 2, 3, 49], device="cuda")).all()
    with pytest.raises(ValueError, match="outside"):
        skv.page_select(q, bounds, steps, table, _lens([400]), 8, 5, check=True)


def test_selection_refusals(skv):
    bounds, steps = torch.zeros(4, 2, 2, 16, dtype=torch.int8, device="cuda"), torch.ones(4, 2, device="cuda")
    q, table, lens = torch.randn(1, 4, 1, 16, device="cuda"), torch.zeros(1, 5, dtype=torch.int32, device="cuda"), _lens([9])
    good = (q, bounds, steps, table, lens, 8, 3)
    skv.page_select(*good)
    for i, wrong in ((0, q[0]), (0, q[:, :3]), (0, q[..., :8]), (1, bounds.cpu()), (1, bounds.float()), (1, bounds[0]), (2, steps[:3]),
                     (2, steps.double()), (3, table[0]), (3, table.repeat(2, 1)), (3, table.float()), (4, lens.repeat(2)), (5, 0), (6, 1)):
        with pytest.raises(ValueError):
            skv.page_select(*good[:i], wrong, *good[i + 1:])
    for kw in (dict(first=-1), dict(recent=0), dict(first=3), dict(new_lengths=_lens([1, 1]))):
        with pytest.raises(ValueError):
            skv.page_select(*good, **kw)
    big = torch.zeros(1, 1, 2, 1032, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError):
        skv.page_select(torch.zeros(1, 1, 1, 1032, device="cuda"), big, torch.ones(1, 1, device="cuda"), table, lens, 8, 3)


# ------------------------------------------------------------------------------------------ attention
def _sparse64(q, pages_kv, scales, table, counts, new, causal, pages):
    """Attention of the listed pages in 64 bits, and the bound of test_gpu_paged_pool.py."""
    B, Hq, Sq, D = q.shape
    H, P = pages_kv[0].shape[1:3]
    out, bound = (torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device="cuda") for _ in range(2))
    es, ep = (2.0 ** -19, 2.0 ** -19) if q.dtype == torch.float32 else (2.0 ** -17, 2.0 ** -11)
    for b, n in enumerate(counts):
        if n == 0:
            continue
        k, v = (_dense64(p, s, table, b, n, D) for p, s in zip(pages_kv, scales))
        for i in range(Sq):
            see = 0 if i >= new[b] else max(0, n - new[b] + 1 + i) if causal else n
            for h in range(H):
                top, tokens = -1, []
                for e in pages[b, h, i].tolist():
                    if e > top and e * P < see:
                        tokens += range(e * P, min(see, e * P + P))
                    top = max(top, e)
                if not tokens:
                    continue
                kh, vh = k[h, tokens], v[h, tokens]
                qh = q[b].unflatten(0, (H, -1))[h, :, i].double()
                s = qh @ kh.T / math.sqrt(D)
                size = qh.abs() @ kh.abs().T / math.sqrt(D)
                w = torch.softmax(s, -1)
                ds = ((D * U + es) * size + 4 * U * s.abs()).amax(-1, keepdim=True)
                to = out[b].unflatten(0, (H, -1))[h, :, i], bound[b].unflatten(0, (H, -1))[h, :, i]
                to[0].copy_(w @ vh)
                to[1].copy_((2 * ds + len(tokens) * U + ep) * (w @ vh.abs()))
    return out, bound + HALF[q.dtype] * (out.abs() + bound) + TINY[q.dtype]


SPARSE = [  # counts, H, rep, Sq, D, P, G, causal, keep
    ([1], 1, 1, 1, 64, 16, 16, False, 1),
    ([512], 4, 1, 1, 128, 32, 16, False, 5),
    ([0, 1, 15, 16, 17, 33, 129, 2000], 2, 4, 1, 128, 16, 16, False, 9),
    ([257, 3, 96], 2, 2, 4, 128, 16, 16, True, 4),
    ([200, 5], 1, 5, 7, 64, 32, 16, True, 2),
    ([130, 0, 77], 3, 3, 3, 80, 7, 16, True, 6),
    ([61, 20], 2, 2, 2, 33, 5, 16, False, 4),
    ([100], 2, 6, 2, 256, 8, 16, True, 7),
    ([40], 1, 1, 1, 300, 8, 16, False, 3),
    ([333, 700], 1, 12, 2, 128, 32, 64, False, 33),
    ([300], 1, 50, 2, 64, 16, 32, False, 7),                # enough rows a key head for the kernel of prompts
    ([170] * 40, 4, 3, 3, 64, 16, 16, True, 8),             # more units than CTAs: whole ones, one after the other
    ([300, 20] * 30, 8, 2, 1, 64, 16, 16, False, 15),       # in even shares
]


@pytest.mark.parametrize("counts,H,rep,Sq,D,P,G,causal,keep", SPARSE)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", FLOATS)
def test_attention_of_listed_pages(skv, counts, H, rep, Sq, D, P, G, causal, keep, kv, dtype):
    pages_kv, scales, table, lens = _filled(skv, kv, counts, H, P, D, G, sum(counts) + Sq)
    gen = _gen(D + keep)
    B = len(counts)
    layout = ["bhsd", "projection", "odd"][(D + Sq) % 3]
    q = _rows(gen, B, H * rep, Sq, D, dtype, layout)
    width = table.shape[1]
    pages = torch.stack([torch.randperm(width, generator=gen, device="cuda") for _ in range(B * H * Sq)])[:, :keep]
    if pages.shape[1] < keep:
        pages = torch.cat((pages, pages.new_full((B * H * Sq, keep - pages.shape[1]), -1)), 1)
    pages = pages.view(B, H, Sq, keep).sort(-1).values.int()
    new = [max(0, Sq - b) for b in range(B)]
    for listed in (pages, pages.flip(-1), pages.roll(1, -1)):    # ascending, and lists of which not all counts
        got = skv.paged_attention(q, *pages_kv, table, lens, *scales, causal=causal, new_lengths=_lens(new), pages=listed)
        want, bound = _sparse64(q, pages_kv, scales, table, counts, new, causal, listed)
        assert got.shape == q.shape and got.dtype == dtype
        assert ((got.double() - want).abs() <= bound).all()
        assert (got[want == 0] == 0).all() or (want == 0).sum() < D


CUTS = [  # counts, H, rep, keep: units of 1 to 150, of few and of many tokens, whole or over some CTAs
    ([4096], 8, 4, 128), ([2048, 40], 8, 4, 64), ([2048, 2000], 8, 1, 63), ([3000, 3000, 10], 20, 1, 90), ([1100] * 2, 32, 2, 32),
    ([600] * 4, 37, 1, 16), ([1000] * 5, 30, 1, 20), ([512], 1, 8, 16), ([5000], 1, 1, 157), ([250] * 10, 10, 1, 8), ([1024] * 8, 16, 1, 31),
]


@pytest.mark.parametrize("counts,H,rep,keep", CUTS)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_listed_pages_however_units_are_cut(skv, counts, H, rep, keep, kv, dtype):
    pages_kv, scales, table, lens = _filled(skv, kv, counts, H, 32, 128, 16, sum(counts))
    gen = _gen(keep)
    B = len(counts)
    q = _rows(gen, B, H * rep, 1, 128, dtype, "bhsd")
    pages = torch.rand(B, H, 1, max(keep, table.shape[1]), generator=gen, device="cuda").argsort(-1)[..., :keep].sort(-1).values.int()
    got = skv.paged_attention(q, *pages_kv, table, lens, *scales, pages=pages)
    want, bound = _sparse64(q, pages_kv, scales, table, counts, [1] * B, False, pages)
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(skv.paged_attention(q, *pages_kv, table, lens, *scales, pages=pages), got)


def test_listed_pages_broadcast_and_tell_nothing_else(skv):
    """Lists are broadcast, 64-bit lists are not cut, and what is in a list besides its pages changes nothing."""
    counts, H, P, D = [200, 90], 2, 16, 64
    pages_kv, scales, table, lens = _filled(skv, "int8", counts, H, P, D, 16, 8)
    q = _rows(_gen(1), 2, 4, 3, D, torch.float16, "projection")

    def attend(pages, **kw):
        return skv.paged_attention(q, *pages_kv, table, lens, *scales, pages=pages, **kw)

    some = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    want = attend(some.expand(2, H, 3, 3).contiguous())
    assert torch.equal(attend(some.view(1, 1, 1, 3)), want)
    assert torch.equal(attend(some.view(1, 1, 1, 3).expand(2, H, 3, 3)), want)
    junk = torch.tensor([-5, 0, 0, -1, 2, 1, 5, 5, 2, 2 ** 40, 6, -2 ** 40], device="cuda").view(1, 1, 1, -1)
    assert torch.equal(attend(junk), want)
    with pytest.raises(ValueError, match="outside"):
        attend(junk, check=True)
    assert torch.equal(attend(torch.tensor([0, 2, 5, -1, -1], device="cuda").view(1, 1, 1, -1), check=True), want)
    assert (attend(torch.full((1, 1, 1, 2), -1, device="cuda")) == 0).all()
    for wrong in (some, some.view(1, 1, 3), some.view(1, 1, 1, 3).expand(2, 3, 3, 3), some.view(1, 1, 1, 3)[..., :0], some.view(1, 1, 1, 3).float()):
        with pytest.raises(ValueError):
            attend(wrong)


def test_what_is_not_listed_is_not_read(skv):
    """NaN and infinities in pages that no list names, and behind what a query sees, reach nothing."""
    counts, H, P, D = [160], 2, 16, 128
    for kv in ("fp32", "fp16", "int8", "int4"):
        (kp, vp), scales, table, lens = _filled(skv, kv, counts, H, P, D, 16, 3)
        q = _rows(_gen(2), 1, 2, 2, D, torch.bfloat16)
        pages = torch.tensor([0, 3, 9], device="cuda").view(1, 1, 1, 3)
        want = skv.paged_attention(q, kp, vp, table, lens, *scales, causal=True, pages=pages)
        for j in (1, 2, 4, 5, 6, 7, 8):
            for t in (kp, vp) if scales[0] is None else scales:
                t[int(table[0, j])] = math.nan if j % 2 else math.inf
        assert torch.isfinite(want).all()
        assert torch.equal(skv.paged_attention(q, kp, vp, table, lens, *scales, causal=True, pages=pages), want)


def test_all_pages_listed_is_the_dense_attention(skv):
    counts = [700, 33, 0]
    pages_kv, scales, table, lens = _filled(skv, "fp16", counts, 2, 32, 128, 16, 4)
    q = _rows(_gen(3), 3, 8, 1, 128, torch.float32)
    every = torch.arange(table.shape[1], device="cuda").view(1, 1, 1, -1)
    a, b = (skv.paged_attention(q, *pages_kv, table, lens, pages=p) for p in (None, every))
    want, bound = _sparse64(q, pages_kv, scales, table, counts, [1] * 3, False, every.expand(3, 2, 1, -1))
    assert ((a.double() - want).abs() <= bound).all() and ((b.double() - want).abs() <= bound).all()


# -------------------------------------------------------------------------------------- streams, graphs, the pool
def test_selection_in_a_graph_and_on_another_stream(skv):
    counts, H, P, D = [500, 300], 2, 16, 128
    pages_kv, scales, table, lens = _filled(skv, "int8", counts, H, P, D, 16, 6)
    q = _rows(_gen(5), 2, 8, 1, D, torch.float16)
    bounds, steps = torch.zeros(pages_kv[0].shape[0], H, 2, D, dtype=torch.int8, device="cuda"), torch.ones(pages_kv[0].shape[0], H, device="cuda")

    def step():
        skv.page_bounds(pages_kv[0], table, lens, scales[0], None, bounds, steps)
        pages = skv.page_select(q, bounds, steps, table, lens, P, 6)
        return pages, skv.paged_attention(q, *pages_kv, table, lens, *scales, pages=pages)

    want = step()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = step()
    other.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    bounds.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (7, 8):
        q.copy_(_rows(_gen(seed), 2, 8, 1, D, torch.float16))
        lens.copy_(_lens([400 + seed, 299]))
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, step()))


def test_sparse_calls_from_two_threads_on_one_stream(skv):
    """Selection and attention of both kinds (units split by number, and in even shares) from two host threads that share workspaces."""
    import threading

    calls = []
    for seed, (counts, H, rep, Sq, keep) in enumerate((([3000, 16], 2, 4, 1, 30), ([2000] * 64, 8, 3, 1, 20))):
        pages_kv, scales, table, lens = _filled(skv, "fp16", counts, H, 32, 128, 16, seed)
        bounds, steps = skv.page_bounds(pages_kv[0], table, lens)
        q = _rows(_gen(seed), len(counts), H * rep, Sq, 128, torch.bfloat16)

        def call(q=q, pages_kv=pages_kv, table=table, lens=lens, bounds=bounds, steps=steps, keep=keep):
            pages = skv.page_select(q, bounds, steps, table, lens, 32, keep)
            return pages, skv.paged_attention(q, *pages_kv, table, lens, pages=pages)
        calls.append(call)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(2)

    def work(i):
        go.wait()
        for _ in range(200):
            if not all(torch.equal(a, b) for a, b in zip(calls[i](), want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_calls_that_start_early_read_what_was_written_last(skv):
    """Inputs change in place behind a slow kernel, and a choice of pages, behind which the next calls are set up early, stands between."""
    gen = _gen(30)
    counts, H, D, P, keep = [700, 333, 512], 2, 64, 16, 9
    pages_kv, scales, table, lens = _filled(skv, "fp16", counts, H, P, D, 16, 7)
    bounds, steps = skv.page_bounds(pages_kv[0], table, lens)
    q, other = torch.randn(2, 3, 2 * H, 1, D, generator=gen, device="cuda")
    logits, scores, lengths = torch.zeros(2, 4, 5003, device="cuda"), torch.zeros(2, 4, device="cuda"), lens.clone()
    slow = torch.randn(4096, 4096, generator=gen, device="cuda")

    def calls():
        skv.page_select(other, bounds, steps, table, lens, P, keep)
        beams = skv.beam_select(logits, scores, 7)
        skv.page_select(other, bounds, steps, table, lens, P, keep)
        chosen = skv.page_select(q, bounds, steps, table, lengths, P, keep)
        return [*beams, chosen, skv.paged_attention(q, *pages_kv, table, lengths, pages=chosen)]

    for _ in range(20):
        new = torch.randn(2, 4, 5003, generator=gen, device="cuda"), torch.randn(2, 4, generator=gen, device="cuda"), \
            lens - torch.randint(300, (3,), generator=gen, device="cuda", dtype=torch.int32), torch.randn(q.shape, generator=gen, device="cuda")
        torch.cuda.synchronize()
        slow @ slow
        for to, x in zip((logits, scores, lengths, q), new):
            to.copy_(x)
        got = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, calls()))


def test_two_graphs_do_not_share_workspaces(skv):
    """Graphs captured on one stream and replayed on two."""
    made = []
    for seed, counts in enumerate(([2000, 1500], [900, 3000])):
        pages_kv, scales, table, lens = _filled(skv, "int8", counts, 2, 16, 128, 16, seed)
        bounds, steps = skv.page_bounds(pages_kv[0], table, lens, scales[0])
        q = _rows(_gen(seed), 2, 8, 4, 128, torch.float16, "projection")
        logits, scores = torch.randn(2, 4, 20000, generator=_gen(seed), device="cuda"), torch.zeros(2, 4, device="cuda")

        def step(q=q, pages_kv=pages_kv, scales=scales, table=table, lens=lens, bounds=bounds, steps=steps, logits=logits, scores=scores):
            pages = skv.page_select(q, bounds, steps, table, lens, 16, 12, causal=True)
            return (pages, skv.paged_attention(q, *pages_kv, table, lens, *scales, causal=True, pages=pages),
                    *skv.beam_select(logits, scores, 9))

        want = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        made.append((graph, got, want, step))   # (a graph does not keep what it reads)
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(20):
        for _, got, _, _ in made:
            for x in got:
                x.zero_()
        torch.cuda.synchronize()
        for (graph, *_), s in zip(made, streams):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _ in made:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("precision", ["fp32", "fp16", "int8", "int4"])
def test_pool_keeps_its_bounds(skv, precision):
    """Appends of prompts and single tokens leave the bounds that a look at the whole pool gives, and the choice reads them."""
    pool = skv.PagedKVPool(64, 3, 2, 64, max_tokens=320, page_size=8, precision=precision, bounds=True)
    gen = _gen(9)
    for new in ([100, 3, 0], [1, 1, 1], [50, 8, 20], [1, 1, 1]):
        k, v = (torch.randn(3, 2, max(new), 64, generator=gen, device="cuda") for _ in range(2))
        pool.append(k, v, new_lengths=new)
        for b in range(3):
            for j in range(-(-pool.token_counts[b] // 8)):
                want = skv.page_bounds(pool.k_pages, pool.block_table, pool.lengths, pool.scale_k)
                page = int(pool.block_table[b, j])
                assert torch.equal(pool.bounds[page], want[0][page]) and torch.equal(pool.steps[page], want[1][page])
    q = torch.randn(3, 4, 1, 64, generator=gen, device="cuda")
    pages = skv.page_select(q, pool.bounds, pool.steps, pool.block_table, pool.lengths, 8, 5, 2, 1)
    want = skv.paged_attention(q, pool.k_pages, pool.v_pages, pool.block_table, pool.lengths, pool.scale_k, pool.scale_v, pages=pages)
    assert torch.equal(pool.attention(q, keep=5, first=2), want)
    with pytest.raises(ValueError, match="bounds"):
        skv.PagedKVPool(4, 1, 1, 16, 32).attention(torch.zeros(1, 1, 1, 16, device="cuda"), keep=3)


def test_block_forward_over_chosen_pages(skv):
    """With as many pages as there are the block's result is the dense one's; with fewer, that of its own parts."""
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.hidden_dim, self.num_heads, self.head_dim, self.num_kv_heads = 256, 4, 64, 2
            self.ln1, self.ln2 = torch.nn.LayerNorm(256), torch.nn.LayerNorm(256)
            self.q_proj, self.o_proj, self.up_proj, self.down_proj = (torch.nn.Linear(256, 256) for _ in range(4))
            self.k_proj, self.v_proj = (torch.nn.Linear(256, 128) for _ in range(2))

    torch.manual_seed(0)
    block = Block().cuda()
    cos, sin = skv.rotary_tables(64, 512)
    x = torch.randn(2, 120, 256, generator=_gen(4), device="cuda")

    def run(**kw):
        pool = skv.PagedKVPool(64, 2, 2, 64, max_tokens=256, page_size=8, bounds=True)
        with torch.no_grad():
            skv.paged_block_forward(block, x, pool, cos, sin, causal=True)
            return skv.paged_block_forward(block, x[:, :1], pool, cos, sin, **kw), pool

    dense, _ = run()
    every, _ = run(keep=16)
    few, pool = run(keep=4)
    assert (dense - every).abs().max() < 1e-4 * dense.abs().max() and not torch.equal(few, dense)
    with torch.no_grad():
        normed = block.ln1(x[:, :1])
        pos = torch.full((2, 1), 120, device="cuda")
        q = skv.apply_rotary(block.q_proj(normed).view(2, 1, 4, 64).transpose(1, 2), cos, sin, positions=pos)
        attn = pool.attention(q, keep=4).transpose(1, 2).reshape(2, 1, 256)
        hidden = x[:, :1] + block.o_proj(attn)
        want = hidden + block.down_proj(torch.nn.functional.gelu(block.up_proj(block.ln2(hidden))))
    assert torch.equal(few, want)
