"""Beam selection and reordering on the GPU against plain implementations in 64 bits.

The sum of a row's exponentials is computed in 32 bits: an exponential is off by at most 2^-22 (the instruction's bound)
and |d| 2^-23 (its argument d, weighted by e^-|d|: below 2^-24), sums and rescalings of a thread's 16 values a piece by 2^-24 each.
Averages of such errors stay below 2^-20 in the logarithm; a result is rounded once more.  Continuations that
are nearer than that may change places; all others are where the definition has them.
"""

import math

import pytest
import torch

from test_gpu_paged_pool import PAGE_TYPE, _gen, _pool, skv  # noqa: F401

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]
OFF = 2.0 ** -20


def _continuations(logits, scores, finished, pad):
    """All continuations' scores [B, beams * V] in 64 bits."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    none = torch.full_like(x, -math.inf)
    out = torch.where(x == math.inf, -torch.log((x == math.inf).sum(-1, keepdim=True).double()), none)
    plain = (x < math.inf).all(-1, keepdim=True) & (x > -math.inf).any(-1, keepdim=True)
    # (relative to the largest: next to the type's lowest value 64 bits lose a logarithm)
    less = torch.where(plain, x - torch.where(plain, x, torch.zeros_like(x)).amax(-1, keepdim=True), torch.zeros_like(x))
    out = torch.where(plain, less - torch.log(torch.exp(less).sum(-1, keepdim=True)), out)
    cum = scores.double()[..., None]
    live = cum.isfinite()
    out = torch.where(live & (out > -math.inf), torch.where(live, cum, torch.zeros_like(cum)) + out, none)
    if finished is not None:
        only = none.clone()
        only[..., pad] = torch.where(live[..., 0], scores.double(), -math.inf)
        out = torch.where(finished.bool()[..., None], only, out)
    return out.flatten(1)


def _check(skv, logits, scores, keep, finished=None, pad=0):
    V = logits.shape[2]
    values, parents, tokens = skv.beam_select(logits, scores, keep, finished, pad)
    every = _continuations(logits, scores, finished, pad)
    want, at = (t[:, :keep] for t in torch.sort(every, dim=1, descending=True, stable=True))
    flat = parents * V + tokens
    assert parents.dtype == tokens.dtype == torch.int64 and values.dtype == torch.float32
    assert ((parents >= 0) & (parents < logits.shape[1]) & (tokens >= 0) & (tokens < V)).all()
    assert (flat.sort(1).values.diff(dim=1) > 0).all()                       # no continuation twice
    mine = every.gather(1, flat)
    near = lambda a, b: (a == b) | ((a - b).abs() <= OFF + b.abs() * 2.0 ** -23)   # noqa: E731
    assert near(values.double(), mine).all() and near(mine, want).all()
    # in place, unless a neighbour is too near (or one that was left out)
    padded = torch.sort(every, dim=1, descending=True).values[:, :keep + 1]
    gap = (padded[:, :-1] - padded[:, 1:]).nan_to_num(nan=0.0)
    if padded.shape[1] == keep:
        gap = torch.cat((gap, torch.full_like(gap[:, :1], math.inf)), 1)[:, :keep] if keep > 1 else torch.full_like(want, math.inf)
    clear = (gap > 4 * OFF) & (torch.cat((torch.full_like(gap[:, :1], math.inf), gap[:, :-1]), 1) > 4 * OFF)
    assert (flat == at)[clear].all()
    same = parents[:, 1:] == parents[:, :-1]                                 # a beam's own are exact, ties to the lowest
    wrong = same & ((mine[:, 1:] > mine[:, :-1]) | ((mine[:, 1:] == mine[:, :-1]) & (flat[:, 1:] < flat[:, :-1])))
    assert not wrong.any()
    return values, parents, tokens


BEAM = [  # B, beams, V, keep
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 32000, 4), (3, 2, 4096, 9), (2, 5, 4097, 10), (2, 3, 8191, 128), (5, 3, 40009, 7),
    (1, 1, 300000, 128), (7, 16, 1000, 32), (2, 64, 5000, 64), (1, 1500, 64, 100), (300, 2, 333, 4),
    (37, 2, 4500, 17), (38, 2, 4500, 17), (1, 2, 9000, 32), (3, 2, 70000, 24), (40, 1, 60000, 33), (1, 64, 700, 8), (1, 65, 700, 8), (2, 8, 131072, 16), (25, 8, 70001, 16),
]


@pytest.mark.parametrize("B,beams,V,keep", BEAM)
@pytest.mark.parametrize("dtype", FLOATS)
def test_selection_is_the_definitions(skv, B, beams, V, keep, dtype):
    gen = _gen(V + beams)
    logits = (3 * torch.randn(B, beams, V, generator=gen, device="cuda")).to(dtype)
    scores = -20 * torch.rand(B, beams, generator=gen, device="cuda")
    _check(skv, logits, scores, keep)
    done = torch.rand(B, beams, generator=gen, device="cuda") < 0.4
    _check(skv, logits, scores, keep, done, V - 1)
    _check(skv, logits, scores, keep, done.to(torch.uint8))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("copies", [1, 20])                  # searches of one launch, of two
def test_equal_logits_go_to_the_lowest(skv, dtype, copies):
    """Everything alike, alike but for a few, alike in steps: more candidates than a block's list holds."""
    B, beams, V = 2, 2, 20000
    for case in range(5):
        logits = torch.zeros(B, beams, V, device="cuda", dtype=dtype)
        if case == 1:
            logits[:, :, 12345], logits[:, 1, 19999] = 1.0, 2.0
        if case == 2:
            logits[:] = (torch.arange(V, device="cuda") // 5000).to(dtype)             # better and better
        if case == 3:
            logits[:] = -(torch.arange(V, device="cuda") % 7).to(dtype)
        if case == 4:
            logits[:, 1:] = -0.0
        for keep in (1, 5, 33, 128):
            scores = torch.tensor([[-1.0, -1.0], [-2.0, -5.0]], device="cuda")
            values, parents, tokens = skv.beam_select(logits.repeat(copies, 1, 1), scores.repeat(copies, 1), keep)
            every = _continuations(logits, scores, None, 0)
            at = torch.sort((every * 2 ** 30).round(), dim=1, descending=True, stable=True).indices[:, :keep]
            assert torch.equal(parents * V + tokens, at.repeat(copies, 1)), (case, keep)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("V", [50, 9001])
@pytest.mark.parametrize("copies", [1, 7])                   # searches of one launch, of two
def test_masked_logits_and_beams_that_end(skv, dtype, V, copies):
    """Masks of -inf and of the type's lowest value, rows that nothing is left of, infinities, NaN, scores that are not finite."""
    B, beams = 6, 4
    gen = _gen(V)
    logits = torch.randn(B, beams, V, generator=gen, device="cuda").to(dtype)
    scores = -torch.rand(B, beams, generator=gen, device="cuda")
    logits[0] = -math.inf                                    # nothing at all
    logits[1, :, 3:] = -math.inf                             # 12 continuations, most of them alike in place
    logits[2, 0], logits[2, 1, ::2], logits[2, 2] = math.nan, math.nan, torch.finfo(dtype).min
    logits[2, 3, 5:] = torch.finfo(dtype).min
    logits[3, 1, 7], logits[3, 1, 40], logits[3, 2, 0] = math.inf, math.inf, math.inf
    logits[3, 3] = math.inf
    scores[4] = torch.tensor([0.0, -math.inf, math.nan, math.inf], device="cuda")
    scores[5] = -math.inf
    done = torch.zeros(B, beams, dtype=torch.bool, device="cuda")
    done[1, 2] = done[4, 0] = done[5, 1] = done[3, 1] = True
    logits, scores, done = logits.repeat(copies, 1, 1), scores.repeat(copies, 1), done.repeat(copies, 1)
    for keep in (1, 4, 13, 40, 128):
        _check(skv, logits, scores, keep)
        _check(skv, logits, scores, keep, done, 2)
    values, parents, tokens = skv.beam_select(logits, scores, 5)
    assert (values[0] == -math.inf).all() and (parents[0] == 0).all() and tokens[0].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("dtype", FLOATS)
def test_rows_of_any_alignment_and_stride(skv, dtype):
    gen = _gen(11)
    B, beams, V = 2, 3, 5003
    flat = torch.randn(B * beams * (V + 3) + 40, generator=gen, device="cuda").to(dtype)
    for at in range(1, 9):
        flat[:at], flat[at + V] = 1000.0, 1000.0             # neighbours are not looked at
        x = flat[at:at + B * beams * (V + 3)].view(B, beams, V + 3)[..., :V]
        x[:, :, -1] = torch.linspace(4.0, 6.0, B * beams, device="cuda").view(B, beams).to(dtype)
        x[:, 1, 0] = 5.5
        _check(skv, x, torch.zeros(B, beams, device="cuda"), 6)
    x = torch.randn(beams, B, V, generator=gen, device="cuda").to(dtype)
    _check(skv, x.transpose(0, 1), torch.zeros(B, beams, device="cuda"), 6)
    _check(skv, x[:1, :1].expand(B, beams, V), torch.linspace(0, -3, 6, device="cuda").view(B, beams), 6)
    assert torch.equal(skv.beam_select(x.transpose(1, 2).contiguous().transpose(1, 2), torch.zeros(beams, B, device="cuda"))[2],
                       skv.beam_select(x, torch.zeros(beams, B, device="cuda"))[2])


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("B,beams,V,keep", [(1, 4, 50257, 13), (3, 8, 20001, 24), (2, 5, 333, 40), (40, 4, 20001, 9), (64, 8, 5003, 17), (24, 8, 50257, 16),
                                            (1, 2, 300007, 5), (2, 40, 1003, 128)])
def test_equal_beams_tie_wherever_their_rows_begin(skv, dtype, B, beams, V, keep):
    """Copies of one row with equal scores: the order is that of the logits, then of the beams, exactly."""
    gen = _gen(V)
    for at, pitch in ((0, V), (1, V), (3, V + 2), (0, V + 7), (5, (V + 15) // 8 * 8)):
        row = (3 * torch.randn(B, 1, V, generator=gen, device="cuda")).to(dtype)
        row[:, :, ::7] = -math.inf
        row[0, 0, 5], row[0, 0, 11] = math.nan, -1e-6
        x = torch.full((at + B * beams * pitch,), 1000.0, device="cuda", dtype=dtype)[at:].view(B, beams, pitch)[..., :V]
        x.copy_(row.expand(B, beams, V))
        scores = -torch.rand(B, 1, generator=gen, device="cuda").expand(B, beams)
        values, parents, tokens = skv.beam_select(x, scores, keep)
        every = torch.where(x.isnan(), -math.inf, x.double()).flatten(1)
        assert torch.equal(parents * V + tokens, torch.sort(every, dim=1, descending=True, stable=True).indices[:, :keep])
        # beams that tie have one score, whichever group of lanes added it up
        same = every.gather(1, parents * V + tokens)
        assert ((values[:, 1:] == values[:, :-1]) | (same[:, 1:] < same[:, :-1])).all()
        _check(skv, x, -3 * torch.rand(B, beams, generator=gen, device="cuda"), keep)


@pytest.mark.parametrize("B,V", [(1, 300), (2, 20001), (40, 20001), (40, 20000)])      # searches of one launch, of two
@pytest.mark.parametrize("near", [40, 700])
def test_logits_that_64_bits_do_not_tell_apart(skv, B, V, near):
    """Scores that are equal in 64 bits: a beam's own continuations by their logits, as the lists that are cut have them, behind lower beams'."""
    near = min(near, V)
    gen = _gen(V + near)
    logits = torch.full((B, 2, V), -9.0, device="cuda")
    for b in range(B):
        at = torch.randperm(V, generator=gen, device="cuda")[:near]
        logits[b, :, at] = -1e-20 * torch.rand(2, near, generator=gen, device="cuda")
    for keep in (1, 2, 13, 60, 128):
        order = torch.sort(logits, dim=2, descending=True, stable=True).indices[:, :, :near]   # equal beams: all of the first one's
        want = torch.cat((order[:, 0], order[:, 1] + V), 1)[:, :keep]
        _, parents, tokens = skv.beam_select(logits, torch.zeros(B, 2, device="cuda"), keep)
        n = min(keep, 2 * near)
        assert torch.equal((parents * V + tokens)[:, :n], want[:, :n])
        _, parents, tokens = skv.beam_select(logits, torch.tensor([-50.0, 0.0], device="cuda").expand(B, 2), min(keep, near))
        assert (parents == 1).all() and torch.equal(tokens, order[:, 1, :keep])


@pytest.mark.parametrize("B", [3, 40])                       # one launch, two
def test_selection_in_a_graph_on_streams_and_for_host_tensors(skv, B):
    gen = _gen(12)
    logits, scores = torch.randn(B, 4, 9000, generator=gen, device="cuda"), torch.zeros(B, 4, device="cuda")
    logits.requires_grad_(True)
    want = skv.beam_select(logits, scores)
    assert not want[0].requires_grad
    logits = logits.detach()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(want, skv.beam_select(logits.cpu(), scores.cpu())))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = skv.beam_select(logits, scores)
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = skv.beam_select(logits, scores, 7)
    for _ in range(2):
        logits.copy_(torch.randn(B, 4, 9000, generator=gen, device="cuda"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, skv.beam_select(logits, scores, 7)))


@pytest.mark.parametrize("B,beams,V,keep", [(125, 4, 4096, 5), (125, 4, 2048, 5), (148, 4, 1024, 8), (1, 1, 100000, 3), (2, 16, 33000, 32),
                                            (74, 8, 6144, 16), (1, 4, 512, 4), (32, 8, 70000, 16)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shift", [0, 1])
def test_scratch_is_as_large_as_said(skv, B, beams, V, keep, dtype, shift):
    """Nothing is written behind the scratch's stated size, whatever the rows' type and alignment (which decide how rows are cut)."""
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import beam
    from shadow_infer_b200.shadowkv.rotary import _DTYPE_CODE
    lib = _lib.load()
    pitch = V + 8 if shift == 0 else V + 1
    flat = torch.randn(B * beams * pitch + 1, generator=_gen(V), device="cuda").to(dtype)
    x = flat[shift:shift + B * beams * pitch].view(B, beams, pitch)[..., :V]
    scores = torch.zeros(B, beams, device="cuda")
    need = lib.skv_beam_scratch_bytes(B, beams, V, keep)
    scratch = torch.full((need + (1 << 16),), 77, dtype=torch.uint8, device="cuda")
    values, parents, tokens = torch.empty(B, keep, device="cuda"), *torch.empty(2, B, keep, dtype=torch.int64, device="cuda")
    args = beam._BEAM.pack(x.data_ptr(), x.stride(0), x.stride(1), scores.data_ptr(), 0, values.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                           scratch.data_ptr(), need, _DTYPE_CODE[dtype], B, beams, V, keep, 0)
    assert lib.skv_beam_select(args, torch.cuda.current_stream().cuda_stream) == 0
    assert (scratch[need:] == 77).all()
    want = skv.beam_select(x, scores, keep)
    assert all(torch.equal(a, b) for a, b in zip((values, parents, tokens), want))


def test_more_beams_than_a_merge_holds_entries_for(skv):
    """Searches whose lists do not fit the merge's shared memory: all beams alike, and all different."""
    gen = _gen(5)
    for beams, V, keep in ((4096, 9, 2), (4096, 3, 128), (2000, 40, 5), (64, 300, 128)):
        logits = torch.randn(1, beams, V, generator=gen, device="cuda")
        _check(skv, logits, -30 * torch.rand(1, beams, generator=gen, device="cuda"), keep)
        _check(skv, torch.zeros_like(logits), torch.linspace(0, -1, beams, device="cuda")[None], keep)


def test_selection_from_threads_on_one_stream(skv):
    """A call's launches share a scratch that the stream's other calls use too."""
    import threading

    calls = []
    for seed, (B, beams, V, keep) in enumerate(((4, 4, 30000, 8), (2, 7, 50001, 12), (40, 3, 20001, 12))):   # one launch, two, two of another type
        x = torch.randn(B, beams, V, generator=_gen(seed), device="cuda").to(torch.float16 if seed == 2 else torch.float32)
        calls.append(lambda x=x, keep=keep: skv.beam_select(x, torch.zeros(x.shape[:2], device="cuda"), keep))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(3)

    def work(i):
        go.wait()
        for _ in range(200):
            if not all(torch.equal(a, b) for a, b in zip(calls[i](), want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_empty_batch(skv):
    assert [tuple(t.shape) for t in skv.beam_select(torch.zeros(0, 2, 9, device="cuda"), torch.zeros(0, 2, device="cuda"))] == [(0, 2)] * 3


# ------------------------------------------------------------------------------------------ reordering
def _reordered(table, lengths, parents, P, arrays):
    """The definition, group by group, on host lists; `arrays` are changed in place."""
    G, R = parents.shape
    new_table, new_lengths = [], []
    for g in range(G):
        rows, lens, ps = table[g * R:(g + 1) * R], lengths[g * R:(g + 1) * R], parents[g].tolist()
        childless = [r for r in range(R) if r not in ps]
        extra = 0
        for c, p in enumerate(ps):
            n = lens[p]
            row = rows[p][:-(-n // P)] + rows[c][-(-n // P):]       # entries behind the tokens are each beam's own
            keeper = p if ps[p] == p else ps.index(p)
            if c != keeper:
                j, held = divmod(n, P)
                if held:
                    source, target = row[j], rows[childless[extra]][j]
                    row[j] = target
                    for x in arrays:
                        x[target, :, :held] = x[source, :, :held]
                extra += 1
            new_table.append(row)
            new_lengths.append(n)
    return new_table, new_lengths


REORDER = [  # groups, beams, tokens, H, D, P, G
    (1, 1, 5, 1, 16, 4, 16), (2, 4, 37, 2, 128, 16, 16), (3, 3, 32, 2, 64, 16, 16), (1, 8, 1, 3, 80, 7, 16), (2, 5, 30, 1, 33, 8, 16),
    (1, 40, 11, 2, 64, 8, 32), (1, 300, 3, 1, 8, 2, 8), (2, 2, 0, 1, 16, 4, 16),
]


@pytest.mark.parametrize("groups,beams,tokens,H,D,P,G", REORDER)
@pytest.mark.parametrize("kv", ["fp32", "fp16", "int8", "int4"])
def test_reordering_follows_the_parents(skv, groups, beams, tokens, H, D, P, G, kv):
    gen = _gen(beams * 100 + tokens)
    rows, full = groups * beams, tokens // P
    width = full + 2
    N = groups * full + rows + 1
    order = torch.randperm(N, generator=torch.Generator().manual_seed(tokens)).int()
    table = torch.full((rows, width), -1, dtype=torch.int32)
    table[:, :full] = order[:groups * full].view(groups, 1, full).expand(-1, beams, -1).reshape(rows, full)
    table[:, full] = order[groups * full:groups * full + rows]
    (kp, vp), (sk, sv) = _pool(kv, N, H, P, D, G)
    bounds = torch.randint(-127, 128, (N, H, 2, D), generator=gen, device="cuda", dtype=torch.int8)
    steps = torch.rand(N, H, generator=gen, device="cuda")
    for t in (kp, vp, sk, sv):
        if t is not None:
            t.normal_(generator=gen) if t.dtype.is_floating_point else t.random_(0, 100, generator=gen)
    lengths = torch.full((rows,), tokens, dtype=torch.int32, device="cuda")
    for case in range(6):
        parents = torch.randint(beams, (groups, beams), generator=gen, device="cuda")
        if case == 1:
            parents[:] = torch.arange(beams, device="cuda")
        if case == 2:
            parents[:] = beams - 1
        if case == 3:
            parents[:] = torch.arange(beams, device="cuda").flip(0)
        if case == 4:
            parents = parents.int()
        held = [t for t in (kp, vp, sk, sv) if t is not None]
        before = [t.clone() for t in held]
        same = bounds.clone(), steps.clone()
        # the bounds are those of the pages that were copied
        want_table, want_lengths = _reordered(table.tolist(), lengths.tolist(), parents.cpu(), P, before)
        got = skv.paged_reorder(kp, vp, table.cuda(), lengths, parents, sk, sv, bounds, steps, head_dim=D, check=True)
        assert got[0].tolist() == want_table and got[1].tolist() == want_lengths
        assert all(torch.equal(a, b) for a, b in zip(held, before))
        for r in range(rows):
            p = r // beams * beams + int(parents.flatten()[r])
            if tokens % P:
                mine, theirs = want_table[r][full], int(table[p, full])
                assert torch.equal(bounds[mine], same[0][theirs]) and torch.equal(steps[mine], same[1][theirs])
        assert torch.equal(bounds[table[:, :full].flatten().long().cuda()], same[0][table[:, :full].flatten().long().cuda()])
        # every sequence's last page is its own again
        assert len({row[full] for row in want_table}) == rows


def test_reordering_names_bad_parents_and_pages(skv):
    kp = torch.randn(6, 1, 4, 8, device="cuda")
    table = torch.tensor([[0, 1], [0, 2], [3, 4], [3, 5]], dtype=torch.int32, device="cuda")
    lens = torch.full((4,), 6, dtype=torch.int32, device="cuda")
    for bad in (-1, 2, 2 ** 40):
        parents = torch.tensor([[0, bad], [1, 1]], device="cuda")
        with pytest.raises(ValueError, match="outside"):
            skv.paged_reorder(kp, kp.clone(), table, lens, parents, check=True)
        was = kp.clone()
        t, n = skv.paged_reorder(kp, kp.clone(), table, lens, parents)
        assert t.tolist() == [[0, 1], [-1, -1], [3, 4], [3, 5]] or t.tolist() == [[0, 1], [-1, -1], [3, 5], [3, 4]]
        assert n.tolist() == [6, 0, 6, 6] and torch.equal(kp[[0, 1, 2, 3]], was[[0, 1, 2, 3]])
    # beams of different lengths, of which one has no page to give; a page outside the pool
    for change in ((1, 1, -1), (1, 1, 6), (0, 1, 99)):
        t = table.clone()
        t[change[0], change[1]] = change[2]
        was = kp.clone()
        parents = torch.tensor([[0, 0], [0, 1]], device="cuda")
        with pytest.raises(ValueError, match="outside"):
            skv.paged_reorder(kp, kp.clone(), t, lens, parents, check=True)
        got, _ = skv.paged_reorder(kp, kp.clone(), t, lens, parents)
        assert got[1].tolist() == [0, -1] and torch.equal(kp, was)
    with pytest.raises(ValueError, match="outside"):
        skv.paged_reorder(kp, kp.clone(), table, lens - 20, torch.tensor([[0, 0], [0, 1]], device="cuda"), check=True)
    for wrong in (dict(bounds=torch.zeros(6, 1, 2, 8, dtype=torch.int8, device="cuda")), dict(scale_k=kp)):
        if "bounds" in wrong:
            with pytest.raises(ValueError):
                skv.paged_reorder(kp, kp.clone(), table, lens, torch.zeros(2, 2, dtype=torch.int64, device="cuda"), **wrong)
    with pytest.raises(ValueError):
        skv.paged_reorder(kp, kp.clone(), table, lens, torch.zeros(3, 2, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("beams", [3, 40])                   # a warp's beams, a block's
def test_reordering_leaves_full_pages_of_longer_beams_alone(skv, beams):
    """A beam without children that is longer than a child has a full page, which others share, where the child wants one."""
    kp = torch.randn(2 * beams + 3, 1, 4, 8, generator=_gen(1), device="cuda")
    vp, bounds = kp + 1, torch.randint(-9, 9, (2 * beams + 3, 1, 2, 8), dtype=torch.int8, device="cuda")
    steps = torch.rand(2 * beams + 3, 1, device="cuda")
    # beam 0: 6 tokens in pages 0 and 1; beams 1 and 2: 11 tokens in pages 2 and 3, which they share, and one of their own; the others: 6 tokens
    table = torch.full((beams, 3), -1, dtype=torch.int32)
    lens = torch.full((beams,), 6, dtype=torch.int32)
    table[0, :2] = torch.tensor([0, 1])
    table[1], table[2] = torch.tensor([2, 3, 4]), torch.tensor([2, 3, 5])
    lens[1:3] = 11
    for r in range(3, beams):
        table[r, :2] = torch.tensor([2 * r, 2 * r + 1])
    table, lens = table.cuda(), lens.cuda()
    parents = torch.arange(beams, device="cuda")[None].clone()
    parents[0, 1] = 0                                        # beam 1 goes on from beam 0, beam 2 from itself
    was = [t.clone() for t in (kp, vp, bounds, steps)]
    for check in (False, True):
        if check:
            with pytest.raises(ValueError, match="outside"):
                skv.paged_reorder(kp, vp, table, lens, parents, bounds=bounds, steps=steps, check=True)
        else:
            got, n = skv.paged_reorder(kp, vp, table, lens, parents, bounds=bounds, steps=steps)
            assert got[:3].tolist() == [[0, 1, -1], [0, -1, -1], [2, 3, 5]] and n[:3].tolist() == [6, 6, 11]
            assert torch.equal(got[3:], table[3:])
        assert all(torch.equal(a, b) for a, b in zip(was, (kp, vp, bounds, steps)))
    # a shorter one has its own page there, or one taken ahead
    lens[1] = 5
    got, n = skv.paged_reorder(kp, vp, table, lens, parents, bounds=bounds, steps=steps, check=True)
    assert got[:3].tolist() == [[0, 1, -1], [0, 3, 4], [2, 3, 5]] and n[:3].tolist() == [6, 6, 11]
    assert torch.equal(kp[3, :, :2], was[0][1, :, :2]) and torch.equal(bounds[3], was[2][1])


@pytest.mark.parametrize("precision", ["fp16", "int8", "int4"])
def test_pool_forks_and_reorders(skv, precision):
    """A pool's sequences against one dense copy each: forks, steps of a search, ends, and new sequences in the pages that became free."""
    H, D, P, beams = 2, 32, 4, 3
    pool = skv.PagedKVPool(60, 2 * beams, H, D, max_tokens=64, page_size=P, precision=precision, bounds=True)
    gen = _gen(21)
    dense = [torch.zeros(H, 0, D, device="cuda") for _ in range(2 * beams)]

    def append(new):
        k = torch.randn(2 * beams, H, max(new), D, generator=gen, device="cuda")
        pool.append(k, -k, new_lengths=new)
        for b, n in enumerate(new):
            dense[b] = torch.cat((dense[b], k[b, :, :n]), 1)

    def check():
        counts = [x.shape[1] for x in dense]
        assert pool.token_counts == counts == pool.lengths.tolist()
        k, v = pool.read()
        for b, n in enumerate(counts):
            other = skv.PagedKVPool(20, 1, H, D, 64, P, precision)
            if n:
                other.append(dense[b][None], -dense[b][None])
                want = other.read()
                assert torch.equal(k[b, :, :n], want[0][0]) and torch.equal(v[b, :, :n], want[1][0])
                held = pool.block_table[b, :-(-n // P)].long()
                mine = skv.page_bounds(other.k_pages, other.block_table, other.lengths, other.scale_k)
                ids = other.block_table[0, :-(-n // P)].long()
                assert torch.equal(pool.bounds[held], mine[0][ids]) and torch.equal(pool.steps[held], mine[1][ids])

    free = pool.free_pages
    for start in (10, 8, 3):
        append([start, 0, 0, 5, 0, 0])
        check()
        pool.fork(0, [1, 2])
        pool.fork(3, [4])
        dense[1] = dense[2] = dense[0]
        dense[4] = dense[3]
        append([0, 0, 0, 0, 0, 5])
        check()
        for step in range(9):
            append([1] * 6)
            parents = torch.randint(beams, (2, beams), generator=gen, device="cuda")
            if len({dense[3].shape[1], dense[4].shape[1], dense[5].shape[1]}) == 1:
                pool.reorder(parents, check=step % 2 == 0)
                dense = [dense[g * beams + int(parents[g, c])] for g in range(2) for c in range(beams)]
            check()
        assert pool.release(1) == 0 and pool.free_pages < free          # its pages may be the others'
        dense[1] = dense[1][:, :0]
        check()
        with pytest.raises(ValueError, match="equally long"):
            pool.reorder(torch.zeros(2, beams, dtype=torch.int64, device="cuda"))
        for b in (0, 2, 3, 4, 5):
            pool.release(b)
            dense[b] = dense[b][:, :0]
        assert pool.free_pages == free
        check()


def _same_as_dense(pool, dense):
    counts = [x.shape[1] for x in dense]
    assert pool.token_counts == counts == pool.lengths.tolist()
    k, _ = pool.read()
    assert all(torch.equal(k[b, :, :n], x) for b, (n, x) in enumerate(zip(counts, dense)))


def test_forks_that_end_return_their_pages(skv):
    """A prefix that stays, forked for one request after another: what a request took is free again when it ends."""
    H, D, P, B = 2, 16, 4, 4
    for prefix in (7, 8):                                    # a last page that is partly filled, or none
        pool = skv.PagedKVPool(12, B, H, D, max_tokens=32, page_size=P, precision="fp32", bounds=True)
        gen = _gen(prefix)
        dense = [torch.zeros(H, 0, D, device="cuda") for _ in range(B)]

        def append(new):
            k = torch.randn(B, H, max(new), D, generator=gen, device="cuda")
            pool.append(k, -k, new_lengths=new)
            for b, n in enumerate(new):
                dense[b] = torch.cat((dense[b], k[b, :, :n]), 1)
            _same_as_dense(pool, dense)

        append([prefix, 0, 0, 0])
        free = pool.free_pages
        for _ in range(8):
            pool.fork(0, [1, 2])
            dense[1] = dense[2] = dense[0]
            append([0, 5, 1, 0])
            pool.fork(1, [3])                                # a request's own fork, which outlives it
            dense[3] = dense[1]
            _same_as_dense(pool, dense)
            held = {p for b in (0, 2, 3) for p in pool.block_table[b].tolist() if p >= 0}
            own = [p for p in pool.block_table[1].tolist() if p >= 0 and p not in held]
            was = pool.free_pages
            assert pool.release(1) == len(own) == pool.free_pages - was
            dense[1] = dense[1][:, :0]
            append([0, 4, 0, 3])                             # in the pages that became free
            for b in (3, 1, 2):
                pool.release(b)
                dense[b] = dense[b][:, :0]
            assert pool.free_pages == free
            _same_as_dense(pool, dense)
            assert torch.equal(pool.block_table.cpu(), pool._table)   # (which appends copy as long as nothing was reordered)
        pool.fork(0, [1])
        assert pool.release(0) == prefix % P // 3 and pool.release(1) == 2 and pool.free_pages == 12


@pytest.mark.parametrize("order", [(0, 1, 2, 3, 4, 5), (5, 4, 3, 2, 1, 0), (3, 0, 4, 2, 5, 1)])
def test_searches_that_share_a_prompt_end_one_by_one(skv, order):
    """Two searches of one prompt (rows 0 and 1, rows 2 and 3) and a fork of a beam of each (4, 5): no page is free that a sequence reads."""
    H, D, P, B = 1, 16, 4, 6
    gen = _gen(8)
    pool = skv.PagedKVPool(40, B, H, D, max_tokens=48, page_size=P, precision="fp32")
    dense = [torch.zeros(H, 0, D, device="cuda") for _ in range(B)]

    def append(new):
        k = torch.randn(B, H, max(new), D, generator=gen, device="cuda")
        pool.append(k, -k, new_lengths=new)
        for b, n in enumerate(new):
            dense[b] = torch.cat((dense[b], k[b, :, :n]), 1)
        check()

    def check():
        for p in pool._free:
            pool.k_pages[p] = math.nan
        _same_as_dense(pool, dense)

    append([9, 0, 0, 0, 0, 0])
    pool.fork(0, [1, 2, 3])
    dense[1] = dense[2] = dense[3] = dense[0]
    for parents in ([[1, 1], [0, 1], [0, 0]], [[0, 0], [1, 0], [1, 1]], [[1, 0], [1, 1], [0, 1]]):
        append([3, 3, 3, 3, 0, 0])
        pool.reorder(torch.tensor(parents, device="cuda"))
        dense = [dense[2 * g + p] for g, ps in enumerate(parents) for p in ps]
        check()
    pool.fork(1, [4])
    pool.fork(3, [5])
    dense[4], dense[5] = dense[1], dense[3]
    append([1, 0, 2, 0, 3, 6])
    for b in order:
        pool.release(b)
        dense[b] = dense[b][:, :0]
        check()
    assert sorted(pool._free) == list(range(40))
    append([5, 1, 0, 9, 4, 4])
    assert pool.release(4) == 1 and pool.release(3) == 3


def test_pool_fork_refusals(skv):
    pool = skv.PagedKVPool(4, 4, 1, 8, max_tokens=16, page_size=4)
    x = torch.randn(4, 1, 6, 8, device="cuda")
    pool.append(x, x, new_lengths=[6, 1, 0, 0])

    def unchanged(error, *args):
        was = pool.block_table.clone(), pool.lengths.clone(), pool.free_pages, list(pool.token_counts)
        with pytest.raises(error):
            pool.fork(*args)
        assert torch.equal(was[0], pool.block_table) and torch.equal(was[1], pool.lengths)
        assert was[2:] == (pool.free_pages, pool.token_counts)

    unchanged(ValueError, 0, [1])
    unchanged(ValueError, 0, [0])
    unchanged(ValueError, 0, [2, 2])
    unchanged(ValueError, 0, [2, -2])
    unchanged(RuntimeError, 0, [2, 3])
    with pytest.raises(IndexError):
        pool.fork(0, [4])
    pool.fork(2, [3])                      # nothing to share
    pool.fork(0, [])
    pool.fork(0, [2])
    assert pool.token_counts == [6, 1, 6, 0] and pool.free_pages == 0
    for wrong in (torch.zeros(4, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.int64)):
        with pytest.raises(ValueError):
            pool.reorder(wrong.cuda())
    with pytest.raises(ValueError, match="outside"):
        skv.PagedKVPool(4, 2, 1, 8, 16).reorder(torch.tensor([[0, 2]], device="cuda"), check=True)


def test_search_step_does_not_wait_for_the_gpu(skv):
    pool = skv.PagedKVPool(64, 4, 2, 32, max_tokens=128, page_size=8, precision="int8", bounds=True)
    x = torch.randn(4, 2, 11, 32, generator=_gen(1), device="cuda")
    logits = torch.randn(1, 4, 1000, generator=_gen(2), device="cuda")

    def steps():
        pool.append(x, x, new_lengths=[11, 0, 0, 0])
        pool.fork(0, [1, 2, 3])
        scores = torch.zeros(1, 4, device="cuda")
        for _ in range(3):
            pool.append(x[:, :, :1], x[:, :, :1])
            pool.attention(x[:, :, :1], keep=2)
            scores, parents, _ = skv.beam_select(logits, scores)
            pool.reorder(parents)
        for b in range(4):
            pool.release(b)

    steps()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        steps()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert pool.free_pages == 64


def test_search_through_a_block(skv):
    """A search over a small model's block: its beams' pages give the attention that each beam's own tokens give."""
    H, D, V, beams, B, steps = 2, 32, 101, 3, 2, 6
    torch.manual_seed(3)
    embed, to_logits = torch.randn(V, H * D, device="cuda"), torch.randn(H * D, V, device="cuda") / 4

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.hidden_dim, self.num_heads, self.head_dim = H * D, H, D
            self.ln1, self.ln2 = torch.nn.LayerNorm(H * D), torch.nn.LayerNorm(H * D)
            for name in ("q_proj", "k_proj", "v_proj", "o_proj", "up_proj", "down_proj"):
                setattr(self, name, torch.nn.Linear(H * D, H * D))

    block = Block().cuda()
    cos, sin = skv.rotary_tables(D, 64)
    prompt = torch.randint(V, (B, 9), generator=_gen(1), device="cuda")
    with torch.no_grad():
        pool = skv.PagedKVPool(80, B * beams, H, D, max_tokens=32, page_size=4, precision="fp32")
        wide = torch.zeros(B * beams, 9, H * D, device="cuda")
        wide[::beams] = embed[prompt]
        first = [9 if b % beams == 0 else 0 for b in range(B * beams)]
        hidden = skv.paged_block_forward(block, wide, pool, cos, sin, causal=True, new_lengths=first)
        for g in range(B):
            pool.fork(g * beams, [g * beams + 1, g * beams + 2])
        logits = (hidden[::beams, -1:] @ to_logits).expand(B, beams, V)
        scores = torch.tensor([0.0] + [-math.inf] * (beams - 1), device="cuda").expand(B, beams)
        history = prompt[:, None].expand(B, beams, 9)
        for _ in range(steps):
            scores, parents, tokens = skv.beam_select(logits, scores)
            pool.reorder(parents)
            history = torch.cat((history.gather(1, parents[..., None].expand_as(history)), tokens[..., None]), -1)
            hidden = skv.paged_block_forward(block, embed[tokens].view(B * beams, 1, H * D), pool, cos, sin)
            logits = (hidden[:, 0] @ to_logits).view(B, beams, V)
            # every beam by itself, from its tokens
            alone = skv.PagedKVPool(80, B * beams, H, D, max_tokens=32, page_size=4, precision="fp32")
            want = skv.paged_block_forward(block, embed[history].flatten(0, 1), alone, cos, sin, causal=True)[:, -1]
            assert (hidden[:, 0] - want).abs().max() < 1e-4 * want.abs().max()
    assert len({tuple(h) for h in history[0].tolist()}) == beams
