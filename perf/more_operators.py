"""Operators of serving from a page pool beyond dense attention: which pages a query reads, and which sequences go on.

Four operators over plain tensors:

* ``bounds``   the least and the largest value of every channel of a page's keys, in 8 bits with one
               power-of-two step for a page and head, rounded outwards;
* ``sparse``   for every query the pages whose keys may score highest by those bounds (the first and the
               newest pages always among them), and attention over the tokens of these pages;
* ``beam``     the best continuations of all beams of a sequence over the vocabulary;
* ``reorder``  beams go on from their parents: block tables follow them, pages that are full are shared, and a last
               page that several go on from is copied.

``run`` computes them in elementary torch operations in 32 bits (log-probabilities that are ranked: in 64), or, where
``own`` is true, through ``shadow_infer_b200.shadowkv``.  ``exact`` holds the definitions in 64 bits.
"""

import math
import random

import torch

own = False

_TYPE = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
GROUP = 16  # values that share one int4 scale


def listed():
    return [
        # a long prompt has been written: the bounds of all its pages
        dict(name="bounds_prompt_fp16", op="bounds", B=1, lo=32768, hi=32768, new=32768, Hk=32, D=128, page=32, kv="fp16"),
        # a decoding step: the page that each sequence's newest token fell into, bound by latency
        dict(name="bounds_token_int8", op="bounds", B=8, lo=1, hi=2048, new=1, Hk=8, D=128, page=32, kv="int8"),
        # one token of a long int4 sequence, a key head for every query head, a sixteenth of the pages
        dict(name="sparse_long_int4", op="sparse", B=1, Sq=1, lo=32768, hi=32768, Hk=32, rep=1, D=128, page=32, keep=64,
             first=1, recent=2, kv="int4", dtype="fp16", causal=False),
        # the longest sequence, shared key heads, int8, 32-bit queries and outputs
        dict(name="sparse_longest_int8", op="sparse", B=1, Sq=1, lo=131071, hi=131071, Hk=8, rep=4, D=128, page=64, keep=64,
             first=1, recent=1, kv="int8", dtype="fp32", causal=False),
        # a full serving batch, the largest call: short sequences keep all of their pages
        dict(name="sparse_full_fp16", op="sparse", B=64, Sq=1, lo=64, hi=8192, Hk=8, rep=4, D=128, page=32, keep=32,
             first=1, recent=2, kv="fp16", dtype="bf16", causal=False),
        # a block of new tokens, each with pages of its own
        dict(name="sparse_block_int8", op="sparse", B=4, Sq=16, lo=1024, hi=4096, Hk=8, rep=4, D=128, page=32, keep=16,
             first=1, recent=1, kv="int8", dtype="bf16", causal=True),
        # odd everything: empty sequences, a page size and a head size that divide nothing, 32-bit pages
        dict(name="sparse_odd_fp32", op="sparse", B=5, Sq=3, lo=0, hi=777, Hk=3, rep=3, D=80, page=7, keep=11,
             first=0, recent=1, kv="fp32", dtype="fp32", causal=True),
        # the smallest search: four beams of one sequence
        dict(name="beam_one_fp32", op="beam", B=1, beams=4, V=32000, keep=4, dtype="fp32", masked=False, ended=False),
        # a batch of searches over a large vocabulary, with spare candidates for beams that end
        dict(name="beam_batch_bf16", op="beam", B=32, beams=8, V=131072, keep=16, dtype="bf16", masked=False, ended=True),
        # odd sizes, most of the vocabulary not allowed, a beam to which nothing is
        dict(name="beam_odd_fp16", op="beam", B=5, beams=3, V=40009, keep=7, dtype="fp16", masked=True, ended=True),
        # one step of a search over 8 sequences
        dict(name="reorder_step_fp16", op="reorder", groups=8, beams=4, tokens=1001, Hk=8, D=128, page=32, kv="fp16"),
        # a large batch in large pages, odd heads, int8 with scales
        dict(name="reorder_batch_int8", op="reorder", groups=32, beams=8, tokens=1983, Hk=10, D=128, page=64, kv="int8"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _drawn(rng):
    op = rng.choice(["bounds", "sparse", "sparse", "sparse", "beam", "beam", "reorder"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "beam":
        beams = _log(rng, 1, 16)
        V = _log(rng, 500, 131072)
        return dict(op=op, B=_log(rng, 1, 32), beams=beams, V=V, keep=rng.choice([beams, 2 * beams, _log(rng, 1, 32)]),
                    dtype=dtype, masked=rng.random() < 0.4, ended=rng.random() < 0.5)
    pool = dict(Hk=rng.choice([1, 2, 3, 5, 8, 8, 16, 32]), D=rng.choice([64, 128, 128, 128, 96, 80, 256]),
                page=rng.choice([16, 32, 32, 64, 7, 17, 128]), kv=rng.choice(["fp32", "fp16", "fp16", "int8", "int8", "int4", "int4"]))
    if op == "reorder":
        return dict(op=op, groups=_log(rng, 1, 32), beams=_log(rng, 2, 16), tokens=_log(rng, 1, 4096), **pool)
    B, hi = _log(rng, 1, 64), _log(rng, 1, 131072)
    lo = hi if B == 1 else rng.choice([0, 1, hi // 2, hi])
    if op == "bounds":
        return dict(op=op, B=B, lo=lo, hi=hi, new=rng.choice([1, _log(rng, 1, hi), hi]), **pool)
    recent, first = rng.choice([1, 1, 2, 4]), rng.choice([0, 1, 1, 2])
    return dict(op=op, B=B, Sq=rng.choice([1, 1, 1, 2, 5, 16, 31]), lo=lo, hi=hi, rep=rng.choice([1, 1, 2, 3, 4, 4, 7, 8]),
                keep=max(recent + first, _log(rng, 1, 128)), first=first, recent=recent, dtype=dtype,
                causal=rng.random() < 0.4, **pool)


def draw(rng):
    """One more case: sizes over the listed ones' ranges, drawn again until it costs no more than the largest of them."""
    while True:
        case = _drawn(rng)
        cost = work(case)
        most = [work(c) for c in listed() if c["op"] == case["op"]]
        if (all(cost[n] <= max(m[n] for m in most) for n in cost)
                and _pool_values(case) <= max(_pool_values(c) for c in listed() if c["op"] in (case["op"], "bounds"))):
            return case


def _pool_values(case):
    """Values of the keys (or logits) that the inputs hold."""
    if case["op"] == "beam":
        return case["B"] * case["beams"] * case["V"]
    if case["op"] == "reorder":
        return case["groups"] * (case["tokens"] + case["beams"] * case["page"]) * case["Hk"] * case["D"]
    return sum(_lengths(case)) * case["Hk"] * case["D"]


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """The sequences' lengths, from `lo` to `hi`: the same for every seed, so that the work is."""
    lo, hi, B = case["lo"], case["hi"], case["B"]
    rng = random.Random(lo * 1000003 + hi * 101 + B)
    return [hi] + [rng.randint(lo, hi) for _ in range(B - 2)] + ([lo] if B > 1 else [])


def _fill(case, gen, N):
    """N pages of keys and values in the case's precision, and their scales."""
    P, H, D, kv = case["page"], case["Hk"], case["D"], case["kv"]
    s = {}
    for name in ("k", "v"):
        x = torch.randn(N, H, P, D, generator=gen, device="cuda", dtype=torch.float32 if kv == "fp32" else torch.float16)
        if name == "k":  # a few channels of K are larger, and neighbouring tokens' keys are alike
            x[..., :: max(1, D // 4)] *= 3.0
            x += torch.randn(N, H, 1, D, generator=gen, device="cuda", dtype=x.dtype)
        scale = None
        if kv in ("int8", "int4"):
            g = x.view(N, H, P, -1, GROUP if kv == "int4" else D)
            scale = g.abs().amax(-1, keepdim=True).float() / (7.0 if kv == "int4" else 127.0)
            x = (g / scale).round_().to(torch.int8).view(N, H, P, D)
            if kv == "int4":
                x = (x + 8).to(torch.uint8)
                x = x[..., 0::2] * 16 + x[..., 1::2]
            else:
                scale = scale.view(N, H, P, 1)
        s[name + "_pages"], s["scale_" + name] = x, scale
    return s


def _pages(case, gen):
    """Pages in shuffled order, their table, and NaN in the rows past each sequence's end."""
    counts, P = _lengths(case), case["page"]
    per = [-(-n // P) for n in counts]
    N, M = sum(per) + 3, max(per) + 1
    order = torch.randperm(N, generator=torch.Generator().manual_seed(gen.initial_seed())).tolist()
    table, used, at = torch.full((len(per), M), -1, dtype=torch.int32), torch.zeros(N, P, dtype=torch.bool), 0
    for b, n in enumerate(per):
        ids = order[at:at + n]
        at += n
        if n:
            table[b, :n] = torch.tensor(ids, dtype=torch.int32)
            used[ids] = True
            used[ids[-1]] = torch.arange(P) < counts[b] - (n - 1) * P
    s = _fill(case, gen, N)
    unused = ~used.cuda()
    for name in ("k", "v"):
        x = s["scale_" + name] if s["scale_" + name] is not None else s[name + "_pages"]
        x.masked_fill_(unused.view(N, 1, P, *[1] * (x.dim() - 3)), math.nan)
    s["block_table"], s["lengths"] = table.cuda(), torch.tensor(counts, dtype=torch.int32, device="cuda")
    return s, used.cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "beam":
        B, beams, V = case["B"], case["beams"], case["V"]
        x = 3.0 * torch.randn(B, beams, V, generator=gen, device="cuda")
        if case["masked"]:
            banned = torch.rand(B, 1, V, generator=gen, device="cuda") < 0.9
            x.masked_fill_(banned, -math.inf)
            x[0, 0] = -math.inf
        s = {"logits": x.to(_TYPE[case["dtype"]]),
             "scores": -10.0 * torch.rand(B, beams, generator=gen, device="cuda"), "finished": None}
        if case["ended"]:
            s["finished"] = torch.rand(B, beams, generator=gen, device="cuda") < 0.2
    elif case["op"] == "reorder":
        G, R, P, L = case["groups"], case["beams"], case["page"], case["tokens"]
        full, M = L // P, -(-L // P) + 1
        own_pages = L % P > 0   # beams share the pages that are full; a last page that is not is each beam's own
        N = G * (full + R) + 3
        order = torch.randperm(N, generator=torch.Generator().manual_seed(gen.initial_seed())).int()
        table = torch.full((G, R, M), -1, dtype=torch.int32)
        table[:, :, :full] = order[:G * full].view(G, 1, full)
        if own_pages:
            table[:, :, full] = order[G * full:G * (full + R)].view(G, R)
        s = _fill(case, gen, N)
        s["block_table"] = table.view(G * R, M).cuda()
        s["lengths"] = torch.full((G * R,), L, dtype=torch.int32, device="cuda")
        s["parents"] = torch.randint(R, (G, R), generator=gen, device="cuda")
    else:
        s, used = _pages(case, gen)
        N = used.shape[0]
        if case["op"] == "bounds":
            s["start"] = (s["lengths"] - case["new"]).clamp_min(0)
            s["bounds"] = torch.zeros(N, case["Hk"], 2, case["D"], dtype=torch.int8, device="cuda")
            s["steps"] = torch.ones(N, case["Hk"], device="cuda")
        else:
            s["bounds"], s["steps"] = _bounds_of(s["k_pages"], s["scale_k"], used)
            s["q"] = torch.randn(case["B"], case["Sq"], case["Hk"] * case["rep"], case["D"], generator=gen,
                                 device="cuda").to(_TYPE[case["dtype"]]).transpose(1, 2)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------- the plain forms
def _values(pages, scale):
    """What page rows stand for, in 32 bits."""
    if pages.dtype == torch.uint8:
        x = torch.stack((pages >> 4, pages & 15), -1).flatten(-2).float() - 8.0
        return (x.unflatten(-1, (scale.shape[-2], -1)) * scale).flatten(-2)
    return pages.float() if scale is None else pages.float() * scale


def _step(top):
    """The least power of two of which 127 reach `top` (one where it is zero)."""
    m, e = torch.frexp(top)   # top = m 2^e, m in [0.5, 1)
    e = torch.where(m * 128.0 <= 127.0, e - 7, e - 6).clamp_min(-126)
    return torch.where(top == 0, torch.ones_like(top), torch.ldexp(torch.ones_like(top), e))


def _bounds_of(k_pages, scale, held):
    """Bounds [N, H, 2, D] and steps [N, H] of pages whose rows `held` [N, P] are tokens."""
    x = _values(k_pages, scale)
    there = held[:, None, :, None]
    inf = torch.full((), math.inf, device=x.device)
    low, high = torch.where(there, x, inf).amin(2), torch.where(there, x, -inf).amax(2)
    empty = ~held.any(1)[:, None, None]
    low, high = low.masked_fill(empty, 0.0), high.masked_fill(empty, 0.0)
    step = _step(torch.maximum(-low, high).amax(-1).clamp_min(0))[..., None]
    return torch.stack((torch.floor(low / step), torch.ceil(high / step)), 2).to(torch.int8), step[..., 0]


def _bounds(s):
    case, P = s["case"], s["case"]["page"]
    table, lens = s["block_table"].long(), s["lengths"].long()
    j = torch.arange(table.shape[1], device="cuda")
    touched = (j >= (s["start"].long() // P)[:, None]) & (j * P < lens[:, None]) & (s["start"].long() < lens)[:, None]
    page = table[touched]
    held = (j[:, None] * P + torch.arange(P, device="cuda") < lens[:, None, None])[touched]
    scale = None if s["scale_k"] is None else s["scale_k"][page]
    s["bounds"][page], s["steps"][page] = _bounds_of(s["k_pages"][page], scale, held)
    return [s["bounds"], s["steps"]]


def _seen(s):
    """Tokens that each query sees [B, Sq]."""
    Sq, lens = s["case"]["Sq"], s["lengths"].long()
    i = torch.arange(Sq, device="cuda")
    return (lens[:, None] - Sq + 1 + i if s["case"]["causal"] else lens[:, None] + 0 * i).clamp_min(0)


def _select(s):
    case = s["case"]
    B, Hk, rep, Sq, P, keep = (case[n] for n in ("B", "Hk", "rep", "Sq", "page", "keep"))
    table = s["block_table"].long().clamp_min(0)
    M = table.shape[1]
    q = s["q"].float().reshape(B, Hk, rep * Sq, -1)
    t = _step(q.abs().amax(-1))
    n = torch.round(q / t[..., None])
    low, high = (s["bounds"][table][:, :, :, i].float().permute(0, 2, 3, 1) for i in (0, 1))   # [B, Hk, D, M]
    dots = n.clamp_min(0) @ high + n.clamp_max(0) @ low    # whole numbers below 2^24
    score = dots * t[..., None] * s["steps"][table].transpose(1, 2)[:, :, None]
    score = score.view(B, Hk, rep, Sq, M).amax(2)
    pages = ((_seen(s) + P - 1) // P)[:, None, :, None]
    j = torch.arange(M, device="cuda")
    score = torch.where((j < case["first"]) | (j >= pages - case["recent"]), torch.full((), math.inf, device="cuda"), score)
    score = torch.where(j < pages, score, torch.full((), -math.inf, device="cuda"))
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    if M < keep:
        best = torch.cat((best, best.new_full((*best.shape[:-1], keep - M), M)), -1)
    best = torch.where(best < pages, best, torch.full((), 1 << 30, device="cuda", dtype=torch.long)).sort(-1).values
    return torch.where(best < pages, best, torch.full((), -1, device="cuda", dtype=torch.long)).int()


def _sparse(s):
    case = s["case"]
    B, Hk, rep, Sq, P, D = (case[n] for n in ("B", "Hk", "rep", "Sq", "page", "D"))
    pages = _select(s)
    listed_ = pages.long().clamp_min(0)
    physical = s["block_table"].long().clamp_min(0)[:, None, None, :].expand(B, Hk, Sq, -1).gather(-1, listed_)
    head = torch.arange(Hk, device="cuda").view(1, Hk, 1, 1)
    token = listed_[..., None] * P + torch.arange(P, device="cuda")
    seen = (pages >= 0)[..., None] & (token < _seen(s)[:, None, :, None, None])
    past = []
    for n in ("k", "v"):
        scale = s["scale_" + n]
        x = _values(s[n + "_pages"][physical, head], None if scale is None else scale[physical, head])
        past.append(torch.where(seen[..., None], x, torch.zeros((), device="cuda")).flatten(3, 4))
    q = s["q"].float().view(B, Hk, rep, Sq, D).transpose(2, 3)
    score = (q @ past[0].transpose(-1, -2)) * (1.0 / math.sqrt(D))
    score = torch.where(seen.flatten(3)[:, :, :, None], score, torch.full((), -math.inf, device="cuda"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ past[1]) / torch.where(total == 0, torch.ones_like(total), total)
    return [pages, out.transpose(2, 3).reshape(B, Hk * rep, Sq, D).to(s["q"].dtype)]


def _beam(s):
    case = s["case"]
    V, keep = case["V"], case["keep"]
    none = torch.full((), -math.inf, dtype=torch.float64, device="cuda")
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    shift = torch.where(top == -math.inf, torch.zeros_like(top), top)
    total = torch.exp(x - shift).sum(-1, keepdim=True)
    score = s["scores"].double()[..., None] + (x - shift - torch.log(total))
    score = torch.where(x == -math.inf, none, score)
    if s["finished"] is not None:
        only = torch.where(torch.arange(V, device="cuda") == 0, s["scores"].double()[..., None], none)
        score = torch.where(s["finished"][..., None], only, score)
    value, at = (t[:, :keep] for t in torch.sort(score.flatten(1), dim=1, descending=True, stable=True))
    return [value.float(), at // V, at % V]


def _reorder(s):
    case = s["case"]
    G, R, P, L = case["groups"], case["beams"], case["page"], case["tokens"]
    old = s["block_table"].view(G, R, -1)
    parents = s["parents"]
    table = old.gather(1, parents[..., None].expand_as(old)).clone()
    j, rows = L // P, L % P
    if rows:
        me = torch.arange(R, device="cuda")
        child = parents[:, None, :] == me[:, None]                       # [G, parent, child]
        # the child that keeps its parent's last page: the parent itself, else the first
        rank = torch.where(torch.eye(R, dtype=torch.bool, device="cuda"), -1, me.expand(R, R))
        rank = torch.where(child, rank, R)
        keeper = rank.argmin(-1)                                        # [G, parent]
        extra = keeper.gather(1, parents) != me                         # [G, child]
        dropped = ~child.any(-1)                                        # [G, row]
        g, c = extra.nonzero(as_tuple=True)                             # both in ascending order: the n-th extra child
        g2, d = dropped.nonzero(as_tuple=True)                          # takes the last page of the n-th dropped beam
        source, target = old[g, parents[g, c], j].long(), old[g2, d, j].long()
        table[g, c, j] = target.int()
        for n in ("k", "v"):
            s[n + "_pages"][target, :, :rows] = s[n + "_pages"][source, :, :rows]
            if s["scale_" + n] is not None:
                s["scale_" + n][target, :, :rows] = s["scale_" + n][source, :, :rows]
    lengths = s["lengths"].view(G, R).gather(1, parents).view(-1)
    return [table.view(G * R, -1), lengths] + [s[n] for n in ("k_pages", "v_pages", "scale_k", "scale_v") if s[n] is not None]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"bounds": _bounds, "sparse": _sparse, "beam": _beam, "reorder": _reorder}[op](s)
    from shadow_infer_b200 import shadowkv

    case = s["case"]
    if op == "beam":
        return list(shadowkv.beam_select(s["logits"], s["scores"], case["keep"], finished=s["finished"], pad_token=0))
    if op == "bounds":
        return list(shadowkv.page_bounds(s["k_pages"], s["block_table"], s["lengths"], scale_k=s["scale_k"], start=s["start"],
                                         bounds=s["bounds"], steps=s["steps"]))
    if op == "reorder":
        out = shadowkv.paged_reorder(s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], s["parents"],
                                     scale_k=s["scale_k"], scale_v=s["scale_v"])
        return list(out) + [s[n] for n in ("k_pages", "v_pages", "scale_k", "scale_v") if s[n] is not None]
    pages = shadowkv.page_select(s["q"], s["bounds"], s["steps"], s["block_table"], s["lengths"], case["page"], case["keep"],
                                 first=case["first"], recent=case["recent"], causal=case["causal"])
    out = shadowkv.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], scale_k=s["scale_k"],
                                   scale_v=s["scale_v"], causal=case["causal"], pages=pages)
    return [pages, out]


# --------------------------------------------------------------------------------------- what it costs
def _row_bytes(kv, D):
    """Bytes of one page row and its scales."""
    return {"fp32": 4 * D, "fp16": 2 * D, "int8": D + 4, "int4": D // 2 + D // GROUP * 4}[kv]


def work(case):
    if case["op"] == "beam":
        rows, keep = case["B"] * case["beams"], case["keep"]
        return {"bytes": rows * case["V"] * _BYTES[case["dtype"]] + rows * 5 + case["B"] * keep * 20,
                "flops": 3 * rows * case["V"]}
    H, D, P = case["Hk"], case["D"], case["page"]
    row = _row_bytes(case["kv"], D)
    if case["op"] == "reorder":
        G, R, L = case["groups"], case["beams"], case["tokens"]
        copied = R * (1.0 - 1.0 / R) ** R    # beams that no other goes on from, on average
        return {"bytes": int(G * copied * 2 * 2 * H * (L % P) * row) + 2 * 4 * G * R * (-(-L // P) + 1) + 12 * G * R, "flops": 0}
    if case["op"] == "bounds":
        b, values = 8 * case["B"], 0
        for n in _lengths(case):
            j = max(0, n - case["new"]) // P     # the first page that is looked at
            rows, pages = n - j * P, -(-n // P) - j
            b += 4 * pages + H * (rows * row + pages * (2 * D + 4))
            values += H * rows * D
        return {"bytes": b, "flops": 2 * values}
    B, Sq, rep, keep, e = case["B"], case["Sq"], case["rep"], case["keep"], _BYTES[case["dtype"]]
    b, flops = 4 * B * (1 + H * Sq * keep) + 2 * B * Sq * H * rep * D * e, 0
    for n in _lengths(case):
        total, most = -(-n // P), 0
        b += 4 * total
        if total > keep:
            b += total * H * (2 * D + 4)
        for i in range(Sq):
            seen = max(0, n - Sq + 1 + i) if case["causal"] else n
            pages = -(-seen // P)
            read = seen if pages <= keep else seen - (pages - keep) * P
            most = max(most, read)
            flops += H * rep * (4 * read * D + (4 * pages * D if pages > keep else 0))
        b += 2 * H * most * row     # queries of one block may read the same pages
    return {"bytes": b, "flops": flops}


# ------------------------------------------------------------------------- the definitions in 64 bits
def _held(pages, scale, ids, head=None):
    """Tokens [n * P, H, D] (or [n * P, D] of one head) of the pages `ids`, in 64 bits."""
    x, scale = (pages[ids], scale if scale is None else scale[ids]) if head is None else (
        pages[ids, head:head + 1], scale if scale is None else scale[ids, head:head + 1])
    if scale is None:
        x = x.double()
    elif x.dtype == torch.int8:
        x = x.double() * scale.double()
    else:
        n = torch.stack((x.int().div(16, rounding_mode="floor"), x.int() % 16), -1) - 8
        x = (n.reshape(*x.shape[:-1], -1, GROUP).double() * scale.double()).reshape(*x.shape[:-1], -1)
    x = x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])
    return x if head is None else x[:, 0]


def _power(top):
    """2 to the least exponent with 127 * 2^e >= top, found by its logarithm; 1 for zero."""
    safe = torch.where(top > 0, top, torch.ones_like(top))
    e = torch.ceil(torch.log2(safe / 127.0)).clamp_min(-126)
    e = torch.where(127.0 * torch.exp2(e - 1) >= safe, e - 1, e).clamp_min(-126)
    e = torch.where(127.0 * torch.exp2(e) < safe, e + 1, e)
    return torch.where(top > 0, torch.exp2(e), torch.ones_like(top))


def _exact_bounds(s, case):
    P = case["page"]
    bounds, steps = s["bounds"].clone(), s["steps"].clone()
    for b, n in enumerate(_lengths(case)):
        first, last = max(0, n - case["new"]) // P, -(-n // P)
        if last == first:
            continue
        ids = s["block_table"][b, first:last].long()
        # what a cache holds is a 32-bit product
        x = _held(s["k_pages"], s["scale_k"], ids).float().double()
        x = torch.cat((x[:n - first * P], x[:n - first * P][-1:].expand(last * P - n, -1, -1))).unflatten(0, (last - first, P))
        low, high = x.min(1).values, x.max(1).values
        step = _power(torch.maximum(low.abs(), high.abs()).max(-1).values)
        bounds[ids] = torch.stack((torch.floor(low / step[..., None]), torch.ceil(high / step[..., None])), -2).to(torch.int8)
        steps[ids] = step.float()
    return [bounds, steps]


def _exact_sparse(s, case):
    Hk, rep, Sq, P, D, keep = (case[n] for n in ("Hk", "rep", "Sq", "page", "D", "keep"))
    lens = _lengths(case)
    pages = torch.full((case["B"], Hk, Sq, keep), -1, dtype=torch.int32, device="cuda")
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = s["block_table"][b, :-(-n // P)].long()
        q = s["q"][b].double().unflatten(0, (Hk, rep))                       # [Hk, rep, Sq, D]
        t = _power(q.abs().max(-1).values)
        whole = torch.round(q / t[..., None]) * t[..., None]
        low, high = (s["bounds"][ids, :, i].double() * s["steps"][ids].double()[..., None] for i in (0, 1))
        score = (torch.einsum("hrsd,phd->hsrp", whole * (whole > 0), high)
                 + torch.einsum("hrsd,phd->hsrp", whole * (whole < 0), low)).max(2).values
        score = score.cpu()
        for i in range(Sq):
            seen = n - Sq + 1 + i if case["causal"] else n
            total = max(0, -(-seen // P))
            for h in range(Hk):
                if total <= keep:
                    chosen = list(range(total))
                else:
                    always = set(range(case["first"])) | set(range(total - case["recent"], total))
                    ranked = torch.sort(score[h, i, :total], descending=True, stable=True).indices.tolist()
                    others = [p for p in ranked if p not in always][:keep - len(always)]
                    chosen = sorted(always | set(others))
                if not chosen:
                    continue
                pages[b, h, i, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
                where = ids[chosen]
                k, v = (_held(s[x + "_pages"], s["scale_" + x], where, h) for x in ("k", "v"))
                count = (len(chosen) - 1) * P + seen - chosen[-1] * P if chosen[-1] == total - 1 else len(chosen) * P
                w = torch.softmax(q[h, :, i] @ k[:count].T / math.sqrt(D), -1)
                out[b, h * rep:(h + 1) * rep, i] = w @ v[:count]
    return [pages, out]


def _exact_beam(s, case):
    V, keep, none = case["V"], case["keep"], -math.inf
    values, parents, tokens = [], [], []
    for b in range(case["B"]):
        found = []    # the best of each beam, then the best of those
        for r in range(case["beams"]):
            cum = float(s["scores"][b, r])
            if s["finished"] is not None and bool(s["finished"][b, r]):
                found += [(cum, r, 0)] + [(none, r, t) for t in range(1, min(V, keep))]
                continue
            x = s["logits"][b, r].double()
            logp = x - torch.logsumexp(x, 0) if bool((x > none).any()) else x
            order = torch.sort(x, descending=True, stable=True).indices[:keep]
            found += [(cum + p, r, t) for p, t in zip(logp[order].tolist(), order.tolist())]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        values.append([c[0] for c in found[:keep]])
        parents.append([c[1] for c in found[:keep]])
        tokens.append([c[2] for c in found[:keep]])
    return [torch.tensor(values, dtype=torch.float64, device="cuda"), torch.tensor(parents, device="cuda"),
            torch.tensor(tokens, device="cuda")]


def _exact_reorder(s, case):
    R, P, L = case["beams"], case["page"], case["tokens"]
    old, parents = s["block_table"].tolist(), s["parents"].tolist()
    new, j, rows = [], L // P, L % P
    outs = {n: s[n].clone() for n in ("k_pages", "v_pages", "scale_k", "scale_v") if s[n] is not None}
    for g, ps in enumerate(parents):
        mine = old[g * R:(g + 1) * R]
        free = [mine[r][j] for r in range(R) if r not in ps] if rows else []
        kept = {p: (p if ps[p] == p else ps.index(p)) for p in ps}
        for c, p in enumerate(ps):
            row = list(mine[p])
            if rows and kept[p] != c:
                source, row[j] = row[j], free.pop(0)
                for x in outs.values():
                    x[row[j], :, :rows] = x[source, :, :rows]
            new.append(row)
    return [torch.tensor(new, dtype=torch.int32, device="cuda"), s["lengths"].clone()] + list(outs.values())


def exact(case, seed):
    if case["op"] == "sparse" and case["B"] * case["Hk"] * case["Sq"] > 12000:   # one by one they would take too long
        return None
    s = prepare(case, seed)
    return {"bounds": _exact_bounds, "sparse": _exact_sparse, "beam": _exact_beam, "reorder": _exact_reorder}[case["op"]](s, case)
