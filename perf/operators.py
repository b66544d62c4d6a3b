"""Single-token and prompt operators of a paged KV cache: rotary positions, the quantising append, and attention.

Three operators that one decoding step runs in a row, over plain tensors:

* ``rotary``     rotates queries and keys by their positions (half-split or interleaved pairs, all
                 or part of the head, tables scaled for long contexts, forwards or backwards);
* ``append``     rotates the new queries and keys, and writes keys and values into the sequences'
                 pages in the cache's precision (fp32, fp16, int8 per row, int4 per 16 values); what
                 is held in 8 or 4 bits is read back as the values it stands for;
* ``attention``  attention of the newest tokens of each sequence over its pages.

``run`` computes them in elementary torch operations in 32 bits, or, where ``own`` is true, through
``shadow_infer_b200.shadowkv``.  ``exact`` holds the definitions in 64 bits.
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
        # a prompt of the longest benchmark step, q and k cut from one fused projection, 4x longer
        # context than the base frequencies cover
        dict(name="rotary_prompt", op="rotary", B=1, S=8192, Hq=32, Hk=8, D=128, rot=128, dtype="bf16",
             interleaved=False, inverse=False, scaling="ntk_parts", offset=24576),
        # odd sizes, a quarter of the head rotated, pairs next to each other, turned back (the gradient's direction)
        dict(name="rotary_part_back", op="rotary", B=3, S=517, Hq=6, Hk=3, D=96, rot=24, dtype="fp32",
             interleaved=True, inverse=True, scaling="linear", offset=5),
        # one new token for each of 8 sequences: a decoding step's write, bound by its latency
        dict(name="append_token_fp16", op="append", B=8, S=1, lo=100, hi=2047, Hq=32, Hk=8, D=128, rot=128, page=32,
             kv="fp16", dtype="bf16", interleaved=False),
        # ragged prompts of a batch into an int8 cache
        dict(name="append_prompt_int8", op="append", B=8, S=2048, lo=0, hi=0, Hq=0, Hk=32, D=128, rot=128, page=32,
             kv="int8", dtype="fp16", interleaved=False),
        # odd lengths and an odd page size, interleaved partial rotation, behind tokens that are there already
        dict(name="append_odd_int4", op="append", B=3, S=1001, lo=1, hi=300, Hq=10, Hk=5, D=64, rot=32, page=17,
             kv="int4", dtype="fp32", interleaved=True),
        # the smallest call: one short sequence, one token
        dict(name="attend_token_short", op="attention", B=1, Sq=1, lo=512, hi=512, Hk=32, rep=1, D=128, page=32,
             kv="fp16", dtype="fp16", causal=False),
        # a decoding batch over ragged int8 sequences, shared key heads
        dict(name="attend_batch_int8", op="attention", B=8, Sq=1, lo=1, hi=2048, Hk=8, rep=4, D=128, page=32,
             kv="int8", dtype="bf16", causal=False),
        # the long-context cache: one sequence, a key head for every query head, int4
        dict(name="attend_long_int4", op="attention", B=1, Sq=1, lo=32768, hi=32768, Hk=32, rep=1, D=128, page=32,
             kv="int4", dtype="fp16", causal=False),
        # four times longer, shared key heads, int8, 32-bit queries and outputs: few heads, so the length has to be split
        dict(name="attend_longest_int8", op="attention", B=1, Sq=1, lo=131071, hi=131071, Hk=8, rep=4, D=128, page=64,
             kv="int8", dtype="fp32", causal=False),
        # a full serving batch, the largest call
        dict(name="attend_full_fp16", op="attention", B=64, Sq=1, lo=64, hi=8192, Hk=8, rep=4, D=128, page=32,
             kv="fp16", dtype="bf16", causal=False),
        # a block of new tokens that see the past and each other up to themselves
        dict(name="attend_block_int8", op="attention", B=4, Sq=16, lo=1024, hi=4096, Hk=8, rep=4, D=128, page=32,
             kv="int8", dtype="bf16", causal=True),
        # odd everything: empty and one-token sequences, a page size and a head size that divide nothing, 32-bit pages
        dict(name="attend_odd_fp32", op="attention", B=5, Sq=3, lo=0, hi=777, Hk=3, rep=3, D=80, page=7,
             kv="fp32", dtype="fp32", causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    """One more case: sizes over the listed ones' ranges, the batch cut until the cost is no more than theirs."""
    op = rng.choice(["rotary", "append", "append", "attention", "attention", "attention"])
    D = rng.choice([64, 128, 128, 128, 96, 80, 256])
    Hk = rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32])
    rep = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    rep = min(rep, 64 // Hk)
    B = _log(rng, 1, 64)
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    page = rng.choice([16, 32, 32, 64, 7, 17, 128])
    kv = rng.choice(["fp32", "fp16", "fp16", "int8", "int8", "int4", "int4"])
    if op == "attention":
        Sq = rng.choice([1, 1, 1, 1, 2, 5, 16, 31])
        hi = _log(rng, 1, 131072)
        while B > 1 and B * hi * Hk * D > 1.3e8:
            B //= 2
        while B * hi * Hk * D > 1.3e8 or B * hi * Hk * D * rep * Sq > 4e9:
            hi = hi * 2 // 3
        lo = hi if B == 1 else rng.choice([0, 1, hi // 2, hi])
        return dict(op=op, B=B, Sq=Sq, lo=lo, hi=hi, Hk=Hk, rep=rep, D=D, page=page, kv=kv, dtype=dtype,
                    causal=rng.random() < 0.4)
    rot = rng.choice([D, D, D // 2, 16])
    S = rng.choice([1, _log(rng, 1, 8192)])
    while B > 1 and B * S * Hk * (rep + 2) * D > 6e7:
        B //= 2
    while B * S * Hk * (rep + 2) * D > 6e7:
        S = S * 2 // 3
    if op == "rotary":
        return dict(op=op, B=B, S=S, Hq=Hk * rep, Hk=Hk, D=D, rot=rot, dtype=dtype, interleaved=rng.random() < 0.5,
                    inverse=rng.random() < 0.3, scaling=rng.choice(["none", "linear", "ntk", "ntk_parts"]),
                    offset=_log(rng, 1, 20000))
    hi = _log(rng, 1, 2048)
    return dict(op=op, B=B, S=S, lo=rng.choice([0, hi // 3, hi]), hi=hi, Hq=Hk * rep * rng.choice([0, 1, 1]), Hk=Hk, D=D,
                rot=rot, page=page, kv=kv, dtype=dtype, interleaved=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """The sequences' lengths, from `lo` to `hi`: the same for every seed, so that the work is."""
    lo, hi, B = case["lo"], case["hi"], case["B"]
    rng = random.Random(lo * 1000003 + hi * 101 + B)
    return [hi] + [rng.randint(lo, hi) for _ in range(B - 2)] + ([lo] if B > 1 else [])


def _new_lengths(case):
    """How many of the S new rows of each sequence are tokens (the rest is padding of a ragged prompt)."""
    S, B = case["S"], case["B"]
    rng = random.Random(S * 7919 + B)
    return [S] + [rng.randint((S + 1) // 2, S) for _ in range(B - 1)]


def _frequencies(rot, scaling):
    """The angle of each pair per position, and the factor on cos and sin."""
    base, half = 10000.0, rot // 2
    if scaling == "ntk":
        base *= 4.0 ** (rot / max(1, rot - 2))
    inv = base ** (-torch.arange(half, dtype=torch.float64) * 2 / rot)
    if scaling == "linear":
        return inv / 4.0, 1.0
    if scaling == "ntk_parts":
        # pairs that turn over 32 times within the trained length keep their frequency, those that
        # turn less than once are slowed down, a ramp in between
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return inv / 4.0 * (1 - keep) + inv * keep, 0.1 * math.log(4.0) + 1.0
    return inv, 1.0


def _tables(rot, scaling, n):
    inv, factor = _frequencies(rot, scaling)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv.cuda()
    return (a.cos() * factor).float(), (a.sin() * factor).float()


def _pages(case, gen, counts, stale):
    """Pages in shuffled order, their table, and rows past each sequence's end that hold `stale` values."""
    P, H, D, kv, B = case["page"], case["Hk"], case["D"], case["kv"], case["B"]
    per = [-(-n // P) for n in counts]
    N, M = sum(per) + 3, max(per) + 1
    order = torch.randperm(N, generator=torch.Generator().manual_seed(gen.initial_seed())).tolist()
    table, used, at = torch.full((B, M), -1, dtype=torch.int32), torch.zeros(N, P, dtype=torch.bool), 0
    for b, n in enumerate(per):
        ids = order[at:at + n]
        at += n
        if n:
            table[b, :n] = torch.tensor(ids, dtype=torch.int32)
            used[ids] = True
            used[ids[-1]] = torch.arange(P) < counts[b] - (n - 1) * P
    unused = ~used.cuda()
    s = {"block_table": table.cuda()}
    for name in ("k", "v"):
        x = torch.randn(N, H, P, D, generator=gen, device="cuda", dtype=torch.float32 if kv == "fp32" else torch.float16)
        if name == "k":  # a few channels of K are larger than the others
            x[..., :: max(1, D // 4)] *= 3.0
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
            scale.masked_fill_(unused.view(N, 1, P, *[1] * (scale.dim() - 3)), stale)
        else:
            x.masked_fill_(unused.view(N, 1, P, 1), stale)
        s[name + "_pages"], s["scale_" + name] = x, scale
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _TYPE[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dt)

    if case["op"] == "attention":
        lens = _lengths(case)
        s = _pages(case, gen, lens, math.nan)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = rand(case["B"], case["Sq"], case["Hk"] * case["rep"], case["D"]).transpose(1, 2)
    else:
        B, S, Hq, Hk, D = (case[n] for n in ("B", "S", "Hq", "Hk", "D"))
        # one projection's output [B, S, heads, D]; q, k and v are its slices, seen as [B, heads, S, D]
        x = rand(B, S, Hq + 2 * Hk, D).transpose(1, 2)
        s = {"q": x[:, :Hq] if Hq else None, "k": x[:, Hq:Hq + Hk], "v": x[:, Hq + Hk:]}
        if case["op"] == "rotary":
            steps = [case["offset"] + 11 * b for b in range(B)]
            s["positions"] = torch.tensor(steps, device="cuda")[:, None] + torch.arange(S, device="cuda")
            s["cos"], s["sin"] = _tables(case["rot"], case["scaling"], max(steps) + S)
        else:
            lens, new = _lengths(case), _new_lengths(case)
            total = [a + b for a, b in zip(lens, new)]
            s |= _pages(case, gen, total, 0.5)
            for name, v in (("lengths", lens), ("new_lengths", new), ("total", total)):
                s[name] = torch.tensor(v, dtype=torch.int32, device="cuda")
            s["cos"], s["sin"] = _tables(case["rot"], "none", max(lens) + S)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin, interleaved):
    """x [B, H, S, D] in 32 bits, cos and sin [B, S, rot / 2]."""
    half = cos.shape[-1]
    c, s, part = cos[:, None], sin[:, None], x[..., :2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    u, v = a * c - b * s, b * c + a * s
    part = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((part, x[..., 2 * half:]), -1)


def _values(pages, scale):
    """What page rows stand for, in 32 bits."""
    if pages.dtype == torch.uint8:
        x = torch.stack((pages >> 4, pages & 15), -1).flatten(-2).float() - 8.0
        return (x.unflatten(-1, (scale.shape[-2], -1)) * scale).flatten(-2)
    return pages.float() if scale is None else pages.float() * scale


def _quantise(x, kv):
    """x [..., D] in 32 bits as page rows and their scales: amax / 127 (int8) or / 7 (int4), one where a row is zero."""
    if kv not in ("int8", "int4"):
        return x.to(_TYPE[kv]), None
    top = torch.full((), 7.0 if kv == "int4" else 127.0, device=x.device)
    g = x.unflatten(-1, (-1, GROUP)) if kv == "int4" else x
    scale = g.abs().amax(-1, keepdim=True) / top.expand(1)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    n = torch.clamp(torch.round(g / scale), -8 if kv == "int4" else -128, 7 if kv == "int4" else 127)
    if kv == "int8":
        return n.to(torch.int8), scale
    n = (n + 8).to(torch.uint8).flatten(-2)
    return n[..., 0::2] * 16 + n[..., 1::2], scale


def _rotary(s):
    case = s["case"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    sin = -sin if case["inverse"] else sin
    return [_rotate(s[n].float(), cos, sin, case["interleaved"]).to(s[n].dtype) for n in ("q", "k")]


def _append(s):
    case, P = s["case"], s["k_pages"].shape[2]
    S = s["k"].shape[2]
    step = torch.arange(S, device="cuda")
    at = s["lengths"].long()[:, None] + step
    cos, sin = s["cos"][at], s["sin"][at]
    out = {} if s["q"] is None else {"q": _rotate(s["q"].float(), cos, sin, case["interleaved"]).to(s["q"].dtype)}
    here = step < s["new_lengths"].long()[:, None]
    page = s["block_table"].long().gather(1, (at // P).clamp_max(s["block_table"].shape[1] - 1))
    page, row = page[here], (at % P)[here]
    for name in ("k", "v"):
        x = s[name].float()
        x = _rotate(x, cos, sin, case["interleaved"]) if name == "k" else x
        x, scale = _quantise(x, case["kv"])
        s[name + "_pages"][page, :, row] = x.transpose(1, 2)[here]
        if scale is None:
            out[name + "_pages"] = s[name + "_pages"]
        else:
            s["scale_" + name][page, :, row] = scale.transpose(1, 2)[here]
            y = torch.zeros(s[name].shape[0], S, *s[name].shape[1::2], device="cuda")
            y[here] = _values(s[name + "_pages"][page, :, row], s["scale_" + name][page, :, row])
            out[name] = y.transpose(1, 2)
    return out


def _attention(s):
    case, q, table = s["case"], s["q"].float(), s["block_table"].long()
    B, H, Sq, D = q.shape
    Hk, P, M = case["Hk"], case["page"], table.shape[1]
    lens = s["lengths"].long()
    token = torch.arange(M * P, device="cuda")
    there = (token < lens[:, None])[:, None, :, None]
    past = [None, None]
    for i, n in enumerate(("k", "v")):
        scale = s["scale_" + n]
        x = _values(s[n + "_pages"][table], None if scale is None else scale[table]).transpose(1, 2).flatten(2, 3)
        past[i] = torch.where(there, x, torch.zeros((), device="cuda"))
    score = q.reshape(B, Hk, -1, D) @ past[0].transpose(-1, -2) * (1.0 / math.sqrt(D))
    last = lens[:, None] - (Sq - torch.arange(Sq, device="cuda") if case["causal"] else 0 * torch.arange(Sq, device="cuda") + 1)
    seen = (token <= last[:, :, None])[:, None, None]
    score = torch.where(seen, score.view(B, Hk, -1, Sq, M * P), torch.full((), -math.inf, device="cuda")).flatten(2, 3)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ past[1]) / torch.where(total == 0, torch.ones_like(total), total)
    return out.view(B, H, Sq, D).to(s["q"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"rotary": _rotary, "append": _append, "attention": _attention}[op](s)
    from shadow_infer_b200 import shadowkv

    case = s["case"]
    if op == "rotary":
        return list(shadowkv.apply_rotary(s["q"], s["cos"], s["sin"], k=s["k"], positions=s["positions"],
                                          interleaved=case["interleaved"], inverse=case["inverse"]))
    pool = (s["k_pages"], s["v_pages"], s["block_table"])
    scales = dict(scale_k=s["scale_k"], scale_v=s["scale_v"])
    if op == "attention":
        return shadowkv.paged_attention(s["q"], *pool, s["lengths"], **scales, causal=case["causal"])
    q = shadowkv.paged_append(s["k"], s["v"], *pool, s["lengths"], **scales, new_lengths=s["new_lengths"], q=s["q"],
                              cos=s["cos"], sin=s["sin"], interleaved=case["interleaved"])
    out = {} if q is None else {"q": q}
    if s["scale_k"] is None:
        return {**out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    k, v = shadowkv.paged_read(*pool, s["total"], case["S"], **scales, start=s["lengths"])
    return {**out, "k": k, "v": v}


# --------------------------------------------------------------------------------------- what it costs
def _row_bytes(kv, D):
    """Bytes of one page row and its scales."""
    return {"fp32": 4 * D, "fp16": 2 * D, "int8": D + 4, "int4": D // 2 + D // GROUP * 4}[kv]


def work(case):
    B, D, e = case["B"], case["D"], _BYTES[case["dtype"]]
    if case["op"] == "attention":
        lens, Sq, R = _lengths(case), case["Sq"], case["Hk"] * case["rep"]
        kv = 2 * sum(lens) * case["Hk"] * _row_bytes(case["kv"], D)
        seen = sum(max(0, n - Sq + 1 + i) for n in lens for i in range(Sq)) if case["causal"] else sum(lens) * Sq
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": kv + 2 * B * Sq * R * D * e + 4 * (pages + B), "flops": 4 * seen * R * D}
    S, Hq, Hk, rot = case["S"], case["Hq"], case["Hk"], case["rot"]
    if case["op"] == "rotary":
        table = 4 * rot * (S + 11 * (B - 1) if B > 1 else S)
        return {"bytes": 2 * B * S * (Hq + Hk) * D * e + table + 8 * B * S, "flops": 3 * B * S * (Hq + Hk) * rot}
    n = sum(_new_lengths(case))
    table = 4 * rot * min(n, S + max(_lengths(case)))
    b = B * S * Hq * D * e * 2 + 2 * n * Hk * (D * e + _row_bytes(case["kv"], D)) + table
    if case["kv"] in ("int8", "int4"):
        b += 2 * n * Hk * _row_bytes(case["kv"], D) + 2 * B * S * Hk * D * 4
    return {"bytes": b, "flops": 3 * n * (Hq + Hk) * rot + 4 * n * Hk * D}


# ------------------------------------------------------------------------- the definitions in 64 bits
def _turn(x, cos, sin, interleaved, sign=1.0):
    """Each pair of x [n, H, D] times a unit complex number: cos, sin [n, rot / 2]."""
    x, half = x.double().clone(), cos.shape[-1]
    first = torch.arange(half, device=x.device) * 2 if interleaved else torch.arange(half, device=x.device)
    second = first + (1 if interleaved else half)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos.double(), sign * sin.double())[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _stored(x, kv):
    """What a row of x keeps when it is written, in 64 bits."""
    if kv not in ("int8", "int4"):
        return x
    width, top = (GROUP, 7) if kv == "int4" else (x.shape[-1], 127)
    g = x.reshape(-1, width)
    scale = g.abs().max(-1, keepdim=True).values / top
    scale[scale == 0] = 1
    return (torch.round(g / scale).clamp(-top - 1, top) * scale).reshape(x.shape)


def _held(pages, scale, ids):
    """Tokens [n * P, H, D] of the pages `ids`, in 64 bits."""
    x = pages[ids]
    if scale is None:
        x = x.double()
    elif x.dtype == torch.int8:
        x = x.double() * scale[ids].double()
    else:
        sign = torch.stack((x.int().div(16, rounding_mode="floor"), x.int() % 16), -1) - 8
        x = (sign.reshape(*x.shape[:-1], -1, GROUP).double() * scale[ids].double()).reshape(*x.shape[:-1], -1)
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])


def exact(case, seed):
    s = prepare(case, seed)
    P = case.get("page")
    if case["op"] == "attention":
        q, outs = s["q"].double(), []
        Sq = case["Sq"]
        for b, n in enumerate(_lengths(case)):
            if n == 0:
                outs.append(torch.zeros_like(q[b]))
                continue
            ids = s["block_table"][b, :-(-n // P)].long()
            k, v = (_held(s[x + "_pages"], s["scale_" + x], ids)[:n] for x in ("k", "v"))
            w = torch.einsum("grsd,tgd->grst", q[b].unflatten(0, (case["Hk"], -1)), k) / math.sqrt(case["D"])
            if case["causal"]:
                w = w.masked_fill(torch.ones(Sq, n, device="cuda").triu(n - Sq + 1).bool(), -math.inf)
            w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
            outs.append(torch.einsum("grst,tgd->grsd", w, v).flatten(0, 1))
        return torch.stack(outs)
    if case["op"] == "rotary":
        outs = []
        for n in ("q", "k"):
            rows = [_turn(s[n][b].transpose(0, 1), s["cos"][s["positions"][b]], s["sin"][s["positions"][b]],
                          case["interleaved"], -1.0 if case["inverse"] else 1.0).transpose(0, 1) for b in range(case["B"])]
            outs.append(torch.stack(rows))
        return outs
    out = {} if s["q"] is None else {"q": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")}
    quantised = case["kv"] in ("int8", "int4")
    for n in ("k", "v"):
        out[n if quantised else n + "_pages"] = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") if quantised
                                                 else s[n + "_pages"].double())
    for b, (first, new) in enumerate(zip(_lengths(case), _new_lengths(case))):
        where = torch.arange(first, first + case["S"], device="cuda")
        cos, sin = s["cos"][where], s["sin"][where]
        if s["q"] is not None:
            out["q"][b] = _turn(s["q"][b].transpose(0, 1), cos, sin, case["interleaved"]).transpose(0, 1)
        for n in ("k", "v"):
            x = s[n][b].transpose(0, 1)
            x = _stored(_turn(x, cos, sin, case["interleaved"]) if n == "k" else x.double(), case["kv"])[:new]
            if quantised:
                out[n][b, :, :new] = x.transpose(0, 1)
            else:
                ids = s["block_table"][b].long()[where[:new] // P]
                out[n + "_pages"][ids, :, where[:new] % P] = x
    return out
