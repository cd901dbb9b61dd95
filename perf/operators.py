"""The operators of a paged key/value cache that is held in 8 bits, as cases to be measured.

  plan       request lengths -> block tables, slot maps, row offsets (on the GPU)
  write      new keys and values -> e4m3 values and one power-of-two scale for each page and head, in place
  attention  queries over the cache: one token of each sequence (decode), several (verification, a prompt in pieces),
             whole prompts, or a fixed set of keys that every query sees (an encoder's states)

A scale is an exponent: 8-bit code s stands for 2^(s - 127).  A key or value is its e4m3 code times its page's scale.
"""
import random

import numpy as np
import torch

own = False

EMIN = 27           # the smallest code of a scale: 2^-100, also that of a page of zeros
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # one step of a small server: 16 requests, one new token each
        {"name": "plan_step", "op": "plan", "B": 16, "ctx_lo": 1, "ctx_hi": 4000, "new_lo": 1, "new_hi": 1, "long": 0, "page": 64,
         "mix": 1},
        # a large scheduler step: 1000 requests of which most bring one token and some a prompt of up to 4000
        {"name": "plan_mixed", "op": "plan", "B": 1000, "ctx_lo": 0, "ctx_hi": 3000, "new_lo": 1, "new_hi": 4000, "long": 70,
         "page": 32, "mix": 2},
        # the append of one decode step: 64 sequences, grouped heads
        {"name": "write_step", "op": "write", "B": 64, "ctx_lo": 1, "ctx_hi": 4000, "new_lo": 1, "new_hi": 1, "long": 0,
         "page": 64, "Hkv": 8, "D": 128, "dtype": "bf16", "mix": 3},
        # prompts written whole
        {"name": "write_prompts", "op": "write", "B": 9, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 500, "new_hi": 8000, "long": 9,
         "page": 64, "Hkv": 8, "D": 128, "dtype": "bf16", "mix": 4},
        # decode steps and pieces of prompts together, small pages, every head its own, sequences that bring nothing
        {"name": "write_mixed", "op": "write", "B": 65, "ctx_lo": 0, "ctx_hi": 1000, "new_lo": 0, "new_hi": 700, "long": 6,
         "page": 16, "Hkv": 32, "D": 64, "dtype": "fp16", "mix": 5},
        # one request, a short context: latency
        {"name": "decode_one", "op": "attention", "B": 1, "ctx_lo": 512, "ctx_hi": 512, "new_lo": 1, "new_hi": 1, "long": 0,
         "page": 64, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "mix": 6},
        # an ordinary decode batch of uneven contexts
        {"name": "decode_batch", "op": "attention", "B": 48, "ctx_lo": 60, "ctx_hi": 8000, "new_lo": 1, "new_hi": 1, "long": 0,
         "page": 64, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "mix": 7},
        # few requests of very long contexts
        {"name": "decode_long", "op": "attention", "B": 6, "ctx_lo": 20000, "ctx_hi": 131000, "new_lo": 1, "new_hi": 1, "long": 0,
         "page": 128, "Hq": 64, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "mix": 8},
        # every head its own keys, head dim 64, small pages, sequences without a token among them
        {"name": "decode_heads", "op": "attention", "B": 33, "ctx_lo": 0, "ctx_hi": 2500, "new_lo": 0, "new_hi": 1, "long": 0,
         "page": 16, "Hq": 16, "Hkv": 16, "D": 64, "dtype": "fp16", "causal": True, "mix": 9},
        # two prompts whole
        {"name": "prompt", "op": "attention", "B": 2, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 2900, "new_hi": 4100, "long": 2,
         "page": 64, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "mix": 10},
        # pieces of prompts and decode steps together
        {"name": "prompt_pieces", "op": "attention", "B": 8, "ctx_lo": 500, "ctx_hi": 8000, "new_lo": 1, "new_hi": 500, "long": 4,
         "page": 64, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "mix": 11},
        # a decoder's few tokens over an encoder's states, head dim 256
        {"name": "encoder_states", "op": "attention", "B": 16, "ctx_lo": 300, "ctx_hi": 1500, "new_lo": 1, "new_hi": 7, "long": 16,
         "page": 32, "Hq": 8, "Hkv": 4, "D": 256, "dtype": "fp16", "causal": False, "mix": 12},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(("plan", "write", "attention", "attention"))
    page = rng.choice((16, 32, 64, 128))
    mix = rng.randrange(1000, 1 << 20)
    if op == "plan":
        B = log(1, 1000)
        c = {"op": op, "B": B, "ctx_lo": 0, "ctx_hi": log(1, 3000), "new_lo": rng.choice((0, 1)), "new_hi": log(1, 4000),
             "long": rng.randint(0, min(B, 70)), "page": max(page, 32), "mix": mix}
        return c
    D = rng.choice((64, 128, 128, 256))
    dtype = rng.choice(("bf16", "fp16"))
    Hkv = rng.choice((1, 2, 4, 8))
    if op == "write":
        B = log(1, 128)
        hi = max(1, min(log(1, 8000), 32000 * 128 * 8 // (B * Hkv * D)))
        return {"op": op, "B": B, "ctx_lo": 0, "ctx_hi": log(1, 3000), "new_lo": rng.choice((0, 1)), "new_hi": hi,
                "long": rng.randint(0, B), "page": page, "Hkv": Hkv, "D": D, "dtype": dtype, "mix": mix}
    group = rng.choice((1, 2, 4, 8))
    kind = rng.choice(("decode", "decode", "few", "prompt"))
    if kind == "prompt":
        B, Hkv = rng.randint(1, 3), rng.choice((1, 2, 4))
        new = log(20, 2500)
        ctx = log(1, 3000) if rng.random() < 0.5 else 0
    elif kind == "few":
        B, new = log(1, 32), rng.randint(2, 16)
        ctx = log(10, 6000)
    else:
        B, new = log(1, 64), 1
        ctx = min(log(10, 100000), 130000 * 8 * 128 * 3 // (B * Hkv * D))
    return {"op": op, "B": B, "ctx_lo": ctx // 4, "ctx_hi": ctx, "new_lo": 1, "new_hi": new, "long": B if new > 1 else 0,
            "page": page, "Hq": Hkv * group, "Hkv": Hkv, "D": D, "dtype": dtype, "causal": rng.random() < 0.8, "mix": mix}


def lengths(case):
    """(cached, new) tokens of each sequence, from the case alone: `long` sequences bring up to new_hi tokens, the others
    new_lo (or, where that is 0, none or one)."""
    r = random.Random(case["mix"])
    B = case["B"]
    many = set(r.sample(range(B), case["long"]))
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(B)]
    new = [r.randint(max(1, case["new_lo"]), case["new_hi"]) if b in many else r.randint(case["new_lo"], min(1, case["new_hi"]))
           for b in range(B)]
    if not any(new):
        new[r.randrange(B)] = 1
    return ctx, new


def cdiv(a, b):
    return -(-a // b)


def pow2(code):
    """2^(code - 127) in 32 bits, exactly (exp2 of a whole number may be off by a rounding)."""
    return (code.int() << 23).view(torch.float32)


# ---- inputs -----------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ctx, new = lengths(case)
    P, B, T = case["page"], case["B"], sum(new)
    total = [a + b for a, b in zip(ctx, new)]
    width = max(cdiv(n, P) for n in total) + 2
    held = [cdiv(n, P) for n in (ctx if case["op"] == "plan" else total)]
    pages = sum(cdiv(n, P) for n in total) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(width, device="cuda")
    held_t = torch.tensor(held, device="cuda")
    first = held_t.cumsum(0) - held_t
    table = torch.where(col < held_t[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).to(torch.int32)
    i32 = dict(dtype=torch.int32, device="cuda")
    s = {"case": case, "T": T, "P": P, "pages": pages, "table": table}
    if case["op"] == "plan":
        s |= {"ctx": torch.tensor(ctx, **i32), "new": torch.tensor(new, **i32), "free": order[sum(held):].contiguous()}
        return s
    H, D = case["Hkv"], case["D"]
    dt = DTYPES[case["dtype"]]
    ctx_t, new_t = torch.tensor(ctx, device="cuda"), torch.tensor(new, device="cuda")
    total_t = ctx_t + new_t
    cu = torch.zeros(B + 1, dtype=torch.int64, device="cuda")
    cu[1:] = new_t.cumsum(0)
    # rows that hold a token: all but those behind a sequence's end, which hold NaN codes
    live = torch.zeros(pages, P, dtype=torch.bool, device="cuda")
    known = ctx_t if case["op"] == "write" else total_t
    inside = (torch.arange(width * P, device="cuda") < known[:, None]).view(B, width, P)
    live[table[table >= 0].long()] = inside[table >= 0]

    def codes():
        x = torch.empty(pages, H, P, D, dtype=torch.float8_e4m3fn, device="cuda")
        for at in range(0, pages, 4096):        # pieces: the random numbers are four times as wide
            n = min(4096, pages - at)
            x[at:at + n] = (torch.randn(n, H, P, D, generator=g, device="cuda") * 100).clamp_(-448, 448).to(x.dtype)
        x.view(torch.uint8).masked_fill_(~live[:, None, :, None], 0x7F)
        return x

    def scales():
        return torch.randint(119, 122, (pages, H), generator=g, device="cuda", dtype=torch.uint8)

    s |= {"k": codes(), "v": codes(), "ks": scales(), "vs": scales()}
    if case["op"] == "write":
        t = torch.arange(T, device="cuda")
        b = torch.searchsorted(cu[1:], t, right=True)
        pos = ctx_t[b] + t - cu[b]
        s["slots"] = (table[b, pos // P].long() * P + pos % P).to(torch.int32)
        # a token now and then is several times larger than the page so far: its page's scale grows
        loud = torch.where(torch.rand(T, 1, 1, generator=g, device="cuda") < 0.1, 8.0, 1.0)
        s["k_new"] = (torch.randn(T, H, D, generator=g, device="cuda") * loud).to(dt)
        s["v_new"] = (torch.randn(T, H, D, generator=g, device="cuda") * loud).to(dt)
    else:
        s |= {"q": (2 * torch.randn(T, case["Hq"], D, generator=g, device="cuda")).to(dt), "cu": cu.to(torch.int32),
              "lens": total_t.to(torch.int32), "max_q": max(new), "scale": D ** -0.5, "causal": case["causal"]}
    return s


# ---- the operators ----------------------------------------------------------
def run(s):
    if own:
        from triton_tenstorrent_amd import kernels as K
        if "new" in s:
            p = K.paged_plan(s["ctx"], s["new"], s["table"], s["free"], s["P"], s["T"])
            return {"table": s["table"], "lens": p.lens, "cu": p.cu_new, "slots": p.slot_map, "free_end": p.free_end}
        cache = K.PagedCache(s["k"], s["v"], s["ks"], s["vs"])
        if "slots" in s:
            K.paged_write(s["k_new"], s["v_new"], s["slots"], cache)
            return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
        o, lse = K.paged_attention(s["q"], cache, s["table"], s["lens"], s["cu"], s["scale"], max_q=s["max_q"],
                                   causal=s["causal"], return_lse=True)
        return {"o": o, "lse": lse}
    if "new" in s:
        return plain_plan(s)
    if "slots" in s:
        plain_write(s["k_new"], s["slots"], s["k"], s["ks"])
        plain_write(s["v_new"], s["slots"], s["v"], s["vs"])
        return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
    return plain_attention(s)


def plain_plan(s):
    P, T, table, free = s["P"], s["T"], s["table"], s["free"]
    width = table.shape[1]
    ctx = s["ctx"].long().clamp(0, width * P)
    fits = torch.minimum(s["new"].long().clamp(min=0), width * P - ctx)
    cu = torch.zeros(len(ctx) + 1, dtype=torch.int64, device=ctx.device)
    cu[1:] = fits.cumsum(0).clamp(max=T)
    lens = ctx + cu[1:] - cu[:-1]
    had = (ctx + P - 1) // P
    has = (lens + P - 1) // P
    start = (has - had).cumsum(0) - (has - had)
    free_end = (has - had).sum()
    # the table's new entries
    col = torch.arange(width, device=ctx.device)
    at = start[:, None] + col - had[:, None]
    taken = torch.where(at < len(free), free[at.clamp(0, len(free) - 1)], -1)
    table.copy_(torch.where((col >= had[:, None]) & (col < has[:, None]), taken, table))
    # every new token's slot
    t = torch.arange(T, device=ctx.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=len(ctx) - 1)
    pos = (ctx[b] + t - cu[b]).clamp(0, width * P - 1)
    page = table[b, pos // P].long()
    slots = torch.where((t < cu[-1]) & (page >= 0), page * P + pos % P, -1)
    i32 = torch.int32
    return {"table": table, "lens": lens.to(i32), "cu": cu.to(i32), "slots": slots.to(i32), "free_end": free_end.to(i32).reshape(1)}


def plain_write(x, slots, codes, scales):
    pages, H, P, D = codes.shape
    x = x.float()
    page, row = (slots // P).long(), (slots % P).long()
    touched, of = torch.unique(page, return_inverse=True)
    # the largest magnitude and the first row that each touched page gets
    amax = torch.zeros(len(touched), H, device=x.device).index_reduce_(0, of, x.abs().amax(-1), "amax")
    first = torch.full((len(touched), ), P, device=x.device).index_reduce_(0, of, row, "amin")
    # smallest exponent e with amax <= 448 * 2^e = 1.75 * 2^(e + 8)
    bits = amax.view(torch.int32)
    need = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=EMIN)
    old = scales[touched].int()
    new = torch.where((first > 0)[:, None], torch.maximum(need, old), need)
    # the tokens that were there are put to the new scale, then the new tokens go in
    held = codes.view(torch.uint8)[touched].view(codes.dtype)
    moved = (held.float() * pow2(old - new + 127)[..., None, None]).to(codes.dtype)
    keep = (torch.arange(P, device=x.device) < first[:, None])[:, None, :, None]
    held = torch.where(keep, moved.view(torch.uint8), held.view(torch.uint8))
    q = (x * pow2(254 - new[of])[..., None]).clamp(-448, 448).to(codes.dtype)
    held[of, :, row] = q.view(torch.uint8)
    codes.view(torch.uint8)[touched] = held
    scales[touched] = new.to(torch.uint8)


def plain_attention(s):
    q, table, lens, cu, max_q = s["q"], s["table"], s["lens"].long(), s["cu"].long(), s["max_q"]
    pages, H, P, D = s["k"].shape
    B, width = table.shape
    T, Hq, _ = q.shape
    group, L = Hq // H, width * P
    at = table.clamp(min=0).long()
    key = torch.arange(L, device=q.device)

    def real(codes, scales):        # [B, H, L, D]; the rows behind a sequence's end count as zeros
        x = codes.view(torch.uint8)[at].view(codes.dtype).float() * pow2(scales[at])[..., None, None]
        x = x.transpose(1, 2).reshape(B, H, L, D)
        return torch.where((key < lens[:, None])[:, None, :, None], x, 0.0)

    k, v = real(s["k"], s["ks"]), real(s["v"], s["vs"])
    i = torch.arange(max_q, device=q.device)
    n_q = cu[1:] - cu[:-1]
    rows = q[(cu[:-1, None] + i).clamp(max=T - 1)].float()                                   # [B, max_q, Hq, D]
    rows = rows.view(B, max_q, H, group, D).permute(0, 2, 3, 1, 4).reshape(B, H, group * max_q, D)
    sc = (rows @ k.transpose(-1, -2)).view(B, H, group, max_q, L) * s["scale"]
    last = (lens - n_q)[:, None] + i if s["causal"] else (lens - 1)[:, None].expand(B, max_q)
    sees = (key <= last[..., None]) & (key < lens[:, None, None])                            # [B, max_q, L]
    sc = torch.where(sees[:, None, None], sc, -torch.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -torch.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, H, group * max_q, L) @ v).view(B, H, group, max_q, D) / torch.where(l > 0, l, 1.0)
    lse = torch.where(l > 0, (m + torch.log(l)) * 1.4426950408889634, -torch.inf)
    # back to packed rows
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, max_q, Hq, D)[b, t - cu[b]]
    lse = lse[..., 0].permute(0, 3, 1, 2).reshape(B, max_q, Hq)[b, t - cu[b]]
    return {"o": o.to(q.dtype), "lse": lse}


# ---- what a pass cannot do without ------------------------------------------
def work(case):
    ctx, new = lengths(case)
    P, T, B = case["page"], sum(new), case["B"]
    if case["op"] == "plan":
        fresh = sum(cdiv(a + b, P) - cdiv(a, P) for a, b in zip(ctx, new))
        return {"bytes": 16 * B + 4 * T + 8 * fresh + 8, "flops": T}
    H, D = case["Hkv"], case["D"]
    if case["op"] == "write":
        touched = sum(cdiv(a + b, P) - a // P for a, b in zip(ctx, new) if b)
        return {"bytes": 2 * T * H * D * 3 + 4 * T + 4 * touched * H, "flops": 4 * T * H * D}
    Hq = case["Hq"]
    keys = sum(a + b for a, b in zip(ctx, new) if b)
    used = sum(cdiv(a + b, P) for a, b in zip(ctx, new) if b)
    pairs = sum(b * a + b * (b + 1) // 2 if case["causal"] else b * (a + b) for a, b in zip(ctx, new))
    return {"bytes": 2 * keys * H * D + 2 * used * H + 4 * used + 8 * B + T * Hq * (4 * D + 4), "flops": 4 * pairs * Hq * D}


# ---- the definition, in 64 bits ---------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return exact_plan(case, s)
    if case["op"] == "write":
        k, ks = exact_write(s["k_new"], s["slots"], s["k"], s["ks"])
        v, vs = exact_write(s["v_new"], s["slots"], s["v"], s["vs"])
        return {"k": k, "v": v, "ks": ks, "vs": vs}
    return exact_attention(case, s)


def exact_plan(case, s):
    """Request by request, token by token."""
    ctx, new = lengths(case)
    P, table, free = case["page"], s["table"].cpu().numpy().copy(), s["free"].cpu().numpy()
    used, cu, slots, lens = 0, [0], [], []
    for b, (a, n) in enumerate(zip(ctx, new)):
        for page in range(cdiv(a, P), cdiv(a + n, P)):
            table[b, page] = free[used]
            used += 1
        pos = np.arange(a, a + n)
        slots.append(table[b, pos // P].astype(np.int64) * P + pos % P)
        lens.append(a + n)
        cu.append(cu[-1] + n)
    a32 = lambda v: np.asarray(v, dtype=np.int32)
    return {"table": table, "lens": a32(lens), "cu": a32(cu), "slots": a32(np.concatenate(slots)), "free_end": a32([used])}


TWO = torch.from_numpy(np.ldexp(1.0, np.arange(-300, 301)))


def two(e):
    """2^e in 64 bits, |e| <= 300."""
    return TWO.to(e.device)[e.long() + 300]


def e4m3(x):
    """x rounded to e4m3 (ties to even), |x| <= 448; 64 bits in and out."""
    _, e = torch.frexp(x)                                       # x = m * 2^e, m in [0.5, 1)
    step = two((e - 1).clamp(-6, 8) - 3)
    return torch.round(x / step) * step


def exact_write(x, slots, codes, scales):
    """Token by token, as a sequence of appends would leave the cache: a page's scale is the one that its largest token
    needs, and a token that was there before is rounded again where the scale grows."""
    pages, H, P, D = codes.shape
    out, sc = codes.double(), scales.long()
    x, slots = x.double(), slots.long()
    at = slots.cpu().numpy()
    starts = [0] + [i for i in range(1, len(at)) if at[i] // P != at[i - 1] // P] + [len(at)]
    for i, j in zip(starts, starts[1:]):
        page, row = int(at[i]) // P, int(at[i]) % P
        new = x[i:j]                                            # [n, H, D]
        e = torch.ceil(torch.log2(new.abs().amax((0, 2)) / 448)).long() + 127
        # log2 may round across a whole number: the exponent is checked and moved by one where it has to be
        e = torch.where(new.abs().amax((0, 2)) > 448 * two(e - 127), e + 1, e)
        e = torch.where(new.abs().amax((0, 2)) <= 448 * two(e - 128), e - 1, e).clamp(min=EMIN)
        if row > 0:
            e = torch.maximum(e, sc[page])
            out[page, :, :row] = e4m3(out[page, :, :row] * two(sc[page] - e)[:, None, None])
        sc[page] = e
        out[page, :, row:row + j - i] = e4m3(new * two(127 - e)[:, None]).transpose(0, 1)
    return out, sc.to(torch.uint8)


def exact_attention(case, s):
    """Sequence by sequence and head by head."""
    ctx, new = lengths(case)
    P, H, Hq, D = case["page"], case["Hkv"], case["Hq"], case["D"]
    group = Hq // H
    o = torch.zeros(s["T"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((s["T"], Hq), -torch.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (a, n) in enumerate(zip(ctx, new)):
        used = s["table"][b, :cdiv(a + n, P)].long()
        for h in range(H):
            def real(codes, scales):
                x = codes[:, h].view(torch.uint8)[used].view(codes.dtype).double()
                return (x * two(scales[used, h].long() - 127)[:, None, None]).reshape(-1, D)[:a + n]
            if n == 0 or a + n == 0:
                continue
            k, v = real(s["k"], s["ks"]), real(s["v"], s["vs"])
            hide = torch.arange(a + n, device="cuda") > torch.arange(a, a + n, device="cuda")[:, None]
            for j in range(h * group, (h + 1) * group):
                x = s["q"][at:at + n, j].double() @ k.T * (D ** -0.5)
                if case["causal"]:
                    x = x.masked_fill(hide, -torch.inf)
                z = torch.logsumexp(x, -1)
                o[at:at + n, j] = torch.exp(x - z[:, None]) @ v
                lse[at:at + n, j] = z / np.log(2.0)
        at += n
    return {"o": o, "lse": lse}
