"""Performance cases of the operators around attention: rotary positions, the paged cache, and the attention that reads it.

A case is one layer's work for one step:

  rotary   q and k turned to their positions; with "order" 1 also the gradients, with 2 also the gradients' gradient
  append   the keys (turned to their positions) and values of new tokens written into the pages of a cache; with 4-bit
           pages the whole cache is read back too, which is how its contents are seen
  attend   attention of new tokens' queries (turned to their positions) over the cache, 16-bit or 4-bit

Sequences of a batch have lengths of their own, given by the case alone; the values are N(0, 1), keys with a mean of
their own for each channel.  Pages lie in random order.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ----------------------------------------------------------------------------------------------------
def _rotary(name, B, Hq, Hkv, N, D, dtype="bf16", order=1, rd=0, interleaved=False, scaling="none", factor=1.0, first=0, layout="bnhd"):
    return _named(name, dict(op="rotary", B=B, Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, order=order, rd=rd or D, interleaved=interleaved,
                             scaling=scaling, factor=factor, first=first, layout=layout))


def _append(name, B, Hkv, N, L, D, page, bits=16, dtype="bf16", rd=0, interleaved=False, ragged=True):
    return _named(name, dict(op="append", B=B, Hq=Hkv, Hkv=Hkv, N=N, L=L, D=D, page=page, bits=bits, dtype=dtype, rd=rd or D,
                             interleaved=interleaved, scaling="none", factor=1.0, ragged=ragged))


def _attend(name, B, Hq, Hkv, N, L, D, page, bits=16, dtype="bf16", causal=True, window=0, rd=-1, interleaved=False, ragged=True):
    return _named(name, dict(op="attend", B=B, Hq=Hq, Hkv=Hkv, N=N, L=L, D=D, page=page, bits=bits, dtype=dtype, causal=causal, window=window,
                             rd=D if rd < 0 else rd, interleaved=interleaved, scaling="none", factor=1.0, ragged=ragged))


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # positions of one new token per sequence, where only latency counts
        _rotary("rotary step b8 h16 d64", 8, 16, 16, 1, 64, order=0, first=4095),
        # a grouped-head training layer: the rotation and its gradients
        _rotary("rotary train b2 gqa32/8 n2048 d128", 2, 32, 8, 2048, 128),
        # a long-context layer that turns half of each head, neighbours paired, for a second-order step
        _rotary("rotary second h16 n8191 d64 fp16", 1, 16, 16, 8191, 64, dtype="fp16", order=2, rd=32, interleaved=True, scaling="yarn", factor=4.0),
        # a generation step of 64 sequences stores its tokens
        _append("append step b64 kv8 d128", 64, 8, 1, 4096, 128, 16),
        # ragged prompts are stored before generation
        _append("append prompts b8 kv8 n2048 d128", 8, 8, 2048, 2048, 128, 64),
        # a prompt is stored in 4 bits, and read back
        _append("append 4-bit b2 kv16 n4001 d64 fp16", 2, 16, 4001, 4001, 64, 32, bits=4, dtype="fp16"),
        # one conversation's next token, short cache: latency
        _attend("step b1 gqa32/8 k500 d128", 1, 32, 8, 1, 500, 128, 16),
        # a serving batch of ragged sequences
        _attend("step b64 gqa32/8 k8192 d128", 64, 32, 8, 1, 8192, 128, 64),
        # four tokens to verify per sequence, multi-head, sliding window, fp16
        _attend("verify b8 h16 4x4096 w1024 d64 fp16", 8, 16, 16, 4, 4096, 64, 32, dtype="fp16", window=1024),
        # the next chunk of long prompts, against what is cached of them
        _attend("chunk b4 gqa32/8 1024x8192 d128", 4, 32, 8, 1024, 8192, 128, 64),
        # long contexts in 4 bits
        _attend("4-bit step b16 gqa32/8 k16384 d128", 16, 32, 8, 1, 16384, 128, 64, bits=4),
        # a short chunk against a 4-bit cache, multi-head, no rotation, fp16
        _attend("4-bit chunk b3 h16 100x2500 d64 fp16", 3, 16, 16, 100, 2500, 64, 16, bits=4, dtype="fp16", rd=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "append", "append", "attend", "attend", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    D = rng.choice((32, 64, 64, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    interleaved = rng.choice((False, False, True))
    rd = rng.choice((D, D, D // 2, D // 4))
    while True:
        B, Hkv = _log_int(rng, 1, 64), rng.choice((1, 2, 4, 8, 8, 16, 32))
        G = rng.choice((1, 1, 2, 3, 4, 4, 7, 8))
        if op == "rotary":
            c = _rotary("", B, Hkv * G, Hkv, _log_int(rng, 1, 8192), D, dtype=dtype, order=rng.choice((0, 1, 1, 2)), rd=rd, interleaved=interleaved,
                        scaling=rng.choice(("none", "linear", "ntk", "yarn")), factor=rng.choice((2.0, 4.0, 8.0)), first=rng.choice((0, 0, 1000, 100000)),
                        layout=rng.choice(("bnhd", "bhnd")))
        elif op == "append":
            L = _log_int(rng, 1, 8192)
            bits = rng.choice((16, 16, 4))
            N = L if bits == 4 else rng.choice((1, L, _log_int(rng, 1, L)))
            c = _append("", B, Hkv, N, L, D, page, bits=bits, dtype=dtype, rd=rd, interleaved=interleaved, ragged=rng.choice((True, False)))
        else:
            L = _log_int(rng, 1, 32768)
            N = min(L, rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048))))
            causal = rng.choice((True, True, True, False))
            window = _log_int(rng, 16, 4096) if causal and rng.random() < 0.25 else 0
            c = _attend("", B, Hkv * G, Hkv, N, L, D, page, bits=rng.choice((16, 16, 4)), dtype=dtype, causal=causal, window=window,
                        rd=rng.choice((rd, 0)) if causal else 0, interleaved=interleaved, ragged=rng.choice((True, False)))
        w = work(c)
        # no more than the largest listed cases, and dense scores and keys of the plain form that fit
        if w["bytes"] <= 1e9 and w["flops"] <= 5e11 and c["B"] * c["Hq"] * c["N"] * c.get("L", 1) <= 1.2e9 and c["B"] * c["Hkv"] * c.get("L", 1) * c["D"] <= 6e8:
            return c


# ---- inputs ---------------------------------------------------------------------------------------------------
def _sequences(case):
    """(cached tokens with the new ones, new tokens) of each sequence; a function of the case alone."""
    B, N, L = case["B"], case["N"], case["L"]
    if not case["ragged"]:
        return [(L, N)] * B
    out = []
    for b in range(B):
        length = L - (b * 7919) % max(1, L - L // 4)        # L, and down to a quarter of it, in no order
        new = min(length, N) if N == 1 or case["op"] == "append" else min(length, max(1, N - (b * 31) % max(1, N // 2)))
        out.append((length, new))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Hq, Hkv, N, D = (case[x] for x in ("B", "Hq", "Hkv", "N", "D"))
    dtype = _DTYPES[case["dtype"]]
    state = dict(case=case)

    def heads(H, n, layout="bnhd", grad=False):
        t = torch.randn((B, n, H, D) if layout == "bnhd" else (B, H, n, D), dtype=dtype, device="cuda", generator=gen)
        return (t.transpose(1, 2) if layout == "bnhd" else t).requires_grad_(grad)

    if case["op"] == "rotary":
        grad = case["order"] > 0
        state.update(q=heads(Hq, N, case["layout"], grad), k=heads(Hkv, N, case["layout"], grad))
        # sequences of a batch start at positions of their own
        state["positions"] = case["first"] + torch.arange(N, device="cuda") + 17 * torch.arange(B, device="cuda")[:, None]
        if grad:
            state["dO"] = (heads(Hq, N, "bhnd", case["order"] == 2), heads(Hkv, N, "bhnd", case["order"] == 2))
        if case["order"] == 2:
            state["directions"] = (heads(Hq, N, "bhnd"), heads(Hkv, N, "bhnd"))
    else:
        seqs, page, L = _sequences(case), case["page"], case["L"]
        per = -(-L // page)
        used = [-(-n // page) for n, _ in seqs]
        n_pages = sum(used) + 3
        order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
        table = torch.zeros(B, per, dtype=torch.int32)
        at = 0
        slots = torch.full((B, per), -1, dtype=torch.int64)
        for b, n in enumerate(used):
            slots[b, :n] = torch.arange(at, at + n)
            at += n
        slots = slots.cuda()
        table = torch.where(slots >= 0, order[slots.clamp(min=0)], -1).to(torch.int32)
        state["page_table"] = table
        state["lengths"] = torch.tensor([n for n, _ in seqs], dtype=torch.int32, device="cuda")
        state["counts"] = torch.tensor([c for _, c in seqs], dtype=torch.int32, device="cuda")
        shape = (n_pages, Hkv, page, D)
        mean = torch.randn((1, Hkv, 1, D), device="cuda", generator=gen)
        cached = (torch.randn(shape, dtype=dtype, device="cuda", generator=gen) + mean.to(dtype), torch.randn(shape, dtype=dtype, device="cuda", generator=gen))
        if case["bits"] == 16:
            state["cache"] = dict(k=cached[0], v=cached[1])
        else:
            (kc, ks), (vc, vs) = (_quantise(t) for t in cached)
            state["cache"] = dict(k=kc, v=vc, k_scales=ks, v_scales=vs)
        if case["op"] == "append":
            state.update(k=heads(Hkv, N), v=heads(Hkv, N))
        else:
            state["q"] = heads(Hq, N)
    if own:                                     # the handles that a user's program keeps
        from flashbob_b200 import paged, rotary

        rd = case["rd"]
        state["rotary"] = rotary.Rotary(D, rotary_dim=rd, interleaved=case["interleaved"], scaling=None if case["scaling"] == "none" else case["scaling"],
                                        factor=case["factor"], original_length=4096 if case["scaling"] == "yarn" else None) if rd else None
        if "cache" in state:
            state["handle"] = paged.PagedCache(dtype=dtype, **state["cache"])
    return state


# ---- one pass -------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "rotary":
        return _plain_rotary(state, case)
    if case["op"] == "append":
        return _plain_append(state, case)
    return _plain_attend(state, case)


def _run_own(state, case):
    from flashbob_b200 import paged, rotary

    if case["op"] == "rotary":
        leaves = (state["q"], state["k"])
        out = rotary.apply_rotary(*leaves, state["rotary"], positions=state["positions"])
        if case["order"] == 0:
            return out
        first = torch.autograd.grad(out, leaves, state["dO"], create_graph=case["order"] == 2)
        if case["order"] == 1:
            return (*(t.detach() for t in out), *first)
        second = torch.autograd.grad(first, state["dO"], state["directions"])
        return (*(t.detach() for t in out), *(t.detach() for t in first), *second)
    seqs = (state["page_table"], state["lengths"])
    if case["op"] == "append":
        paged.append_kv(state["k"], state["v"], state["handle"], *seqs, counts=state["counts"], rotary=state["rotary"])
        if case["bits"] == 16:
            return state["cache"]["k"], state["cache"]["v"]
        return paged.read_kv(state["handle"], *seqs, case["L"])
    return paged.sdpa_paged(state["q"], state["handle"], *seqs, counts=state["counts"], is_causal=case["causal"], window_size=case["window"],
                            rotary=state["rotary"])


# ---- plain forms ----------------------------------------------------------------------------------------------
def _frequencies(case):
    """Angle per position of each pair, and the factor on the result; 64 bits."""
    rd, theta, factor = case["rd"], 10000.0, case["factor"]
    i = torch.arange(rd // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk":
        theta *= factor ** (rd / (rd - 2))
    f = theta ** (-2 * i / rd)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] != "yarn":
        return f, 1.0
    low, high = (rd * math.log(4096 / (beta * 2 * math.pi)) / (2 * math.log(theta)) for beta in (32.0, 1.0))
    low, high = max(math.floor(low), 0), min(math.ceil(high), rd - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1


def _turn(x, positions, case, inverse=False):
    """x [B, H, N, D] (computed in its own type) turned to positions [B, N]."""
    rd = case["rd"]
    if not rd:
        return x
    f, m = _frequencies(case)
    angle = positions.double()[:, None, :, None] * f
    c, s = (m * angle.cos()).to(x.dtype), (m * angle.sin()).to(x.dtype)
    if inverse:
        s = -s
    if case["interleaved"]:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        return torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), x[..., rd:]), -1)
    a, b = x[..., : rd // 2], x[..., rd // 2 : rd]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., rd:]), -1)


def _plain_rotary(state, case):
    def both(tensors, inverse):
        return tuple(_turn(t.detach().float(), state["positions"], case, inverse).to(t.dtype) for t in tensors)

    out = both((state["q"], state["k"]), False)
    if case["order"] == 0:
        return out
    first = both(state["dO"], True)                         # the gradient turns back
    return (*out, *first) if case["order"] == 1 else (*out, *first, *both(state["directions"], False))


def _quantise(x):
    """16-bit x [..., D] -> codes [..., D / 2] (element 2 j in the low half of byte j) and fp32 (scale, zero) of each row."""
    x = x.float()
    zero, top = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = torch.where(top > zero, (top - zero) / 15, 1.0)
    codes = ((x - zero) / scale).round().clamp(0, 15).to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.cat((scale, zero), -1)


def _values(codes, scales, dtype):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return c.to(dtype) * scales[..., 0:1].to(dtype) + scales[..., 1:2].to(dtype)


def _new_rows(state, case):
    """Position, page and place in the page of each new token, and which of them there are; [B, N]."""
    i = torch.arange(case["N"], device="cuda")
    position = (state["lengths"] - state["counts"])[:, None].long() + i
    there = i < state["counts"][:, None]
    page = state["page_table"].long().gather(1, (position // case["page"]).clamp(max=state["page_table"].shape[1] - 1))
    return position, page, position % case["page"], there


def _plain_append(state, case):
    position, page, place, there = _new_rows(state, case)
    b, i = there.nonzero(as_tuple=True)
    page, place = page[b, i], place[b, i]
    cache, dtype = state["cache"], state["k"].dtype
    if case["bits"] == 16:
        k = _turn(state["k"].float(), position, case).to(dtype)
        cache["k"][page, :, place] = k[b, :, i]
        cache["v"][page, :, place] = state["v"][b, :, i]
        return cache["k"], cache["v"]
    k = _turn(state["k"].double(), position, case).to(dtype)        # (64 bits: a code's border may be near)
    for name, t in (("k", k), ("v", state["v"])):
        codes, scales = _quantise(t)
        cache[name][page, :, place] = codes[b, :, i]
        cache[name + "_scales"][page, :, place] = scales[b, :, i]
    return tuple(t.to(dtype) for t in _gather(state, case, torch.float32))


def _gather(state, case, dtype):
    """The cached keys and values, [B, Hkv, L, D] each; rows behind a sequence are zero."""
    cache, L = state["cache"], case["L"]
    table = state["page_table"].long().clamp(min=0)
    keep = (torch.arange(L, device="cuda") < state["lengths"][:, None])[:, None, :, None]

    def rows(t):
        return t[table].transpose(1, 2).flatten(2, 3)[:, :, :L]

    out = []
    for name in ("k", "v"):
        x = rows(cache[name])
        x = x.to(dtype) if case["bits"] == 16 else _values(x, rows(cache[name + "_scales"]), dtype)
        out.append(torch.where(keep, x, torch.zeros((), dtype=dtype, device="cuda")))
    return out


def _plain_attend(state, case):
    B, Hq, Hkv, N, L, D = (case[x] for x in ("B", "Hq", "Hkv", "N", "L", "D"))
    k, v = _gather(state, case, torch.float32)
    position = (state["lengths"] - state["counts"])[:, None].long() + torch.arange(N, device="cuda")
    q = _turn(state["q"].float(), position, case).reshape(B, Hkv, Hq // Hkv * N, D)
    s = (q @ k.transpose(-1, -2)).view(B, Hkv, -1, N, L) * D ** -0.5
    distance = position[:, :, None] - torch.arange(L, device="cuda")
    keep = (torch.arange(L, device="cuda") < state["lengths"][:, None])[:, None, :] & (torch.arange(N, device="cuda") < state["counts"][:, None])[:, :, None]
    if case["causal"]:
        keep = keep & (distance >= 0)
    if case["window"]:
        keep = keep & (distance < case["window"])
    s = s.masked_fill_(~keep[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    out = s.view(B, Hkv, -1, L) @ v / total.clamp(min=1e-30).view(B, Hkv, -1, 1)
    return out.view(B, Hq, N, D).to(state["q"].dtype)


# ---- 64 bits --------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    dtype = _DTYPES[case["dtype"]]
    rd = case["rd"]

    def turned(x, p, sign=1.0):
        """One sequence's x [H, n, D] at positions p [n]: each pair as a complex number."""
        x = x.detach().double().clone()
        if not rd:
            return x
        freq, m = _exact_frequencies(case)
        e = m * torch.exp(1j * sign * p.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device))
        first, second = (slice(0, rd, 2), slice(1, rd, 2)) if case["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
        z = torch.complex(x[..., first], x[..., second]) * e
        x[..., first], x[..., second] = z.real, z.imag
        return x

    if case["op"] == "rotary":
        def each(t, sign):
            return torch.stack([turned(t[b], state["positions"][b], sign) for b in range(case["B"])])

        out = [each(state[x], 1.0) for x in ("q", "k")]
        if case["order"]:
            out += [each(t, -1.0) for t in state["dO"]]
        if case["order"] == 2:
            out += [each(t, 1.0) for t in state["directions"]]
        return tuple(out)

    cache, page, table = state["cache"], case["page"], state["page_table"].long()
    seqs = _sequences(case)

    def rows(name, b, n):
        """Cached rows 0 .. n - 1 of sequence b, [Hkv, n, D], in 64 bits."""
        at = table[b, torch.arange(n, device="cuda") // page], torch.arange(n, device="cuda") % page
        x = cache[name][at[0], :, at[1]].transpose(0, 1)
        if case["bits"] == 16:
            return x.double()
        sc = cache[name + "_scales"][at[0], :, at[1]].transpose(0, 1).double()
        y = torch.empty(*x.shape[:-1], case["D"], dtype=torch.float64, device="cuda")
        y[..., 0::2], y[..., 1::2] = (x % 16).double(), (x // 16).double()
        return y * sc[..., :1] + sc[..., 1:]

    if case["op"] == "append" and case["bits"] == 16:
        k, v = cache["k"].double(), cache["v"].double()
        for b, (n, new) in enumerate(seqs):
            p = torch.arange(n - new, n, device="cuda")
            k[table[b, p // page], :, p % page] = turned(state["k"][b, :, :new], p).transpose(0, 1)
            v[table[b, p // page], :, p % page] = state["v"][b, :, :new].double().transpose(0, 1)
        return k, v
    if case["op"] == "append":
        out = []
        for name in ("k", "v"):
            whole = torch.zeros(case["B"], case["Hkv"], case["L"], case["D"], dtype=torch.float64, device="cuda")
            for b, (n, new) in enumerate(seqs):
                whole[b, :, : n - new] = rows(name, b, n)[:, : n - new]
                x = state[name][b, :, :new]
                x = (turned(x, torch.arange(n - new, n, device="cuda")) if name == "k" else x).to(dtype).double()
                low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
                step = torch.where(high > low, (high - low) / 15, torch.ones_like(low)).float().double()   # (held in 32 bits)
                whole[b, :, n - new : n] = torch.round((x - low) / step).clamp(0, 15) * step + low
            out.append(whole)
        return tuple(out)

    out = torch.zeros(case["B"], case["Hq"], case["N"], case["D"], dtype=torch.float64, device="cuda")
    G = case["Hq"] // case["Hkv"]
    for b, (n, new) in enumerate(seqs):
        k, v = rows("k", b, n), rows("v", b, n)
        p = torch.arange(n - new, n, device="cuda")
        j = torch.arange(n, device="cuda")
        seen = torch.ones(new, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen &= j <= p[:, None]
        if case["window"]:
            seen &= j > p[:, None] - case["window"]
        q = turned(state["q"][b, :, :new], p)
        for h in range(case["Hq"]):
            s = (q[h] @ k[h // G].T / math.sqrt(case["D"])).masked_fill(~seen, -math.inf)
            out[b, h, :new] = torch.softmax(s, -1) @ v[h // G]
    return out


def _exact_frequencies(case):
    rd, factor = case["rd"], case["factor"]
    base = 10000.0 * factor ** (rd / (rd - 2)) if case["scaling"] == "ntk" else 10000.0
    freq = [base ** (-2.0 * i / rd) for i in range(rd // 2)]
    if case["scaling"] == "linear":
        return [x / factor for x in freq], 1.0
    if case["scaling"] == "yarn":
        # pairs that turn over 32 times within the original 4096 positions stay, those that turn less than once are interpolated
        def pair(turns):
            return rd * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))

        low, high = max(0, math.floor(pair(32.0))), min(rd - 1, math.ceil(pair(1.0)))
        part = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(rd // 2)]
        return [x * (1 - r) + x / factor * r for x, r in zip(freq, part)], 1.0 + 0.1 * math.log(factor)
    return freq, 1.0


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def work(case):
    B, Hq, Hkv, N, D = (case[x] for x in ("B", "Hq", "Hkv", "N", "D"))
    if case["op"] == "rotary":
        passes = 1 + case["order"]
        return {"bytes": passes * B * N * D * (Hq + Hkv) * 2 * 2, "flops": passes * 3 * B * N * case["rd"] * (Hq + Hkv)}
    seqs = _sequences(case)
    row = 2 * D if case["bits"] == 16 else D // 2 + 8
    if case["op"] == "append":
        new = sum(c for _, c in seqs)
        moved = new * Hkv * 2 * (2 * D + row)
        if case["bits"] == 4:                   # read back
            moved += Hkv * 2 * (sum(n for n, _ in seqs) * row + B * case["L"] * 2 * D)
        return {"bytes": moved, "flops": 3 * new * Hkv * case["rd"]}
    pairs, keys = 0, 0
    for n, c in seqs:
        w = case["window"] or n
        first = max(0, n - c - w + 1)           # the first key that the first of the queries sees
        keys += n - first
        if case["causal"]:
            full = max(0, n - max(n - c, w - 1))                        # queries that see a whole window
            seen = c - full                                             # the others see all keys up to their own
            pairs += full * min(w, n) + seen * (n - c + 1) + seen * (seen - 1) // 2
        else:
            pairs += c * n
    return {"bytes": Hkv * 2 * keys * row + 2 * 2 * B * N * Hq * D, "flops": 4 * pairs * Hq * D}
