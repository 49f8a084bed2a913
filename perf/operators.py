"""The operators around an 8-bit key/value cache whose speed matters, as a user's
program calls them, and their plain forms.

Every case is one of four kinds:

  norm     add_rms_norm: a decoder layer's residual sum and root-mean-square
           norm, the result in 8 bits with scales (or in 16)
  write    kv_write: new keys and values quantised into the pages of a cache
           (int8 caches: written and read back, as the values they stand for)
  read     kv_read: cached tokens back in 16 bits, packed
  attend   KvAttention.run: a chunk of new tokens (one token per sequence when
           decoding) over the paged cache that already holds them

Sizes are the Llama-3-8B and -70B layers' (hidden 4096 and 8192, 32 or 64 query
heads over 8 key/value heads of 128) and generic ones around them.

A sequence s of a case has `starts[s]` tokens in the cache before its chunk of
`lens[s]` tokens; token i of the chunk has position starts[s] + i and lies in
slot (position % page) of the cache page table[s, position // page].
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
TOP = {"f8": 448.0, "i8": 127.0}   # largest value of a code
TINY = 2.0 ** -100                 # rows whose largest magnitude is below this are stored as zeros
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of a decoding step through a layer's norm, the smallest call
        dict(name="norm_token", kind="norm", rows=1, hidden=4096, type="bf16", out="f8", group=0),
        # a prefill chunk
        dict(name="norm_chunk", kind="norm", rows=2048, hidden=4096, type="bf16", out="f8", group=0),
        # a large batch of the 70B hidden size, scales per 128 values
        dict(name="norm_large", kind="norm", rows=16384, hidden=8192, type="f16", out="f8", group=128),
        # a decoding step of 64 sequences: one new token each
        dict(name="write_step", kind="write", cache="f8", type="bf16", kv_heads=8, dim=128, page=64, seqs=64,
             new_lo=1, new_hi=1, old_lo=100, old_hi=4000, shape=1),
        # a prefill batch of ragged prompts
        dict(name="write_chunk", kind="write", cache="f8", type="bf16", kv_heads=8, dim=128, page=64, seqs=9,
             new_lo=300, new_hi=4000, old_lo=0, old_hi=2000, shape=2),
        # the same in int8 with other heads, each row read back
        dict(name="write_int8", kind="write", cache="i8", type="f16", kv_heads=4, dim=64, page=16, seqs=5,
             new_lo=1000, new_hi=9000, old_lo=0, old_hi=777, shape=3),
        # whole sequences out of the cache, to hand them to another program
        dict(name="read_sequences", kind="read", cache="f8", type="bf16", kv_heads=8, dim=128, page=64, seqs=16,
             new_lo=1000, new_hi=16000, old_lo=0, old_hi=0, shape=4),
        # a few tokens that a user wants back
        dict(name="read_tail", kind="read", cache="i8", type="bf16", kv_heads=8, dim=128, page=32, seqs=3,
             new_lo=5, new_hi=50, old_lo=100, old_hi=900, shape=5),
        # one sequence decoding its next token, a short context: latency
        dict(name="attend_token", kind="attend", cache="f8", type="bf16", kv_heads=8, group=4, dim=128, page=64,
             seqs=1, new_lo=1, new_hi=1, old_lo=1000, old_hi=1000, window=0, shape=6),
        # a decoding step of 64 sequences with ragged contexts
        dict(name="attend_step", kind="attend", cache="f8", type="bf16", kv_heads=8, group=4, dim=128, page=64,
             seqs=64, new_lo=1, new_hi=1, old_lo=200, old_hi=16000, window=0, shape=7),
        # a prefill chunk of 2048 tokens behind 30 thousand in the cache
        dict(name="attend_chunk", kind="attend", cache="f8", type="bf16", kv_heads=8, group=4, dim=128, page=64,
             seqs=1, new_lo=2048, new_hi=2048, old_lo=30000, old_hi=30000, window=0, shape=8),
        # ragged prompts from their first token on, the cache in the model's own type
        dict(name="attend_prompts", kind="attend", cache="f16", type="f16", kv_heads=8, group=8, dim=128, page=16,
             seqs=6, new_lo=150, new_hi=3000, old_lo=0, old_hi=0, window=0, shape=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "write", "read", "attend", "attend", "attend", "attend"])
    shape = rng.randrange(1 << 30)
    if kind == "norm":
        hidden = rng.choice([1024, 2048, 4096, 5120, 8192, 2 * rng.randrange(32, 6000) + 1, 2 * rng.randrange(32, 6000) + 1])
        out = rng.choice(["f8", "f8", "f8", "same"])
        group = rng.choice([0, 0, 32, 128]) if out == "f8" else 0
        return dict(kind=kind, rows=_log(rng, 1, max(2, (1 << 25) // hidden)), hidden=hidden,
                    type=rng.choice(["bf16", "bf16", "f16", "f32"]), out=out, group=group if group and hidden % group == 0 else 0)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8])
    base = dict(kind=kind, cache=rng.choice(["f8", "f8", "i8", "same"]), type=rng.choice(["bf16", "bf16", "f16"]),
                kv_heads=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), shape=shape)
    if base["cache"] == "same":
        base["cache"] = base["type"]
    if kind in ("write", "read"):
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 60000 // seqs)
        return dict(base, seqs=seqs, new_lo=max(1, new // 4), new_hi=new, old_lo=0, old_hi=rng.choice([0, 100, 3000]))
    group = rng.choice([1, 2, 4, 4, 8])
    window = rng.choice([0, 0, 0, _log(rng, 100, 4000)])
    if rng.random() < 0.5:      # decoding, one or a few drafted tokens
        seqs = _log(rng, 1, 64)
        old = _log(rng, 1, max(2, min(131072, (1 << 28) // (seqs * kv * dim))))
        new = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return dict(base, group=group, seqs=seqs, new_lo=1, new_hi=new, old_lo=max(1, old // rng.choice([1, 4, 50])),
                    old_hi=old, window=window)
    seqs = rng.randint(1, 4)    # prefill
    new = _log(rng, 16, 2048 // seqs)
    old = rng.choice([0, _log(rng, 1, 30000 // seqs)])
    return dict(base, group=group, seqs=seqs, new_lo=max(1, new // 3), new_hi=new, old_lo=old // 3, old_hi=old, window=window)


def _lengths(c):
    """(tokens in the cache before, new tokens) of each sequence."""
    r = random.Random(c["shape"])
    return ([r.randint(c["old_lo"], c["old_hi"]) for _ in range(c["seqs"])],
            [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])])


def work(case):
    if case["kind"] == "norm":
        n, e = case["rows"] * case["hidden"], 4 if case["type"] == "f32" else 2
        out = n * e if case["out"] == "same" else n + 4 * (n // case["group"] if case["group"] else case["rows"])
        return {"bytes": 3 * n * e + case["hidden"] * e + out, "flops": 8 * n}
    old, new = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    wide = 2 * row * 2                                                     # a token's keys and values in 16 bits
    held = wide if case["cache"] in TYPES else 2 * row + 8 * case["kv_heads"]
    if case["kind"] == "write":
        again = wide + held if case["cache"] == "i8" else 0
        return {"bytes": sum(new) * (wide + held + again), "flops": 6 * sum(new) * row}
    if case["kind"] == "read":
        return {"bytes": sum(new) * (wide + held), "flops": 2 * sum(new) * row}
    w, pairs, seen = case["window"], 0, 0
    for o, n in zip(old, new):
        first = o + 1                                                     # keys that the chunk's first token sees
        if w:
            full = max(0, min(n, w - first))                              # tokens whose window is not yet full
            pairs += full * first + full * (full - 1) // 2 + (n - full) * min(w, first + n - 1 if n == full else w)
            seen += min(o + n, w + n - 1)
        else:
            pairs += n * first + n * (n - 1) // 2
            seen += o + n
    heads = case["kv_heads"] * case["group"]
    return {"bytes": seen * held + sum(new) * heads * (case["dim"] * 4 + 4), "flops": 4 * pairs * heads * case["dim"]}


# ------------------------------------------------------------------ the inputs
def _codes(x, fmt):
    """Rows of `x` (32 bits) as codes with one scale a row."""
    top = x.abs().amax(-1)
    scale = torch.where(top >= TINY, top / TOP[fmt], 0.0)
    inv = torch.where(top >= TINY, torch.full_like(top, TOP[fmt]) / top, 0.0)  # one rounding: a number / tensor takes two
    v = x * inv[..., None]
    return (v.round().to(torch.int8) if fmt == "i8" else v.to(F8)), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    st = {"case": case}
    if case["kind"] == "norm":
        t = TYPES[case["type"]]
        rows, n = case["rows"], case["hidden"]
        spread = torch.exp(0.5 * normal(n))                               # a few loud channels, as hidden states have
        st["x"] = (normal(rows, n) * spread).to(t)
        st["residual"] = (normal(rows, n) * 2 * spread).to(t)
        st["weight"] = (1 + 0.1 * normal(n)).to(t)
        if own:
            import checkers_amd as ck
            q = case["out"] == "f8"
            per = n // case["group"] if case["group"] else 1
            st["out"] = torch.empty(rows, n, dtype=F8 if q else t, device=dev)
            st["scales"] = torch.empty((rows, per) if case["group"] else (rows,), dtype=torch.float32, device=dev) if q else None
            st["total"] = torch.empty(rows, n, dtype=t, device=dev)
            st["tag"] = ck.F8 if q else ck.torch_tag(t)
        return st
    t, fmt, ps, heads, dim = TYPES[case["type"]], case["cache"], case["page"], case["kv_heads"], case["dim"]
    old, new = _lengths(case)
    pages = [-(-(o + n) // ps) for o, n in zip(old, new)]
    width = max(pages)
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32)
    for s, p in enumerate(pages):
        table[s, :p] = torch.tensor(order[sum(pages[:s]):sum(pages[:s]) + p], dtype=torch.int32)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    st["table"] = table.to(dev)
    st["starts"] = torch.tensor(old, dtype=torch.int32, device=dev)
    st["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
    st["tokens"], st["longest"], st["context"] = offsets[-1], max(new), max(o + n for o, n in zip(old, new))
    loud = torch.exp(0.7 * normal(heads, 1, dim))                         # some key channels are louder than others
    st["k"], st["k_scale"], st["v"], st["v_scale"] = None, None, None, None
    for name in ("k", "v"):
        x = normal(n_pages, heads, ps, dim) * loud if name == "k" else normal(n_pages, heads, ps, dim)
        if fmt in TYPES:
            st[name] = x.to(TYPES[fmt])
        else:
            st[name], st[name + "_scale"] = _codes(x, fmt)
        del x
    if case["kind"] == "write":
        st["new_k"] = (normal(offsets[-1], heads, dim) * loud.view(heads, dim)).to(t)
        st["new_v"] = normal(offsets[-1], heads, dim).to(t)
    if case["kind"] == "attend":
        st["scale"] = dim ** -0.5
        st["q"] = (normal(offsets[-1], heads * case["group"], dim) * 1.5).to(t)
    if own:
        import checkers_amd as ck
        st["cache"] = ck.KvCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["batch"] = ck.KvBatch(st["table"], st["starts"], st["offsets"], st["tokens"], st["longest"], st["context"])
        if case["kind"] == "attend":
            st["plan"] = ck.KvAttention(heads * case["group"], heads, dim, case["seqs"], st["tokens"], st["longest"], st["context"])
            st["out"] = torch.empty_like(st["q"])
            st["lse"] = torch.empty(st["tokens"], heads * case["group"], dtype=torch.float32, device=dev)
        elif case["kind"] == "read" or fmt == "i8":
            st["out"] = tuple(torch.empty(st["tokens"], heads, dim, dtype=t, device=dev) for _ in range(2))
            st["tag"] = ck.torch_tag(t)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if not own:
        return {"norm": _norm, "write": _write, "read": _read, "attend": _attend}[c["kind"]](state)
    import checkers_amd as ck
    if c["kind"] == "norm":
        ck.add_rms_norm(state["x"], state["residual"], state["weight"], EPS, state["tag"], group=c["group"],
                        out=state["out"], scales=state["scales"], total=state["total"])
        return {"out": state["out"], "scales": state["scales"], "total": state["total"]}
    if c["kind"] == "write":
        ck.kv_write(state["cache"], state["batch"], state["new_k"], state["new_v"])
        if c["cache"] == "i8":
            k, v = ck.kv_read(state["cache"], state["batch"], state["tag"], out=state["out"])
            return {"k": k, "v": v}
        return {"k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if c["kind"] == "read":
        k, v = ck.kv_read(state["cache"], state["batch"], state["tag"], out=state["out"])
        return {"k": k, "v": v}
    state["plan"].run(state["cache"], state["batch"], state["q"], scale=state["scale"], window=c["window"],
                      out=state["out"], lse=state["lse"])
    return {"out": state["out"], "lse": state["lse"]}


def _norm(st):
    c, x = st["case"], st["x"]
    total = x.float() + st["residual"].float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + EPS) * st["weight"].float()
    if c["out"] == "same":
        return {"out": y.to(x.dtype), "scales": None, "total": total.to(x.dtype)}
    if not c["group"]:
        codes, scales = _codes(y, "f8")
    else:
        codes, scales = _codes(y.view(c["rows"], -1, c["group"]), "f8")
        codes = codes.view(c["rows"], -1)
    return {"out": codes, "scales": scales, "total": total.to(x.dtype)}


def _tokens(st):
    """(sequence, index in its chunk) of every token of the batch."""
    lens = (st["offsets"][1:] - st["offsets"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device=lens.device), lens, output_size=st["tokens"])
    return seq, torch.arange(st["tokens"], device=lens.device) - st["offsets"].long()[seq]


def _places(st):
    """(page, slot) of every token of the batch."""
    seq, at = _tokens(st)
    pos = st["starts"].long()[seq] + at
    return st["table"].long()[seq, pos // st["case"]["page"]], pos % st["case"]["page"]


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == F8 else x


def _write(st):
    c = st["case"]
    page, slot = _places(st)
    for name in ("k", "v"):
        new, pool = st["new_" + name], st[name]
        if c["cache"] in TYPES:
            pool[page, :, slot] = new
        else:
            codes, scales = _codes(new.float(), c["cache"])
            _bytes(pool)[page, :, slot] = _bytes(codes)
            st[name + "_scale"][page, :, slot] = scales
    if c["cache"] == "i8":
        return _read(st)
    return {"k": st["k"], "v": st["v"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _read(st):
    c = st["case"]
    page, slot = _places(st)
    out = {}
    for name in ("k", "v"):
        x = _bytes(st[name])[page, :, slot]
        if c["cache"] not in TYPES:
            x = (x.view(F8) if c["cache"] == "f8" else x).float() * st[name + "_scale"][page, :, slot][..., None]
        out[name] = x.to(TYPES[c["type"]])
    return out


def _attend(st):
    c = st["case"]
    S, H, G, D, n = c["seqs"], c["kv_heads"], c["group"], c["dim"], st["longest"]
    dev = st["q"].device
    pages = st["table"].long().clamp(min=0)
    kv = []
    for name in ("k", "v"):
        x = _bytes(st[name])[pages]                                       # [S, pages, H, page, D]
        if c["cache"] in TYPES:
            x = x.float()
        else:
            x = (x.view(F8) if c["cache"] == "f8" else x).float() * st[name + "_scale"][pages][..., None]
        kv.append(x.transpose(1, 2).reshape(S, H, -1, D))
    k, v = kv
    step = torch.arange(n, device=dev)
    rows = (st["offsets"][:-1, None].long() + step).clamp(max=st["tokens"] - 1)
    q = st["q"][rows].float().view(S, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * n, D)
    s = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * st["scale"]).view(S, H, G, n, -1)
    pos = (st["starts"][:, None].long() + step)[:, None, None, :, None]
    key = torch.arange(s.shape[-1], device=dev)
    hidden = key > pos
    if c["window"]:
        hidden = hidden | (key <= pos - c["window"])
    s.masked_fill_(hidden, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, H, G * n, -1), v).view(S, H, G, n, D) / total
    lse = top + torch.log(total)
    seq, at = _tokens(st)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, n, H * G, D)[seq, at]
    lse = lse[..., 0].permute(0, 3, 1, 2).reshape(S, n, H * G)[seq, at]
    return {"out": o.to(st["q"].dtype), "lse": lse}


# ------------------------------------------------------------------ in 64 bits
def _e4m3(v):
    """Values rounded to three fractional bits (ties to even), the smallest step 2^-9."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _quantised(x, fmt):
    """What the codes of a 64-bit row mean before scaling, and the scale."""
    top = x.abs().max(dim=-1).values
    v = x / (top / TOP[fmt]).unsqueeze(-1)
    return (_e4m3(v) if fmt == "f8" else torch.round(v)), top / TOP[fmt]


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        h = st["x"].double() + st["residual"].double()
        y = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / case["hidden"] + EPS) * st["weight"].double()
        if case["out"] == "same":
            return {"out": y, "scales": None, "total": h}
        parts = y.unflatten(-1, (-1, case["group"] or case["hidden"]))
        codes, scales = _quantised(parts, "f8")
        return {"out": codes.flatten(-2), "scales": scales if case["group"] else scales[:, 0], "total": h}
    old, new = _lengths(case)
    table, ps, fmt = st["table"].cpu(), case["page"], case["cache"]

    def held(name, page):
        x = st[name][page] if fmt != "f8" else st[name].view(torch.uint8)[page].view(F8)
        return x.double() if fmt in TYPES else x.double() * st[name + "_scale"][page].double()[..., None]

    def sequence(name, s, first, last):
        """Tokens first to last of sequence s, [tokens, heads, dim]."""
        pages = table[s, : -(-last // ps)].to(st[name].device).long()
        return held(name, pages).permute(0, 2, 1, 3).flatten(0, 1)[first:last]

    if case["kind"] == "read":
        return {n: torch.cat([sequence(n, s, o, o + m) for s, (o, m) in enumerate(zip(old, new))]) for n in ("k", "v")}
    if case["kind"] == "write":
        back = {}
        for name in ("k", "v"):
            x = st["new_" + name].double()
            if fmt in TYPES:
                codes, scales = x, None
            else:
                codes, scales = _quantised(x, fmt)
            if fmt == "i8":
                back[name] = codes * scales.unsqueeze(-1)
                continue
            pool = st[name].double()
            ps_scale = None if scales is None else st[name + "_scale"].double()
            t = 0
            for s, (o, m) in enumerate(zip(old, new)):
                at = torch.arange(o, o + m)
                page, slot = table[s][at // ps].long().to(pool.device), (at % ps).to(pool.device)
                pool[page, :, slot] = codes[t:t + m]
                if scales is not None:
                    ps_scale[page, :, slot] = scales[t:t + m]
                t += m
            back[name], back[name + "_scale"] = pool, ps_scale
        return back
    G, out, lse, t = case["group"], [], [], 0
    for s, (o, m) in enumerate(zip(old, new)):
        k, v = sequence("k", s, 0, o + m), sequence("v", s, 0, o + m)
        at, key = torch.arange(o, o + m, device=k.device)[:, None], torch.arange(o + m, device=k.device)[None]
        seen = (key <= at) & (key > at - case["window"]) if case["window"] else key <= at
        rows_o, rows_l = [], []
        for h in range(case["kv_heads"] * G):
            e = st["q"][t:t + m, h].double() @ k[:, h // G].t() * st["scale"]
            e = torch.where(seen, e, -torch.inf)
            z = torch.logsumexp(e, -1)
            rows_o.append(torch.exp(e - z[:, None]) @ v[:, h // G])
            rows_l.append(z)
        out.append(torch.stack(rows_o, 1))
        lse.append(torch.stack(rows_l, 1))
        t += m
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
