"""Cases of the 4-bit serving operators, for measuring them.

Four operators, each as ``run`` calls it when ``own`` is true, and in elementary torch operations
when it is false:

  linear   products with 4-bit weights and group scales (``int4_linear.int4_linear``)
  attend   decode attention over a 4-bit KV cache (``ops.decode_attention_int4``)
  append   RoPE + append of new tokens to a 4-bit KV cache, and the values that the cache then
           holds for them (``ops.rope_kv_append_int4``, ``ops.kv_read_int4``)
  read     a stretch of a 4-bit KV cache in 16 bits, as a later prompt chunk needs it
           (``ops.kv_read_int4``)

Formats.  A cache row of D dims is D/2 bytes -- byte j holds dim j in its low and dim j + D/2 in its
high four bits -- and four 16-bit numbers (s0, m0, s1, m1): a code c of the lower half stands for
s0 * c + m0, one of the upper half for s1 * c + m1.  A weight row of k columns is k/2 bytes (column
2j low, 2j + 1 high), with s and m per group of columns.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # -- products with 4-bit weights -------------------------------------
        # output projection of the 7B shape, one sequence: the smallest call, launch latency counts
        {"name": "o_proj, 1 token", "op": "linear", "tokens": 1, "n": 4096, "k": 4096, "group": 128,
         "epilogue": "residual", "type": "bf16"},
        # gate/up of the 7B shape for four sequences, with the SiLU * up epilogue
        {"name": "gate_up, 4 tokens", "op": "linear", "tokens": 4, "n": 11008, "k": 4096,
         "group": 128, "epilogue": "swiglu", "type": "bf16"},
        # odd row count, more than one tile of tokens, short groups
        {"name": "1003 rows, 13 tokens, fp16", "op": "linear", "tokens": 13, "n": 1003, "k": 4160,
         "group": 64, "epilogue": "store", "type": "fp16"},
        # the 128,256-row vocabulary projection of one sequence: the largest weight
        {"name": "lm_head, 1 token", "op": "linear", "tokens": 1, "n": 128256, "k": 4096,
         "group": 128, "epilogue": "store", "type": "bf16"},
        # -- decode attention over a 4-bit cache -----------------------------
        # one chat of about a thousand tokens, 7B heads: latency
        {"name": "1 sequence, 1000 keys", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 32,
         "dim": 128, "cap": 1064, "shortest": 1000, "longest": 1000, "layout": "dense",
         "type": "bf16"},
        # a serving batch of mixed lengths, 7B heads
        {"name": "32 sequences up to 4096", "op": "attend", "batch": 32, "heads": 32,
         "kv_heads": 32, "dim": 128, "cap": 4096, "shortest": 1, "longest": 4096,
         "layout": "dense", "type": "bf16"},
        # few long documents with shared KV heads (64 heads on 8, as in 70B)
        {"name": "3 sequences of 60000, 64:8", "op": "attend", "batch": 3, "heads": 64,
         "kv_heads": 8, "dim": 128, "cap": 60017, "shortest": 59000, "longest": 60017,
         "layout": "dense", "type": "bf16"},
        # packed cache of odd capacities, small heads, an empty sequence among them
        {"name": "ragged, 17 sequences, D=64", "op": "attend", "batch": 17, "heads": 12,
         "kv_heads": 6, "dim": 64, "cap": 1501, "shortest": 0, "longest": 1501,
         "layout": "ragged", "type": "fp16"},
        # -- append, and the rows as the cache holds them --------------------
        # the decode step of 32 sequences
        {"name": "append 32 x 1", "op": "append", "batch": 32, "seq": 1, "heads": 32,
         "kv_heads": 32, "dim": 128, "cap": 616, "layout": "dense", "type": "bf16"},
        # the prefill of four 2048-token prompts, 32 heads on 8
        {"name": "append 4 x 2048", "op": "append", "batch": 4, "seq": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 2304, "layout": "ragged", "type": "bf16"},
        # -- the cache read back for the next prompt chunk -------------------
        {"name": "read 3 x 777, D=64", "op": "read", "batch": 3, "seq": 777, "kv_heads": 6,
         "dim": 64, "cap": 1024, "layout": "ragged", "type": "fp16"},
        {"name": "read 2 x 16000", "op": "read", "batch": 2, "seq": 16000, "kv_heads": 32,
         "dim": 128, "cap": 16384, "layout": "dense", "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "attend", "attend", "append", "read"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "linear":
        group = rng.choice([32, 64, 128])
        unit = max(group, 64)
        k = unit * _log(rng, 1, 14336 // unit)
        epilogue = rng.choice(["store", "residual", "swiglu"])
        n = _log(rng, 17, min(128256, 128256 * 4096 // k) // (2 if epilogue == "swiglu" else 1))
        return {"op": op, "tokens": _log(rng, 1, 64), "n": n, "k": k, "group": group,
                "epilogue": epilogue, "type": kind}
    kv_heads = rng.choice([1, 2, 5, 8, 16, 32])
    shared = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 128, 128])
    layout = rng.choice(["dense", "ragged"])
    if op == "attend":
        cap = _log(rng, 1, 131072)
        batch = _log(rng, 1, max(1, min(64, 2 ** 22 // (cap * kv_heads))))
        longest = rng.randint((cap + 1) // 2, cap)
        return {"op": op, "batch": batch, "heads": kv_heads * shared, "kv_heads": kv_heads,
                "dim": dim, "cap": cap, "shortest": rng.randint(0, longest), "longest": longest,
                "layout": layout, "type": kind}
    seq = _log(rng, 1, 8192)
    batch = _log(rng, 1, max(1, min(64, 2 ** 18 // (seq * kv_heads))))
    case = {"op": op, "batch": batch, "seq": seq, "heads": kv_heads * shared, "kv_heads": kv_heads,
            "dim": dim, "cap": seq + rng.randint(0, 300), "layout": layout, "type": kind}
    if op == "read":
        del case["heads"]
    return case


def _lengths(case):
    """Keys of each sequence: spread over [shortest, longest], both ends among them; a matter of the
    case alone."""
    r = random.Random(case["batch"] * 7919 + case["longest"])
    got = [r.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    got[0] = case["longest"]
    if case["batch"] > 1:
        got[-1] = case["shortest"]
    return got


def _capacities(case):
    """Rows that each sequence of a packed cache owns: odd numbers of them, at most `cap`."""
    if case["op"] == "attend":
        r = random.Random(case["cap"])
        return [min(case["cap"], max(1, n + r.randint(0, 9))) for n in _lengths(case)]
    return [case["cap"] - b % 2 if case["cap"] > case["seq"] else case["cap"]
            for b in range(case["batch"])]


def _starts(case):
    """First position that each row of the batch appends or reads: sequences stand at different
    places."""
    caps = _capacities(case) if case["layout"] == "ragged" else [case["cap"]] * case["batch"]
    return [(37 * b) % (c - case["seq"] + 1) for b, c in enumerate(caps)]


def work(case):
    if case["op"] == "linear":
        rows = case["n"] * (2 if case["epilogue"] == "swiglu" else 1)
        moved = rows * case["k"] / 2 + 4 * rows * (case["k"] // case["group"])
        moved += 2 * case["tokens"] * (case["k"] + case["n"])
        if case["epilogue"] == "residual":
            moved += 2 * case["tokens"] * case["n"]
        return {"bytes": moved, "flops": 2 * case["tokens"] * rows * case["k"]}
    kv, dim = case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        keys = sum(_lengths(case))
        return {"bytes": keys * kv * (dim + 16) + 4 * case["batch"] * case["heads"] * dim,
                "flops": 4 * keys * case["heads"] * dim}
    tokens = case["batch"] * case["seq"]
    rows = tokens * kv
    if case["op"] == "read":
        return {"bytes": rows * (dim + 16) + 4 * rows * dim + 8 * tokens, "flops": 4 * rows * dim}
    heads = case["heads"]
    moved = 2 * tokens * (heads + 2 * kv) * dim + 2 * tokens * heads * dim + 8 * tokens
    moved += rows * (dim + 16) + 4 * rows * dim
    return {"bytes": moved, "flops": 3 * tokens * (heads + kv) * dim + 8 * rows * dim}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _quantised_weight(gen, rows, k, group, kind):
    """Codes [rows, k/2] and s, m [rows, k/group] of a weight of the usual spread, in stretches of
    rows."""
    codes = torch.empty(rows, k // 2, dtype=torch.uint8, device=DEV)
    s = torch.empty(rows, k // group, dtype=kind, device=DEV)
    m = torch.empty(rows, k // group, dtype=kind, device=DEV)
    for at in range(0, rows, 16384):
        n = min(16384, rows - at)
        w = torch.randn(n, k // group, group, device=DEV, generator=gen) * 0.02
        lo = w.amin(-1).to(kind)
        sc = ((w.amax(-1) - lo.float()) / 15).to(kind)
        c = ((w - lo.float()[..., None]) / sc.float()[..., None]).round().clamp_(0, 15)
        c = c.to(torch.uint8).view(n, k // 2, 2)
        codes[at:at + n] = c[..., 0] | (c[..., 1] << 4)
        s[at:at + n], m[at:at + n] = sc, lo
    return codes, s, m


def _held_rows(gen, shape, dim, kind, spread):
    """A cache's codes and numbers for values around zero of about `spread`, as quantised rows of
    such values have them."""
    codes = torch.randint(0, 256, (*shape, dim // 2), dtype=torch.uint8, device=DEV, generator=gen)
    # the range of dim/2 normal values is about 4.7 times their spread; no two rows alike
    s = (torch.rand(*shape, 2, device=DEV, generator=gen) * 0.5 + 0.75) * (spread * 4.7 / 15)
    m = -7.5 * s * (torch.rand(*shape, 2, device=DEV, generator=gen) * 0.4 + 0.8)
    return codes, torch.stack([s[..., 0], m[..., 0], s[..., 1], m[..., 1]], -1).to(kind)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] == "linear":
        swiglu = case["epilogue"] == "swiglu"
        rows = case["n"] * (2 if swiglu else 1)
        codes, s, m = _quantised_weight(gen, rows, case["k"], case["group"], kind)
        st = {"x": torch.randn(case["tokens"], case["k"], device=DEV, generator=gen).to(kind),
              "codes": codes, "s": s, "m": m}
        if case["epilogue"] == "residual":
            st["resid"] = torch.randn(case["tokens"], case["n"], device=DEV, generator=gen).to(kind)
        if own:
            from llama_pure_compute_b200.int4_linear import Int4Weight
            st["weight"] = Int4Weight.from_codes(codes, s, m, group_size=case["group"],
                                                 layout="swiglu" if swiglu else "linear")
        return {"case": case, **st}
    kv, dim, batch = case["kv_heads"], case["dim"], case["batch"]
    ragged = case["layout"] == "ragged"
    st = {"base": None, "caps": None}
    if ragged:
        caps = _capacities(case)
        bases = [sum(caps[:b]) for b in range(batch)]
        st["base"] = torch.tensor(bases, dtype=torch.int64, device=DEV)
        st["caps"] = torch.tensor(caps, dtype=torch.int32, device=DEV)
        shape = (kv, sum(caps))
    else:
        shape = (batch, kv, case["cap"])
    # keys carry the rotation and spread wider than values
    st["kc"], st["ks"] = _held_rows(gen, shape, dim, kind, 1.3)
    st["vc"], st["vs"] = _held_rows(gen, shape, dim, kind, 0.8)
    if case["op"] == "attend":
        st["q"] = torch.randn(batch, case["heads"], dim, device=DEV, generator=gen).to(kind)
        st["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    else:
        at = torch.tensor(_starts(case), dtype=torch.int64, device=DEV)
        st["pos"] = at[:, None] + torch.arange(case["seq"], device=DEV)
    if case["op"] == "append":
        width = (case["heads"] + 2 * kv) * dim
        st["qkv"] = torch.randn(batch, case["seq"], width, device=DEV, generator=gen).to(kind)
        # the model's rotation tables, [positions, dim] in the data's type
        turn = 10000.0 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
        angle = torch.arange(case["cap"], device=DEV, dtype=torch.float64)[:, None] * turn
        st["cos"] = angle.cos().repeat(1, 2).to(kind)
        st["sin"] = angle.sin().repeat(1, 2).to(kind)
    if own:
        from llama_pure_compute_b200 import ops
        st["kv"] = ops.Int4KV(st["kc"], st["ks"], st["vc"], st["vs"], st["base"], st["caps"],
                              case["cap"] if ragged else None)
        if case["op"] == "attend":
            st["workspace"] = ops.decode_attention_int4_workspace(st["kv"], batch, case["heads"])
    return {"case": case, **st}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(st):
    from llama_pure_compute_b200 import int4_linear, ops
    case = st["case"]
    if case["op"] == "linear":
        return int4_linear.int4_linear(st["x"], st["weight"], case["epilogue"], st.get("resid"))
    if case["op"] == "attend":
        return ops.decode_attention_int4(st["q"], st["kv"], st["lens"], workspace=st["workspace"])
    if case["op"] == "read":
        k, v = ops.kv_read_int4(st["kv"], st["pos"])
        return {"k": k, "v": v}
    q = ops.rope_kv_append_int4(st["qkv"], st["pos"], st["cos"], st["sin"], st["kv"], case["heads"])
    k, v = ops.kv_read_int4(st["kv"], st["pos"])
    return {"q": q, "k": k, "v": v}


def _values(codes, numbers):
    """fp32 values [..., D] of cache rows."""
    n = numbers.float()
    low = (codes & 15).float() * n[..., 0:1] + n[..., 1:2]
    high = (codes >> 4).float() * n[..., 2:3] + n[..., 3:4]
    return torch.cat([low, high], -1)


def _rows(st, t, pos):
    """Rows of the cache tensor t at positions [B, n], as [B, kv heads, n, ...]."""
    if st["base"] is not None:
        return t[:, st["base"][:, None] + pos].transpose(0, 1)
    b = torch.arange(pos.shape[0], device=DEV)[:, None]
    return t[b, :, pos].transpose(1, 2)


def _plain(st):
    case = st["case"]
    kind = TYPES[case["type"]]
    if case["op"] == "linear":
        k, group = case["k"], case["group"]
        c = torch.stack([st["codes"] & 15, st["codes"] >> 4], -1).float().view(-1, k // group, group)
        w = (c * st["s"].float()[..., None] + st["m"].float()[..., None]).view(-1, k)
        y = st["x"].float() @ w.t()
        if case["epilogue"] == "residual":
            y = st["resid"].float() + y
        if case["epilogue"] == "swiglu":
            gate, up = y[:, :case["n"]], y[:, case["n"]:]
            y = gate / (1 + torch.exp(-gate)) * up
        return y.to(kind)
    if case["op"] == "read":
        return {"k": _values(_rows(st, st["kc"], st["pos"]), _rows(st, st["ks"], st["pos"])).to(kind),
                "v": _values(_rows(st, st["vc"], st["pos"]), _rows(st, st["vs"], st["pos"])).to(kind)}
    if case["op"] == "append":
        return _plain_append(st, case, kind)
    batch, kv, dim = case["batch"], case["kv_heads"], case["dim"]
    longest = case["longest"]
    if longest == 0:
        return torch.zeros_like(st["q"])
    held = [st["kc"], st["ks"], st["vc"], st["vs"]]
    if st["base"] is not None:
        # rows past a sequence's end belong to others: they are masked, and kept inside the tensor
        at = st["base"][:, None] + torch.arange(longest, device=DEV)
        at = at.clamp(max=st["kc"].shape[1] - 1)
        held = [t[:, at].transpose(0, 1) for t in held]
    else:
        held = [t[:, :, :longest] for t in held]
    q = st["q"].float().view(batch, kv, -1, dim)
    score = torch.matmul(q, _values(held[0], held[1]).transpose(2, 3)) * dim ** -0.5
    seen = torch.arange(longest, device=DEV) < st["lens"][:, None, None, None]
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _values(held[2], held[3])) / torch.where(total == 0, total + 1, total)
    return out.view(batch, -1, dim).to(kind)


def _plain_append(st, case, kind):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    batch, seq = case["batch"], case["seq"]
    x = st["qkv"].float().view(batch, seq, heads + 2 * kv, dim)
    turned, v = x[:, :, :heads + kv], x[:, :, heads + kv:]
    cos, sin = st["cos"][st["pos"]].float()[:, :, None], st["sin"][st["pos"]].float()[:, :, None]
    low, high = turned[..., :dim // 2], turned[..., dim // 2:]
    half = torch.cat([-high, low], -1)
    turned = (turned * cos + half * sin).to(kind)
    q, k = turned[:, :, :heads], turned[:, :, heads:].float()
    got = {"q": q.transpose(1, 2).contiguous()}
    for name, rows, codes, numbers in (("k", k, st["kc"], st["ks"]), ("v", v, st["vc"], st["vs"])):
        g = rows.reshape(batch, seq, kv, 2, dim // 2)
        m = g.amin(-1)
        s = ((g.amax(-1) - m) / 15).to(kind).float()
        s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
        c = torch.round((g - m[..., None]) * (1 / s)[..., None]).clamp(0, 15)
        c = torch.where(s[..., None] == 0, torch.zeros_like(c), c).to(torch.uint8)
        byte = c[..., 0, :] | (c[..., 1, :] << 4)
        number = torch.stack([s[..., 0], m[..., 0], s[..., 1], m[..., 1]], -1).to(kind)
        if st["base"] is not None:
            at = st["base"][:, None] + st["pos"]
            codes[:, at], numbers[:, at] = byte.permute(2, 0, 1, 3), number.permute(2, 0, 1, 3)
        else:
            b = torch.arange(batch, device=DEV)[:, None]
            codes[b, :, st["pos"]], numbers[b, :, st["pos"]] = byte, number
        got[name] = _values(_rows(st, codes, st["pos"]), _rows(st, numbers, st["pos"])).to(kind)
    return got


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _wide_rows(codes, numbers):
    half = codes.shape[-1]
    n = numbers.double()
    got = torch.empty(*codes.shape[:-1], 2 * half, dtype=torch.float64, device=codes.device)
    got[..., :half] = n[..., 1:2] + n[..., 0:1] * codes.remainder(16).double()
    got[..., half:] = n[..., 3:4] + n[..., 2:3] * codes.div(16, rounding_mode="floor").double()
    return got


def _once(x):
    """The fp32 number nearest to each value: the operator's definition names these roundings."""
    return x.float().double()


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        x, group = st["x"].double(), case["group"]
        parts = x.view(case["tokens"], -1, group)
        y = torch.empty(case["tokens"], st["codes"].shape[0], dtype=torch.float64, device=DEV)
        for at in range(0, y.shape[1], 8192):
            b = st["codes"][at:at + 8192]
            even = torch.einsum("tgj,ngj->ngt", parts[..., 0::2],
                                b.remainder(16).double().view(b.shape[0], -1, group // 2))
            odd = torch.einsum("tgj,ngj->ngt", parts[..., 1::2],
                               (b // 16).double().view(b.shape[0], -1, group // 2))
            s, m = st["s"][at:at + 8192].double(), st["m"][at:at + 8192].double()
            y[:, at:at + 8192] = (torch.einsum("ng,ngt->tn", s, even + odd)
                                  + parts.sum(-1) @ m.t())
        if case["epilogue"] == "residual":
            y += st["resid"].double()
        if case["epilogue"] == "swiglu":
            y = y[:, :case["n"]] * torch.sigmoid(y[:, :case["n"]]) * y[:, case["n"]:]
        return y
    kv, dim, batch = case["kv_heads"], case["dim"], case["batch"]

    def stretch(codes, numbers, b, lo, hi):
        if case["layout"] == "ragged":
            at = int(st["base"][b])
            return _wide_rows(codes[:, at + lo:at + hi], numbers[:, at + lo:at + hi])
        return _wide_rows(codes[b, :, lo:hi], numbers[b, :, lo:hi])

    if case["op"] == "attend":
        out = torch.zeros(batch, case["heads"], dim, dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lengths(case)):
            if n:
                q = st["q"][b].double().view(kv, -1, dim)
                p = torch.softmax(q @ stretch(st["kc"], st["ks"], b, 0, n).mT / math.sqrt(dim), -1)
                out[b] = (p @ stretch(st["vc"], st["vs"], b, 0, n)).view(-1, dim)
        return out
    starts, seq = _starts(case), case["seq"]
    if case["op"] == "read":
        return {n: torch.stack([stretch(st[n + "c"], st[n + "s"], b, lo, lo + seq)
                                for b, lo in enumerate(starts)]) for n in ("k", "v")}
    heads, half, kind = case["heads"], dim // 2, TYPES[case["type"]]
    x = st["qkv"].double().view(batch, seq, -1, dim).transpose(1, 2)
    a, b = x[:, :heads + kv, :, :half], x[:, :heads + kv, :, half:]
    cos, sin = (st[n][st["pos"]].double()[:, None] for n in ("cos", "sin"))
    turned = torch.empty_like(x[:, :heads + kv])
    turned[..., :half] = _once(_once(a * cos[..., :half]) - _once(b * sin[..., :half]))
    turned[..., half:] = _once(_once(b * cos[..., half:]) + _once(a * sin[..., half:]))
    turned = turned.to(kind).double()
    got = {"q": turned[:, :heads]}
    for name, rows in (("k", turned[:, heads:]), ("v", x[:, heads + kv:])):
        held = torch.empty_like(rows)
        for part in (slice(0, half), slice(half, dim)):
            g = rows[..., part]
            lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            s = _once(_once(hi - lo) / 15).to(kind).double()
            s = s * (s >= 2.0 ** -126)
            inverse = _once(1 / torch.where(s == 0, torch.ones_like(s), s))
            c = torch.round(_once(_once(g - lo) * inverse)).clamp(0, 15) * (s != 0)
            held[..., part] = lo + s * c
        got[name] = held
    return got
