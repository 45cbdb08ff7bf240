"""The paged-cache operators of a serving step, as cases that can be timed and compared.

A step of a server that checks drafted tokens (or decodes one token) over a paged KV cache:

- ``slots``: block tables and slot maps from request lengths (``ops.cache_slots``);
- ``rope``: rotary positions of one tensor, forward or backward (``ops.rope``);
- ``cache``: rotary positions of Q and K, and K and V written to their slots (``ops.rope_cache``);
- ``tree``: attention of a tree of drafted tokens over the paged cache (``ops.tree_attn``).

``run`` computes them in elementary torch operations, or, where ``own`` is set, through the
library. Sequence lengths are the quantiles of a range, in an order drawn from the seed, so that
the work of a case does not depend on the seed.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # eight requests decode one token each: the smallest step, all launch latency
        {"name": "slots_step_b8", "op": "slots", "B": 8, "lo": 1024, "hi": 8192, "new_lo": 1,
         "new_hi": 1, "bs": 16},
        # 256 requests with drafted trees of 1 to 16 tokens
        {"name": "slots_draft_b256", "op": "slots", "B": 256, "lo": 0, "hi": 8192, "new_lo": 1,
         "new_hi": 16, "bs": 64},
        # new prompts of up to 4095 tokens, every block newly taken from the pool
        {"name": "slots_prompt_b64", "op": "slots", "B": 64, "lo": 0, "hi": 0, "new_lo": 1,
         "new_hi": 4095, "bs": 16},
        # the query heads of 64 sequences decoding one token each
        {"name": "rope_step_n64", "op": "rope", "N": 64, "H": 32, "D": 128, "rot": 128, "dt": "bf16",
         "inter": False, "inverse": False, "far": 8192, "stretch": 1.0},
        # a prompt far into a stretched context: part of the head, interleaved pairs, odd length
        {"name": "rope_part_n4099", "op": "rope", "N": 4099, "H": 32, "D": 128, "rot": 64,
         "dt": "f16", "inter": True, "inverse": False, "far": 1000000, "stretch": 32.0},
        # the gradient of a training batch of 8 x 4096 tokens
        {"name": "rope_back_n32768", "op": "rope", "N": 32768, "H": 32, "D": 128, "rot": 128,
         "dt": "bf16", "inter": False, "inverse": True, "far": 4096, "stretch": 1.0},
        # 64 sequences with eight drafted tokens each: Q, K rotated, K, V to the cache
        {"name": "cache_draft_n512", "op": "cache", "N": 512, "Hq": 32, "Hkv": 8, "D": 128,
         "rot": 128, "dt": "bf16", "inter": False, "far": 8192, "stretch": 1.0, "bs": 64},
        # a chunk of prompts
        {"name": "cache_prompt_n16384", "op": "cache", "N": 16384, "Hq": 32, "Hkv": 8, "D": 128,
         "rot": 128, "dt": "f16", "inter": True, "far": 131072, "stretch": 8.0, "bs": 16},
        # one sequence, eight drafted tokens, an odd length: latency
        {"name": "tree_b1_t8", "op": "tree", "B": 1, "lo": 1003, "hi": 1003, "t_lo": 8, "t_hi": 8,
         "Hq": 32, "Hkv": 8, "D": 128, "bs": 16, "dt": "bf16", "br": 2},
        # the ordinary serving step: 64 sequences, lengths 1024 to 8192, eight drafted tokens
        {"name": "tree_b64_t8", "op": "tree", "B": 64, "lo": 1024, "hi": 8192, "t_lo": 8, "t_hi": 8,
         "Hq": 32, "Hkv": 8, "D": 128, "bs": 64, "dt": "bf16", "br": 2},
        # single tokens of a few very long contexts
        {"name": "tree_b4_t1_long", "op": "tree", "B": 4, "lo": 131071, "hi": 131071, "t_lo": 1,
         "t_hi": 1, "Hq": 32, "Hkv": 8, "D": 128, "bs": 16, "dt": "f16", "br": 1},
        # large ragged trees of 33 to 64 tokens, eight query heads to a KV head: many rows
        {"name": "tree_b32_t64_g8", "op": "tree", "B": 32, "lo": 2048, "hi": 8192, "t_lo": 33,
         "t_hi": 64, "Hq": 64, "Hkv": 8, "D": 128, "bs": 32, "dt": "bf16", "br": 3},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["slots", "rope", "cache", "tree", "tree"])
    if op == "slots":
        B = _log(rng, 1, 512)
        new_hi = _log(rng, 1, max(1, min(4095, 2 * 131072 // B - 1)))
        hi = rng.choice([0, _log(rng, 1, 8192)])
        return {"op": op, "B": B, "lo": hi // rng.randint(1, 8), "hi": hi,
                "new_lo": rng.randint(1, new_hi), "new_hi": new_hi, "bs": rng.choice([16, 32, 64, 128])}
    dt = rng.choice(["bf16", "f16"])
    if op in ("rope", "cache"):
        D = rng.choice([64, 128])
        rot = rng.choice([D, D // 2, 48])
        far, stretch = _log(rng, 2048, 1000000), rng.choice([1.0, 4.0, 32.0])
        if op == "rope":
            H = rng.choice([1, 4, 7, 8, 32])
            return {"op": op, "N": _log(rng, 1, 32768), "H": H, "D": D, "rot": rot, "dt": dt,
                    "inter": rng.random() < 0.5, "inverse": rng.random() < 0.5, "far": far,
                    "stretch": stretch}
        Hkv = rng.choice([1, 2, 4, 8])
        return {"op": op, "N": _log(rng, 1, 16384), "Hq": Hkv * rng.choice([1, 3, 4]), "Hkv": Hkv,
                "D": D, "rot": rot, "dt": dt, "inter": rng.random() < 0.5, "far": far,
                "stretch": stretch, "bs": rng.choice([16, 32, 64, 128])}
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 5, 7, 8, 16])
    hi = _log(rng, 1, 131072)
    t_hi = _log(rng, 1, 64)
    rows = 64 * 48 * 5120 * 32  # query rows x keys of the largest listed case, at most
    B = _log(rng, 1, max(1, min(64, 4 * 131072 // hi, rows // (t_hi * G * Hkv * hi))))
    return {"op": op, "B": B, "lo": hi // rng.randint(1, 8), "hi": hi, "t_lo": rng.randint(1, t_hi),
            "t_hi": t_hi, "Hq": Hkv * G, "Hkv": Hkv, "D": rng.choice([64, 128, 128]),
            "bs": rng.choice([16, 32, 64, 128]), "dt": dt, "br": rng.randint(1, 4)}


# ---- inputs ------------------------------------------------------------------------------


def _quantiles(n, lo, hi):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case, new):
    """Tokens in the cache and new tokens of each request, before they are put in order."""
    lo, hi = new
    return _quantiles(case["B"], case["lo"], case["hi"]), _quantiles(case["B"], lo, hi)


def _parents(t, br):
    """A complete tree: token i continues token (i - 1) // br, the first one the context."""
    return [(i - 1) // br if i else -1 for i in range(t)]


def _tree_bits(t, br):
    """Per token the tokens that it sees: itself and those that it continues, one bit each."""
    bits = []
    for i, parent in enumerate(_parents(t, br)):
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def _freqs(rot, stretch):
    """Radians per position of each pair. Stretched contexts divide the low frequencies by
    `stretch` and keep the high ones, with a ramp between 32 turns and 1 turn in 4096 tokens."""
    f = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot
    f = 10000.0 ** -f
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return f * (keep + (1 - keep) / stretch) if stretch != 1.0 else f


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dt, gen):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=gen).to(_DTYPES[dt])


def _ints(values, dtype):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = _gen(seed)
    host = torch.Generator().manual_seed(seed)
    s = dict(case)
    if case["op"] == "slots":
        B, bs = case["B"], case["bs"]
        ctx, new = _lengths(case, (case["new_lo"], case["new_hi"]))
        order = torch.randperm(B, generator=host).tolist()
        ctx, new = [ctx[i] for i in order], [new[i] for i in order]
        held = [-(-c // bs) for c in ctx]
        need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
        ids = torch.randperm(sum(need) + 32, generator=host).tolist()
        wide = max(need) + 8
        rows = []
        for h in held:
            rows.append(ids[:h] + [-1] * (wide - h))
            del ids[:h]
        s.update(ctx=_ints(ctx, torch.int32), new=_ints(new, torch.int32),
                 tables=_ints(rows, torch.int32), free=_ints(ids, torch.int32),
                 room=-(-sum(new) // 64) * 64)
        return s
    if case["op"] in ("rope", "cache"):
        n = case["N"]
        s["freqs"] = _freqs(case["rot"], case["stretch"])
        s["scale"] = 1.0 if case["stretch"] == 1.0 else 1.0 + 0.1 * math.log(case["stretch"])
        s["pos"] = torch.randint(case["far"], (n,), device="cuda", generator=gen, dtype=torch.int32)
        if case["op"] == "rope":
            s["x"] = _randn((n, case["H"], case["D"]), case["dt"], gen)
            return s
        for name, heads in (("q", case["Hq"]), ("k", case["Hkv"]), ("v", case["Hkv"])):
            s[name] = _randn((n, heads, case["D"]), case["dt"], gen)
        blocks = -(-n // case["bs"]) + 2
        s["slots"] = torch.randperm(blocks * case["bs"], device="cuda", generator=gen)[:n]
        shape = (blocks, case["bs"], case["Hkv"], case["D"])
        s["kc"], s["vc"] = _randn(shape, case["dt"], gen), _randn(shape, case["dt"], gen)
        return s
    B, bs = case["B"], case["bs"]
    ctx, new = _lengths(case, (case["t_lo"], case["t_hi"]))
    order = torch.randperm(B, generator=host).tolist()
    ctx, new = [ctx[i] for i in order], [new[i] for i in order]
    need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    blocks = sum(need) + 3
    ids = torch.randperm(blocks, generator=host).tolist()
    wide = max(need)
    rows, bits, offsets = [], [], [0]
    for m, n in zip(need, new):
        rows.append(ids[:m] + [-1] * (wide - m))
        del ids[:m]
        bits += _tree_bits(n, case["br"])
        offsets.append(offsets[-1] + n)
    shape = (blocks, bs, case["Hkv"], case["D"])
    s.update(tables=_ints(rows, torch.int32), ctx=_ints(ctx, torch.int32),
             offsets=_ints(offsets, torch.int32), tree=_ints(bits, torch.int64),
             longest=max(c + n for c, n in zip(ctx, new)),
             q=_randn((offsets[-1], case["Hq"], case["D"]), case["dt"], gen),
             kc=_randn(shape, case["dt"], gen), vc=_randn(shape, case["dt"], gen))
    return s


# ---- the operators -----------------------------------------------------------------------


def _slots(s):
    ctx, new, tables, free, bs = s["ctx"].long(), s["new"].long(), s["tables"], s["free"], s["bs"]
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    offsets = torch.cat([zero, new.cumsum(0)])
    held, need = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    taken = torch.cat([zero, (need - held).cumsum(0)])
    col = torch.arange(tables.shape[1], device="cuda")
    pick = (taken[:-1, None] + col - held[:, None]).clamp(0, free.numel() - 1)
    fresh = (col >= held[:, None]) & (col < need[:, None])
    tables.copy_(torch.where(fresh, free[pick], tables))
    n = torch.arange(s["room"], device="cuda")
    b = torch.searchsorted(offsets[1:], n, right=True).clamp(max=ctx.numel() - 1)
    live = n < offsets[-1]
    pos = torch.where(live, ctx[b] + n - offsets[b], 0)
    slots = torch.where(live, tables[b, pos // bs].long() * bs + pos % bs, -1)
    return {"tables": tables, "slots": slots, "positions": pos.int(), "offsets": offsets.int(),
            "used": taken[-1:].int()}


def _rotate(x, pos, freqs, inter, inverse, scale):
    """x [N, H, D] in 32 bits with its first 2 len(freqs) dimensions rotated in pairs."""
    rot = 2 * freqs.numel()
    angle = pos.double()[:, None] * freqs
    cos, sin = (angle.cos() * scale).float()[:, None], (angle.sin() * scale).float()[:, None]
    if inverse:
        sin = -sin
    x = x.float()
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :rot // 2], part[..., rot // 2:])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    part = torch.stack([lo, hi], -1).flatten(-2) if inter else torch.cat([lo, hi], -1)
    return torch.cat([part, x[..., rot:]], -1)


def _rope(s):
    return _rotate(s["x"], s["pos"], s["freqs"], s["inter"], s["inverse"], s["scale"]).to(s["x"].dtype)


def _cache(s):
    turn = (s["pos"], s["freqs"], s["inter"], False, s["scale"])
    s["kc"].flatten(0, 1)[s["slots"]] = _rotate(s["k"], *turn).to(s["k"].dtype)
    s["vc"].flatten(0, 1)[s["slots"]] = s["v"]
    return {"q": _rotate(s["q"], *turn).to(s["q"].dtype), "k_cache": s["kc"], "v_cache": s["vc"]}


def _tree(s):
    B, Hkv, D, bs, T = s["B"], s["Hkv"], s["D"], s["bs"], s["t_hi"]
    G = s["Hq"] // Hkv
    ctx, offsets = s["ctx"].long(), s["offsets"].long()
    new = offsets[1:] - offsets[:-1]
    p = torch.arange(s["longest"], device="cuda")
    held = p < (ctx + new)[:, None]
    slot = torch.where(held, s["tables"][:, p // bs].long() * bs + p % bs, 0)
    k = s["kc"].flatten(0, 1)[slot].float().permute(0, 2, 3, 1)
    v = (s["vc"].flatten(0, 1)[slot].float() * held[:, :, None, None]).transpose(1, 2)
    t = torch.arange(T, device="cuda")
    row = (offsets[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().view(B, T, Hkv, G, D).transpose(1, 2).reshape(B, Hkv, T * G, D)
    j = p - ctx[:, None]
    drafted = (s["tree"][row][:, :, None] >> j.clamp(0, 63)[:, None] & 1).bool() & (j >= 0)[:, None]
    seen = (drafted | (j < 0)[:, None]) & held[:, None]
    seen = seen[:, None, :, None].expand(B, 1, T, G, p.numel()).reshape(B, 1, T * G, -1)
    a = ((q @ k) * D ** -0.5).masked_fill(~seen, -math.inf)
    top = a.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    a = (a - top).exp()
    total = a.sum(-1, keepdim=True)
    o = torch.where(total > 0, (a @ v) / total, 0.0)
    lse = (top + total.log())[..., 0]
    n = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(offsets[1:], n, right=True)
    o = o.view(B, Hkv, T, G, D).transpose(1, 2)[b, n - offsets[b]].reshape(-1, Hkv * G, D)
    lse = lse.view(B, Hkv, T, G).transpose(1, 2)[b, n - offsets[b]].reshape(-1, Hkv * G)
    return {"out": o.to(s["q"].dtype), "lse": lse}


def _own(s):
    from kta_b200 import ops

    if s["op"] == "slots":
        slots, positions, offsets, used = ops.cache_slots(s["ctx"], s["new"], s["tables"], s["free"],
                                                          s["bs"], s["room"])
        return {"tables": s["tables"], "slots": slots, "positions": positions, "offsets": offsets,
                "used": used}
    if s["op"] == "rope":
        return ops.rope(s["x"], s["pos"], s["freqs"], interleaved=s["inter"], inverse=s["inverse"],
                        scale=s["scale"])
    if s["op"] == "cache":
        q = ops.rope_cache(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["freqs"], s["kc"], s["vc"],
                           interleaved=s["inter"], scale=s["scale"])
        return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}
    out, lse = ops.tree_attn(s["q"], s["kc"], s["vc"], s["tables"], s["ctx"], s["offsets"], s["t_hi"],
                             s["tree"])
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"slots": _slots, "rope": _rope, "cache": _cache, "tree": _tree}[state["op"]](state)


def work(case):
    if case["op"] == "slots":
        ctx, new = _lengths(case, (case["new_lo"], case["new_hi"]))
        bs = case["bs"]
        fresh = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        begun = sum(c % bs != 0 for c in ctx)
        # lengths, the blocks begun and those taken; the new table entries, the token map
        return {"bytes": 8 * case["B"] + 4 * begun + 8 * fresh + 12 * sum(new) + 4 * (case["B"] + 2),
                "flops": 0}
    if case["op"] == "rope":
        n = case["N"] * case["H"]
        return {"bytes": 4 * n * case["D"] + 4 * case["N"] + 4 * case["rot"], "flops": 3 * n * case["rot"]}
    if case["op"] == "cache":
        n = case["N"]
        rows = n * (case["Hq"] + 2 * case["Hkv"])
        return {"bytes": 4 * rows * case["D"] + 12 * n + 4 * case["rot"],
                "flops": 3 * n * (case["Hq"] + case["Hkv"]) * case["rot"]}
    ctx, new = _lengths(case, (case["t_lo"], case["t_hi"]))
    D, bs, rows = case["D"], case["bs"], sum(new) * case["Hq"]
    seen = sum(n * c + sum(bin(b & (1 << 64) - 1).count("1") for b in _tree_bits(n, case["br"]))
               for c, n in zip(ctx, new))
    held = sum(ctx) + sum(new)
    blocks = sum(-(-(c + n) // bs) for c, n in zip(ctx, new))
    return {"bytes": 4 * held * case["Hkv"] * D + 4 * rows * D + 4 * rows + 8 * sum(new) + 4 * blocks
            + 8 * case["B"], "flops": 4 * seen * case["Hq"] * D}


# ---- the same in 64 bits -----------------------------------------------------------------


def _exact_slots(s):
    ctx, new, bs = s["ctx"].tolist(), s["new"].tolist(), s["bs"]
    tables, pool = s["tables"].tolist(), s["free"].tolist()
    offsets, slots, positions, used = [0], [], [], 0
    for row, c, n in zip(tables, ctx, new):
        for p in range(c, c + n):
            if p // bs >= -(-c // bs) and (p % bs == 0 or p == c):
                row[p // bs] = pool[used]
                used += 1
            slots.append(row[p // bs] * bs + p % bs)
            positions.append(p)
        offsets.append(offsets[-1] + n)
    pad = s["room"] - len(slots)
    return {"tables": _ints(tables, torch.int32), "slots": _ints(slots + [-1] * pad, torch.int64),
            "positions": _ints(positions + [0] * pad, torch.int32),
            "offsets": _ints(offsets, torch.int32), "used": _ints([used], torch.int32)}


def _exact_turn(x, s, inverse):
    """Each pair as a complex number times scale e^(i angle)."""
    half = s["freqs"].numel()
    y = x.double().clone()
    lo = torch.arange(half, device="cuda")
    lo, hi = (2 * lo, 2 * lo + 1) if s["inter"] else (lo, lo + half)
    angle = torch.outer(s["pos"].double(), s["freqs"])
    turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if inverse else angle)
    z = torch.complex(y[..., lo], y[..., hi]) * turn.unsqueeze(1)
    y[..., lo], y[..., hi] = z.real, z.imag
    return y


def _exact_tree(s):
    G, D = s["Hq"] // s["Hkv"], s["D"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    ctx, offsets = s["ctx"].tolist(), s["offsets"].tolist()
    for i, c in enumerate(ctx):
        a, z = offsets[i], offsets[i + 1]
        blocks = s["tables"][i, :-(-(c + z - a) // s["bs"])].long()
        k = s["kc"][blocks].reshape(-1, s["Hkv"], D)[:c + z - a].double()
        v = s["vc"][blocks].reshape(-1, s["Hkv"], D)[:c + z - a].double()
        sight = torch.zeros(z - a, c + z - a, dtype=torch.bool)
        sight[:, :c] = True
        for t, parent in enumerate(_parents(z - a, s["br"])):
            if parent >= 0:
                sight[t] = sight[parent]
            sight[t, c + t] = True
        sight = sight.to("cuda")
        for h in range(s["Hkv"]):
            q = s["q"][a:z, h * G:(h + 1) * G].double()
            w = torch.einsum("tgd,ld->tgl", q, k[:, h]) / math.sqrt(D)
            w = w.masked_fill(~sight[:, None], -math.inf)
            lse[a:z, h * G:(h + 1) * G] = torch.logsumexp(w, -1)
            out[a:z, h * G:(h + 1) * G] = torch.einsum("tgl,ld->tgd", torch.softmax(w, -1), v[:, h])
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "slots":
        return _exact_slots(s)
    if case["op"] == "rope":
        return _exact_turn(s["x"], s, case["inverse"])
    if case["op"] == "cache":
        k_cache, v_cache = s["kc"].double(), s["vc"].double()
        k_cache.view(-1, case["Hkv"], case["D"])[s["slots"]] = _exact_turn(s["k"], s, False)
        v_cache.view(-1, case["Hkv"], case["D"])[s["slots"]] = s["v"].double()
        return {"q": _exact_turn(s["q"], s, False), "k_cache": k_cache, "v_cache": v_cache}
    return _exact_tree(s)
