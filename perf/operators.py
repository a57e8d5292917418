"""What is measured of the operators on a KV cache held in 4 bits: the append (per-head norm, rotary positions on one or
several axes, quantisation), attention of single tokens and attention of prompts.

A cache is one uint8 tensor ``[blocks, kv heads, block size / 16, 10 D]`` for the keys and one for the values: units of 16
tokens of one head.  32 neighbouring dims of a row form a group with a 16-bit scale ``s`` and least value ``m``; a 4-bit
code ``n`` stands for ``n * s + m``.  A unit is 8 D bytes of codes, then the scales, then the least values (D bytes each);
inside, keys and values are ordered for the kernels' operand registers:

* codes of keys: ``[D / 128][16 tokens][4 t][4 g]`` 32-bit words (``D == 64``: ``[16][4 t][2 g]``), word (t, g) = dims
  ``32 g + 8 t ..+7`` of its 128, lowest nibble first; scales and least values ``[16 tokens][groups]``
* codes of values: ``[D / 128][16 places][8 slots][4 g]`` 16-bit words (``D == 64``: ``[16][8][2]``), word g of slot c =
  dims ``32 g + 4 c' ..+3`` with ``c' = c ^ ((place & 2) << 1)`` (``D == 64``: ``c' = c``); token ``b3 b2 b1 b0`` (its bits)
  stands at place ``b3 b0 b2 b1``; scales and least values ``[8 token pairs][groups][2]``
"""
import math
import random

import torch

own = False

GROUP = 32
LARGEST_ROWS, LARGEST_KEYS, LARGEST_PAIRS = 8192, 400_000, 40_000_000     # limits of draw(): the largest listed cases' work


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    heads8b, heads70b, heads235b = dict(hq=32, hkv=8, d=128), dict(hq=64, hkv=8, d=128), dict(hq=64, hkv=4, d=128)
    oss, wide = dict(hq=64, hkv=8, d=64), dict(hq=16, hkv=2, d=256)
    plain, whole = dict(window=0, sinks=False, bs=16), dict(ragged=False)
    return [
        # one user's next token (Llama-3.1-8B's heads): launch latency
        dict(name="append 1 token", op="append", T=1, rot=128, norm=False, axes=1, bs=16, **heads8b),
        # a decode step of 64 users, heads normalised (Qwen3-235B's heads)
        dict(name="append 64 tokens", op="append", T=64, rot=128, norm=True, axes=1, bs=16, **heads235b),
        # a quarter of wide heads turned (Qwen3-Next's heads), a prompt chunk of odd length
        dict(name="append 4097 wide", op="append", T=4097, rot=64, norm=True, axes=1, bs=16, **wide),
        # a prompt with images: time, height and width positions (Qwen3-VL's heads)
        dict(name="append 8192 3 axes", op="append", T=8192, rot=128, norm=True, axes=3, bs=16, **heads8b),
        # a chat's first answers: one short sequence
        dict(name="decode 1 x 203", op="decode", B=1, len=203, **heads8b, **plain, **whole),
        # the serving batch: 32 sequences around 2048
        dict(name="decode 32 x 2048", op="decode", B=32, len=4095, ragged=True, **heads8b, **plain),
        # one long document, the whole card on one sequence (Llama-3.1-70B's heads)
        dict(name="decode 1 x 131000", op="decode", B=1, len=131000, **heads70b, **plain, **whole),
        # 16 query heads to a key head, a full serving batch
        dict(name="decode 64 x 6000", op="decode", B=64, len=6001, **heads235b, **plain, **whole),
        # attention sinks and 64-wide heads (GPT-OSS's full layers)
        dict(name="decode 40 x 3000 sinks", op="decode", B=40, len=6000, ragged=True, window=0, sinks=True, bs=16, **oss),
        # a whole prompt in one chunk
        dict(name="prompt 8192", op="prompt", B=1, new=8192, cached=0, **heads8b, **plain, **whole),
        # several prompts' chunks of odd lengths behind cached prefixes, sliding window and sinks
        dict(name="prompt 7 ragged window", op="prompt", B=7, new=801, cached=1500, ragged=True, window=128, sinks=True,
             bs=16, **oss),
        # a short follow-up to a long cached document: few rows, many keys (Qwen3-Next's wide heads)
        dict(name="prompt 200 after 30000", op="prompt", B=1, new=200, cached=30000, **wide, **plain, **whole),
    ]


def _spread(rng, lo, hi):
    """Whole numbers spread over their logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    hq, hkv, d = rng.choice([(32, 8, 128), (64, 8, 128), (64, 4, 128), (64, 8, 64), (16, 2, 256), (96, 8, 128), (20, 4, 128),
                             (12, 12, 64), (6, 1, 256)])
    c = dict(hq=hq, hkv=hkv, d=d, bs=rng.choice([16, 16, 32]))
    op = rng.choice(["append", "decode", "prompt"])
    if op == "append":
        return dict(op=op, T=_spread(rng, 1, LARGEST_ROWS * 48 // (hq + 2 * hkv) * 128 // d // 2), rot=rng.choice([d, d // 2, d // 4]),
                    norm=rng.random() < 0.5, axes=rng.choice([1, 1, 3]), **c)
    c.update(window=rng.choice([0, 0, 0, _spread(rng, 20, 2000)]), sinks=rng.random() < 0.3, ragged=rng.random() < 0.6)
    if op == "decode":
        b = _spread(rng, 1, 200)
        return dict(op=op, B=b, len=_spread(rng, 1, min(131000, LARGEST_KEYS * 512 // (hkv * d) // b)), **c)
    b = _spread(rng, 1, 12)
    new = _spread(rng, 2, 4000 // b)
    return dict(op=op, B=b, new=new, cached=rng.choice([0, _spread(rng, 1, max(2, min(20000, LARGEST_PAIRS * 16 // hq // (b * new))))]), **c)


def _lens(c):
    """(new tokens, keys) of each sequence: part of the case, not of the seed."""
    r = random.Random("%s" % sorted((k, v) for k, v in c.items() if k != "name"))
    n, out = c["B"], []
    for _ in range(n):
        if c["op"] == "decode":
            out.append((1, r.randint(1, c["len"]) if c["ragged"] else c["len"]))
        else:
            new = r.randint(1, c["new"]) if c["ragged"] else c["new"]
            out.append((new, new + (r.randint(0, c["cached"]) if c["ragged"] else c["cached"])))
    return out


def _pairs(new, keys, window):
    """Visible (query, key) pairs, and keys that some query sees."""
    w = window or keys
    first = keys - new + 1                                   # keys the first query would see without a window
    full = max(0, min(new, w - first + 1))                   # queries that the window does not cut
    pairs = full * first + full * (full - 1) // 2 + (new - full) * w
    return pairs, min(keys, w + new - 1)


def work(case):
    c = case
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    if c["op"] == "append":
        t = c["T"]
        kept = 10 * d // 16                                  # bytes of one row of one head in the cache
        return {"bytes": t * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * kept + 2 * hkv * d * 2 + 4 * c["axes"] + 4),
                "flops": t * (hq + 2 * hkv) * d * 12}
    nbytes, flops = 0, 0
    for new, keys in _lens(c):
        pairs, seen = _pairs(new, keys, c["window"])
        nbytes += 2 * new * hq * d * 2 + 2 * seen * hkv * 10 * d // 16
        flops += 4 * hq * d * pairs
    return {"bytes": nbytes, "flops": flops}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _random_units(gen, n_blocks, hkv, units, d):
    """Cache contents of rows that are normal with a standard deviation of about one, as a model's keys and values are."""
    data = torch.randint(0, 256, (n_blocks, hkv, units, 10 * d), dtype=torch.uint8, device="cuda", generator=gen)
    n = (n_blocks, hkv, units, d // 2)
    meta = torch.empty(*n[:3], d, dtype=torch.float16, device="cuda")
    scale = 0.16 + 0.24 * torch.rand(n, device="cuda", generator=gen)
    meta[..., :d // 2] = scale
    meta[..., d // 2:] = -scale * (6.5 + 2.0 * torch.rand(n, device="cuda", generator=gen))
    data[..., 8 * d:] = meta.view(torch.uint8)
    return data


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d, hq, hkv, bs = c["d"], c["hq"], c["hkv"], c["bs"]
    if c["op"] == "append":
        t = c["T"]
        n_blocks = -(-t // bs) + 3
        s = dict(c)
        s["qkv"] = torch.randn(t, (hq + 2 * hkv) * d, device="cuda", generator=gen).to(torch.bfloat16)
        s["q_norm"] = (1 + 0.2 * torch.randn(d, device="cuda", generator=gen)).to(torch.bfloat16) if c["norm"] else None
        s["k_norm"] = (1 + 0.2 * torch.randn(d, device="cuda", generator=gen)).to(torch.bfloat16) if c["norm"] else None
        s["inv_freq"] = (500000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])).float()
        start = int(torch.randint(0, 120000, (1,), device="cuda", generator=gen))
        line = torch.arange(t, device="cuda")
        if c["axes"] == 1:           # consecutive tokens, or (few rows) users anywhere in their contexts
            pos = line + start if t > 200 else torch.randint(0, 131072, (t,), device="cuda", generator=gen)
            s["positions"], s["axes"] = pos.int(), None
        else:                        # pictures of 32 x 40 tokens with text between them
            pic, text = line % 1500 < 1280, line + start
            at = torch.where(pic, text - line % 1500, text)
            s["positions"] = torch.stack((at, torch.where(pic, at + line % 1500 // 40, at),
                                          torch.where(pic, at + line % 1500 % 40, at))).int().contiguous()
            s["axes"] = (torch.arange(c["rot"] // 2, device="cuda") % 3).int()
        blocks = torch.randperm(n_blocks, device="cuda", generator=gen)
        s["slots"] = (blocks[line // bs] * bs + line % bs).int()
        s["k"] = _random_units(gen, n_blocks, hkv, bs // 16, d)
        s["v"] = _random_units(gen, n_blocks, hkv, bs // 16, d)
        return s
    lens = _lens(c)
    pages = [-(-keys // bs) for _, keys in lens]
    n_blocks = sum(pages) + 5
    blocks = torch.randperm(n_blocks, device="cuda", generator=gen).int()
    width = max(pages) + 1
    rows = torch.tensor(pages, device="cuda")
    first = torch.cumsum(rows, 0) - rows
    col = torch.arange(width, device="cuda")
    table = torch.where(col < rows[:, None], blocks[(first[:, None] + col).clamp_max(n_blocks - 1)], 0).int()
    new = [n for n, _ in lens]
    total = sum(new)
    s = dict(c, max_q=max(new), max_keys=max(k for _, k in lens))
    s["q"] = (1.5 * torch.randn(total, hq, d, device="cuda", generator=gen)).to(torch.bfloat16)
    s["k"] = _random_units(gen, n_blocks, hkv, bs // 16, d)
    s["v"] = _random_units(gen, n_blocks, hkv, bs // 16, d)
    s["table"] = table.contiguous()
    s["seq_lens"] = torch.tensor([k for _, k in lens], dtype=torch.int32, device="cuda")
    s["cu_q"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["sinks_w"] = torch.randn(hq, device="cuda", generator=gen).to(torch.bfloat16) if c["sinks"] else None
    s["scale"] = d ** -0.5
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return _append_plain(s) if s["op"] == "append" else _attention_plain(s)


def _run_own(s):
    from exo_b200 import ops
    kc, vc = ops.Kv4Cache(s["k"], s["d"], "k"), ops.Kv4Cache(s["v"], s["d"], "v")
    if s["op"] == "append":
        q = ops.qk_rope_append(s["qkv"], s["positions"], s["inv_freq"], 1.0, s["hq"], s["hkv"], s["d"], kc, vc, s["slots"],
                               s["q_norm"], s["k_norm"], 1e-6, axes=s["axes"])
        k, v = ops.kv4_read(kc, vc, s["slots"])
        return q, k, v
    return ops.paged_attention(s["q"], kc, vc, s["table"], s["seq_lens"], s["cu_q"], s["scale"], s["window"], s["sinks_w"],
                               s["max_q"])


def _held(x):
    """The values that a 4-bit cache holds of the rows ``x [..., D]`` (32 bits)."""
    g = x.clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    least = g.amin(-1, keepdim=True)
    m = least.half()
    bits = m.view(torch.int16)
    below = torch.where(bits > 0, bits - 1, torch.where(bits == 0, torch.full_like(bits, -32767), bits + 1)).view(torch.float16)
    m = torch.where(m.float() > least, below, m).float()
    step = (g.amax(-1, keepdim=True) - m) / torch.full_like(m, 15.0)        # a quotient, not a product with a rounded 1/15
    s = step.half()
    s = torch.where(s.float() < step, (s.view(torch.int16) + 1).view(torch.float16), s).float()
    n = torch.where(s > 0, (g - m) / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g)).round().clamp(0, 15)
    return (n * s + m).flatten(-2)


def _append_plain(s):
    d, hq, hkv, half = s["d"], s["hq"], s["hkv"], s["rot"] // 2
    x = s["qkv"].float().unflatten(1, (-1, d))
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        w = torch.cat((s["q_norm"].float().expand(hq, d), s["k_norm"].float().expand(hkv, d)))
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    p = s["positions"].double()
    p = p[:, None] if s["axes"] is None else p[s["axes"].long()].T
    angle = p * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = qk[..., :half], qk[..., half:2 * half]
    qk = torch.cat((a * cos - b * sin, b * cos + a * sin, qk[..., 2 * half:]), -1)
    return qk[:, :hq].to(torch.bfloat16), _held(qk[:, hq:]).to(torch.bfloat16), _held(v).to(torch.bfloat16)


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2).float()


def _unpack_keys(u, d):
    """Units ``[..., 10 D]`` -> rows ``[..., 16, D]``."""
    half, g = (d // 128, 4) if d > 64 else (1, 2)
    n = _nibbles(u[..., :8 * d]).unflatten(-1, (half, 16, 4, g, 8))                   # half, token, t, g, dim
    n = n.movedim(-5, -4).movedim(-2, -3)                                             # token, half, g, t, dim
    meta = u[..., 8 * d:].contiguous().view(torch.float16).float().unflatten(-1, (2, 16, half * g, 1))
    x = n.flatten(-2).flatten(-3, -2) * meta[..., 0, :, :, :] + meta[..., 1, :, :, :]
    return x.flatten(-2)


def _unpack_values(u, d):
    half, g = (d // 128, 4) if d > 64 else (1, 2)
    n = _nibbles(u[..., :8 * d]).unflatten(-1, (half, 16, 8, g, 4))                   # half, place, slot, g, dim
    token = torch.arange(16, device=u.device)
    place = (token & 8) | ((token & 1) << 2) | ((token >> 1) & 3)
    slot = torch.arange(8, device=u.device).expand(16, 8)
    if d > 64:
        slot = slot ^ ((place & 2) << 1)[:, None]
    n = n[..., :, place[:, None], slot, :, :]                                         # half, token, c, g, dim
    n = n.movedim(-5, -4).movedim(-2, -3)                                             # token, half, g, c, dim
    meta = u[..., 8 * d:].contiguous().view(torch.float16).float().unflatten(-1, (2, 8, half * g, 2))
    meta = meta.movedim(-1, -2).flatten(-3, -2)[..., None]                            # scales / least values, token, group
    x = n.flatten(-2).flatten(-3, -2) * meta[..., 0, :, :, :] + meta[..., 1, :, :, :]
    return x.flatten(-2)


def _attention_plain(s):
    d, hq, hkv = s["d"], s["hq"], s["hkv"]
    pages = s["table"][:, :-(-s["max_keys"] // s["bs"])].long()
    k = _unpack_keys(s["k"][pages], d).movedim(2, 1).flatten(2, 4)                    # sequence, head, key, dim
    v = _unpack_values(s["v"][pages], d).movedim(2, 1).flatten(2, 4)
    n_keys, new = k.shape[2], s["cu_q"].diff()
    step = torch.arange(s["max_q"], device="cuda")
    rows = (s["cu_q"][:-1, None] + step).clamp_max(s["q"].shape[0] - 1)
    q = s["q"][rows].float().unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4)           # sequence, kv head, head, row, dim
    sc = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (-1, s["max_q"])) * s["scale"]
    at = (s["seq_lens"] - new)[:, None] + step                                        # position of each row
    key = torch.arange(n_keys, device="cuda")
    seen = key <= at[..., None]
    if s["window"]:
        seen &= key > at[..., None] - s["window"]
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    if s["sinks_w"] is not None:
        sink = s["sinks_w"].float().view(1, hkv, -1, 1, 1)
        top = torch.maximum(top, sink)
    sc = sc.sub_(top).exp_()
    den = sc.sum(-1, keepdim=True)
    if s["sinks_w"] is not None:
        den = den + (sink - top).exp()
    o = (sc.flatten(2, 3) @ v).unflatten(2, (-1, s["max_q"])) / den
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                        # sequence, row, head, dim
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["cu_q"][1:].contiguous(), token.int(), right=True)
    return o[seq, token - s["cu_q"][seq]].to(torch.bfloat16)


# ---- the same from the definition, in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _append_exact(s) if s["op"] == "append" else _attention_exact(s)


def _rounded(x, up):
    """The nearest 16-bit number not below (above) ``x``, both in 64 bits."""
    e = torch.frexp(x.abs()).exponent.clamp_min(-13).double()
    ulp = torch.exp2(e - 11)
    return (torch.ceil(x / ulp) if up else torch.floor(x / ulp)) * ulp


def _held_exact(x):
    out = torch.empty_like(x)
    for i in range(0, x.shape[-1], GROUP):
        g = x[..., i:i + GROUP]
        m = _rounded(g.min(-1, keepdim=True).values, False)
        sc = _rounded((g.max(-1, keepdim=True).values - m) / 15, True)
        out[..., i:i + GROUP] = torch.where(sc > 0, torch.round((g - m) / sc.clamp_min(1e-300)), 0.0 * g) * sc + m
    return out


def _append_exact(s):
    d, hq, hkv, rot = s["d"], s["hq"], s["hkv"], s["rot"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    parts = [x[:, :hq].clone(), x[:, hq:hq + hkv].clone(), x[:, hq + hkv:].clone()]
    for part, w in ((parts[0], s["q_norm"]), (parts[1], s["k_norm"])):
        if w is not None:
            part /= torch.sqrt((part * part).sum(-1, keepdim=True) / d + 1e-6)
            part *= w.double()
        turned = part.clone()
        for i in range(rot // 2):
            pos = s["positions"] if s["axes"] is None else s["positions"][int(s["axes"][i])]
            phase = (pos.double() * float(s["inv_freq"][i]))[:, None]
            z = torch.polar(torch.ones_like(phase), phase) * torch.complex(part[..., i], part[..., i + rot // 2])
            turned[..., i], turned[..., i + rot // 2] = z.real, z.imag
        part.copy_(turned)
    return parts[0], _held_exact(parts[1]), _held_exact(parts[2])


def _places(d, values):
    """(byte, shift, scale, least): where the code of (token, dim) and its group's two numbers stand in a unit, by index."""
    byte, shift, scale = [], [], []
    groups = d // GROUP
    for tok in range(16):
        for x in range(d):
            h, r = divmod(x, 128)
            g, i = divmod(r, 32)
            per = min(4, groups)
            if not values:
                at = ((h * 16 + tok) * 4 + i // 8) * per * 4 + g * 4 + i % 8 // 2
                byte.append(at), shift.append(4 * (i % 2))
                scale.append(tok * groups + x // 32)
            else:
                place = (tok // 8) * 8 + (tok % 2) * 4 + (tok // 2) % 4
                slot = i // 4 if d == 64 or place // 2 % 2 == 0 else (i // 4 + 4) % 8
                at = ((h * 16 + place) * 8 + slot) * per * 2 + g * 2 + i % 4 // 2
                byte.append(at), shift.append(4 * (i % 2))
                scale.append((tok // 2 * groups + x // 32) * 2 + tok % 2)
    return tuple(torch.tensor(t, device="cuda") for t in (byte, shift, scale))


def _rows_exact(units, d, values):
    """Units ``[n, 10 D]`` -> rows ``[n * 16, D]`` in 64 bits."""
    byte, shift, scale = _places(d, values)
    code = (units[:, byte].long() >> shift) & 15
    meta = units[:, 8 * d:].contiguous().view(torch.float16).double()
    return (code * meta[:, scale] + meta[:, d // 2 + scale]).view(-1, d)


def _attention_exact(s):
    d, hq, hkv, bs = s["d"], s["hq"], s["hkv"], s["bs"]
    per = hq // hkv
    out = torch.zeros(s["q"].shape[0], hq, d, dtype=torch.float64, device="cuda")
    lens, cu = s["seq_lens"].tolist(), s["cu_q"].tolist()
    if sum(_pairs(cu[b + 1] - cu[b], lens[b], s["window"])[0] for b in range(s["B"])) * hq * d > 1e13:
        return None
    for b in range(s["B"]):
        n, first = lens[b], cu[b]
        blocks = s["table"][b, :-(-n // bs)].long()
        for h in range(hkv):
            k = _rows_exact(s["k"][blocks, h].flatten(0, 1), d, False)[:n]
            v = _rows_exact(s["v"][blocks, h].flatten(0, 1), d, True)[:n]
            for lo in range(first, cu[b + 1], 1024):
                hi = min(cu[b + 1], lo + 1024)
                pos = torch.arange(lo - first, hi - first, device="cuda") + n - (cu[b + 1] - first)
                key = torch.arange(n, device="cuda")
                hidden = key[None] > pos[:, None]
                if s["window"]:
                    hidden |= key[None] <= pos[:, None] - s["window"]
                for j in range(h * per, (h + 1) * per):
                    logit = (s["q"][lo:hi, j].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
                    if s["sinks_w"] is not None:
                        logit = torch.cat((logit, s["sinks_w"][j].double().expand(hi - lo, 1)), 1)
                    p = torch.softmax(logit, 1)[:, :n]
                    out[lo:hi, j] = p @ v
    return out
