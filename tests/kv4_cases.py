"""Inputs, 64-bit definitions and derived tolerances shared by the CPU and GPU tests of the 4-bit KV cache."""
import math

import torch

from exo_b200 import ops
from exo_b200.ops import kv4


def unpacked(cache):
    """(codes, scales, least values) of every slot of a cache in 64 bits, by walking the format's definition byte by byte:
    ``[n_slots, heads, D]``, ``[n_slots, heads, D / 32]`` twice."""
    d = cache.head_dim
    nb, bs, h, _ = cache.shape
    units = cache.data.cpu()
    per, groups = min(4, d // 32), d // 32
    byte = torch.empty(16, d, dtype=torch.long)
    num = torch.empty(16, groups, dtype=torch.long)
    for tok in range(16):
        for dim in range(d):
            half, r = divmod(dim, 128)
            g, i = divmod(r, 32)
            if cache.kind == "k":
                byte[tok, dim] = ((half * 16 + tok) * 4 + i // 8) * 4 * per + 4 * g + i % 8 // 2
                num[tok, dim // 32] = tok * groups + dim // 32
            else:
                place = 8 * (tok // 8) + 4 * (tok % 2) + tok // 2 % 4
                slot = i // 4 if d == 64 else (i // 4) ^ (4 * (place // 2 % 2))
                byte[tok, dim] = ((half * 16 + place) * 8 + slot) * 2 * per + 2 * g + i % 4 // 2
                num[tok, dim // 32] = (tok // 2 * groups + dim // 32) * 2 + tok % 2
    codes = (units[..., byte].long() >> (4 * (torch.arange(d) % 2))) & 15               # [nb, h, units, 16, D]
    meta = units[..., 8 * d:].contiguous().view(torch.float16).double()
    flat = lambda t: t.permute(0, 2, 3, 1, 4).reshape(nb * bs, h, -1)                   # noqa: E731
    return flat(codes).double(), flat(meta[..., num]), flat(meta[..., d // 2 + num])


def filled_pair(n_blocks, bs, hkv, d, device, seed=0, spread=1.0, offset=0.0):
    """A cache pair holding normal rows (in every slot)."""
    g = torch.Generator().manual_seed(seed)
    kc, vc = (ops.Kv4Cache.zeros(n_blocks, bs, hkv, d, kind) for kind in "kv")
    slots = torch.arange(n_blocks * bs)
    for c in (kc, vc):
        kv4.write(c, slots, torch.randn(n_blocks * bs, hkv, d, generator=g) * spread + offset)
    return ops.Kv4Cache(kc.data.to(device), d, "k"), ops.Kv4Cache(vc.data.to(device), d, "v")


def batch(lens, bs, n_blocks, seed=0, width=None):
    """Block tables over distinct random pages for sequences ``[(new tokens, keys)]``, lengths and offsets."""
    g = torch.Generator().manual_seed(seed + 1)
    pages = [-(-k // bs) for _, k in lens]
    width = max(1, max(pages)) + 1 if width is None else width
    blocks = torch.randperm(n_blocks, generator=g).int()
    assert sum(pages) <= n_blocks
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = blocks[at:at + n]
        at += n
    cu = torch.tensor([sum(x for x, _ in lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    return table, torch.tensor([k for _, k in lens], dtype=torch.int32), cu


def attention64(q, kc, vc, table, lens, cu, scale, window=0, sinks=None):
    """(out, bound) in 64 bits: ``bound`` is how far a kernel may be off before its result is rounded to q's type.

    The kernels keep scores and sums in fp32, and may round to fp16 (2^-11 each): a key, a value, a weight p, and p times a
    scale.  A rounded key moves a logit by at most e = 2^-11 scale sum |q||k|, fp32 sums by (D + 4) 2^-23 of the same sum
    over codes and least values apart; p moves by exp(2 e) - 1 relative (numerator and denominator).  Then
    |error| <= sum p (c n s + c |m|) with c = exp(2 e) - 1 + 3 * 2^-11, plus fp32 sums."""
    T, hq, d = q.shape
    ks, vs = unpacked(kc), unpacked(vc)
    k_all = (ks[0].unflatten(-1, (-1, 32)) * ks[1][..., None] + ks[2][..., None]).flatten(-2)
    v_mag = (vs[0].unflatten(-1, (-1, 32)) * vs[1][..., None] + vs[2][..., None].abs()).flatten(-2)
    v_all = (vs[0].unflatten(-1, (-1, 32)) * vs[1][..., None] + vs[2][..., None]).flatten(-2)
    k_mag = (ks[0].unflatten(-1, (-1, 32)) * ks[1][..., None] + ks[2][..., None].abs()).flatten(-2)
    hkv, bs = kc.shape[2], kc.shape[1]
    out, bound = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    q, table = q.cpu().double(), table.cpu().long()
    for b in range(lens.numel()):
        lo, hi, n = int(cu[b]), int(cu[b + 1]), int(lens[b])
        if hi == lo or n <= 0:
            continue
        pos = torch.arange(n)
        sl = table[b, pos // bs] * bs + pos % bs
        at = torch.arange(n - (hi - lo), n)[:, None]
        seen = pos[None] <= at
        if window:
            seen = seen & (pos[None] > at - window)
        for h in range(hq):
            kvh = h // (hq // hkv)
            x = q[lo:hi, h]
            logit = (x @ k_all[sl, kvh].T * scale).masked_fill(~seen, -math.inf)
            move = scale * (x.abs() @ k_mag[sl, kvh].T) * (2.0 ** -11 + (d + 4) * 2.0 ** -23)
            if sinks is not None:
                p = torch.softmax(torch.cat((logit, sinks.cpu().double()[h].expand(hi - lo, 1)), 1), 1)[:, :n]
            else:
                p = torch.where(seen.any(1, keepdim=True), torch.softmax(logit, 1), torch.zeros_like(logit))
            c = torch.exp(2 * torch.where(seen, move, torch.zeros_like(move)).amax(1, keepdim=True)) - 1 + 3 * 2.0 ** -11
            v = v_all[sl, kvh]
            out[lo:hi, h] = p @ v.nan_to_num()          # a hidden key may hold anything, a NaN that a row sees makes it NaN
            out[lo:hi, h].masked_fill_(seen.double() @ v.isnan().double() > 0, math.nan)
            bound[lo:hi, h] = c * (p @ v_mag[sl, kvh].nan_to_num()) + 1e-6
    return out, bound


def check_attention(got, out, bound):
    step = torch.finfo(got.dtype).eps / 2
    err = (got.cpu().double() - out).abs()
    limit = bound * (1 + step) + step * out.abs()
    assert torch.equal(got.cpu().isnan(), out.isnan())
    worst = torch.where(out.isnan(), torch.zeros_like(err), err / limit.clamp_min(1e-300))
    assert float(worst.max()) <= 1.0, f"off by {float(worst.max()):.3g} of the bound at {tuple(int(i) for i in torch.nonzero(worst == worst.max())[0])}"


def append64(qkv, positions, inv_freq, mscale, n_q, n_kv, d, q_norm, k_norm, eps, v_unit, axes):
    """q, k, v rows of the append in 64 bits."""
    x = qkv.cpu().double().view(-1, n_q + 2 * n_kv, d)
    q, k, v = x[:, :n_q].clone(), x[:, n_q:n_q + n_kv].clone(), x[:, n_q + n_kv:].clone()
    inv_freq, positions = inv_freq.cpu().double(), positions.cpu().double()
    half = inv_freq.numel()
    rms = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)                 # noqa: E731
    if q_norm is not None:
        q, k = rms(q) * q_norm.cpu().double(), rms(k) * k_norm.cpu().double()
    if v_unit:
        v = rms(v)
    for t in (q, k):
        for i in range(half):
            ang = (positions if axes is None else positions[int(axes[i])]) * inv_freq[i]
            c, s = (ang.cos() * mscale)[:, None], (ang.sin() * mscale)[:, None]
            a, b = t[..., i].clone(), t[..., i + half].clone()
            t[..., i], t[..., i + half] = a * c - b * s, b * c + a * s
    return q, k, v


def check_held(cache, slots, x):
    """The rows of a cache at ``slots`` against the exact rows ``x``: every value within half a stored step (the kernel's x is
    off by some 2^-20 of the row's largest, which may tip a tie), the numbers of a group those of the definition or, for the
    same reason, their neighbours."""
    n, s, m = (t[slots.cpu().long()] for t in unpacked(cache))
    g = x.clamp(-65280, 65280).unflatten(-1, (-1, 32))
    slack = g.abs().amax((-1, -2), keepdim=True) * 2.0 ** -19
    held = n.unflatten(-1, (-1, 32)) * s[..., None] + m[..., None]
    assert bool(((held - g).abs() <= s[..., None] / 2 + slack).all())
    # fp16 steps: of the least value (it is at most one below the group's least), and of the scale
    step16 = lambda t: torch.exp2(torch.frexp(t.abs()).exponent.clamp_min(-13).double() - 11)     # noqa: E731
    least, most = g.amin(-1), g.amax(-1)
    assert bool(((m <= least + slack[..., 0]) & (m >= least - step16(least) - slack[..., 0])).all())
    exact = (most - m) / 15
    assert bool(((s >= exact - slack[..., 0]) & (s <= exact + step16(exact) + slack[..., 0])).all())
