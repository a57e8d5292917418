"""A paged KV cache held in 4 bits: its container, the layout of its bytes, and the fp32 definition of its operators.

The reference quantises its KV cache on request (``kv_bits`` / ``kv_group_size``,
``src/exo/worker/engines/mlx/generator/generate.py:197-202``: affine groups, as MLX quantises weights).  Here the cache is
written in 4 bits from the start, by the kernel that normalises and rotates the keys, and read by attention kernels that
never hold it in more bits than a tile at a time.

Format.  32 neighbouring dims of one head's row form a group.  ``m`` is the group's least value rounded DOWN to fp16, ``s``
is ``(max - m) / 15`` rounded UP to fp16, the code of ``x`` is ``n = rint((x - m) / s)`` in 0..15 (0 where ``s == 0``) and
stands for ``n * s + m``: rounding both numbers outwards keeps every value inside the codes' range, so it is off by at most
``s / 2``.  Values are clamped to +-65280 first (``15 s + m`` then fits fp16); a NaN makes the whole row of that head NaN.  5 bits a
value in all, 0.31 of a bf16 cache.

Storage.  ``data [n_blocks, kv heads, block_size / 16, 10 D]`` bytes; the last axis is a *unit*: 16 tokens of one head, 8 D
bytes of codes, then D bytes of scales and D bytes of least values (all fp16).  A unit is contiguous, so attention fetches
it with one bulk copy, and its bytes stand in the order in which the tensor-core operands take them:

* keys, codes: 32-bit words ``[D / 128][16 tokens][4 t][4 g]`` (64-wide heads: ``[16][4 t][2 g]``), word ``(t, g)`` = dims
  ``32 g + 8 t .. + 7``, lowest nibble first: lane ``t`` of a quad finds its dims of all groups in one 16-byte read.
  Scales and least values: ``[16 tokens][groups]``.
* values, codes: 16-bit words ``[D / 128][16 places][8 slots][4 g]`` (``[16][8][2]``), word ``g`` of slot ``c`` = dims
  ``32 g + 4 c' .. + 3`` with ``c' = c ^ ((place & 2) << 1)`` (64-wide: ``c' = c``).  The token with bits ``b3 b2 b1 b0``
  stands at place ``b3 b0 b2 b1``: the four tokens that the lanes of a quad read together then lie in different banks.
  Scales and least values: ``[8 token pairs][groups][2]``.
"""
from __future__ import annotations

import functools

import torch

GROUP = 32
UNIT = 16                                   # tokens of a unit
HEAD_DIMS = (64, 128, 256)
LARGEST = 65280.0                            # of a value: 15 s + m then stays within fp16 (65504) whatever the roundings


class Kv4Cache:
    """Keys (``kind="k"``) or values (``"v"``) of one layer's paged cache, 4 bits each.

    Stands where the bf16 cache tensor ``[n_blocks, block_size, kv heads, head_dim]`` stands in ``ops.qk_rope_append`` and
    ``ops.paged_attention``; ``shape`` is that tensor's shape."""

    __slots__ = ("data", "head_dim", "kind", "shape")

    def __init__(self, data: torch.Tensor, head_dim: int, kind: str):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"4-bit KV cache: head_dim {head_dim} is not one of {HEAD_DIMS}")
        if kind != "k" and kind != "v":
            raise ValueError(f"4-bit KV cache: kind {kind!r} is neither 'k' nor 'v'")
        shape = data.shape
        if data.dtype is not torch.uint8 or len(shape) != 4 or shape[3] != 10 * head_dim or not data.is_contiguous():
            raise ValueError(f"4-bit KV cache: data must be contiguous uint8 [n_blocks, heads, block_size / 16, {10 * head_dim}], "
                             f"got {data.dtype} {tuple(data.shape)}")
        n, h, u, _ = shape
        if not h or not u:
            raise ValueError(f"4-bit KV cache: {h} heads in blocks of {u * UNIT} tokens")
        if data.data_ptr() % 16:
            raise ValueError("4-bit KV cache: data must start on a 16-byte boundary")
        self.data, self.head_dim, self.kind = data, head_dim, kind
        self.shape = (n, u * UNIT, h, head_dim)

    @classmethod
    def zeros(cls, n_blocks: int, block_size: int, n_kv: int, head_dim: int, kind: str, device="cpu") -> "Kv4Cache":
        if block_size <= 0 or block_size % UNIT:
            raise ValueError(f"4-bit KV cache: block size {block_size} is not a multiple of {UNIT}")
        return cls(torch.zeros(n_blocks, n_kv, block_size // UNIT, 10 * head_dim, dtype=torch.uint8, device=device), head_dim, kind)

    @staticmethod
    def bytes_per_token(n_kv: int, head_dim: int) -> int:
        """Of the keys, or of the values, of one layer."""
        return n_kv * 10 * head_dim // UNIT

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def is_cuda(self) -> bool:
        return self.data.is_cuda

    @property
    def n_slots(self) -> int:
        return self.shape[0] * self.shape[1]

    def nbytes(self) -> int:
        return self.data.numel()


def check_pair(kcache: Kv4Cache, vcache: Kv4Cache, n_kv: int, head_dim: int, device: torch.device) -> None:
    """Refuses a pair that is not the keys and the values of one layer with ``n_kv`` heads of ``head_dim`` on ``device``."""
    if not (isinstance(kcache, Kv4Cache) and isinstance(vcache, Kv4Cache)):
        raise ValueError("a 4-bit cache stands for the keys and the values alike: got one of another kind")
    if kcache.kind != "k" or vcache.kind != "v":
        raise ValueError(f"4-bit KV cache: a pair of kinds {kcache.kind!r}, {vcache.kind!r} where 'k', 'v' is wanted")
    if kcache.shape != vcache.shape:
        raise ValueError(f"4-bit KV cache: keys {kcache.shape} and values {vcache.shape} differ in shape")
    if kcache.shape[2] != n_kv or kcache.head_dim != head_dim:
        raise ValueError(f"4-bit KV cache: {kcache.shape[2]} heads of {kcache.head_dim} where {n_kv} of {head_dim} are wanted")
    if kcache.data.device != device or vcache.data.device != device:
        raise ValueError(f"4-bit KV cache on {kcache.data.device} / {vcache.data.device}, other arguments on {device}")


# ---- definition ----------------------------------------------------------------------------------------------------------
def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Rows ``x [..., D]`` -> codes ``[..., D] uint8``, scales and least values ``[..., D / 32] float16``."""
    x = x.float()
    bad = x.isnan().any(-1, keepdim=True)
    g = x.nan_to_num(nan=0.0).clamp(-LARGEST, LARGEST).unflatten(-1, (-1, GROUP))
    m = _round_f16(g.amin(-1), up=False)
    s = _round_f16((g.amax(-1) - m.float()) / torch.full_like(m, 15.0, dtype=torch.float32), up=True)
    sf = s.float()[..., None]
    n = torch.where(sf > 0, (g - m.float()[..., None]) / torch.where(sf > 0, sf, torch.ones_like(sf)), torch.zeros_like(g))
    n = n.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return n.masked_fill(bad, 0), s.masked_fill(bad, 0.0), m.masked_fill(bad, float("nan"))


def dequantize(n: torch.Tensor, s: torch.Tensor, m: torch.Tensor) -> torch.Tensor:
    """Codes, scales and least values as ``quantize`` gives them -> fp32 rows."""
    return (n.unflatten(-1, (-1, GROUP)).float() * s.float()[..., None] + m.float()[..., None]).flatten(-2)


def _round_f16(x: torch.Tensor, up: bool) -> torch.Tensor:
    """fp32 -> fp16, rounded up or down (``x`` finite and within +-65504)."""
    if up:
        return -_round_f16(-x, up=False)
    h = x.half()
    bits = h.view(torch.int16)
    below = torch.where(bits > 0, bits - 1, torch.where(bits == 0, torch.full_like(bits, -32767), bits + 1)).view(torch.float16)
    return torch.where(h.float() > x, below, h)


@functools.cache
def _layout(head_dim: int, kind: str) -> tuple[torch.Tensor, torch.Tensor]:
    """``(byte [16, D / 2], number [16, D / 32])`` on the CPU: where the byte with the codes of dims ``2 i, 2 i + 1`` of a token
    stands in a unit, and which of the unit's scales (least values) is its group's."""
    d, groups = head_dim, head_dim // GROUP
    per = min(4, groups)
    tok = torch.arange(UNIT)[:, None]
    dim = torch.arange(0, d, 2)[None]
    half, r = dim // 128, dim % 128
    g, i = r // GROUP, r % GROUP
    grp = torch.arange(groups)[None]
    if kind == "k":
        byte = ((half * UNIT + tok) * 4 + i // 8) * (4 * per) + 4 * g + i % 8 // 2
        return byte, tok * groups + grp
    place = (tok & 8) | ((tok & 1) << 2) | ((tok >> 1) & 3)
    slot = i // 4 if d == 64 else (i // 4) ^ ((place & 2) << 1)
    byte = ((half * UNIT + place) * 8 + slot) * (2 * per) + 2 * g + i % 4 // 2
    return byte, (tok // 2 * groups + grp) * 2 + tok % 2


def read(cache: Kv4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The rows ``[n, kv heads, D]`` that the cache holds at flat ``slots [n]`` (zeros for a slot outside the cache)."""
    nb, bs, _, d = cache.shape
    byte, num = (t.to(cache.device) for t in _layout(d, cache.kind))
    ok = (slots >= 0) & (slots < nb * bs)
    sl = torch.where(ok, slots, torch.zeros_like(slots)).long()
    unit = cache.data[sl // bs, :, sl % bs // UNIT]                                   # [n, H, 10 D]
    b = unit.gather(-1, byte[sl % UNIT][:, None].expand(-1, unit.shape[1], -1))
    codes = torch.stack((b & 15, b >> 4), -1).flatten(-2)
    meta = unit[..., 8 * d:].contiguous().view(torch.float16)
    at = num[sl % UNIT][:, None].expand(-1, unit.shape[1], -1)
    x = dequantize(codes, meta.gather(-1, at), meta.gather(-1, at + d // 2))
    return torch.where(ok[:, None, None], x, torch.zeros_like(x)).to(dtype)


def write(cache: Kv4Cache, slots: torch.Tensor, x: torch.Tensor) -> None:
    """Quantise rows ``x [n, kv heads, D]`` into flat ``slots [n]``; a slot outside the cache stores nothing."""
    nb, bs, h, d = cache.shape
    ok = (slots >= 0) & (slots < nb * bs)
    sl, x = slots[ok].long(), x[ok]
    n, s, m = quantize(x)
    byte, num = (t.to(cache.device) for t in _layout(d, cache.kind))
    blk, sub = (sl // bs)[:, None, None], (sl % bs // UNIT)[:, None, None]
    head = torch.arange(h, device=cache.device)[None, :, None]
    cache.data[blk, head, sub, byte[sl % UNIT][:, None]] = n[..., 0::2] | (n[..., 1::2] << 4)
    meta = cache.data.view(torch.float16)                                             # [nb, H, units, 5 D]
    at = num[sl % UNIT][:, None] + 4 * d
    meta[blk, head, sub, at] = s
    meta[blk, head, sub, at + d // 2] = m


def paged_attention(q: torch.Tensor, kcache: Kv4Cache, vcache: Kv4Cache, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                    cu_q: torch.Tensor, scale: float, sliding_window: int = 0, sinks: torch.Tensor | None = None) -> torch.Tensor:
    """Definition of attention over a 4-bit cache: ``reference.paged_attention`` over the rows that the cache holds.  Rows
    that see no key, and rows of ``q`` behind the last sequence, give zeros."""
    T, hq, d = q.shape
    bs, hkv = kcache.shape[1], kcache.shape[2]
    out = torch.zeros_like(q)
    for b in range(seq_lens.numel()):
        lo, hi, n = int(cu_q[b]), int(cu_q[b + 1]), int(seq_lens[b])
        if hi == lo or n <= 0:
            continue
        pos = torch.arange(n, device=q.device)
        slots = block_tables[b].long()[pos // bs] * bs + pos % bs
        k, v = read(kcache, slots), read(vcache, slots)
        qb = q[lo:hi].float().view(hi - lo, hkv, hq // hkv, d)
        sc = torch.einsum("thgd,nhd->hgtn", qb, k) * scale
        at = torch.arange(n - (hi - lo), n, device=q.device)[:, None]
        seen = pos[None] <= at
        if sliding_window:
            seen &= pos[None] > at - sliding_window
        sc = sc.masked_fill(~seen, float("-inf"))
        if sinks is not None:
            sk = sinks.float().view(hkv, -1, 1, 1).expand(-1, -1, hi - lo, 1)
            p = torch.softmax(torch.cat((sc, sk), -1), -1)[..., :-1]
        else:
            p = torch.softmax(sc, -1)
        p = torch.where(seen.any(-1)[..., None], p, torch.zeros_like(sc))
        # a key that a query does not see may hold anything; a NaN that it sees makes its row NaN
        o = torch.einsum("hgtn,nhd->thgd", p, v.nan_to_num(nan=0.0))
        bad = torch.einsum("tn,nh->th", seen.float(), v.isnan().any(-1).float()) > 0
        out[lo:hi] = o.masked_fill(bad[..., None, None], float("nan")).reshape(hi - lo, hq, d).to(q.dtype)
    return out


def rope_axes(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, mscale: float, axes: torch.Tensor | None) -> torch.Tensor:
    """Rotates pairs ``(i, i + rot / 2)`` of fp32 rows ``x [T, heads, D]`` by ``positions[axes[i]] * inv_freq[i]``, the angle
    taken in 64 bits (an fp32 product is off by 2^-8 of a turn at position 2^17); ``positions [T]`` where ``axes`` is None.  An
    axis that ``positions`` has not is taken as the nearest that it has."""
    half = inv_freq.numel()
    pos = positions.double()[:, None] if axes is None else positions.double()[axes.long().clamp(0, positions.shape[0] - 1)].T
    ang = pos * inv_freq.double()
    cos, sin = (ang.cos() * mscale).float()[:, None], (ang.sin() * mscale).float()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)


def qk_rope_append(qkv, positions, inv_freq, mscale, n_q, n_kv, head_dim, kcache, vcache, slots, q_norm=None, k_norm=None,
                   eps=1e-6, v_unit_norm=False, axes=None) -> torch.Tensor:
    """Definition of the append: norm, rotation and quantisation in fp32 with no rounding between them."""
    x = qkv.float().view(qkv.shape[0], n_q + 2 * n_kv, head_dim)
    q, k, v = x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
    unit = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)      # noqa: E731
    if q_norm is not None:
        q = unit(q) * q_norm.float()
        k = unit(k) * k_norm.float() if n_kv else k
    q = rope_axes(q, positions, inv_freq, mscale, axes)
    if n_kv:
        k = rope_axes(k, positions, inv_freq, mscale, axes)
        v = unit(v) if v_unit_norm else v
        if isinstance(kcache, Kv4Cache):
            write(kcache, slots, k)
            write(vcache, slots, v)
        else:
            ok = (slots >= 0) & (slots < kcache.shape[0] * kcache.shape[1])
            for cache, rows in ((kcache, k), (vcache, v)):
                cache.view(-1, *cache.shape[2:])[slots[ok].long()] = rows[ok].to(cache.dtype)
    return q.to(qkv.dtype)
