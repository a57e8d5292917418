"""Hot-op entry points.

Each function takes tensors on one device.  CUDA tensors go to the hand-written
sm_100a kernels in ``exo_b200/ops/csrc`` (bound through ``exo_b200.ops.cuda``); a
missing extension on a CUDA device is an error, never a silent fallback.  CPU tensors
run the fp32 PyTorch definitions in ``exo_b200.ops.reference`` — that path is the
correctness oracle, not a second backend.
"""
from __future__ import annotations

import torch

from . import kv4
from . import reference as ref
from .kv4 import Kv4Cache

_cuda = None


def cuda_ops():
    """The ctypes binding of the kernel library (loaded on first use; raises if absent)."""
    global _cuda
    if _cuda is None:
        from . import cuda as _c
        _c.load()
        _cuda = _c
    return _cuda


def rmsnorm(x, w, eps, residual=None):
    if x.is_cuda:
        return cuda_ops().rmsnorm(x, w, eps, residual)
    return ref.rmsnorm(x, w, eps, residual)


def linear(x, w, bias=None, residual=None, swiglu=False):
    """``y = x @ w.T (+bias) (+residual)``; ``swiglu=True`` returns ``silu(y[:, :F]) * y[:, F:]``."""
    if x.is_cuda:
        return cuda_ops().linear(x, w, bias, residual, None, 0.0, swiglu)
    y = ref.linear(x, w, bias, residual)
    return ref.swiglu(y) if swiglu else y


def norm_linear(h, norm_w, eps, w, bias=None, swiglu=False):
    """``linear(rmsnorm(h, norm_w), w)`` — one kernel on the small-batch path.  ``h`` may be a
    tensor-parallel hand-over (``parallel.fused.Handover``): the reduction then happens in this kernel's prologue."""
    if hasattr(h, "norm_linear"):
        return h.norm_linear(norm_w, eps, w, bias, swiglu)
    if h.is_cuda:
        return cuda_ops().linear(h, w, bias, None, norm_w, eps, swiglu)
    y = ref.linear(ref.rmsnorm(h, norm_w, eps)[0], w, bias)
    return ref.swiglu(y) if swiglu else y


def swiglu(gate_up, limit=0.0):
    """``silu(gate) * up``; ``limit`` > 0 caps the activated gate at ``limit`` and clamps ``up`` to ``+-limit``."""
    if gate_up.is_cuda:
        return cuda_ops().swiglu(gate_up, limit)
    return ref.swiglu(gate_up, limit)


def qk_rope_append(qkv, positions, inv_freq, mscale, n_q, n_kv, head_dim, kcache, vcache, slots,
                   q_norm=None, k_norm=None, eps=1e-6, v_unit_norm=False, axes=None):
    """Split fused ``qkv [T,(n_q+2n_kv)*D]``, apply optional per-head RMSNorm and RoPE to q/k,
    append k/v to the paged cache at ``slots``.  Returns ``q [T, n_q, D]``.  ``v_unit_norm``: v heads are RMS-normalised
    (no weight) before they are stored (Gemma-4).  With ``n_kv == 0`` only q is processed (a layer that reads another
    layer's cache).

    ``kcache`` / ``vcache`` may be a pair of ``Kv4Cache`` (head_dim 64, 128 or 256): k and v are then stored in 4 bits.
    ``axes [rot/2]`` gives each rotated pair its position axis and ``positions`` is then ``[axes, T]`` (time, height, width
    of image and video tokens; an entry of ``axes`` that names no row of ``positions`` is taken as the nearest that does).  In these two forms nothing is
    rounded between norm, rotation and storage, angles are taken in 64 bits, a slot outside the cache (negative, say) stores
    nothing, and of several rows with the same slot it is not defined which is kept (nor that one is kept whole)."""
    if axes is not None or isinstance(kcache, Kv4Cache) or isinstance(vcache, Kv4Cache):
        _check_append(qkv, positions, inv_freq, n_q, n_kv, head_dim, kcache, vcache, slots, q_norm, k_norm, axes)
        if qkv.is_cuda:
            return cuda_ops().kv4_append(qkv, positions, inv_freq, mscale, n_q, n_kv, head_dim, kcache, vcache, slots, q_norm,
                                         k_norm, eps, v_unit_norm, axes)
        return kv4.qk_rope_append(qkv, positions, inv_freq, mscale, n_q, n_kv, head_dim, kcache, vcache, slots, q_norm, k_norm,
                                  eps, v_unit_norm, axes)
    if qkv.is_cuda:
        return cuda_ops().qk_rope_append(qkv, positions, inv_freq, mscale, n_q, n_kv, head_dim, kcache, vcache,
                                         slots, q_norm, k_norm, eps, v_unit_norm)
    T = qkv.shape[0]
    q, k, v = qkv.split((n_q * head_dim, n_kv * head_dim, n_kv * head_dim), dim=-1)
    q, k, v = q.reshape(T, n_q, head_dim), k.reshape(T, n_kv, head_dim), v.reshape(T, n_kv, head_dim)
    if q_norm is not None:
        q = ref.head_rmsnorm(q, q_norm, eps)
        if n_kv:
            k = ref.head_rmsnorm(k, k_norm, eps)
    q = ref.rope(q, positions, inv_freq, mscale)
    if n_kv:
        k = ref.rope(k, positions, inv_freq, mscale)
        if v_unit_norm:
            v = ref.head_rmsnorm(v, torch.ones(head_dim, device=v.device), eps)
        ref.kv_append(k, v, kcache, vcache, slots)
    return q


def _check_append(qkv, positions, inv_freq, n_q, n_kv, head_dim, kcache, vcache, slots, q_norm, k_norm, axes):
    """Arguments of the append to a 4-bit cache, or with several position axes: both run one kernel, whose checks these are."""
    if qkv.dim() != 2 or n_q < 0 or n_kv < 0 or qkv.shape[1] != (n_q + 2 * n_kv) * head_dim:
        raise ValueError(f"qk_rope_append: {tuple(qkv.shape)} for {n_q} + 2 x {n_kv} heads of {head_dim}")
    T, half = qkv.shape[0], inv_freq.numel()
    if head_dim not in kv4.HEAD_DIMS:
        raise ValueError(f"qk_rope_append: head_dim {head_dim} is not one of {kv4.HEAD_DIMS}")
    if 2 * half > head_dim or 2 * half % (head_dim // 16):
        raise ValueError(f"qk_rope_append: {2 * half} rotated dims of {head_dim} are not a multiple of {head_dim // 16}")
    if (q_norm is None) != (k_norm is None) and n_kv:
        raise ValueError("qk_rope_append: q_norm and k_norm come together")
    if axes is None:
        if positions.numel() != T:
            raise ValueError(f"qk_rope_append: {tuple(positions.shape)} positions for {T} tokens")
    elif axes.numel() != half or positions.dim() != 2 or positions.shape[1] != T or not positions.shape[0]:
        raise ValueError(f"qk_rope_append: axes {tuple(axes.shape)} and positions {tuple(positions.shape)} for {half} pairs and {T} tokens")
    if not n_kv:
        return
    if slots.numel() != T:
        raise ValueError(f"qk_rope_append: {slots.numel()} slots for {T} tokens")
    if isinstance(kcache, Kv4Cache) or isinstance(vcache, Kv4Cache):
        kv4.check_pair(kcache, vcache, n_kv, head_dim, qkv.device)
    else:
        for c in (kcache, vcache):
            if tuple(c.shape[2:]) != (n_kv, head_dim) or c.shape != kcache.shape or c.dtype != qkv.dtype or not c.is_contiguous() \
                    or c.device != qkv.device or c.data_ptr() % 16:
                raise ValueError(f"qk_rope_append: cache {tuple(c.shape)} {c.dtype} on {c.device} for {n_kv} heads of {head_dim}, "
                                 f"{qkv.dtype} on {qkv.device}")


def paged_attention(q, kcache, vcache, block_tables, seq_lens, cu_q, scale, sliding_window=0, sinks=None,
                    max_q_len=None):
    """Causal GQA attention of the new tokens ``q [T, Hq, D]`` over a paged cache (``reference.paged_attention`` is the
    definition).  The cache may be a pair of ``Kv4Cache`` (``kv4.paged_attention`` is then the definition: rows that see no
    key and rows behind the last sequence are zero); page numbers outside it and lengths past the table are clamped there."""
    if isinstance(kcache, Kv4Cache) or isinstance(vcache, Kv4Cache):
        if q.dim() != 3 or block_tables.dim() != 2 or block_tables.shape[0] < seq_lens.numel() or cu_q.numel() != seq_lens.numel() + 1:
            raise ValueError(f"paged_attention: q {tuple(q.shape)}, block tables {tuple(block_tables.shape)}, {seq_lens.numel()} "
                             f"lengths and {cu_q.numel()} offsets do not fit")
        kv4.check_pair(kcache, vcache, kcache.shape[2], q.shape[2], q.device)
        if not q.shape[1] or q.shape[1] % kcache.shape[2]:
            raise ValueError(f"paged_attention: {q.shape[1]} query heads over {kcache.shape[2]} key heads")
        if sliding_window < 0:
            raise ValueError(f"paged_attention: sliding window {sliding_window}")
        if q.is_cuda:
            return cuda_ops().kv4_paged_attention(q, kcache, vcache, block_tables, seq_lens, cu_q, scale, sliding_window, sinks,
                                                  max_q_len)
        return kv4.paged_attention(q, kcache, vcache, block_tables, seq_lens, cu_q, scale, sliding_window, sinks)
    if q.is_cuda:
        return cuda_ops().paged_attention(q, kcache, vcache, block_tables, seq_lens, cu_q, scale, sliding_window,
                                          sinks, max_q_len)
    return ref.paged_attention(q, kcache, vcache, block_tables, seq_lens, cu_q, scale, sliding_window, sinks)


def kv4_read(kcache, vcache, slots, dtype=torch.bfloat16):
    """The rows that a 4-bit cache holds at flat ``slots [n]``: ``(k, v)``, each ``[n, kv heads, D]`` in bfloat16 or float32
    (zeros for a slot outside the cache)."""
    kv4.check_pair(kcache, vcache, kcache.shape[2], kcache.head_dim, slots.device)
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"kv4_read: rows are given as bfloat16 or float32, not {dtype}")
    if kcache.is_cuda:
        return cuda_ops().kv4_read(kcache, vcache, slots, dtype)
    return kv4.read(kcache, slots, dtype), kv4.read(vcache, slots, dtype)


def kv4_write(k, v, kcache, vcache, slots):
    """Quantise rows ``k, v [n, kv heads, D]`` into a 4-bit cache at flat ``slots [n]`` (a slot outside it stores nothing)."""
    if k.dim() != 3 or k.shape != v.shape or slots.numel() != k.shape[0] or v.device != k.device:
        raise ValueError(f"kv4_write: {tuple(k.shape)} keys, {tuple(v.shape)} values and {slots.numel()} slots do not fit")
    kv4.check_pair(kcache, vcache, k.shape[1], k.shape[2], k.device)
    if k.is_cuda:
        cuda_ops().kv4_write(k, v, kcache, vcache, slots)
    else:
        kv4.write(kcache, slots, k)
        kv4.write(vcache, slots, v)


def mla_kv_append(kva, norm_w, eps, positions, inv_freq, mscale, cache, slots, kv_lora):
    """Append the new tokens' rows ``[rmsnorm(latent) | rope(k_rope)]`` to the paged latent cache."""
    if kva.is_cuda:
        return cuda_ops().mla_kv_append(kva, norm_w, eps, positions, inv_freq, mscale, cache, slots, kv_lora)
    return ref.mla_kv_append(kva, norm_w, eps, positions, inv_freq, mscale, cache, slots, kv_lora)


def mla_q_absorb(q, w_uk, positions, inv_freq, mscale, nope, kv_lora, w_uk_t=None):
    """``q [T, H, nope + rope]`` -> queries in cache space ``[T, H, kv_lora + rope]`` (``q_nope . W_UK``, rotated rope)."""
    if q.is_cuda:
        return cuda_ops().mla_q_absorb(q, w_uk, positions, inv_freq, mscale, nope, kv_lora, w_uk_t)
    return ref.mla_q_absorb(q, w_uk, positions, inv_freq, mscale, nope)


def mla_o_absorb(o_lat, w_uv):
    """``o_lat [T, H, kv_lora]`` -> ``[T, H * v]`` through ``W_UV``."""
    if o_lat.is_cuda:
        return cuda_ops().mla_o_absorb(o_lat, w_uv)
    return ref.mla_o_absorb(o_lat, w_uv)


def mla_paged_attention(q_full, ckv, block_tables, seq_lens, cu_q, scale, kv_lora, max_q_len=None):
    """Absorbed MLA attention of ``q_full [T, H, kv_lora + rope]`` over the paged latent cache -> ``[T, H, kv_lora]``."""
    if q_full.is_cuda:
        return cuda_ops().mla_paged_attention(q_full, ckv, block_tables, seq_lens, cu_q, scale, kv_lora, max_q_len)
    return ref.mla_paged_attention(q_full[..., :kv_lora], q_full[..., kv_lora:], ckv, block_tables, seq_lens, cu_q, scale,
                                   kv_lora)


def moe_route(logits, top_k, kind, norm_topk, bias, n_group, topk_group, scaling):
    if logits.is_cuda:
        return cuda_ops().moe_route(logits, top_k, kind, norm_topk, bias, n_group, topk_group, scaling)
    return ref.moe_route(logits, top_k, kind, norm_topk, bias, n_group, topk_group, scaling)


def moe_experts(x, w_gate_up, w_down, weights, ids, expert_offset=0, n_experts_total=None, act="silu", limit=0.0):
    """Weighted sum of the routed experts.  ``act``: ``silu`` / ``gelu_tanh`` (gated) or ``relu2`` (``w_gate_up`` is then the
    single up projection ``[E, F, H]``)."""
    if x.is_cuda:
        return cuda_ops().moe_experts(x, w_gate_up, w_down, weights, ids, expert_offset, n_experts_total, act, limit)
    return ref.moe_experts(x, w_gate_up, w_down, weights, ids, expert_offset, act, limit)


def moe_experts_oai(x, w_gate_up, b_gate_up, w_down, b_down, weights, ids, expert_offset=0, limit=7.0):
    """GPT-OSS experts (biases, capped ``(up + 1) * gate * sigmoid(1.702 gate)``): PyTorch ops on either device (the host reads
    which experts are hit, so a step that runs them cannot be captured in a CUDA graph)."""
    return ref.moe_experts_oai(x, w_gate_up, b_gate_up, w_down, b_down, weights, ids, expert_offset, limit)


def embedding(table, ids):
    if table.is_cuda:
        return cuda_ops().embedding(table, ids)
    return table[ids.long()]


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    if logits.is_cuda:
        return cuda_ops().sample(logits, temperature, top_k, top_p, min_p, uniform)
    return ref.sample(logits, temperature, top_k, top_p, min_p, uniform)


def argmax(logits):
    if logits.is_cuda:
        return cuda_ops().argmax(logits)
    return logits.float().argmax(-1)


def gated_delta(proj, conv_w, a_log, dt_bias, norm_w, eps, conv_state, rec_state, seats, cu_q, positions, hk, hv, dk, dv):
    """A gated-delta-rule layer between its projections over a ragged batch: causal convolution + SiLU, L2-normalised
    q/k, the recurrence over each sequence's state seat, gated RMSNorm (``reference.gated_delta`` is the definition)."""
    if proj.is_cuda:
        return cuda_ops().gated_delta(proj, conv_w, a_log, dt_bias, norm_w, eps, conv_state, rec_state, seats, cu_q,
                                      positions, hk, hv, dk, dv)
    return ref.gated_delta(proj, conv_w, a_log, dt_bias, norm_w, eps, conv_state, rec_state, seats, cu_q, positions,
                           hk, hv, dk, dv)


def sigmoid_gate(x, gate):
    """``x * sigmoid(gate)``, element by element (``gate`` may be a column slice of a wider tensor)."""
    if x.is_cuda:
        return cuda_ops().sigmoid_gate(x, gate)
    return (x.float() * torch.sigmoid(gate.float())).to(x.dtype)


def scaled_add(y, x, logit):
    """``y + x * sigmoid(logit)`` with one ``logit`` per row."""
    if x.is_cuda:
        return cuda_ops().scaled_add(y, x, logit)
    return (y.float() + x.float() * torch.sigmoid(logit.float())).to(y.dtype)


def geglu(gate_up):
    """``gelu_tanh(gate_up[:, :F]) * gate_up[:, F:]``."""
    if gate_up.is_cuda:
        return cuda_ops().geglu(gate_up)
    return ref.geglu(gate_up)


def mamba2(proj, conv_w, conv_b, a_log, dt_bias, skip, norm_w, eps, conv_state, ssm_state, seats, cu_q, positions, groups, heads,
           d_state, head_dim):
    """A Mamba-2 mixer between its projections over a ragged batch (``reference.mamba2`` is the definition)."""
    fn = cuda_ops().mamba2 if proj.is_cuda else ref.mamba2
    return fn(proj, conv_w, conv_b, a_log, dt_bias, skip, norm_w, eps, conv_state, ssm_state, seats, cu_q, positions, groups,
              heads, d_state, head_dim)


def relu2(x):
    """``relu(x)^2`` (torch ops on either device: not a hot path of its own, it sits between two GEMMs)."""
    return torch.relu(x).square()
