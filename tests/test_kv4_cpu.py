"""The 4-bit KV cache on the CPU: format, definitions of its operators, refusals, and an engine that serves from it."""
import math

import pytest
import torch

from exo_b200 import ops
from exo_b200.ops import kv4
from kv4_cases import append64, attention64, batch, check_attention, check_held, filled_pair, unpacked


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bs", [16, 48])
def test_rows_in_and_out(d, bs):
    g = torch.Generator().manual_seed(d + bs)
    kc, vc = (ops.Kv4Cache.zeros(4, bs, 3, d, kind) for kind in "kv")
    slots = torch.randperm(4 * bs, generator=g)[:37]
    k, v = torch.randn(37, 3, d, generator=g), torch.randn(37, 3, d, generator=g).to(torch.bfloat16).float() * 50 + 7
    ops.kv4_write(k, v, kc, vc, slots.int())
    check_held(kc, slots, k.double())
    check_held(vc, slots, v.double())
    for cache, got in zip((kc, vc), ops.kv4_read(kc, vc, slots, torch.float32)):
        n, s, m = (t[slots] for t in unpacked(cache))
        want = (n.unflatten(-1, (-1, 32)) * s[..., None] + m[..., None]).flatten(-2)
        assert float((got - want).abs().max()) <= 2.0 ** -22 * float(want.abs().max())
    untouched = torch.ones(4 * bs, dtype=torch.bool)
    untouched[slots] = False
    assert all(not t[untouched].any() for t in unpacked(kc) + unpacked(vc))


def test_slots_outside_store_nothing_and_read_zero():
    kc, vc = filled_pair(2, 16, 2, 64, "cpu")
    before = kc.data.clone()
    slots = torch.tensor([-1, 32, 5])
    ops.kv4_write(torch.ones(3, 2, 64), torch.ones(3, 2, 64), kc, vc, slots)
    k, v = ops.kv4_read(kc, vc, slots, torch.float32)
    assert not k[:2].any() and not v[:2].any() and bool((k[2] == 1).all())
    ops.kv4_write(*(t[2:] for t in (k, v)), kc, vc, slots[2:])
    assert int((kc.data != before).sum()) > 0


def test_extreme_rows():
    kc, vc = (ops.Kv4Cache.zeros(1, 16, 1, 64, kind) for kind in "kv")
    x = torch.zeros(6, 1, 64)
    x[0] = 3.0                                  # a constant group has no step
    x[1, 0, 3], x[1, 0, 40] = float("inf"), -1e30     # clamped to +-65280
    x[2, 0, 9] = float("nan")                   # the whole row is NaN
    x[3] = 2.0 ** -26 * torch.arange(64)        # below fp16's least step
    x[4, 0, 0] = -0.0
    x[5] = torch.linspace(-65504, 65504, 64)
    ops.kv4_write(x, x, kc, vc, torch.arange(6))
    for got in ops.kv4_read(kc, vc, torch.arange(6), torch.float32):
        assert bool((got[0] == 3).all())
        assert got[1, 0, 3] == pytest.approx(65280, rel=2.0 ** -10) and got[1, 0, 40] == -65280
        assert bool(got[2].isnan().all())
        assert float((got[3] - x[3]).abs().max()) <= 2.0 ** -24
        assert not got[4].any()
        assert float((got[5] - x[5]).abs().max()) <= 131008 / 15 / 2 * (1 + 2.0 ** -9)


@pytest.mark.parametrize("d,rot,norm,axes,quantized", [(64, 64, True, False, True), (128, 32, False, True, True),
                                                        (256, 64, True, True, True), (128, 128, True, True, False)])
def test_append_definition(d, rot, norm, axes, quantized):
    g = torch.Generator().manual_seed(d)
    T, nq, nkv = 11, 4, 2
    qkv = torch.randn(T, (nq + 2 * nkv) * d, generator=g)
    qn, kn = ((1 + 0.1 * torch.randn(d, generator=g)) if norm else None for _ in range(2))
    inv = 10000.0 ** (-torch.arange(0, rot, 2) / rot)
    ax = torch.arange(rot // 2) % 3 if axes else None
    pos = torch.randint(0, 100000, (3, T) if axes else (T,), generator=g)
    slots = torch.randperm(32, generator=g)[:T]
    if quantized:
        kc, vc = (ops.Kv4Cache.zeros(2, 16, nkv, d, kind) for kind in "kv")
    else:
        kc, vc = torch.zeros(2, 16, nkv, d), torch.zeros(2, 16, nkv, d)
    q = ops.qk_rope_append(qkv, pos, inv, 1.25, nq, nkv, d, kc, vc, slots, qn, kn, 1e-6, axes=ax)
    want = append64(qkv, pos, inv, 1.25, nq, nkv, d, qn, kn, 1e-6, False, ax)
    assert float((q - want[0]).abs().max()) <= 2.0 ** -20 * float(want[0].abs().max())
    for cache, x in zip((kc, vc), want[1:]):
        if quantized:
            check_held(cache, slots, x)
        else:
            assert float((cache.view(-1, nkv, d)[slots] - x).abs().max()) <= 2.0 ** -20 * float(x.abs().max())


def test_one_axis_for_all_pairs_is_the_plain_rotation():
    g = torch.Generator().manual_seed(3)
    qkv, pos = torch.randn(5, 4 * 64, generator=g), torch.randint(0, 50, (5,), generator=g)
    inv = 10000.0 ** (-torch.arange(0, 64, 2) / 64)
    a, b = ((torch.zeros(1, 16, 1, 64), torch.zeros(1, 16, 1, 64)) for _ in range(2))
    q0 = ops.qk_rope_append(qkv, pos, inv, 1.0, 2, 1, 64, *a, torch.arange(5))
    q1 = ops.qk_rope_append(qkv, pos.expand(3, 5), inv, 1.0, 2, 1, 64, *b, torch.arange(5), axes=torch.arange(32) % 3)
    # angles below 50: an fp32 product is off by 50 * 2^-24
    assert float((q0 - q1).abs().max()) <= 2.0 ** -17 and float((a[0] - b[0]).abs().max()) <= 2.0 ** -17


@pytest.mark.parametrize("d,hq,hkv,bs", [(64, 6, 2, 16), (128, 4, 4, 32), (256, 5, 1, 16)])
@pytest.mark.parametrize("window,sinks", [(0, False), (9, False), (0, True), (9, True)])
def test_attention_definition(d, hq, hkv, bs, window, sinks):
    lens = [(1, 1), (3, 40), (0, 0), (17, 17), (2, 33), (1, 0)]
    kc, vc = filled_pair(12, bs, hkv, d, "cpu", seed=d)
    table, n, cu = batch(lens, bs, 12)
    q = torch.randn(int(cu[-1]) + 2, hq, d, generator=torch.Generator().manual_seed(1))
    sk = torch.linspace(-1, 2, hq) if sinks else None
    out, bound = attention64(q, kc, vc, table, n, cu, d ** -0.5, window, sk)
    got = ops.paged_attention(q, kc, vc, table, n, cu, d ** -0.5, window, sk)
    check_attention(got, out, bound)
    assert not got[-3:].any()               # a sequence without keys, and rows behind the last sequence


def test_what_nobody_sees_may_be_nan():
    """Slots behind a sequence's end, in front of its window and in other pages hold NaN: the output does not change."""
    kc, vc = filled_pair(6, 16, 1, 64, "cpu")
    table, n, cu = batch([(2, 37)], 16, 6)
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(2))
    want = ops.paged_attention(q, kc, vc, table, n, cu, 0.125, 10)
    seen = torch.arange(37 - 11, 37)
    hidden = torch.ones(96, dtype=torch.bool)
    hidden[table[0].long()[seen // 16] * 16 + seen % 16] = False
    for c in (kc, vc):
        kv4.write(c, torch.arange(96)[hidden], torch.full((int(hidden.sum()), 1, 64), float("nan")))
    assert torch.equal(ops.paged_attention(q, kc, vc, table, n, cu, 0.125, 10), want)


def test_a_nan_row_reaches_only_the_queries_that_see_it():
    kc, vc = filled_pair(6, 16, 1, 64, "cpu")
    table, n, cu = batch([(20, 37)], 16, 6)
    slot = table[0, 30 // 16].long() * 16 + 30 % 16
    kv4.write(vc, slot.view(1), torch.full((1, 1, 64), float("nan")))
    q = torch.randn(20, 2, 64, generator=torch.Generator().manual_seed(2))
    got = ops.paged_attention(q, kc, vc, table, n, cu, 0.125)
    out, bound = attention64(q, kc, vc, table, n, cu, 0.125)
    assert bool(got[13:].isnan().all()) and not got[:13].isnan().any()
    check_attention(got, out, bound)


def test_refusals():
    data = torch.zeros(2, 1, 1, 640, dtype=torch.uint8)
    kc, vc = ops.Kv4Cache(data, 64, "k"), ops.Kv4Cache(data.clone(), 64, "v")
    for bad in (lambda: ops.Kv4Cache(data, 96, "k"), lambda: ops.Kv4Cache(data, 128, "k"), lambda: ops.Kv4Cache(data, 64, "x"),
                lambda: ops.Kv4Cache(data.float(), 64, "k"), lambda: ops.Kv4Cache(data[..., :639], 64, "k"),
                lambda: ops.Kv4Cache(torch.zeros(2, 1, 1, 1280, dtype=torch.uint8)[..., ::2], 64, "k"),
                lambda: ops.Kv4Cache.zeros(2, 20, 1, 64, "k"), lambda: ops.Kv4Cache.zeros(2, 0, 1, 64, "k")):
        with pytest.raises(ValueError):
            bad()
    qkv, pos, inv, slots = torch.randn(3, 4 * 64), torch.arange(3), torch.ones(32), torch.arange(3)
    app = lambda **kw: ops.qk_rope_append(**{**dict(qkv=qkv, positions=pos, inv_freq=inv, mscale=1.0, n_q=2, n_kv=1, head_dim=64,   # noqa: E731
                                                    kcache=kc, vcache=vc, slots=slots), **kw})
    app()
    w = torch.ones(64)
    for kw in (dict(kcache=vc, vcache=kc), dict(vcache=torch.zeros(2, 16, 1, 64)), dict(n_q=3), dict(inv_freq=torch.ones(33)),
               dict(inv_freq=torch.ones(31)), dict(slots=slots[:2]), dict(positions=pos[:2]), dict(q_norm=w),
               dict(axes=torch.zeros(32)), dict(axes=torch.zeros(31), positions=pos.expand(3, 3)), dict(head_dim=32, n_q=6),
               dict(vcache=ops.Kv4Cache(torch.zeros(3, 1, 1, 640, dtype=torch.uint8), 64, "v")),
               dict(axes=torch.zeros(32), positions=pos.expand(3, 3), kcache=torch.zeros(2, 16, 2, 64), vcache=torch.zeros(2, 16, 2, 64))):
        with pytest.raises(ValueError):
            app(**kw)
    q, table, n, cu = torch.randn(3, 2, 64), torch.zeros(1, 2, dtype=torch.int32), torch.tensor([3]), torch.tensor([0, 3])
    att = lambda **kw: ops.paged_attention(**{**dict(q=q, kcache=kc, vcache=vc, block_tables=table, seq_lens=n, cu_q=cu,   # noqa: E731
                                                     scale=0.1), **kw})
    att()
    for kw in (dict(q=q[:, :, :32]), dict(q=q[0]), dict(kcache=vc), dict(vcache=torch.zeros(2, 16, 1, 64)), dict(cu_q=cu[:1]),
               dict(seq_lens=torch.tensor([3, 3])), dict(block_tables=table[0]), dict(sliding_window=-1), dict(q=q[:, :0])):
        with pytest.raises(ValueError):
            att(**kw)
    with pytest.raises(ValueError):
        ops.kv4_write(torch.zeros(2, 1, 64), torch.zeros(3, 1, 64), kc, vc, slots[:2])
    with pytest.raises(ValueError):
        ops.kv4_write(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), kc, vc, slots[:2])


def test_half_a_step():
    """fp16 halves of ``kv4._round_f16`` against a walk over neighbours."""
    x = torch.cat((torch.randn(4000) * 10.0 ** torch.randint(-8, 5, (4000,)), torch.tensor([0.0, -0.0, 65504.0, -65504.0, 2.0 ** -25])))
    x = x.clamp(-65504, 65504)
    down, up = kv4._round_f16(x, False).double(), kv4._round_f16(x, True).double()
    step = torch.exp2(torch.frexp(x.double().abs()).exponent.clamp_min(-13).double() - 11)
    assert bool(((down <= x) & (x - down < step)).all()) and bool(((up >= x) & (up - x < step)).all())


# ---- an engine that serves from a 4-bit cache ------------------------------------------------------------------------------
GREEDY = dict(temperature=0.0, ignore_eos=True)


def _engine(cfg=None, weights=None, **kw):
    from exo_b200.engine.engine import Engine
    from exo_b200.models.config import preset
    from exo_b200.models.weights import RandomSource, ShardSpec, build_weights
    cfg = cfg or preset("tiny-llama")
    return Engine(cfg, weights or build_weights(cfg, ShardSpec(), RandomSource(seed=0), device="cpu"), n_blocks=64, device="cpu", **kw)


def _answer(eng, prompt, n):
    from exo_b200.engine.kv import SamplingParams
    rid, toks, logits = eng.submit(prompt, SamplingParams(max_tokens=n, **GREEDY), use_prefix_cache=False), [], []
    while eng.has_work:
        for o in eng.step():
            if o.token is not None:
                toks.append(o.token)
                logits.append(eng.exe.last_logits[0].float().clone())
    assert len(toks) == n and rid
    return toks, torch.stack(logits)


def test_engine_equals_a_dense_cache_of_the_held_values(monkeypatch):
    """The same model over a dense fp32 cache into which the quantised values are written."""
    prompt = torch.randint(0, 32000, (41,), generator=torch.Generator().manual_seed(0)).tolist()
    toks, logits = _answer(_engine(kv_bits=4), prompt, 6)

    def append(qkv, positions, inv_freq, mscale, n_q, n_kv, d, kc, vc, slots, q_norm=None, k_norm=None, eps=1e-6, v_unit_norm=False):
        q = kv4.qk_rope_append(qkv, positions, inv_freq, mscale, n_q, n_kv, d, kc, vc, slots, q_norm, k_norm, eps, v_unit_norm)
        for c in (kc, vc):
            rows = c.view(-1, *c.shape[2:])
            rows[slots.long()] = kv4.dequantize(*kv4.quantize(rows[slots.long()]))
        return q
    monkeypatch.setattr(ops, "qk_rope_append", append)
    want, ref_logits = _answer(_engine(), prompt, 6)
    assert toks == want
    assert float((logits - ref_logits).abs().max()) <= 1e-4 * float(ref_logits.abs().max())      # fp32, other orders of summation


def test_engine_chunks_do_not_matter():
    prompt = torch.randint(0, 32000, (50,), generator=torch.Generator().manual_seed(1)).tolist()
    whole = _answer(_engine(kv_bits=4), prompt, 4)
    parts = _answer(_engine(kv_bits=4, prefill_chunk=7), prompt, 4)
    assert whole[0] == parts[0] and float((whole[1] - parts[1]).abs().max()) <= 1e-4 * float(whole[1].abs().max())


def test_engine_prefix_cache_and_hand_over():
    from exo_b200.engine.kv import SamplingParams
    prompt = torch.randint(0, 32000, (40,), generator=torch.Generator().manual_seed(2)).tolist()
    src = _engine(kv_bits=4)
    want = src.generate(prompt, SamplingParams(max_tokens=5, **GREEDY))
    for _ in range(2):                                    # the second time from cached blocks
        rid = src.submit(prompt, SamplingParams(max_tokens=5, **GREEDY), req_id=None)
        seq, got = src.seqs[rid], []
        while src.has_work:
            got += [o.token for o in src.step() if o.token is not None]
        assert got == want
    assert seq.n_cached_prefix >= 32
    layers = src.export_kv(seq.final_blocks, 32)
    assert layers[0][0].shape == (32, 2, 64) and layers[0][0].dtype == torch.float32
    dst = _engine(kv_bits=4, weights=src.exe.model.w)
    rid, got = dst.submit(prompt, SamplingParams(max_tokens=5, **GREEDY), kv_prefill=(32, layers)), []
    while dst.has_work:
        got += [o.token for o in dst.step() if o.token is not None]
    assert got[0] == want[0]
    # values on the grid of a group's codes: the least is its m, 15 s + m its largest, so s comes back but for a rounding (2^-10)
    # and every value within 15 times that
    blocks = [dst.alloc.alloc() for _ in range(2)]
    dst.import_kv(blocks, 32, layers)
    for pair, again in zip(layers, dst.export_kv(blocks, 32)):
        for x, y in zip(pair, again):
            step = (x.unflatten(-1, (-1, 32)).amax(-1) - x.unflatten(-1, (-1, 32)).amin(-1)) / 15
            assert bool(((x - y).unflatten(-1, (-1, 32)).abs() <= 15 * 2.0 ** -10 * step[..., None] + 1e-6).all())


def test_kv_bits_sizes_and_refusals():
    from exo_b200.models.config import preset
    from exo_b200.models.transformer import KVPool, make_kv_pool
    from exo_b200.models.weights import ShardSpec
    cfg = preset("llama-3.1-8b")
    b16, b4 = KVPool.bytes_per_block(cfg, ShardSpec()), KVPool.bytes_per_block(cfg, ShardSpec(), 16, 4)
    assert b4 * 16 == b16 * 5
    pool = make_kv_pool(preset("tiny-llama"), ShardSpec(), 4, kv_bits=4)
    assert sum(c.nbytes() for kv in pool.layers.values() for c in kv) == 4 * KVPool.bytes_per_block(preset("tiny-llama"), ShardSpec(), 16, 4)
    for bad, bits in ((preset("tiny-llama"), 8), (preset("deepseek-v3"), 4)):
        with pytest.raises(ValueError):
            KVPool.bytes_per_block(bad, ShardSpec(), 16, bits)
        with pytest.raises(ValueError):
            make_kv_pool(bad, ShardSpec(), 4, kv_bits=bits)
    narrow = preset("tiny-llama")
    narrow.head_dim = 32
    with pytest.raises(ValueError):
        make_kv_pool(narrow, ShardSpec(), 4, kv_bits=4)


def test_more_refusals():
    with pytest.raises(ValueError, match="heads"):
        ops.Kv4Cache(torch.zeros(4, 0, 1, 640, dtype=torch.uint8), 64, "k")
    with pytest.raises(ValueError, match="heads"):
        ops.Kv4Cache(torch.zeros(4, 2, 0, 640, dtype=torch.uint8), 64, "k")
    kc, vc = (ops.Kv4Cache.zeros(2, 16, 1, 64, kind) for kind in "kv")
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.kv4_read(kc, vc, torch.zeros(1, dtype=torch.int32), torch.float16)
    inv = torch.ones(32)
    with pytest.raises(ValueError, match="axes"):
        ops.qk_rope_append(torch.zeros(0, 192), torch.zeros(0, 0, dtype=torch.int32), inv, 1.0, 1, 1, 64, kc, vc,
                           torch.zeros(0, dtype=torch.int32), axes=torch.zeros(32, dtype=torch.int32))
    with pytest.raises(ValueError, match="qk_rope_append"):
        ops.qk_rope_append(torch.zeros(()), torch.zeros(0, dtype=torch.int32), inv, 1.0, 1, 1, 64, kc, vc, torch.zeros(0))


def test_sinks_do_not_fill_empty_rows():
    kc, vc = filled_pair(2, 16, 1, 64, "cpu")
    q = torch.ones(3, 2, 64)
    cu, n = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)       # two rows before the first key
    for sinks in (torch.zeros(2), torch.full((2,), -math.inf)):
        out = ops.paged_attention(q, kc, vc, torch.zeros(1, 1, dtype=torch.int32), n, cu, 0.1, 0, sinks)
        assert not out[:2].any() and bool(out[2].abs().sum() > 0) and not out.isnan().any()


def test_axes_outside_positions_are_the_nearest():
    qkv, pos, inv = torch.randn(2, 192), torch.tensor([[1, 2], [5, 9]], dtype=torch.int32), torch.rand(32)
    for given, taken in ((7, 1), (-3, 0)):
        made = []
        for ax in (given, taken):
            kc, vc = (ops.Kv4Cache.zeros(1, 16, 1, 64, kind) for kind in "kv")
            q = ops.qk_rope_append(qkv, pos, inv, 1.0, 1, 1, 64, kc, vc, torch.arange(2), axes=torch.full((32,), ax))
            made.append((q, kc.data, vc.data))
        assert all(torch.equal(a, b) for a, b in zip(*made))
