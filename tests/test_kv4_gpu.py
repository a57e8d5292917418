"""The kernels of the 4-bit KV cache on a B200, against their definitions in 64 bits."""
import os
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from exo_b200 import ops
from exo_b200.ops import kv4
from kv4_cases import append64, attention64, batch, check_attention, check_held, filled_pair

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _append(dtype, T, nq, nkv, d, rot, norm, axes, bs, quantized, device="cuda", v_unit=False, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed + T + d)
    qkv = torch.randn(T, (nq + 2 * nkv) * d + pad, generator=g).to(dtype)
    qn, kn = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype) if norm else None for _ in range(2))
    inv = (10000.0 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))).float()
    ax = (torch.arange(rot // 2) % 3).int() if axes else None
    pos = torch.randint(0, 131072, (3, T) if axes else (T,), generator=g).int()
    nb = -(-T // bs) + 2
    slots = torch.randperm(nb * bs, generator=g)[:T].int()
    if T > 2:
        slots[1], slots[2] = -1, nb * bs            # neither is stored
    if quantized:
        kc, vc = (ops.Kv4Cache.zeros(nb, bs, nkv, d, kind, device) for kind in "kv")
    else:
        kc, vc = (torch.zeros(nb, bs, nkv, d, dtype=dtype, device=device) for _ in range(2))
    dev = lambda t: None if t is None else t.to(device)      # noqa: E731
    rows = dev(qkv)[:, :qkv.shape[1] - pad] if pad else dev(qkv)
    q = ops.qk_rope_append(rows, dev(pos), dev(inv), 1.25, nq, nkv, d, kc, vc, dev(slots), dev(qn), dev(kn), 1e-6, v_unit, axes=dev(ax))
    want = append64(qkv[:, :qkv.shape[1] - pad].contiguous(), pos, inv, 1.25, nq, nkv, d, qn, kn, 1e-6, v_unit, ax)
    # fp32 throughout: a row's norm, its turn and the angle's last reduction are each off by some 2^-22 of the row's largest
    slack = lambda x: 2.0 ** -20 * x.abs().amax(-1, keepdim=True)      # noqa: E731
    half = torch.finfo(dtype).eps / 2
    if nq:
        assert bool(((q.cpu().double() - want[0]).abs() <= half * want[0].abs() + slack(want[0])).all())
    kept = (slots >= 0) & (slots < nb * bs)
    for cache, x in zip((kc, vc), want[1:] if nkv else ()):
        if quantized:
            check_held(cache, slots[kept], x[kept])
        else:
            got = cache.view(-1, nkv, d)[slots[kept].to(device).long()].cpu().double()
            assert bool(((got - x[kept]).abs() <= half * x[kept].abs() + slack(x[kept])).all())
    if quantized:
        left = torch.ones(nb * bs, dtype=torch.bool)
        left[slots[kept].long()] = False
        for t in ops.kv4_read(kc, vc, torch.nonzero(left)[:, 0].int().to(device)):
            assert not t.any()                      # slots that were not named are as they were


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 4), (128, 128), (128, 64), (128, 0), (256, 64), (256, 256), (256, 16)])
@pytest.mark.parametrize("T,nq,nkv", [(1, 8, 2), (3, 5, 5), (67, 6, 1)])
def test_append(dtype, d, rot, T, nq, nkv):
    _append(dtype, T, nq, nkv, d, rot, norm=T != 3, axes=rot > 4 and T == 67, bs=16 if T < 60 else 48, quantized=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_axes_plain_cache(dtype, d):
    _append(dtype, 35, 4, 2, d, d, norm=True, axes=True, bs=16, quantized=False)


def test_append_many_tokens_and_strided_rows():
    _append(BF, 1500, 16, 4, 128, 128, norm=True, axes=True, bs=16, quantized=True)
    _append(BF, 40, 4, 2, 128, 64, norm=True, axes=False, bs=32, quantized=True, pad=8, v_unit=True)
    _append(BF, 40, 4, 2, 128, 64, norm=False, axes=False, bs=32, quantized=True, pad=3)        # rows off their alignment
    _append(BF, 40, 0, 2, 64, 0, norm=False, axes=False, bs=16, quantized=True)
    _append(F32, 40, 4, 0, 64, 64, norm=False, axes=True, bs=16, quantized=False)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_in_and_out(d, dtype):
    g = torch.Generator().manual_seed(d)
    kc, vc = (ops.Kv4Cache.zeros(7, 32, 3, d, kind, "cuda") for kind in "kv")
    slots = torch.randperm(7 * 32, generator=g)[:101].int()
    k, v = ((torch.randn(101, 3, d, generator=g) * 9 + 4).to(dtype) for _ in range(2))
    ops.kv4_write(k.cuda(), v.cuda(), kc, vc, slots.cuda())
    hk, hv = (ops.Kv4Cache.zeros(7, 32, 3, d, kind) for kind in "kv")
    ops.kv4_write(k, v, hk, hv, slots)
    assert torch.equal(kc.data.cpu(), hk.data) and torch.equal(vc.data.cpu(), hv.data)      # the same bytes as the definition's
    for got, want in zip(ops.kv4_read(kc, vc, slots.cuda(), dtype), ops.kv4_read(hk, hv, slots, F32)):
        err = (got.cpu().double() - want.double()).abs()
        # one fp32 rounding here (fma), two there
        assert bool((err <= (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * want.abs() + 2.0 ** -22 * want.abs().max()).all())
    bad = torch.tensor([-5, 7 * 32, int(slots[0])], dtype=torch.int32, device="cuda")
    k2, v2 = ops.kv4_read(kc, vc, bad, F32)
    assert not k2[:2].any() and not v2[:2].any() and k2[2].any()


def test_extreme_rows_match_the_definition():
    x = torch.zeros(6, 2, 128)
    x[0] = 3.0
    x[1, 0, 3], x[1, 0, 40] = float("inf"), -1e30
    x[2, 0, 9] = float("nan")
    x[3] = 2.0 ** -26 * torch.arange(128)
    x[4, 0, 0] = -0.0
    x[5] = torch.linspace(-65504, 65504, 128)
    made = []
    for device in ("cpu", "cuda"):
        kc, vc = (ops.Kv4Cache.zeros(1, 16, 2, 128, kind, device) for kind in "kv")
        ops.kv4_write(x.to(device), x.to(device), kc, vc, torch.arange(6, device=device))
        made.append([t.cpu() for t in ops.kv4_read(kc, vc, torch.arange(6, device=device), F32)])
    for a, b in zip(*made):
        assert torch.equal(a.isnan(), b.isnan())
        # one rounding in the kernel (fma), two in the definition, of numbers up to 16 steps apart
        assert float((a - b).nan_to_num().abs().max()) <= 65504 * 2.0 ** -22


def _attention(dtype, lens, hq, hkv, d, bs=16, window=0, sinks=False, max_q=None, tail=0, seed=0, spread=1.0, offset=0.0, q_spread=1.5):
    pages = sum(-(-k // bs) for _, k in lens)
    kc, vc = filled_pair(pages + 3, bs, hkv, d, "cuda", seed, spread, offset)
    table, n, cu = batch(lens, bs, pages + 3, seed)
    g = torch.Generator().manual_seed(seed + 7)
    q = (torch.randn(int(cu[-1]) + tail, hq, d, generator=g) * q_spread).to(dtype)
    sk = torch.linspace(-1, 2, hq) if sinks else None
    out, bound = attention64(q, kc, vc, table, n, cu, d ** -0.5, window, sk)
    for sink in ((sk, sk.to(BF)) if sinks == "both" else (sk,)):
        got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), n.cuda(), cu.cuda(), d ** -0.5, window,
                                  None if sink is None else sink.cuda(), max_q)
        if sink is not None and sink.dtype is BF:
            out, bound = attention64(q, kc, vc, table, n, cu, d ** -0.5, window, sink)
        check_attention(got, out, bound)
    if tail:
        assert not got[int(cu[-1]):].any()


RAGGED = [(1, 1), (3, 40), (17, 17), (2, 33), (1, 0), (0, 0), (70, 301), (1, 16)]
HEADS = [(4, 4), (6, 2), (8, 1), (16, 2), (12, 1), (24, 1), (20, 4)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_prompt_attention(dtype, d, hq, hkv):
    _attention(dtype, RAGGED, hq, hkv, d, bs=16 if hkv == 1 else 32, tail=3)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 64, 100])
def test_prompt_attention_window_and_sinks(dtype, d, window):
    _attention(dtype, RAGGED, 8, 2, d, window=window, sinks="both" if window == 64 else window == 5)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode_attention(dtype, d, hq, hkv):
    lens = [(1, k) for k in (1, 2, 15, 16, 17, 0, 63, 64, 65, 127, 200, 513, 31, 32, 33)]
    _attention(dtype, lens, hq, hkv, d, bs=16 if hkv == 1 else 48, max_q=1)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 64, 100])
def test_decode_attention_window_and_sinks(dtype, d, window):
    _attention(dtype, [(1, k) for k in (1, 4, 5, 6, 64, 65, 300, 1000, 0)], 16, 2, d, window=window,
               sinks="both" if window == 64 else window == 5, max_q=1)


def test_decode_one_long_sequence():
    _attention(BF, [(1, 20011)], 8, 2, 128, max_q=1)
    _attention(BF, [(1, 9001), (1, 3), (1, 4096)], 16, 1, 128, max_q=1)


def test_prompt_few_rows_many_keys():
    _attention(BF, [(5, 9000), (1, 700)], 8, 2, 128)
    _attention(BF, [(33, 5000)], 8, 1, 256)
    _attention(BF, [(40, 3001)], 8, 1, 64, sinks=True)


@pytest.mark.parametrize("max_q,lens", [(1, [(1, 700), (1, 90)]), (None, [(130, 700), (9, 90)])])
def test_value_and_query_ranges(max_q, lens):
    """Values and scales from fp16's ends, queries of any size (peaked softmax, all-equal logits)."""
    for spread, offset in ((2.0 ** -12, 0.0), (3000.0, 0.0), (0.01, 300.0)):
        _attention(BF, lens, 8, 2, 128, max_q=max_q, spread=spread, offset=offset, q_spread=1.0 / max(spread, 0.01))
    _attention(BF, lens, 8, 2, 128, max_q=max_q, q_spread=12.0)
    _attention(BF, lens, 8, 2, 128, max_q=max_q, q_spread=1e-30)
    _attention(BF, lens, 8, 2, 128, max_q=max_q, q_spread=0.0)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("max_q,lens", [(1, [(1, 37), (1, 130)]), (None, [(2, 37), (20, 130)])])
def test_what_nobody_sees_may_be_nan(d, max_q, lens):
    kc, vc = filled_pair(16, 16, 2, d, "cuda")
    table, n, cu = batch(lens, 16, 16)
    q = torch.randn(int(cu[-1]), 8, d, generator=torch.Generator().manual_seed(2)).to(BF).cuda()
    args = (table.cuda(), n.cuda(), cu.cuda(), d ** -0.5, 10, None, max_q)
    want = ops.paged_attention(q, kc, vc, *args)
    hidden = torch.ones(256, dtype=torch.bool)
    for b, (new, keys) in enumerate(lens):
        seen = torch.arange(max(0, keys - new - 9), keys)
        hidden[table[b].long()[seen // 16] * 16 + seen % 16] = False
    bad = torch.full((int(hidden.sum()), 2, d), float("nan"), device="cuda")
    ops.kv4_write(bad, bad, kc, vc, torch.nonzero(hidden)[:, 0].cuda())
    assert torch.equal(ops.paged_attention(q, kc, vc, *args), want)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("max_q,lens", [(1, [(1, 37), (1, 130)]), (None, [(2, 37), (90, 130)])])
def test_a_nan_row_reaches_the_queries_that_see_it(d, max_q, lens):
    for which in (0, 1):
        kc, vc = filled_pair(16, 16, 2, d, "cuda")
        table, n, cu = batch(lens, 16, 16)
        q = torch.randn(int(cu[-1]), 4, d, generator=torch.Generator().manual_seed(2)).to(BF)
        at = 110                                   # of the second sequence, first head
        slot = table[1].long()[at // 16] * 16 + at % 16
        k, v = ops.kv4_read(kc, vc, slot.view(1).cuda(), F32)
        (k, v)[which][0, 0, 5] = float("nan")
        ops.kv4_write(k, v, kc, vc, slot.view(1).cuda())
        out, bound = attention64(q, kc, vc, table, n, cu, d ** -0.5)
        got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), n.cuda(), cu.cuda(), d ** -0.5, 0, None, max_q).cpu()
        rows = torch.arange(q.shape[0]) - int(cu[1])
        sees = (rows >= 0) & (rows + lens[1][1] - lens[1][0] >= at)
        assert bool(got[sees][:, :2].isnan().all()) and not got[~sees].isnan().any() and not got[:, 2:].isnan().any()
        calm = ~got.isnan()
        assert bool(((got.double() - out).abs() <= bound * 1.01 + 2.0 ** -8 * out.abs())[calm].all())


def test_bad_pages_and_lengths_stay_inside():
    """Page numbers outside the cache and lengths past the table are clamped: nothing faults, other sequences are untouched."""
    for max_q, lens in ((1, [(1, 40), (1, 60)]), (None, [(3, 40), (9, 60)])):
        kc, vc = filled_pair(8, 16, 2, 128, "cuda")
        table, n, cu = batch(lens, 16, 8, width=4)
        q = torch.randn(int(cu[-1]), 8, 128, generator=torch.Generator().manual_seed(2)).to(BF).cuda()
        want = ops.paged_attention(q, kc, vc, table.cuda(), n.cuda(), cu.cuda(), 0.1, 0, None, max_q)
        table[1, 1], table[1, 2], n[1] = 8, -3, 1000
        got = ops.paged_attention(q, kc, vc, table.cuda(), n.cuda(), cu.cuda(), 0.1, 0, None, max_q)
        assert torch.equal(got[:int(cu[1])], want[:int(cu[1])])
        torch.cuda.synchronize()


def test_a_cache_past_32_bits():
    """Units whose byte offset is past 2^32: the last pages of a 5 GiB cache."""
    nb = 270_000
    data = [torch.zeros(nb, 8, 1, 1280 * 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    kc, vc = ops.Kv4Cache(data[0], 256, "k"), ops.Kv4Cache(data[1], 256, "v")
    table = torch.tensor([[nb - 1, 3, nb - 2]], dtype=torch.int32)
    slots = torch.cat([table[0, i] * 16 + torch.arange(16) for i in range(3)]).int().cuda()
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(48, 8, 256, generator=g) for _ in range(2))
    ops.kv4_write(k.cuda(), v.cuda(), kc, vc, slots)
    rk, rv = ops.kv4_read(kc, vc, slots, F32)
    for got, want in ((rk, k), (rv, v)):
        held = kv4.dequantize(*kv4.quantize(want))
        assert float((got.cpu() - held).abs().max()) <= 2.0 ** -20
    small = [ops.Kv4Cache(c.data[torch.tensor([nb - 1, 3, nb - 2], device="cuda")].clone(), 256, c.kind) for c in (kc, vc)]
    for new, max_q in ((1, 1), (30, None)):
        q = torch.randn(new, 16, 256, generator=g).to(BF).cuda()
        cu, n = torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([45], dtype=torch.int32).cuda()
        big = ops.paged_attention(q, kc, vc, table.cuda(), n, cu, 0.06, 0, None, max_q)
        ref = ops.paged_attention(q, *small, torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), n, cu, 0.06, 0, None, max_q)
        assert torch.equal(big, ref)
    del data, kc, vc
    torch.cuda.empty_cache()


# ---- streams, graphs, an engine ---------------------------------------------------------------------------------------------
def _decode_call(seed, lens, hq=8, hkv=2, d=128):
    pages = sum(-(-k // 16) for _, k in lens)
    kc, vc = filled_pair(pages + 2, 16, hkv, d, "cuda", seed)
    table, n, cu = batch(lens, 16, pages + 2, seed)
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(seed)).to(BF).cuda()
    table, n, cu = table.cuda(), n.cuda(), cu.cuda()
    return lambda: ops.paged_attention(q, kc, vc, table, n, cu, d ** -0.5, 0, None, 1), n


LONG = [(1, 9000), (1, 70), (1, 5000)]           # rows that several CTAs share


def test_calls_on_two_streams_at_once():
    calls = [_decode_call(s, LONG)[0] for s in (1, 2)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_two_graphs_replayed_at_once():
    calls = [_decode_call(s, LONG)[0] for s in (3, 4)]
    want = [c() for c in calls]
    side, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for c in calls:                               # both captured on one stream
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append([c() for _ in range(8)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in outs[i])


def test_a_graph_follows_lengths_that_change():
    call, n = _decode_call(5, LONG)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for lens in ([9000, 70, 5000], [1, 0, 3], [8999, 64, 4097], [0, 0, 0]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        assert torch.equal(out, call())


def test_capture_of_append_and_prompt():
    kc, vc = filled_pair(40, 16, 2, 128, "cuda")
    table, n, cu = (t.cuda() for t in batch([(20, 500), (3, 30)], 16, 40))
    qkv = torch.randn(23, 12 * 128, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    pos = torch.cat((torch.arange(480, 500), torch.arange(27, 30))).int().cuda()
    seq = torch.tensor([0] * 20 + [1] * 3).cuda()
    slots = (table[seq, pos.long() // 16] * 16 + pos % 16).int()
    inv = (10000.0 ** (-torch.arange(0, 128, 2, device="cuda") / 128)).float()
    def step():
        q = ops.qk_rope_append(qkv, pos, inv, 1.0, 8, 2, 128, kc, vc, slots)
        return ops.paged_attention(q, kc, vc, table, n, cu, 128 ** -0.5)
    want = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    out.zero_()
    g.replay()
    assert torch.equal(out, want)


def test_prompt_rows_equal_decode_rows():
    """The last row of a prompt and the single-token call of the same query differ by the prompt kernel's roundings alone."""
    for d, hq, hkv in ((64, 8, 1), (128, 32, 8), (256, 16, 2)):
        kc, vc = filled_pair(70, 16, hkv, d, "cuda")
        table, n, cu = batch([(1, 1000)], 16, 70)
        q = torch.randn(1, hq, d, generator=torch.Generator().manual_seed(d)).to(BF)
        out, bound = attention64(q, kc, vc, table, n, cu, d ** -0.5)
        for max_q in (1, None):
            got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), n.cuda(), cu.cuda(), d ** -0.5, 0, None, max_q)
            check_attention(got, out, bound)


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 1), (128, 8, 2), (256, 4, 1)])
def test_engine_serves_from_a_4_bit_cache(d, hq, hkv):
    from exo_b200.engine.engine import Engine
    from exo_b200.engine.kv import SamplingParams
    from exo_b200.models.config import ModelConfig, RopeConfig
    from exo_b200.models.weights import ShardSpec, fast_random_weights
    cfg = ModelConfig(name="t", n_layers=2, hidden=512, n_heads=hq, n_kv_heads=hkv, head_dim=d, ffn=1024, vocab=4096, qk_norm=True,
                      rope=RopeConfig(theta=500000.0), dtype="bf16")
    w = fast_random_weights(cfg, ShardSpec(), "cuda")
    prompts = [torch.randint(0, 4096, (k,), generator=torch.Generator().manual_seed(k)).tolist() for k in (50, 31, 177)]
    runs = []
    for graphs, chunk in ((False, 4096), (True, 4096), (True, 48)):
        eng = Engine(cfg, w, n_blocks=128, device="cuda", use_graphs=graphs, max_seqs=4, prefill_chunk=chunk, kv_bits=4)
        ids = [eng.submit(p, SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True), use_prefix_cache=False) for p in prompts]
        got = {i: [] for i in ids}
        while eng.has_work:
            for o in eng.step():
                if o.token is not None:
                    got[o.req_id].append(o.token)
        runs.append([got[i] for i in ids])
    assert runs[0] == runs[1]                       # a graph replays what an eager step computes
    assert all(len(x) == 12 for r in runs for x in r)
    # the first answer's logits against the same model over a 16-bit cache: what 4 bits cost (a step of a 15th of a group's range
    # is some 0.08 of a normal row's norm, in keys and values alike), and nothing of a mistake's size
    logits = []
    for bits in (4, 16):
        eng = Engine(cfg, w, n_blocks=128, device="cuda", use_graphs=False, max_seqs=4, kv_bits=bits)
        eng.submit(prompts[2], SamplingParams(max_tokens=1, temperature=0.0, ignore_eos=True), use_prefix_cache=False)
        eng.step()
        logits.append(eng.exe.last_logits[0].float())
    assert float((logits[0] - logits[1]).norm() / logits[1].norm()) < 0.2


# ---- calls that few make ----------------------------------------------------------------------------------------------------
def test_unaligned_arguments():
    """Views that start between 16-byte boundaries: the rows are moved, the results the same."""
    off = lambda t, n: torch.cat((t.new_zeros(n), t.reshape(-1)))[n:].view(t.shape)      # noqa: E731
    for d, dtype in ((128, BF), (256, F32), (64, BF)):
        kc, vc = filled_pair(8, 16, 2, d, "cuda")
        g = torch.Generator().manual_seed(3)
        for lens, max_q in (([(1, 40), (1, 60)], 1), ([(3, 40), (9, 60)], None)):
            table, n, cu = (t.cuda() for t in batch(lens, 16, 8))
            q = torch.randn(int(cu[-1]), 8, d, generator=g).to(dtype).cuda()
            sinks = torch.linspace(-1, 1, 8).cuda()
            a = ops.paged_attention(q, kc, vc, table, n, cu, 0.1, 0, sinks, max_q)
            b = ops.paged_attention(off(q, 1), kc, vc, off(table, 1), off(n, 1), off(cu, 1), 0.1, 0, off(sinks, 1), max_q)
            assert torch.equal(a, b)
        T = 5
        qkv = torch.randn(T, 12 * d, generator=g).to(dtype).cuda()
        pos, slots = torch.arange(T).int().cuda(), torch.arange(T).int().cuda() + 3
        inv = torch.rand(d // 2, generator=g).cuda()
        w = torch.rand(2, d, generator=g).to(dtype).cuda()
        made = []
        for mv in (lambda t: t, lambda t: off(t, 1)):
            kc, vc = (ops.Kv4Cache.zeros(2, 16, 2, d, kind, "cuda") for kind in "kv")
            out = ops.qk_rope_append(mv(qkv), mv(pos), mv(inv), 1.0, 8, 2, d, kc, vc, mv(slots), mv(w[0]), mv(w[1]))
            k, v = (mv(torch.ones(T, 2, d, device="cuda", dtype=dtype) * torch.arange(d, device="cuda").to(dtype)) for _ in range(2))
            ops.kv4_write(k, v, kc, vc, mv(slots + 10))
            made.append((out, kc.data, vc.data))
        assert all(torch.equal(a, b) for a, b in zip(*made))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_scales_of_either_sign_and_zero(d, dtype):
    """A negative scale is the same as negated queries; with none, a row is the mean of the values that it sees."""
    for lens, max_q in (([(1, 40), (1, 700)], 1), ([(3, 40), (150, 300)], None)):
        kc, vc = filled_pair(80, 16, 2, d, "cuda")
        table, n, cu = batch(lens, 16, 80)
        q = torch.randn(int(cu[-1]), 8, d, generator=torch.Generator().manual_seed(1)).to(dtype)
        args = (kc, vc, table.cuda(), n.cuda(), cu.cuda())
        out, bound = attention64(-q, kc, vc, table, n, cu, d ** -0.5, 50)
        check_attention(ops.paged_attention(q.cuda(), *args, -(d ** -0.5), 50, None, max_q), out, bound)
        out, bound = attention64(q * 0, kc, vc, table, n, cu, 1.0, 50)
        check_attention(ops.paged_attention(q.cuda(), *args, 0.0, 50, None, max_q), out, bound)
        check_attention(ops.paged_attention((q * 0).cuda(), *args, 1e-12, 50, None, max_q), out, bound)


def test_windows_past_32_bits_hide_nothing():
    for lens, max_q in (([(1, 40), (1, 700)], 1), ([(3, 40), (150, 300)], None)):
        kc, vc = filled_pair(80, 16, 2, 128, "cuda")
        table, n, cu = (t.cuda() for t in batch(lens, 16, 80))
        for dtype in (BF, F32):
            q = torch.randn(int(cu[-1]), 8, 128, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
            want = ops.paged_attention(q, kc, vc, table, n, cu, 0.1, 0, None, max_q)
            for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40):
                assert torch.equal(ops.paged_attention(q, kc, vc, table, n, cu, 0.1, window, None, max_q), want)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_run_of_nan_keys(d):
    """Every key that some warp (or some split) of a row meets is NaN: the row is NaN, not the others' result."""
    for lens, max_q in (([(1, 200), (1, 30)], 1), ([(1, 1), (1, 30)], 1), ([(2, 200), (3, 30)], None), ([(2, 5000), (3, 30)], None)):
        for dtype in (BF, F32):
            if dtype is F32 and lens[0][1] > 200:
                continue
            kc, vc = filled_pair(340, 16, 2, d, "cuda")
            table, n, cu = (t.cuda() for t in batch(lens, 16, 340))
            q = torch.randn(int(cu[-1]), 4, d, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
            for lo, hi in ((0, min(32, lens[0][1])), (lens[0][1] // 2, lens[0][1])):
                at = torch.arange(lo, hi, device="cuda")
                if not len(at):
                    continue
                k, v = filled_pair(340, 16, 2, d, "cuda")
                slots = table[0].long()[at // 16] * 16 + at % 16
                rk, rv = ops.kv4_read(k, v, slots, F32)
                ops.kv4_write(rk * float("nan"), rv, k, v, slots)
                for sinks in (None, torch.zeros(4, device="cuda")):
                    got = ops.paged_attention(q, k, v, table, n, cu, 0.1, 0, sinks, max_q)
                    first = int(cu[1])
                    assert bool(got[first - 1].isnan().all()) and not got[first:].isnan().any()


def test_many_rows_behind_the_last_sequence():
    """A padded batch: the rows behind are zero, whatever was in the output's memory."""
    kc, vc = filled_pair(80, 16, 2, 128, "cuda")
    table, n, cu = (t.cuda() for t in batch([(3, 40), (150, 300)], 16, 80))
    for T in (153, 154, 5000):
        q = torch.randn(T, 8, 128, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
        torch.full((T, 8, 128), float("nan"), dtype=BF, device="cuda")       # (freed: the next output's memory)
        got = ops.paged_attention(q, kc, vc, table, n, cu, 0.1)
        assert not got[153:].any() and not got.isnan().any()
        assert torch.equal(got[:153], ops.paged_attention(q[:153].contiguous(), kc, vc, table, n, cu, 0.1)) or T > 154


def test_single_token_call_of_longer_sequences():
    """``max_q_len=1`` only says how the work is cut: rows of longer sequences come out right all the same."""
    _attention(BF, RAGGED, 8, 2, 128, max_q=1)


def test_indices_past_32_bits():
    kc, vc = filled_pair(4, 16, 2, 64, "cuda")
    before = kc.data.clone()
    slots = torch.tensor([2 ** 32 + 3, -(2 ** 32) + 5, 2 ** 31, -1], device="cuda")
    rows = torch.ones(4, 2, 64, device="cuda")
    ops.kv4_write(rows, rows, kc, vc, slots)
    assert torch.equal(kc.data, before)
    assert not any(x.any() for x in ops.kv4_read(kc, vc, slots, F32))


def test_streams_of_two_threads():
    """First calls of many streams, from two threads at once: none shares another's counters."""
    call, _ = _decode_call(6, LONG)
    want = call()
    torch.cuda.synchronize()
    out = [[], []]

    def run(i):
        for _ in range(12):
            with torch.cuda.stream(torch.cuda.Stream()):
                out[i].append(call())
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(out[0]) == len(out[1]) == 12 and all(torch.equal(x, want) for o in out for x in o)


def test_same_slot_twice_keeps_the_others():
    """Rows with one slot leave it with some row or a mixture; every other slot is what it would be."""
    kc, vc = filled_pair(4, 16, 2, 128, "cuda")
    ref_k = kc.data.clone()
    rows = torch.randn(3, 2, 128, device="cuda")
    ops.kv4_write(rows, rows, kc, vc, torch.tensor([9, 9, 9], device="cuda"))
    changed = ops.Kv4Cache(ref_k, 128, "k")
    others = torch.tensor([i for i in range(64) if i != 9], device="cuda")
    a, _ = ops.kv4_read(kc, vc, others, F32)
    b, _ = ops.kv4_read(changed, vc, others, F32)
    assert torch.equal(a, b)


def test_checks_flavour():
    """With EXO_KERNEL_CHECKS=1 nothing stores behind its output, and a slot outside the cache is still a row not kept."""
    code = """
import torch
from exo_b200 import ops
from exo_b200.ops import cuda
kc, vc = (ops.Kv4Cache.zeros(4, 16, 2, 128, kind, "cuda") for kind in "kv")
pos, slots = torch.arange(5).int().cuda(), torch.tensor([-1, 3, 64, 7, 40]).int().cuda()
q = ops.qk_rope_append(torch.randn(5, 12 * 128, device="cuda").bfloat16(), pos, torch.rand(64, device="cuda"), 1.0, 8, 2, 128, kc, vc, slots)
k, _ = ops.kv4_read(kc, vc, slots)
assert [bool(x.any()) for x in k] == [False, True, False, True, True]
n, table = torch.tensor([5]).int().cuda(), torch.tensor([[0, 1]]).int().cuda()
for max_q in (None, 1):
    ops.paged_attention(q, kc, vc, table, n, torch.tensor([0, 5]).int().cuda(), 0.1, max_q_len=max_q)
cuda.verify_guards()
print("fine")
"""
    out = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, EXO_KERNEL_CHECKS="1"), capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert out.returncode == 0 and out.stdout.strip().endswith("fine"), out.stderr[-2000:]


@pytest.mark.parametrize("bs", [32, 48, 112, 256])
def test_pages_of_other_sizes(bs):
    for d, hq, hkv in ((64, 8, 1), (128, 6, 2), (256, 4, 2)):
        _attention(BF, RAGGED, hq, hkv, d, bs=bs)
        _attention(BF, RAGGED, hq, hkv, d, bs=bs, window=37, sinks=True)
        _attention(BF, [(1, n) for n in (1, 31, 33, 300, 0, 113)], hq, hkv, d, bs=bs, max_q=1)
        _attention(F32, RAGGED, hq, hkv, d, bs=bs)
    _attention(BF, [(5, 3000)], 8, 2, 128, bs=bs)


@pytest.mark.parametrize("hq,hkv", [(160, 1), (300, 2)])
def test_more_heads_to_a_key_head_than_a_tile_has_rows(hq, hkv):
    _attention(BF, [(3, 40), (1, 1), (2, 90)], hq, hkv, 64)
    _attention(BF, [(1, 40), (1, 1), (1, 90)], hq, hkv, 64, max_q=1)
    _attention(F32, [(1, 40), (2, 9)], hq, hkv, 64)
