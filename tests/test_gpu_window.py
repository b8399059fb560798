"""Sliding-window attention with sinks, decode and prefill, against a plain
implementation in 64 bits that only ever touches the tokens a row sees.

The bound of an output element: the weights and the output are each rounded once
to the 16-bit type (half a step u, relative), scores are sums of D products in
32 bits, and a score that is off by s changes every weight by at most
exp(2 s) - 1; fp16 weights below 2^-24 of a row's largest round to multiples
of 2^-24."""

import copy
import math

import numpy as np
import pytest
import torch

import pagedattn
from pagedattn import llama as L
from pagedattn.metadata import decode_metadata, prefill_metadata

from paged_cases import (i32, random_tables, require_fixed_chunks, require_shared_plans,
                         strided_rows, workspace)

pytestmark = pytest.mark.gpu


@pytest.fixture
def general(monkeypatch):
    """The calls' general path: the extension takes nothing."""
    monkeypatch.setattr(pagedattn.ops, "_native", lambda *a: NotImplemented)


HEADS = [(32, 4, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128)]


def make(device, computed, chunks, heads, dtype, fp8, window, sinks, seed, spoil=True):
    """A paged batch whose unseen tokens hold NaN and infinities (spoil) and whose
    unseen pages are gone (-1) or name a page of NaN."""
    hq, hkv, d = heads
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in zip(computed, chunks)]
    tables, num_pages = random_tables(rng, lens, extra_pages=4)
    meta = prefill_metadata(tables, computed, chunks)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    pool = torch.randn((num_pages, 2, hkv, 16, d), generator=g, device=device)
    scales = None
    if fp8:
        scales = (torch.rand((num_pages, 2, hkv), generator=g, device=device) + 0.5) / 64
        pool = (pool / scales[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        pool = pool.to(dtype)
    q = strided_rows(meta.nnz, hq, d, dtype, device, g, tail=2 * hkv)
    if spoil:
        trash = sorted(set(range(num_pages)) - {p for t in tables for p in t})[0]
        bad = [math.nan, math.nan] if fp8 else [math.nan, math.inf]
        pool[trash] = math.nan
        for b, (n, table) in enumerate(zip(lens, tables)):
            first = n - chunks[b] - window  # the first token past the sinks that a row sees
            for t in range(min(sinks, n), min(first, n)):
                pool[table[t // 16], 0, :, t % 16] = bad[t % 2]
                pool[table[t // 16], 1, :, t % 16] = bad[(t + 1) % 2]
            lo, hi = -(-sinks // 16), max(first, 0) // 16
            for s in range(lo, min(hi, len(table))):
                meta.kv_indices[meta.kv_indptr[b] + s] = -1 if s % 2 else trash
    return meta, pool, scales, q


def rows64(pool, scales, ids, kind, tokens):
    page = torch.as_tensor(ids, device=pool.device)[tokens // 16].long()
    x = pool[page, kind, :, tokens % 16].double()
    return x if scales is None else x * scales[page, kind].double()[..., None]


def reference(meta, pool, scales, q, window, sinks, causal=True, b_rows=None, q_err=0.0):
    """(out, lse, bound of out, bound of lse) in 64 bits; q_err: relative rounding of q."""
    dev, (n, hq, d) = q.device, q.shape
    hkv = pool.shape[2]
    g = hq // hkv
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    out = torch.zeros((n, hq, d), dtype=torch.float64, device=dev)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=dev)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(len(meta.kv_last_page_len)):
        ids = meta.kv_indices[meta.kv_indptr[b]:meta.kv_indptr[b + 1]]
        length = (len(ids) - 1) * 16 + int(meta.kv_last_page_len[b]) if len(ids) else 0
        r0, r1 = int(meta.qo_indptr[b]), int(meta.qo_indptr[b + 1])
        for r in range(r0, r1):
            if b_rows is not None and r not in b_rows:
                continue
            at = length - (r1 - r0) + r - r0
            end = min(at + 1, length) if causal else length
            tok = torch.arange(max(end, 0), device=dev)
            tok = tok[(tok >= at - window) | (tok < sinks)]
            if not tok.numel():
                continue
            k, v = (rows64(pool, scales, ids, i, tok).repeat_interleave(g, 1) for i in (0, 1))
            x = q[r].double()[:, None]
            s = (k.transpose(0, 1) * x).sum(-1) / math.sqrt(d)  # [hq, tokens]
            size = (k.transpose(0, 1) * x).abs().sum(-1).amax(-1) / math.sqrt(d)
            lse[r] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[r][:, None])[..., None]
            vt = v.transpose(0, 1)
            out[r] = (p * vt).sum(1)
            spread = (p * vt.abs()).sum(1)
            off = size * (q_err + (d + 8) * 2.0 ** -24) + s.abs().amax(-1) * 2.0 ** -21
            codes = vt.abs().amax(1) if scales is None else vt.abs().amax(1) * 64 * 2
            out_tol[r] = (u * out[r].abs() + spread * (u * 1.01 + torch.expm1(2 * off)[:, None])
                          + tok.numel() * tiny * codes
                          * torch.exp(s.amax(-1) - lse[r])[:, None] + 2.0 ** -24)
            lse_tol[r] = off + lse[r].abs() * 2.0 ** -21 + 2.0 ** -20
    return out, lse, out_tol, lse_tol


def check(out, lse, ref, rows=None):
    want, want_lse, tol, lse_tol = ref
    pick = slice(None) if rows is None else rows
    got = out.double()[pick]
    assert bool(torch.isfinite(got).all()), "an unseen token reached the output"
    worst = ((got - want[pick]).abs() / tol[pick].clamp_min(1e-30)).max()
    assert float(worst) <= 1, f"{float(worst)} times the bound"
    if lse is not None:
        a, b = lse.double()[pick], want_lse[pick]
        assert torch.equal(torch.isinf(a), torch.isinf(b))
        live = ~torch.isinf(b)
        assert bool(((a - b).abs()[live] <= lse_tol[pick][live]).all())


def plan_decode(device, meta, heads, dtype, window, sinks, kind, ws=None):
    w = pagedattn.BatchDecodeWithPagedKVCacheWrapper(
        workspace(device) if ws is None else ws, "HND")
    w.plan(i32(meta.kv_indptr, device), i32(meta.kv_indices, device),
           i32(meta.kv_last_page_len, device), *heads, 16, q_data_type=dtype, window_left=window,
           num_sink_tokens=sinks, device_plan=kind == "device",
           split_pages={"split": 4, "whole": -1}.get(kind, 0))
    return w


LENS = [1, 16, 17, 40, 129, 130, 145, 300, 1000]


@pytest.mark.parametrize("kind", ["host", "split", "whole", "device"])
@pytest.mark.parametrize("window,sinks", [(127, 4), (0, 0), (16, 16), (30, 1), (200, 33),
                                          (5, 40), (100000, 3)])
@pytest.mark.parametrize("heads,dtype,fp8", [
    (HEADS[0], torch.float16, False), (HEADS[1], torch.bfloat16, False),
    (HEADS[1], torch.bfloat16, True), (HEADS[2], torch.float16, True),
    (HEADS[3], torch.bfloat16, False)])
def test_decode(gpu, heads, dtype, fp8, window, sinks, kind):
    meta, pool, scales, q = make(gpu, [n - 1 for n in LENS], [1] * len(LENS), heads, dtype, fp8,
                                 window, sinks, seed=window + sinks)
    w = plan_decode(gpu, meta, heads, dtype, window, sinks, kind)
    out, lse = w.run(q, pool, kv_scales=scales, return_lse=True)
    check(out, lse, reference(meta, pool, scales, q, window, sinks))


@pytest.mark.parametrize("kind", ["host", "device"])
def test_decode_many_sequences(gpu, kind):
    """Enough (sequence, KV head) items for the plans that share whole items."""
    require_shared_plans()
    heads, window, sinks = HEADS[0], 255, 20
    lens = [300 + 37 * (i % 29) for i in range(300)]
    meta, pool, scales, q = make(gpu, [n - 1 for n in lens], [1] * len(lens), heads,
                                 torch.bfloat16, False, window, sinks, seed=5)
    w = plan_decode(gpu, meta, heads, torch.bfloat16, window, sinks, kind)
    assert w.plan_kind == {"host": "shared", "device": "device_shared"}[kind]
    out, lse = w.run(q, pool, return_lse=True)
    rows = list(range(0, len(lens), 7))
    ref = reference(meta, pool, scales, q, window, sinks, b_rows=set(rows))
    check(out, lse, ref, rows)
    if kind == "device":
        require_fixed_chunks()
        w.update_plan()
        again, lse2 = w.run(q, pool, return_lse=True)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


def test_decode_long_window(gpu):
    """A long sequence on its own: its window is cut over the GPU and merged."""
    heads, window, sinks = HEADS[1], 9000, 64
    for kind in ("host", "device"):
        meta, pool, scales, q = make(gpu, [30000], [1], heads, torch.bfloat16, False, window,
                                     sinks, seed=9, spoil=False)
        w = plan_decode(gpu, meta, heads, torch.bfloat16, window, sinks, kind)
        out, lse = w.run(q, pool, return_lse=True)
        check(out, lse, reference(meta, pool, scales, q, window, sinks))


@pytest.mark.parametrize("kind", ["host", "whole", "device"])
@pytest.mark.parametrize("batch", [9, 300])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_fused_append_is_the_separate_calls(gpu, kind, batch, fp8):
    """RoPE + append + windowed attention in one call: the bits of the three."""
    require_fixed_chunks()
    heads, window, sinks, dtype = HEADS[0], 100, 20, torch.bfloat16
    hq, hkv, d = heads
    lens = [LENS[i % len(LENS)] + 16 * (i % 5) for i in range(batch)]
    meta, pool, scales, q = make(gpu, [n - 1 for n in lens], [1] * batch, heads, dtype, fp8,
                                 window, sinks, seed=3)
    g = torch.Generator(device=gpu)
    g.manual_seed(4)
    k, v = (torch.randn((batch, hkv, d), generator=g, device=gpu).to(dtype) for _ in range(2))
    lists = [i32(x, gpu) for x in (meta.kv_indices, meta.kv_indptr, meta.kv_last_page_len)]
    bi, pos = i32(np.arange(batch), gpu), i32(np.asarray(lens) - 1, gpu)
    for rope in (None, (2.0, 10000.0)):
        p1, p2 = pool.clone(), pool.clone()
        q1, k1 = q.clone(), k.clone()
        if rope:
            pagedattn.apply_rope_pos_ids_inplace(q1, k1, pos, rope_scale=rope[0],
                                                 rope_theta=rope[1])
        pagedattn.append_paged_kv_cache(k1, v, bi, pos, p1, *lists, kv_layout="HND",
                                        kv_scales=scales)
        w = plan_decode(gpu, meta, heads, dtype, window, sinks, kind)
        want = w.run(q1, p1, kv_scales=scales)
        got = w.run(q, p2, kv_scales=scales, append_key=k, append_value=v, rope=rope,
                    positions=pos if rope and kind == "host" else None)
        assert torch.equal(p1.view(torch.uint8), p2.view(torch.uint8))
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["host", "device"])
def test_window_past_the_length_is_no_window(gpu, kind):
    """The scores and their sums are those of the call without a window, bit for bit; the
    weights are held in two 16-bit terms instead of one, so the outputs differ by the one
    rounding that reference() allows for."""
    heads, dtype = HEADS[1], torch.bfloat16
    meta, pool, scales, q = make(gpu, [n - 1 for n in LENS], [1] * len(LENS), heads, dtype,
                                 False, 1 << 30, 0, seed=2)
    out, lse = plan_decode(gpu, meta, heads, dtype, 1 << 30, 0, kind).run(q, pool, return_lse=True)
    want, want_lse = plan_decode(gpu, meta, heads, dtype, -1, 0, kind).run(q, pool,
                                                                          return_lse=True)
    assert torch.equal(lse, want_lse)
    ref = reference(meta, pool, scales, q, 1 << 30, 0)
    check(out, lse, ref)
    check(want, want_lse, ref)


def plan_prefill(device, meta, heads, dtype, window, sinks, device_plan, causal=True):
    w = pagedattn.BatchPrefillWithPagedKVCacheWrapper(workspace(device), "HND")
    w.plan(i32(meta.qo_indptr, device), i32(meta.kv_indptr, device), i32(meta.kv_indices, device),
           i32(meta.kv_last_page_len, device), *heads, 16, causal=causal, q_data_type=dtype,
           window_left=window, num_sink_tokens=sinks, device_plan=device_plan,
           max_qo_tokens=meta.nnz)
    return w


CHUNKS = [([0, 5, 300, 0, 77], [1, 40, 70, 200, 0]), ([1500], [33]), ([0], [400])]


@pytest.mark.parametrize("computed,chunks", CHUNKS)
@pytest.mark.parametrize("window,sinks", [(127, 4), (0, 0), (16, 17), (63, 130), (100000, 3)])
@pytest.mark.parametrize("heads,dtype,fp8", [
    (HEADS[0], torch.float16, False), (HEADS[1], torch.bfloat16, False),
    (HEADS[1], torch.bfloat16, True), (HEADS[2], torch.float16, True),
    (HEADS[3], torch.bfloat16, False)])
def test_prefill(gpu, heads, dtype, fp8, window, sinks, computed, chunks):
    meta, pool, scales, q = make(gpu, computed, chunks, heads, dtype, fp8, window, sinks,
                                 seed=window + sinks)
    got = []
    for device_plan in (False, True):
        w = plan_prefill(gpu, meta, heads, dtype, window, sinks, device_plan)
        got.append(w.run(q, pool, kv_scales=scales, return_lse=True))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    rows = sorted({0, 1, meta.nnz - 1, *range(0, meta.nnz, 13)} & set(range(meta.nnz)))
    check(*got[0], reference(meta, pool, scales, q, window, sinks, b_rows=set(rows)), rows)


@pytest.mark.parametrize("heads,dtype,fp8", [(HEADS[1], torch.bfloat16, False),
                                             (HEADS[0], torch.float16, True)])
def test_prefill_cut_windows(gpu, heads, dtype, fp8, monkeypatch):
    """A long window of few rows runs in pieces and is merged; whole, it is the same within the
    bound."""
    window, sinks = 4000, 200
    meta, pool, scales, q = make(gpu, [9000], [64], heads, dtype, fp8, window, sinks, seed=1,
                                 spoil=False)
    rows = [0, 31, 63]
    ref = reference(meta, pool, scales, q, window, sinks, b_rows=set(rows))
    for env in ("1", "0"):
        monkeypatch.setenv("PAGEDATTN_PREFILL_SPLIT", env)
        for device_plan in (False, True):
            w = plan_prefill(gpu, meta, heads, dtype, window, sinks, device_plan)
            check(*w.run(q, pool, kv_scales=scales, return_lse=True), ref, rows)


def test_prefill_not_causal(gpu):
    heads, dtype, window, sinks = HEADS[1], torch.bfloat16, 20, 3
    meta, pool, scales, q = make(gpu, [100, 0], [50, 90], heads, dtype, False, window, sinks,
                                 seed=1)
    w = plan_prefill(gpu, meta, heads, dtype, window, sinks, False, causal=False)
    check(*w.run(q, pool, return_lse=True),
          reference(meta, pool, scales, q, window, sinks, causal=False))


def test_prefill_rows_that_see_nothing(gpu):
    """More query rows than tokens: the rows before the first token are zeros."""
    heads, dtype, window, sinks = HEADS[0], torch.float16, 9, 2
    meta, pool, scales, q = make(gpu, [0], [60], heads, dtype, False, window, sinks, seed=1,
                                 spoil=False)
    meta.kv_indptr[1:] = 2  # 2 pages, the last of 5 tokens
    meta.kv_last_page_len[0] = 5
    w = plan_prefill(gpu, meta, heads, dtype, window, sinks, False)
    out, lse = w.run(q, pool, return_lse=True)
    check(out, lse, reference(meta, pool, scales, q, window, sinks))
    assert not out[:60 - 21].any() and bool(torch.isneginf(lse[:60 - 21]).all())


@pytest.mark.parametrize("heads,fp8", [(HEADS[0], False), (HEADS[1], False), (HEADS[1], True)])
@pytest.mark.parametrize("long", [False, True])
def test_prefill_tokens_not_finite_reach_the_rows_that_see_them_only(gpu, heads, fp8, long):
    """An infinity and a NaN that some rows of a tile see: those rows are not finite as in the
    reference, all others are as if the tokens were not there."""
    dtype, window, sinks = torch.bfloat16, 30, 2
    prefix = 2000 if long else 40
    window = 1500 if long else window
    meta, pool, scales, q = make(gpu, [prefix], [150], heads, dtype, fp8, window, sinks, seed=8)
    table = meta.kv_indices[meta.kv_indptr[0]:]
    for t, x in ((prefix + 60, math.nan), (prefix - window + 20, math.nan if fp8 else math.inf)):
        pool[table[t // 16], 1, :, t % 16] = x
    seen = [r for r in range(150) if any(
        t <= prefix + r and t >= prefix + r - window for t in (prefix + 60, prefix - window + 20))]
    clear = sorted(set(range(150)) - set(seen))
    assert len(clear) > 20 and len(seen) > 20
    w = plan_prefill(gpu, meta, heads, dtype, window, sinks, False)
    out, lse = w.run(q, pool, kv_scales=scales, return_lse=True)
    check(out, lse, reference(meta, pool, scales, q, window, sinks, b_rows=set(clear)), clear)
    assert not bool(torch.isfinite(out[seen]).any())


def test_decode_step_replayed_from_a_graph(gpu):
    """Metadata, plan and fused windowed decode captured once; lengths, rows and tables change
    in place between replays, with eager work between them."""
    heads, window, sinks, dtype, batch = HEADS[0], 70, 17, torch.float16, 5
    hq, hkv, d = heads
    rng = np.random.default_rng(0)
    tables = rng.permutation(batch * 30).reshape(batch, 30)
    bt, lens = i32(tables, gpu), i32(np.ones(batch), gpu)
    g = torch.Generator(device=gpu)
    g.manual_seed(0)
    pool = torch.randn((batch * 30, 2, hkv, 16, d), generator=g, device=gpu).to(dtype)
    q = torch.zeros((batch, hq, d), dtype=dtype, device=gpu)
    k, v = (torch.zeros((batch, hkv, d), dtype=dtype, device=gpu) for _ in range(2))
    out = torch.zeros_like(q)
    for with_update in (False, True):
        buf = pagedattn.ops.new_paged_buffers(batch, batch * 30, batch, gpu)
        w = pagedattn.BatchDecodeWithPagedKVCacheWrapper(
            workspace(gpu), "HND", use_cuda_graph=True, paged_kv_indptr_buffer=buf.kv_indptr,
            paged_kv_indices_buffer=buf.kv_indices,
            paged_kv_last_page_len_buffer=buf.kv_last_page_len)
        w.plan(buf.kv_indptr, buf.kv_indices, buf.kv_last_page_len, hq, hkv, d, 16,
               q_data_type=dtype, window_left=window, num_sink_tokens=sinks)

        def step():
            pagedattn.build_paged_metadata(bt, lens, out=buf)
            if with_update:
                w.update_plan()
            w.run(q, pool, out=out, append_key=k, append_value=v, rope=(1.0, 10000.0),
                  positions=buf.positions)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for i, now in enumerate(([1, 17, 90, 300, 64], [2, 18, 91, 301, 65], [480, 3, 5, 86, 88])):
            lens.copy_(i32(now, gpu))
            for x in (q, k, v):
                x.normal_(generator=g)
            before = pool.clone()
            graph.replay()
            torch.cuda.synchronize()
            got, wrote = out.clone(), pool.clone()
            pool.copy_(before)
            meta = decode_metadata([t.tolist() for t in tables], now)
            we = plan_decode(gpu, meta, heads, dtype, window, sinks, "device")
            want = we.run(q, pool, append_key=k, append_value=v, rope=(1.0, 10000.0))
            assert torch.equal(got, want), i
            assert torch.equal(wrote, pool), i


def test_forward_takes_the_planned_window_only(gpu):
    heads, dtype = HEADS[1], torch.bfloat16
    meta, pool, _, q = make(gpu, [40, 9], [1, 1], heads, dtype, False, 20, 4, seed=1)
    w = plan_decode(gpu, meta, heads, dtype, 20, 4, "device")
    assert torch.equal(w.forward(q, pool, window_left=20), w.forward(q, pool))
    pw = plan_prefill(gpu, meta, heads, dtype, -1, 0, False)
    for x, left in ((w, 21), (w, 0), (pw, 20)):
        with pytest.raises(ValueError, match="window"):
            x.forward(q, pool, window_left=left)
    for left, sinks in ((-2, 0), (-1, 4), (None, 1), (5, -1), (1 << 31, 0)):
        for x in (w, pw):
            args = [i32(meta.kv_indptr, gpu), i32(meta.kv_indices, gpu),
                    i32(meta.kv_last_page_len, gpu), *heads, 16]
            if x is pw:
                args.insert(0, i32(meta.qo_indptr, gpu))
            with pytest.raises(ValueError):
                x.plan(*args, window_left=left, num_sink_tokens=sinks)


def test_an_empty_batch(gpu):
    w = pagedattn.BatchDecodeWithPagedKVCacheWrapper(workspace(gpu), "HND")
    for device_plan in (False, True):
        w.plan(i32([0], gpu), i32([], gpu), i32([], gpu), 8, 2, 64, 16, window_left=5,
               num_sink_tokens=2, device_plan=device_plan)
        out = w.run(torch.zeros((0, 8, 64), dtype=torch.float16, device=gpu),
                    torch.zeros((3, 2, 2, 16, 64), dtype=torch.float16, device=gpu))
        assert out.shape == (0, 8, 64)


def test_patched_llama_with_a_window(gpu):
    """The engine's shim, fused and not, against the model under the window's mask in 32 bits on
    the CPU; pages behind the window are gone by the decode step."""
    from transformers import LlamaConfig, LlamaForCausalLM

    from pagedattn.metadata import decode_metadata, prefill_metadata

    cfg = LlamaConfig(hidden_size=512, intermediate_size=1024, num_attention_heads=8,
                      num_key_value_heads=2, num_hidden_layers=2, vocab_size=512,
                      max_position_embeddings=4096, attn_implementation="eager")
    torch.manual_seed(0)
    ref = LlamaForCausalLM(cfg).eval()
    model = copy.deepcopy(ref).to(device=gpu, dtype=torch.bfloat16)
    L.patch_llama_model(model)
    window, sinks, lens = 24, 5, [37, 100, 5, 64]
    rng = np.random.default_rng(0)
    tokens = torch.as_tensor(rng.integers(0, 512, (len(lens), 128)))
    tables, num_pages = random_tables(rng, [n + 1 for n in lens], extra_pages=4)
    got = []
    try:
        for L.FUSE in (True, False):
            pool = torch.zeros((2, num_pages, 2, 2, 16, 64), dtype=torch.bfloat16, device=gpu)
            L.init_flashinfer_state(kv_pool=pool, page_size=16, device=gpu, window_left=window,
                                    num_sink_tokens=sinks)
            meta = prefill_metadata(tables, [0] * len(lens), lens)
            L.build_batch_indices_positions(i32(meta.qo_indptr, gpu), i32(meta.seq_lens, gpu))
            shape = dict(num_qo_heads=8, num_kv_heads=2, head_dim=64)
            L.plan_prefill(qo_indptr=i32(meta.qo_indptr, gpu), kv_indptr=i32(meta.kv_indptr, gpu),
                           kv_indices=i32(meta.kv_indices, gpu),
                           kv_last_page_len=i32(meta.kv_last_page_len, gpu), **shape)
            packed = torch.cat([tokens[b, :n] for b, n in enumerate(lens)])[None].to(gpu)
            with torch.no_grad():
                pre = model(input_ids=packed, use_cache=False).logits[0]
            kept = [[p if s < 1 or s >= (n - window) // 16 else -1 for s, p in enumerate(t)]
                    for t, n in zip(tables, lens)]
            meta = decode_metadata(kept, [n + 1 for n in lens])
            L.FlashInferState.batch_indices = i32(meta.batch_indices, gpu)
            L.FlashInferState.positions = i32(meta.positions, gpu)
            L.plan_decode(kv_indptr=i32(meta.kv_indptr, gpu),
                          kv_indices=i32(meta.kv_indices, gpu),
                          kv_last_page_len=i32(meta.kv_last_page_len, gpu), **shape)
            step = torch.stack([tokens[b, n] for b, n in enumerate(lens)])[:, None].to(gpu)
            with torch.no_grad():
                dec = model(input_ids=step, use_cache=False).logits[:, 0]
            assert L.append_error_count() == 0
            got.append((pre.float().cpu(), dec.float().cpu()))
    finally:
        L.FUSE = True
        L.init_flashinfer_state(kv_pool=pool, page_size=16, device=gpu)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    ends = np.cumsum(lens)
    for b, n in enumerate(lens):
        i, j = torch.arange(n + 1)[:, None], torch.arange(n + 1)
        seen = (j <= i) & ((j >= i - window) | (j < sinks))
        mask = torch.where(seen, 0.0, torch.finfo(torch.float32).min)[None, None]
        with torch.no_grad():
            full = ref(input_ids=tokens[b:b + 1, :n + 1], attention_mask=mask,
                       use_cache=False).logits[0]
        # the bound that the shim's tests without a window have for bf16
        for mine, want in ((got[0][0][ends[b] - n:ends[b]], full[:n]), (got[0][1][b], full[n])):
            assert float((mine - want).norm() / want.norm()) < 3e-2, b


def test_replanning_between_replays_leaves_the_captured_step_its_lists(gpu):
    """A device plan is captured; the wrapper is planned and run for other batches; the replays
    still give the first batch's results."""
    heads, dtype, window, sinks = HEADS[0], torch.float16, 60, 17
    meta, pool, _, q = make(gpu, [200, 90, 300], [1] * 3, heads, dtype, False, window, sinks, 1)
    w = plan_decode(gpu, meta, heads, dtype, window, sinks, "device")
    want = w.run(q, pool)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(q, pool, out=out)
    lists = (w._indptr, w._indices, w._last)  # the caller's metadata, still alive
    for n, left in ((3, 60), (9, 60), (2, 500), (300, 10)):
        lens = [100 + 3 * i for i in range(n)]
        m2, p2, _, q2 = make(gpu, lens, [1] * n, heads, dtype, False, left, sinks, 2)
        w.plan(*(i32(x, gpu) for x in (m2.kv_indptr, m2.kv_indices, m2.kv_last_page_len)), *heads,
               16, q_data_type=dtype, window_left=left, num_sink_tokens=sinks,
               device_plan=n != 9)
        got = w.run(q2, p2)
        rows = [0, n - 1]
        check(got, None, reference(m2, p2, None, q2, left, sinks, b_rows=set(rows)), rows)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
    del lists


@pytest.mark.parametrize("fp8", [False, True])
def test_prefill_of_nan_scores_is_nan(gpu, fp8):
    """A NaN in a K row: every row that sees it is NaN, the others are as if it were not there."""
    heads, dtype, window, sinks = HEADS[1], torch.bfloat16, 25, 0
    meta, pool, scales, q = make(gpu, [0], [100], heads, dtype, fp8, window, sinks, seed=8)
    page = int(meta.kv_indices[2])
    pool[page, 0, :, 5] = math.nan  # token 37
    w = plan_prefill(gpu, meta, heads, dtype, window, sinks, False)
    out, lse = w.run(q, pool, kv_scales=scales, return_lse=True)
    seen = list(range(37, 37 + window + 1))
    clear = sorted(set(range(100)) - set(seen))
    check(out, lse, reference(meta, pool, scales, q, window, sinks, b_rows=set(clear)), clear)
    assert bool(torch.isnan(out[seen]).all())


def test_a_window_of_the_largest_size(gpu):
    """Rows before the first token (more rows than tokens) and windows up to 2^31 - 1."""
    heads, dtype, window, sinks = HEADS[0], torch.float16, (1 << 31) - 1, (1 << 31) - 1
    meta, pool, scales, q = make(gpu, [0], [60], heads, dtype, False, window, 0, seed=1,
                                 spoil=False)
    meta.kv_indptr[1:] = 2
    meta.kv_last_page_len[0] = 5
    for s in (0, sinks):
        for device_plan in (False, True):
            w = plan_prefill(gpu, meta, heads, dtype, window, s, device_plan)
            check(*w.run(q, pool, return_lse=True),
                  reference(meta, pool, scales, q, window, s))
    one, pool, scales, q = make(gpu, [40, 0], [1, 1], heads, dtype, False, window, 0, seed=1)
    for kind in ("host", "device"):
        w = plan_decode(gpu, one, heads, dtype, window, sinks, kind)
        check(*w.run(q, pool, return_lse=True), reference(one, pool, scales, q, window, sinks))


@pytest.mark.parametrize("kind", ["host", "device"])
def test_decode_by_the_general_path(gpu, kind, request):
    """The same bits as the extension's call, with RoPE and append and without."""
    require_fixed_chunks()
    heads, dtype, window, sinks = HEADS[0], torch.float16, 60, 17
    meta, pool, _, q = make(gpu, [n - 1 for n in LENS], [1] * len(LENS), heads, dtype, False,
                            window, sinks, 1)
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    k, v = (torch.randn((len(LENS), 4, 64), generator=g, device=gpu).to(dtype) for _ in range(2))
    got = []
    for native in (True, False):
        if not native:
            request.getfixturevalue("general")
        p = pool.clone()
        w = plan_decode(gpu, meta, heads, dtype, window, sinks, kind)
        out, lse = w.run(q, p, return_lse=True)
        fused = w.run(q, p, append_key=k, append_value=v, rope=(1.0, 1e4))
        got.append((out, lse, fused, p.view(torch.int16)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_prefill_of_scales_not_finite(gpu):
    """The scale of a page that some rows of a tile see is an infinity, of another NaN: the rows
    that see neither are as if the pages were not there."""
    heads, dtype, window, sinks = HEADS[1], torch.bfloat16, 25, 0
    meta, pool, scales, q = make(gpu, [0], [150], heads, dtype, True, window, sinks, seed=9)
    table = meta.kv_indices
    scales[int(table[3])] = math.inf  # tokens 48 to 63
    scales[int(table[6])] = math.nan  # tokens 96 to 111
    clear = [r for r in range(150) if not (48 <= r <= 63 + window or 96 <= r <= 111 + window)]
    assert len(clear) > 20
    w = plan_prefill(gpu, meta, heads, dtype, window, sinks, False)
    out, lse = w.run(q, pool, kv_scales=scales, return_lse=True)
    check(out, lse, reference(meta, pool, scales, q, window, sinks, b_rows=set(clear)), clear)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
@pytest.mark.parametrize("kind", ["host", "device"])
@pytest.mark.parametrize("way", ["extension", "general"])
def test_decode_on_a_device_that_is_not_current(gpu, kind, way, request):
    if way == "general":
        request.getfixturevalue("general")
    heads, dtype, window, sinks = HEADS[0], torch.float16, 50, 4
    other = torch.device("cuda", 1)
    meta, pool, scales, q = make(other, [99, 300], [1, 1], heads, dtype, False, window, sinks,
                                 seed=3)
    assert torch.cuda.current_device() == 0
    w = plan_decode(other, meta, heads, dtype, window, sinks, kind)
    check(*w.run(q, pool, return_lse=True), reference(meta, pool, scales, q, window, sinks))


@pytest.mark.parametrize("heads,dtype,fp8", [
    (HEADS[0], torch.float16, False), (HEADS[0], torch.bfloat16, True),
    (HEADS[1], torch.bfloat16, False), (HEADS[1], torch.float16, True)])
def test_prefill_of_more_than_two_rounds(gpu, heads, dtype, fp8):
    """More q-tiles than twice those that run at once, whose list does not run in the order of
    their lengths: every row is written, and as the other plan writes it."""
    window, sinks = 127, 4
    rng = np.random.default_rng(4)
    tokens = 256 * heads[1] // heads[0]  # of a q-tile
    tiles = 2 * (256 // heads[1]) + 9
    chunks = [int(x) for x in rng.integers(1, tokens + 1, tiles)]
    chunks[3] += 2 * tokens
    computed = [int(x) for x in rng.integers(0, 300, tiles)]
    meta, pool, scales, q = make(gpu, computed, chunks, heads, dtype, fp8, window, sinks, seed=3)
    got = []
    for device in (False, True):
        out = torch.full_like(q.contiguous(), math.nan)
        w = plan_prefill(gpu, meta, heads, dtype, window, sinks, device)
        got.append(w.run(q, pool, kv_scales=scales, return_lse=True, out=out))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert bool(torch.isfinite(got[0][0]).all())
    rows = sorted(set(rng.integers(0, meta.nnz, 60).tolist()) | {0, meta.nnz - 1})
    check(*got[0], reference(meta, pool, scales, q, window, sinks, b_rows=set(rows)), rows)
