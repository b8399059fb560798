"""The page calls, multi-axis RoPE and windowed attention together, as a serving step uses
them: prompts are admitted, shared with second samples, decoded by a captured step that takes,
forks and releases its pages itself, and the pool is compacted between replays.  Every output
is checked against attention in 64 bits over the sequences' whole history."""

import math

import numpy as np
import pytest
import torch

import pagedattn

from paged_cases import i32, workspace

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, ROWS, WIDTH, PAGES = 2, 8, 2, 64, 6, 30, 70
WINDOW, SINKS, SECTIONS = 37, 5, (12, 10, 10)


class Sequences:
    """What every row has seen: its rotated K and its V rows, layer by layer, in 64 bits."""

    def __init__(self, device):
        empty = torch.zeros((0, HKV, D), dtype=torch.float64, device=device)
        self.kv = [[[empty, empty] for _ in range(ROWS)] for _ in range(LAYERS)]

    def add(self, layer, row, k, v):
        old = self.kv[layer][row]
        self.kv[layer][row] = [torch.cat([old[0], k.double()]), torch.cat([old[1], v.double()])]

    def share(self, src, dst):
        for layer in self.kv:
            layer[dst] = list(layer[src])

    def check(self, layer, row, q, out):
        """out [n, HQ, D] of the row's newest n tokens; one rounding of the weights and one of
        the output, as in the windowed attention's own tests."""
        k, v = (x.repeat_interleave(HQ // HKV, 1).transpose(0, 1) for x in self.kv[layer][row])
        n, length = q.shape[0], k.shape[1]
        u = torch.finfo(q.dtype).eps / 2
        at = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)
        hidden = (j > at) | ((j < at - WINDOW) & (j >= SINKS))
        s = torch.matmul(q.double().transpose(0, 1), k.transpose(1, 2)) / math.sqrt(D)
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        want = torch.matmul(p, v).transpose(0, 1)
        spread = torch.matmul(p, v.abs()).transpose(0, 1)
        size = torch.matmul(q.double().abs().transpose(0, 1), k.abs().transpose(1, 2)).amax()
        off = float(size) / math.sqrt(D) * (D + 8) * 2.0 ** -24 + float(s.abs().max()) * 2.0 ** -21
        tol = u * want.abs() + spread * (1.01 * u + math.expm1(2 * off)) + 2.0 ** -24
        assert bool(((out.double() - want).abs() <= tol).all()), (layer, row)


def axes_of(rng, places):
    """Axis positions of tokens at `places`, as of text and images in turn."""
    t = places - places % 7
    return np.stack([t, t + places % 3, t + places % 5])


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_life_of_a_batch(gpu, dtype):
    rng = np.random.default_rng(0)
    g = torch.Generator(device=gpu)
    g.manual_seed(0)
    pool = torch.full((LAYERS, PAGES, 2, HKV, 16, D), math.nan, dtype=dtype, device=gpu)
    tables = torch.full((ROWS, WIDTH), -1, dtype=torch.int32, device=gpu)
    refs = torch.zeros(PAGES, dtype=torch.int32, device=gpu)
    errors = torch.zeros(2, dtype=torch.int32, device=gpu)
    seqs = Sequences(gpu)

    def consistent():
        t = tables.cpu().numpy()
        assert errors.tolist() == [0, 0]
        assert np.array_equal(refs.cpu().numpy(), np.bincount(t[t >= 0], minlength=PAGES))

    # three prompts; the other rows stay empty
    lens = np.array([50, 17, 5, 0, 0, 0])
    kv_lens, new = i32(lens, gpu), i32(lens, gpu)
    pagedattn.reserve_pages(pool, tables, kv_lens, new, refs, error_flag=errors)
    consistent()
    buf = pagedattn.build_paged_metadata(tables, kv_lens, new, error_flag=errors)
    pw = pagedattn.BatchPrefillWithPagedKVCacheWrapper(workspace(gpu), "HND")
    nnz = int(lens.sum())
    pw.plan(buf.qo_indptr, buf.kv_indptr, buf.kv_indices, buf.kv_last_page_len, HQ, HKV, D, 16,
            causal=True, q_data_type=dtype, window_left=WINDOW, num_sink_tokens=SINKS,
            device_plan=True, max_qo_tokens=nnz)
    places = np.concatenate([np.arange(n) for n in lens])
    axes = i32(axes_of(rng, places), gpu)
    for layer in range(LAYERS):
        rows = torch.randn((nnz, HQ + 2 * HKV, D), generator=g, device=gpu).to(dtype)
        q, k, v = rows[:, :HQ], rows[:, HQ:HQ + HKV], rows[:, HQ + HKV:]
        pagedattn.multi_axis_rope_append_paged_kv_cache(
            q, k, v, axes, SECTIONS, buf.batch_indices, buf.positions, pool[layer],
            buf.kv_indices, buf.kv_indptr, buf.kv_last_page_len, kv_layout="HND", cyclic=True)
        out = pw.run(q, pool[layer])
        at = 0
        for row, n in enumerate(lens):
            seqs.add(layer, row, k[at:at + n], v[at:at + n])
            if n:
                seqs.check(layer, row, q[at:at + n], out[at:at + n])
            at += n
    pagedattn.release_window_pages(tables, kv_lens, refs, WINDOW, SINKS, error_flag=errors)
    consistent()

    # a second sample of every prompt
    pagedattn.share_pages(tables, kv_lens, [0, 1, 2], [3, 4, 5], refs, error_flag=errors)
    for row in range(3):
        seqs.share(row, row + 3)
    lens[3:] = lens[:3]
    assert kv_lens.tolist() == lens.tolist()
    consistent()

    # the captured step
    steps = pagedattn.ops.new_paged_buffers(ROWS, ROWS * WIDTH, ROWS, gpu)
    w = pagedattn.BatchDecodeWithPagedKVCacheWrapper(
        workspace(gpu), "HND", use_cuda_graph=True, paged_kv_indptr_buffer=steps.kv_indptr,
        paged_kv_indices_buffer=steps.kv_indices,
        paged_kv_last_page_len_buffer=steps.kv_last_page_len)
    w.plan(steps.kv_indptr, steps.kv_indices, steps.kv_last_page_len, HQ, HKV, D, 16,
           q_data_type=dtype, window_left=WINDOW, num_sink_tokens=SINKS)
    rows = [torch.zeros((ROWS, HQ + 2 * HKV, D), dtype=dtype, device=gpu) for _ in range(LAYERS)]
    outs = [torch.zeros((ROWS, HQ, D), dtype=dtype, device=gpu) for _ in range(LAYERS)]
    axes = torch.zeros((3, ROWS), dtype=torch.int32, device=gpu)

    def step():
        kv_lens.add_(1)
        pagedattn.reserve_pages(pool, tables, kv_lens, None, refs, error_flag=errors)
        pagedattn.build_paged_metadata(tables, kv_lens, out=steps, error_flag=errors)
        w.update_plan()
        for layer in range(LAYERS):
            q, k, v = (rows[layer][:, a:b] for a, b in ((0, HQ), (HQ, HQ + HKV),
                                                       (HQ + HKV, HQ + 2 * HKV)))
            pagedattn.multi_axis_rope_append_paged_kv_cache(
                q, k, v, axes, SECTIONS, steps.batch_indices, steps.positions, pool[layer],
                steps.kv_indices, steps.kv_indptr, steps.kv_last_page_len, kv_layout="HND",
                cyclic=True)
            w.run(q, pool[layer], out=outs[layer])
        pagedattn.release_window_pages(tables, kv_lens, refs, WINDOW, SINKS, error_flag=errors)

    def prepare():
        axes.copy_(i32(axes_of(rng, lens), gpu))
        for x in rows:
            x.normal_(generator=g)

    def verify():
        torch.cuda.synchronize()
        consistent()
        for layer in range(LAYERS):
            x = rows[layer]
            for row in range(ROWS):
                seqs.add(layer, row, x[row:row + 1, HQ:HQ + HKV], x[row:row + 1, HQ + HKV:])
                seqs.check(layer, row, x[row:row + 1, :HQ], outs[layer][row:row + 1])

    prepare()
    step()  # eager: the three shared partial pages fork
    lens += 1
    verify()
    saved = [x.clone() for x in (kv_lens, tables, refs, errors)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for x, y in zip((kv_lens, tables, refs, errors), saved):  # capture ran nothing
        assert torch.equal(x, y)
    for i in range(60):
        prepare()
        graph.replay()
        lens += 1
        verify()
        if i % 17 == 5:
            before = int((refs > 0).sum())
            remap = pagedattn.compact_pages(pool, tables, refs, error_flag=errors)
            consistent()
            assert bool((refs[:before] > 0).all()) and not refs[before:].any()
            assert int((remap >= 0).sum()) == before
    # sinks, the window and the page being written: the rest has been freed
    assert int((refs > 0).sum()) <= ROWS * 5
    pagedattn.release_pages(tables, refs, error_flag=errors)
    consistent()
    assert not refs.any()
