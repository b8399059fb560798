"""RoPE with several axes, alone and with the page append, against the formula in
64 bits.  A turned element is x0 cos - x1 sin of 16-bit inputs in 32 bits, rounded
once: off by half a step of itself plus what the 32-bit cosine, sine and
products carry, under 2^-21 of |x0| + |x1|."""

import numpy as np
import pytest
import torch

import pagedattn

from paged_cases import i32, strided_rows

pytestmark = pytest.mark.gpu


def axis_list(sections, cyclic):
    if not cyclic:
        return np.repeat(np.arange(len(sections)), sections)
    names = np.zeros(sum(sections), int)
    for a in range(1, len(sections)):
        names[a:len(sections) * sections[a]:len(sections)] = a
    return names


def reference(x, pos, sections, cyclic, rotary, interleave, scale, theta):
    """(turned rows, bound) in 64 bits."""
    x64 = x.double()
    freq = theta ** (-2.0 * torch.arange(rotary // 2, dtype=torch.float64) / rotary)
    ang = pos[axis_list(sections, cyclic)].T.double().cpu() * freq / scale
    cos, sin = (f(ang).to(x.device)[:, None] for f in (torch.cos, torch.sin))
    at = torch.arange(rotary // 2)
    i0, i1 = (2 * at, 2 * at + 1) if interleave else (at, at + rotary // 2)
    a, b = x64[..., i0], x64[..., i1]
    out, tol = x64.clone(), torch.zeros_like(x64)
    u = torch.finfo(x.dtype).eps / 2
    for i, y in ((i0, a * cos - b * sin), (i1, b * cos + a * sin)):
        out[..., i] = y
        tol[..., i] = (a.abs() + b.abs()) * 2.0 ** -21 + y.abs() * u * (1 + 2.0 ** -8)
        tol[..., i] += 2.0 ** -25 if x.dtype == torch.float16 else 0
    return out, tol


def positions_of(rng, axes, n, hi=70000):
    return rng.integers(0, hi, (axes, n))


CASES = [(64, None, (12, 10, 10), True), (64, None, (8, 12, 12), False),
         (128, None, (16, 24, 24), False), (128, 64, (20, 6, 6), False),
         (128, 32, (6, 5, 5), True), (128, None, (64,), False), (256, None, (40, 44, 44), False),
         (96, 48, (0, 24), False), (16, None, (2, 2, 2, 2), True), (80, 80, (14, 13, 13), True)]


@pytest.mark.parametrize("d,rotary,sections,cyclic", CASES)
@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hkv", [(1, 1, 1), (37, 6, 2), (130, 32, 8), (5, 3, 0)])
def test_inplace(gpu, d, rotary, sections, cyclic, interleave, dtype, n, hq, hkv):
    rng = np.random.default_rng(n)
    g = torch.Generator(device=gpu)
    g.manual_seed(n)
    pos = i32(positions_of(rng, len(sections), n), gpu)
    q = strided_rows(n, hq, d, dtype, gpu, g, lead=1, tail=2)
    k = strided_rows(n, max(hkv, 1), d, dtype, gpu, g)[:, :hkv]
    wants = [reference(x, pos, sections, cyclic, rotary or d, interleave, 2.0, 5e5)
             for x in (q, k)]
    pagedattn.apply_multi_axis_rope_inplace(q, k, pos, sections, cyclic=cyclic, rotary_dim=rotary,
                                            interleave=interleave, rope_scale=2.0, rope_theta=5e5)
    for x, (want, tol) in zip((q, k), wants):
        assert bool(((x.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("rotary,interleave", [(None, False), (64, False), (None, True), (32, True)])
def test_equal_positions_are_the_one_position_call(gpu, rotary, interleave):
    rng = np.random.default_rng(0)
    g = torch.Generator(device=gpu)
    g.manual_seed(0)
    q, k = (torch.randn((50, h, 128), generator=g, device=gpu).bfloat16() for h in (8, 2))
    pos = i32(rng.integers(0, 130000, 50), gpu)
    q2, k2 = q.clone(), k.clone()
    pagedattn.apply_rope_pos_ids_inplace(q, k, pos, rotary_dim=rotary, interleave=interleave)
    f = (rotary or 128) // 2
    # int64 positions whose rows are one row: any strides and types
    pagedattn.apply_multi_axis_rope_inplace(q2, k2, pos.long().expand(3, 50), (f - 2, 1, 1),
                                            rotary_dim=rotary, interleave=interleave)
    assert torch.equal(q, q2) and torch.equal(k, k2)


@pytest.mark.parametrize("d,rotary,sections,cyclic", [CASES[0], CASES[2], CASES[3], CASES[6]])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("chunks", [[1] * 9, [40, 1, 130, 17]])
@pytest.mark.parametrize("native", [True, False])
def test_append_is_the_two_calls(gpu, d, rotary, sections, cyclic, fp8, interleave, chunks,
                                 native, monkeypatch):
    """By the extension's call and by the general path."""
    if native:
        real = pagedattn.ops._native

        def taken(fn, *args):
            r = real(fn, *args)
            assert r is not NotImplemented, fn
            return r

        monkeypatch.setattr(pagedattn.ops, "_native", taken)
    else:
        monkeypatch.setattr(pagedattn.ops, "_native", lambda *a: NotImplemented)
    dtype, hq, hkv, n = torch.bfloat16, 8, 2, sum(chunks)
    rng = np.random.default_rng(n)
    g = torch.Generator(device=gpu)
    g.manual_seed(n)
    computed = [3, 0, 20, 16, 5, 0, 31, 2, 9][:len(chunks)]
    need = [-(-(c + x) // 16) for c, x in zip(computed, chunks)]
    num_pages = sum(need) + 2
    meta = [i32(x, gpu) for x in (
        np.repeat(np.arange(len(chunks)), chunks),
        np.concatenate([np.arange(c, c + x) for c, x in zip(computed, chunks)]),
        rng.permutation(num_pages)[:sum(need)], np.concatenate([[0], np.cumsum(need)]),
        [(c + x - 1) % 16 + 1 for c, x in zip(computed, chunks)])]
    bi, at, ind, indptr, last = meta
    at[0] = 100000  # outside its sequence's pages: skipped and counted
    pool = torch.zeros((num_pages, 2, hkv, 16, d), device=gpu)
    pool = pool.to(torch.float8_e4m3fn) if fp8 else pool.to(dtype)
    scales = torch.rand((num_pages, 2, hkv), generator=g, device=gpu) / 8 if fp8 else None
    pos = i32(positions_of(rng, len(sections), n), gpu)
    rows = strided_rows(n, hq + 2 * hkv, d, dtype, gpu, g)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
    q2, k2, v2, pool2 = q.clone(), k.clone(), v.clone(), pool.clone()
    err, err2 = (torch.zeros(2, dtype=torch.int32, device=gpu) for _ in range(2))
    turn = dict(cyclic=cyclic, rotary_dim=rotary, interleave=interleave, rope_theta=1e6)
    pagedattn.multi_axis_rope_append_paged_kv_cache(
        q, k, v, pos, sections, bi, at, pool, ind, indptr, last, kv_layout="HND",
        kv_scales=scales, error_flag=err, **turn)
    pagedattn.apply_multi_axis_rope_inplace(q2, k2, pos, sections, **turn)
    pagedattn.append_paged_kv_cache(k2, v2, bi, at, pool2, ind, indptr, last, kv_layout="HND",
                                    kv_scales=scales, error_flag=err2)
    assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(v, v2)
    assert torch.equal(pool.view(torch.uint8), pool2.view(torch.uint8))
    assert err.tolist() == err2.tolist() and err[0] == 1


def test_few_heads_and_many_tokens(gpu):
    """Tokens past 16 a workgroup, and a step whose last workgroup is not full."""
    n, d, sections = 40001, 64, (12, 10, 10)
    rng = np.random.default_rng(0)
    pos = i32(positions_of(rng, 3, n), gpu)
    q = torch.randn((n, 2, d), device=gpu).half()
    k = torch.randn((n, 1, d), device=gpu).half()
    wants = [reference(x, pos, sections, True, d, False, 1.0, 1e4) for x in (q, k)]
    pagedattn.apply_multi_axis_rope_inplace(q, k, pos, sections, cyclic=True)
    for x, (want, tol) in zip((q, k), wants):
        assert bool(((x.double() - want).abs() <= tol).all())


def test_no_tokens(gpu):
    q, k = (torch.zeros((0, h, 64), device=gpu).half() for h in (4, 2))
    pagedattn.apply_multi_axis_rope_inplace(q, k, i32(np.zeros((3, 0)), gpu), (12, 10, 10))
