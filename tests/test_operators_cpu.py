"""Refusals of the windowed, paging and multi-axis calls, on the host: nothing here reaches a
device (the C entry points fail before they touch their pointers)."""

import ctypes

import numpy as np
import pytest
import torch

import pagedattn
from pagedattn import _lib, ops

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
A = 4096  # an aligned address that is never followed


def status(name, *args):
    lib = _lib.lib()
    rc = getattr(lib, name)(*args)
    return rc, lib.pagedattn_last_error().decode()


def refused(name, args, code, needle):
    rc, message = status(name, *args)
    assert rc == code and needle in message, (rc, message)


@pytest.mark.parametrize("left,sinks", [(-1, 0), (None, 0), (0, 0), (7, 3), ((1 << 31) - 1, 5)])
def test_windows_that_are_taken(left, sinks):
    assert ops._window(left, sinks) == (-1 if left is None else left, sinks)


@pytest.mark.parametrize("left,sinks,error", [
    (-2, 0, ValueError), (-1, 1, ValueError), (None, 4, ValueError), (4, -1, ValueError),
    (1 << 31, 0, ValueError), (4, 1 << 31, ValueError), (1.5, 0, TypeError), (4, "2", TypeError)])
def test_windows_that_are_not(left, sinks, error):
    with pytest.raises(error):
        ops._window(left, sinks)


@pytest.mark.parametrize("left,sinks", [(-2, 0), (-1, 3), (5, -1)])
def test_plans_refuse_bad_windows(left, sinks):
    lib = _lib.lib()
    plan = lib.pagedattn_plan_create()
    ptr = np.array([0, 2], np.int32).ctypes.data
    last = np.array([3], np.int32).ctypes.data
    for name, args in (
            ("pagedattn_decode_plan_window", (plan, ptr, last, 1, 8, 2, 64, 16, 0, left, sinks, A,
                                              1 << 20, None)),
            ("pagedattn_prefill_plan_window", (plan, ptr, ptr, last, 1, 8, 2, 64, 16, left, sinks,
                                               A, 1 << 20, None)),
            ("pagedattn_prefill_plan_device_window", (plan, 1, 8, 2, 64, 16, 10, left, sinks, A,
                                                      1 << 20))):
        refused(name, args, INVALID, "window")
    lib.pagedattn_plan_destroy(plan)


@pytest.mark.parametrize("indptr,last,kw,code,needle", [
    ([0, 3, 2], [5, 5], {}, INVALID, "monotone"),
    ([0, 2], [17], {}, INVALID, "kv_last_page_len"),
    ([0, 2], [5], {"page": 32}, UNSUPPORTED, "page_size"),
    ([0, 2], [5], {"d": 96}, UNSUPPORTED, "head_dim"),
    ([0, 2], [5], {"bsz": -1}, INVALID, "batch_size"),
    ([0, 9], [5], {"ws": 64}, WORKSPACE, "workspace")])
def test_windowed_decode_plan_checks_its_metadata(indptr, last, kw, code, needle):
    lib = _lib.lib()
    plan = lib.pagedattn_plan_create()
    indptr, last = np.asarray(indptr, np.int32), np.asarray(last, np.int32)
    refused("pagedattn_decode_plan_window",
            (plan, indptr.ctypes.data, last.ctypes.data, kw.get("bsz", len(last)), 8, 2,
             kw.get("d", 64), kw.get("page", 16), 4, 20, 4, A, kw.get("ws", 1 << 20), None), code,
            needle)
    lib.pagedattn_plan_destroy(plan)
    refused("pagedattn_decode_plan_window", (None, indptr.ctypes.data, last.ctypes.data, 1, 8, 2,
                                             64, 16, 0, 20, 4, A, 1 << 20, None), INVALID, "plan")


def test_window_metadata_refuses():
    def args(**kw):
        d = dict(indptr=A, indices=A, n=4, last=A, b=1, left=3, sinks=0, oi=A, ox=A, cap=4,
                 holes=A)
        d.update(kw)
        return (*d.values(), None)

    for kw in ({"b": -1}, {"n": -1}, {"cap": -1}, {"left": -1}, {"sinks": -1}):
        refused("pagedattn_decode_window_metadata", args(**kw), INVALID, "bad sizes")
    for kw in ({"indptr": None}, {"indices": None}, {"last": None}, {"oi": None}, {"ox": None},
               {"holes": None}):
        refused("pagedattn_decode_window_metadata", args(**kw), INVALID, "null")
    assert status("pagedattn_decode_window_metadata", *args(b=0, indptr=None, holes=None))[0] == 0


def pool_args(**kw):
    d = dict(pool=A, dtype=_lib.BF16, layers=2, pages=10, hkv=2, d=64, page=16, scales=None)
    d.update(kw)
    return list(d.values())


BAD_POOLS = [({"page": 8}, UNSUPPORTED, "page_size"), ({"dtype": _lib.F32}, UNSUPPORTED, "dtype"),
             ({"layers": 0}, INVALID, "shape"), ({"hkv": 0}, INVALID, "shape"),
             ({"d": 4}, INVALID, "16 bytes"), ({"d": 8, "dtype": _lib.E4M3}, INVALID, "16 bytes"),
             ({"dtype": _lib.E4M3}, INVALID, "kv_scales"), ({"pool": None}, INVALID, "pool"),
             ({"pool": A + 8}, INVALID, "pool"), ({"pages": -1}, INVALID, "shape"),
             ({"hkv": 1 << 30, "d": 1 << 30}, INVALID, "shape")]
BAD_TABLES = [({"tables": None}, INVALID, "null block_tables"), ({"refs": None}, INVALID, "ref"),
              ({"stride": 3}, INVALID, "bad sizes"), ({"b": -1}, INVALID, "bad sizes"),
              ({"width": -1}, INVALID, "bad sizes"), ({"b": 65536}, UNSUPPORTED, "65535"),
              ({"b": 65535, "width": 1 << 15, "stride": 1 << 15}, UNSUPPORTED, "entries")]
BAD_SCRATCH = [({"scratch": None}, INVALID, "scratch"), ({"scratch": A + 64}, INVALID, "scratch"),
               ({"size": 100}, WORKSPACE, "scratch")]


def split(kw):
    pool = {k: v for k, v in kw.items() if k in ("pool", "dtype", "layers", "pages", "hkv", "d",
                                                 "page", "scales")}
    return pool_args(**pool), {k: v for k, v in kw.items() if k not in pool}


@pytest.mark.parametrize("kw,code,needle", BAD_POOLS + BAD_TABLES + BAD_SCRATCH
                         + [({"lens": None}, INVALID, "kv_lens")])
def test_reserve_refuses(kw, code, needle):
    pool, rest = split(kw)
    d = dict(tables=A, stride=4, width=4, lens=A, new=None, b=3, refs=A, err=None, scratch=A,
             size=1 << 20)
    d.update(rest)
    refused("pagedattn_reserve_pages", (*pool, *d.values(), None), code, needle)


@pytest.mark.parametrize("kw,code,needle", BAD_POOLS + BAD_TABLES + BAD_SCRATCH
                         + [({"remap": None}, INVALID, "remap")])
def test_compact_refuses(kw, code, needle):
    pool, rest = split(kw)
    d = dict(tables=A, stride=4, width=4, b=3, refs=A, remap=A, err=None, scratch=A, size=1 << 20)
    d.update(rest)
    refused("pagedattn_compact_pages", (*pool, *d.values(), None), code, needle)


@pytest.mark.parametrize("kw,code,needle", BAD_TABLES)
def test_release_and_share_refuse(kw, code, needle):
    d = dict(tables=A, stride=4, width=4, b=3, refs=A)
    d.update(kw)
    t, s, w, b, r = d.values()
    refused("pagedattn_release_pages", (t, s, w, b, r, 10, None, None, None, None), code, needle)
    refused("pagedattn_release_window_pages", (t, s, w, A, b, r, 10, 5, 0, None, None), code,
            needle)
    refused("pagedattn_share_pages", (t, s, w, A, b, A, A, 1, r, 10, None, None), code, needle)


def test_release_window_and_share_arguments():
    for left, sinks in ((-1, 0), (3, -1)):
        refused("pagedattn_release_window_pages", (A, 4, 4, A, 3, A, 10, left, sinks, None, None),
                INVALID, "window")
    refused("pagedattn_release_window_pages", (A, 4, 4, None, 3, A, 10, 3, 0, None, None),
            INVALID, "kv_lens")
    refused("pagedattn_share_pages", (A, 4, 4, A, 3, A, A, -1, A, 10, None, None), INVALID,
            "num_shares")
    for i in (3, 5, 6):
        args = [A, 4, 4, A, 3, A, A, 1, A, 10, None, None]
        args[i] = None
        refused("pagedattn_share_pages", args, INVALID, "null")
    # nothing to do is no error
    assert status("pagedattn_release_pages", None, 0, 0, 0, None, 0, None, None, None, None)[0] == 0
    assert status("pagedattn_share_pages", A, 4, 4, None, 3, None, None, 0, A, 10, None,
                  None)[0] == 0


def axes_args(sections=(12, 10, 10), **kw):
    d = dict(q=A, k=A, axes=A, stride=5, n_axes=len(sections),
             sections=(ctypes.c_int32 * len(sections))(*sections), cyclic=0, nnz=5, hq=4, hkv=2,
             d=64, rotary=64, qn=256, qh=64, kn=128, kh=64, interleave=0, scale=1.0, theta=1e4,
             dtype=_lib.BF16)
    d.update(kw)
    return (*d.values(), None)


BAD_AXES = [
    (dict(sections=(12, 10)), INVALID, "sections"), (dict(sections=(30, 3, -1)), INVALID, "negative"),
    (dict(sections=(8, 12, 12), cyclic=1), INVALID, "cyclic"),
    (dict(sections=(8, 8, 8, 4, 4)), INVALID, "axes"), (dict(n_axes=0), INVALID, "axes"),
    (dict(rotary=72), INVALID, "rotary_dim"), (dict(rotary=128), INVALID, "rotary_dim"),
    (dict(d=72), INVALID, "head_dim"), (dict(scale=0.0), INVALID, "rope_scale"),
    (dict(theta=-1.0), INVALID, "rope_theta"), (dict(theta=float("nan")), INVALID, "rope_theta"),
    (dict(stride=4), INVALID, "stride"), (dict(axes=None), INVALID, "axis positions"),
    (dict(qh=60), UNSUPPORTED, "aligned"), (dict(q=A + 8), UNSUPPORTED, "aligned"),
    (dict(k=A + 2), UNSUPPORTED, "aligned"), (dict(kn=129), UNSUPPORTED, "aligned"),
    (dict(q=None), INVALID, "null"), (dict(k=None), INVALID, "null"),
    (dict(dtype=_lib.F32), UNSUPPORTED, "dtype"), (dict(nnz=-1), INVALID, "shape")]


@pytest.mark.parametrize("kw,code,needle", BAD_AXES)
def test_multi_axis_rope_refuses(kw, code, needle):
    refused("pagedattn_apply_multi_axis_rope_inplace", axes_args(**kw), code, needle)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(sections=(12, 10)), INVALID, "sections"), (dict(rotary=72), INVALID, "rotary_dim"),
    (dict(q=None), INVALID, "null"), (dict(q=A + 8), UNSUPPORTED, "aligned"),
    (dict(hq=-1), INVALID, "shape"), (dict(page=8), UNSUPPORTED, "page_size"),
    (dict(cache_dtype=_lib.F16), UNSUPPORTED, "cache dtype"),
    (dict(cache_dtype=_lib.E4M3), INVALID, "kv_scales"), (dict(bi=None), INVALID, "null")])
def test_multi_axis_append_refuses(kw, code, needle):
    sections = kw.pop("sections", (12, 10, 10))
    d = dict(q=A, qn=256, qh=64, hq=4, k=A, v=A, kn=128, kh=64, vn=128, vh=64, dtype=_lib.BF16,
             axes=A, stride=5, n=len(sections), sections=(ctypes.c_int32 * len(sections))(*sections),
             cyclic=0, bi=A, pos=A, nnz=5, rotary=64, interleave=0, scale=1.0, theta=1e4, cache=A,
             cache_dtype=_lib.BF16, scales=None, pages=9, ind=A, n_ind=9, indptr=A, b=2, hkv=2,
             d=64, page=16, err=None)
    d.update(kw)
    refused("pagedattn_multi_axis_rope_append_paged_kv_cache", (*d.values(), None), code, needle)


def test_host_tensors_are_refused():
    t = torch.zeros((2, 4), dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    refs = torch.zeros(10, dtype=torch.int32)
    pool = torch.zeros((1, 10, 2, 2, 16, 64), dtype=torch.float16)
    q = torch.zeros((3, 2, 64), dtype=torch.float16)
    for call in (lambda: pagedattn.reserve_pages(pool, t, n, None, refs),
                 lambda: pagedattn.release_pages(t, refs),
                 lambda: pagedattn.release_window_pages(t, n, refs, 5),
                 lambda: pagedattn.share_pages(t, n, [0], [1], refs),
                 lambda: pagedattn.compact_pages(pool, t, refs),
                 lambda: pagedattn.apply_multi_axis_rope_inplace(q, q, t, (32,))):
        with pytest.raises(ValueError, match="device"):
            call()
    with pytest.raises(ValueError, match="window"):
        pagedattn.release_window_pages(t, n, refs, -1)


def test_scratch_covers_both_calls():
    size = _lib.lib().pagedattn_page_scratch_bytes
    assert size(0, 0, 0) > 0 and size(-1, 1, 1) == 0
    # five int32 a row, three a page, whatever the other is
    assert size(1000, 65535, 4) >= 4 * 5 * 65535 and size(100000, 1, 1) >= 12 * 100000
