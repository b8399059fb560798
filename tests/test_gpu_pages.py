"""Page upkeep on the device (reserve, share, release, compact) against plain
Python over lists, bit for bit: tables, counts, pools of every layer and scales."""

import numpy as np
import pytest
import torch

import pagedattn

from paged_cases import i32

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "general"], autouse=True)
def path(request, monkeypatch):
    """Every test by the extension's calls and by the general path."""
    if request.param == "general":
        monkeypatch.setattr(pagedattn.ops, "_native", lambda *a: NotImplemented)


POOLS = [(2, 3, 64, torch.bfloat16), (3, 1, 128, torch.float16), (1, 8, 128, torch.bfloat16),
         (2, 2, 64, torch.float8_e4m3fn), (1, 1, 16, torch.float8_e4m3fn)]


def make_pool(device, num_pages, shape, seed=0):
    """(pool, scales) of random bits."""
    layers, hkv, d, dtype = shape
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (layers, num_pages, 2, hkv, 16, d * size), generator=g,
                        device=device, dtype=torch.uint8)
    scales = None
    if dtype == torch.float8_e4m3fn:
        scales = torch.rand((layers, num_pages, 2, hkv), generator=g, device=device)
    return raw.view(dtype), scales


def bits(pool):
    return pool.view(torch.uint8).cpu().numpy()


class Oracle:
    def __init__(self, tables, refs, pool, scales):
        self.tables, self.refs = np.array(tables), np.array(refs)
        self.pool, self.scales = bits(pool).copy(), \
            None if scales is None else scales.cpu().numpy().copy()
        self.rows_bad = self.short = 0

    def reserve(self, lens, new):
        width = self.tables.shape[1]
        plan, forked = [], {}
        for b, (length, n) in enumerate(zip(lens, new)):
            held = length - n
            if n < 0 or held < 0 or -(-length // 16) > width:
                self.rows_bad += 1
                continue
            if n > 0 and held % 16:
                page = self.tables[b, held // 16]
                if not (0 <= page < len(self.refs)) or self.refs[page] <= 0:
                    self.rows_bad += 1
                    continue
                if self.refs[page] - forked.get(page, 0) > 1:
                    forked[page] = forked.get(page, 0) + 1
                    plan.append((b, held // 16, page, held % 16))
            plan += [(b, s, -1, 0) for s in range(-(-held // 16), -(-length // 16))]
        free = np.flatnonzero(self.refs == 0)
        if len(plan) > len(free):
            self.short = len(plan) - len(free)
            return
        for (b, s, old, rows), page in zip(plan, free):
            self.tables[b, s] = page
            self.refs[page] = 1
            if old >= 0:
                self.refs[old] -= 1
                self.pool[:, page, :, :, :rows] = self.pool[:, old, :, :, :rows]
                if self.scales is not None:
                    self.scales[:, page] = self.scales[:, old]

    def release(self, first, last):
        bad = 0
        for b in range(len(self.tables)):
            for s in range(max(first[b], 0), min(last[b], self.tables.shape[1])):
                page = self.tables[b, s]
                if page < 0:
                    continue
                self.tables[b, s] = -1
                if page >= len(self.refs) or self.refs[page] <= 0:
                    bad += 1
                else:
                    self.refs[page] -= 1
        return bad

    def compact(self):
        live = np.flatnonzero(self.refs > 0)
        n = len(live)
        src, dst = live[live >= n], np.flatnonzero(self.refs[:n] == 0)
        remap = np.where(self.refs > 0, np.arange(len(self.refs)), -1)
        remap[src] = dst
        self.pool[:, dst] = self.pool[:, src]
        if self.scales is not None:
            self.scales[:, dst] = self.scales[:, src]
        self.refs[dst] = self.refs[src]
        self.refs[src] = 0
        hit = (self.tables >= 0) & (self.tables < len(remap))
        ok = hit & (remap[np.where(hit, self.tables, 0)] >= 0)
        self.tables[ok] = remap[self.tables[ok]]
        return remap, int(((self.tables >= 0) & ~ok).sum())

    def check(self, tables, refs, pool, scales):
        assert np.array_equal(tables.cpu().numpy(), self.tables)
        assert np.array_equal(refs.cpu().numpy(), self.refs)
        assert np.array_equal(bits(pool), self.pool)
        if scales is not None:
            assert np.array_equal(scales.cpu().numpy(), self.scales)


def held_tables(rng, num_pages, lens, width, samples=()):
    """Tables of sequences of `lens` tokens over scattered pages; (row, of) in
    `samples`: row holds the pages of row `of`.  With their counts."""
    perm = rng.permutation(num_pages)
    tables = np.full((len(lens), width), -1, np.int64)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // 16)
        tables[b, :k] = perm[at:at + k]
        at += k
    for row, of in samples:
        tables[row] = tables[of]
    refs = np.bincount(tables[tables >= 0], minlength=num_pages)
    return tables, refs


def flags(device, n=2):
    return torch.zeros(n, dtype=torch.int32, device=device)


@pytest.mark.parametrize("shape", POOLS)
@pytest.mark.parametrize("num_pages", [60, 4096, 9001])
def test_reserve(gpu, shape, num_pages):
    rng = np.random.default_rng(num_pages)
    lens = [0, 1, 15, 16, 17, 40, 40, 40, 31, 31, 64, 5]
    new = np.array([3, 1, 1, 1, 16, 1, 40, 1, 0, 2, 0, 70])
    samples = [(6, 5), (7, 5), (9, 8)]
    tables, refs = held_tables(rng, num_pages, lens, 9, samples)
    pool, scales = make_pool(gpu, num_pages, shape)
    want = Oracle(tables, refs, pool, scales)
    want.reserve(np.array(lens) + new, new)
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu)
    pagedattn.reserve_pages(pool, t, i32(np.array(lens) + new, gpu), i32(new, gpu), r,
                            kv_scales=scales, error_flag=err)
    want.check(t, r, pool, scales)
    assert err.tolist() == [0, 0] and want.rows_bad == want.short == 0
    # rows 5 and 6 fork, row 7 keeps the page; row 9 forks since row 8 holds it still
    assert t[7, 2] == tables[7, 2] and t[5, 2] != tables[5, 2] and t[9, 1] != tables[9, 1]


def test_reserve_decode_step_of_many_samples(gpu):
    """A step without new_lens: 700 rows, whole families on one partial page."""
    rng = np.random.default_rng(1)
    n = 700
    lens = rng.integers(1, 200, n)
    samples = [(b, b // 20 * 20) for b in range(n) if b % 20 and b % 3]
    for row, of in samples:
        lens[row] = lens[of]
    tables, refs = held_tables(rng, 12000, lens, 14, samples)
    pool, scales = make_pool(gpu, 12000, POOLS[1])
    want = Oracle(tables, refs, pool, scales)
    want.reserve(lens + 1, np.ones(n, int))
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu)
    pagedattn.reserve_pages(pool, t, i32(lens + 1, gpu), None, r, error_flag=err)
    want.check(t, r, pool, scales)
    assert err.tolist() == [0, 0]


def test_reserve_skips_bad_rows_and_counts_them(gpu):
    tables = np.array([[0, 1, -1], [2, -1, -1], [99, -1, -1], [3, 4, 5], [6, -1, -1], [7, 8, -1]])
    refs = np.zeros(20, int)
    refs[[0, 1, 2, 3, 4, 5, 7, 8]] = 1  # page 6 is held by nobody
    lens = np.array([33, 20, 5, 50, 9, -4])
    new = np.array([1, -1, 1, 3, 1, 0])
    pool, scales = make_pool(gpu, 20, POOLS[0])
    want = Oracle(tables, refs, pool, scales)
    want.reserve(lens, new)
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu)
    pagedattn.reserve_pages(pool, t, i32(lens, gpu), i32(new, gpu), r, error_flag=err)
    want.check(t, r, pool, scales)
    assert err.tolist() == [want.rows_bad, 0] == [5, 0]


@pytest.mark.parametrize("free,short", [(7, 0), (6, 1), (0, 7)])
def test_reserve_takes_all_or_nothing(gpu, free, short):
    """Six new pages and a fork: the last free page is taken; one short, nothing changes."""
    tables = np.array([[0, 1, -1, -1], [0, 1, -1, -1], [2, -1, -1, -1]])
    refs = np.zeros(3 + free, int)
    refs[:3] = [2, 2, 1]
    lens = np.array([20 + 44, 20, 16 + 48])
    new = np.array([44, 0, 48])
    pool, scales = make_pool(gpu, len(refs), POOLS[3])
    want = Oracle(tables, refs, pool, scales)
    want.reserve(lens, new)
    # row 0 appends to a page that row 1 holds: one fork, two pages; row 2: three
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu)
    pagedattn.reserve_pages(pool, t, i32(lens, gpu), i32(new, gpu), r, kv_scales=scales,
                            error_flag=err)
    want.check(t, r, pool, scales)
    assert err.tolist() == [0, want.short]
    assert want.short == max(0, 6 - free)


def test_reserve_of_nothing(gpu):
    pool, _ = make_pool(gpu, 4, POOLS[0])
    before = bits(pool).copy()
    r = i32([0, 0, 0, 0], gpu)
    pagedattn.reserve_pages(pool, i32(np.zeros((0, 5)), gpu), i32([], gpu), None, r)
    t = i32(-np.ones((2, 0)), gpu)
    pagedattn.reserve_pages(pool, t, i32([0, 0], gpu), i32([0, 0], gpu), r)
    empty = pool[:, :0].contiguous()
    err = flags(gpu)
    pagedattn.reserve_pages(empty, i32(-np.ones((1, 2)), gpu), i32([3], gpu), None, r[:0],
                            error_flag=err)
    assert not r.any() and np.array_equal(bits(pool), before)
    # row of 3 tokens, 2 of them in no page
    assert err.tolist() == [1, 0]


@pytest.mark.parametrize("width", [3, 300, 5000])
def test_release(gpu, width):
    rng = np.random.default_rng(width)
    n, num_pages = 9, 4000
    tables = rng.integers(-1, num_pages, (n, width))
    refs = np.bincount(tables[tables >= 0], minlength=num_pages)
    wide = i32(np.full((n, width + 7), 5), gpu)  # rows of a wider tensor
    t = wide[:, :width]
    t.copy_(i32(tables, gpu))
    first, last = rng.integers(-3, width // 2 + 1, n), rng.integers(-3, width + 9, n)
    pool = torch.zeros((1, num_pages, 2, 1, 16, 8), dtype=torch.float16)
    want = Oracle(tables, refs, pool, None)
    r, err = i32(refs, gpu), flags(gpu, 1)
    bad = want.release(first, last)
    pagedattn.release_pages(t, r, i32(first, gpu), i32(last, gpu), error_flag=err)
    assert np.array_equal(t.cpu().numpy(), want.tables)
    assert np.array_equal(r.cpu().numpy(), want.refs)
    assert err.item() == bad == 0 and bool((wide[:, width:] == 5).all())
    pagedattn.release_pages(t, r, error_flag=err)
    assert bool((t == -1).all()) and not r.any() and err.item() == 0


def test_release_counts_what_nobody_holds(gpu):
    """A page named three times that is held once, and one outside the pool."""
    t, r, err = i32([[1, 1], [1, 7], [0, -1]], gpu), i32([1, 1, 0], gpu), flags(gpu, 1)
    pagedattn.release_pages(t, r, error_flag=err)
    assert r.tolist() == [0, 0, 0] and err.item() == 3 and bool((t == -1).all())


@pytest.mark.parametrize("window,sinks", [(0, 0), (15, 1), (16, 16), (31, 17), (100, 40),
                                          (5000, 3)])
def test_release_window_frees_what_no_later_token_sees(gpu, window, sinks):
    rng = np.random.default_rng(window)
    lens = np.array([0, 1, 16, 17, 33, 64, 100, 129, 640])
    tables, refs = held_tables(rng, 200, lens, 41)
    t, r = i32(tables, gpu), i32(refs, gpu)
    pagedattn.release_window_pages(t, i32(lens, gpu), r, window_left=window,
                                   num_sink_tokens=sinks)
    for b, n in enumerate(lens):
        seen = {j // 16 for j in range(n) if j >= n - 1 - window or j < sinks}
        kept = np.array([tables[b, s] if s in seen else -1 for s in range(41)])
        # a page between the sinks' and the window's is freed when none of it is seen
        assert np.array_equal(t[b].cpu().numpy(), kept), (b, n)
    refs = np.bincount(t[t >= 0].cpu().numpy(), minlength=200)
    assert np.array_equal(r.cpu().numpy(), refs)


@pytest.mark.parametrize("on_device", [False, True])
def test_share(gpu, on_device):
    rng = np.random.default_rng(0)
    lens = np.array([33, 16, 5, 0, 90, 1])
    tables, refs = held_tables(rng, 64, lens, 6)
    tables[0, 1] = -1  # a page behind a window
    refs = np.bincount(tables[tables >= 0], minlength=64)
    src, dst = [0, 0, 3, 4], [1, 2, 5, 3]
    if on_device:
        src, dst = i32([0, 0, 9, 4, 4, 0, 2], gpu), i32([1, 2, 1, 5, 5, 4, 3], gpu)
    t, r, n, err = i32(tables, gpu), i32(refs, gpu), i32(lens, gpu), flags(gpu, 1)
    if not on_device:
        with pytest.raises(ValueError, match="also a source"):
            pagedattn.share_pages(t, n, src, dst, r)
        src, dst = [0, 0, 4], [1, 2, 3]
        pairs = list(zip(src, dst))
    else:
        # 9 is no row, the second 5 is taken, destinations 4 and 2 are sources too
        pairs = [(0, 1), (4, 5), (2, 3)]
    pagedattn.share_pages(t, n, src, dst, r, error_flag=err)
    for s, d in pairs:
        tables[d] = np.where(np.arange(6) < -(-lens[s] // 16), tables[s], -1)
        refs += np.bincount(tables[d][tables[d] >= 0], minlength=64)
        lens[d] = lens[s]
    assert np.array_equal(t.cpu().numpy(), tables)
    assert np.array_equal(r.cpu().numpy(), refs)
    assert np.array_equal(n.cpu().numpy(), lens)
    assert err.item() == (4 if on_device else 0)


@pytest.mark.parametrize("shape", POOLS)
@pytest.mark.parametrize("num_pages,live", [(1, 1.0), (1, 0.0), (37, 0.4), (4096, 0.9),
                                            (4097, 0.5), (9001, 0.1), (600, 1.0),
                                            (65536, 0.3)])
def test_compact(gpu, shape, num_pages, live):
    rng = np.random.default_rng(num_pages)
    refs = (rng.random(num_pages) < live) * rng.integers(1, 4, num_pages)
    held = np.flatnonzero(refs)
    tables = np.full((5, 40), -1)
    if len(held):
        tables[:, 3:] = rng.choice(held, (5, 37))
    pool, scales = make_pool(gpu, num_pages, shape)
    want = Oracle(tables, refs, pool, scales)
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu, 1)
    remap = pagedattn.compact_pages(pool, t, r, kv_scales=scales, error_flag=err)
    want_remap, _ = want.compact()
    want.check(t, r, pool, scales)
    assert np.array_equal(remap.cpu().numpy(), want_remap) and err.item() == 0
    n = int((refs > 0).sum())
    assert bool((r[:n] > 0).all()) and not r[n:].any()


@pytest.mark.parametrize("num_pages", [65537, 300001])
def test_compact_of_many_pages(gpu, num_pages):
    """Past the pools whose blocks every workgroup counts itself."""
    rng = np.random.default_rng(num_pages)
    refs = (rng.random(num_pages) < 0.4).astype(int)
    tables = rng.choice(np.flatnonzero(refs), (3, 700))
    pool, _ = make_pool(gpu, num_pages, (1, 1, 16, torch.float16))
    want = Oracle(tables, refs, pool, None)
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu, 1)
    remap = pagedattn.compact_pages(pool, t, r, error_flag=err)
    want_remap, _ = want.compact()
    want.check(t, r, pool, None)
    assert np.array_equal(remap.cpu().numpy(), want_remap) and err.item() == 0


def test_compact_leaves_entries_of_no_held_page(gpu):
    t, r, err = i32([[4, 9], [1, -1]], gpu), i32([0, 0, 0, 0, 2], gpu), flags(gpu, 1)
    pool, _ = make_pool(gpu, 5, POOLS[0])
    remap = pagedattn.compact_pages(pool, t, r, error_flag=err)
    assert t.tolist() == [[0, 9], [1, -1]] and r.tolist() == [2, 0, 0, 0, 0]
    assert remap.tolist() == [-1, -1, -1, -1, 0] and err.item() == 2


def test_pool_past_32_bits(gpu):
    """Offsets of a 6 GB pool: forks and moves at its far end."""
    num_pages = 50000
    pool = torch.zeros((2, num_pages, 2, 8, 16, 128), dtype=torch.bfloat16, device=gpu)
    last = num_pages - 1
    pool[:, last] = 3.0
    pool[0, last, 1, 7, 15] = 5.0
    refs = torch.ones(num_pages, dtype=torch.int32, device=gpu)
    refs[last] = 2
    refs[last - 1] = 0
    t = i32([[last], [last]], gpu)
    pagedattn.reserve_pages(pool, t, i32([9, 8], gpu), i32([1, 0], gpu), refs)
    assert t.tolist() == [[last - 1], [last]]
    assert bool((pool[:, last - 1, :, :, :8] == 3).all()) and not pool[:, last - 1, :, :, 8:].any()
    refs.zero_()
    refs[last] = 1
    remap = pagedattn.compact_pages(pool, t, refs)
    assert int(remap[last]) == 0 and t.tolist() == [[last - 1], [0]]
    assert torch.equal(pool[:, 0], pool[:, last]) and float(pool[0, 0, 1, 7, 15, 0]) == 5.0


def test_calls_on_another_stream(gpu):
    """Tables made on one stream and used on another, in order by an event."""
    rng = np.random.default_rng(3)
    lens = np.array([40, 40, 7])
    tables, refs = held_tables(rng, 5000, lens, 8, [(1, 0)])
    pool, scales = make_pool(gpu, 5000, POOLS[0])
    want = Oracle(tables, refs, pool, scales)
    want.reserve(lens + 1, np.ones(3, int))
    remap_want, _ = want.compact()
    side = torch.cuda.Stream()
    t, r, n = i32(tables, gpu), i32(refs, gpu), i32(lens + 1, gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pagedattn.reserve_pages(pool, t, n, None, r)
        remap = pagedattn.compact_pages(pool, t, r)
    side.synchronize()
    want.check(t, r, pool, scales)
    assert np.array_equal(remap.cpu().numpy(), remap_want)


def test_the_extension_takes_the_plain_form(gpu, path, monkeypatch):
    """And leaves what it does not take to the general path, which refuses or converts."""
    assert pagedattn.ops._native("reserve", "reserve", *[None] * 7) is NotImplemented
    pool, scales = make_pool(gpu, 9, POOLS[3])
    t, r, n = i32([[-1, -1]], gpu), i32([0] * 9, gpu), i32([3], gpu)
    took = []
    real = pagedattn.ops._native
    monkeypatch.setattr(pagedattn.ops, "_native",
                        lambda *a: took.append(real(*a)) or took[-1])
    pagedattn.reserve_pages(pool, t, n, i32([3], gpu), r, kv_scales=scales,
                            error_flag=flags(gpu))
    pagedattn.release_window_pages(t, n, r, 0)
    assert t.tolist() == [[0, -1]] and r.tolist() == [1] + [0] * 8
    assert len(took) == 2 and len({x is None for x in took}) == 1
    for bad in (dict(pool=pool[:, :, :, :, :, ::2]), dict(pool=pool[0]), dict(t=t.long()),
                dict(t=t.t()), dict(n=i32([3, 3], gpu)), dict(n=n.long()), dict(r=r[:5]),
                dict(r=r.cpu()), dict(s=None), dict(s=scales.half()), dict(s=scales[:, :5]),
                dict(new=i32([1, 1], gpu)), dict(err=flags(gpu, 1)), dict(err=flags(gpu).long())):
        x = {**dict(pool=pool, t=t, n=n, new=None, r=r, s=scales, err=None), **bad}
        with pytest.raises((ValueError, RuntimeError)):
            pagedattn.reserve_pages(x["pool"], x["t"], x["n"], x["new"], x["r"],
                                    kv_scales=x["s"], error_flag=x["err"])
    with pytest.raises(pagedattn.PagedAttnError, match="dtype"):
        pagedattn.reserve_pages(pool.float(), t, n, None, r)
    for bad in (dict(t=t.long()), dict(n=n[:0]), dict(r=r.float()), dict(w=-1), dict(s=-1),
                dict(err=flags(gpu).float())):
        x = {**dict(t=t, n=n, r=r, w=3, s=0, err=None), **bad}
        with pytest.raises(ValueError):
            pagedattn.release_window_pages(x["t"], x["n"], x["r"], x["w"], x["s"],
                                           error_flag=x["err"])
    assert t.tolist() == [[0, -1]] and r.tolist() == [1] + [0] * 8


@pytest.mark.parametrize("num_pages", [8192, 8193, 40000])
@pytest.mark.parametrize("n", [1, 127, 128, 129, 257])
@pytest.mark.parametrize("short", [False, True])
def test_reserve_counted_by_every_workgroup_or_ahead(gpu, num_pages, n, short):
    """Batches and pools on both sides of the sizes that a call counts in a launch of its own:
    families on one partial page, rows that are skipped, and pools that are nearly full."""
    rng = np.random.default_rng(num_pages + n + short)
    lens = rng.integers(1, 300, n)
    new = rng.integers(0, 40, n)
    samples = [(b, b // 8 * 8) for b in range(n) if b % 8 and b % 3]
    for row, of in samples:
        lens[row] = lens[of]
    tables, refs = held_tables(rng, num_pages, lens, 24, samples)
    new[n // 2] = 2000  # past the table
    wanted = 8 * n if not short else 0
    others = np.flatnonzero(refs == 0)  # pages of other tables
    refs[rng.permutation(others)[:max(len(others) - wanted - 1, 0)]] = 3
    pool, scales = make_pool(gpu, num_pages, POOLS[4])
    want = Oracle(tables, refs, pool, scales)
    want.reserve(lens + new, new)
    t, r, err = i32(tables, gpu), i32(refs, gpu), flags(gpu)
    pagedattn.reserve_pages(pool, t, i32(lens + new, gpu), i32(new, gpu), r, kv_scales=scales,
                            error_flag=err)
    want.check(t, r, pool, scales)
    assert err.tolist() == [want.rows_bad, want.short] and want.rows_bad == 1
    assert (want.short > 0) == (short and n > 1)
