"""The 8-bit cache on the GPU (sixi_kv8_write, sixi_kv8_read, sixi_kv8_attn) against 64-bit restatements.

Store and read-back are exact (powers of two as scales), so they must agree bit for bit; the attention within the
bound that kv8_ref.attention derives from the roundings it makes, plus half a step of the output's type."""
import sys

import numpy as np
import pytest
import torch

import sixi_attn as sa
from kv8_ref import BLOCK, PAGE, Cells, attention, random_cells, to_pages

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", file=sys.stderr, flush=True)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(k, v, rng=None):
    """A Kv8Cache over the cells, as one range per stream or (rng) as shuffled pages; and the table."""
    packed, table = [*k.pack_key(), *v.pack_value()], None
    if rng is not None:
        packed, table = to_pages(rng, packed)
        table = table.cuda()
    return sa.Kv8Cache(*[t.cuda() for t in packed]), table


def _cells_of(cache, table=None):
    """The cells a cache holds now."""
    ts = [cache.k, cache.k_exp, cache.v, cache.v_exp]
    if table is not None:
        s, per = table.shape
        ts = [t[table.long()].transpose(1, 2).flatten(2, 3) for t in ts]
    return Cells.unpack_key(ts[0], ts[1]), Cells.unpack_value(ts[2], ts[3])


# ---- store and read-back ----

def _rows(rng, s, n, heads, d, f16):
    """Rows whose size varies by 2^12 from row to row."""
    x = rng.standard_normal((s, n, heads, d)) * np.exp2(rng.uniform(-8, 4, (s, n, heads, 1)))
    return x.astype(np.float16 if f16 else np.float32)


STORES = [
    # streams, rows, heads, D, first cell of each stream, rows of each stream, f16
    (1, 1, 1, 128, [0], None, False),
    (1, 1, 4, 256, [31], None, True),
    (1, 1, 4, 128, [32], None, False),
    (3, 7, 2, 128, [0, 30, 250], [7, 5, 0], True),
    (2, 64, 4, 256, [32, 1], None, False),
    (2, 33, 1, 128, [31, 63], [33, 32], False),
    (1, 300, 3, 128, [5], [299], True),
    (4, 16, 4, 128, [500, 511, 512, 496], None, False),   # 512 cells: the last rows have no cell
    (2, 40, 2, 256, [-3, -40], None, False),              # the first rows have none
]


@pytest.mark.parametrize("s,n,heads,d,first,count,f16", STORES)
@pytest.mark.parametrize("paged", [False, True])
def test_write_and_read_back_are_exact(s, n, heads, d, first, count, f16, paged):
    _say(f"kv8 write s={s} n={n} heads={heads} d={d} first={first} count={count} f16={f16} paged={paged}")
    rng = np.random.default_rng(n * 1000 + d + s)
    cells = 512
    k, v = random_cells(rng, s, cells, heads, d), random_cells(rng, s, cells, heads, d)
    cache, table = _cache(k, v, rng if paged else None)
    rk, rv = _rows(rng, s, n, heads, d, f16), _rows(rng, s, n, heads, d, f16)
    args = dict(kv_len=_i32(first), q_len=None if count is None else _i32(count), page_table=table)
    sa.kv8_write(torch.from_numpy(rk).cuda(), torch.from_numpy(rv).cuda(), cache, **args)
    count = [n] * s if count is None else count
    k.write(rk.astype(np.float64), first, count)
    v.write(rv.astype(np.float64), first, count)
    gk, gv = _cells_of(cache, table)
    for got, want in ((gk, k), (gv, v)):
        assert np.array_equal(got.exps, want.exps)
        assert np.array_equal(got.codes, want.codes)
    # back: the rows just written, in both types; rows without a cell stay as they were
    for dtype in (torch.float32, torch.float16):
        bk, bv = (torch.full((s, n, heads, d), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        sa.kv8_read(cache, bk, bv, **args)
        for got, want in ((bk, k.values()), (bv, v.values())):
            ref = np.full((s, n, heads, d), 7.0)
            for i in range(s):
                for j in range(count[i]):
                    if 0 <= first[i] + j < cells:
                        ref[i, j] = want[i, first[i] + j]
            ref = ref.astype(np.float32 if dtype == torch.float32 else np.float16)
            assert np.array_equal(got.cpu().numpy(), ref)
    if paged:  # pages that no stream holds are untouched
        free = sorted(set(range(cache.n)) - set(table.cpu().flatten().tolist()))
        assert free and all(bool((t[free] == 1).all()) for t in (cache.k, cache.k_exp, cache.v, cache.v_exp))


def test_write_token_by_token_grows_the_scale_and_starts_it_anew():
    """100 one-row writes: louder rows grow the block's scale (kept codes are rounded again), a block begun at its
    first cell forgets what it held."""
    rng = np.random.default_rng(5)
    s, heads, d = 2, 2, 128
    k, v = random_cells(rng, s, 256, heads, d, 5, 9), random_cells(rng, s, 256, heads, d, 5, 9)
    cache, _ = _cache(k, v)
    for i in range(100):
        r = _rows(rng, s, 1, heads, d, False)
        first = [i, 64 + i // 2]
        sa.kv8_write(torch.from_numpy(r).cuda(), torch.from_numpy(-r).cuda(), cache, kv_len=_i32(first))
        k.write(r.astype(np.float64), first, [1, 1])
        v.write(-r.astype(np.float64), first, [1, 1])
    gk, gv = _cells_of(cache)
    for got, want in ((gk, k), (gv, v)):
        assert np.array_equal(got.exps, want.exps) and np.array_equal(got.codes, want.codes)


def test_write_of_extremes():
    """Zeros, subnormals, values at the borders of the scale rule, values past the exponents' range, infinities, NaN."""
    d = 128
    rows = np.zeros((1, 320, 1, d), np.float32)
    tops = [0.0, 1e-45, 127.0, np.nextafter(np.float32(127), np.float32(128)), 127 * 2.0 ** -40, 65504.0, 3e38, np.inf, np.nan, 63.5]
    for b, t in enumerate(tops):
        rows[0, b * 32:(b + 1) * 32, 0] = np.linspace(-1, 1, 32 * d, dtype=np.float32).reshape(32, d)
        if t == 0.0:
            rows[0, b * 32:(b + 1) * 32] = 0.0
        rows[0, b * 32 + 5, 0, 17] = t
        if t not in (np.inf,) and np.isfinite(t):
            x = rows[0, b * 32:(b + 1) * 32, 0]
            x[np.abs(x) > abs(t)] = np.float32(t) * np.float32(0.5)
    k = Cells(1, 512, 1, d)
    cache, _ = _cache(k, k)
    sa.kv8_write(torch.from_numpy(rows).cuda(), torch.from_numpy(rows).cuda(), cache, kv_len=_i32([0]))
    k.write(rows.astype(np.float64), [0], [320])
    for got in _cells_of(cache):
        assert np.array_equal(got.exps, k.exps) and np.array_equal(got.codes, k.codes)


def test_write_reads_strided_rows_and_strided_blocks():
    """Rows as a slice of a wider projection, a cache whose heads lie in a wider tensor."""
    rng = np.random.default_rng(9)
    s, n, heads, d = 2, 5, 3, 128
    wide = torch.from_numpy(_rows(rng, s, n, 2 * heads + 2, 2 * d, True)).cuda()
    rk, rv = wide[:, :, 0:2 * heads:2, :d], wide[:, :, 1:2 * heads + 1:2, d:]
    k, v = random_cells(rng, s, 256, heads + 2, d), random_cells(rng, s, 256, heads + 2, d)
    packed = [t.cuda() for t in (*k.pack_key(), *v.pack_value())]
    cache = sa.Kv8Cache(*[t[:, 1:heads + 1] for t in packed])
    first = [40, 3]
    sa.kv8_write(rk, rv, cache, kv_len=_i32(first))
    part = [Cells(s, 256, heads, d, x.codes[:, :, 1:heads + 1].copy(), x.exps[:, :, 1:heads + 1].copy()) for x in (k, v)]
    for x, r in zip(part, (rk, rv)):
        x.write(r.cpu().numpy().astype(np.float64), first, [n] * s)
    for got, want in zip((Cells.unpack_key(*packed[:2]), Cells.unpack_value(*packed[2:])), zip((k, v), part)):
        whole, mine = want
        whole.codes[:, :, 1:heads + 1], whole.exps[:, :, 1:heads + 1] = mine.codes, mine.exps
        assert np.array_equal(got.exps, whole.exps) and np.array_equal(got.codes, whole.codes)


def test_exponents_out_of_range_count_as_the_nearest():
    d = 128
    k = Cells(1, 256, 1, d, np.full((1, 256, 1, d), 3), np.array([[[-128], [-41], [41], [127], [0], [0], [0], [0]]]))
    cache, _ = _cache(k, k)
    out = [torch.zeros((1, 256, 1, d), device="cuda") for _ in range(2)]
    sa.kv8_read(cache, *out)
    assert all(np.array_equal(o.cpu().numpy(), k.values().astype(np.float32)) for o in out)
    half = [torch.zeros((1, 256, 1, d), dtype=torch.float16, device="cuda") for _ in range(2)]
    sa.kv8_read(cache, *half)
    assert float(half[0][0, 70, 0, 0]) == 65504.0 and float(half[0][0, 3, 0, 0]) == 0.0


# ---- attention ----

def _attend(s, n_q, H, heads, d, cached, rows, cells, mode=sa.MASK_BLOCK_CAUSAL, paged=False, q16=True, o16=True,
            scale=None, seed=0, mask=None, exps=(-6, -3), q_size=2.0, no_lens=False, no_rows=False, handle=None):
    _say(f"kv8 attention s={s} n_q={n_q} H={H} heads={heads} d={d} cached={cached} rows={rows} cells={cells} mode={mode} "
         f"paged={paged} q16={q16} o16={o16} scale={scale} exps={exps}")
    rng = np.random.default_rng(seed + n_q * 7 + d + sum(cached))
    k, v = random_cells(rng, s, cells, heads, d, *exps), random_cells(rng, s, cells, heads, d, *exps)
    q = (rng.standard_normal((s, n_q, H, d)) * q_size).astype(np.float16 if q16 else np.float32)
    for i in range(s):  # what no row may look at: queries past a stream's rows, exponents past its cells
        q[i, rows[i]:] = np.nan
        k.exps[i, -(-(cached[i] + rows[i]) // BLOCK):] = 127
        v.exps[i, -(-(cached[i] + rows[i]) // BLOCK):] = 127
    cache, table = _cache(k, v, rng if paged else None)
    out = torch.full((s, n_q, H, d), float("nan"), dtype=torch.float16 if o16 else torch.float32, device="cuda")
    sc = d ** -0.5 if scale is None else scale
    fa = handle or sa.Kv8Attention()
    fa(torch.from_numpy(q).cuda(), cache, out, kv_len=None if no_lens else _i32(cached), q_len=None if no_rows else _i32(rows), mask_mode=mode,
       mask=None if mask is None else torch.from_numpy(mask).cuda(), scale=scale, page_table=table)
    want, tol = attention(q.astype(np.float16).astype(np.float64), k.values(), v.values(), v.exps, cached, rows, sc, mode,
                          None if mask is None else mask.astype(np.float64))
    got = out.cpu().numpy().astype(np.float64)
    live = np.zeros((s, n_q), bool)
    for i in range(s):
        live[i, :rows[i]] = True
    assert np.isnan(got[~live]).all()
    # half a step of the output's type; f16 outputs below its normal numbers have steps of 2^-24
    tol = tol + np.abs(want) * (2.0 ** -11 if o16 else 2.0 ** -22) + (2.0 ** -25 if o16 else 0.0)
    off = np.abs(got - want)[live] / np.maximum(tol[live], 1e-300)
    _say(f"  worst {off.max() if off.size else 0:.3f} of the bound")
    assert (off <= 1.0).all()
    return got


SHAPES = [
    # streams, rows, H, heads, cached, rows of each, cells
    (1, 1, 4, 4, [0], [1], 32),
    (1, 1, 24, 4, [30], [1], 32),
    (2, 1, 24, 4, [31, 32], [1, 1], 64),
    (3, 1, 15, 3, [255, 256, 700], [1, 0, 1], 1024),
    (2, 5, 24, 4, [0, 97], [5, 3], 256),
    (2, 16, 24, 4, [1000, 17], [16, 9], 1024 + 32),
    (1, 16, 32, 1, [100], [16], 256),
    (2, 17, 8, 8, [250, 3], [17, 17], 512),
    (1, 33, 12, 2, [400], [33], 448),
    (1, 100, 6, 1, [0], [100], 128),
    (1, 70, 24, 4, [300], [70], 512),
]


@pytest.mark.parametrize("s,n_q,H,heads,cached,rows,cells", SHAPES)
@pytest.mark.parametrize("d", [128, 256])
def test_attention_shapes(s, n_q, H, heads, cached, rows, cells, d):
    _attend(s, n_q, H, heads, d, cached, rows, cells)
    _attend(s, n_q, H, heads, d, cached, rows, cells, q16=False, o16=False, mode=sa.MASK_NONE, seed=3)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("rows", [1, 6, 16, 40])
def test_attention_pages(d, rows):
    _attend(3, rows, 24, 4, d, [513, 0, 1400], [rows, rows, max(1, rows - 2)], 1536, paged=True)


@pytest.mark.parametrize("d", [128, 256])
def test_attention_long(d):
    _attend(1, 2, 6, 1, d, [20011], [2], 20480)
    _attend(2, 1, 6, 1, d, [9000, 33], [1, 1], 9216, paged=True, seed=1)


@pytest.mark.parametrize("d", [128, 256])
def test_attention_rows_of_every_stream(d):
    """Without q_len the host can tell whether there is anything to join: few tiles, just enough of them, and more."""
    for s, n_q in ((2, 20), (15, 127), (16, 128), (17, 129)):
        _attend(s, n_q, 12, 4, d, [5 * i % 70 for i in range(s)], [n_q] * s, 256, no_rows=True)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("n_q,H,heads", [(6, 24, 4), (8, 24, 4), (11, 24, 4), (16, 24, 4), (64, 2, 2), (90, 1, 1), (3, 32, 1)])
def test_attention_of_33_to_96_rows(d, n_q, H, heads):
    """Two and three tiles of rows in one work-group: lengths about its steps of 128 cells and their pieces, ragged rows,
    pages, and scales that outgrow the reference again and again."""
    for i, cached in enumerate([[0, 1, 90], [127, 128, 129], [255, 700, 1023 - n_q], [1500, 0, 5]]):
        rows = [n_q, max(1, n_q // 2), n_q if i % 2 else 0]
        _attend(3, n_q, H, heads, d, cached, rows, 1792, paged=i % 2 == 1, q16=i < 2, o16=i > 0, seed=i)
        _attend(3, n_q, H, heads, d, cached, rows, 1792, exps=(-16, 8), q_size=0.05, mode=sa.MASK_NONE if i == 3 else sa.MASK_BLOCK_CAUSAL,
                seed=10 + i)
    rng = np.random.default_rng(n_q)
    for hidden in (-np.inf, -65504.0):
        m = _tree(rng, 2, n_q, 1024, [800, 90], [n_q, n_q], hidden)
        _attend(2, n_q, H, heads, d, [800, 90], [n_q, n_q], 1024, mode=sa.MASK_EXPLICIT, mask=m, seed=5)


@pytest.mark.parametrize("s", [64, 65, 130, 512])
def test_attention_of_many_streams(s):
    """Past 64 streams the cut goes over the lanes more than once."""
    rng = np.random.default_rng(s)
    cached = [int(x) for x in rng.integers(0, 250, s)]
    rows = [int(x) for x in rng.integers(0, 3, s)]
    _attend(s, 2, 6, 1, 128, cached, rows, 256)
    cached[s // 2], rows[s // 2] = 3000, 2      # one long among short ones: its pieces are numbered between theirs
    cached[-1], rows[-1] = 1200, 1
    _attend(s, 2, 2, 1, 128, cached, rows, 3104, seed=1)


@pytest.mark.parametrize("d,n_q,H,masked", [(128, 1, 6, False), (128, 8, 6, False), (128, 5, 6, True), (256, 5, 6, False), (256, 3, 6, True),
                                            (128, 40, 6, False)])
def test_attention_in_a_cache_of_gigabytes(d, n_q, H, masked):
    """A pool larger than the chip's caches, read past them where one work-group reads each cell: the same bits as a small
    cache that holds the same cells."""
    pages, n = (1 << 29) // (2 * PAGE * d) + 9, 2900
    big, small = sa.Kv8Cache.empty(pages, PAGE, 1, d), sa.Kv8Cache.empty(1, 12 * PAGE, 1, d)
    gen = torch.Generator(device="cuda").manual_seed(d + n_q)
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[None].contiguous()
    rows = [torch.randn((1, n + n_q, 1, d), generator=gen, device="cuda") for _ in range(2)]
    sa.kv8_write(*rows, big, page_table=table)
    sa.kv8_write(*rows, small)
    q = torch.randn((1, n_q, H, d), generator=gen, device="cuda").half()
    outs = [torch.zeros((1, n_q, H, d), device="cuda") for _ in range(2)]
    mask = None
    if masked:
        mask = torch.full((1, 1, n_q, pages * PAGE), -float("inf"), dtype=torch.float16, device="cuda")
        mask[..., :n] = torch.randn((n_q, n), generator=gen, device="cuda").half()
    mode = sa.MASK_EXPLICIT if masked else sa.MASK_BLOCK_CAUSAL
    for cache, out, pt in ((big, outs[0], table), (small, outs[1], None)):
        m = None if mask is None else mask[..., :cache.n_blocks * BLOCK] if pt is None else mask
        sa.Kv8Attention()(q, cache, out, kv_len=_i32([n]), q_len=_i32([n_q]), mask_mode=mode, mask=m, page_table=pt)
    assert torch.equal(*outs) and bool((outs[0].abs().sum(-1) > 0).all())


@pytest.mark.parametrize("d,n_q", [(128, 2), (128, 40), (256, 40)])
def test_offsets_past_32_bits(d, n_q):
    """Blocks half a GiB apart: a stream's cells lie up to 5 GiB behind one another."""
    rng = np.random.default_rng(d + n_q)
    cells, step = 320, 1 << 29
    k, v = random_cells(rng, 1, cells, 1, d), random_cells(rng, 1, cells, 1, d)
    packed = [*k.pack_key(), *v.pack_value()]
    room = [torch.empty((cells // BLOCK - 1) * step + 2 * BLOCK * d, dtype=torch.int8, device="cuda") for _ in range(2)]
    codes = []
    for t, r in zip((packed[0], packed[2]), room):
        inner = [x for x in t.stride()[3:]]
        far = r.as_strided(t.shape, (r.numel(), BLOCK * d, step, *inner))
        far.copy_(t)
        codes.append(far)
    cache = sa.Kv8Cache(codes[0], packed[1].cuda(), codes[1], packed[3].cuda())
    rk, rv = _rows(rng, 1, 40, 1, d, False), _rows(rng, 1, 40, 1, d, False)
    first = cells - 41
    sa.kv8_write(torch.from_numpy(rk).cuda(), torch.from_numpy(rv).cuda(), cache, kv_len=_i32([first]))
    k.write(rk.astype(np.float64), [first], [40])
    v.write(rv.astype(np.float64), [first], [40])
    back = [torch.zeros((1, cells, 1, d), device="cuda") for _ in range(2)]
    sa.kv8_read(cache, *back)
    for got, want in zip(back, (k, v)):
        assert np.array_equal(got.cpu().numpy(), want.values().astype(np.float32))
    q = rng.standard_normal((1, n_q, 3, d)).astype(np.float16)
    out = torch.zeros((1, n_q, 3, d), device="cuda")
    sa.Kv8Attention()(torch.from_numpy(q).cuda(), cache, out, kv_len=_i32([cells - 1 - n_q]))
    want, tol = attention(q.astype(np.float64), k.values(), v.values(), v.exps, [cells - 1 - n_q], [n_q], d ** -0.5, sa.MASK_BLOCK_CAUSAL)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol + 2.0 ** -22 * np.abs(want)).all()


def test_attention_few_rows_of_a_long_block():
    """Rows for many tiles, few of them there: their cells are cut and joined."""
    _attend(2, 2000, 24, 4, 128, [1500, 2000], [40, 3], 4096)
    _attend(1, 700, 8, 1, 256, [900], [90], 2048, paged=True)


def test_attention_without_lengths_sees_every_cell():
    _attend(2, 3, 8, 2, 128, [253, 253], [3, 3], 256, mode=sa.MASK_NONE, no_lens=True)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0, 1e-30, 7.5])
def test_attention_scales(d, scale):
    _attend(1, 3, 12, 2, d, [77], [3], 128, scale=scale, q_size=0.3)


@pytest.mark.parametrize("d", [128, 256])
def test_attention_over_unequal_scales(d):
    """Blocks whose scales differ by up to 2^24, the loud ones seen by few: the weights keep their precision."""
    _attend(1, 4, 6, 1, d, [700], [4], 1024, exps=(-16, 8), q_size=0.02)
    _attend(1, 4, 6, 1, d, [90], [4], 128, exps=(-40, -30), q_size=40.0, o16=False)
    _attend(1, 40, 6, 1, d, [90], [40], 256, exps=(20, 40), q_size=1e-4, scale=1e-9, o16=False)


def _tree(rng, s, n_q, cells, cached, rows, hidden):
    """Random trees: a row sees the cached cells but some, and its ancestors."""
    m = np.full((s, 1, n_q, cells), hidden, np.float16)
    for i in range(s):
        for j in range(rows[i]):
            m[i, 0, j, :cached[i]] = np.where(rng.random(cached[i]) < 0.8, rng.standard_normal(cached[i]) * 0.5, hidden)
            if j:
                p = int(rng.integers(0, j))
                m[i, 0, j, cached[i]:] = m[i, 0, p, cached[i]:]
            m[i, 0, j, cached[i] + j] = 0.0
    return m


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("s,n_q,cached,rows,cells", [(1, 1, [0], [1], 32), (2, 12, [100, 31], [12, 7], 256),
                                                      (1, 16, [999], [16], 1024), (2, 50, [64, 5], [50, 41], 256)])
def test_attention_masks(d, s, n_q, cached, rows, cells):
    rng = np.random.default_rng(cells + n_q)
    for hidden in (-np.inf, np.finfo(np.float16).min):
        m = _tree(rng, s, n_q, cells, cached, rows, hidden)
        for i in range(s):  # cells that the stream does not have: never looked at
            m[i, :, :, cached[i] + rows[i]:] = np.nan
        _attend(s, n_q, 12, 2, d, cached, rows, cells, mode=sa.MASK_EXPLICIT, mask=m, seed=int(hidden == -np.inf))


def test_attention_masks_that_leave_rows_empty():
    rng = np.random.default_rng(2)
    m = _tree(rng, 2, 6, 128, [40, 90], [6, 6], -np.inf)
    m[0, 0, 2] = -np.inf
    m[1, 0, 5] = -np.inf
    got = _attend(2, 6, 12, 2, 128, [40, 90], [6, 6], 128, mode=sa.MASK_EXPLICIT, mask=m)
    assert (got[0, 2] == 0).all() and (got[1, 5] == 0).all()
    # one mask for every stream, of lowest values only: the cells weigh alike
    m = np.full((1, 1, 6, 128), np.finfo(np.float16).min, np.float16)
    _attend(2, 6, 12, 2, 256, [40, 90], [6, 6], 128, mode=sa.MASK_EXPLICIT, mask=m, q_size=0.0)


def test_attention_strides():
    """Q as the first half of the heads' rows of a wider tensor, the output into every second row of another, a mask
    whose rows begin at odd addresses."""
    rng = np.random.default_rng(4)
    s, n_q, H, heads, d, cached, cells = 2, 4, 12, 2, 128, [70, 20], 128
    k, v = random_cells(rng, s, cells, heads, d), random_cells(rng, s, cells, heads, d)
    cache, _ = _cache(k, v)
    qg = torch.from_numpy(rng.standard_normal((s, n_q, H, 2 * d)).astype(np.float32)).cuda()
    wide = torch.full((s, 2 * n_q, H, d + 8), float("nan"), dtype=torch.float16, device="cuda")
    m = _tree(rng, s, n_q, cells, cached, [n_q] * s, -np.inf)
    odd = torch.full((s, 1, n_q, cells + 3), float("nan"), dtype=torch.float16, device="cuda")
    odd[..., 1:cells + 1] = torch.from_numpy(m).cuda()
    sa.Kv8Attention()(qg[..., :d], cache, wide[:, ::2, :, :d], kv_len=_i32(cached), mask_mode=sa.MASK_EXPLICIT,
                      mask=odd[..., 1:cells + 1])
    want, tol = attention(qg[..., :d].half().double().cpu().numpy(), k.values(), v.values(), v.exps, cached, [n_q] * s,
                          d ** -0.5, 2, m.astype(np.float64))
    got = wide.cpu().double().numpy()
    assert (np.abs(got[:, ::2, :, :d] - want) <= tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
    assert np.isnan(got[:, 1::2]).all() and np.isnan(got[..., d:]).all()


def test_attention_nan_stays_in_its_row():
    rng = np.random.default_rng(6)
    k, v = random_cells(rng, 1, 64, 1, 128), random_cells(rng, 1, 64, 1, 128)
    cache, _ = _cache(k, v)
    q = torch.randn((1, 4, 6, 128), device="cuda", dtype=torch.float16)
    outs = []
    for bad in (False, True):
        if bad:
            q[0, 1, 2, 5] = float("nan")
            q[0, 3, 0, 0] = float("inf")
        out = torch.zeros((1, 4, 6, 128), device="cuda")
        sa.Kv8Attention()(q, cache, out, kv_len=_i32([50]))
        outs.append(out.cpu().numpy())
    same = np.ones((4, 6), bool)
    same[1, 2] = same[3, 0] = False
    assert np.isnan(outs[1][0, 1, 2]).all() and np.isnan(outs[1][0, 3, 0]).any()
    assert np.array_equal(outs[0][0][same], outs[1][0][same])


def test_attention_is_the_same_every_time_and_in_a_poisoned_workspace():
    rng = np.random.default_rng(8)
    k, v = random_cells(rng, 2, 2048, 2, 256), random_cells(rng, 2, 2048, 2, 256)
    cache, _ = _cache(k, v)
    q = torch.randn((2, 8, 12, 256), device="cuda", dtype=torch.float16)
    fa, kv = sa.Kv8Attention(), _i32([2040, 900])
    outs = []
    for fill in (0, 255, 127):
        out = torch.zeros((2, 8, 12, 256), device="cuda")
        p = fa.params(q, cache, out, kv_len=kv)
        ws = torch.full((fa.workspace_bytes(p),), fill, dtype=torch.uint8, device="cuda")
        fa(q, cache, out, kv_len=kv, workspace=ws)
        outs.append(out.cpu().numpy())
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


def test_page_entries_out_of_range_are_clamped():
    """Entries of pages that no row sees may hold anything; a bad one that is seen reads some page of the pool."""
    rng = np.random.default_rng(3)
    k, v = random_cells(rng, 1, 1024, 2, 128), random_cells(rng, 1, 1024, 2, 128)
    cache, table = _cache(k, v, rng)
    q = torch.randn((1, 1, 12, 128), device="cuda", dtype=torch.float16)
    outs = []
    for junk in (None, -1, 1 << 30):
        t = table.clone()
        if junk is not None:
            t[0, 2:] = junk
        out = torch.zeros((1, 1, 12, 128), device="cuda")
        sa.Kv8Attention()(q, cache, out, kv_len=_i32([500]), page_table=t)
        outs.append(out.cpu().numpy())
        if junk is not None:
            sa.Kv8Attention()(q, cache, out, kv_len=_i32([900]), page_table=t)
            assert np.isfinite(out.cpu().numpy()).all()
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


def test_lengths_out_of_range_are_clamped():
    """kv_len past the cells counts as the last place for the block, a negative one as 0; q_len as [0, n_q]."""
    rng = np.random.default_rng(13)
    k, v = random_cells(rng, 2, 128, 2, 128), random_cells(rng, 2, 128, 2, 128)
    cache, _ = _cache(k, v)
    q = torch.randn((2, 4, 12, 128), device="cuda", dtype=torch.float16)
    outs = []
    for kv, ql in (([124, 0], [4, 4]), ([1 << 30, -5], [9, 1 << 30])):
        out = torch.zeros((2, 4, 12, 128), device="cuda")
        sa.Kv8Attention()(q, cache, out, kv_len=_i32(kv), q_len=_i32(ql))
        outs.append(out.cpu().numpy())
    assert np.array_equal(outs[0], outs[1])
    out = torch.full((2, 4, 12, 128), 5.0, device="cuda")
    sa.Kv8Attention()(q, cache, out, kv_len=_i32([3, 3]), q_len=_i32([0, -1]))
    assert bool((out == 5.0).all())


def test_streams_and_handles_side_by_side():
    """Two handles on two streams at once, each the same as alone."""
    rng = np.random.default_rng(21)
    k, v = random_cells(rng, 1, 4096, 2, 128), random_cells(rng, 1, 4096, 2, 128)
    cache, _ = _cache(k, v)
    qs = [torch.randn((1, 4, 12, 128), device="cuda", dtype=torch.float16) for _ in range(2)]
    want = []
    for q in qs:
        out = torch.zeros((1, 4, 12, 128), device="cuda")
        sa.Kv8Attention()(q, cache, out, kv_len=_i32([4000]))
        want.append(out)
    handles, kv = [sa.Kv8Attention() for _ in qs], _i32([4000])
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [torch.zeros((1, 4, 12, 128), device="cuda") for _ in qs]
    torch.cuda.synchronize()
    for _ in range(5):
        for q, h, st, out in zip(qs, handles, streams, outs):
            with torch.cuda.stream(st):
                h(q, cache, out, kv_len=kv)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_pool_copies_codes_and_exponents():
    """A stream that shares a page and then writes into it gets a copy, codes and exponents."""
    rng = np.random.default_rng(17)
    pool = sa.KvPool(4, 2, 2)
    cache = sa.Kv8Cache.empty(4, PAGE, 2, 128)
    cache.attach(pool)
    pool.prepare_write(0, 0, 40)
    r = torch.from_numpy(_rows(rng, 2, 40, 2, 128, False)).cuda()
    sa.kv8_write(r, r, cache, kv_len=_i32([0, 0]), q_len=_i32([40, 0]), page_table=pool.upload())
    pool.seq_cp(0, 1)
    pool.prepare_write(1, 40, 5)
    table = pool.upload()
    assert int(table[0, 0]) != int(table[1, 0])
    a, b = int(table[0, 0]), int(table[1, 0])
    assert all(torch.equal(t[a], t[b]) for t in (cache.k, cache.k_exp, cache.v, cache.v_exp))
    before = [t[a].clone() for t in (cache.k, cache.k_exp, cache.v, cache.v_exp)]
    sa.kv8_write(r, r, cache, kv_len=_i32([0, 40]), q_len=_i32([0, 5]), page_table=table)
    assert all(torch.equal(t[a], x) for t, x in zip((cache.k, cache.k_exp, cache.v, cache.v_exp), before))
    back = [torch.zeros((2, 45, 2, 128), device="cuda") for _ in range(2)]
    sa.kv8_read(cache, *back, kv_len=_i32([0, 0]), q_len=_i32([40, 45]), page_table=table)
    k = Cells(1, 64, 2, 128)
    k.write(r[:1].double().cpu().numpy(), [0], [40])
    assert np.array_equal(back[0][0, :40].cpu().numpy(), k.values()[0, :40])
    k.write(r[1:2, :5].double().cpu().numpy(), [40], [5])
    assert np.array_equal(back[1][1].cpu().numpy(), k.values()[0, :45])
