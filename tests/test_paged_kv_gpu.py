"""The paged key-value cache functions against plain 64-bit forms: formats, head layouts, lengths around every tile and page
border, poisoned free slots, masks, bad page numbers, strides, streams and graphs, and a run of them together."""
import math

import numpy as np
import pytest
import torch

from helpers import adversarial, assert_bits_equal, bits
from paged_reference import FORMATS, HALF, Pool, attend, evict, values

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16)
EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 257]


def F():
    from mase_amd.quantized import functional

    return functional


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------------------------------------------------------------
# gather
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 16)])
def test_gather_reads_sequences_back(dev, fmt, dim, page, dtype):
    p = Pool(gen(1), [0, 1, 17, 40, 33], 3, dim, page, fmt, dtype, extra_slots=3, strided=True)
    k, v = F().paged_kv_gather(**p.to(dev), lengths=i32(p.lengths, dev), max_length=p.max_length, dtype=dtype)
    for b, n in enumerate(p.lengths):
        for got, want in zip((k, v), p.rows(b, n)):
            assert_bits_equal(got[b, :, :n], want.to(dtype), f"sequence {b}")  # every value is exact in dtype
            assert not bool(got[b, :, n:].any())


@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_every_code_and_scale_widens_to_its_value(dev, fmt):
    """all 256 bytes of codes under all scale bytes: exact where bf16 holds the value, NaN under byte 255"""
    n = 256
    k = torch.arange(256).repeat(n, 1).to(torch.uint8)
    if fmt == "mxfp8_e4m3":
        k[(k & 127) == 127] = 0
    elif fmt == "mxfp8_e5m2":
        k[(k & 124) == 124] = 0
    width = 128 if fmt == "mxfp4" else 256
    codes = k[:, :width].reshape(n // 16, 1, 16, width)
    s = torch.arange(256).to(torch.uint8)
    ks = s.view(n // 16, 1, 16, 1).expand(-1, -1, -1, 8).contiguous()
    vs = s.view(n // 16, 1, 1, 16).expand(-1, -1, 8, -1).contiguous()
    pages = codes.view(torch.int8) if fmt == "mxint8" else codes
    table = torch.arange(n // 16, dtype=torch.int32).view(1, -1)
    got = F().paged_kv_gather(pages.to(dev), pages.to(dev), table.to(dev), i32([n], dev), n, dtype=torch.bfloat16, kv_format=fmt,
                              k_scales=ks.to(dev), v_scales=vs.to(dev))
    want = values(pages.reshape(n, width), ks.reshape(n, 8), fmt)
    ok = want.isnan() | (want == want.to(torch.bfloat16).double())  # within bf16's range and steps
    top = 2.0 ** 127 * (2 - 2.0 ** -7)
    ok &= want.isnan() | (want.abs() <= top)
    assert float(ok.float().mean()) > 0.9
    for g in got:
        g = g[0, 0].cpu().double()
        same = (g == want) | (g.isnan() & want.isnan())
        bad = (~same & ok).nonzero()
        assert bad.numel() == 0, (fmt, bad[:4].tolist(), [(float(g[tuple(i)]), float(want[tuple(i)])) for i in bad[:4]])


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def _empty_pool(n, heads, dim, page, fmt, dtype, dev, fill=0x5A):
    width = dim // 2 if fmt == "mxfp4" else dim
    if fmt is None:
        k = torch.full((n, heads, page, width), 0x5A5A, dtype=torch.int16, device=dev).view(dtype)
        return dict(k_pages=k, v_pages=k.clone())
    code = torch.int8 if fmt == "mxint8" else torch.uint8
    k = torch.full((n, heads, page, width), fill, dtype=code, device=dev)
    return dict(k_pages=k, v_pages=k.clone(), kv_format=fmt, k_scales=torch.full((n, heads, page, dim // 32), fill, dtype=torch.uint8, device=dev),
                v_scales=torch.full((n, heads, dim // 32, page), fill, dtype=torch.uint8, device=dev))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 1), (128, 64, 3), (256, 16, 2)])
def test_append_writes_its_slots_and_no_others(dev, fmt, dim, page, heads, dtype):
    g = gen(2)
    starts, counts, tokens = [0, 5, 15, 30, 2, 40], [21, 0, 2, 18, 1, 21], 21
    b, n_tab = len(starts), -(-64 // page)
    n = b * n_tab + 2
    table = torch.randperm(n, generator=g)[: b * n_tab].view(b, n_tab).to(torch.int32)
    # states as a fused projection leaves them: [batch, tokens, (keys | values), heads, dim]
    states = torch.randn(b, tokens, 2, heads, dim, generator=g).mul_(3).to(dtype)
    key, value = states[:, :, 0].transpose(1, 2), states[:, :, 1].transpose(1, 2)
    sd = states.to(dev)
    pool = _empty_pool(n, heads, dim, page, fmt, dtype, dev)
    before = {k: t.clone() for k, t in pool.items() if torch.is_tensor(t)}
    positions = torch.full((b, heads, n_tab * page + 3), -7, dtype=torch.int32, device=dev)
    F().paged_kv_append(sd[:, :, 0].transpose(1, 2), sd[:, :, 1].transpose(1, 2), page_table=table.to(dev), starts=i32(starts, dev),
                        counts=i32(counts, dev), positions=positions, first_positions=i32([100 * i for i in range(b)], dev), **pool)
    from mase_amd._gemm import mxfp_pack
    from mase_amd.quantizers import _ops

    def packed(x):  # what the package's packing functions make of the same states
        flat = x.to(dev).contiguous()
        if fmt == "mxint8":
            _, c, s = _ops.mxint_qdq(flat, 32, 8, -1, 8, pack=True)
            return c.view(flat.shape).cpu(), s.view(*flat.shape[:-1], -1).cpu()
        e, f = {"mxfp8_e4m3": (4, 3), "mxfp8_e5m2": (5, 2), "mxfp4": (2, 1)}[fmt]
        c, s = mxfp_pack(flat.view(-1, dim), e, f)
        return c.view(*flat.shape[:-1], -1).cpu(), s.view(*flat.shape[:-1], -1).cpu()

    want = {k: t.cpu() for k, t in before.items()}
    want_pos = torch.full(positions.shape, -7, dtype=torch.int32)
    if fmt is not None:
        (kc, ksc), (vc, vsc) = packed(key), packed(value)
    for i in range(b):
        for j in range(counts[i]):
            slot = starts[i] + j
            if slot >= n_tab * page:
                continue  # past the table: not written
            pg, at = int(table[i, slot // page]), slot % page
            if fmt is None:
                want["k_pages"][pg, :, at], want["v_pages"][pg, :, at] = key[i, :, j], value[i, :, j]
            else:
                want["k_pages"][pg, :, at], want["v_pages"][pg, :, at] = kc[i, :, j], vc[i, :, j]
                want["k_scales"][pg, :, at], want["v_scales"][pg, :, :, at] = ksc[i, :, j], vsc[i, :, j]
            want_pos[i, :, slot] = 100 * i + j
    for k, t in want.items():
        got = pool[k].cpu()
        if fmt is None:
            assert_bits_equal(got, t, k)
        else:
            assert torch.equal(got, t), k
    assert torch.equal(positions.cpu(), want_pos)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS[1:])
def test_append_then_gather_are_the_quantizers_values(dev, fmt, dtype):
    """adversarial states (ties, powers of two, tiny and huge blocks, non-finite elements): what comes back is what the
    quantizer functions give; their packed forms re-express blocks with reserved codes, checked through those"""
    import mase_amd.quantizers as Q
    from mase_amd._gemm import mxfp_pack

    rng = np.random.default_rng(3)
    x = adversarial(rng, (1, 2, 96, 128), dtype)
    x[0, 1, 5, 7], x[0, 1, 6, 40], x[0, 0, 9, 100] = math.nan, math.inf, -math.inf
    xd = x.to(dev)
    pool = _empty_pool(8, 2, 128, 16, fmt, dtype, dev)
    table = i32([[5, 2, 7, 0, 3, 1]], dev)
    F().paged_kv_append(xd, xd, page_table=table, starts=i32([0], dev), **pool)
    k, v = F().paged_kv_gather(page_table=table, lengths=i32([96], dev), max_length=96, dtype=dtype, **pool)
    if fmt == "mxint8":
        want = Q.mxint_quantizer(xd, 32, 8)
    else:
        e, f = {"mxfp8_e4m3": (4, 3), "mxfp8_e5m2": (5, 2), "mxfp4": (2, 1)}[fmt]
        c, s = mxfp_pack(xd.view(-1, 128), e, f)
        want = values(c.cpu().view(192, -1), s.cpu().view(192, 4), fmt).view(x.shape).to(dtype).to(dev)
    for got in (k, v):
        same = (got == want) | (got.isnan() & want.isnan())  # a zero's sign is not kept by codes
        if dtype == torch.float16:  # and values below fp16's range come out as its rounding of them
            same |= (got.double() - want.double()).abs() <= 2.0 ** -25
        assert bool(same.all()), (int((~same).sum()), got[~same][:4].tolist(), want[~same][:4].tolist())


# ---------------------------------------------------------------------------------------------------------------------
# attention of one token
# ---------------------------------------------------------------------------------------------------------------------
def check_decode(dev, p, group, seed, mask=None, scaling=None, weights=False, absent=None, max_length=None, runs=1):
    g = gen(seed)
    b, dim, kvh = len(p.lengths), p.dim, p.heads
    q = torch.randn(b, kvh * group, dim, generator=g).to(p.dtype)
    scale = dim ** -0.5 if scaling is None else scaling
    args = dict(p.to(dev), lengths=i32(p.lengths, dev), max_length=p.max_length if max_length is None else max_length)
    w = w0 = None
    if weights:
        w0 = torch.rand(b, kvh, p.table.shape[1] * p.page + 5, generator=g)
        w = w0.to(dev)
    for _ in range(runs):
        out = F().paged_attention_decode(q.to(dev), **args, mask=None if mask is None else mask.to(dev), scaling=scaling, weights=w).cpu()
    want_w = None if w is None else w0.double()
    tol_w = None if w is None else torch.zeros_like(want_w)
    for i, n in enumerate(p.lengths):
        k, v = p.rows(i, n)
        row = None if mask is None else mask[i if mask.shape[0] > 1 else 0].reshape(-1)[:n].double()
        if absent is not None:
            row = (torch.zeros(n, dtype=torch.float64) if row is None else row).masked_fill(absent[i][:n], -math.inf)
        o, pr, to, tp = attend(q[i], k, v, scale, row, p.dtype)
        off = (out[i].double() - o).abs()
        assert bool((off <= to).all()), f"sequence {i} of length {n}: off by {float((off - to).max()):.3g} more than {float(to.max()):.3g}"
        if w is not None:
            # each run adds the group's probabilities: group + 1 roundings of numbers up to the running sum
            for _ in range(runs):
                add = pr.view(kvh, group, n).sum(1)
                want_w[i, :, :n] += add
                tol_w[i, :, :n] += tp.view(kvh, group, n).sum(1) + (group + 1) * HALF[torch.float32] * (add + want_w[i, :, :n])
    if w is not None:
        off = (w.cpu().double() - want_w).abs()
        assert bool((off <= tol_w).all()), f"weights off by {float((off - tol_w).max()):.3g}"
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_at_every_edge_length(dev, fmt, dim, dtype):
    p = Pool(gen(4), EDGES, 2, dim, 16, fmt, dtype)
    check_decode(dev, p, 4, 5)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 15, 16, 17, 33])
@pytest.mark.parametrize("fmt", [None, "mxint8"])
def test_decode_head_layouts(dev, group, fmt):
    p = Pool(gen(6), [3, 70, 200], 3, 64 if fmt else 128, 32, fmt, torch.bfloat16, extra_slots=10, strided=True)
    check_decode(dev, p, group, 7, weights=True)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 4096])
def test_decode_page_sizes(dev, page):
    p = Pool(gen(8), [1, 129, 500], 1, 128, page, "mxfp8_e4m3", torch.bfloat16)
    check_decode(dev, p, 4, 9, weights=True)


def test_decode_many_short_sequences(dev):
    """more sequences than a work-group has threads, more than the launch has shares; some empty"""
    g = gen(65)
    n = 700
    k, v = (torch.randn(n, 1, 16, 64, generator=g).bfloat16() for _ in range(2))
    table = torch.randperm(n, generator=g).to(torch.int32).view(n, 1)
    lengths = torch.randint(0, 17, (n,), generator=g).to(torch.int32)
    q = torch.randn(n, 4, 64, generator=g).bfloat16()
    w = torch.zeros(n, 1, 16, device=dev)
    out = F().paged_attention_decode(q.to(dev), k.to(dev), v.to(dev), table.to(dev), lengths.to(dev), 16, weights=w).cpu().double()
    rows = torch.arange(16) < lengths[:, None]
    kk, vv = k[table[:, 0].long(), 0].double(), v[table[:, 0].long(), 0].double()
    x = torch.where(rows[:, None], q.double() @ kk.transpose(1, 2) / 8, -math.inf)
    p = torch.where(lengths[:, None, None] > 0, torch.softmax(x, -1), 0.0)
    want = p @ vv
    # fp32 statistics (1e-5 covers them at 16 slots and scores below 10) and one rounding
    assert bool(((out - want).abs() <= HALF[torch.bfloat16] * want.abs() + 1e-5 * (p @ vv.abs()) + 1e-30).all())
    assert bool(((w[:, 0].cpu().double() - p.sum(1)).abs() <= 1e-5 * 4).all()) and not bool(out[lengths == 0].any())


@pytest.mark.parametrize("fmt", [None, "mxfp4"])
def test_decode_splits_one_long_sequence_and_joins(dev, fmt):
    p = Pool(gen(10), [40001], 1, 128, 256, fmt, torch.bfloat16)
    check_decode(dev, p, 4, 11, weights=True, runs=2)
    check_decode(dev, p, 1, 12)


def test_decode_without_weights_equals_decode_with(dev):
    p = Pool(gen(13), [700, 3000], 2, 64, 64, None, torch.float16)
    assert_bits_equal(check_decode(dev, p, 4, 14), check_decode(dev, p, 4, 14, weights=True))


@pytest.mark.parametrize("mask_dtype", ["own", torch.float32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_masks(dev, dtype, mask_dtype):
    """biases, the type's lowest value, -inf (over slots that hold NaN and infinities), rows that keep nothing"""
    g = gen(15)
    lengths = [90, 64, 33, 50, 40, 1]
    p = Pool(g, lengths, 2, 64, 16, None, dtype)
    mt = dtype if mask_dtype == "own" else mask_dtype
    mask = torch.randn(len(lengths), 1, 1, p.max_length + 4, generator=g).to(mt)
    low = torch.finfo(mt).min
    mask[0, ..., :20] = low
    mask[1, ..., :] = low                      # nothing but the lowest value: every slot counts the same
    mask[2, ..., :] = -math.inf                # nothing at all
    mask[3, ..., 10:30] = -math.inf
    mask[4, ..., ::2] = -math.inf
    mask[5, ..., 0] = -math.inf
    for t in (list(range(10, 30)), []):
        for s in t:
            pg, at = int(p.table[3, s // 16]), s % 16
            p.k[pg, :, at] = math.nan if s % 2 else math.inf
            p.v[pg, :, at] = -math.inf if s % 3 else math.nan
    # lowest values: x = s + lowest rounds to lowest in fp32, so the sum forgets s (the plain form must too)
    q_mask = mask.clone()
    out = check_decode_lowest(dev, p, 2, 16, q_mask, 1)
    assert not bool(out[2].any()) and not bool(out[5].any())


def check_decode_lowest(dev, p, group, seed, mask, lowest_row):
    """check_decode, with the row of lowest values held to the mean of the values (fp32 absorbs the scores)"""
    b = len(p.lengths)
    q = torch.randn(b, p.heads * group, p.dim, generator=gen(seed)).to(p.dtype)
    w = torch.zeros(b, p.heads, p.table.shape[1] * p.page, device=dev)
    out = F().paged_attention_decode(q.to(dev), **p.to(dev), lengths=i32(p.lengths, dev), max_length=p.max_length, mask=mask.to(dev), weights=w).cpu()
    for i, n in enumerate(p.lengths):
        k, v = p.rows(i, n)
        row = mask[i, 0, 0, :n].double()
        if i == lowest_row and torch.finfo(mask.dtype).min < -1e30:
            row, k = torch.zeros_like(row), torch.zeros_like(k)
        elif i != lowest_row and bool((row == torch.finfo(mask.dtype).min).any()):
            row = row.masked_fill(row == torch.finfo(mask.dtype).min, -math.inf)  # next to others: nothing left of them
        o, pr, to, tp = attend(q[i], k, v, p.dim ** -0.5, row, p.dtype)
        assert bool(((out[i].double() - o).abs() <= to).all()), (i, n)
        got = w[i, :, :n].cpu().double()
        want = pr.view(p.heads, group, n).sum(1)
        assert bool(((got - want).abs() <= tp.view(p.heads, group, n).sum(1) + (group + 1) * HALF[torch.float32] * want + 1e-30).all()), i
    return out


def test_decode_one_mask_row_for_all(dev):
    p = Pool(gen(17), [60, 128], 1, 128, 16, "mxint8", torch.bfloat16)
    check_decode(dev, p, 4, 18, mask=torch.randn(1, 128, generator=gen(19)))


@pytest.mark.parametrize("mask_dtype", ["own", torch.float32])
@pytest.mark.parametrize("n,offset,stride", [(1, 0, 1), (2, 1, 5), (3, 0, 3), (4, 3, 7), (5, 1, 6), (130, 1, 131), (257, 2, 263)])
def test_decode_mask_rows_of_any_alignment(dev, n, offset, stride, mask_dtype):
    """masks that end with the last slot, start at any element and have odd strides; short ones"""
    p = Pool(gen(60), [n, max(1, n - 1)], 2, 128, 16, "mxfp8_e5m2" if n % 2 else None, torch.bfloat16)
    mt = torch.bfloat16 if mask_dtype == "own" else mask_dtype
    flat = torch.full((offset + stride + n,), math.nan, dtype=mt)  # what lies around the rows is never added
    mask = flat.as_strided((2, n), (stride, 1), offset)
    mask.copy_(torch.randn(2, n, generator=gen(61)))
    check = flat.to(dev)
    g = gen(62)
    q = torch.randn(2, 8, 128, generator=g).bfloat16()
    w = torch.zeros(2, 2, p.table.shape[1] * 16, device=dev)
    out = F().paged_attention_decode(q.to(dev), **p.to(dev), lengths=i32(p.lengths, dev), max_length=n,
                                     mask=check.as_strided((2, n), (stride, 1), offset), weights=w).cpu()
    for i, m in enumerate(p.lengths):
        k, v = p.rows(i, m)
        o, pr, to, tp = attend(q[i], k, v, 128 ** -0.5, mask[i, :m].double(), torch.bfloat16)
        assert bool(((out[i].double() - o).abs() <= to).all())
        assert bool(((w[i, :, :m].cpu().double() - pr.view(2, 4, m).sum(1)).abs() <= tp.view(2, 4, m).sum(1) + 5 * HALF[torch.float32]).all())


@pytest.mark.parametrize("scaling", [0.0, -0.2, 3.0])
def test_decode_scalings(dev, scaling):
    p = Pool(gen(20), [200, 77], 2, 64, 16, None, torch.bfloat16)
    check_decode(dev, p, 4, 21, scaling=scaling, weights=True)


def test_decode_follows_no_page_outside_the_pool(dev):
    """wrong page numbers and lengths past the table: those slots are absent, for every reader"""
    p = Pool(gen(22), [100, 64, 40], 2, 64, 16, None, torch.bfloat16)
    absent = [torch.zeros(112, dtype=torch.bool) for _ in range(3)]
    good = p.table.clone()
    for i, at, bad in ((0, 1, -1), (0, 4, p.k.shape[0]), (1, 0, 0x7FFFFFFF), (2, 0, -0x80000000), (2, 1, 1 << 20), (2, 2, -5)):
        p.table[i, at] = bad
        absent[i][16 * at:16 * at + 16] = True
    args = p.to(dev)
    q = torch.randn(3, 4, 64, generator=gen(23)).bfloat16()
    w = torch.zeros(3, 2, p.table.shape[1] * 16, device=dev)
    out = F().paged_attention_decode(q.to(dev), **args, lengths=i32([100, 64, 1 << 30], dev), max_length=p.max_length, weights=w).cpu()
    k, v = F().paged_kv_gather(**args, lengths=i32([100, 64, 1 << 30], dev), max_length=p.max_length)
    p.table = good
    for i, n in enumerate([100, 64, 40]):
        kk, vv = p.rows(i, n)
        row = torch.zeros(n, dtype=torch.float64).masked_fill(absent[i][:n], -math.inf)
        o, pr, to, tp = attend(q[i], kk, vv, 64 ** -0.5, row, torch.bfloat16)
        if i == 2:  # its length is a lie: slots 40 .. are NaN in valid pages, and no slot below 48 is there
            continue
        assert bool(((out[i].double() - o).abs() <= to).all())
        assert not bool(k[i, :, :n].cpu()[:, absent[i][:n]].any()) and not bool(w[i, :, :n].cpu()[:, absent[i][:n]].any())
        assert torch.equal(k[i, :, :n].cpu()[:, ~absent[i][:n]].double(), kk[:, ~absent[i][:n]])


def test_append_and_evict_write_nothing_through_bad_pages(dev):
    pool = _empty_pool(3, 1, 64, 16, None, torch.bfloat16, dev)
    before = pool["k_pages"].clone()
    table = i32([[-1, 3, 1 << 30, 1]], dev)
    x = torch.randn(1, 1, 80, 64, generator=gen(24)).bfloat16().to(dev)
    F().paged_kv_append(x, x, page_table=table, starts=i32([0], dev), **pool)
    want = before.cpu()
    want[1, 0] = x[0, 0, 48:64].cpu()
    assert_bits_equal(pool["k_pages"], want)
    F().paged_kv_append(x, x, page_table=table, starts=i32([-40], dev), **pool)   # a negative start names no slot
    F().paged_kv_append(x, x, page_table=table, starts=i32([0x7FFFFFF0], dev), **pool)
    assert_bits_equal(pool["k_pages"], want)
    w = torch.rand(1, 1, 64, generator=gen(25)).to(dev)
    pos = torch.arange(64, dtype=torch.int32, device=dev).view(1, 1, 64)
    F().paged_kv_evict(page_table=table, lengths=i32([64], dev), weights=w, positions=pos, max_length=64, keep=16, **pool)
    assert_bits_equal(pool["k_pages"], want)  # every target lies in a page that is not there


def test_decode_far_into_a_large_pool(dev):
    """rows more than 4 GiB into the pages, and slots in pages of both ends"""
    n, heads, page, dim = 70000, 4, 64, 256
    k = torch.empty((n, heads, page, dim), dtype=torch.int8, device=dev)  # 4.6 GB
    v = torch.empty_like(k)
    ks = torch.empty((n, heads, page, dim // 32), dtype=torch.uint8, device=dev)
    vs = torch.empty((n, heads, dim // 32, page), dtype=torch.uint8, device=dev)
    table = torch.tensor([[n - 1, 0, n - 2, 65536, 32768]], dtype=torch.int32)
    p = Pool(gen(26), [300], heads, dim, page, "mxint8", torch.bfloat16)
    for j in range(5):
        src, dst = int(p.table[0, j]), int(table[0, j])
        k[dst], v[dst], ks[dst], vs[dst] = (t[src].to(dev) for t in (p.k, p.v, p.ks, p.vs))
    kw = dict(kv_format="mxint8", k_scales=ks, v_scales=vs)
    q = torch.randn(1, heads * 2, dim, generator=gen(27)).bfloat16()
    out = F().paged_attention_decode(q.to(dev), k, v, table.to(dev), i32([300], dev), 300, **kw).cpu()
    kk, vv = p.rows(0, 300)
    o, _, to, _ = attend(q[0], kk, vv, dim ** -0.5, None, torch.bfloat16)
    assert bool(((out[0].double() - o).abs() <= to).all())
    gk, _ = F().paged_kv_gather(k, v, table.to(dev), i32([300], dev), 300, dtype=torch.bfloat16, **kw)
    assert torch.equal(gk[0].cpu().double(), kk)
    x = torch.randn(1, heads, 1, dim, generator=gen(28)).bfloat16().to(dev)
    F().paged_kv_append(x, x, k, v, table.to(dev), i32([5], dev), **kw)
    gk, _ = F().paged_kv_gather(k, v, table.to(dev), i32([300], dev), 6, dtype=torch.bfloat16, **kw)
    from mase_amd.quantizers import mxint_quantizer

    assert torch.equal(gk[0, :, 5], mxint_quantizer(x, 32, 8)[0, :, 0])


# ---------------------------------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------------------------------
def _run_evict(dev, p, w, pos, keep, recent, first, max_length=None):
    kw = p.to(dev)
    nw, npos, nlen = F().paged_kv_evict(**kw, lengths=i32(p.lengths, dev), weights=w.to(dev), positions=pos.to(dev),
                                        max_length=p.max_length if max_length is None else max_length, keep=keep, recent=recent, first=first)
    return kw, nw.cpu(), npos.cpu(), nlen.cpu()


def check_evict(dev, p, w, pos, keep, recent, first):
    kw, nw, npos, nlen = _run_evict(dev, p, w, pos, keep, recent, first)
    assert nlen.tolist() == [min(n, keep) for n in p.lengths]
    want = {n: getattr(p, a).clone() for n, a in (("k_pages", "k"), ("v_pages", "v"), ("k_scales", "ks"), ("v_scales", "vs")) if getattr(p, a) is not None}
    for b, n in enumerate(p.lengths):
        for h in range(p.heads):
            src = evict(pos[b, h].tolist(), w[b, h].tolist(), n, keep, recent, first)
            m = len(src)
            assert npos[b, h, :m].tolist() == pos[b, h, src].tolist(), (b, h)
            assert_bits_equal(nw[b, h, :m], w[b, h, src])
            assert not bool(nw[b, h, m:].any()) and bool((npos[b, h, m:] == -1).all())
            for to, s in enumerate(src):
                if s == to:
                    continue
                pt, at, pf, af = int(p.table[b, to // p.page]), to % p.page, int(p.table[b, s // p.page]), s % p.page
                want["k_pages"][pt, h, at], want["v_pages"][pt, h, at] = p.k[pf, h, af], p.v[pf, h, af]
                if p.ks is not None:
                    want["k_scales"][pt, h, at], want["v_scales"][pt, h, :, at] = p.ks[pf, h, af], p.vs[pf, h, :, af]
    for name, t in want.items():  # all of the pool: what is not a target stays as it was
        got = kw[name].cpu().contiguous()
        assert torch.equal(bits(got) if p.ks is None else got, bits(t) if p.ks is None else t), name


@pytest.mark.parametrize("keep,recent,first", [(1, 0, 0), (1, 1, 0), (16, 4, 2), (33, 33, 0), (33, 0, 33), (64, 10, 10), (130, 1, 1), (400, 5, 5)])
@pytest.mark.parametrize("fmt", [None, "mxint8", "mxfp4"])
def test_evict_keeps_protected_then_heaviest(dev, fmt, keep, recent, first):
    g = gen(30)
    lengths = [0, 1, 17, 64, 65, 257, 300]
    p = Pool(g, lengths, 2, 64, 16, fmt, torch.bfloat16, strided=True)
    cap = p.table.shape[1] * 16
    w = torch.rand(len(lengths), 2, cap, generator=g).mul_(4).round_().div_(4)  # many ties
    w[:, 0] = torch.rand(len(lengths), cap, generator=g)
    pos = torch.stack([torch.stack([torch.randperm(2 * cap, generator=g)[:cap] for _ in range(2)]) for _ in lengths]).to(torch.int32)
    check_evict(dev, p, w, pos, keep, recent, first)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("fmt", FORMATS)
def test_evict_moves_whole_rows_of_every_format(dev, fmt, dim):
    g = gen(31)
    p = Pool(g, [100, 31], 3, dim, 32, fmt, torch.float16, strided=True)
    cap = p.table.shape[1] * 32
    check_evict(dev, p, torch.rand(2, 3, cap, generator=g), torch.arange(cap, dtype=torch.int32).expand(2, 3, cap).contiguous(), 30, 7, 3)


def test_evict_orders_odd_weights(dev):
    """NaN below every weight, infinities and both zeros in place, all weights alike, more protected ones than places"""
    g = gen(32)
    p = Pool(g, [200] * 4, 1, 64, 16, None, torch.bfloat16)
    cap = p.table.shape[1] * 16
    w = torch.rand(4, 1, cap, generator=g) - 0.5
    w[0, 0, ::3], w[0, 0, 1::9], w[0, 0, 5::50], w[0, 0, 7::50] = 0.0, -0.0, math.inf, -math.inf
    w[1, 0, ::2] = math.nan
    w[2] = 1.0
    pos = torch.arange(cap, dtype=torch.int32).expand(4, 1, cap).clone()
    pos[3] = 5  # every slot at one position: all of them recent
    check_evict(dev, p, w, pos, 90, 3, 1)
    w[1] = math.nan
    check_evict(dev, p, w, pos, 101, 0, 0)


def test_evict_to_more_than_there_is_copies_what_there_is(dev):
    p = Pool(gen(63), [30, 64], 2, 64, 16, None, torch.bfloat16)
    cap = p.table.shape[1] * 16
    w, pos = torch.rand(2, 2, cap, generator=gen(64)), torch.arange(cap, dtype=torch.int32).expand(2, 2, cap).contiguous()
    for keep, recent in ((64, 64), (1 << 30, 1 << 29)):  # the second would take 32 GB to list moves that cannot be
        kw, nw, npos, nlen = _run_evict(dev, p, w, pos, keep, recent, 5 if keep > 64 else 0)
        assert nlen.tolist() == [30, 64] and torch.equal(nw[1], w[1]) and torch.equal(npos[0, :, :30], pos[0, :, :30])
        assert not bool(nw[0, :, 30:].any()) and bool((npos[0, :, 30:] == -1).all())
        assert_bits_equal(kw["k_pages"], p.k)


@pytest.mark.parametrize("n,keep", [(5000, 4096), (70001, 35000), (33000, 100)])
def test_evict_long_rows(dev, n, keep):
    """the same choice by torch's stable sort"""
    g = gen(33)
    cap = -(-n // 256) * 256
    k = torch.randint(-128, 128, (cap // 256, 2, 256, 64), generator=g).to(torch.int8)
    s = torch.randint(100, 140, (cap // 256, 2, 256, 2), generator=g).to(torch.uint8)
    vs = s.transpose(2, 3).contiguous()
    table = torch.randperm(cap // 256, generator=g).to(torch.int32).view(1, -1)
    w = torch.rand(1, 2, cap, generator=g).mul_(1000).floor_()
    w[0, 0, : n // 3] = 0
    pos = torch.arange(cap, dtype=torch.int32).expand(1, 2, cap).contiguous()
    kd, vd, ksd, vsd = k.to(dev), k.to(dev), s.to(dev), vs.to(dev)
    nw, npos, nlen = F().paged_kv_evict(kd, vd, table.to(dev), i32([n], dev), w.to(dev), pos.to(dev), n, keep, recent=50, first=4,
                                        kv_format="mxint8", k_scales=ksd, v_scales=vsd)
    assert nlen.tolist() == [keep]
    flat = lambda t: t[table[0].long()].transpose(0, 1).flatten(1, 2)  # noqa: E731  [heads, slots, ...]
    for h in range(2):
        rank = w[0, h, :n].clone()
        rank[:4] = math.inf
        rank[n - 50:] = math.inf
        kept = torch.sort(rank, descending=True, stable=True).indices[:keep].sort().values
        src = torch.arange(keep)
        free = torch.ones(keep, dtype=torch.bool)
        free[kept[kept < keep]] = False
        src[free] = kept[kept >= keep]
        assert torch.equal(npos[0, h, :keep].cpu().long(), src)
        assert torch.equal(nw[0, h, :keep].cpu(), w[0, h, src]) and not bool(nw[0, h, keep:].any())
        assert torch.equal(flat(kd.cpu())[h, :keep], flat(k)[h, src]) and torch.equal(flat(vd.cpu())[h, :keep], flat(k)[h, src])
        assert torch.equal(flat(ksd.cpu())[h, :keep], flat(s)[h, src])
        assert torch.equal(flat(vsd.transpose(2, 3).cpu())[h, :keep], flat(s)[h, src])
        assert torch.equal(flat(kd.cpu())[h, keep:], flat(k)[h, keep:])


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_functions_run_on_the_current_stream(dev):
    p = Pool(gen(40), [900, 300], 2, 128, 64, "mxint8", torch.bfloat16)
    kw = p.to(dev)
    lengths = i32(p.lengths, dev)
    q = torch.randn(2, 8, 128, generator=gen(41)).bfloat16().to(dev)
    want = F().paged_attention_decode(q, **kw, lengths=lengths, max_length=900)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    with torch.cuda.stream(side):
        a = torch.randn(4096, 4096, device=dev)
        for _ in range(20):
            a = a @ a * 1e-4        # keeps the stream busy: a launch on another stream would read zeros
        late.copy_(q)
        got = F().paged_attention_decode(late, **kw, lengths=lengths, max_length=900)
    side.synchronize()
    assert_bits_equal(got, want)


def test_calls_on_two_streams_do_not_meet(dev):
    """two pools worked on at the same time from two streams: the results of one after the other"""
    jobs = []
    for i, (lengths, fmt) in enumerate((([3000, 500], "mxint8"), ([2500, 2600], "mxfp4"))):
        p = Pool(gen(66 + i), lengths, 2, 64, 64, fmt, torch.bfloat16)
        jobs.append(dict(kw=p.to(dev), n=i32(lengths, dev), top=max(lengths), q=torch.randn(2, 8, 64, generator=gen(68 + i)).bfloat16().to(dev),
                         pos=torch.arange(p.table.shape[1] * 64, dtype=torch.int32, device=dev).expand(2, 2, -1).contiguous()))

    def work(j):
        w = torch.zeros(2, 2, j["pos"].shape[2], device=dev)
        kw = {k: v.clone() if torch.is_tensor(v) else v for k, v in j["kw"].items()}
        outs = [F().paged_attention_decode(j["q"], **kw, lengths=j["n"], max_length=j["top"], weights=w) for _ in range(5)]
        w2, pos, n = F().paged_kv_evict(**kw, lengths=j["n"], weights=w, positions=j["pos"], max_length=j["top"], keep=400, recent=9)
        outs.append(F().paged_attention_decode(j["q"], **kw, lengths=n, max_length=400, weights=w2))
        return outs + [w2, pos, kw["k_pages"], kw["v_pages"]]

    want = [work(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for s, j in zip(streams, jobs):
        with torch.cuda.stream(s):
            got.append(work(j))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x, y.view(torch.int16) if y.dtype == torch.bfloat16 else y)


@pytest.mark.parametrize("fmt", [None, "mxfp8_e5m2"])
def test_a_step_replays_from_two_graphs(dev, fmt):
    """append + decode with weights captured at two batch layouts; lengths move on inside the graph; replays alternate with
    eager work and equal the eager steps"""
    g = gen(42)
    state = []
    for lengths in ([5, 140], [60, 200]):
        p = Pool(g, lengths, 2, 64, 16, fmt, torch.bfloat16, extra_slots=40)
        kw, ew = p.to(dev), p.to(dev)
        st = dict(p=p, x=torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, device=dev), q=torch.zeros(2, 8, 64, dtype=torch.bfloat16, device=dev))
        for name, pool in (("graph", kw), ("eager", ew)):
            st[name] = dict(pool=pool, n=i32(lengths, dev), w=torch.zeros(2, 2, p.table.shape[1] * 16, device=dev))
        state.append(st)

    def step(st, side):
        d = st[side]
        F().paged_kv_append(st["x"], st["x"], starts=d["n"], **d["pool"])
        d["n"] += 1
        return F().paged_attention_decode(st["q"], **d["pool"], lengths=d["n"], max_length=st["p"].max_length, weights=d["w"])

    graphs = []
    warm = torch.cuda.Stream()
    for st in state:
        saved = {k: v.clone() for k, v in st["graph"]["pool"].items() if torch.is_tensor(v)}
        n0 = st["graph"]["n"].clone()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            step(st, "graph")
        torch.cuda.current_stream().wait_stream(warm)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            st["out"] = step(st, "graph")
        for k, v in saved.items():
            st["graph"]["pool"][k].copy_(v)
        st["graph"]["n"].copy_(n0)
        st["graph"]["w"].zero_()
        graphs.append(gr)
    for _ in range(4):
        for st in state:
            st["x"].copy_(torch.randn(st["x"].shape, generator=g).bfloat16())
            st["q"].copy_(torch.randn(st["q"].shape, generator=g).bfloat16())
        for gr in graphs:
            gr.replay()
        for st in state:
            want = step(st, "eager")
            torch.cuda.synchronize()
            assert_bits_equal(st["out"], want)
            assert torch.equal(st["graph"]["w"], st["eager"]["w"]) and torch.equal(st["graph"]["n"], st["eager"]["n"])


def test_evict_replays_from_a_graph(dev):
    g = gen(43)
    p = Pool(g, [300, 90], 2, 64, 16, None, torch.bfloat16)
    cap = p.table.shape[1] * 16
    kw = p.to(dev)
    k0, v0 = kw["k_pages"].clone(), kw["v_pages"].clone()
    w = torch.zeros(2, 2, cap, device=dev)
    pos = torch.arange(cap, dtype=torch.int32, device=dev).expand(2, 2, cap).contiguous()
    lengths = i32(p.lengths, dev)
    run = lambda: F().paged_kv_evict(**kw, lengths=lengths, weights=w, positions=pos, max_length=300, keep=64, recent=8, first=2)  # noqa: E731
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run()
    torch.cuda.current_stream().wait_stream(warm)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = run()
    for _ in range(3):
        w.copy_(torch.rand(w.shape, generator=g))
        got = []
        for replay in (True, False):
            kw["k_pages"].copy_(k0)
            kw["v_pages"].copy_(v0)
            res = (gr.replay(), out)[1] if replay else run()
            torch.cuda.synchronize()
            got.append([t.clone() for t in res] + [kw["k_pages"].clone(), kw["v_pages"].clone()])
        for a, b in zip(*got):
            assert torch.equal(a.view(torch.int16) if a.is_floating_point() else a, b.view(torch.int16) if b.is_floating_point() else b)


def test_functions_refuse_what_they_do_not_take(dev):
    from mase_amd._lib import MaseAmdError

    p = Pool(gen(44), [20, 30], 2, 64, 16, "mxint8", torch.bfloat16)
    kw = p.to(dev)
    n = i32(p.lengths, dev)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    dec = lambda query=q, lengths=n, max_length=30, **k: F().paged_attention_decode(query, **{**kw, **k.pop("pool", {})}, lengths=lengths, max_length=max_length, **k)  # noqa: E731
    dec()
    for bad in (dict(query=q[:1]), dict(query=q[:, :3]), dict(query=q[..., :32]), dict(query=q.float()), dict(lengths=n.long()),
                dict(lengths=n[:1]), dict(max_length=33), dict(max_length=-1), dict(mask=torch.zeros(2, 29, device=dev)),
                dict(mask=torch.zeros(3, 30, device=dev)), dict(mask=torch.zeros(2, 4, 30, device=dev)), dict(mask=torch.zeros(2, 30, dtype=torch.float64, device=dev)),
                dict(mask=torch.zeros(2, 30, dtype=torch.float16, device=dev)), dict(mask=torch.zeros(2, 30)),
                dict(weights=torch.zeros(2, 2, 29, device=dev)), dict(weights=torch.zeros(2, 2, 32, dtype=torch.bfloat16, device=dev)),
                dict(weights=torch.zeros(2, 1, 32, device=dev).expand(2, 2, 32)), dict(weights=torch.zeros(1, 2, 32, device=dev).expand(2, 2, 32)),
                dict(pool=dict(k_scales=None)), dict(pool=dict(k_scales=kw["v_scales"])), dict(pool=dict(kv_format=None)), dict(pool=dict(kv_format="mxfp4")),
                dict(pool=dict(k_pages=kw["k_pages"][:, :, :8])), dict(pool=dict(v_pages=kw["v_pages"][:1])),
                dict(pool=dict(page_table=kw["page_table"].long())), dict(pool=dict(page_table=kw["page_table"][:1].expand(2, -1))),
                dict(pool=dict(k_pages=kw["k_pages"][:1].expand_as(kw["k_pages"]))), dict(pool=dict(v_pages=kw["v_pages"][:, :1].expand_as(kw["v_pages"]))),
                dict(pool=dict(page_table=kw["page_table"].cpu()))):
        with pytest.raises(ValueError):
            dec(**bad)
    with pytest.raises(MaseAmdError, match="gradient"):
        dec(query=q.clone().requires_grad_())
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16, device=dev)
    app = lambda key=x, value=x, starts=n, **k: F().paged_kv_append(key, value, starts=starts, **kw, **k)  # noqa: E731
    for bad in (dict(key=x[:1]), dict(value=x[:, :, :2]), dict(value=x.half()), dict(key=x.float(), value=x.float()), dict(starts=n.cpu()),
                dict(counts=n[:1]), dict(positions=torch.zeros(2, 2, 31, dtype=torch.int32, device=dev)), dict(first_positions=n),
                dict(positions=torch.zeros(2, 2, 32, device=dev)), dict(key=x.cpu(), value=x.cpu())):
        with pytest.raises(ValueError):
            app(**bad)
    w, pos = torch.zeros(2, 2, 32, device=dev), torch.zeros(2, 2, 32, dtype=torch.int32, device=dev)
    ev = lambda weights=w, positions=pos, max_length=30, keep=8, **k: F().paged_kv_evict(**kw, lengths=n, weights=weights, positions=positions, max_length=max_length, keep=keep, **k)  # noqa: E731
    for bad in (dict(keep=0), dict(recent=9), dict(recent=-1), dict(first=5, recent=4), dict(max_length=33), dict(weights=w[..., :29]),
                dict(positions=pos[..., :31]), dict(weights=w.double()), dict(positions=pos.long())):
        with pytest.raises(ValueError):
            ev(**bad)
    with pytest.raises(ValueError):
        F().paged_kv_gather(**kw, lengths=n, max_length=30)  # codes need a type to be read as
    with pytest.raises(ValueError):
        F().paged_kv_gather(**kw, lengths=n, max_length=-1, dtype=torch.bfloat16)


def test_empty_calls(dev):
    p = Pool(gen(45), [0, 0], 2, 64, 16, None, torch.bfloat16)
    kw, n = p.to(dev), i32([0, 0], dev)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    w = torch.full((2, 2, 16), 3.0, device=dev)
    assert not bool(F().paged_attention_decode(q, **kw, lengths=n, max_length=0).any())
    assert not bool(F().paged_attention_decode(q, **kw, lengths=n, max_length=16, weights=w).any()) and bool((w == 3).all())
    assert F().paged_kv_gather(**kw, lengths=n, max_length=0)[0].shape == (2, 2, 0, 64)
    F().paged_kv_append(torch.zeros(2, 2, 0, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 2, 0, 64, dtype=torch.bfloat16, device=dev), starts=n, **kw)
    none = dict(kw, page_table=kw["page_table"][:0])
    assert F().paged_attention_decode(q[:0], **none, lengths=n[:0], max_length=16).shape == (0, 4, 64)


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
def test_prompt_steps_eviction_and_more_steps(dev, fmt):
    """a prompt, decoding steps that add up weights, an eviction, further steps over what is left: the cache object against
    a dense simulation of the same (keys and values as the cache reads them back)"""
    from mase_amd.quantized import PagedKVCache

    g = gen(50)
    B, H, G, D, dtype = 2, 2, 2, 64, torch.bfloat16
    c = PagedKVCache(B, H, D, 120, num_layers=2, page_size=16, num_pages=14, kv_format=fmt, dtype=dtype, device=dev, track_weights=True)
    prompt = torch.randn(2, 2, B, H, 50, D, generator=g).to(dtype).to(dev)
    sim = []   # per layer: per sequence: dict(k, v [H, n, D], pos, w [H, n])
    for layer in range(2):
        c.append(prompt[layer, 0], prompt[layer, 1], layer, counts=[50, 37])
        k, v = c.gather(layer)
        sim.append([dict(k=k[b, :, :n].double().cpu(), v=v[b, :, :n].double().cpu(), pos=torch.arange(n).expand(H, n).clone(),
                         w=torch.zeros(H, n, dtype=torch.float64)) for b, n in enumerate([50, 37])])
    assert c.lengths() == [50, 37] and c.get_seq_length() == 50

    def steps(count, seen):
        for s in range(count):
            for layer in range(2):
                kv = torch.randn(2, B, H, 1, D, generator=g).to(dtype)
                q = torch.randn(B, H * G, D, generator=g).to(dtype)
                k, v = c.update(kv[0].to(dev), kv[1].to(dev), layer)
                out = c.attend(q.to(dev), layer).cpu().double()
                w = c.weights(layer).cpu().double()
                for b in range(B):
                    d = sim[layer][b]
                    n = d["k"].shape[1] + 1
                    d["k"] = torch.cat((d["k"], k[b, :, n - 1:n].double().cpu()), 1)
                    d["v"] = torch.cat((d["v"], v[b, :, n - 1:n].double().cpu()), 1)
                    d["pos"] = torch.cat((d["pos"], torch.full((H, 1), seen[b] + s)), 1)
                    assert torch.equal(k[b, :, :n].double().cpu(), d["k"]) and torch.equal(v[b, :, :n].double().cpu(), d["v"])
                    assert torch.equal(c.positions(layer)[b, :, :n].cpu().long(), d["pos"])
                    o, pr, to, tp = attend(q[b], d["k"], d["v"], D ** -0.5, None, dtype)
                    assert bool(((out[b] - o).abs() <= to).all())
                    d["w"] = torch.cat((d["w"], torch.zeros(H, 1, dtype=torch.float64)), 1) + pr.view(H, G, n).sum(1)
                    assert bool(((w[b, :, :n] - d["w"]).abs() <= 1e-5).all())
                    d["w"] = w[b, :, :n].clone()  # go on from the same numbers, so that the eviction sorts the same ones

    steps(5, [50, 37])
    assert c.lengths(1) == [55, 42]
    used = len(c._free)
    c.evict(40, recent=6, first=2)
    assert c.lengths(0) == [40, 40] and c.lengths(1) == [40, 40] and len(c._free) == used + 1  # 4 + 3 pages before, 3 + 3 after
    for layer in range(2):
        for b in range(B):
            d = sim[layer][b]
            for h in range(H):
                src = evict(d["pos"][h].tolist(), d["w"][h].tolist(), d["k"].shape[1], 40, 6, 2)
                for name in ("k", "v", "pos", "w"):
                    d[name][h, :40] = d[name][h, src].clone()
            for name in ("k", "v", "pos", "w"):
                d[name] = d[name][:, :40]
    steps(4, [55, 42])
    assert c.get_seq_length() == 59
    c.reset()
    assert c.lengths() == [0, 0] and len(c._free) == 14
