"""Attention masks on a PagedKVCache whose slots are no longer its positions: left-padded batches after an eviction, chunks
of several tokens after one, and sequences of different lengths, through the modules and through ``attend``."""
import math

import pytest
import torch

from helpers import assert_bits_equal
from paged_reference import HALF, attend
from test_paged_attention_modules_gpu import E4M3, INT8, MINI, build, tables

pytestmark = pytest.mark.gpu

DTYPE = torch.bfloat16
LOW = torch.finfo(DTYPE).min
OFF = {"bypass": True}
PADS = (7, 0)


def module(dev, kind="mxint", quantized=False, fmt=None):
    """an attention module whose output is the heads' (no output projection); quantized: the scores, so that every step is dense"""
    import mase_amd.quantized as Q

    quant = INT8 if kind == "mxint" else E4M3
    qc = {"qk_matmul": quant, "av_matmul": OFF, "rope": MINI, "softmax": MINI, "kv_cache": quant} if quantized else {
        "qk_matmul": OFF, "av_matmul": OFF, "rope": OFF, "softmax": OFF, "kv_cache": OFF if fmt is None else quant}
    m = build(Q.LlamaAttentionMXInt if kind == "mxint" else Q.LlamaAttentionMXFP, dev, DTYPE, qc, layer=0)
    m.o_proj = torch.nn.Identity()
    return m


def position_mask(tokens, total, dev, pads=PADS):
    """[2, 1, tokens, total]: causal by position, the first pads[b] positions hidden"""
    at = torch.arange(total)
    m = torch.zeros(2, 1, tokens, total, dtype=DTYPE)
    for t in range(tokens):
        m[:, 0, t, at > total - tokens + t] = LOW
    for b, p in enumerate(pads):
        m[b, :, :, :p] = LOW
    return m.to(dev)


def run(dev, m, cache, seed, chunk, pad_seed=None, last_seed=None):
    """a left-padded prompt of 20, four decoding steps, an eviction to 16 (a few padding slots among the protected ones), then
    a step of `chunk` tokens, an eviction to 14 and another such step, every step with its mask over positions"""
    g = torch.Generator().manual_seed(seed)
    outs = []

    def step(n, seen):
        x = torch.randn(2, n, 256, generator=g).to(DTYPE)
        if pad_seed is not None and seen == 0:
            x[0, :PADS[0]] = torch.randn(PADS[0], 256, generator=torch.Generator().manual_seed(pad_seed)).to(DTYPE)
        if last_seed is not None and n > 1 and seen:
            x[:, -1] = torch.randn(2, 256, generator=torch.Generator().manual_seed(last_seed)).to(DTYPE)
        x = x.to(dev)
        cos_sin, mask = tables(n, 64, seen, dev, DTYPE), position_mask(n, seen + n, dev)
        with torch.no_grad():
            y, w = m(x, cos_sin, mask, past_key_value=cache)
        outs.append(dict(x=x, cos_sin=cos_sin, mask=mask, y=y, w=w, n=n))

    step(20, 0)
    for s in range(4):
        step(1, 20 + s)
    cache.evict(16, recent=5, first=4)
    step(chunk, 24)
    yield outs
    cache.evict(14, recent=5, first=2)
    step(chunk, 24 + chunk)
    yield outs


def make(dev, fmt=None):
    from mase_amd.quantized import PagedKVCache

    return PagedKVCache(2, 4, 64, 64, page_size=16, kv_format=fmt, dtype=DTYPE, device=dev, track_weights=True)


def queries(m, o):
    """the module's own query states of a step [2, heads, tokens, 64]"""
    from mase_amd.quantized.modules.llama import apply_rotary_pos_emb

    with torch.no_grad():
        q, k, _ = m._project(o["x"], (2, o["n"], -1, 64))
        return apply_rotary_pos_emb(q, k, *o["cos_sin"])[0]


def check_step(m, cache, o):
    """a step against 64 bits: each slot hidden or not by the position that its token stood at"""
    q = queries(m, o).cpu()
    k, v = (t.double().cpu() for t in cache.gather(0))
    pos, mask = cache.positions(0).cpu(), o["mask"].double().cpu()
    got = o["y"].view(2, o["n"], 8, 64).double().cpu()
    half = HALF[DTYPE]
    for b in range(2):
        n = cache.lengths(0)[b]
        for hk in range(4):
            for t in range(o["n"]):
                row = mask[b, 0, t, pos[b, hk, :n].long()]
                row = row.masked_fill(row < -1e30, -math.inf)
                qq, kk, vv = q[b, 2 * hk:2 * hk + 2, t], k[b, hk:hk + 1, :n], v[b, hk:hk + 1, :n]
                want, p, tol, _ = attend(qq, kk, vv, m.scaling, row, DTYPE)
                if o["n"] > 1:
                    # the dense chain rounds scores twice (products, scaling), the probabilities and the result
                    x = (qq.double() @ kk[0].T).abs().max() * m.scaling
                    rel = math.expm1(2 * 2.1 * half * float(x)) + half
                    tol = tol + (p @ vv[0].abs()) * rel * (1 + half)
                off = (got[b, t, 2 * hk:2 * hk + 2] - want).abs()
                assert bool((off <= tol).all()), (b, hk, t, float((off - tol).max()))


@pytest.mark.parametrize("chunk", [1, 2, 5])
@pytest.mark.parametrize("kind,fmt", [("mxint", None), ("mxint", "mxint8"), ("mxfp", "mxfp8_e4m3")])
def test_masks_over_positions_after_evictions(dev, kind, fmt, chunk):
    m, cache = module(dev, kind, fmt=fmt), make(dev, fmt)
    for outs in run(dev, m, cache, 70, chunk):
        check_step(m, cache, outs[-1])
    assert cache.lengths(0) == [14 + chunk] * 2 and cache.get_seq_length(0) == 24 + 2 * chunk


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("chunk", [1, 4])
def test_padding_stays_hidden_after_evictions(dev, chunk, quantized):
    """what the padding held changes nothing, to the last bit"""
    m = module(dev, quantized=quantized)
    a, b = (list(run(dev, m, make(dev), 71, chunk, pad_seed=s))[-1] for s in (1, 2))
    assert len(a) == 7
    for x, y in zip(a[1:], b[1:]):
        assert_bits_equal(x["y"], y["y"])


@pytest.mark.parametrize("quantized", [False, True])
def test_tokens_of_a_chunk_see_no_later_ones_after_an_eviction(dev, quantized):
    m = module(dev, quantized=quantized)
    a, b = (next(iter(run(dev, m, make(dev), 72, 4, last_seed=s))) for s in (1, 2))
    assert_bits_equal(a[-1]["y"][:, :3], b[-1]["y"][:, :3])
    assert not torch.equal(a[-1]["y"][:, 3], b[-1]["y"][:, 3])


@pytest.mark.parametrize("most", [65535, 4, 1])
def test_attend_takes_its_mask_by_positions(dev, most, monkeypatch):
    """the cache's own method: unequal lengths, an eviction, biases by position, weights; more cached heads of sequences than
    one call takes"""
    from mase_amd.quantized import PagedKVCache

    monkeypatch.setattr(PagedKVCache, "_most_sequences", most)
    g = torch.Generator().manual_seed(73)
    c = PagedKVCache(3, 2, 64, 80, page_size=16, kv_format="mxint8", dtype=DTYPE, device=dev, track_weights=True)
    kv = torch.randn(2, 3, 2, 40, 64, generator=g).to(DTYPE).to(dev)
    c.append(kv[0], kv[1], counts=[40, 12, 33])
    for _ in range(2):
        c.attend(torch.randn(3, 6, 64, generator=g).to(DTYPE).to(dev))
    c.evict(17, recent=3, first=1)
    c.append(kv[0][:, :, :2], kv[1][:, :, :2])
    assert c.lengths() == [19, 14, 19]
    q = torch.randn(3, 6, 64, generator=g).to(DTYPE)
    before = c.weights(0).cpu().double()
    for shape, mt in (((3, 42), torch.float32), ((1, 1, 1, 50), DTYPE)):
        mask = torch.randn(shape, generator=g).to(mt)
        mask[..., 5:20] = -math.inf
        out = c.attend(q.to(dev), mask=mask.to(dev)).cpu().double()
        k, v = (t.double().cpu() for t in c.gather())
        pos, after = c.positions(0).cpu().long(), c.weights(0).cpu().double()
        for b, n in enumerate(c.lengths()):
            row = mask.reshape(mask.shape[0], -1)[b if mask.shape[0] > 1 else 0].double()
            for h in range(2):
                want, p, tol, tol_p = attend(q[b, 3 * h:3 * h + 3], k[b, h:h + 1, :n], v[b, h:h + 1, :n], 64 ** -0.5, row[pos[b, h, :n]], DTYPE)
                assert bool(((out[b, 3 * h:3 * h + 3] - want).abs() <= tol).all()), (b, h)
                off = (after[b, h, :n] - before[b, h, :n] - p.sum(0)).abs()
                assert bool((off <= tol_p.sum(0) + 5 * HALF[torch.float32] * after[b, h, :n]).all()), (b, h)
        before = after
    for bad in (torch.zeros(3, 41), torch.zeros(2, 42), torch.zeros(3, 2, 42), torch.zeros(3, 42, dtype=torch.float64)):
        with pytest.raises(ValueError, match="mask"):
            c.attend(q.to(dev), mask=bad.to(dev))


def test_a_refused_mask_leaves_the_cache_as_it_was(dev):
    m, cache = module(dev), make(dev)
    x = torch.randn(2, 20, 256, generator=torch.Generator().manual_seed(74)).to(DTYPE).to(dev)
    with torch.no_grad():
        m(x, tables(20, 64, 0, dev, DTYPE), position_mask(20, 20, dev), past_key_value=cache)

        def refused(n, seen, mask):
            free, held = list(cache._free), cache.lengths(0)
            with pytest.raises(ValueError, match="mask"):
                m(x[:, :n], tables(n, 64, seen, dev, DTYPE), mask, past_key_value=cache)
            assert cache.lengths(0) == held and cache._free == free and cache._held_dev[0].tolist() == held

        refused(1, 20, position_mask(1, 20, dev))                    # one column too few
        cache.evict(12, recent=4)
        refused(1, 20, position_mask(1, 13, dev))                    # columns of slots, not of positions
        refused(3, 20, position_mask(3, 15, dev))
        refused(3, 20, position_mask(3, 23, dev)[:, 0])
        refused(3, 20, position_mask(3, 23, dev) == 0)
        refused(3, 20, position_mask(3, 23, dev).expand(2, 3, 3, 23))  # neither one head nor all of them
        for n in (1, 3):                                             # these fit
            m(x[:, :n], tables(n, 64, 20, dev, DTYPE), position_mask(n, cache.get_seq_length() + n, dev), past_key_value=cache)


@pytest.mark.parametrize("evicted", [False, True])
def test_dense_steps_of_unequal_sequences_see_only_their_own_slots(dev, evicted):
    """several tokens at once, without a mask, on a cache whose sequences hold different numbers of slots"""
    m, cache = module(dev), make(dev)
    kv = torch.randn(2, 2, 4, 30, 64, generator=torch.Generator().manual_seed(75)).to(DTYPE).to(dev)
    cache.append(kv[0], kv[1], counts=[30, 9])
    if evicted:
        cache.evict(14, recent=4)
    x = torch.randn(2, 2, 256, generator=torch.Generator().manual_seed(76)).to(DTYPE).to(dev)
    cos_sin = tables(2, 64, 9, dev, DTYPE)
    with torch.no_grad():
        y, _ = m(x, cos_sin, None, past_key_value=cache)
    assert cache.lengths(0) == [16 if evicted else 32, 11]
    check_step(m, cache, dict(x=x, cos_sin=cos_sin, y=y, n=2, mask=torch.zeros(2, 1, 2, 32)))


def test_masks_of_positions_are_refused_where_sequences_stand_at_different_ones(dev):
    """a column cannot be one position of all sequences for the new tokens; nothing is appended"""
    m, cache = module(dev), make(dev)
    kv = torch.randn(2, 2, 4, 30, 64, generator=torch.Generator().manual_seed(77)).to(DTYPE).to(dev)
    cache.append(kv[0], kv[1], counts=[30, 9])
    x = torch.randn(2, 3, 256, generator=torch.Generator().manual_seed(78)).to(DTYPE).to(dev)
    with torch.no_grad():
        for n in (1, 3):
            with pytest.raises(ValueError, match="mask"):
                m(x[:, :n], tables(n, 64, 30, dev, DTYPE), position_mask(n, 30 + n, dev, pads=(0, 0)), past_key_value=cache)
    assert cache.lengths(0) == [30, 9]
