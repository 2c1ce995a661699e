"""The paged cache on the host: masks over positions laid over slots, and what is refused before anything changes."""
import pytest
import torch


def cache(held, seen, positions=None, heads=2, capacity=32, dtype=torch.bfloat16):
    """a cache on the CPU that holds `held` of the `seen` tokens of each sequence at the given positions"""
    from mase_amd.quantized import PagedKVCache

    c = PagedKVCache(len(held), heads, 64, capacity, page_size=16, dtype=dtype, device="cpu", track_weights=True)
    c._held, c._seen = [list(held)], [list(seen)]
    c._held_dev[0], c._seen_dev[0] = torch.tensor(held, dtype=torch.int32), torch.tensor(seen, dtype=torch.int32)
    if positions is not None:
        c._positions[0] = positions
    return c


def scattered(held, seen, heads, capacity, gen):
    """an order of slots of its own for each head"""
    pos = torch.full((len(held), heads, capacity), -1, dtype=torch.int32)
    for b, (n, total) in enumerate(zip(held, seen)):
        for h in range(heads):
            pos[b, h, :n] = torch.randperm(total, generator=gen)[:n].to(torch.int32)
    return pos


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 3, 24), (2, 1, 3, 24), (2, 6, 3, 24), (2, 1, 1, 24), (1, 6, 1, 40)])
def test_columns_of_positions_become_columns_of_slots(shape, dtype):
    g = torch.Generator().manual_seed(110)
    pos = scattered([10, 10], [24, 24], 2, 32, g)
    c = cache([10, 10], [24, 24], pos)
    mask = torch.randn(shape, generator=g).to(dtype)
    got = c.slot_mask(mask, 6)
    assert got.dtype == dtype and got.shape == (2, 6, shape[2], 10)
    for b in range(2):
        for h in range(6):
            for t in range(shape[2]):
                for s in range(10):
                    want = mask[b if shape[0] > 1 else 0, h if shape[1] > 1 else 0, t, int(pos[b, h // 3, s])]
                    assert got[b, h, t, s] == want


def test_masks_stay_as_they_are_until_a_layer_is_evicted_from():
    c = cache([10, 10], [10, 10])
    mask = torch.zeros(2, 1, 3, 13)
    c.require_mask(mask, 3)
    assert c.slot_mask(mask, 6) is mask and c.slot_mask(None, 6) is None
    c.require_mask(torch.zeros(2, 1, 1, 11, dtype=torch.bool), 1)  # the dense chain's own business
    with pytest.raises(ValueError, match="mask"):
        c.require_mask(torch.zeros(2, 1, 1, 10), 1)


@pytest.mark.parametrize("bad", [torch.zeros(2, 1, 3, 26), torch.zeros(2, 1, 2, 27), torch.zeros(3, 1, 3, 27), torch.zeros(2, 3, 3, 27),
                                 torch.zeros(2, 3, 27), torch.zeros(2, 1, 3, 27, dtype=torch.bool)])
def test_masks_that_are_no_masks_of_positions_are_refused_after_an_eviction(bad):
    c = cache([10, 10], [24, 24])
    c.require_mask(torch.zeros(2, 1, 3, 27), 3)
    c.require_mask(torch.zeros(1, 6, 1, 40), 3)
    c.require_mask(None, 3)
    with pytest.raises(ValueError, match="mask"):
        c.require_mask(bad, 3)


@pytest.mark.parametrize("evicted", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_behind_shorter_sequences_are_hidden(dtype, evicted):
    held, seen = [10, 4, 7], [24, 24, 24] if evicted else [10, 4, 7]
    g = torch.Generator().manual_seed(111)
    c = cache(held, seen, scattered(held, seen, 2, 32, g), dtype=dtype)
    behind = torch.arange(10) >= torch.tensor(held)[:, None]
    got = c.slot_mask(None, 6)
    assert got.dtype == dtype and got.shape == (3, 1, 1, 10)
    assert bool((got[:, 0, 0][behind] == torch.finfo(dtype).min).all()) and not bool(got[:, 0, 0][~behind].any())
    if evicted:
        mask = torch.randn(3, 1, 2, 24, generator=g)
        got = c.slot_mask(mask, 6)
        for b in range(3):
            assert bool((got[b, :, :, behind[b]] == torch.finfo(torch.float32).min).all())
            for h in range(6):
                assert torch.equal(got[b, h, :, :held[b]], mask[b, 0][:, c._positions[0][b, h // 3, :held[b]].long()])


@pytest.mark.parametrize("tokens", [1, 3])
def test_masks_need_sequences_that_stand_at_one_position(tokens):
    c = cache([10, 4], [10, 4])
    c.require_mask(None, tokens)
    with pytest.raises(ValueError, match="4 to 10 tokens"):
        c.require_mask(torch.zeros(2, 1, tokens, 10 + tokens), tokens)


def test_a_refused_append_takes_no_pages():
    """states that the functions refuse (here: no GPU, other shapes) leave pages, table and lengths as they were"""
    from mase_amd._lib import MaseAmdError
    from mase_amd.quantized import PagedKVCache

    c = PagedKVCache(2, 1, 64, 100, page_size=16, num_pages=7, device="cpu")
    c._grow([17, 0])
    c._held[0][0] = 17
    free, table = list(c._free), c._table.clone()
    x = torch.zeros(2, 1, 30, 64, dtype=torch.bfloat16)
    for key, value, counts in ((x, x, None), (x, x, [30, 0]), (x.expand(2, 2, 30, 64), x, None), (x, x[:, :, :4], None), (x[..., :32], x, None)):
        with pytest.raises((MaseAmdError, ValueError)):
            c.append(key, value, counts=counts)
        assert c._free == free and torch.equal(c._table, table) and [len(p) for p in c._pages] == [2, 0]
        assert c.lengths() == [17, 0] and c._held_dev[0].tolist() == [0, 0]


def test_functions_refuse_whatever_records_gradients():
    """pages, masks and weights like queries and states: none of the functions has a backward pass"""
    from mase_amd._lib import MaseAmdError
    from mase_amd.quantized import functional as F

    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    kg = k.clone().requires_grad_()
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x, q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    m, w, pos = torch.zeros(1, 16), torch.zeros(1, 1, 16), torch.zeros(1, 1, 16, dtype=torch.int32)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: F.paged_kv_append(grad(x), x, k, k, t, n), lambda: F.paged_kv_append(x, grad(x), k, k, t, n)]
    calls += [lambda: F.paged_attention_decode(grad(q), k, k, t, n, 16), lambda: F.paged_attention_decode(q, k, k, t, n, 16, mask=grad(m)),
              lambda: F.paged_attention_decode(q, k, k, t, n, 16, weights=grad(w)), lambda: F.paged_kv_evict(k, k, t, n, grad(w), pos, 16, 8)]
    for pages in ((kg, k), (k, kg)):
        calls += [lambda p=pages: F.paged_kv_append(x, x, *p, t, n), lambda p=pages: F.paged_kv_gather(*p, t, n, 1),
                  lambda p=pages: F.paged_attention_decode(q, *p, t, n, 16), lambda p=pages: F.paged_kv_evict(*p, t, n, w, pos, 16, 8)]
    for call in calls:
        with pytest.raises(MaseAmdError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(MaseAmdError, match="ROCm device"):
            call()


@pytest.mark.parametrize("keep,recent,first", [(0, 0, 0), (20, 21, 0), (20, -1, 0), (20, 0, -1), (20, 11, 10), (-3, 0, 0)])
def test_evictions_that_cannot_be_are_refused_at_any_length(keep, recent, first):
    c = cache([10, 10], [10, 10])
    c.evict(20, recent=10, first=10)  # shorter than that: nothing to do
    for held in ([10, 10], [0, 0]):
        c._held = [held]
        with pytest.raises(ValueError, match="keep"):
            c.evict(keep, recent=recent, first=first)


@pytest.mark.parametrize("bad", [torch.zeros(2, 1, 3, 23), torch.zeros(2, 4, 3, 24), torch.zeros(3, 1, 3, 24), torch.zeros(2, 3, 24),
                                 torch.zeros(2, 1, 3, 24, dtype=torch.bool)])
def test_no_position_is_looked_up_past_a_mask(bad):
    """an index past the columns would end a kernel, and with it the process"""
    held, seen = [10, 10], [24, 24]
    c = cache(held, seen, scattered(held, seen, 2, 32, torch.Generator().manual_seed(112)))
    assert c.slot_mask(torch.zeros(2, 6, 3, 24), 6).shape == (2, 6, 3, 10)
    with pytest.raises(ValueError, match="mask"):
        c.slot_mask(bad, 6)
    c.require_mask(torch.zeros(2, 6, 1, 25), 1, heads=6)
    with pytest.raises(ValueError, match="mask"):
        c.require_mask(torch.zeros(2, 4, 1, 25), 1, heads=6)
