"""The paged key-value cache without a GPU: where slots lie and which page numbers are followed (the kernels' own index
functions in a host program), refusals of the C entry points and of the Python functions, the cache object's page keeping."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include "paged_kv_index.hpp"
#include <cstdio>
using namespace mase;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  const int32_t table[4] = {2, -1, 7, 3};  // a pool of 7 pages: entry 2 names a page that is not there
  CHECK(kv_page(table, 4, 4, 7, 0) == 2 && kv_page(table, 4, 4, 7, 15) == 2);
  CHECK(kv_page(table, 4, 4, 7, 16) == -1 && kv_page(table, 4, 4, 7, 32) == -1);
  CHECK(kv_page(table, 4, 4, 7, 48) == 3 && kv_page(table, 4, 4, 7, 63) == 3);
  CHECK(kv_page(table, 4, 4, 7, 64) == -1 && kv_page(table, 4, 4, 7, -1) == -1 && kv_page(table, 4, 4, 7, 0x7FFFFFFF) == -1);
  const int32_t wild[2] = {0x7FFFFFFF, (int32_t)0x80000000};
  CHECK(kv_page(wild, 2, 4, 7, 0) == -1 && kv_page(wild, 2, 4, 7, 16) == -1);
  CHECK(kv_length(10, 100, 4, 4) == 10 && kv_length(200, 100, 4, 4) == 64 && kv_length(200, 50, 4, 4) == 50);
  CHECK(kv_length(-5, 100, 4, 4) == 0 && kv_length(0, 100, 4, 4) == 0 && kv_length(0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFFF >> 12, 12) > 0);
  CHECK(kv_length((int)0x80000000, 100, 4, 4) == 0);
  CHECK(kv_new_slot(5, 3, 2, 4, 4) == 7 && kv_new_slot(5, 3, 3, 4, 4) == -1 && kv_new_slot(-1, 3, 0, 4, 4) == -1);
  CHECK(kv_new_slot(60, 10, 3, 4, 4) == 63 && kv_new_slot(60, 10, 4, 4, 4) == -1 && kv_new_slot(0x7FFFFFFF, 10, 5, 4, 4) == -1);
  CHECK(kv_new_slot(0, 0, 0, 4, 4) == -1 && kv_new_slot(0, -3, 0, 4, 4) == -1);
  // every slot of a table, every page shift: a row inside the pool or none
  for (int shift = 4; shift <= 12; ++shift)
    for (int s = -3; s < (5 << shift); ++s) {
      const int pg = kv_page(table, 4, shift, 7, s);
      CHECK(pg >= -1 && pg < 7);
      if (s >= 0 && (s >> shift) < 4) CHECK(pg == (table[s >> shift] < 7 ? table[s >> shift] : -1));
      else CHECK(pg == -1);
    }
  return 0;
}
'''


def test_index_functions_follow_no_page_outside_the_pool(tmp_path):
    src = tmp_path / "index.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "index"
    flags = ["-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined"]
    subprocess.run(["g++", *flags, "-I", os.path.join(ROOT, "mase_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr


@pytest.fixture(scope="module")
def lib():
    from mase_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g

        g.build()
    return _lib.load()


def _pool(**kw):
    from mase_amd import _lib

    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    d = dict(k=p, v=p, k_scales=None, v_scales=None, page_table=p, num_pages=4, page_size=16, kv_heads=2, head_dim=64, batch=1,
             table_pages=2, table_stride=2, k_stride_page=4096, k_stride_head=2048, k_stride_slot=128, v_stride_page=4096,
             v_stride_head=2048, v_stride_slot=128, format=0, dtype=1)
    d.update(kw)
    return _lib.PagedKv(**d), p, buf


BAD_POOLS = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(page_table=None), -1),
    (dict(dtype=0), -4), (dict(dtype=3), -4), (dict(format=5), -5), (dict(format=-1), -5),
    (dict(format=1), -1),                                                          # codes without scales
    (dict(head_dim=96), -2), (dict(head_dim=32), -2), (dict(head_dim=0), -2), (dict(head_dim=512), -2),
    (dict(page_size=8), -2), (dict(page_size=24), -2), (dict(page_size=8192), -2), (dict(page_size=0), -2),
    (dict(num_pages=0), -2), (dict(num_pages=1 << 31), -2), (dict(table_pages=0), -2), (dict(table_stride=1), -2),
    (dict(table_pages=1 << 28, table_stride=1 << 28), -2),                           # slots pass 31 bits
    (dict(batch=65536), -2), (dict(kv_heads=0), -2), (dict(kv_heads=65536), -2),
    (dict(k_stride_slot=64), -2), (dict(v_stride_slot=112), -2), (dict(k_stride_slot=136), -3), (dict(v_stride_page=4100), -3),
    (dict(v_stride_slot=1 << 28), -2),
]


@pytest.mark.parametrize("bad,code", BAD_POOLS)
def test_entry_points_refuse_bad_pools(lib, bad, code):
    c, p, _buf = _pool(**bad)
    a = ctypes.addressof(c)
    assert lib.mase_paged_kv_append(a, p, p, 1, 128, 64, 64, 128, 64, 64, p, None, None, 0, 0, None, None, None) == code
    assert lib.mase_paged_kv_gather(a, p, 16, p, p, None) == code
    assert lib.mase_paged_attention_decode(a, p, 128, 64, 2, p, 16, 0.1, None, 0, 0, None, 0, 0, p, None, 0, None) == code
    assert lib.mase_paged_kv_evict(a, p, 16, p, p, 32, 8, 0, 0, p + 4096, p + 8192, p, p, 1 << 20, None) == code


def test_entry_points_refuse_bad_arguments(lib):
    c, p, _buf = _pool()
    a = ctypes.addressof(c)

    def append(**kw):
        d = dict(key=p, value=p, tokens=1, ks=(128, 64, 64), vs=(128, 64, 64), starts=p, tab=None)
        d.update(kw)
        return lib.mase_paged_kv_append(a, d["key"], d["value"], d["tokens"], *d["ks"], *d["vs"], d["starts"], None, None, 0, 0, None,
                                        d["tab"], None)

    assert append(key=None) == -1 and append(value=None) == -1 and append(starts=None) == -1
    assert append(key=p + 8) == -3 and append(vs=(128, 64, 60)) == -3 and append(tokens=1 << 40) == -2
    assert append(tokens=0) == 0
    cm, pm, _b2 = _pool(format=1, k_scales=p, v_scales=p)
    assert lib.mase_paged_kv_append(ctypes.addressof(cm), pm, pm, 1, 128, 64, 64, 128, 64, 64, pm, None, None, 0, 0, None, None, None) == -1
    cm.k_scales = p + 4
    assert lib.mase_paged_kv_gather(ctypes.addressof(cm), p, 16, p, p, None) == -3
    assert lib.mase_paged_kv_append(None, p, p, 1, 128, 64, 64, 128, 64, 64, p, None, None, 0, 0, None, None, None) == -1
    assert lib.mase_paged_kv_gather(a, None, 16, p, p, None) == -1 and lib.mase_paged_kv_gather(a, p, 16, None, p, None) == -1
    assert lib.mase_paged_kv_gather(a, p, 16, p + 2, p, None) == -3 and lib.mase_paged_kv_gather(a, p, 1 << 40, p, p, None) == -2
    assert lib.mase_paged_kv_gather(a, p, 0, p, p, None) == 0

    def decode(**kw):
        d = dict(q=p, qs=(128, 64), heads=2, lengths=p, n=16, scaling=0.1, mask=None, mdt=1, w=None, out=p, ws=p, wsb=1 << 16)
        d.update(kw)
        return lib.mase_paged_attention_decode(a, d["q"], *d["qs"], d["heads"], d["lengths"], d["n"], d["scaling"], d["mask"], d["mdt"], 0,
                                               d["w"], 0, 0, d["out"], d["ws"], d["wsb"], None)

    assert decode(q=None) == -1 and decode(lengths=None) == -1 and decode(out=None) == -1
    assert decode(heads=3) == -2 and decode(heads=0) == -2 and decode(heads=2 * 257) == -2 and decode(n=1 << 40) == -2
    many, _p, _b3 = _pool(kv_heads=8192)  # 9 tiles of 16 query heads for each: too many rows for a grid
    assert lib.mase_paged_attention_decode(ctypes.addressof(many), p, 128, 64, 8192 * 144, p, 16, 0.1, None, 0, 0, None, 0, 0, p, p, 1 << 40, None) == -2
    assert decode(scaling=float("nan")) == -5 and decode(scaling=float("inf")) == -5
    assert decode(mask=p, mdt=2) == -4 and decode(q=p + 8) == -3 and decode(qs=(128, 60)) == -3 and decode(out=p + 8) == -3
    assert decode(w=p, ws=None, wsb=0) == -7 and decode(w=p, wsb=16) == -7 and decode(w=p, ws=p + 8) == -3
    assert decode(ws=None, wsb=0) == -7 and decode(wsb=8) == -7
    size = lib.mase_paged_attention_decode_workspace_bytes
    assert 0 < size(1, 2, 2, 64, 0, 16, 0) < size(1, 2, 2, 64, 0, 16, 1)  # (batch, heads, kv_heads, head_dim, format, max_length, weights)
    assert size(1, 3, 2, 64, 0, 16, 1) == 0 and size(1, 2, 2, 96, 0, 16, 1) == 0 and size(1, 2, 2, 64, 5, 16, 1) == 0

    def evict(**kw):
        d = dict(lengths=p, n=32, w=p, pos=p + 1024, cap=32, keep=8, recent=2, first=2, wo=p + 2048, po=p + 4096, lo=p, ws=p, wsb=1 << 16)
        d.update(kw)
        return lib.mase_paged_kv_evict(a, d["lengths"], d["n"], d["w"], d["pos"], d["cap"], d["keep"], d["recent"], d["first"], d["wo"],
                                       d["po"], d["lo"], d["ws"], d["wsb"], None)

    assert evict(keep=0) == -5 and evict(recent=9) == -5 and evict(recent=5, first=4) == -5 and evict(first=9, recent=0) == -5
    assert all(evict(**{k: None}) == -1 for k in ("lengths", "w", "pos", "wo", "po", "lo"))
    assert evict(wo=p) == -5 and evict(po=p + 1024) == -5 and evict(cap=0) == -2
    assert evict(ws=None) == -7 and evict(wsb=8) == -7 and evict(ws=p + 4) == -3


def test_the_packed_record_is_the_struct():
    """what the Python functions pack has the layout of mase_paged_kv, field by field"""
    import struct

    from mase_amd import _lib
    from mase_amd.quantized.functional import paged_kv

    values = list(range(1, 21))
    blob = paged_kv._record(*values)
    assert len(blob) == ctypes.sizeof(_lib.PagedKv) == struct.calcsize("@5P13N2i")
    c = _lib.PagedKv.from_buffer_copy(blob)
    assert [getattr(c, n) for n, _ in _lib.PagedKv._fields_] == values
    text = open(os.path.join(ROOT, "include", "mase_amd.h")).read()
    body = text[text.index("typedef struct mase_paged_kv {"):text.index("} mase_paged_kv;")]
    names = [n.strip(" *\n") for line in body.split("{")[1].split(";") for n in line.split("*/")[-1].replace("uint8_t*", "").replace(
        "const int32_t*", "").replace("void*", "").replace("size_t", "").replace("int32_t", "").split(",") if n.strip(" *\n")]
    assert names == [n for n, _ in _lib.PagedKv._fields_], names


def test_functions_have_no_cpu_path():
    from mase_amd._lib import MaseAmdError
    from mase_amd.quantized import functional as F

    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    w, pos = torch.zeros(1, 1, 16), torch.zeros(1, 1, 16, dtype=torch.int32)
    for call in (lambda: F.paged_kv_append(x, x, k, k, t, n), lambda: F.paged_kv_gather(k, k, t, n, 1),
                 lambda: F.paged_attention_decode(x[:, :, 0], k, k, t, n, 1), lambda: F.paged_kv_evict(k, k, t, n, w, pos, 16, 8)):
        with pytest.raises(MaseAmdError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="kv_format"):
        F.paged_kv_gather(k, k, t, n, 1, kv_format="mxint4")


def test_cache_object_keeps_its_pages():
    """allocation and refusals, on the host (nothing here launches a kernel)"""
    from mase_amd.quantized import PagedKVCache

    for bad in (dict(kv_format="int8"), dict(head_dim=80), dict(page_size=24), dict(page_size=8), dict(dtype=torch.float32),
                dict(batch_size=0), dict(max_length=0), dict(num_pages=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(batch_size=2, num_kv_heads=1, head_dim=64, max_length=100, device="cpu"), **bad})
    c = PagedKVCache(2, 1, 64, 100, num_layers=2, page_size=16, num_pages=9, device="cpu", track_weights=True)
    c._grow([17, 1])
    assert [len(p) for p in c._pages] == [2, 1] and len(c._free) == 6
    c._grow([17, 16])
    assert [len(p) for p in c._pages] == [2, 1]
    with pytest.raises(ValueError, match="max_length"):
        c._grow([101, 1])
    with pytest.raises(ValueError, match="free pages"):
        c._grow([100, 100])
    c._grow([96, 48])
    assert len(c._free) == 0 and len(set(sum(c._pages, []))) == 9
    assert c._table[0].tolist() == c._pages[0] + [-1] and c._table[1].tolist() == c._pages[1] + [-1] * 4
    c.reset()
    assert len(c._free) == 9 and int(c._table.max()) == -1
    states = torch.zeros(2, 1, 3, 64)
    with pytest.raises(ValueError, match="states must be"):
        c.append(states, states)
    with pytest.raises(ValueError, match="counts"):
        c.append(states.bfloat16(), states.bfloat16(), counts=[4, 0])
    c._held = [[5, 5], [4, 5]]
    with pytest.raises(ValueError, match="between steps"):
        c.evict(2)
    plain = PagedKVCache(2, 1, 64, 100, device="cpu")
    with pytest.raises(ValueError, match="track_weights"):
        plain.evict(2)


def test_cache_object_takes_only_the_quantizer_whose_values_it_holds():
    from mase_amd.quantized import PagedKVCache

    make = lambda fmt: PagedKVCache(1, 1, 64, 16, kv_format=fmt, device="cpu")  # noqa: E731
    i8 = {"data_in_block_size": 32, "data_in_width": 8}
    e4 = {"data_in_block_size": 32, "data_in_exponent_width": 4, "data_in_frac_width": 3}
    make(None).require_kind("mxint", {"data_in_block_size": 16, "data_in_width": 4})
    make(None).require_kind(None, {})
    make("mxint8").require_kind("mxint", i8)
    make("mxfp8_e4m3").require_kind("mxfp", e4)
    make("mxfp4").require_kind("mxfp", dict(e4, data_in_exponent_width=2, data_in_frac_width=1))
    for fmt, kind, cfg in (("mxint8", None, {}), ("mxint8", "mxint", dict(i8, data_in_width=6)), ("mxint8", "mxint", dict(i8, data_in_block_size=16)),
                           ("mxint8", "mxfp", e4), ("mxfp8_e5m2", "mxfp", e4), ("mxfp4", "mxint", i8)):
        with pytest.raises(ValueError, match="kv_format=None"):
            make(fmt).require_kind(kind, cfg)
