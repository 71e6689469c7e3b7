"""Host side of the paged cache: struct layouts, refusals before any launch, the
page table's bookkeeping, and the 64-bit reference's own rounding (no GPU)."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import cache_reference as ref
import ssa_amd
from conftest import ROOT
from ssa_amd import _lib

F8 = torch.float8_e4m3fn


def test_cache_structs_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    mirrors = {"ssa_kv_cache": _lib.KVCacheStruct, "ssa_batch_rows": _lib.BatchRows,
               "ssa_page_plan_args": _lib.PagePlanArgs,
               "ssa_cache_append_args": _lib.CacheAppendArgs,
               "ssa_select_pages_args": _lib.SelectPagesArgs,
               "ssa_cached_attention_args": _lib.CachedAttentionArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ssa_amd.h"',
             'int main(void) {']
    for c, py in mirrors.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ['return 0;', '}']) + "\n")
    subprocess.check_call([gcc, "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                           str(exe)])
    got = {}
    for line in subprocess.check_output([str(exe)], text=True).splitlines():
        c, f, n = line.split()
        got[c, f] = int(n)
    for c, py in mirrors.items():
        assert got[c, "size"] == ctypes.sizeof(py), c
        for f in py._fields_:
            assert got[c, f[0]] == getattr(py, f[0]).offset, (c, f[0])


def test_reference_rounds_as_the_e4m3_cast():
    """Every bf16 number up to 448 in magnitude, and the midpoints of codes."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).double()
    x = x[x.abs() <= 448]
    v = ref.VALUES[ref.VALUES >= 0].sort().values
    x = torch.cat([x, (v[1:] + v[:-1]) / 2, -(v[1:] + v[:-1]) / 2])
    assert torch.equal(ref.to_code(x), x.float().to(F8).double())


@pytest.mark.parametrize("a,e", [(0.0, -100), (448.0, 0), (448.0001, 1), (224.0, -1), (1e-40, -100),
                                 (2.0 ** 120, 112), (1.0, -8), (1.75, -8), (1.76, -7)])
def test_reference_scale_exponent(a, e):
    assert ref.exponent(a) == e


# ---------------------------------------------------------------------------- refusals
def _cache(P=3, H=2, ps=32, d=48):
    return ssa_amd.PagedKVCache(P, H, d, ps, device="cpu")


def _plan(T=2, R=2, W=3):
    return ssa_amd.PagePlan(torch.zeros(R, W, dtype=torch.int32),
                            torch.zeros(R + 1, dtype=torch.int32),
                            torch.zeros(T, dtype=torch.int32), torch.zeros(T, dtype=torch.int32))


@pytest.mark.parametrize("kw", [dict(d=0), dict(d=257), dict(ps=16), dict(ps=48), dict(P=0)])
def test_cache_refuses_sizes(kw):
    with pytest.raises(RuntimeError):
        _cache(**kw)


@pytest.mark.parametrize("which", ["v_layout", "dtype", "scale_dtype", "strides", "bounds"])
def test_cache_refuses_buffers(which):
    c = _cache()
    t = dict(k_codes=c.k_codes, v_codes=c.v_codes, bounds=c.bounds, k_scale=c.k_scale,
             v_scale=c.v_scale, d_head=48)
    if which == "v_layout":
        t["v_codes"] = c.k_codes.contiguous()
    elif which == "dtype":
        t["k_codes"] = c.k_codes.view(torch.uint8)
    elif which == "scale_dtype":
        t["k_scale"] = c.k_scale.double()
    elif which == "strides":
        t["k_codes"] = torch.zeros(3, 32, 2, 64, dtype=torch.uint8).view(F8).transpose(1, 2)
    elif which == "bounds":
        t["bounds"] = c.bounds[:2]
    with pytest.raises(RuntimeError, match="PagedKVCache"):
        ssa_amd.PagedKVCache.from_tensors(**t)


@pytest.mark.parametrize("bad", ["heads", "dim", "shapes", "dtypes", "slots_dtype", "slots_len",
                                 "float64", "grad", "device"])
def test_append_refusals(bad):
    c = _cache()
    k, v = torch.zeros(4, 2, 48), torch.zeros(4, 2, 48)
    s = torch.zeros(4, dtype=torch.int64)
    if bad == "heads":
        k, v = torch.zeros(4, 3, 48), torch.zeros(4, 3, 48)
    elif bad == "dim":
        k, v = torch.zeros(4, 2, 64), torch.zeros(4, 2, 64)
    elif bad == "shapes":
        v = v[:3]
    elif bad == "dtypes":
        v = v.half()
    elif bad == "slots_dtype":
        s = s.int()
    elif bad == "slots_len":
        s = s[:3]
    elif bad == "float64":
        k, v = k.double(), v.double()
    elif bad == "grad":
        k.requires_grad_()
    with pytest.raises(RuntimeError, match="ROCm" if bad == "device" else "ssa_amd"):
        ssa_amd.cache_append(c, k, v, s)


@pytest.mark.parametrize("bad", ["heads", "dim", "rows", "starts", "table_dtype", "table_strides",
                                 "rank", "grad", "device"])
def test_attention_and_selection_refusals(bad):
    c, p, q = _cache(), _plan(), torch.zeros(2, 4, 48)
    if bad == "heads":
        q = torch.zeros(2, 3, 48)
    elif bad == "dim":
        q = torch.zeros(2, 4, 40)
    elif bad == "rows":
        p.positions = p.positions[:1]
    elif bad == "starts":
        p.starts = p.starts[:2]
    elif bad == "table_dtype":
        p.block_table = p.block_table.long()
    elif bad == "table_strides":
        p.block_table = torch.zeros(3, 2, dtype=torch.int32).T
    elif bad == "rank":
        q = q[0]
    elif bad == "grad":
        q.requires_grad_()
    m = "ROCm" if bad == "device" else "inference only" if bad == "grad" else "ssa_amd"
    with pytest.raises(RuntimeError, match=m):
        ssa_amd.cached_attention(q, c, p)
    with pytest.raises(RuntimeError, match=m):
        ssa_amd.select_pages(q, c, p, 3)


@pytest.mark.parametrize("top,first,recent", [(3, 0, 0), (3, 2, 2), (3, -1, 1), (0, 0, 1)])
def test_selection_refuses_budgets(top, first, recent):
    with pytest.raises(RuntimeError, match="recent"):
        ssa_amd.select_pages(torch.zeros(2, 4, 48), _cache(), _plan(), top, first=first,
                             recent=recent)


def test_plan_refusals():
    i = dict(dtype=torch.int32)
    good = [torch.zeros(2, **i), torch.zeros(2, **i), torch.zeros(2, 3, **i), torch.zeros(5, **i),
            torch.zeros(1, **i)]
    with pytest.raises(RuntimeError, match="ROCm"):
        ssa_amd.plan_pages(*good, page_size=64, num_rows=2)
    for at, t in ((0, torch.zeros(2)), (0, torch.zeros(3, **i)), (1, torch.zeros(2).long()),
                  (2, torch.zeros(3, 2, **i).T), (2, torch.zeros(0, 3, **i)), (3, torch.zeros(5)),
                  (4, torch.zeros(2, **i))):
        args = list(good)
        args[at] = t
        with pytest.raises(RuntimeError, match="plan_pages"):
            ssa_amd.plan_pages(*args, page_size=64, num_rows=2)


def _c_cache(**kw):
    a = dict(k_codes=256, v_codes=256, bounds=256, k_scale=256, v_scale=256, num_pages=4, Hkv=2,
             page=64, D=64, d=64)
    return _lib.KVCacheStruct(**(a | kw))


def _c_rows(**kw):
    a = dict(block_table=256, table_stride=4, R=2, width=4, starts=256, requests=256,
             positions=256, T=2)
    return _lib.BatchRows(**(a | kw))


@pytest.mark.parametrize("cache,rows,top,code", [
    (dict(page=48), {}, 0, -2), (dict(d=65), {}, 0, -2), (dict(d=300, D=256), {}, 0, -2),
    (dict(Hkv=3), {}, 0, -1), (dict(num_pages=0), {}, 0, -1), (dict(k_codes=264), {}, 0, -1),
    (dict(v_scale=None), {}, 0, -1), ({}, dict(R=0), 0, -1), ({}, dict(table_stride=3), 0, -1),
    ({}, dict(starts=None), 0, -1), ({}, dict(T=-1), 0, -1), ({}, dict(T=1 << 30), 0, -1),
    ({}, dict(width=1 << 26, table_stride=1 << 26), 0, -1), ({}, {}, -1, -1)])
def test_c_entry_points_refuse_before_a_launch(cache, rows, top, code):
    """The pointers here are never followed."""
    L = _lib.lib()
    a = _lib.CachedAttentionArgs(_c_cache(**cache), _c_rows(**rows), 256, 256, _lib.SSA_BF16, 4,
                                 256, 64, 256, 64, 0.125, 256 if top else None, top)
    assert L.ssa_cached_attention_workspace_bytes(ctypes.byref(a)) == code
    assert L.ssa_cached_attention(ctypes.byref(a), None, 0, None) == code
    assert L.ssa_last_error()


def test_c_entry_points_refuse_other_arguments():
    L = _lib.lib()
    a = _lib.CachedAttentionArgs(_c_cache(), _c_rows(T=64, width=4096, table_stride=4096), 256,
                                 256, _lib.SSA_BF16, 4, 256, 64, 256, 64, 0.125, None, 0)
    n = L.ssa_cached_attention_workspace_bytes(ctypes.byref(a))
    assert n > 0
    assert L.ssa_cached_attention(ctypes.byref(a), 256, n - 1, None) == -3
    assert b"workspace" in L.ssa_last_error()
    assert L.ssa_cached_attention(ctypes.byref(a), 8, n, None) == -1
    a.dtype = 7
    assert L.ssa_cached_attention_workspace_bytes(ctypes.byref(a)) == -1
    s = _lib.SelectPagesArgs(_c_cache(), _c_rows(), 256, _lib.SSA_BF16, 4, 256, 64, 2, 1, 2, 256)
    assert L.ssa_select_pages(ctypes.byref(s), None) == -1
    s = _lib.SelectPagesArgs(_c_cache(), _c_rows(width=20000, table_stride=20000), 256,
                             _lib.SSA_BF16, 4, 256, 64, 4, 1, 2, 256)
    assert L.ssa_select_pages(ctypes.byref(s), None) == -2
    p = _lib.PagePlanArgs(256, 256, 256, 4, 16385, 4, 64, 2, 256, 8, 256, 256, 256, 256, 256, 256,
                          256, 256)
    assert L.ssa_page_plan(ctypes.byref(p), None) == -2
    p.R, p.slots = 2, None
    assert L.ssa_page_plan(ctypes.byref(p), None) == -1
    p.slots, p.page = 256, 16
    assert L.ssa_page_plan(ctypes.byref(p), None) == -2
    c = _lib.CacheAppendArgs(_c_cache(), None, 256, _lib.SSA_F32, 2, 64, 64, 64, 64, 256)
    assert L.ssa_cache_append(ctypes.byref(c), None) == -1
    for f in (L.ssa_page_plan, L.ssa_cache_append, L.ssa_select_pages):
        assert f(None, None) == -1
    # nothing to do is no error
    c.T = 0
    assert L.ssa_cache_append(ctypes.byref(c), None) == 0


@pytest.mark.parametrize("T,R,Hq,Hkv,width,top", [
    (1, 1, 32, 1, 1 << 14, 0), (1000, 1, 32, 1, 2048, 0), (70, 1, 8, 8, 1 << 14, 0),
    (8192, 4, 32, 8, 512, 0), (1 << 17, 1, 32, 8, 2048, 0), (4096, 4096, 32, 8, 1 << 14, 0),
    (300, 9, 64, 64, 4096, 0), (64, 64, 32, 8, 4096, 2048), (1 << 16, 8, 32, 1, 4096, 16)])
def test_workspace_is_bounded(T, R, Hq, Hkv, width, top):
    """Chunks are cut for about 2,048 workgroups: 128 columns of 258 floats each at
    most, whatever the rows, the requests and the table's width."""
    a = _lib.CachedAttentionArgs(
        _c_cache(Hkv=Hkv, D=256, d=256), _c_rows(T=T, R=R, width=width, table_stride=width), 256,
        256, _lib.SSA_BF16, Hq, Hq * 256, 256, Hq * 256, 256, 0.0625, 256 if top else None, top)
    n = _lib.lib().ssa_cached_attention_workspace_bytes(ctypes.byref(a))
    assert 0 <= n <= (2 * 2048 + 512) * 64 * 258 * 4


# ---------------------------------------------------------------------------- page table
def test_rows_beyond_32_bits_are_refused():
    x = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="rows"):
        ssa_amd.plan_pages(x[0], x[0], x, x[0], x[0], page_size=32, num_rows=1 << 31)
    c = ssa_amd.PagedKVCache(1, 1, 64, 32, device="cpu")
    k = torch.zeros(1, 1, 64).expand(1 << 31, 1, 64)
    with pytest.raises(RuntimeError, match="2\\^31 rows"):
        ssa_amd.cache_append(c, k, k, torch.zeros(1, dtype=torch.int64))


def test_released_pages_return_once():
    t = ssa_amd.PageTable(4, 3, 10, 32, device="cpu")
    free, table = t._free[:10].tolist(), t.block_table.tolist()
    cached, new = t.lengths.tolist(), [70, 10, 0, 33]
    out = ref.plan(cached, new, table, free, 10, 32, 200)
    t.block_table.copy_(torch.tensor(table))
    t.lengths.copy_(torch.tensor(out[1]))
    t.free_count.fill_(out[5])
    assert out[5] == 4
    t.release(torch.tensor([3, 0, 3, 0]))                 # a place named twice
    assert t.lengths.tolist() == [0, 10, 0, 0]
    assert t.free_count.item() == 9
    held = [p for p in t.block_table.flatten().tolist() if p >= 0]
    assert sorted(t._free[:9].tolist() + held) == list(range(10))
    t.release(torch.tensor([], dtype=torch.int64))
    t.release(torch.tensor([1, 7, -1]))                   # 7 and -1 name no place
    assert sorted(t._free[:10].tolist()) == list(range(10)) and t.free_count.item() == 10


# ---------------------------------------------------------------------------- modules
def _attn(**kw):
    a = dict(d_model=64, num_heads=4, num_kv_heads=2, num_neighbors=128, window_size=16,
             causal=True)
    return ssa_amd.SparseAttention(ssa_amd.SSAConfig(**(a | kw)))


def test_page_budget_holds_the_window_and_the_globals():
    assert _attn().page_budget(64) == (4, 1, 2)
    assert _attn().page_budget(32) == (4, 1, 2)
    assert _attn(num_neighbors=1024).page_budget(64) == (16, 1, 2)
    assert _attn(num_global_tokens=0, window_size=0).page_budget(128) == (2, 0, 1)
    with pytest.raises(ValueError, match="global_token_indices"):
        _attn(global_token_indices=[0, 9]).page_budget(64)


def test_forward_cached_refusals():
    a, p = _attn(causal=False), _plan()
    with pytest.raises(ValueError, match="causal"):
        a.forward_cached(torch.zeros(2, 64), a.new_cache(2), p)
    a = _attn()
    with pytest.raises(ValueError, match="packed"):
        a.forward_cached(torch.zeros(1, 2, 64), a.new_cache(2), p)
    m = ssa_amd.SparseTransformer(a.config, num_layers=2, vocab_size=11)
    with pytest.raises(ValueError, match="caches"):
        m.forward_cached(torch.zeros(2, dtype=torch.int64), m.new_caches(2)[:1], p)
