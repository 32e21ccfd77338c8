"""Paged caches without a GPU: what the calls refuse before they launch anything, and the argument structures as C lays them out."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BADARG, TOOLARGE = -1, -2
P = 1 << 20                                                   # an address that is never used


def pages(pkg, **more):
    a = pkg.PagesArgs(n_req=4, page=16, table_ld=8, n_pages=40, max_rows=64)
    for f in ("d_len", "d_len_out", "d_new", "d_base", "d_table", "d_free", "d_free_n", "d_free_n_out", "d_row_start", "d_slot", "d_pos"):
        setattr(a, f, P)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def store(pkg, **more):
    a = pkg.PagedStoreArgs(wtype=pkg.B200_WT_F16, n_q=8, n_kv=2, hd=64, page=16, n_pages=40, max_rows=4, eps=1e-6, qkv_ld=12 * 64, q_ld=8 * 64)
    for f in ("d_qkv", "d_rows", "d_slot", "d_pos", "d_k_pool", "d_v_pool", "d_q"):
        setattr(a, f, P)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def attn(pkg, **more):
    a = pkg.PagedAttnArgs(wtype=pkg.B200_WT_BF16, n_q=8, n_kv=2, hd=64, page=16, n_pages=40, max_rows=4, scale=0.125, q_ld=512, out_ld=512, n_req=4, table_ld=8, n_groups=1, prefix_ld=3)
    for f in ("d_q", "d_k_pool", "d_v_pool", "d_out", "d_row_start", "d_len", "d_table", "d_group_start", "d_prefix_len", "d_prefix_table", "d_work"):
        setattr(a, f, P)
    for k, v in more.items():
        setattr(a, k, v)
    if "work_bytes" not in more:
        a.work_bytes = 1 << 40
    return a


@pytest.mark.parametrize("name", ["b200_pages_extend", "b200_pages_release"])
@pytest.mark.parametrize("more,code", [
    (dict(n_req=-1), BADARG), (dict(n_req=1025), BADARG), (dict(page=8), BADARG), (dict(page=48), BADARG), (dict(page=512), BADARG), (dict(page=0), BADARG),
    (dict(table_ld=-1), BADARG), (dict(table_ld=(1 << 20) + 1), BADARG), (dict(n_pages=-1), BADARG), (dict(n_pages=1 << 27), TOOLARGE),
    (dict(d_len=None), BADARG), (dict(d_len_out=None), BADARG), (dict(d_new=None), BADARG), (dict(d_table=None), BADARG), (dict(d_free=None), BADARG),
    (dict(d_free_n=None), BADARG), (dict(d_free_n_out=None), BADARG)])
def test_pages_refusals(pkg, lib, name, more, code):
    assert getattr(lib, name)(C.byref(pages(pkg, **more)), None) == code
    assert getattr(lib, name)(None, None) == BADARG


@pytest.mark.parametrize("more", [dict(max_rows=-1), dict(max_rows=(1 << 20) + 1), dict(d_row_start=None), dict(d_slot=None), dict(d_pos=None)])
def test_extend_refusals(pkg, lib, more):
    assert lib.b200_pages_extend(C.byref(pages(pkg, **more)), None) == BADARG


SHAPES = [
    (dict(wtype=0), BADARG), (dict(wtype=3), BADARG), (dict(hd=96), BADARG), (dict(hd=512), BADARG), (dict(hd=0), BADARG), (dict(n_q=0), BADARG), (dict(n_kv=0), BADARG),
    (dict(n_kv=3), BADARG), (dict(n_q=2048), BADARG), (dict(max_rows=-1), BADARG), (dict(max_rows=(1 << 20) + 1), BADARG), (dict(n_pages=0), BADARG), (dict(page=24), BADARG),
    (dict(page=8), BADARG), (dict(n_pages=1 << 27), TOOLARGE), (dict(d_q=None), BADARG), (dict(d_k_pool=None), BADARG), (dict(d_v_pool=None), BADARG), (dict(d_q=P + 8), BADARG),
    (dict(d_k_pool=P + 2), BADARG), (dict(d_v_pool=P + 8), BADARG), (dict(q_ld=504), BADARG), (dict(q_ld=516), BADARG)]


@pytest.mark.parametrize("more,code", SHAPES + [
    (dict(d_qkv=None), BADARG), (dict(d_rows=None), BADARG), (dict(d_slot=None), BADARG), (dict(d_pos=None), BADARG), (dict(d_qkv=P + 4), BADARG), (dict(d_q_gamma=P + 4), BADARG),
    (dict(d_k_gamma=P + 8), BADARG), (dict(d_inv_freq=P + 4), BADARG), (dict(qkv_ld=764), BADARG), (dict(qkv_ld=770), BADARG)])
def test_store_refusals(pkg, lib, more, code):
    assert lib.b200_paged_store(C.byref(store(pkg, **more)), None) == code
    assert lib.b200_paged_store(None, None) == BADARG


@pytest.mark.parametrize("more,code", SHAPES + [
    (dict(d_out=None), BADARG), (dict(d_row_start=None), BADARG), (dict(d_len=None), BADARG), (dict(d_table=None), BADARG), (dict(d_group_start=None), BADARG),
    (dict(d_prefix_len=None), BADARG), (dict(d_prefix_table=None), BADARG), (dict(d_work=None), BADARG), (dict(d_work=P + 8), BADARG), (dict(d_out=P + 8), BADARG),
    (dict(out_ld=500), BADARG), (dict(out_ld=518), BADARG), (dict(n_req=-1), BADARG), (dict(n_req=1025), BADARG), (dict(n_groups=-1), BADARG), (dict(n_groups=5), BADARG),
    (dict(table_ld=-1), BADARG), (dict(table_ld=(1 << 20) + 1), BADARG), (dict(prefix_ld=(1 << 20) + 1), BADARG), (dict(work_bytes=100), BADARG),
    (dict(scale=float("nan")), BADARG), (dict(scale=-float("inf")), BADARG)])
def test_attention_refusals(pkg, lib, more, code):
    assert lib.b200_paged_attn(C.byref(attn(pkg, **more)), None) == code
    assert lib.b200_paged_attn(None, None) == BADARG


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38])
def test_scales_that_overflow_as_powers_of_two(pkg, lib, scale):
    assert lib.b200_paged_attn(C.byref(attn(pkg, scale=scale)), None) == BADARG


def test_nothing_to_do_is_no_error(pkg, lib):
    assert lib.b200_paged_store(C.byref(store(pkg, max_rows=0)), None) == 0
    assert lib.b200_paged_attn(C.byref(attn(pkg, max_rows=0)), None) == 0
    assert lib.b200_paged_attn(C.byref(attn(pkg, n_req=0, n_groups=0)), None) == 0


def test_work_bytes(pkg, lib):
    size = lambda **more: lib.b200_paged_attn_work_bytes(C.byref(attn(pkg, **more)))          # noqa: E731
    assert size() > 0 and size() % 8 == 0
    assert size(d_q=None, d_work=None, work_bytes=0) == size()                                # sizes alone count
    assert size(max_rows=400) > size() and size(hd=128) > size()
    assert size(page=24) == 0 and size(wtype=0) == 0 and lib.b200_paged_attn_work_bytes(None) == 0


def test_structures_are_those_of_the_header(pkg, tmp_path):
    """Sizes and offsets of every field, from the C compiler."""
    classes = {"b200_pages_args": pkg.PagesArgs, "b200_paged_store_args": pkg.PagedStoreArgs, "b200_paged_attn_args": pkg.PagedAttnArgs}
    lines, want = [], []
    for name, cls in classes.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for field, kind in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "llmb200_paged_kernels.h"\nint main(void) { ' + " ".join(lines) + " return 0; }\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    assert list(map(int, subprocess.run([exe], check=True, stdout=subprocess.PIPE, text=True).stdout.split())) == want
