"""C entries of the windowed attention and the gated norms without a GPU: struct layouts, workspace sizes, and what they refuse before any launch."""
import ctypes as C
import importlib
import os
import re

import pytest

dic = importlib.import_module("diffusion-image-captioning_amd")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CTYPES = {"int": C.c_int, "float": C.c_float, "size_t": C.c_size_t, "int64_t": C.c_int64}


def header_fields(name):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "dic_hip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"(?:const\s+)?(\w+)\s*(.*)", decl, re.S).groups()
        for n in names.split(","):
            n = n.strip()
            fields.append((n.lstrip("* "), "ptr" if n.startswith("*") else kind))
    return fields


@pytest.mark.parametrize("struct,mirror", [("DicWinAttnParams", "WinAttnParams"), ("DicGatedNormParams", "GatedNormParams")])
def test_struct_mirrors_follow_the_header(struct, mirror):
    want = []
    for name, kind in header_fields(struct):
        if kind == "DicStrides":
            want += [(f"{name}_{d}", C.c_int64) for d, _ in header_fields("DicStrides")]
        elif kind == "DicNorm":
            want += [(f"{name}_{d}", C.c_void_p if k == "ptr" else CTYPES[k]) for d, k in header_fields("DicNorm")]
        else:
            want.append((name, C.c_void_p if kind == "ptr" else CTYPES[kind]))
    assert getattr(dic._lib, mirror)._fields_ == want


def test_packed_params_have_the_structs_sizes():
    from importlib import import_module
    block = import_module("diffusion-image-captioning_amd.block")
    for packed, mirror in ((block._WIN, dic._lib.WinAttnParams), (block._NORM, dic._lib.GatedNormParams)):
        assert packed.size == C.sizeof(mirror)
        values = list(range(1, len(mirror._fields_) + 1))
        got = mirror.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, n) for n, _ in mirror._fields_] == values


def attn(**kw):
    p = dic._lib.WinAttnParams()
    base = dict(N=2, Tq=8, Tk=8, H=4, Hkv=2, dh=64, left=-1, right=-1, scale=0.125, ws=4096, ws_bytes=1 << 20)
    base.update({n: 4096 * (i + 1) for i, n in enumerate(("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"))})
    for n in ("q", "out", "dout", "dq"):
        base.update({f"{n}_stride_n": 8 * 256, f"{n}_stride_t": 256, f"{n}_stride_h": 64})
    for n in ("k", "v", "dk", "dv"):
        base.update({f"{n}_stride_n": 8 * 128, f"{n}_stride_t": 128, f"{n}_stride_h": 64})
    for k, v in {**base, **kw}.items():
        setattr(p, k, v)
    return p


BAD_ATTENTION = [
    dict(dh=65), dict(dh=32), dict(H=3), dict(Hkv=0), dict(H=0), dict(N=-1), dict(Tq=-1), dict(Tk=-5), dict(Tq=1 << 30), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=4098), dict(v=4104), dict(k_stride_t=130), dict(q_stride_h=-64),
    dict(v_stride_t=1 << 24), dict(out_stride_t=0), dict(N=1 << 20, H=4096, Hkv=2),
]


@pytest.mark.parametrize("kw", BAD_ATTENTION, ids=str)
def test_attention_refuses(kw):
    L, p = dic.lib(), attn(**kw)
    backward = {k: ({"out": "dq", "out_stride_t": "dq_stride_t"}.get(k, k)) for k in kw}
    assert L.dic_win_attn_fwd(1, C.byref(p), None) == 1001 and L.dic_last_error().startswith(b"dic_win_attn")
    assert L.dic_win_attn_bwd(1, C.byref(attn(**{backward[k]: v for k, v in kw.items()})), None) == 1001


def test_attention_refuses_outputs_in_place_of_anything_else():
    L = dic._lib.lib()
    at = {n: getattr(attn(), n) for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")}
    for x in ("q", "k", "v"):
        assert L.dic_win_attn_fwd(1, C.byref(attn(out=at[x])), None) == 1001 and b"in place of" in L.dic_last_error()
    for y in ("dq", "dk", "dv"):
        for x in ("q", "k", "v", "out", "dout"):
            assert L.dic_win_attn_bwd(1, C.byref(attn(**{y: at[x]})), None) == 1001 and b"in place of" in L.dic_last_error()
        for z in ("dq", "dk", "dv"):
            if z != y:
                assert L.dic_win_attn_bwd(1, C.byref(attn(**{y: at[z]})), None) == 1001 and b"in one place" in L.dic_last_error()


def test_attention_refuses_other_types_and_missing_workspaces():
    L = dic.lib()
    for dtype in (-1, 2, 0x201):
        assert L.dic_win_attn_fwd(dtype, C.byref(attn()), None) == 1001
    assert L.dic_win_attn_fwd(1, None, None) == 1001
    size = L.dic_win_attn_ws_bytes(1, 1, C.byref(attn()))
    assert size >= 2 * 2 * 4 * 8 * 4
    for kw in (dict(ws=None), dict(ws_bytes=size - 1), dict(ws=4100), dict(lse=None), dict(dout=None), dict(dk=None), dict(dk_stride_t=0)):
        assert L.dic_win_attn_bwd(1, C.byref(attn(**kw)), None) == 1001, kw
    assert L.dic_win_attn_ws_bytes(1, 1, C.byref(attn(dh=65))) == 0


MORE_THAN_ONE_LAUNCH = [
    dict(N=1 << 26, H=1, Hkv=1, Tq=1, Tk=1),                                  # a workgroup of 64 threads for each row: 2^32 threads
    dict(N=1 << 25, H=2, Hkv=2, Tq=32, Tk=40), dict(N=1 << 24, H=4, Hkv=1, Tq=32, Tk=40), dict(N=3 << 22, H=2, Hkv=2, Tq=128, Tk=128),
    dict(N=1 << 30, H=1 << 30, Hkv=1, Tq=15 * 32, Tk=1),                      # 2^64 tiles: the product passes 64 bits
    dict(N=1 << 30, H=1 << 30, Hkv=1 << 30, Tq=1, Tk=15 * 32),
]


@pytest.mark.parametrize("kw", MORE_THAN_ONE_LAUNCH, ids=str)
@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_refuses_what_no_launch_holds_in_front_of_any(dtype, kw):
    L, p = dic.lib(), attn(**kw)
    assert L.dic_win_attn_fwd(dtype, C.byref(p), None) == 1001 and L.dic_last_error().endswith(b"for one launch")
    assert L.dic_win_attn_bwd(dtype, C.byref(p), None) == 1001 and L.dic_last_error().endswith(b"for one launch")


def test_attention_refuses_too_many_workgroups_of_the_few_rows_form():
    L, p = dic.lib(), attn(N=1 << 24, H=8, Hkv=1, Tq=2, Tk=65)                # four waves each (two in fp32 at dh 128)
    assert L.dic_win_attn_fwd(1, C.byref(p), None) == 1001 and L.dic_last_error().endswith(b"for one launch")


def norms(**kw):
    p = dic._lib.GatedNormParams()
    base = dict(rows=8, rows_per_gate=4, D=96, residual_scale=1.0, post_kind=1, pre_kind=2, post_eps=1e-6, pre_eps=1e-6, ws=4096, ws_bytes=1 << 20)
    base.update({n: 4096 for n in ("x", "y", "x_new", "a", "gate", "saved", "dx_new", "da", "dx", "dy", "dgate", "dpost_w", "dpre_b")})
    for k, v in {**base, **kw}.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw", [dict(D=0), dict(D=8193), dict(rows=-1), dict(rows=7), dict(rows_per_gate=0), dict(post_kind=3), dict(pre_kind=-1), dict(post_eps=-1.0), dict(pre_eps=float("nan")),
                                dict(post_kind=0, post_weight=4096), dict(residual_scale=float("inf")), dict(y=None)], ids=str)
def test_norms_refuse(kw):
    L = dic.lib()
    assert L.dic_gated_norm_fwd(0, C.byref(norms(**kw)), None) == 1001 and L.dic_last_error().startswith(b"dic_gated_norm")
    assert L.dic_gated_norm_bwd(0, C.byref(norms(**kw)), None) == 1001


def test_norms_refuse_missing_pointers():
    L = dic.lib()
    for kw in (dict(x=None), dict(x_new=None), dict(a=None)):
        assert L.dic_gated_norm_fwd(0, C.byref(norms(**kw)), None) == 1001, kw
    size = L.dic_gated_norm_ws_bytes(0, C.byref(norms()))
    assert size > 0
    for kw in (dict(da=None), dict(x_new=None), dict(dx=None), dict(dy=None), dict(saved=None), dict(ws=None), dict(ws_bytes=size - 1), dict(gate=None), dict(pre_kind=0), dict(post_kind=0)):
        assert L.dic_gated_norm_bwd(0, C.byref(norms(**kw)), None) == 1001, kw
    for dtype in (-1, 2, 0x200):
        assert L.dic_gated_norm_fwd(dtype, C.byref(norms()), None) == 1001
    assert L.dic_gated_norm_fwd(0, None, None) == 1001
