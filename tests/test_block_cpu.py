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


def packed(N, Tq, Tk, H, Hkv):
    """Sizes with the strides of contiguous tensors."""
    strides = {f"{x}_stride_{d}": v for names, t, h in ((("q", "out", "dout", "dq"), Tq, H), (("k", "v", "dk", "dv"), Tk, Hkv)) for x in names
               for d, v in (("n", 64 * t * h), ("t", 64 * h), ("h", 64))}
    return attn(N=N, Tq=Tq, Tk=Tk, H=H, Hkv=Hkv, **strides)


@pytest.mark.parametrize("kw", MORE_THAN_ONE_LAUNCH, ids=str)
@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_refuses_what_no_launch_holds_in_front_of_any(dtype, kw):
    L, p = dic.lib(), packed(**kw)
    assert L.dic_win_attn_fwd(dtype, C.byref(p), None) == 1001 and L.dic_last_error().endswith(b"for one launch")
    assert L.dic_win_attn_bwd(dtype, C.byref(p), None) == 1001 and L.dic_last_error().endswith(b"for one launch")


def test_attention_refuses_too_many_workgroups_of_the_few_rows_form():
    L, p = dic.lib(), packed(N=1 << 24, H=8, Hkv=1, Tq=2, Tk=65)                # four waves each (two in fp32 at dh 128)
    assert L.dic_win_attn_fwd(1, C.byref(p), None) == 1001 and L.dic_last_error().endswith(b"for one launch")


def apart(**kw):
    """Far from each other unless `kw` moves one; without a workspace, so that no call gets as far as a launch."""
    return attn(**{**{n: 1 << 20 << i for i, n in enumerate(("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"))}, "ws": None, **kw})


def told(p):
    assert dic.lib().dic_win_attn_bwd(1, C.byref(p), None) == 1001
    return dic.lib().dic_last_error()


def test_attention_refuses_outputs_that_overlap_in_part():
    at = {n: getattr(apart(), n) for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv")}
    assert b"workspace" in told(apart())
    row, flat = 256 * 2, 4 * 2 * 4 * 8                                        # bytes of a token row of q, of lse
    for y in ("dq", "dk", "dv"):
        size = 2 * 8 * (row if y == "dq" else row // 2)
        for x in ("q", "k", "v", "out", "dout"):
            other = 2 * 8 * (row if x in ("q", "out", "dout") else row // 2)
            assert b"overlaps" in told(apart(**{y: at[x] + other - 16})) and b"overlaps" in told(apart(**{y: at[x] - size + 16})), (y, x)
            assert b"workspace" in told(apart(**{y: at[x] + other})) and b"workspace" in told(apart(**{y: at[x] - size})), (y, x)
        assert b"overlaps" in told(apart(**{y: at["lse"] + flat - 16})) and b"workspace" in told(apart(**{y: at["lse"] + flat}))
        for n, bytes_ in (("key_mask", 16), ("kv_len", 8), ("q_pos", 8)):
            assert b"overlaps" in told(apart(**{n: at[y] + 16})) and b"workspace" in told(apart(**{n: at[y] - bytes_}))
        for z in ("dq", "dk", "dv"):
            if z != y:
                assert b"overlaps" in told(apart(**{y: at[z] + 16}))
    p = apart(ws=at["dq"] + 2 * 8 * row - 16, ws_bytes=1 << 20)
    assert b"overlaps" in told(p)
    L = dic.lib()
    for kw in (dict(out=at["q"] + 16), dict(out=at["v"] - 16), dict(lse=at["out"] + 64), dict(lse=at["k"]), dict(key_mask=at["out"] + 8)):
        assert L.dic_win_attn_fwd(1, C.byref(apart(**kw)), None) == 1001 and b"overlaps" in L.dic_last_error(), kw


def test_attention_takes_outputs_that_lie_between_each_other():
    """Views of one packed tensor [N, T, heads, dh], of its transposed form, and of caches of which a call reads every other sequence."""
    for n, t, h in ((8 * 512, 512, 64), (8 * 512, 64, 8 * 64)):
        kw = {f"{x}_stride_{d}": v for x in ("dq", "dk", "dv") for d, v in (("n", n), ("t", t), ("h", h))}
        at = 1 << 30
        assert b"workspace" in told(apart(dq=at, dk=at + 2 * (4 * h), dv=at + 2 * (6 * h), **kw))
        assert b"overlaps" in told(apart(dq=at, dk=at + 2 * (4 * h) - 16, dv=at + 2 * (6 * h), **kw))
        assert b"overlaps" in told(apart(dq=at, dk=at + 2 * (3 * h), dv=at + 2 * (6 * h), **kw))
    k = {f"k_stride_{d}": v for d, v in (("n", 2 * 8 * 128), ("t", 128), ("h", 64))}
    dk = {f"dk_stride_{d}": v for d, v in (("n", 2 * 8 * 128), ("t", 128), ("h", 64))}
    assert b"workspace" in told(apart(k=1 << 30, dk=(1 << 30) + 2 * 8 * 128, **k, **dk))
    assert b"overlaps" in told(apart(k=1 << 30, dk=(1 << 30) + 2 * 7 * 128, **k, **dk))


def test_overlaps_of_small_layouts_are_told_exactly():
    """Random strides, compared with the rows counted out."""
    import itertools
    import random
    rng, seen = random.Random(5), {True: 0, False: 0}
    for _ in range(1500):
        N, T, H = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 4)
        a, b = ([8 * rng.randint(0 if which else 8, rng.choice((9, 20, 60, 200))) for _ in range(3)] for which in (0, 1))
        if a[0] == a[1] or a[1] == a[2] or a[0] == a[2]:                       # (an output's own rows are another matter)
            continue
        at = 1 << 30, (1 << 30) + 16 * rng.randint(-300, 300)
        starts = [{p + 2 * (n * s[0] + t * s[1] + h * s[2]) for n, t, h in itertools.product(range(N), range(T), range(H))} for p, s in zip(at, (a, b))]
        want = any(abs(x - y) < 128 for x in starts[0] for y in starts[1])
        kw = {f"{n}_stride_{d}": s[i] for n, s in (("dq", a), ("q", b), *((n, (64 * T * H, 64 * H, 64)) for n in ("k", "v", "dk", "dv")))
              for i, d in enumerate("nth")}
        got = told(apart(N=N, Tq=T, Tk=T, H=H, Hkv=H, q=at[1], dq=at[0], out=1 << 40, dout=1 << 41, lse=1 << 42, dk=1 << 43, dv=1 << 44, k=1 << 45, v=1 << 46, **kw))
        if at[0] == at[1]:
            continue
        if b"rows of an output overlap" in got:
            continue
        assert (b"overlaps an input" in got) == want and (b"workspace" in got) == (not want), (N, T, H, a, b, at)
        seen[want] += 1
    assert min(seen.values()) > 100


def test_an_output_whose_rows_overlap_is_refused():
    """Every stride at least a row long, and yet: two strides the same, or one that another's steps reach.  Random ones, compared with the rows counted out."""
    import itertools
    import random
    for s in ((4096, 64, 64), (64, 256, 64), (4096, 192, 128), (1984, 1000, 64)):
        p = apart(N=2, Tq=8, H=4, **{f"dq_stride_{d}": v for d, v in zip("nth", s)})
        assert b"rows of an output overlap" in told(p), s
    rng, seen = random.Random(6), {True: 0, False: 0}
    for _ in range(3000):
        N, T, H = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 4)
        s = [8 * rng.randint(8, rng.choice((9, 20, 60, 200))) for _ in range(3)]
        starts = [n * s[0] + t * s[1] + h * s[2] for n, t, h in itertools.product(range(N), range(T), range(H))]
        want = any(abs(x - y) < 64 for x, y in itertools.combinations(starts, 2))
        kw = {f"{n}_stride_{d}": st[i] for n, st in (("dq", s), *((n, (64 * T * H, 64 * H, 64)) for n in ("q", "k", "v", "out", "dout", "dk", "dv"))) for i, d in enumerate("nth")}
        got = told(apart(N=N, Tq=T, Tk=T, H=H, Hkv=H, **kw))
        assert (b"rows of an output overlap" in got) == want and (b"workspace" in got) == (not want), (N, T, H, s)
        seen[want] += 1
    assert min(seen.values()) > 300


def test_strides_beyond_the_address_space_are_refused():
    for kw in (dict(q_stride_n=1 << 60), dict(k_stride_h=1 << 55), dict(dv_stride_n=1 << 62)):
        assert b"strides" in told(apart(**kw)), kw


def test_attention_refuses_a_scale_that_is_infinite_times_log2_e():
    """The kernels' exponentials are powers of two: 2.5e38 log2(e) is infinite, and 0 times that no logit."""
    for entry in (dic.lib().dic_win_attn_fwd, dic.lib().dic_win_attn_bwd):
        assert entry(1, C.byref(attn(scale=2.5e38)), None) == 1001 and b"scale" in dic.lib().dic_last_error()


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


def test_an_older_library_can_be_loaded_for_a_comparison(tmp_path):
    """DIC_HIP_LIB with a library of the same version that has no such entries (a stand-in built here): it loads, and a call of one names the file."""
    import subprocess
    import sys
    older = [n for n in dic._lib.EXPORTS if n not in dic._lib.LATER_EXPORTS]
    assert set(dic._lib.LATER_EXPORTS) < set(dic._lib.EXPORTS)

    def build(path, names):
        src = tmp_path / "stub.c"
        src.write_text("".join("const char* %s(void) { return \"\"; }\n" % n if n == "dic_last_error" else
                               "int %s(void) { return %d; }\n" % (n, dic._lib.ABI_VERSION if n == "dic_version" else 0) for n in names))
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(path), str(src)], check=True)
        code = ("import importlib\ndic = importlib.import_module('diffusion-image-captioning_amd')\nL = dic.lib()\nassert L.dic_version() == %d\n"
                "from importlib import import_module\nblock = import_module('diffusion-image-captioning_amd.block')\nblock._fn('dic_win_attn_fwd')" % dic._lib.ABI_VERSION)
        run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, "DIC_HIP_LIB": str(path)}, capture_output=True, text=True)
        return run.stderr

    said = build(tmp_path / "older.so", older)
    assert "older.so does not export dic_win_attn_fwd: an older build" in said, said
    said = build(tmp_path / "broken.so", [n for n in older if n != "dic_gemm"])
    assert "broken.so does not export dic_gemm" in said and "an older build" not in said, said


def test_a_library_older_than_the_flags_is_not_reused(monkeypatch):
    """The flags decide which instructions the kernels hold, and stand in _lib.py."""
    class Compiles(Exception):
        pass

    def popen(*_, **__):
        raise Compiles

    lib = dic._lib
    monkeypatch.setattr(lib.subprocess, "Popen", popen)
    monkeypatch.setattr(lib, "LAST_BUILD", None)
    monkeypatch.setattr(lib.os.path, "exists", lambda p: True)
    times = {lib.LIB_PATH: 2.0}
    monkeypatch.setattr(lib.os.path, "getmtime", lambda p: times.get(p, 1.0))
    assert lib.build() == lib.LIB_PATH and lib.LAST_BUILD == "reused"
    for newer in (os.path.abspath(lib.__file__), os.path.join(lib.CSRC, "wattn.hip"), os.path.join(ROOT, "include", "dic_hip.h")):
        times[newer] = 3.0
        with pytest.raises(Compiles):
            lib.build()
        del times[newer]


def test_the_script_for_variants_builds_every_source_with_its_flags(tmp_path):
    """scripts/build_variant.sh in a copy of the tree's layout, with a compiler that writes down how it is called."""
    import shutil
    import subprocess
    root, log = tmp_path / "tree", tmp_path / "calls"
    (root / "scripts").mkdir(parents=True)
    shutil.copy(os.path.join(ROOT, "scripts", "build_variant.sh"), root / "scripts")
    os.symlink(os.path.dirname(dic._lib.__file__), root / "diffusion-image-captioning_amd")
    hipcc = tmp_path / "hipcc"
    hipcc.write_text('#!/bin/bash\necho "$@" >> %s\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then touch "$2"; fi; shift; done\n' % log)
    hipcc.chmod(0o755)
    run = subprocess.run(["bash", str(root / "scripts" / "build_variant.sh"), "x", "-DONE -DTWO=2"], env={**os.environ, "HIPCC": str(hipcc)}, capture_output=True, text=True)
    assert run.returncode == 0 and (root / "abl" / "libdic_x.so").exists(), run.stderr
    calls = log.read_text().splitlines()
    for s in dic._lib.SOURCES:
        call, = (c for c in calls if f"/{s} " in c)
        assert "-DONE -DTWO=2" in call and ("-packed-fp32-ops" in call) == (s in dic._lib.NO_PACKED_F32_SOURCES) and ("-ffp-contract=off" in call) == (s == "misc.hip"), call
    link, = (c for c in calls if "-shared" in c)
    assert all(f"/{s[:-4]}.o" in link for s in dic._lib.SOURCES)
