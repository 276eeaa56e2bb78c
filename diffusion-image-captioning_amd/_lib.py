"""Builds and loads `libdic_hip.so` (the C-ABI of include/dic_hip.h) and exposes thin ctypes callers.

No CPU fallback exists: every op goes through the HIP library, and a missing library or missing GPU is a
loud `RuntimeError` (GPU tests cannot pass on a silent eager path).
"""
from __future__ import annotations

import ctypes as C
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_PATH = os.path.join(HERE, "libdic_hip.so")
_AB_LIB = os.environ.get("DIC_HIP_LIB")      # measurement aid: load another build of the same library for within-run A/B timing
SOURCES = ["gemm.hip", "attn.hip", "norm.hip", "misc.hip", "wattn.hip", "gnorm.hip"]
# Packed fp32 instructions off: some of their forms have given wrong results now and then.  gemm.hip holds them in its generated assembly text, which the
# assembler would refuse under this feature setting.
NO_PACKED_F32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
NO_PACKED_F32_SOURCES = ("wattn.hip", "gnorm.hip")

DIC_F32, DIC_BF16 = 0, 1
ABI_VERSION = 19          # include/dic_hip.h DIC_HIP_VERSION the struct mirrors / argtypes below were written for; lib() refuses any other library
EPI_AFFINE, EPI_BIAS_GELU, EPI_GELU_BWD, EPI_CE_PARTIAL, EPI_CE_DLOGITS, EPI_CE_EXP, EPI_BIAS_GELU_D, EPI_MUL_AUX = range(8)

EXPORTS = [
    "dic_version", "dic_last_error", "dic_gemm", "dic_gemm_set_two_heights", "dic_gemm_set_w4a", "dic_gemm_two_heights_plan", "dic_gemm_w4a_rows_plan", "dic_ce_combine", "dic_ce_target_logit", "dic_head_center", "dic_head_center_ws_bytes", "dic_ce_exp_combine", "dic_add_rows_scaled", "dic_embed_gather", "dic_qsample",
    "dic_fuse_ln_fwd", "dic_fuse_ln_bwd", "dic_ln_fwd", "dic_ln_fwd_r32", "dic_ln_bwd", "dic_lo_mean_bias", "dic_lo_mean_bias_ws_bytes", "dic_gelu_ln_fwd", "dic_gelu_ln_bwd",
    "dic_attn_fwd", "dic_attn_bwd", "dic_emb_loss", "dic_add_rows", "dic_seg_sum", "dic_cfg_mix_fwd",
    "dic_cfg_mix_bwd", "dic_seq_sum", "dic_colsum", "dic_colsum_pair", "dic_adamw", "dic_adamw_hl", "dic_cast_bf16", "dic_cast_bf16_hl", "dic_probe_tr16", "dic_prof_begin", "dic_prof_end", "dic_prof_algorithmic_bytes", "dic_prof_get",
    "dic_gemm_split_ws_bytes", "dic_ce_n_partials", "dic_ce_partial_bytes", "dic_colsum_ws_bytes", "dic_ln_partial_bytes",
    "dic_te_dx0", "dic_embed_scatter", "dic_temb_grad", "dic_step_prep", "dic_randint", "dic_zero", "dic_wgrad_group", "dic_wgrad_group_ws_bytes",
    "dic_gemm_set_variant", "dic_fuse_ln_fwd_x", "dic_cfg_prep", "dic_step_ctx_set", "dic_step_advance",
    "dic_lin_prep", "dic_lin_prep_ws_bytes", "dic_ln_fwd_cen", "dic_ln_bwd_cen", "dic_set_option", "dic_rank1_add",
    "dic_win_attn_fwd", "dic_win_attn_bwd", "dic_win_attn_ws_bytes", "dic_gated_norm_fwd", "dic_gated_norm_bwd", "dic_gated_norm_ws_bytes",
]
# Entries that came without a change to what was there before, at the same version: a library loaded through DIC_HIP_LIB may be older, and what it has is used.
LATER_EXPORTS = ("dic_win_attn_fwd", "dic_win_attn_bwd", "dic_win_attn_ws_bytes", "dic_gated_norm_fwd", "dic_gated_norm_bwd", "dic_gated_norm_ws_bytes")


class GemmParams(C.Structure):
    _fields_ = [
        ("A", C.c_void_p), ("B", C.c_void_p), ("C", C.c_void_p),
        ("M", C.c_int), ("N", C.c_int), ("K", C.c_int),
        ("lda", C.c_int), ("ldb", C.c_int), ("ldc", C.c_int),
        ("bias", C.c_void_p),
        ("R", C.c_void_p), ("ldr", C.c_int),
        ("aux", C.c_void_p), ("ldaux", C.c_int),
        ("p_drop", C.c_float), ("seed", C.c_uint64),
        ("out_f32", C.c_int), ("accumulate", C.c_int),
        ("tgt", C.c_void_p), ("lse", C.c_void_p), ("partial", C.c_void_p), ("tgt_logit", C.c_void_p),
        ("ce_rows_a", C.c_int), ("ce_scale_a", C.c_float), ("ce_scale_b", C.c_float),
        ("split_k", C.c_int), ("split_ws", C.c_void_p), ("tile", C.c_int), ("cu_cap", C.c_int), ("colsum_out", C.c_void_p),
        ("B2", C.c_void_p),                                          # low-order half of a split weight (bf16 forward GEMMs) or NULL
        ("step_ctr", C.c_void_p), ("step_ctr0", C.c_int64),          # reserved (filled by dic_gemm from the step context)
        ("b2_col0", C.c_int),                                        # with B2: first output column that takes the low-order pass
        ("bias2", C.c_void_p),                                       # bias row behind the dropout (centred residual stream) or NULL
    ]


class WgradItem(C.Structure):
    """Mirror of DicWgradItem (include/dic_hip.h)."""
    _fields_ = [("dY", C.c_void_p), ("ldy", C.c_int), ("X", C.c_void_p), ("ldx", C.c_int), ("dW", C.c_void_p), ("db", C.c_void_p),
                ("M", C.c_int), ("N", C.c_int)]


class WinAttnParams(C.Structure):
    """Mirror of DicWinAttnParams (include/dic_hip.h); a DicStrides member is three int64 in a row."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv")] + [
        (f"{n}_stride_{d}", C.c_int64) for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv") for d in "nth"] + [
        ("key_mask", C.c_void_p), ("kv_len", C.c_void_p), ("q_pos", C.c_void_p),
        ("N", C.c_int), ("Tq", C.c_int), ("Tk", C.c_int), ("H", C.c_int), ("Hkv", C.c_int), ("dh", C.c_int),
        ("left", C.c_int), ("right", C.c_int), ("sinks", C.c_int), ("scale", C.c_float), ("ws", C.c_void_p), ("ws_bytes", C.c_size_t)]


class GatedNormParams(C.Structure):
    """Mirror of DicGatedNormParams (include/dic_hip.h); a DicNorm member is weight, bias, kind, eps."""
    _fields_ = [(n, C.c_void_p) for n in ("x", "y", "x_new", "a", "gate", "saved", "dx_new", "da", "dx", "dy", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b",
                                          "post_weight", "post_bias")] + [
        ("post_kind", C.c_int), ("post_eps", C.c_float), ("pre_weight", C.c_void_p), ("pre_bias", C.c_void_p), ("pre_kind", C.c_int), ("pre_eps", C.c_float),
        ("rows", C.c_int64), ("rows_per_gate", C.c_int64), ("D", C.c_int), ("residual_scale", C.c_float), ("ws", C.c_void_p), ("ws_bytes", C.c_size_t)]


LAST_BUILD = None        # "compiled" | "reused": what the last build() call did (printed by __graft_entry__.build)


def compile_command(source: str, obj: str, extra=()) -> list:
    """The command that compiles one of SOURCES into `obj`."""
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O3", "-std=c++20", "-fPIC", "-Wno-unused-value", *extra, "-c", os.path.join(CSRC, source), "-o", obj]
    if source == "misc.hip":
        # q_sample must round a*x, eps*b and their sum separately to be bit-exact with the reference (ref :360-362);
        # everything in misc.hip is HBM-bound, so no FMA contraction in this file costs nothing
        cmd.insert(3, "-ffp-contract=off")
    if source in NO_PACKED_F32_SOURCES:
        cmd[3:3] = NO_PACKED_F32
    return cmd


def build(verbose: bool = False, force: bool = False) -> str:
    """Compile every HIP source for gfx950 into one shared library, in-tree (it travels with the snapshot).
    force: compile even when the library is newer than every source and this file, which holds the flags (a check that everything builds must compile, not trust mtimes)."""
    global LAST_BUILD
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.abspath(__file__)] + [os.path.join(CSRC, h) for h in ("common.h", "gemm_w4a.h", "gemm_w4a_asm.inc", "gemm_w4n.h", "gemm_w4n_asm.inc")] + [os.path.join(os.path.dirname(HERE), "include", "dic_hip.h")]
    if not force and os.path.exists(LIB_PATH) and all(os.path.getmtime(LIB_PATH) >= os.path.getmtime(d) for d in deps):
        LAST_BUILD = "reused"
        return LIB_PATH
    LAST_BUILD = "compiled"
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs = []
    procs = []
    for s in srcs:
        o = s[:-4] + ".o"
        objs.append(o)
        cmd = compile_command(os.path.basename(s), o)
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for cmd, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError("hipcc failed: " + " ".join(cmd) + "\n" + out.decode(errors="replace"))
        if verbose and out:
            print(out.decode(errors="replace"))
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH] + objs
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if r.returncode != 0:
        raise RuntimeError("link failed: " + r.stdout.decode(errors="replace"))
    return LIB_PATH


_lib = None


def lib():
    """The loaded library; raises if it has not been built (run `python __graft_entry__.py` / `build()`)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: the HIP extension must be built (no CPU fallback exists); "
                               "run __graft_entry__.build()")
        L = C.CDLL(_AB_LIB if _AB_LIB else LIB_PATH)
        for name in EXPORTS:
            if not hasattr(L, name) and not (_AB_LIB and name in LATER_EXPORTS):
                raise RuntimeError(f"{_AB_LIB or LIB_PATH} does not export {name}")
        L.dic_last_error.restype = C.c_char_p
        if L.dic_version() != ABI_VERSION:
            raise RuntimeError(f"{_AB_LIB or LIB_PATH} reports ABI version {L.dic_version()}, this binding was written for {ABI_VERSION} "
                               "(struct layouts / signatures differ): rebuild with __graft_entry__.build()")
        for fn, args in (("dic_gemm_split_ws_bytes", 4), ("dic_ce_partial_bytes", 3), ("dic_colsum_ws_bytes", 3), ("dic_ln_partial_bytes", 3)):
            getattr(L, fn).restype = C.c_size_t
            getattr(L, fn).argtypes = [C.c_int] * args
        L.dic_ce_n_partials.restype = C.c_int
        L.dic_te_dx0.argtypes = [C.c_void_p] * 5 + [C.c_int] * 7 + [C.c_void_p, C.c_void_p]
        L.dic_embed_scatter.argtypes = [C.c_void_p] * 3 + [C.c_int] * 3 + [C.c_void_p, C.c_void_p]
        L.dic_ce_n_partials.argtypes = [C.c_int, C.c_int]
        L.dic_gemm_w4a_rows_plan.argtypes = [C.c_int] * 4
        L.dic_gemm.argtypes = [C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(GemmParams), C.c_void_p]
        P, I, F, U64, I64 = C.c_void_p, C.c_int, C.c_float, C.c_uint64, C.c_int64
        L.dic_ce_combine.argtypes = [P, P, I, I, P, P, P, P]
        L.dic_embed_gather.argtypes = [P, P, P, I, I, I, P, P]
        L.dic_qsample.argtypes = [P, P, P, P, P, P, P, I, I, I, I, U64, P]
        L.dic_fuse_ln_fwd.argtypes = [I, I, P, P, P, P, P, P, P, P, P, P, P, P, P, I, I, I, F, F, U64, P]
        L.dic_fuse_ln_fwd_x.argtypes = [I, I, P, I64, P, P, P, P, P, P, P, P, P, P, P, P, I, I, I, F, F, U64, P]
        L.dic_fuse_ln_bwd.argtypes = [I, I, P, P, P, P, P, P, P, P, P, P, P, P, P, P, I, I, I, I, F, U64, P]
        L.dic_temb_grad.argtypes = [P, P, I, I, I, I, P, P]
        L.dic_ln_fwd.argtypes = [I, P, P, P, P, P, P, I, I, F, P]
        L.dic_ln_fwd_r32.argtypes = [P, P, P, P, P, P, P, I, I, F, P]
        L.dic_lo_mean_bias.argtypes = [P, I, I, I, I, P, I, I, P, P, P, P]
        L.dic_lo_mean_bias_ws_bytes.argtypes = [I]
        L.dic_lo_mean_bias_ws_bytes.restype = C.c_size_t
        L.dic_ln_bwd.argtypes = [I, P, P, P, P, P, P, P, F, U64, P, I, I, I, P]
        L.dic_lin_prep.argtypes = [P, I, I, I, I, P, P, I, I, P, P, I, P, P, P, P, P]
        L.dic_lin_prep_ws_bytes.argtypes = [I]
        L.dic_lin_prep_ws_bytes.restype = C.c_size_t
        L.dic_ln_fwd_cen.argtypes = [P, P, P, P, P, P, P, P, P, I, I, F, P, P, I, I, P, P, P]
        L.dic_rank1_add.argtypes = [P, P, P, I, I, P]
        L.dic_ln_bwd_cen.argtypes = [P, P, P, P, P, P, P, P, F, U64, P, I, I, I, P]
        L.dic_gelu_ln_fwd.argtypes = [I, P, P, P, P, P, P, I, I, F, P]
        L.dic_gelu_ln_bwd.argtypes = [I, P, P, P, P, P, P, P, I, I, I, P]
        L.dic_attn_fwd.argtypes = [I, P, P, P, I, I, I, I, F, U64, P]
        L.dic_attn_bwd.argtypes = [I, P, P, P, P, I, I, I, I, F, U64, P]
        L.dic_emb_loss.argtypes = [I, I, P, P, I, P, P, P, P, I, I, I, I, P]
        L.dic_add_rows.argtypes = [P, P, I, I, I, I, P]
        L.dic_add_rows_scaled.argtypes = [P, P, P, C.c_float, I, I, I, I, P]
        L.dic_ce_target_logit.argtypes = [P, P, P, I, I, I, C.c_float, P, P, P, P]
        L.dic_head_center.argtypes = [P, I, P, I, I, I, I, P, I, P, P, P, P, P]
        L.dic_head_center_ws_bytes.argtypes = [I]
        L.dic_head_center_ws_bytes.restype = C.c_size_t
        L.dic_ce_exp_combine.argtypes = [P, I, P, P, P, I, I, P, I, P, P, P, P]
        L.dic_seg_sum.argtypes = [P, I, I, F, F, P, P, P]
        L.dic_step_prep.argtypes = [P, P, P, P, I, I, I, I, P, P, P, P, P, P, F, F, P]
        L.dic_cfg_prep.argtypes = [P, P, P, P, P, I, I, I, I, I, I, P, P, P, P, P, P, F, F, P, P, P]
        L.dic_randint.argtypes = [P, I, I, U64, P]
        L.dic_step_ctx_set.argtypes = [P, I64, U64, P]
        L.dic_step_advance.argtypes = [P, P]
        L.dic_zero.argtypes = [P, I64, P]
        L.dic_wgrad_group.argtypes = [C.POINTER(WgradItem), I, I, P, C.c_size_t, I, P]
        L.dic_wgrad_group_ws_bytes.argtypes = [C.POINTER(WgradItem), I, I, I]
        L.dic_wgrad_group_ws_bytes.restype = C.c_size_t
        L.dic_cfg_mix_fwd.argtypes = [P, P, P, I, I, F, P]
        L.dic_cfg_mix_bwd.argtypes = [P, P, P, I, I, F, P]
        L.dic_seq_sum.argtypes = [P, P, P, P, I, I, I, P]
        L.dic_colsum.argtypes = [I, P, I, I, I, P, I, P, P]
        L.dic_colsum_pair.argtypes = [P, P, P, P, I, I, I, P]
        L.dic_adamw.argtypes = [P, P, P, P, P, I64, F, F, F, F, F, F, F, F, P]
        L.dic_cast_bf16.argtypes = [P, P, I64, P]
        L.dic_adamw_hl.argtypes = [P, P, P, P, P, P, I64, F, F, F, F, F, F, F, F, P]
        L.dic_cast_bf16_hl.argtypes = [P, P, P, I64, P]
        L.dic_probe_tr16.argtypes = [P, P, P]
        for fn in LATER_EXPORTS:
            if hasattr(L, fn):
                params = C.POINTER(WinAttnParams if "win_attn" in fn else GatedNormParams)
                getattr(L, fn).argtypes = [I, params, P] if not fn.endswith("ws_bytes") else [I, I, params] if "win_attn" in fn else [I, params]
                getattr(L, fn).restype = C.c_size_t if fn.endswith("ws_bytes") else I
        L.dic_gemm_set_variant.argtypes = [I]
        L.dic_set_option.argtypes = [C.c_char_p, I]
        L.dic_gemm_set_w4a.argtypes = [I]
        L.dic_prof_begin.argtypes = [I]
        L.dic_prof_algorithmic_bytes.restype = C.c_double
        L.dic_prof_algorithmic_bytes.argtypes = []
        L.dic_prof_get.argtypes = [I, C.POINTER(C.c_double), C.POINTER(C.c_double), C.POINTER(C.c_double)]
        L.dic_prof_end.argtypes = [C.POINTER(C.c_double), C.POINTER(C.c_double), C.POINTER(C.c_int)]
        from . import options
        options.push_to_library(L)          # the library reads no environment: its process-global switches come from the one record
        _lib = L
    return _lib


def entry(name):
    """A C entry as an object of its own (argument types set on it are seen by nobody else)."""
    try:
        return lib()[name]
    except AttributeError:
        raise RuntimeError(f"{_AB_LIB or LIB_PATH} does not export {name}: an older build, which has other operators only") from None


def loaded() -> bool:
    """True once lib() has dlopened the library in this process."""
    return _lib is not None


def check(rc: int, what: str = ""):
    if rc != 0:
        msg = lib().dic_last_error().decode(errors="replace")
        raise RuntimeError(f"HIP op {what} failed (code {rc}): {msg}")


def require_gpu():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("no MI355X visible: this path has no CPU fallback (the CPU oracle lives under oracle/ "
                           "and is test infrastructure only)")
