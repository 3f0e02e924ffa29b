"""Host-side mirror of the engines' attention ops over the C ABI.

The reference engines launch ``qwen3_attend`` (crates/omni-qwen3/src/stack.rs:
207-241), ``lm_attend`` (crates/omni-personaplex/src/helium.rs:256-275) and
``hidream_attend`` (crates/omni-hidream-o1/src/model.rs:362-380) with raw
device pointers. This module exposes the same calls, argument for argument,
over ``libomni_attn.so`` via ctypes, taking torch tensors only as holders of
device memory and streams. There is no fallback: if the HIP library is absent
or a launch fails, the call raises.
"""
from __future__ import annotations

import ctypes
import os
import sys
from dataclasses import dataclass

# torch brings its own HIP runtime; it is loaded before the library so that the
# library binds to the same one instead of pulling in a second copy from /opt/rocm.
import torch as _torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libomni_attn.so")
HEAD_DIM = 128

OK = 0
EINVAL = -1
EUNSUPPORTED = -2
ELAUNCH = -3
EWORKSPACE = -4
ETABLE = -5

EXPORTS = (
    "omni_attn_decode_plan_init",
    "omni_attn_decode_plan_init_fp8",
    "omni_qwen3_attend",
    "omni_qwen3_attend_noalloc",
    "omni_lm_attend",
    "omni_lm_attend_fp8",
    "omni_attn_decode_run_lastlen",
    "omni_attn_check_table",
    "omni_attn_gather_kv",
    "omni_attn_prefill_plan_init",
    "omni_hidream_rows",
    "omni_attn_prefill_run",
    "omni_hidream_attend",
    "omni_hidream_attend_batched",
    "omni_hidream_attend_ws",
    "omni_hidream_workspace_bytes",
    "omni_qwen3_attend_dense",
    "omni_mimi_attend",
    "omni_mimi_rope_kv",
    "omni_lm_copy_kv",
    "omni_codec_attention",
    "omni_lm_dep_kv_attend",
    "omni_qwen3_rope",
    "omni_qwen3_rope_dense",
    "omni_qwen3_rope_attend",
    "omni_lm_rope_attend_fp8",
    "omni_lm_rope",
    "omni_hidream_qk_rope",
    "omni_attn_step_tables",
    "omni_qwen3_rope_q8",
    "omni_attn_decode_plan_init_q8",
    "omni_qwen3_attend_q8",
    "omni_attn_prompt_plan_init",
    "omni_attn_prompt_run",
    "omni_attn_extend_plan_init",
    "omni_attn_cross_plan_init",
    "omni_qwen3_extend_q8",
    "omni_attn_cross_run",
    "omni_attn_pages_fork",
    "omni_attn_pages_free",
    "omni_attn_pages_compact",
    "omni_attn_pages_copy",
    "omni_attn_rows_new",
    "omni_attn_rows_free",
    "omni_attn_rows_clear",
    "omni_attn_rows_push",
    "omni_attn_rows_count",
    "omni_attn_rows_get",
    "omni_attn_version",
    "omni_attn_last_error",
)


class OmniAttnError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"omni_attn error {code}: {msg}")
        self.code = code


class DecodePlan(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int32),
        ("hq", ctypes.c_int32),
        ("hk", ctypes.c_int32),
        ("page", ctypes.c_int32),
        ("max_len", ctypes.c_int32),
        ("chunk", ctypes.c_int32),
        ("splits", ctypes.c_int32),
        ("group_heads", ctypes.c_int32),  # FP8 kernel: heads per workgroup, 0 = auto
        ("workspace_bytes", ctypes.c_int64),
    ]


class PrefillPlan(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int32),
        ("hq", ctypes.c_int32),
        ("hk", ctypes.c_int32),
        ("page", ctypes.c_int32),
        ("tiles", ctypes.c_int32),
        ("tile_rows", ctypes.c_int32),
        ("work_bytes", ctypes.c_int64),
        ("workgroups", ctypes.c_int32),
        ("exact_p", ctypes.c_int32),
    ]


class PromptPlan(ctypes.Structure):
    _fields_ = [
        ("nseq", ctypes.c_int32),
        ("rows", ctypes.c_int32),
        ("hq", ctypes.c_int32),
        ("hk", ctypes.c_int32),
        ("tiles", ctypes.c_int32),
        ("tile_rows", ctypes.c_int32),
        ("workgroups", ctypes.c_int32),
        ("exact_p", ctypes.c_int32),
        ("work_bytes", ctypes.c_int64),
    ]


class MultiPlan(ctypes.Structure):
    _fields_ = [
        ("cross", ctypes.c_int32),
        ("nseq", ctypes.c_int32),
        ("rows", ctypes.c_int32),
        ("hq", ctypes.c_int32),
        ("hk", ctypes.c_int32),
        ("max_len", ctypes.c_int32),
        ("groups", ctypes.c_int32 * 2),
        ("group_rows", ctypes.c_int32),
        ("chunk", ctypes.c_int32),
        ("splits", ctypes.c_int32),
        ("tiles", ctypes.c_int32),
        ("tile_chunk", ctypes.c_int32),
        ("tile_units", ctypes.c_int32),
        ("split_tiles", ctypes.c_int32),
        ("tile_segments", ctypes.c_int32),
        ("exact_p", ctypes.c_int32),
        ("work_bytes", ctypes.c_int64),
        ("workspace_bytes", ctypes.c_int64),
    ]


_lib = None


def load(path: str | None = None):
    """Load the HIP library (raises if it was not built). OMNI_ATTN_LIB names
    another build of the same library (A/B measurements)."""
    global _lib
    if _lib is not None:
        return _lib
    path = path or os.environ.get("OMNI_ATTN_LIB") or LIB_PATH
    if not os.path.exists(path):
        raise OmniAttnError(ELAUNCH, f"{path} is missing: build it with pega-omni_amd/build.py")
    L = ctypes.CDLL(path)
    P, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
    dplan = ctypes.POINTER(DecodePlan)
    pplan = ctypes.POINTER(PrefillPlan)
    qplan = ctypes.POINTER(PromptPlan)
    mplan = ctypes.POINTER(MultiPlan)
    sig = {
        "omni_attn_decode_plan_init": [i32, i32, i32, i32, i32, i32, dplan],
        "omni_attn_decode_plan_init_fp8": [i32, i32, i32, i32, i32, dplan],
        "omni_qwen3_attend": [P, P, P, P, i32, P, P, i32, P, i32, i32, f32, dplan, P, P],
        "omni_qwen3_attend_noalloc": [P, P, P, P, i32, P, P, i32, P, i32, i32, f32, dplan, P],
        "omni_lm_attend": [P, P, P, P, i32, P, P, i32, P, i32, f32, i32, dplan, P, P],
        "omni_lm_attend_fp8": [P, P, P, P, i32, P, P, i32, P, i32, f32, i32, dplan, P, P],
        "omni_attn_decode_run_lastlen": [P, P, P, P, i32, P, P, i32, P, i32, i32, f32, dplan, P, P],
        "omni_attn_check_table": [P, i32, P, i32, P, P, i32, i32, i32, i32],
        "omni_attn_gather_kv": [P, i32, P, P, i32, P, P, P, i32, P, P],
        "omni_attn_prefill_plan_init": [i32, i32, i32, i32, P, P, P, i64, pplan],
        "omni_hidream_rows": [i32, i32, i32, i32, P, P, P, P, P],
        "omni_attn_prefill_run": [pplan, P, P, P, P, P, P, P, f32, P, P],
        "omni_hidream_attend": [P, P, P, P, i32, P, i32, i32, f32, i32, i32, P],
        "omni_hidream_attend_batched": [P, P, P, P, i32, P, i32, i32, f32, i32, i32, i32, i64, i64, i64, P],
        "omni_hidream_attend_ws": [P, P, P, P, i32, P, i32, i32, f32, i32, i32, i32, i64, i64, i64, P, i64, P],
        "omni_hidream_workspace_bytes": [],
        "omni_qwen3_attend_dense": [P, P, i32, i32, i32, P, i32, i32, f32, dplan, P, P],
        "omni_mimi_attend": [P, P, P, P, P, i32, i32, i32, f32, i32, i64, P],
        "omni_mimi_rope_kv": [P, P, P, P, i32, i32, i32, f32, i32, i64, P],
        "omni_lm_copy_kv": [P, P, P, i32, i32, P],
        "omni_codec_attention": [P, P, P, P, P, i32, i64, i32, f32, P],
        "omni_lm_dep_kv_attend": [P, P, i32, P, i32, i32, f32, P],
        "omni_qwen3_rope": [P, P, P, P, P, P, i32, i32, i32, f32, f32, P],
        "omni_qwen3_rope_dense": [P, P, P, P, i32, i32, i32, i32, i32, i32, f32, f32, P],
        "omni_qwen3_rope_attend": [P, P, P, P, P, P, P, P, i32, P, i32, i32, f32, f32, f32, dplan, P, P],
        "omni_lm_rope_attend_fp8": [P, P, P, P, P, P, i32, P, i32, f32, f32, i32, dplan, P, P],
        "omni_lm_rope": [P, P, P, P, i32, i32, f32, P],
        "omni_hidream_qk_rope": [P, i32, P, P, P, P, P, P, i32, i32, i32, i32, f32, f32, P],
        "omni_attn_version": [],
        "omni_attn_last_error": [],
    }
    sig.update({
        "omni_attn_step_tables": [P, P, P, i32, i32, i32, P, i64, i32, P, i32, P, i32, i32, P, P, P, P, P, P, P, P],
        "omni_qwen3_rope_q8": [P, i64, P, P, P, P, P, i64, P, i64, P, P, i32, i32, i32, i32, f32, f32, P],
        "omni_attn_decode_plan_init_q8": [i32, i32, i32, i32, i32, i32, dplan],
        "omni_qwen3_attend_q8": [P, i64, P, P, i32, P, P, i32, P, P, i32, P, i32, i32, f32, dplan, P, P],
        "omni_attn_prompt_plan_init": [i32, P, i32, i32, P, i64, qplan],
        "omni_attn_prompt_run": [qplan, P, i64, P, i64, P, i64, P, f32, P, P],
        "omni_attn_extend_plan_init": [i32, P, P, i32, i32, i32, i32, P, i64, mplan],
        "omni_attn_cross_plan_init": [i32, P, P, i32, i32, i32, i32, P, i64, mplan],
        "omni_qwen3_extend_q8": [mplan, P, i64, P, P, i32, P, P, P, i32, P, f32, P, P, P],
        "omni_attn_cross_run": [mplan, P, i64, P, i64, P, i64, P, P, P, P, f32, P, P, P],
        "omni_attn_pages_fork": [P, P, P, i32, i32, P, i64, i32, P, i32, P, P, P, P, P, P],
        "omni_attn_pages_free": [P, P, i32, i32, P, i64, i32, P, i32, P, P, P, P],
        "omni_attn_pages_compact": [P, i64, i32, P, i32, P, P, i32, P, P, P, P, P, P, i32, P, P],
        "omni_attn_pages_copy": [P, i64, i64, P, i64, i64, i32, i32, P, P, i32, P, P],
        "omni_attn_rows_new": [i32, i32],
        "omni_attn_rows_free": [P],
        "omni_attn_rows_clear": [P],
        "omni_attn_rows_push": [P, P, i32, i32, i32, i32],
        "omni_attn_rows_count": [P, P, P, P],
        "omni_attn_rows_get": [P, i32],
    })
    for name, args in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = (ctypes.c_char_p if name == "omni_attn_last_error"
                      else ctypes.c_int64 if name == "omni_hidream_workspace_bytes"
                      else ctypes.c_void_p if name == "omni_attn_rows_new"
                      else ctypes.POINTER(ctypes.c_int32) if name == "omni_attn_rows_get"
                      else None if name in ("omni_attn_rows_free", "omni_attn_rows_clear") else ctypes.c_int)
    _lib = L
    return L


def _check(rc: int):
    if rc != OK:
        raise OmniAttnError(rc, load().omni_attn_last_error().decode())


# A call's host time is most of a small launch's (4 sessions of one talker
# layer: 13 us of host against 11 us of kernels), so the checks below read each
# attribute once, pointers go to ctypes as plain integers (every pointer
# parameter is declared c_void_p) and the stream is asked for as a raw handle
# instead of a torch.cuda.Stream object (torch's own call for it is not a public
# one: where a build lacks it, the public one answers).
_raw_stream = getattr(_torch._C, "_cuda_getCurrentRawStream", None)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream):
    if stream is None:
        if _raw_stream is not None:
            return _raw_stream(_torch.cuda.current_device())
        stream = _torch.cuda.current_stream()
    return stream.cuda_stream


def _bf16_dev(t, name):
    if t.dtype != _torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
        raise OmniAttnError(EINVAL, f"{name} must be a contiguous bf16 device tensor")


def _i32_dev(t, name):
    if t is None:
        return
    if t.dtype != _torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise OmniAttnError(EINVAL, f"{name} must be a contiguous int32 device tensor")


def _ws(plan, workspace):
    """The workspace pointer for a decode run, after checking that it holds the
    plan's split partials (the C call takes no size: a smaller buffer would be
    written past its end)."""
    if workspace is None:
        return None
    need = plan.workspace_bytes
    if workspace.nbytes < need:
        raise OmniAttnError(EWORKSPACE, f"workspace holds {workspace.nbytes} bytes, the plan needs {need}")
    if not workspace.is_cuda or not workspace.is_contiguous():
        raise OmniAttnError(EINVAL, "workspace must be a contiguous device tensor")
    return workspace.data_ptr()


# --------------------------------------------------------------------- decode
def decode_plan(rows: int, hq: int, hk: int, page: int, max_len: int, chunk: int = 0) -> DecodePlan:
    plan = DecodePlan()
    _check(load().omni_attn_decode_plan_init(rows, hq, hk, page, max_len, chunk, ctypes.byref(plan)))
    return plan


def decode_plan_fp8(rows: int, heads: int, page: int, max_len: int, chunk: int = 0) -> DecodePlan:
    """The plan for lm_attend over FP8 slots (split size picked for the FP8 kernel)."""
    plan = DecodePlan()
    _check(load().omni_attn_decode_plan_init_fp8(rows, heads, page, max_len, chunk, ctypes.byref(plan)))
    return plan


def workspace_for(plan, device="cuda"):
    """Device workspace for a plan (None when the plan needs none)."""
    n = int(plan.workspace_bytes)
    return _torch.empty(n, dtype=_torch.uint8, device=device) if n > 0 else None


def check_table(indptr_h, pages_h, num_pages, pos_h=None, seq_h=None, ragged=False, page=16, context=0):
    """Host validation of a page table (numpy int32 arrays)."""
    import numpy as np

    indptr_h = np.ascontiguousarray(indptr_h, dtype=np.int32)
    pages_h = np.ascontiguousarray(pages_h, dtype=np.int32)
    rows = 0 if pos_h is None else len(pos_h)
    pos_a = None if pos_h is None else np.ascontiguousarray(pos_h, dtype=np.int32)
    seq_a = None if seq_h is None else np.ascontiguousarray(seq_h, dtype=np.int32)
    rc = load().omni_attn_check_table(
        indptr_h.ctypes.data_as(ctypes.c_void_p), len(indptr_h) - 1, pages_h.ctypes.data_as(ctypes.c_void_p),
        num_pages, None if pos_a is None else pos_a.ctypes.data_as(ctypes.c_void_p),
        None if seq_a is None else seq_a.ctypes.data_as(ctypes.c_void_p), int(ragged), rows, page, context)
    _check(rc)


def qwen3_attend(qkv, kv, pos, seq, ragged, indptr, pages, page, out, hq, hk, scale, plan, workspace=None,
                 stream=None):
    """``qwen3_attend`` (crates/omni-qwen3/kernels/qwen3.cu:234-240) on the GPU."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(kv, "kv"), _bf16_dev(out, "out")
    for t, n in ((pos, "pos"), (seq, "seq"), (indptr, "indptr"), (pages, "pages")):
        _i32_dev(t, n)
    _check(load().omni_qwen3_attend(_ptr(qkv), _ptr(kv), _ptr(pos), _ptr(seq), int(ragged), _ptr(indptr),
                                    _ptr(pages), page, _ptr(out), hq, hk, float(scale), ctypes.byref(plan),
                                    _ws(plan, workspace), _stream(stream)))
    return out


def qwen3_attend_noalloc(qkv, kv, pos, seq, ragged, indptr, pages, page, out, hq, hk, scale, plan, stream=None):
    """``qwen3_attend`` without a workspace argument: the split partials go to
    the library's static per-GPU scratch (no allocation; calls that overlap on
    one GPU race). No counterpart in the reference."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(kv, "kv"), _bf16_dev(out, "out")
    for t, n in ((pos, "pos"), (seq, "seq"), (indptr, "indptr"), (pages, "pages")):
        _i32_dev(t, n)
    _check(load().omni_qwen3_attend_noalloc(_ptr(qkv), _ptr(kv), _ptr(pos), _ptr(seq), int(ragged), _ptr(indptr),
                                            _ptr(pages), page, _ptr(out), hq, hk, float(scale), ctypes.byref(plan),
                                            _stream(stream)))
    return out


def lm_attend(qkv, kv, pos, seq, ragged, indptr, pages, page, out, heads, scale, context, plan, workspace=None,
              stream=None):
    """``lm_attend`` (crates/omni-personaplex/kernels/lm.cu:275-290) over bf16 slots."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(kv, "kv"), _bf16_dev(out, "out")
    for t, n in ((pos, "pos"), (seq, "seq"), (indptr, "indptr"), (pages, "pages")):
        _i32_dev(t, n)
    _check(load().omni_lm_attend(_ptr(qkv), _ptr(kv), _ptr(pos), _ptr(seq), int(ragged), _ptr(indptr), _ptr(pages),
                                 page, _ptr(out), heads, float(scale), context, ctypes.byref(plan),
                                 _ws(plan, workspace), _stream(stream)))
    return out


def lm_attend_fp8(qkv, kv, pos, seq, ragged, indptr, pages, page, out, heads, scale, context, plan, workspace=None,
                  stream=None):
    """``lm_attend`` over FP8 E4M3 slots (crates/omni-personaplex/kernels/lm.cu:196-290).
    kv is a uint8 device tensor of slots of 2*heads*128 + 2*heads*4 bytes."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(out, "out")
    if kv.dtype != _torch.uint8 or not kv.is_cuda or not kv.is_contiguous():
        raise OmniAttnError(EINVAL, "kv must be a contiguous uint8 device tensor of FP8 slots")
    for t, n in ((pos, "pos"), (seq, "seq"), (indptr, "indptr"), (pages, "pages")):
        _i32_dev(t, n)
    _check(load().omni_lm_attend_fp8(_ptr(qkv), _ptr(kv), _ptr(pos), _ptr(seq), int(ragged), _ptr(indptr),
                                     _ptr(pages), page, _ptr(out), heads, float(scale), context, ctypes.byref(plan),
                                     _ws(plan, workspace), _stream(stream)))
    return out


def decode_lastlen(qkv, kv, last_page_len, seq, ragged, indptr, pages, page, out, hq, hk, scale, plan,
                   workspace=None, stream=None):
    """Decode with per-sequence last-page lengths instead of positions."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(kv, "kv"), _bf16_dev(out, "out")
    _check(load().omni_attn_decode_run_lastlen(_ptr(qkv), _ptr(kv), _ptr(last_page_len), _ptr(seq), int(ragged),
                                               _ptr(indptr), _ptr(pages), page, _ptr(out), hq, hk, float(scale),
                                               ctypes.byref(plan), _ws(plan, workspace), _stream(stream)))
    return out


def gather_kv(kv, hk, indptr, pages, page, seq_ids, lens, out_indptr, out, stream=None):
    """Bit-exact paged -> dense copy of K/V slots (the page-table rule)."""
    nseq = int(seq_ids.numel())
    _check(load().omni_attn_gather_kv(_ptr(kv), hk, _ptr(indptr), _ptr(pages), page, _ptr(seq_ids), _ptr(lens),
                                      _ptr(out_indptr), nseq, _ptr(out), _stream(stream)))
    return out


# -------------------------------------------------------------------- prefill
@dataclass
class Prefill:
    plan: PrefillPlan
    work: object  # device int32 tensor


def prefill_plan(rows, hq, hk, page, seq_h, pos_h, device="cuda", exact_p=False) -> Prefill:
    """Host plan of a ragged causal prefill; uploads the work list. exact_p:
    P carried as two bf16 terms through P.V (qwen3_attend's f32 P, ~1.4x the time)."""
    import numpy as np
    seq_a = np.ascontiguousarray(seq_h, dtype=np.int32)
    pos_a = np.ascontiguousarray(pos_h, dtype=np.int32)
    plan = PrefillPlan()
    L = load()
    rc = L.omni_attn_prefill_plan_init(rows, hq, hk, page, seq_a.ctypes.data_as(ctypes.c_void_p),
                                       pos_a.ctypes.data_as(ctypes.c_void_p), None, 0, ctypes.byref(plan))
    if rc not in (OK, EWORKSPACE):
        _check(rc)
    cap = max(1, int(plan.work_bytes) // 4)
    work_h = np.zeros(cap, dtype=np.int32)
    _check(L.omni_attn_prefill_plan_init(rows, hq, hk, page, seq_a.ctypes.data_as(ctypes.c_void_p),
                                         pos_a.ctypes.data_as(ctypes.c_void_p),
                                         work_h.ctypes.data_as(ctypes.c_void_p), cap, ctypes.byref(plan)))
    plan.exact_p = 1 if exact_p else 0
    return Prefill(plan, _torch.from_numpy(work_h).to(device))


def prefill_run(pf: Prefill, qkv, kv, pos, seq, indptr, pages, out, scale, stream=None):
    """Ragged causal prefill with qwen3_attend(ragged = 1) semantics (MFMA)."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(kv, "kv"), _bf16_dev(out, "out")
    _check(load().omni_attn_prefill_run(ctypes.byref(pf.plan), _ptr(qkv), _ptr(kv), _ptr(pos), _ptr(seq),
                                        _ptr(indptr), _ptr(pages), _ptr(out), float(scale), _ptr(pf.work),
                                        _stream(stream)))
    return out


# ------------------------------------------------------------------------ DiT
def hidream_attend(q, k, v, out, q_len, kv_len_at, q_stride, causal, scale_log2, hq, hk, stream=None):
    """``hidream_attend`` (crates/omni-hidream-o1/kernels/hidream.cu:209-347)."""
    _check(load().omni_hidream_attend(_ptr(q), _ptr(k), _ptr(v), _ptr(out), q_len, _ptr(kv_len_at), q_stride,
                                      int(causal), float(scale_log2), hq, hk, _stream(stream)))
    return out


def hidream_attend_batched(q, k, v, out, q_len, kv_len_at, q_stride, causal, scale_log2, hq, hk, batch, q_bstride,
                           kv_bstride, out_bstride, stream=None):
    _check(load().omni_hidream_attend_batched(_ptr(q), _ptr(k), _ptr(v), _ptr(out), q_len, _ptr(kv_len_at), q_stride,
                                              int(causal), float(scale_log2), hq, hk, batch, q_bstride, kv_bstride,
                                              out_bstride, _stream(stream)))
    return out


# ------------------------------------------------ rotary embedding + K/V scatter
def qwen3_rope(qkv, q_norm, k_norm, pos, slots, kv, rows, hq, hk, eps, theta, stream=None):
    """``qwen3_rope`` (crates/omni-qwen3/kernels/qwen3.cu:64-103): q rotated in
    place, K and V written to slot ``slots[n]`` of the bf16 paged cache."""
    for t, n in ((qkv, "qkv"), (q_norm, "q_norm"), (k_norm, "k_norm"), (kv, "kv")):
        _bf16_dev(t, n)
    _i32_dev(pos, "pos"), _i32_dev(slots, "slots")
    _check(load().omni_qwen3_rope(_ptr(qkv), _ptr(q_norm), _ptr(k_norm), _ptr(pos), _ptr(slots), _ptr(kv), rows, hq,
                                  hk, float(eps), float(theta), _stream(stream)))


def qwen3_rope_attend(qkv, q_norm, k_norm, pos, slots, kv, indptr, pages, page, out, hq, hk, eps, theta, scale, plan,
                      workspace=None, stream=None):
    """``qwen3_rope`` then ``qwen3_attend`` (ragged = 0) in one launch: K and V
    of row n written to ``slots[n]`` (which must be the slot of key pos[n]),
    q rotated in registers only (qkv is not written)."""
    for t, n in ((qkv, "qkv"), (q_norm, "q_norm"), (k_norm, "k_norm"), (kv, "kv"), (out, "out")):
        _bf16_dev(t, n)
    for t, n in ((pos, "pos"), (slots, "slots"), (indptr, "indptr"), (pages, "pages")):
        _i32_dev(t, n)
    _check(load().omni_qwen3_rope_attend(_ptr(qkv), _ptr(q_norm), _ptr(k_norm), _ptr(pos), _ptr(slots), _ptr(kv),
                                         _ptr(indptr), _ptr(pages), page, _ptr(out), hq, hk, float(eps), float(theta),
                                         float(scale), ctypes.byref(plan), _ws(plan, workspace), _stream(stream)))
    return out


def lm_rope_attend_fp8(qkv, pos, slots, kv, indptr, pages, page, out, heads, coef, scale, context, plan,
                       workspace=None, stream=None):
    """``lm_rope`` then ``lm_attend`` over FP8 slots (ragged = 0) in one launch:
    K and V of row n quantized into ``slots[n]`` (which must be the slot of ring
    index pos[n] % context), q rotated in registers only (qkv is not written)."""
    for t, n in ((qkv, "qkv"), (out, "out")):
        _bf16_dev(t, n)
    if kv.dtype != _torch.uint8 or not kv.is_cuda or not kv.is_contiguous():
        raise OmniAttnError(EINVAL, "kv must be a contiguous uint8 device tensor of FP8 slots")
    for t, n in ((pos, "pos"), (slots, "slots"), (indptr, "indptr"), (pages, "pages")):
        _i32_dev(t, n)
    _check(load().omni_lm_rope_attend_fp8(_ptr(qkv), _ptr(pos), _ptr(slots), _ptr(kv), _ptr(indptr), _ptr(pages), page,
                                          _ptr(out), heads, float(coef), float(scale), context, ctypes.byref(plan),
                                          _ws(plan, workspace), _stream(stream)))
    return out


def qwen3_rope_dense(qkv, q_norm, k_norm, kv, rows, per, base, span, hq, hk, eps, theta, stream=None):
    """``qwen3_rope_dense`` (qwen3.cu:105-111)."""
    for t, n in ((qkv, "qkv"), (q_norm, "q_norm"), (k_norm, "k_norm"), (kv, "kv")):
        _bf16_dev(t, n)
    _check(load().omni_qwen3_rope_dense(_ptr(qkv), _ptr(q_norm), _ptr(k_norm), _ptr(kv), rows, per, base, span, hq,
                                        hk, float(eps), float(theta), _stream(stream)))


def lm_rope(qkv, pos, slots, kv, rows, heads, coef, stream=None):
    """``lm_rope`` (crates/omni-personaplex/kernels/lm.cu:125-182): kv is a
    uint8 device tensor of FP8 slots."""
    _bf16_dev(qkv, "qkv"), _i32_dev(pos, "pos"), _i32_dev(slots, "slots")
    if kv.dtype != _torch.uint8 or not kv.is_cuda or not kv.is_contiguous():
        raise OmniAttnError(EINVAL, "kv must be a contiguous uint8 device tensor of FP8 slots")
    _check(load().omni_lm_rope(_ptr(qkv), _ptr(pos), _ptr(slots), _ptr(kv), rows, heads, float(coef),
                               _stream(stream)))


def hidream_qk_rope(qkv, ld, q_norm, k_norm, positions, slots, k_cache, v_cache, rows, hq, hk, mrope_hw, eps, theta,
                    stream=None):
    """``hidream_qk_rope`` (crates/omni-hidream-o1/kernels/hidream.cu:55-106)."""
    for t, n in ((qkv, "qkv"), (q_norm, "q_norm"), (k_norm, "k_norm"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _bf16_dev(t, n)
    _i32_dev(positions, "positions"), _i32_dev(slots, "slots")
    _check(load().omni_hidream_qk_rope(_ptr(qkv), ld, _ptr(q_norm), _ptr(k_norm), _ptr(positions), _ptr(slots),
                                       _ptr(k_cache), _ptr(v_cache), rows, hq, hk, mrope_hw, float(eps),
                                       float(theta), _stream(stream)))


# ------------------------------------------------- dense and head-64 attentions
def qwen3_attend_dense(qkv, kv, per, base, span, out, hq, hk, scale, plan, workspace=None, stream=None):
    """``qwen3_attend_dense`` (crates/omni-qwen3/kernels/qwen3.cu:243-248); the
    plan is made with page = 1 and max_len >= base + per."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(kv, "kv"), _bf16_dev(out, "out")
    _check(load().omni_qwen3_attend_dense(_ptr(qkv), _ptr(kv), per, base, span, _ptr(out), hq, hk, float(scale),
                                          ctypes.byref(plan), _ws(plan, workspace), _stream(stream)))
    return out


def mimi_rope_kv(qkv, pos, lines, state, rows, T, heads, coef, context, stride, stream=None):
    """``mimi_rope_kv`` (crates/omni-personaplex/kernels/mimi.cu:226-246): q turned
    in place, k turned and v copied into each row's ring slot of ``state``."""
    _bf16_dev(qkv, "qkv"), _i32_dev(pos, "pos"), _i32_dev(lines, "lines")
    _check(load().omni_mimi_rope_kv(_ptr(qkv), _ptr(pos), _ptr(lines), _ptr(state), rows, T, heads, float(coef),
                                    context, int(stride), _stream(stream)))
    return qkv


def lm_copy_kv(kv, src_slot, dst_slot, tokens, slot_bytes, stream=None):
    """``lm_copy_kv`` (crates/omni-personaplex/kernels/lm.cu:583-593): slot
    dst_slot[r] takes the bytes of slot src_slot[r] (prefix K/V reuse)."""
    _i32_dev(src_slot, "src_slot"), _i32_dev(dst_slot, "dst_slot")
    _check(load().omni_lm_copy_kv(_ptr(kv), _ptr(src_slot), _ptr(dst_slot), tokens, slot_bytes, _stream(stream)))
    return kv


def mimi_attend(qkv, pos, lines, state, out, rows, T, heads, scale, context, stride, stream=None):
    """``mimi_attend`` (crates/omni-personaplex/kernels/mimi.cu:248-263); state is
    any contiguous device tensor holding the per-session rings."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(out, "out"), _i32_dev(pos, "pos"), _i32_dev(lines, "lines")
    _check(load().omni_mimi_attend(_ptr(qkv), _ptr(pos), _ptr(lines), _ptr(state), _ptr(out), rows, T, heads,
                                   float(scale), context, int(stride), _stream(stream)))
    return out


def codec_attention(qkv, pos, lines, kv, out, rows, stride, heads, theta, stream=None):
    """``codec_attention`` (crates/omni-qwen3-tts/kernels/codec.cu:168-277)."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(out, "out"), _i32_dev(pos, "pos"), _i32_dev(lines, "lines")
    _check(load().omni_codec_attention(_ptr(qkv), _ptr(pos), _ptr(lines), _ptr(kv), _ptr(out), rows, int(stride),
                                       heads, float(theta), _stream(stream)))
    return out


def lm_dep_kv_attend(qkv, ws, step, out, rows, heads, scale, stream=None):
    """``lm_dep_kv_attend`` (crates/omni-personaplex/kernels/lm.cu:314-366)."""
    _bf16_dev(qkv, "qkv"), _bf16_dev(ws, "ws"), _bf16_dev(out, "out")
    _check(load().omni_lm_dep_kv_attend(_ptr(qkv), _ptr(ws), step, _ptr(out), rows, heads, float(scale),
                                        _stream(stream)))
    return out


def hidream_workspace(device="cuda"):
    """A workspace for hidream_attend_ws on the current device."""
    return _torch.empty(int(load().omni_hidream_workspace_bytes()), dtype=_torch.uint8, device=device)


def hidream_attend_ws(q, k, v, out, q_len, kv_len_at, q_stride, causal, scale_log2, hq, hk, batch, q_bstride,
                      kv_bstride, out_bstride, workspace, stream=None):
    """The batched DiT call with the tail split (a workspace from hidream_workspace)."""
    nbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(load().omni_hidream_attend_ws(_ptr(q), _ptr(k), _ptr(v), _ptr(out), q_len, _ptr(kv_len_at), q_stride,
                                         int(causal), float(scale_log2), hq, hk, batch, int(q_bstride),
                                         int(kv_bstride), int(out_bstride), _ptr(workspace), nbytes,
                                         _stream(stream)))
    return out


# ------------------------------------------ serving over an 8-bit block cache
TABLES_OK, TABLES_BAD, TABLES_ROWS, TABLES_PAGES, TABLES_LINE, TABLES_EXHAUSTED = range(6)
_Q8_DTYPES = (_torch.float8_e4m3fn, _torch.int8)


# A call launches on the current device, whose stream it takes: every tensor has
# to lie there. omni_tensors checks them all in one call (its source lists the
# kinds); the device is asked for once (the raw call where torch has it; -1, where
# nothing lies, if the first tensor is the host's).
_current_device = getattr(_torch._C, "_cuda_getDevice", None) or _torch.cuda.current_device


def _load_tensors():
    import importlib.machinery
    import importlib.util

    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "omni_tensors.so")
    if not os.path.exists(path):
        raise OmniAttnError(ELAUNCH, f"{path} is missing: build it with pega-omni_amd/build.py")
    loader = importlib.machinery.ExtensionFileLoader("omni_tensors", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("omni_tensors", loader))
    loader.exec_module(module)
    here = "torch %s, Python %d.%d" % (_torch.__version__, *sys.version_info[:2])
    if module.built_for != here:
        raise OmniAttnError(ELAUNCH, f"{path} was built for {module.built_for}, this is {here}: build it again")
    module.set_error(OmniAttnError, EINVAL)
    return module


def _take(*args):
    """omni_tensors.take, in whose place it stands until the first call."""
    global _take
    _take = _load_tensors().take
    return _take(*args)


def _stream_on(stream, d):
    if stream is None and _raw_stream is not None:
        return _raw_stream(d)
    return _stream(stream)


def q8_cache(pages, page, hk, dtype=_torch.float8_e4m3fn, device="cuda"):
    """A zeroed 8-bit cache of `pages` pages: (kv [blocks][2 hk][2048], kv_scale [blocks][2 hk] exponents)."""
    if page <= 0 or page % 16 or dtype not in _Q8_DTYPES or pages < 0 or hk <= 0:
        raise OmniAttnError(EINVAL, f"q8_cache: pages={pages} page={page} hk={hk} dtype={dtype}")
    blocks = pages * (page // 16)
    kv = _torch.zeros(blocks, 2 * hk, 16 * HEAD_DIM, dtype=_torch.uint8, device=device).view(dtype)
    return kv, _torch.full((blocks, 2 * hk), 1, dtype=_torch.uint8, device=device).view(_torch.float8_e8m0fnu)


def step_tables(first, count, lines, table, free_pages, free_state, pos, slots, seq, row_indptr, indptr, pages, status,
                page=16, ring=0, stream=None):
    """The step's row tables on the GPU from the request lengths: ``pos``,
    ``slots``, ``seq``, ``row_indptr``, ``indptr`` and ``pages`` of every new row
    and sequence, pages taken from the free queue (free_pages, free_state =
    [head, free entries]) into ``table`` [lines][pages per line], pages of done
    requests (count < 0) given back. lines None: line s; free_pages None: the
    table holds every page. ``status`` = [code, rows, pages, head, free entries];
    ``status[3:5]`` is the next call's free_state, with another status. ring > 0:
    tables for the calls with a context cap (``lm_attend`` with context = ring),
    not for the 8-bit cache's."""
    d = _current_device() if first.is_cuda else -1
    n, rows = first.numel(), pos.numel()
    shape = table.shape
    if len(shape) != 2:
        raise OmniAttnError(EINVAL, "table must be an int32 tensor [lines][pages]")
    num_pages = 0 if free_pages is None else free_pages.numel()
    (p_first, p_count, p_lines, p_table, p_free, p_state, p_pos, p_slots, p_seq, p_rows, p_indptr, p_pages, p_status) = _take(
        "iiIiIIiiiiiii", "first count lines table free_pages free_state pos slots seq row_indptr indptr pages status", d,
        first, 0, count, n, lines, n, table, 0, free_pages, 1, None if free_pages is None else free_state, 2, pos, 0,
        slots, rows, seq, rows, row_indptr, n + 1, indptr, n + 1, pages, 0, status, 5)
    _check(load().omni_attn_step_tables(p_first, p_count, p_lines, n, page, ring, p_table, shape[1], shape[0], p_free,
                                        num_pages, p_state, rows, pages.numel(), p_pos, p_slots, p_seq, p_rows, p_indptr,
                                        p_pages, p_status, _stream_on(stream, d)))
    return status


def qwen3_rope_q8(qkv, q_norm, k_norm, pos, slots, q_out, k_out, kv, kv_scale, hq, hk, eps, theta, stream=None):
    """``qwen3_rope`` with the quantized cache write: q to ``q_out`` rows, the
    turned k to ``k_out`` rows (None: not written), K and V to slot ``slots[n]``
    of the 8-bit cache. Rows may be strided; rows with a negative slot are
    skipped."""
    rows = pos.numel()
    d = _current_device() if qkv.is_cuda else -1
    src, ld, p_qn, p_kn, p_pos, p_slots, q, q_ld, k, k_ld, cache, scales, fmt = _take(
        "rbbiirRc", "qkv q_norm k_norm pos slots q_out k_out kv", d, qkv, rows, (hq + 2 * hk) * HEAD_DIM, q_norm, HEAD_DIM,
        k_norm, HEAD_DIM, pos, 0, slots, rows, q_out, rows, hq * HEAD_DIM, k_out, rows, hk * HEAD_DIM, kv, kv_scale, 2 * hk)
    _check(load().omni_qwen3_rope_q8(src, ld, p_qn, p_kn, p_pos, p_slots, q, q_ld, k, k_ld, cache, scales, fmt, rows, hq,
                                     hk, eps, theta, _stream_on(stream, d)))


def decode_plan_q8(rows: int, hq: int, hk: int, page: int, max_len: int, chunk: int = 0) -> DecodePlan:
    """The plan for qwen3_attend_q8."""
    plan = DecodePlan()
    _check(load().omni_attn_decode_plan_init_q8(rows, hq, hk, page, max_len, chunk, ctypes.byref(plan)))
    return plan


def qwen3_attend_q8(q, kv, kv_scale, pos, seq, ragged, indptr, pages, page, out, hq, hk, scale, plan, workspace=None,
                    stream=None):
    """``qwen3_attend`` over the 8-bit cache: q rows [hq * 128], possibly strided;
    rows with a negative position store zeros."""
    rows = plan.rows
    d = _current_device() if q.is_cuda else -1
    src, stride, cache, scales, fmt, p_pos, p_seq, p_indptr, p_pages, p_out = _take(
        "rciIiib", "q kv pos seq indptr pages out", d, q, rows, hq * HEAD_DIM, kv, kv_scale, 2 * hk, pos, rows, seq, rows,
        indptr, 1 if ragged else rows + 1, pages, 0, out, rows * hq * HEAD_DIM)
    if workspace is not None and workspace.get_device() != d:
        raise OmniAttnError(EINVAL, "workspace must lie on the current device, with the other tensors")
    _check(load().omni_qwen3_attend_q8(src, stride, cache, scales, fmt, p_pos, p_seq, 1 if ragged else 0, p_indptr, p_pages,
                                       page, p_out, hq, hk, scale, ctypes.byref(plan), _ws(plan, workspace),
                                       _stream_on(stream, d)))
    return out


@dataclass
class Prompt:
    plan: PromptPlan
    work: object  # device int32 tensor


def prompt_plan(lens, hq, hk, device="cuda", exact_p=False) -> Prompt:
    """Host plan of causal attention over packed prompts of these lengths;
    uploads the work list. exact_p: as in prefill_plan."""
    import numpy as np

    lens_a = np.ascontiguousarray(lens, dtype=np.int32)
    plan = PromptPlan()
    L = load()
    ptr = lens_a.ctypes.data_as(ctypes.c_void_p)
    rc = L.omni_attn_prompt_plan_init(len(lens_a), ptr, hq, hk, None, 0, ctypes.byref(plan))
    if rc not in (OK, EWORKSPACE):
        _check(rc)
    work_h = np.zeros(max(1, int(plan.work_bytes) // 4), dtype=np.int32)
    _check(L.omni_attn_prompt_plan_init(len(lens_a), ptr, hq, hk, work_h.ctypes.data_as(ctypes.c_void_p), len(work_h),
                                        ctypes.byref(plan)))
    plan.exact_p = 1 if exact_p else 0
    return Prompt(plan, _torch.from_numpy(work_h).to(device))


def prompt_run(pp: Prompt, q, k, v, out, scale, stream=None):
    """Causal attention of packed prompts: q rows [hq * 128], k and v rows
    [hk * 128], possibly strided (parts of one qkv row); out contiguous rows."""
    plan = pp.plan
    rows, hq, hk = plan.rows, plan.hq, plan.hk
    d = _current_device() if q.is_cuda else -1
    p_q, q_ld, p_k, k_ld, p_v, v_ld, p_out, p_work = _take(
        "rrrbi", "q k v out work", d, q, rows, hq * HEAD_DIM, k, rows, hk * HEAD_DIM, v, rows, hk * HEAD_DIM, out,
        rows * hq * HEAD_DIM, pp.work, plan.work_bytes >> 2)
    _check(load().omni_attn_prompt_run(ctypes.byref(plan), p_q, q_ld, p_k, k_ld, p_v, v_ld, p_out, scale, p_work,
                                       _stream_on(stream, d)))
    return out


# ------------------------------------- several rows per sequence, encoder states
@dataclass
class Multi:
    plan: MultiPlan
    work: object  # device int32 tensor


def _multi_plan(init, counts, keys, hq, hk, max_len, chunk, device, exact_p) -> Multi:
    import numpy as np

    counts_a = np.ascontiguousarray(counts, dtype=np.int32)
    keys_a = None if keys is None else np.ascontiguousarray(keys, dtype=np.int32)
    if keys_a is not None and len(keys_a) != len(counts_a):
        raise OmniAttnError(EINVAL, f"{len(keys_a)} lengths for {len(counts_a)} sequences")
    ptr = lambda a: None if a is None else a.ctypes.data_as(ctypes.c_void_p)
    plan = MultiPlan()
    rc = init(len(counts_a), ptr(counts_a), ptr(keys_a), hq, hk, max_len, chunk, None, 0, ctypes.byref(plan))
    if rc not in (OK, EWORKSPACE):
        _check(rc)
    work_h = np.zeros(max(4, int(plan.work_bytes) // 4), dtype=np.int32)
    _check(init(len(counts_a), ptr(counts_a), ptr(keys_a), hq, hk, max_len, chunk, ptr(work_h), len(work_h), ctypes.byref(plan)))
    plan.exact_p = 1 if exact_p else 0
    return Multi(plan, _torch.from_numpy(work_h).to(device))


def extend_plan(counts, hq, hk, max_len, keys=None, chunk=0, device="cuda", exact_p=False) -> Multi:
    """Host plan of qwen3_extend_q8 for ``counts[s]`` rows of each sequence;
    uploads the work list. ``keys``: how many keys each sequence's last row sees
    now, if known (for the choice of kernels, the order and the split sizes alone);
    exact_p: P in 16 bits in every row (else rounded to bf16 in rows that run in
    tiles); the workspace is ``workspace_for(plan.plan)``."""
    return _multi_plan(load().omni_attn_extend_plan_init, counts, keys, hq, hk, max_len, chunk, device, exact_p)


def cross_plan(counts, hq, hk, max_len, keys=None, chunk=0, device="cuda", exact_p=False) -> Multi:
    """Host plan of cross_run for ``counts[s]`` rows over each source, as extend_plan."""
    return _multi_plan(load().omni_attn_cross_plan_init, counts, keys, hq, hk, max_len, chunk, device, exact_p)


def _multi_ws(plan, workspace, d):
    if workspace is not None and workspace.get_device() != d:
        raise OmniAttnError(EINVAL, "workspace must lie on the current device, with the other tensors")
    return _ws(plan, workspace)


def qwen3_extend_q8(mp: Multi, q, kv, kv_scale, pos, indptr, pages, page, out, scale, workspace=None, stream=None):
    """Attention of several new rows per sequence over the 8-bit cache: row n of
    the plan's sequence s sees keys 0..pos[n] (the call's rows among them); rows
    with a negative position store zeros. q rows [hq * 128], possibly strided."""
    plan = mp.plan
    rows, hq = plan.rows, plan.hq
    d = _current_device() if q.is_cuda else -1
    src, stride, cache, scales, fmt, p_pos, p_indptr, p_pages, p_out, p_work = _take(
        "rciiibi", "q kv pos indptr pages out work", d, q, rows, hq * HEAD_DIM, kv, kv_scale, 2 * plan.hk, pos, rows, indptr,
        plan.nseq + 1, pages, 0, out, rows * hq * HEAD_DIM, mp.work, plan.work_bytes >> 2)
    _check(load().omni_qwen3_extend_q8(ctypes.byref(plan), src, stride, cache, scales, fmt, p_pos, p_indptr, p_pages, page, p_out,
                                       scale, p_work, _multi_ws(plan, workspace, d), _stream_on(stream, d)))
    return out


def cross_run(mp: Multi, q, k, v, of, first, length, out, scale, workspace=None, stream=None):
    """Cross attention: the plan's rows of sequence s see rows first[e] ..
    first[e] + length[e] - 1 of k and v, e = of[s] (of None: s); zeros where there
    are none. q rows [hq * 128], k and v rows [hk * 128], possibly strided (k and v
    parts of one row)."""
    plan = mp.plan
    rows, hq, hk = plan.rows, plan.hq, plan.hk
    d = _current_device() if q.is_cuda else -1
    p_q, q_ld, p_k, k_ld, p_v, v_ld, p_of, p_first, p_len, p_out, p_work = _take(
        "rrrIiibi", "q k v of first length out work", d, q, rows, hq * HEAD_DIM, k, 0, hk * HEAD_DIM, v, 0, hk * HEAD_DIM, of,
        plan.nseq, first, 0 if of is not None else plan.nseq, length, first.numel(), out, rows * hq * HEAD_DIM, mp.work,
        plan.work_bytes >> 2)
    _check(load().omni_attn_cross_run(ctypes.byref(plan), p_q, q_ld, p_k, k_ld, p_v, v_ld, p_of, p_first, p_len, p_out, scale, p_work,
                                      _multi_ws(plan, workspace, d), _stream_on(stream, d)))
    return out


# ------------------------------------------------- pages that requests share
PAGES_UNHELD = 6


def _table_shape(table):
    shape = table.shape
    if len(shape) != 2:
        raise OmniAttnError(EINVAL, "table must be an int32 tensor [lines][pages]")
    return shape


def pages_fork(parents, children, tokens, table, free_pages, free_state, shares, src, dst, status, page=16, stream=None):
    """Line ``children[i]`` of ``table`` begins with the first ``tokens[i]`` tokens
    of line ``parents[i]``: whole pages shared (``shares`` counts a page's holders
    beside the first), the part-filled one a page of its own from the free queue,
    to be copied by ``pages_copy(.., src, dst)``. ``status`` = [code, pages taken,
    pages shared, head, free entries]; ``status[3:5]`` is the next call's free_state.
    tokens < 0: no fork. Lines that share pages take tables without a ring, whose
    rows would come round to the shared pages."""
    d = _current_device() if parents.is_cuda else -1
    n, (lines, ld), pool = parents.numel(), _table_shape(table), free_pages.numel()
    (p_par, p_chi, p_tok, p_table, p_free, p_state, p_shares, p_src, p_dst, p_status) = _take(
        "iiiiiiiiii", "parents children tokens table free_pages free_state shares src dst status", d, parents, 0, children, n,
        tokens, n, table, 0, free_pages, 1, free_state, 2, shares, pool, src, n, dst, n, status, 5)
    _check(load().omni_attn_pages_fork(p_par, p_chi, p_tok, n, page, p_table, ld, lines, p_free, pool, p_state, p_shares, p_src,
                                       p_dst, p_status, _stream_on(stream, d)))
    return status


def pages_free(lines, tokens, table, free_pages, free_state, shares, status, page=16, stream=None):
    """Lines ``lines[i]`` of ``tokens[i]`` tokens end: pages that nobody else holds
    go to the free queue's end, in ascending order. ``status`` = [code, pages that
    came free, pages that the lines held, head, free entries]."""
    d = _current_device() if lines.is_cuda else -1
    n, (num_lines, ld), pool = lines.numel(), _table_shape(table), free_pages.numel()
    p_lines, p_tok, p_table, p_free, p_state, p_shares, p_status = _take(
        "iiiiiii", "lines tokens table free_pages free_state shares status", d, lines, 0, tokens, n, table, 0, free_pages, 1,
        free_state, 2, shares, pool, status, 5)
    _check(load().omni_attn_pages_free(p_lines, p_tok, n, page, p_table, ld, num_lines, p_free, pool, p_state, p_shares, p_status,
                                       _stream_on(stream, d)))
    return status


def pages_compact(table, free_pages, free_state, shares, limit, table_out, free_out, shares_out, new_ids, src, dst, status,
                  stream=None):
    """Pages in use from id ``limit`` on move to free ones below it: ``src`` and
    ``dst`` (-1 past the last) for ``pages_copy(.., count=status[1:2])``, the table
    (in place if table_out is it), the free queue in ascending order, the holders
    and every page's new id. ``status`` = [code, moves, free pages below the limit,
    0, free pages]."""
    d = _current_device() if table.is_cuda else -1
    (lines, ld), pool, cap = _table_shape(table), free_pages.numel(), src.numel()
    (p_table, p_free, p_state, p_shares, p_tout, p_fout, p_sout, p_ids, p_src, p_dst, p_status) = _take(
        "iiiiiiiiiii", "table free_pages free_state shares table_out free_out shares_out new_ids src dst status", d, table, 0,
        free_pages, 1, free_state, 2, shares, pool, table_out, lines * ld, free_out, pool, shares_out, pool, new_ids, pool, src, 0,
        dst, cap, status, 5)
    _check(load().omni_attn_pages_compact(p_table, ld, lines, p_free, pool, p_state, p_shares, limit, p_tout, p_fout, p_sout, p_ids,
                                          p_src, p_dst, cap, p_status, _stream_on(stream, d)))
    return status


def pages_copy(kv, kv_scale, src, dst, page=16, count=None, stream=None):
    """Page ``dst[k]`` takes the bytes of page ``src[k]`` in every layer (ids outside
    the pool: no copy; ``count``: a device int32, how many pairs count). kv and
    kv_scale: the 8-bit cache, [blocks][2 hk][2048] and [blocks][2 hk]; kv_scale None:
    bf16 slots [slots][2 hk][128], or uint8 slots [slots][bytes] (FP8 slots, of a
    multiple of 16 bytes a page); each may have a dimension of layers before."""
    d = _current_device() if kv.is_cuda else -1
    n = src.numel()
    p_kv, p_scale, layers, units, width, scales, per, p_src, p_dst, p_count = _take(
        "piiI", "kv src dst count", d, kv, kv_scale, page, src, 0, dst, n, count, 1)
    _check(load().omni_attn_pages_copy(p_kv, width * per, width * units, p_scale, scales * per, scales * units, layers, units // per,
                                       p_src, p_dst, n, p_count, _stream_on(stream, d)))
    return kv


# ------------------------------------------------------------ host row builder
class Rows:
    """The engines' ``Rows`` (crates/omni-qwen3-tts/src/model.rs:266-303,
    crates/omni-personaplex/src/model.rs:472-499) on the native builder:
    ``push(page_ids, first, count, seq)`` per sequence, then the int32 arrays
    ``pos``, ``slot``, ``seq``, ``indptr``, ``pages`` (numpy copies)."""

    _WHICH = {"pos": 0, "slot": 1, "seq": 2, "indptr": 3, "pages": 4}

    def __init__(self, page: int = 16, ring: int = 0):
        h = load().omni_attn_rows_new(page, ring)
        if not h:
            raise OmniAttnError(EINVAL, load().omni_attn_last_error().decode())
        self._h = ctypes.c_void_p(h)

    def __del__(self):
        if getattr(self, "_h", None) and _lib is not None:
            _lib.omni_attn_rows_free(self._h)
            self._h = None

    def push(self, page_ids, first: int, count: int, seq: int):
        import numpy as np

        ids = np.ascontiguousarray(page_ids, dtype=np.int32)
        _check(load().omni_attn_rows_push(self._h, ids.ctypes.data_as(ctypes.c_void_p), len(ids), first, count, seq))

    def clear(self):
        load().omni_attn_rows_clear(self._h)

    def counts(self):
        r, s, p = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        _check(load().omni_attn_rows_count(self._h, ctypes.byref(r), ctypes.byref(s), ctypes.byref(p)))
        return r.value, s.value, p.value

    def __getattr__(self, name):
        if name not in Rows._WHICH:
            raise AttributeError(name)
        import numpy as np

        rows, seqs, pages = self.counts()
        n = {"pos": rows, "slot": rows, "seq": rows, "indptr": seqs + 1 if seqs else 0, "pages": pages}[name]
        if n == 0:
            return np.zeros(0, np.int32)
        ptr = load().omni_attn_rows_get(self._h, Rows._WHICH[name])
        return np.ctypeslib.as_array(ptr, shape=(n,)).copy()


def hidream_rows(causal, grid, image_position=4096):
    """HiDream-O1's host row arrays (``model.rs:123-160``): (text_pos [causal][3],
    text_slots, gen_pos [rows][3], gen_slots, step_kv) as numpy int32."""
    import numpy as np

    rows = 1 + grid[0] * grid[1]
    tp = np.zeros((causal, 3), np.int32)
    ts = np.zeros(causal, np.int32)
    gp = np.zeros((rows, 3), np.int32)
    gs = np.zeros(rows, np.int32)
    kv = np.zeros(1, np.int32)
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)
    _check(load().omni_hidream_rows(causal, grid[0], grid[1], image_position, ptr(tp), ptr(ts), ptr(gp), ptr(gs),
                                    ptr(kv)))
    return tp, ts, gp, gs, int(kv[0])
