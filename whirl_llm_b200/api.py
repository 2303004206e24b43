"""ctypes bindings of libwhirl_b200.so over torch tensors (device memory and streams only; all arithmetic is in the
library).  Function names and argument meaning follow include/whirl_b200.h, which follows the reference's kernel and
ServerModel interfaces."""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass, field
from typing import Optional

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("WHIRL_B200_LIB") or os.path.join(_HERE, "libwhirl_b200.so")

F32, BF16 = 0, 1
ROW_DONE, ROW_ESCALATE, ROW_OPEN_TAIL = 0, 1, 2
CNT_ESCALATED, CNT_OPEN_TAIL, CNT_UNRESOLVED, CNT_TIMEOUT, CNT_REDO, CNT_NAN_ROWS, CNT_WORDS = 0, 1, 2, 3, 4, 5, 8
ERR_TIMEOUT = 5
MAX_K, STREAM_MAX_K, MAX_HIST, Q_WORDS, Q_MAX, CTL_WORDS = 16384, 1024, 4096, 72, 32, 64
STATIC_MAX_ROWS = 256


class WhirlError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"whirl_b200 status {status}: {msg}")
        self.status = status


class SampleParams(C.Structure):
    _fields_ = [("inv_t", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p), ("min_p", C.c_void_p),
                ("greedy", C.c_void_p), ("u", C.c_void_p), ("race_key", C.c_void_p), ("hist", C.c_void_p),
                ("hist_len", C.c_void_p), ("hist_stride", C.c_int64), ("rep", C.c_void_p), ("pres", C.c_void_p),
                ("freq", C.c_void_p)]


class DSampArgs(C.Structure):
    _fields_ = [("on", C.c_void_p), ("top_k", C.c_void_p), ("qoff", C.c_void_p), ("inv_t", C.c_void_p), ("top_p", C.c_void_p),
                ("min_p", C.c_void_p), ("key_lo", C.c_void_p), ("key_hi", C.c_void_p)]


class RelaxParams(C.Structure):
    _fields_ = [("k", C.c_uint32), ("alpha", C.c_float), ("eps", C.c_float), ("delta", C.c_float)]


class AcceptIn(C.Structure):
    _fields_ = [("tokens", C.c_void_p), ("drafts", C.c_void_p), ("draft_stride", C.c_int64), ("nd", C.c_void_p), ("row0", C.c_void_p),
                ("greedy", C.c_void_p), ("relax_on", C.c_void_p), ("next", C.c_void_p), ("hist", C.c_void_p),
                ("hist_stride", C.c_int64), ("hist_len", C.c_void_p), ("rk_ids", C.c_void_p), ("rk_vals", C.c_void_p),
                ("rk_stats", C.c_void_p), ("rk", C.c_int32), ("kept_cap", C.c_int32), ("kept_ids", C.c_void_p),
                ("kept_p", C.c_void_p), ("n_kept", C.c_void_p), ("closed", C.c_void_p), ("stats", C.c_void_p), ("x", C.c_void_p),
                ("dtype", C.c_int32), ("n", C.c_int32), ("inv_t", C.c_void_p)]


class SampleOut(C.Structure):
    _fields_ = [("token", C.c_void_p), ("status", C.c_void_p), ("n_kept", C.c_void_p), ("closed", C.c_void_p),
                ("stats", C.c_void_p), ("kept_ids", C.c_void_p), ("kept_p", C.c_void_p), ("kept_cap", C.c_int32),
                ("counters", C.c_void_p)]


class PolicyParams(C.Structure):
    _fields_ = [("token", C.c_void_p), ("adv", C.c_void_p), ("old_logp", C.c_void_p), ("ref_logp", C.c_void_p), ("weight", C.c_void_p),
                ("seq_start", C.c_void_p), ("seqs", C.c_int32), ("mean", C.c_int32), ("inv_t_rows", C.c_void_p), ("inv_t", C.c_float),
                ("clip_low", C.c_float), ("clip_high", C.c_float), ("dual_clip", C.c_float), ("kl_coef", C.c_float),
                ("ent_coef", C.c_float)]


class PolicyOut(C.Structure):
    _fields_ = [("loss", C.c_void_p), ("logp", C.c_void_p), ("stats", C.c_void_p), ("entropy", C.c_void_p), ("kl", C.c_void_p),
                ("row_loss", C.c_void_p), ("g_logp", C.c_void_p), ("row_scale", C.c_void_p), ("dx", C.c_void_p), ("ld_dx", C.c_int64)]


class PreferenceParams(C.Structure):
    _fields_ = [("token", C.c_void_p), ("seq_start", C.c_void_p), ("ref_logp", C.c_void_p), ("weight", C.c_void_p),
                ("inv_t_rows", C.c_void_p), ("pairs", C.c_int32), ("kind", C.c_int32), ("average", C.c_int32), ("inv_t", C.c_float),
                ("beta", C.c_float), ("smoothing", C.c_float), ("margin", C.c_float)]


class PreferenceOut(C.Structure):
    _fields_ = [("loss", C.c_void_p), ("pair_loss", C.c_void_p), ("reward", C.c_void_p), ("logp", C.c_void_p), ("stats", C.c_void_p),
                ("g_logp", C.c_void_p), ("dx", C.c_void_p), ("ld_dx", C.c_int64)]


class BlockTables(C.Structure):
    _fields_ = [("table", C.c_void_p), ("owned", C.c_void_p), ("free_ids", C.c_void_p), ("free_count", C.c_void_p), ("seqs", C.c_int32),
                ("max_blocks", C.c_int32), ("num_blocks", C.c_int32), ("block_size", C.c_int32)]


class StepRowsOut(C.Structure):
    _fields_ = [("slot", C.c_void_p), ("position", C.c_void_p), ("seq", C.c_void_p), ("row0", C.c_void_p), ("status", C.c_void_p),
                ("max_rows", C.c_int32)]


def _load() -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python -m whirl_llm_b200.build` "
                          "(there is no fallback implementation)")
    lib = C.CDLL(LIB_PATH)
    vp, i, f, sz, i64 = C.c_void_p, C.c_int, C.c_float, C.c_size_t, C.c_int64
    sigs = {
        "whirl_status_string": (C.c_char_p, [i]),
        "whirl_last_error": (C.c_char_p, []),
        "whirl_version": (i, []),
        "whirl_workspace_bytes": (sz, [i, i]),
        "whirl_argmax": (i, [vp, i, i, vp, vp, vp, i, vp, sz, vp]),
        "whirl_argmax_rows": (i, [vp, i, i, i, vp, vp, sz, vp]),
        "whirl_argmax_rows_to": (i, [vp, i, i, i, vp, vp, vp, sz, vp]),
        "whirl_argmax_rows_static": (i, [vp, i, i, i, vp, vp]),
        "whirl_argmax_prob": (i, [vp, i, i, i, vp, vp, vp, sz, vp]),
        "whirl_draft_pick": (i, [vp, i, i, vp, vp, vp, i, i, f, vp, vp, sz, vp]),
        "whirl_draft_pick_rows": (i, [vp, i, i, i, vp, vp, i, i, f, vp, vp, sz, vp]),
        "whirl_topk_rows": (i, [vp, i, i, i, i, f, vp, vp, vp, vp, vp, sz, vp]),
        "whirl_draft_sample_rows": (i, [vp, i, i, i, vp, vp, i, vp, C.POINTER(DSampArgs), vp, vp]),
        "whirl_accept_tokens": (i, [vp, vp, i, vp, vp, i, vp, vp, vp]),
        "whirl_spec_workspace_bytes": (sz, [i, i]),
        "whirl_spec_accept_residual": (i, [vp, vp, i, i, i, i, vp, vp, vp, vp, vp, vp, vp, sz, vp]),
        "whirl_topk_rows_shard": (i, [vp, i, i, i, i, i, f, vp, vp, vp, vp, vp, sz, vp]),
        "whirl_merge_sample_rows": (i, [vp, vp, vp, i, i, i, i, C.POINTER(SampleParams), C.POINTER(SampleOut), vp]),
        "whirl_sample_rows": (i, [vp, i, i, i, C.POINTER(SampleParams), C.POINTER(SampleOut), vp, sz, vp]),
        "whirl_sample_rows_host": (i, [vp, i, i, i, C.POINTER(SampleParams), C.POINTER(SampleOut), i]),
        "whirl_host_release": (None, []),
        "whirl_host_last_error": (C.c_char_p, []),
        "whirl_launch_counts": (None, [vp, i]),
        "whirl_check": (i, [vp, sz, i, vp, vp]),
        "whirl_shard_block_words": (sz, [i, i]),
        "whirl_merge_sample_rows_packed": (i, [vp, i, i, i, i, C.POINTER(SampleParams), C.POINTER(SampleOut), vp]),
        "whirl_accept_rows": (i, [C.POINTER(AcceptIn), C.POINTER(RelaxParams), i, vp, vp, vp, vp, vp, vp]),
        "whirl_uniform_splitmix": (C.c_double, [C.c_uint64, C.c_uint64, C.c_uint32]),
        "whirl_race_base": (C.c_uint64, [C.c_uint64, C.c_uint64]),
        "whirl_philox4x32_10": (None, [C.POINTER(C.c_uint32), C.POINTER(C.c_uint32), C.POINTER(C.c_uint32)]),
        "whirl_uniform_philox4x32": (C.c_double, [C.c_uint64, C.c_uint64, C.c_uint32, C.c_uint32]),
        "whirl_fill_draws": (i, [vp, vp, i, i, C.c_uint32, vp, vp, vp]),
        "whirl_test_waits": (None, [C.c_uint32, i]),
        "whirl_token_logprobs": (i, [vp, i, i, i, i64, vp, f, vp, vp, vp, vp, vp]),
        "whirl_token_logprobs_grad": (i, [vp, i, i, i, i64, vp, f, vp, vp, vp, vp, vp, vp, i64, vp]),
        "whirl_loss_workspace_bytes": (sz, [i, i]),
        "whirl_policy_loss": (i, [vp, i, i, i, i64, C.POINTER(PolicyParams), C.POINTER(PolicyOut), vp, sz, vp]),
        "whirl_loss_check": (i, [vp, sz, vp, C.POINTER(C.c_uint32)]),
        "whirl_preference_loss": (i, [vp, i, i, i, i64, C.POINTER(PreferenceParams), C.POINTER(PreferenceOut), vp, sz, vp]),
        "whirl_block_workspace_bytes": (sz, [i]),
        "whirl_block_tables_step": (i, [vp, vp, C.POINTER(BlockTables), C.POINTER(StepRowsOut), vp, sz, vp]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


lib = _load()
DECLARED = ["whirl_status_string", "whirl_last_error", "whirl_version", "whirl_workspace_bytes", "whirl_argmax",
            "whirl_argmax_rows", "whirl_argmax_rows_static", "whirl_argmax_rows_to", "whirl_argmax_prob", "whirl_draft_pick", "whirl_draft_pick_rows", "whirl_draft_sample_rows", "whirl_accept_tokens", "whirl_spec_workspace_bytes",
            "whirl_spec_accept_residual",
            "whirl_topk_rows", "whirl_topk_rows_shard", "whirl_merge_sample_rows", "whirl_sample_rows", "whirl_sample_rows_host", "whirl_host_release", "whirl_host_last_error",
            "whirl_launch_counts", "whirl_check", "whirl_shard_block_words", "whirl_merge_sample_rows_packed", "whirl_test_waits", "whirl_accept_rows",
            "whirl_uniform_splitmix", "whirl_race_base", "whirl_philox4x32_10", "whirl_uniform_philox4x32", "whirl_fill_draws",
            "whirl_token_logprobs", "whirl_token_logprobs_grad", "whirl_loss_workspace_bytes", "whirl_policy_loss", "whirl_loss_check", "whirl_preference_loss",
            "whirl_block_workspace_bytes", "whirl_block_tables_step"]


def _check(status: int):
    if status != 0:
        raise WhirlError(status, (lib.whirl_last_error() or b"").decode())


def _dtype(x: torch.Tensor) -> int:
    if x.dtype == torch.float32:
        return F32
    if x.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"logits must be float32 or bfloat16, got {x.dtype}")


def _rows(x: torch.Tensor):
    if not x.is_cuda:
        raise ValueError("logits must be on a CUDA device (this library has no CPU path)")
    if x.dim() == 1:
        x = x.unsqueeze(0)
    if x.dim() != 2 or x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) != x.shape[1]):
        raise ValueError("logits must be dense rows [rows, n]")
    return x, x.shape[0], x.shape[1]


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(x: torch.Tensor):
    return torch.cuda.current_stream(x.device).cuda_stream


def workspace_bytes(rows: int, n: int) -> int:
    return lib.whirl_workspace_bytes(rows, n)


_ws_cache: dict = {}


def workspace(rows: int, n: int, device) -> torch.Tensor:
    """A cached workspace tensor for (rows, n) on `device` (callers that manage memory pass their own)."""
    device = torch.device(device)
    need = workspace_bytes(rows, n)
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    ws = _ws_cache.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(need, dtype=torch.uint8, device=device)
        _ws_cache[key] = ws
    return ws


def argmax(x, out=None, ids=None, pos=None, advance=0, ws=None):
    x, rows, n = _rows(x)
    assert rows == 1
    out = torch.empty(1, dtype=torch.int32, device=x.device) if out is None else out
    ws = workspace(1, n, x.device) if ws is None else ws
    _check(lib.whirl_argmax(x.data_ptr(), _dtype(x), n, out.data_ptr(), _p(ids), _p(pos), advance, ws.data_ptr(), ws.numel(),
                            _stream(x)))
    return out


def argmax_rows(x, out=None, ws=None):
    x, rows, n = _rows(x)
    out = torch.empty(rows, dtype=torch.int32, device=x.device) if out is None else out
    ws = workspace(rows, n, x.device) if ws is None else ws
    _check(lib.whirl_argmax_rows(x.data_ptr(), _dtype(x), rows, n, out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(x)))
    return out


def argmax_rows_static(x, out=None):
    """The greedy pick with the library's own fixed scratch: no workspace, no allocation by the library (at most
    WHIRL_STATIC_MAX_ROWS rows).  `out` is the caller's."""
    x, rows, n = _rows(x)
    out = torch.empty(rows, dtype=torch.int32, device=x.device) if out is None else out
    _check(lib.whirl_argmax_rows_static(x.data_ptr(), _dtype(x), rows, n, out.data_ptr(), _stream(x)))
    return out


def argmax_rows_to(x, out, dst, ws=None):
    x, rows, n = _rows(x)
    ws = workspace(rows, n, x.device) if ws is None else ws
    _check(lib.whirl_argmax_rows_to(x.data_ptr(), _dtype(x), rows, n, out.data_ptr(), dst.data_ptr(), ws.data_ptr(), ws.numel(),
                                    _stream(x)))
    return out


def argmax_prob(x, ws=None):
    x, rows, n = _rows(x)
    tok = torch.empty(rows, dtype=torch.int32, device=x.device)
    prob = torch.empty(rows, dtype=torch.float32, device=x.device)
    ws = workspace(rows, n, x.device) if ws is None else ws
    _check(lib.whirl_argmax_prob(x.data_ptr(), _dtype(x), rows, n, tok.data_ptr(), prob.data_ptr(), ws.data_ptr(), ws.numel(),
                                 _stream(x)))
    return tok, prob


def draft_pick(x, tok, prob, ctl, r, n_min, p_min, vmap=None, ws=None):
    x, rows, n = _rows(x)
    assert rows == 1
    ws = workspace(1, n, x.device) if ws is None else ws
    _check(lib.whirl_draft_pick(x.data_ptr(), _dtype(x), n, tok.data_ptr(), prob.data_ptr(), ctl.data_ptr(), r, n_min, p_min,
                                _p(vmap), ws.data_ptr(), ws.numel(), _stream(x)))


def draft_pick_rows(x, ctl_all, area, r, n_min, p_min, vmap=None, ws=None):
    x, rows, n = _rows(x)
    ws = workspace(rows, n, x.device) if ws is None else ws
    _check(lib.whirl_draft_pick_rows(x.data_ptr(), _dtype(x), rows, n, ctl_all.data_ptr(), area.data_ptr(), r, n_min, p_min,
                                     _p(vmap), ws.data_ptr(), ws.numel(), _stream(x)))


def draft_sample_rows(x, ctl_all, area, r, on, top_k, qoff, inv_t, top_p, min_p, race_key, qbuf, vmap=None):
    """draft_sample_rows: per-row arrays are device tensors (int32 / float32); race_key int64 holding the uint64 keys."""
    x, rows, n = _rows(x)
    lo = (race_key & 0xFFFFFFFF).to(torch.int32).contiguous()
    hi = ((race_key >> 32) & 0xFFFFFFFF).to(torch.int32).contiguous()
    d = DSampArgs(on=_p(on), top_k=_p(top_k), qoff=_p(qoff), inv_t=_p(inv_t), top_p=_p(top_p), min_p=_p(min_p), key_lo=_p(lo),
                  key_hi=_p(hi))
    _check(lib.whirl_draft_sample_rows(x.data_ptr(), _dtype(x), rows, n, ctl_all.data_ptr(), area.data_ptr(), r, _p(vmap),
                                       C.byref(d), qbuf.data_ptr(), _stream(x)))


def topk_rows(x, K, inv_t=1.0, inv_t_rows=None, ws=None):
    """ids [rows, K] i32, vals [rows, K] f32, stats [rows, 2] f32 (ServerModel::topkRows)."""
    x, rows, n = _rows(x)
    ids = torch.full((rows, K), -1, dtype=torch.int32, device=x.device)
    vals = torch.zeros((rows, K), dtype=torch.float32, device=x.device)
    stats = torch.zeros((rows, 2), dtype=torch.float32, device=x.device)
    ws = workspace(rows, n, x.device) if ws is None else ws
    _check(lib.whirl_topk_rows(x.data_ptr(), _dtype(x), rows, n, K, float(inv_t), _p(inv_t_rows), ids.data_ptr(), vals.data_ptr(),
                               stats.data_ptr(), ws.data_ptr(), ws.numel(), _stream(x)))
    return ids, vals, stats


def shard_block_views(block: torch.Tensor, rows: int, K: int):
    """The ids / vals / stats views of one rank's packed block (int32 tensor of whirl_shard_block_words words)."""
    assert block.dtype == torch.int32 and block.is_contiguous() and block.numel() == lib.whirl_shard_block_words(rows, K)
    ids = block[: rows * K].view(rows, K)
    vals = block[rows * K: 2 * rows * K].view(torch.float32).view(rows, K)
    stats = block[2 * rows * K:].view(torch.float32).view(rows, 2)
    return ids, vals, stats


def topk_rows_shard(x, K, id_offset, inv_t=1.0, inv_t_rows=None, ws=None, out=None):
    """topk_rows of one vocabulary slice with global token ids (ids pre-filled with -1).  out: (ids, vals, stats) to
    write into, e.g. the views of a packed block."""
    x, rows, n = _rows(x)
    if out is None:
        ids = torch.full((rows, K), -1, dtype=torch.int32, device=x.device)
        vals = torch.zeros((rows, K), dtype=torch.float32, device=x.device)
        stats = torch.zeros((rows, 2), dtype=torch.float32, device=x.device)
    else:
        ids, vals, stats = out
        if K > n:
            ids.fill_(-1)
    ws = workspace(rows, n, x.device) if ws is None else ws
    _check(lib.whirl_topk_rows_shard(x.data_ptr(), _dtype(x), rows, n, K, int(id_offset), float(inv_t), _p(inv_t_rows),
                                     ids.data_ptr(), vals.data_ptr(), stats.data_ptr(), ws.data_ptr(), ws.numel(), _stream(x)))
    return ids, vals, stats


@dataclass
class RowParams:
    """Device tensors of per-row sampler settings (None = the library default)."""
    inv_t: Optional[torch.Tensor] = None      # float32
    top_k: Optional[torch.Tensor] = None      # int32
    top_p: Optional[torch.Tensor] = None      # float64
    min_p: Optional[torch.Tensor] = None      # float64
    greedy: Optional[torch.Tensor] = None     # uint8
    u: Optional[torch.Tensor] = None          # float64
    race_key: Optional[torch.Tensor] = None   # int64 holding the uint64 bit pattern
    hist: Optional[torch.Tensor] = None       # int32 [rows, H]
    hist_len: Optional[torch.Tensor] = None   # int32
    rep: Optional[torch.Tensor] = None        # float32
    pres: Optional[torch.Tensor] = None       # float32
    freq: Optional[torch.Tensor] = None       # float32

    _DT = dict(inv_t=torch.float32, top_k=torch.int32, top_p=torch.float64, min_p=torch.float64, greedy=torch.uint8,
               u=torch.float64, race_key=torch.int64, hist=torch.int32, hist_len=torch.int32, rep=torch.float32,
               pres=torch.float32, freq=torch.float32)

    def struct(self, rows: int) -> SampleParams:
        s = SampleParams()
        for k, dt in self._DT.items():
            t = getattr(self, k)
            if t is not None:
                if t.dtype != dt or not t.is_cuda or not t.is_contiguous():
                    raise TypeError(f"{k}: want a contiguous CUDA tensor of {dt}, got {t.dtype} on {t.device}")
                if k != "hist" and t.shape != (rows,):
                    raise ValueError(f"{k}: want shape ({rows},), got {tuple(t.shape)}")
                if k == "hist" and (t.dim() != 2 or t.shape[0] != rows):
                    raise ValueError(f"hist: want [rows, H], got {tuple(t.shape)}")
            setattr(s, k, _p(t))
        s.hist_stride = 0 if self.hist is None else self.hist.shape[1]
        return s


@dataclass
class SampleResult:
    token: torch.Tensor
    status: torch.Tensor
    n_kept: torch.Tensor
    closed: torch.Tensor
    stats: Optional[torch.Tensor]
    kept_ids: Optional[torch.Tensor]
    kept_p: Optional[torch.Tensor]
    counters: torch.Tensor


def sample_rows(x, params: RowParams, kept_cap: int = 0, ws=None, result: Optional[SampleResult] = None,
                want_stats: bool = True) -> SampleResult:
    """One token per row: penalties -> candidates -> top-k / top-p / min-p -> draw (whirl_sample_rows)."""
    x, rows, n = _rows(x)
    dev = x.device
    if result is None:
        result = SampleResult(
            token=torch.empty(rows, dtype=torch.int32, device=dev), status=torch.empty(rows, dtype=torch.int32, device=dev),
            n_kept=torch.empty(rows, dtype=torch.int32, device=dev), closed=torch.empty(rows, dtype=torch.int32, device=dev),
            stats=torch.empty((rows, 2), dtype=torch.float32, device=dev) if want_stats else None,
            kept_ids=torch.full((rows, kept_cap), -1, dtype=torch.int32, device=dev) if kept_cap else None,
            kept_p=torch.zeros((rows, kept_cap), dtype=torch.float64, device=dev) if kept_cap else None,
            counters=torch.zeros(CNT_WORDS, dtype=torch.int32, device=dev))
    o = SampleOut(token=_p(result.token), status=_p(result.status), n_kept=_p(result.n_kept), closed=_p(result.closed),
                  stats=_p(result.stats), kept_ids=_p(result.kept_ids), kept_p=_p(result.kept_p),
                  kept_cap=0 if result.kept_ids is None else result.kept_ids.shape[1], counters=_p(result.counters))
    ws = workspace(rows, n, dev) if ws is None else ws
    ps = params.struct(rows)
    _check(lib.whirl_sample_rows(x.data_ptr(), _dtype(x), rows, n, C.byref(ps), C.byref(o), ws.data_ptr(), ws.numel(), _stream(x)))
    return result


def check(ws: torch.Tensor, rows: int) -> int:
    """whirl_check: reads the device error word of the last sample_rows / topk_rows call on `ws` (synchronises the
    stream).  Returns the code of the wait that ran out (0: none)."""
    where = C.c_uint32(0)
    st = lib.whirl_check(ws.data_ptr(), ws.numel(), rows, torch.cuda.current_stream(ws.device).cuda_stream, C.byref(where))
    if st not in (0, ERR_TIMEOUT):
        _check(st)
    return int(where.value)


def test_waits(wait_us: int = 0, lose_copy: bool = False) -> None:
    """whirl_test_waits: a testing aid; see include/whirl_b200.h."""
    lib.whirl_test_waits(wait_us, int(lose_copy))


GEN_SPLITMIX, GEN_PHILOX = 0, 1


def uniform_splitmix(seed: int, pos_idx: int, stream_id: int = 0) -> float:
    """Sampler::uniform / spec::uniform of the reference, on the host."""
    return lib.whirl_uniform_splitmix(seed, pos_idx, stream_id)


def race_base(seed: int, pos_idx: int) -> int:
    return lib.whirl_race_base(seed, pos_idx)


def philox4x32_10(ctr, key):
    c, k, o = (C.c_uint32 * 4)(*ctr), (C.c_uint32 * 2)(*key), (C.c_uint32 * 4)()
    lib.whirl_philox4x32_10(c, k, o)
    return list(o)


def uniform_philox4x32(seed: int, pos_idx: int, row: int, stream_id: int = 0) -> float:
    return lib.whirl_uniform_philox4x32(seed, pos_idx, row, stream_id)


def fill_draws(seed: torch.Tensor, pos_idx: torch.Tensor, generator: int = GEN_SPLITMIX, stream_id: int = 0, want_u: bool = True,
               want_race_key: bool = True):
    """seed, pos_idx: int64 CUDA tensors holding the u64 bit patterns -> (u f64, race_key int64 bit patterns)."""
    rows = seed.numel()
    u = torch.empty(rows, dtype=torch.float64, device=seed.device) if want_u else None
    rk = torch.empty(rows, dtype=torch.int64, device=seed.device) if want_race_key else None
    _check(lib.whirl_fill_draws(seed.data_ptr(), pos_idx.data_ptr(), rows, generator, stream_id, _p(u), _p(rk),
                                torch.cuda.current_stream(seed.device).cuda_stream))
    return u, rk


def launch_counts() -> dict:
    """Kernel launches made through the library by this process so far, per family."""
    a = (C.c_uint64 * 6)()
    lib.whirl_launch_counts(a, 6)
    return dict(rowscan=a[0], select_generic=a[1], single_pass=a[2], aux=a[3], loss=a[4], blocks=a[5])


def sample_rows_host(x_host, params: dict, rows: int, n: int, dtype: int, out: dict, kept_cap: int = 0, device: int = 0):
    """whirl_sample_rows_host on host buffers: `x_host`, the values of `params` and of `out` are CPU tensors (pinned for
    full copy speed) or None.  Blocks until the tokens are in out['token']."""
    ps = SampleParams()
    for k, _ in SampleParams._fields_:
        if k == "hist_stride":
            continue
        t = params.get(k)
        setattr(ps, k, None if t is None else t.data_ptr())
    ps.hist_stride = 0 if params.get("hist") is None else params["hist"].shape[1]
    o = SampleOut(kept_cap=kept_cap)
    for k, _ in SampleOut._fields_:
        if k == "kept_cap":
            continue
        t = out.get(k)
        setattr(o, k, None if t is None else t.data_ptr())
    st = lib.whirl_sample_rows_host(x_host.data_ptr(), dtype, rows, n, C.byref(ps), C.byref(o), device)
    if st != 0:
        raise WhirlError(st, (lib.whirl_host_last_error() or b"").decode())


def merge_sample_rows(ids, vals, stats, n_total: int, params: RowParams, kept_cap: int = 0) -> SampleResult:
    """ids / vals [shards, rows, K_s], stats [shards, rows, 2] (all-gathered slices) -> one token per row."""
    shards, rows, ks = ids.shape
    dev = ids.device
    res = SampleResult(
        token=torch.empty(rows, dtype=torch.int32, device=dev), status=torch.empty(rows, dtype=torch.int32, device=dev),
        n_kept=torch.empty(rows, dtype=torch.int32, device=dev), closed=torch.empty(rows, dtype=torch.int32, device=dev),
        stats=torch.empty((rows, 2), dtype=torch.float32, device=dev),
        kept_ids=torch.full((rows, kept_cap), -1, dtype=torch.int32, device=dev) if kept_cap else None,
        kept_p=torch.zeros((rows, kept_cap), dtype=torch.float64, device=dev) if kept_cap else None,
        counters=torch.zeros(CNT_WORDS, dtype=torch.int32, device=dev))
    o = SampleOut(token=_p(res.token), status=_p(res.status), n_kept=_p(res.n_kept), closed=_p(res.closed), stats=_p(res.stats),
                  kept_ids=_p(res.kept_ids), kept_p=_p(res.kept_p), kept_cap=kept_cap, counters=_p(res.counters))
    ps = params.struct(rows)
    assert ids.is_contiguous() and vals.is_contiguous() and stats.is_contiguous()
    _check(lib.whirl_merge_sample_rows(ids.data_ptr(), vals.data_ptr(), stats.data_ptr(), shards, rows, ks, n_total, C.byref(ps),
                                       C.byref(o), torch.cuda.current_stream(dev).cuda_stream))
    return res


def merge_sample_rows_packed(blocks: torch.Tensor, shards: int, rows: int, ks: int, n_total: int, params: RowParams,
                             kept_cap: int = 0) -> SampleResult:
    """blocks: int32 tensor of `shards` packed blocks (the all-gather of every rank's block) -> one token per row."""
    dev = blocks.device
    assert blocks.is_contiguous() and blocks.numel() == shards * lib.whirl_shard_block_words(rows, ks)
    res = SampleResult(
        token=torch.empty(rows, dtype=torch.int32, device=dev), status=torch.empty(rows, dtype=torch.int32, device=dev),
        n_kept=torch.empty(rows, dtype=torch.int32, device=dev), closed=torch.empty(rows, dtype=torch.int32, device=dev),
        stats=torch.empty((rows, 2), dtype=torch.float32, device=dev),
        kept_ids=torch.full((rows, kept_cap), -1, dtype=torch.int32, device=dev) if kept_cap else None,
        kept_p=torch.zeros((rows, kept_cap), dtype=torch.float64, device=dev) if kept_cap else None,
        counters=torch.zeros(CNT_WORDS, dtype=torch.int32, device=dev))
    o = SampleOut(token=_p(res.token), status=_p(res.status), n_kept=_p(res.n_kept), closed=_p(res.closed), stats=_p(res.stats),
                  kept_ids=_p(res.kept_ids), kept_p=_p(res.kept_p), kept_cap=kept_cap, counters=_p(res.counters))
    ps = params.struct(rows)
    _check(lib.whirl_merge_sample_rows_packed(blocks.data_ptr(), shards, rows, ks, n_total, C.byref(ps), C.byref(o),
                                              torch.cuda.current_stream(dev).cuda_stream))
    return res


def accept_tokens(tokens, drafts, nd, row0):
    """Device accept loop: tokens [rows] i32, drafts [seqs, D] i32, nd / row0 [seqs] i32 -> (acc, chosen) [seqs] i32."""
    seqs = drafts.shape[0]
    acc = torch.empty(seqs, dtype=torch.int32, device=tokens.device)
    chosen = torch.empty(seqs, dtype=torch.int32, device=tokens.device)
    _check(lib.whirl_accept_tokens(tokens.data_ptr(), drafts.data_ptr(), drafts.shape[1], nd.data_ptr(), row0.data_ptr(), seqs,
                                   acc.data_ptr(), chosen.data_ptr(), torch.cuda.current_stream(tokens.device).cuda_stream))
    return acc, chosen


def accept_rows(tokens, drafts, nd, row0, relax: RelaxParams, greedy=None, relax_on=None, next_tok=None, hist=None, hist_len=None,
                rk_ids=None, rk_vals=None, rk_stats=None, kept: Optional[SampleResult] = None, x=None, inv_t=None):
    """whirl_accept_rows: the accept step with the relaxed rules.  tokens [rows] i32; drafts [seqs, D] i32; nd / row0 / next_tok
    [seqs] i32; greedy / relax_on [seqs] u8; hist [seqs, H] i32 + hist_len [seqs] i32; rk_* the outputs of topk_rows with
    K = rk; kept: a SampleResult with kept_ids / kept_p (the typical rule); x / inv_t the verify logits for open rows.
    Returns (acc, chosen, relaxed, relax_gap, flags)."""
    seqs = drafts.shape[0]
    dev = tokens.device
    a = AcceptIn(tokens=_p(tokens), drafts=_p(drafts), draft_stride=drafts.shape[1], nd=_p(nd), row0=_p(row0), greedy=_p(greedy),
                 relax_on=_p(relax_on), next=_p(next_tok), hist=_p(hist), hist_stride=0 if hist is None else hist.shape[1],
                 hist_len=_p(hist_len), rk_ids=_p(rk_ids), rk_vals=_p(rk_vals), rk_stats=_p(rk_stats),
                 rk=0 if rk_ids is None else rk_ids.shape[1])
    if kept is not None:
        a.kept_cap = 0 if kept.kept_ids is None else kept.kept_ids.shape[1]
        a.kept_ids, a.kept_p, a.n_kept, a.closed, a.stats = _p(kept.kept_ids), _p(kept.kept_p), _p(kept.n_kept), _p(kept.closed), _p(kept.stats)
    if x is not None:
        x, _, n = _rows(x)
        a.x, a.dtype, a.n = x.data_ptr(), _dtype(x), n
    a.inv_t = _p(inv_t)
    acc = torch.empty(seqs, dtype=torch.int32, device=dev)
    chosen = torch.empty(seqs, dtype=torch.int32, device=dev)
    relaxed = torch.zeros(seqs, dtype=torch.int32, device=dev)
    gap = torch.zeros(seqs, dtype=torch.float64, device=dev)
    flags = torch.zeros(seqs, dtype=torch.int32, device=dev)
    _check(lib.whirl_accept_rows(C.byref(a), C.byref(relax), seqs, acc.data_ptr(), chosen.data_ptr(), relaxed.data_ptr(), gap.data_ptr(),
                                 flags.data_ptr(), torch.cuda.current_stream(dev).cuda_stream))
    return acc, chosen, relaxed, gap, flags


def spec_accept_residual(target, draft, draft_tok, inv_t, u_acc, u_res):
    """target [seqs, L + 1, n], draft [seqs, L, n] logits; draft_tok [seqs, L] i32; inv_t [seqs] f32 or None;
    u_acc [seqs, L], u_res [seqs, L + 1] f64 -> (n_acc, next_tok) [seqs] i32."""
    seqs, L1, n = target.shape
    L = L1 - 1
    dev = target.device
    n_acc = torch.empty(seqs, dtype=torch.int32, device=dev)
    nxt = torch.empty(seqs, dtype=torch.int32, device=dev)
    ws = torch.empty(lib.whirl_spec_workspace_bytes(seqs, L), dtype=torch.uint8, device=dev)
    _check(lib.whirl_spec_accept_residual(target.data_ptr(), _p(draft), _dtype(target), seqs, L, n, _p(draft_tok), _p(inv_t), _p(u_acc),
                                          u_res.data_ptr(), n_acc.data_ptr(), nxt.data_ptr(), ws.data_ptr(), ws.numel(),
                                          torch.cuda.current_stream(dev).cuda_stream))
    return n_acc, nxt


# ---- training on sampled tokens -------------------------------------------------------------------------------------------

MEAN_SUM, MEAN_TOKENS, MEAN_SEQS = 0, 1, 2
PREF_SIGMOID, PREF_HINGE, PREF_SQUARED = 0, 1, 2


def _i32(v: int, name: str) -> int:
    """v, refused where a C int does not hold it (ctypes would cut it)."""
    if not -2 ** 31 <= v < 2 ** 31:
        raise ValueError(f"{name} = {v} does not fit 32 bits")
    return v


def _loss_rows(x: torch.Tensor):
    """Logits [rows, n] whose rows may lie further apart than n (a padded vocabulary): (dtype, rows, n, ld)."""
    if not x.is_cuda:
        raise ValueError("logits must be on a CUDA device (this library has no CPU path)")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"logits must be [rows, n], got {tuple(x.shape)}")
    rows, n = x.shape
    s0, s1 = x.stride()
    if (n > 1 and s1 != 1) or (rows > 1 and s0 < n):
        raise ValueError(f"logits must be rows of consecutive elements that do not overlap, got strides {(s0, s1)}")
    return _dtype(x), _i32(rows, "rows"), _i32(n, "n"), (s0 if rows > 1 else n)


def _vec(t: Optional[torch.Tensor], name: str, dtype, shape, dev: int):
    """The address of a contiguous tensor of the given type and shape on CUDA device `dev` (None stays None)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"{name}: want a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{dev}, got {t.dtype} {tuple(t.shape)} "
                        f"on {t.device}")
    return t.data_ptr()


def _grad_out(x: torch.Tensor, dx: Optional[torch.Tensor], ld: int) -> torch.Tensor:
    """dx, checked; a new one has rows as x has them to 16 bytes (the kernels' fast case), and no more of a gap than that takes."""
    if dx is None:
        rows, n = x.shape
        gap = (ld - n) % (16 // x.element_size())
        return torch.empty((rows, n + gap), dtype=x.dtype, device=x.device)[:, :n] if gap else torch.empty((rows, n), dtype=x.dtype, device=x.device)
    if dx.dtype != x.dtype or dx.device != x.device or dx.shape != x.shape:
        raise TypeError(f"dx: want {x.dtype} {tuple(x.shape)} on {x.device}, got {dx.dtype} {tuple(dx.shape)} on {dx.device}")
    torch.autograd.graph.increment_version(dx)  # (autograd does not see the kernels' writes: a graph that kept dx, or x where they are one, has to)
    return dx


def _call(dev: int, fn, *args):
    """fn(*args, stream) on the device's current stream, with that device current.  (The raw calls: a Stream object and a device
    context cost several microseconds, as much as a small kernel.)"""
    if dev == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if status:
        _check(status)


@dataclass
class LogprobResult:
    logp: torch.Tensor                # [rows] float32
    stats: torch.Tensor               # [rows, 2] float32: max, sum exp((x - max) * inv_t)
    entropy: Optional[torch.Tensor]   # [rows] float32


def token_logprobs(x, token, inv_t: float = 1.0, inv_t_rows=None, want_entropy: bool = False) -> LogprobResult:
    """Log-probability of token[r] under row r of the logits, the row's softmax statistics, and its entropy
    (whirl_token_logprobs).  x [rows, n] float32 / bfloat16, rows may be padded; token [rows] int32.  A row whose token lies
    outside [0, n) is not read and gets zeros."""
    dt, rows, n, ld = _loss_rows(x)
    f32, rs, dev = torch.float32, (rows,), x.get_device()
    tok, it = _vec(token, "token", torch.int32, rs, dev), _vec(inv_t_rows, "inv_t_rows", f32, rs, dev)
    logp = torch.empty(rows, dtype=f32, device=dev)
    stats = torch.empty((rows, 2), dtype=f32, device=dev)
    entropy = torch.empty(rows, dtype=f32, device=dev) if want_entropy else None
    _call(dev, lib.whirl_token_logprobs, x.data_ptr(), dt, rows, n, ld, tok, inv_t, it, logp.data_ptr(), stats.data_ptr(), _p(entropy))
    return LogprobResult(logp, stats, entropy)


def token_logprobs_grad(x, token, stats, g_logp, inv_t: float = 1.0, inv_t_rows=None, entropy=None, g_entropy=None, dx=None) -> torch.Tensor:
    """The gradient by the logits of a loss whose gradients by logp and (optionally) entropy are g_logp and g_entropy [rows]
    float32 (whirl_token_logprobs_grad).  stats, entropy: what token_logprobs returned.  dx may be x itself."""
    dt, rows, n, ld = _loss_rows(x)
    f32, rs, dev = torch.float32, (rows,), x.get_device()
    args = (_vec(token, "token", torch.int32, rs, dev), inv_t, _vec(inv_t_rows, "inv_t_rows", f32, rs, dev), _vec(stats, "stats", f32, (rows, 2), dev),
            _vec(entropy, "entropy", f32, rs, dev), _vec(g_logp, "g_logp", f32, rs, dev), _vec(g_entropy, "g_entropy", f32, rs, dev))
    dx = _grad_out(x, dx, ld)
    _call(dev, lib.whirl_token_logprobs_grad, x.data_ptr(), dt, rows, n, ld, *args, dx.data_ptr(), _loss_rows(dx)[3])
    return dx


@dataclass
class PolicyResult:
    loss: torch.Tensor                # [] float32
    logp: torch.Tensor                # [rows] float32, and so on
    entropy: Optional[torch.Tensor]   # (with ent_coef or want_entropy)
    kl: Optional[torch.Tensor]        # (with ref_logp)
    row_loss: torch.Tensor
    dx: Optional[torch.Tensor]        # d loss / d x: logits.backward(result.dx) goes on from there
    aux: torch.Tensor                 # what the properties below are views of (an allocation of its own each would cost more than the view)

    @property
    def stats(self) -> torch.Tensor:  # [rows, 2]: max, sum exp((x - max) * inv_t)
        n = self.logp.numel()
        return self.aux[: 2 * n].view(n, 2)

    @property
    def g_logp(self) -> torch.Tensor:  # d loss / d logp
        n = self.logp.numel()
        return self.aux[2 * n: 3 * n]

    @property
    def row_scale(self) -> torch.Tensor:  # a row's share of the loss; the entropy's gradient is -ent_coef * row_scale
        n = self.logp.numel()
        return self.aux[3 * n: 4 * n]


def policy_loss(x, token, adv, old_logp=None, ref_logp=None, weight=None, seq_start=None, inv_t: float = 1.0, inv_t_rows=None,
                clip_low: float = 0.2, clip_high: float = 0.2, dual_clip: float = 0.0, kl_coef: float = 0.0, ent_coef: float = 0.0,
                mean: int = MEAN_TOKENS, want_grad: bool = True, want_entropy: bool = False, dx=None) -> PolicyResult:
    """The clipped policy loss with a KL term on logits x [rows, n] and the tokens sampled from them, with its gradient by the
    logits (whirl_policy_loss).  adv, old_logp, ref_logp, weight: [rows] float32 (weight 0: a prompt or padding row, not read);
    seq_start: [seqs + 1] int32, needed by MEAN_SEQS.  dx may be x itself."""
    dt, rows, n, ld = _loss_rows(x)
    f32, i32, rs, dev = torch.float32, torch.int32, (rows,), x.get_device()
    if mean == MEAN_SEQS and (seq_start is None or seq_start.dim() != 1 or seq_start.numel() < 1):
        raise ValueError("policy_loss: MEAN_SEQS needs seq_start [seqs + 1]")
    seqs = 0 if seq_start is None else _i32(seq_start.numel() - 1, "seqs")
    p = PolicyParams(_vec(token, "token", i32, rs, dev), _vec(adv, "adv", f32, rs, dev), _vec(old_logp, "old_logp", f32, rs, dev),
                     _vec(ref_logp, "ref_logp", f32, rs, dev), _vec(weight, "weight", f32, rs, dev),
                     None if seq_start is None else _vec(seq_start, "seq_start", i32, (seqs + 1,), dev), seqs, mean,
                     _vec(inv_t_rows, "inv_t_rows", f32, rs, dev), inv_t, clip_low, clip_high, dual_clip, kl_coef, ent_coef)
    ent, kl = want_entropy or ent_coef != 0.0, ref_logp is not None
    loss, logp, row_loss = torch.empty((), dtype=f32, device=dev), torch.empty(rows, dtype=f32, device=dev), torch.empty(rows, dtype=f32, device=dev)
    entropy = torch.empty(rows, dtype=f32, device=dev) if ent else None
    kl = torch.empty(rows, dtype=f32, device=dev) if kl else None
    nbytes = lib.whirl_loss_workspace_bytes(rows, seqs)
    aux = torch.empty(4 * rows + (nbytes + 3) // 4, dtype=f32, device=dev)  # stats, g_logp, row_scale, and the workspace behind them
    base = aux.data_ptr()
    dx = _grad_out(x, dx, ld) if want_grad else None
    o = PolicyOut(loss.data_ptr(), logp.data_ptr(), base, _p(entropy), _p(kl), row_loss.data_ptr(), base + 8 * rows, base + 12 * rows, _p(dx),
                  _loss_rows(dx)[3] if want_grad else 0)
    _call(dev, lib.whirl_policy_loss, x.data_ptr(), dt, rows, n, ld, p, o, base + 16 * rows, nbytes)
    return PolicyResult(loss, logp, entropy, kl, row_loss, dx, aux)


def loss_check(r: PolicyResult) -> int:
    """whirl_loss_check: 1 if a wait of the policy_loss call that returned r ran out (rows are NaN that need not be), else 0.
    Synchronises the stream."""
    where, ws = C.c_uint32(0), r.aux[4 * r.logp.numel():]
    with torch.cuda.device(r.aux.device):
        st = lib.whirl_loss_check(ws.data_ptr(), 4 * ws.numel(), torch.cuda.current_stream().cuda_stream, C.byref(where))
    if st not in (0, ERR_TIMEOUT):
        _check(st)
    return int(where.value)


@dataclass
class PreferenceResult:
    loss: torch.Tensor          # [] float32
    pair_loss: torch.Tensor     # [pairs]
    reward: torch.Tensor        # [pairs, 2]: chosen, rejected
    logp: torch.Tensor          # [rows]
    dx: Optional[torch.Tensor]  # d loss / d x: logits.backward(result.dx) goes on from there
    aux: torch.Tensor

    @property
    def stats(self) -> torch.Tensor:  # [rows, 2]: max, sum exp((x - max) * inv_t)
        n = self.logp.numel()
        return self.aux[: 2 * n].view(n, 2)

    @property
    def g_logp(self) -> torch.Tensor:  # d loss / d logp
        n = self.logp.numel()
        return self.aux[2 * n: 3 * n]


def preference_loss(x, token, seq_start, ref_logp=None, weight=None, inv_t: float = 1.0, inv_t_rows=None, beta: float = 0.1,
                    kind: int = PREF_SIGMOID, smoothing: float = 0.0, margin: float = 0.0, average: bool = False, want_grad: bool = True,
                    dx=None) -> PreferenceResult:
    """The preference loss of pairs of sequences packed row after row in x [rows, n] (chosen, rejected, chosen, rejected ...;
    sequence s holds the rows seq_start[s] to seq_start[s + 1]), with its gradient by the logits (whirl_preference_loss).
    ref_logp, weight: [rows] float32.  dx may be x itself."""
    dt, rows, n, ld = _loss_rows(x)
    f32, i32, rs, dev = torch.float32, torch.int32, (rows,), x.get_device()
    if seq_start.dim() != 1 or seq_start.numel() % 2 != 1:
        raise ValueError(f"preference_loss: seq_start is [2 * pairs + 1], got {tuple(seq_start.shape)}")
    pairs = _i32(seq_start.numel() // 2, "pairs")
    p = PreferenceParams(_vec(token, "token", i32, rs, dev), _vec(seq_start, "seq_start", i32, (2 * pairs + 1,), dev),
                         _vec(ref_logp, "ref_logp", f32, rs, dev), _vec(weight, "weight", f32, rs, dev), _vec(inv_t_rows, "inv_t_rows", f32, rs, dev),
                         pairs, kind, int(average), inv_t, beta, smoothing, margin)
    loss, logp = torch.empty((), dtype=f32, device=dev), torch.empty(rows, dtype=f32, device=dev)
    pair_loss, reward = torch.empty(pairs, dtype=f32, device=dev), torch.empty((pairs, 2), dtype=f32, device=dev)
    nbytes = lib.whirl_loss_workspace_bytes(rows, pairs)
    aux = torch.empty(3 * rows + (nbytes + 3) // 4, dtype=f32, device=dev)  # stats, g_logp, and the workspace behind them
    base = aux.data_ptr()
    dx = _grad_out(x, dx, ld) if want_grad else None
    o = PreferenceOut(loss.data_ptr(), pair_loss.data_ptr(), reward.data_ptr(), logp.data_ptr(), base, base + 8 * rows, _p(dx),
                      _loss_rows(dx)[3] if want_grad else 0)
    _call(dev, lib.whirl_preference_loss, x.data_ptr(), dt, rows, n, ld, p, o, base + 12 * rows, nbytes)
    return PreferenceResult(loss, pair_loss, reward, logp, dx, aux)


# ---- the rows of the next step --------------------------------------------------------------------------------------------

SEQ_OK, SEQ_REFUSED, SEQ_INVALID = 0, 1, 2
MAX_SEQS = 65536


@dataclass
class StepRows:
    slot: torch.Tensor      # [max_rows] int64, -1 behind the last row
    position: torch.Tensor  # [max_rows] int32
    seq: torch.Tensor       # [max_rows] int32, -1 behind the last row
    row0: torch.Tensor      # [seqs + 1] int32
    status: torch.Tensor    # [seqs] int32: SEQ_*


def block_tables_step(length, n_new, table, owned, free_ids, free_count, block_size: int, max_rows: int,
                      rows: Optional[StepRows] = None) -> StepRows:
    """Blocks, slots and positions of the next step's rows from the sequences' lengths (whirl_block_tables_step).  length, n_new,
    owned [seqs], table [seqs, max_blocks], free_ids [num_blocks], free_count [1]: int32; the last four are updated."""
    if table.dim() != 2 or not table.is_cuda:
        raise ValueError("block_tables_step: table must be [seqs, max_blocks] on a CUDA device")
    i32, dev = torch.int32, table.get_device()
    seqs, width = table.shape
    blocks, ss = _i32(free_ids.numel(), "num_blocks"), (seqs,)
    block_size, max_rows, seqs, width = (_i32(v, k) for v, k in ((block_size, "block_size"), (max_rows, "max_rows"), (seqs, "seqs"), (width, "max_blocks")))
    if rows is None:
        rows = StepRows(torch.empty(max_rows, dtype=torch.int64, device=dev), torch.empty(max_rows, dtype=i32, device=dev),
                        torch.empty(max_rows, dtype=i32, device=dev), torch.empty(seqs + 1, dtype=i32, device=dev),
                        torch.empty(seqs, dtype=i32, device=dev))
        out = rows.slot.data_ptr(), rows.position.data_ptr(), rows.seq.data_ptr(), rows.row0.data_ptr(), rows.status.data_ptr()
    else:
        mr = (max_rows,)
        out = (_vec(rows.slot, "slot", torch.int64, mr, dev), _vec(rows.position, "position", i32, mr, dev), _vec(rows.seq, "seq", i32, mr, dev),
               _vec(rows.row0, "row0", i32, (seqs + 1,), dev), _vec(rows.status, "status", i32, ss, dev))
    t = BlockTables(_vec(table, "table", i32, (seqs, width), dev), _vec(owned, "owned", i32, ss, dev), _vec(free_ids, "free_ids", i32, (blocks,), dev),
                    _vec(free_count, "free_count", i32, (1,), dev), seqs, width, blocks, block_size)
    o = StepRowsOut(*out, max_rows)
    nbytes = lib.whirl_block_workspace_bytes(seqs)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call(dev, lib.whirl_block_tables_step, _vec(length, "length", i32, ss, dev), _vec(n_new, "n_new", i32, ss, dev), t, o, ws.data_ptr(), nbytes)
    return rows
