"""Device-tensor front end of the C ABI.

Torch is used only to hold device memory and the current HIP stream; every
computation runs in libstrim_sampler.so. Inputs must already live on the GPU. A call with a
`stream` is queued there: the caller makes that stream wait for the inputs, and whoever
uses the results wait for that stream.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple

import numpy as np
import torch

from . import _native as N


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream=None) -> ctypes.c_void_p:
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _tensors(*xs):
    """The tensors among a call's arguments or results."""
    for x in xs:
        if isinstance(x, torch.Tensor):
            yield x
        elif isinstance(x, Q4Weight):
            yield from _tensors(x.words, x.scales, x.biases)
        elif isinstance(x, tuple):
            yield from _tensors(*x)


def _elsewhere(stream, device: torch.device) -> bool:
    """Whether a call on `device` has to be made by _there: on a given stream, or with another
    device current."""
    return stream is not None or torch._C._cuda_getDevice() != device.index


def _there(fn, stream, device: torch.device, *args):
    """fn(*args) with `device` current (the default stream, and what a kernel is told once, are the
    current device's). With a given stream that stream is current too: temporary memory is taken from
    it and goes back to it, in the order of its work (taken from the caller's stream it would be
    handed out again while the kernels still use it); the caller's tensors are not handed out again
    before that stream is done with them, nor the results before the caller's is."""
    if stream is None:
        with torch.cuda.device(device):
            return fn(*args)
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(stream.cuda_stream, device)
    if stream.device != device:
        raise ValueError(f"the stream is one of {stream.device}, the tensors are on {device}")
    caller = torch.cuda.current_stream(device)
    for t in _tensors(*args):
        t.record_stream(stream)
    with torch.cuda.stream(stream):
        out = fn(*args)
    for t in _tensors(out):
        t.record_stream(caller)
    return out


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return N.DTYPE_BF16
    if t.dtype == torch.float32:
        return N.DTYPE_F32
    raise TypeError(f"logits must be bfloat16 or float32, got {t.dtype}")


def host_params(params) -> np.ndarray:
    """strim_sampling_params rows as a contiguous host array (the C ABI reads them at
    call time; the caller may reuse the memory as soon as the call returns)."""
    return np.ascontiguousarray(params, dtype=N.PARAMS_DTYPE).reshape(-1)


def _pp(p: np.ndarray) -> ctypes.c_void_p:
    return p.ctypes.data_as(ctypes.c_void_p)


def _check_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("every tensor argument must be on the GPU")
        if t is not None and not t.is_contiguous():
            raise ValueError("tensor arguments must be contiguous")


def as_rows(t: torch.Tensor) -> torch.Tensor:
    """[..., n] as [R, n], also where R or n is 0."""
    return t.unsqueeze(0) if t.dim() == 1 else t.flatten(0, -2)


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows (a single row may carry any stride, e.g. 0 from a
    broadcast view: its own length is passed)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_rows(t: torch.Tensor) -> None:
    """Logits may have a row stride > V, but each row must be contiguous."""
    if not t.is_cuda:
        raise ValueError("logits must be on the GPU")
    if t.dim() != 2 or t.stride(1) != 1 or _row_stride(t) < t.shape[1]:
        raise ValueError("logits must be [R, V] with contiguous rows (row stride >= V)")


class Context:
    """strim_ctx: scratch for up to max_rows rows of up to max_vocab tokens."""

    def __init__(self, device: int = 0, max_rows: int = 64, max_vocab: int = 262144):
        self.device = device
        self.max_rows = max_rows
        self.max_vocab = max_vocab
        h = ctypes.c_void_p()
        with torch.cuda.device(device):
            N.check(N.lib().strim_ctx_create(ctypes.byref(h), device, max_rows, max_vocab),
                    "strim_ctx_create")
        self._h = h

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            torch.cuda.synchronize(self.device)
            N.check(N.lib().strim_ctx_destroy(self._h), "strim_ctx_destroy")
            self._h = None

    def __del__(self):  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass

    # -------------------------------------------------------------------------
    def profile_begin(self, max_launches: int) -> None:
        N.check(N.lib().strim_profile_begin(self._h, max_launches), "strim_profile_begin")

    def profile_end(self) -> dict:
        """{kernel name: (total ms, launches)} since profile_begin (synchronises)."""
        tot = np.zeros(N.KERNEL_COUNT, np.float64)
        cnt = np.zeros(N.KERNEL_COUNT, np.int64)
        N.check(N.lib().strim_profile_end(self._h, tot.ctypes.data_as(ctypes.c_void_p),
                                          cnt.ctypes.data_as(ctypes.c_void_p)),
                "strim_profile_end")
        return {N.lib().strim_kernel_name(i).decode(): (float(tot[i]), int(cnt[i]))
                for i in range(N.KERNEL_COUNT)}

    def sample(self, logits: torch.Tensor, params, mask: torch.Tensor | None = None,
               history: torch.Tensor | None = None, history_len: torch.Tensor | None = None,
               noise_mode: int = N.NOISE_ICDF, noise: torch.Tensor | None = None,
               want_probs: bool = False, out_ids: torch.Tensor | None = None,
               out_status: torch.Tensor | None = None, stream=None):
        """strim_sample over logits [B,V]. Returns (ids int32[B], status int32[B],
        probs float32[B,V] or None), all on the device."""
        if logits.dim() == 1:
            logits = logits.unsqueeze(0)
        B, V = logits.shape
        dev = logits.device
        p = host_params(params)
        if p.size != B:
            raise ValueError(f"need {B} param rows, got {p.size}")
        _check_rows(logits)
        _check_cuda(mask, history, history_len, noise)
        if out_ids is None:
            out_ids = torch.empty(B, dtype=torch.int32, device=dev)
        if out_status is None:
            out_status = torch.empty(B, dtype=torch.int32, device=dev)
        probs = torch.empty(B, V, dtype=torch.float32, device=dev) if want_probs else None
        H = 0 if history is None else history.shape[-1]
        mstride = 0 if mask is None else mask.shape[-1]
        rc = N.lib().strim_sample(self._h, _stream(stream), _ptr(logits), _dtype_code(logits),
                                  B, V, _row_stride(logits), _pp(p), _ptr(mask), mstride,
                                  _ptr(history), _ptr(history_len), H, noise_mode, _ptr(noise),
                                  _ptr(out_ids), _ptr(out_status), _ptr(probs))
        N.check(rc, "strim_sample")
        return out_ids, out_status, probs

    def bind_sample(self, logits: torch.Tensor, params, mask: torch.Tensor | None = None,
                    history: torch.Tensor | None = None,
                    history_len: torch.Tensor | None = None, noise_mode: int = N.NOISE_ICDF,
                    noise: torch.Tensor | None = None, out_ids: torch.Tensor | None = None,
                    out_status: torch.Tensor | None = None, stream=None) -> "BoundCall":
        """strim_sample with every argument converted once: calling the result launches
        the step again on the same buffers (the tensors must stay alive). For loops that
        reuse buffers, such as a decode loop or HIP-graph capture."""
        if logits.dim() == 1:
            logits = logits.unsqueeze(0)
        B, V = logits.shape
        dev = logits.device
        p = host_params(params)
        if p.size != B:
            raise ValueError(f"need {B} param rows, got {p.size}")
        _check_rows(logits)
        _check_cuda(mask, history, history_len, noise)
        if out_ids is None:
            out_ids = torch.empty(B, dtype=torch.int32, device=dev)
        if out_status is None:
            out_status = torch.empty(B, dtype=torch.int32, device=dev)
        H = 0 if history is None else history.shape[-1]
        mstride = 0 if mask is None else mask.shape[-1]
        args = [self._h, None, _ptr(logits), _dtype_code(logits), B, V,
                _row_stride(logits), _pp(p), _ptr(mask), mstride, _ptr(history), _ptr(history_len),
                H, noise_mode, _ptr(noise), _ptr(out_ids), _ptr(out_status), None]
        keep = (logits, p, mask, history, history_len, noise, out_ids, out_status)
        return BoundCall(N.lib().strim_sample, args, keep, out_ids, out_status, stream)

    def verify(self, target_logits: torch.Tensor, draft_tokens: torch.Tensor | None, params,
               draft_logits: torch.Tensor | None = None,
               draft_to_full: torch.Tensor | None = None, mask: torch.Tensor | None = None,
               history: torch.Tensor | None = None, history_len: torch.Tensor | None = None,
               noise_mode: int = N.NOISE_ICDF, noise: torch.Tensor | None = None,
               row_outputs: bool = True, stream=None):
        """strim_verify over target [B,k+1,V]. Returns a dict of device tensors:
        accepted [B], token [B], status [B], row_accept [B,k], row_token [B,k+1]."""
        B, k1, V = target_logits.shape
        k = k1 - 1
        dev = target_logits.device
        p = host_params(params)
        if p.size != B:
            raise ValueError(f"need {B} param rows, got {p.size}")
        _check_cuda(target_logits, draft_tokens, draft_logits, draft_to_full, mask, history,
                    history_len, noise)
        acc = torch.empty(B, dtype=torch.int32, device=dev)
        tok = torch.empty(B, dtype=torch.int32, device=dev)
        st = torch.empty(B, dtype=torch.int32, device=dev)
        racc = torch.empty(B, max(k, 1), dtype=torch.int32, device=dev) if row_outputs else None
        rtok = torch.empty(B, k + 1, dtype=torch.int32, device=dev) if row_outputs else None
        H = 0 if history is None else history.shape[-1]
        mstride = 0 if mask is None else mask.shape[-1]
        Vd = 0 if draft_logits is None else draft_logits.shape[-1]
        if draft_logits is not None:
            if draft_logits.dtype != target_logits.dtype:
                raise ValueError("draft_logits must have the target logits' dtype")
            if tuple(draft_logits.shape) != (B, k, Vd) or not draft_logits.is_contiguous():
                raise ValueError(f"draft_logits must be contiguous [{B}, {k}, Vd]")
            if draft_to_full is None or draft_to_full.numel() != Vd:
                raise ValueError("draft_to_full must hold Vd ids")
        rc = N.lib().strim_verify(self._h, _stream(stream), _ptr(target_logits),
                                  _dtype_code(target_logits), B, k, V, _ptr(draft_logits), Vd,
                                  _ptr(draft_to_full), _ptr(draft_tokens), _pp(p), _ptr(mask),
                                  mstride, _ptr(history), _ptr(history_len), H, noise_mode,
                                  _ptr(noise), _ptr(acc), _ptr(tok), _ptr(racc), _ptr(rtok),
                                  _ptr(st))
        N.check(rc, "strim_verify")
        return {"accepted": acc, "token": tok, "status": st,
                "row_accept": None if racc is None else racc[:, :k], "row_token": rtok}


    def bind_verify(self, target_logits: torch.Tensor, draft_tokens: torch.Tensor, params,
                    draft_logits: torch.Tensor | None = None,
                    draft_to_full: torch.Tensor | None = None,
                    noise_mode: int = N.NOISE_GUMBEL, noise: torch.Tensor | None = None,
                    stream=None) -> "BoundCall":
        """strim_verify with every argument converted and the outputs allocated once:
        calling the result launches the verify again on the same buffers (for HIP-graph
        capture). Its out_ids / out_status are the accepted counts and the tokens."""
        B, k1, V = target_logits.shape
        k = k1 - 1
        dev = target_logits.device
        p = host_params(params)
        if p.size != B:
            raise ValueError(f"need {B} param rows, got {p.size}")
        _check_cuda(target_logits, draft_tokens, draft_logits, draft_to_full, noise)
        Vd = 0 if draft_logits is None else draft_logits.shape[-1]
        if draft_logits is not None and (tuple(draft_logits.shape) != (B, k, Vd)
                                         or not draft_logits.is_contiguous()
                                         or draft_logits.dtype != target_logits.dtype):
            raise ValueError(f"draft_logits must be contiguous [{B}, {k}, Vd] of the target dtype")
        acc = torch.empty(B, dtype=torch.int32, device=dev)
        tok = torch.empty(B, dtype=torch.int32, device=dev)
        st = torch.empty(B, dtype=torch.int32, device=dev)
        args = [self._h, None, _ptr(target_logits), _dtype_code(target_logits), B, k, V,
                _ptr(draft_logits), Vd, _ptr(draft_to_full), _ptr(draft_tokens), _pp(p), None, 0,
                None, None, 0, noise_mode, _ptr(noise), _ptr(acc), _ptr(tok), None, None,
                _ptr(st)]
        keep = (target_logits, draft_tokens, p, draft_logits, draft_to_full, noise, acc, tok, st)
        call = BoundCall(N.lib().strim_verify, args, keep, acc, tok, stream, "strim_verify")
        call.status = st
        return call


def mask_logits(logits: torch.Tensor, mask_words: torch.Tensor | None, stream=None):
    """maskLogits (TokenMask.swift:15-17): float32 logits with disallowed tokens at -inf."""
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    R, V = logits.shape
    _check_rows(logits)
    _check_cuda(mask_words)
    out = torch.empty(R, V, dtype=torch.float32, device=logits.device)
    mstride = 0 if mask_words is None else mask_words.shape[-1]
    N.check(N.lib().strim_mask_logits(_stream(stream), _ptr(logits), _dtype_code(logits), R, V,
                                      _row_stride(logits), _ptr(mask_words), mstride, _ptr(out)),
            "strim_mask_logits")
    return out


def head_logits(hidden: torch.Tensor, lm_head: torch.Tensor,
                norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                out: torch.Tensor | None = None, xn: torch.Tensor | None = None, stream=None):
    """The producer of the logits: final RMSNorm and dense lm_head of the decode step
    (QwenModel.swift:202-212; Weights.swift:244-255,270-273) on the GPU. hidden bf16 [B, K],
    lm_head bf16 [V, K], norm_weight bf16 [K] (None: hidden is already normalised).
    Returns bf16 logits [B, V] (or fills `out`), the layout sample/verify take."""
    if hidden.dim() == 1:
        hidden = hidden.unsqueeze(0)
    for t in (hidden, lm_head, norm_weight, out, xn):
        _check_cuda(t)
        if t is not None and t.dtype != torch.bfloat16:
            raise TypeError("head_logits takes bf16 tensors")
    B, K = hidden.shape
    V = lm_head.shape[0]
    if lm_head.shape[1] != K:
        raise ValueError(f"lm_head is [{lm_head.shape[0]}, {lm_head.shape[1]}], hidden K={K}")
    if _elsewhere(stream, hidden.device):
        return _there(head_logits, stream, hidden.device, hidden, lm_head, norm_weight, eps, out, xn)
    if out is None:
        out = torch.empty(B, V, dtype=torch.bfloat16, device=hidden.device)
    if norm_weight is not None and xn is None:
        xn = torch.empty(B, K, dtype=torch.bfloat16, device=hidden.device)
    N.check(N.lib().strim_head_logits(_stream(), _ptr(hidden), _row_stride(hidden), B, K,
                                      _ptr(norm_weight), float(eps), _ptr(xn), _ptr(lm_head),
                                      _row_stride(lm_head), V, _ptr(out), _row_stride(out)),
            "strim_head_logits")
    return out


def head_greedy(ctx: "Context", hidden: torch.Tensor, lm_head: torch.Tensor,
                norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                out_logits: torch.Tensor | None = None, xn: torch.Tensor | None = None,
                ids: torch.Tensor | None = None, status: torch.Tensor | None = None,
                stream=None):
    """Hidden -> greedy token with the pick fused into the producer (strim_head_greedy):
    the first maximum of each row's bf16 logits, which strim_sample gives for a T <= 0 row
    without penalties, mask or filters. out_logits None: the logits are not written.
    Returns (ids, status) int32 [B]."""
    if hidden.dim() == 1:
        hidden = hidden.unsqueeze(0)
    for t in (hidden, lm_head, norm_weight, out_logits, xn):
        _check_cuda(t)
        if t is not None and t.dtype != torch.bfloat16:
            raise TypeError("head_greedy takes bf16 tensors")
    B, K = hidden.shape
    V = lm_head.shape[0]
    if lm_head.shape[1] != K:
        raise ValueError(f"lm_head is [{lm_head.shape[0]}, {lm_head.shape[1]}], hidden K={K}")
    if _elsewhere(stream, hidden.device):
        return _there(head_greedy, stream, hidden.device, ctx, hidden, lm_head, norm_weight, eps,
                      out_logits, xn, ids, status)
    if norm_weight is not None and xn is None:
        xn = torch.empty(B, K, dtype=torch.bfloat16, device=hidden.device)
    if ids is None:
        ids = torch.empty(B, dtype=torch.int32, device=hidden.device)
    if status is None:
        status = torch.empty(B, dtype=torch.int32, device=hidden.device)
    N.check(N.lib().strim_head_greedy(ctx.handle, _stream(), _ptr(hidden),
                                      _row_stride(hidden), B, K, _ptr(norm_weight), float(eps),
                                      _ptr(xn), _ptr(lm_head), _row_stride(lm_head), V,
                                      _ptr(out_logits),
                                      _row_stride(out_logits) if out_logits is not None else 0,
                                      _ptr(ids), _ptr(status)),
            "strim_head_greedy")
    return ids, status


# What a small call costs is mostly this file's own time, so the checks of the loss and of the
# 4-bit projections ask each tensor for as little as they can.
def _check_bf16_rows(name: str, t: torch.Tensor) -> None:
    """A bf16 operand of the loss: [R, K] with contiguous rows, 16-byte aligned."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError("every tensor argument must be on the GPU")
    if t.dim() != 2 or (not t.is_contiguous() and t.stride(1) != 1):
        raise ValueError(f"{name} must be [rows, K] with contiguous rows")


def _stream_of(device: torch.device) -> int:
    """The handle of `device`'s current stream (without the Stream object that
    torch.cuda.current_stream makes, 2.6 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _check_with(device: torch.device, *ts) -> None:
    """Contiguous tensors (or None) on `device`."""
    for t in ts:
        if t is None:
            continue
        if t.device != device:
            raise ValueError("every tensor argument must be on the same GPU")
        if not t.is_contiguous():
            raise ValueError("tensor arguments must be contiguous")


def check_ignore_index(ignore_index: int) -> None:
    if not -2 ** 31 <= ignore_index < 2 ** 31:
        raise ValueError(f"ignore_index must be a 32-bit number, got {ignore_index}")


def _loss_args(hidden, lm_head, targets, ignore_index):
    check_ignore_index(ignore_index)
    _check_bf16_rows("hidden", hidden)
    _check_bf16_rows("lm_head", lm_head)
    _check_with(hidden.device, targets)
    R, K = hidden.shape
    V, KW = lm_head.shape
    if lm_head.device != hidden.device:
        raise ValueError("every tensor argument must be on the same GPU")
    if KW != K:
        raise ValueError(f"lm_head is [{V}, {KW}], hidden K={K}")
    if targets.dtype != torch.int32 or targets.shape != (R,):
        raise ValueError(f"targets must be int32 [{R}]")
    return R, K, V


def _workspace(workspace, need: int, device) -> torch.Tensor | None:
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    _check_with(device, workspace)
    if workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace must hold {need} bytes")
    return workspace


def _bytes(t) -> int:
    return 0 if t is None else t.numel() * t.element_size()


@lru_cache(maxsize=256)
def head_loss_workspace(rows: int, K: int, V: int, want_hidden: bool = False,
                        want_lm_head: bool = False) -> int:
    """Bytes of workspace that head_loss (no gradient wanted) or head_loss_grad takes."""
    need = N.lib().strim_head_loss_workspace(rows, K, V, int(want_hidden), int(want_lm_head))
    if need < 0:
        raise N.StrimError(need, "strim_head_loss_workspace")
    return need


@lru_cache(maxsize=256)
def head_logits_q4_workspace(B: int, K: int) -> int:
    """Bytes of workspace that head_logits_q4 takes (0 for a few rows)."""
    need = N.lib().strim_head_logits_packed_workspace(B, K)
    if need < 0:
        raise N.StrimError(need, "strim_head_logits_packed_workspace")
    return need


def head_loss(hidden: torch.Tensor, lm_head: torch.Tensor, targets: torch.Tensor,
              ignore_index: int = -100, workspace: torch.Tensor | None = None, stream=None):
    """Cross entropy of hidden bf16 [N, K] projected by lm_head bf16 [V, K] against targets
    int32 [N], without keeping the logits. Returns (loss float32 [N], lse float32 [N], status
    int32 [N]): minus the targets' log-probabilities, the logits' log-sum-exp, and OK, EINVAL
    (a target outside [0, V) that is not ignore_index) or ENONFINITE. Ignored rows have loss
    0. strim_amd.loss has the differentiable form."""
    R, K, V = _loss_args(hidden, lm_head, targets, ignore_index)
    dev = hidden.device
    if _elsewhere(stream, dev):
        return _there(head_loss, stream, dev, hidden, lm_head, targets, ignore_index, workspace)
    loss = torch.empty(R, dtype=torch.float32, device=dev)
    lse = torch.empty(R, dtype=torch.float32, device=dev)
    status = torch.empty(R, dtype=torch.int32, device=dev)
    ws = _workspace(workspace, head_loss_workspace(R, K, V), dev)
    N.check(N.lib().strim_head_loss(_stream_of(dev), _ptr(hidden), _row_stride(hidden), R, K,
                                    _ptr(lm_head), _row_stride(lm_head), V, _ptr(targets),
                                    ignore_index, _ptr(ws), _bytes(ws), _ptr(loss), _ptr(lse),
                                    _ptr(status)), "strim_head_loss")
    return loss, lse, status


def head_loss_grad(hidden: torch.Tensor, lm_head: torch.Tensor, targets: torch.Tensor,
                   lse: torch.Tensor, grad_loss: torch.Tensor,
                   grad_lse: torch.Tensor | None = None, want_hidden: bool = True,
                   want_lm_head: bool = True, ignore_index: int = -100,
                   workspace: torch.Tensor | None = None, stream=None):
    """Gradients of head_loss: (d_hidden bf16 [N, K] or None, d_lm_head bf16 [V, K] or None)
    from lse as head_loss gave it and the float32 [N] gradients of its loss and (optional)
    its lse."""
    R, K, V = _loss_args(hidden, lm_head, targets, ignore_index)
    dev = hidden.device
    _check_with(dev, lse, grad_loss, grad_lse)
    for t in (lse, grad_loss, grad_lse):
        if t is not None and (t.dtype != torch.float32 or t.shape != (R,)):
            raise ValueError(f"lse and the gradients must be float32 [{R}]")
    if not (want_hidden or want_lm_head):
        return None, None
    if _elsewhere(stream, dev):
        return _there(head_loss_grad, stream, dev, hidden, lm_head, targets, lse, grad_loss, grad_lse,
                      want_hidden, want_lm_head, ignore_index, workspace)
    dh = torch.empty(R, K, dtype=torch.bfloat16, device=dev) if want_hidden else None
    dw = torch.empty(V, K, dtype=torch.bfloat16, device=dev) if want_lm_head else None
    ws = _workspace(workspace, head_loss_workspace(R, K, V, want_hidden, want_lm_head), dev)
    N.check(N.lib().strim_head_loss_grad(_stream_of(dev), _ptr(hidden), _row_stride(hidden), R, K,
                                         _ptr(lm_head), _row_stride(lm_head), V, _ptr(targets),
                                         ignore_index, _ptr(lse), _ptr(grad_loss), _ptr(grad_lse),
                                         _ptr(ws), _bytes(ws), _ptr(dh), K, _ptr(dw), K),
            "strim_head_loss_grad")
    return dh, dw


class Q4Weight:
    """A projection [V, K] in 4 bits: words int32 [V, K / 8] (eight codes a word, the lowest
    bits first), scales bf16 [V, K / group], biases alike or None (symmetric); the element is
    scale q + bias, or scale (q - 8). The layout of the reference's 4-bit groupwise weights
    (QGEMV.swift:14-15,68-69)."""

    def __init__(self, words: torch.Tensor, scales: torch.Tensor,
                 biases: torch.Tensor | None = None, group: int = 64):
        if words.dtype != torch.int32 or words.dim() != 2:
            raise ValueError("words must be int32 [V, K / 8]")
        if not words.is_cuda:
            raise ValueError("every tensor argument must be on the GPU")
        V, W = words.shape
        if group not in (32, 64, 128) or 8 * W % group:
            raise ValueError(f"group must be 32, 64 or 128 and divide K={8 * W}, got {group}")
        for t in (scales, biases):
            if t is not None and (t.dtype != torch.bfloat16 or t.shape != (V, 8 * W // group)):
                raise ValueError(f"scales and biases must be bfloat16 [{V}, {8 * W // group}]")
        _check_with(words.device, words, scales, biases)
        self.words, self.scales, self.biases, self.group = words, scales, biases, group
        self.V, self.K = V, 8 * W


def q4_pack(weight: torch.Tensor, group: int = 64, symmetric: bool = False,
            stream=None) -> Q4Weight:
    """weight [V, K] (bf16 or float32) in 4 bits with a scale (and, unless symmetric, a bias)
    for every `group` elements of a row."""
    code = _dtype_code(weight)
    _check_rows(weight)
    V, K = weight.shape
    if group not in (32, 64, 128) or K % group:
        raise ValueError(f"group must be 32, 64 or 128 and divide K={K}, got {group}")
    dev = weight.device
    if _elsewhere(stream, dev):
        return _there(q4_pack, stream, dev, weight, group, symmetric)
    words = torch.empty(V, K // 8, dtype=torch.int32, device=dev)
    scales = torch.empty(V, K // group, dtype=torch.bfloat16, device=dev)
    biases = None if symmetric else torch.empty_like(scales)
    N.check(N.lib().strim_pack_weights(_stream_of(dev), _ptr(weight), code, _row_stride(weight), V,
                                       K, group, _ptr(words), _ptr(scales), _ptr(biases)),
            "strim_pack_weights")
    return Q4Weight(words, scales, biases, group)


def q4_unpack(q: Q4Weight, dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """The values [V, K] that a packed projection stands for, as bf16 or float32."""
    dev = q.words.device
    if _elsewhere(stream, dev):
        return _there(q4_unpack, stream, dev, q, dtype)
    out = torch.empty(q.V, q.K, dtype=dtype, device=dev)
    N.check(N.lib().strim_unpack_weights(_stream_of(dev), _ptr(q.words), q.K // 8, _ptr(q.scales),
                                         _ptr(q.biases), q.K // q.group, q.V, q.K, q.group,
                                         _ptr(out), _dtype_code(out), q.K),
            "strim_unpack_weights")
    return out


def head_logits_q4(hidden: torch.Tensor, q: Q4Weight, norm_weight: torch.Tensor | None = None,
                   eps: float = 1e-6, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.bfloat16, xn: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """head_logits over a projection held in 4 bits: logits [B, V] in bf16 or float32 (or
    `out`), the layout sample / verify take. Any number of rows."""
    if hidden.dim() == 1:
        hidden = hidden.unsqueeze(0)
    _check_bf16_rows("hidden", hidden)
    dev = q.words.device
    _check_with(dev, norm_weight, out, xn)
    B, K = hidden.shape
    if hidden.device != dev:
        raise ValueError("every tensor argument must be on the same GPU")
    if K != q.K:
        raise ValueError(f"the projection has K={q.K}, hidden K={K}")
    if _elsewhere(stream, dev):
        return _there(head_logits_q4, stream, dev, hidden, q, norm_weight, eps, out, out_dtype, xn, workspace)
    if norm_weight is not None:
        if norm_weight.dtype != torch.bfloat16 or norm_weight.shape != (K,):
            raise ValueError(f"norm_weight must be bfloat16 [{K}]")
        if xn is None:
            xn = torch.empty(B, K, dtype=torch.bfloat16, device=dev)
        elif xn.dtype != torch.bfloat16 or xn.shape != (B, K):
            raise ValueError(f"xn must be bfloat16 [{B}, {K}]")
    if out is None:
        out = torch.empty(B, q.V, dtype=out_dtype, device=dev)
    elif out.shape != (B, q.V):
        raise ValueError(f"out must be [{B}, {q.V}]")
    ws = _workspace(workspace, head_logits_q4_workspace(B, K), dev)
    N.check(N.lib().strim_head_logits_packed(
        _stream_of(dev), _ptr(hidden), _row_stride(hidden), B, K, _ptr(norm_weight), eps,
        _ptr(xn), _ptr(q.words), K // 8, _ptr(q.scales), _ptr(q.biases), K // q.group, q.group,
        q.V, _ptr(ws), _bytes(ws), _ptr(out), _dtype_code(out), q.V), "strim_head_logits_packed")
    return out


class TokenScores(NamedTuple):
    """What token_scores returns: log-probabilities of the given tokens (as tokens is shaped; None
    without tokens), entropy and log-sum-exp float32 [R], the alternatives' ids int32 and
    log-probabilities float32 [R, top] (None for top 0), status int32 [R]."""

    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None
    status: torch.Tensor


def _check_logits(logits: torch.Tensor, temperature: float) -> int:
    """The dtype code of logits [R, V] with contiguous rows."""
    code = _dtype_code(logits)
    if not logits.is_cuda:
        raise ValueError("logits must be on the GPU")
    if logits.dim() != 2 or (not logits.is_contiguous() and
                             (logits.stride(1) != 1 or _row_stride(logits) < logits.shape[1])):
        raise ValueError("logits must be [R, V] with contiguous rows (row stride >= V)")
    if not N.SCORE_MIN_TEMPERATURE <= temperature < float("inf"):
        raise ValueError(f"temperature must be finite and at least {N.SCORE_MIN_TEMPERATURE}, got {temperature}")
    R, V = logits.shape
    if R > N.SCORE_MAX_ROWS or not 0 < V <= N.SCORE_MAX_VOCAB:
        raise ValueError(f"logits must be at most [{N.SCORE_MAX_ROWS}, {N.SCORE_MAX_VOCAB}], got [{R}, {V}]")
    return code


def _check_list(name: str, t: torch.Tensor, dtype: torch.dtype, R: int) -> int:
    """Entries a row of a list int32 or float32 [R] or [R, S]."""
    if t.dtype != dtype or t.dim() not in (1, 2) or t.shape[0] != R:
        raise ValueError(f"{name} must be {dtype} [{R}] or [{R}, n], got {t.dtype} {tuple(t.shape)}")
    S = 1 if t.dim() == 1 else t.shape[1]
    if S > N.SCORE_MAX_LIST:
        raise ValueError(f"{name} may have {N.SCORE_MAX_LIST} entries a row, got {S}")
    return S


def _check_mask(mask: torch.Tensor | None, R: int, V: int) -> int:
    if mask is None:
        return 0
    if mask.dtype != torch.int32 or mask.dim() != 2 or mask.shape[0] != R or 32 * mask.shape[1] < V:
        raise ValueError(f"mask must be int32 words [{R}, {(V + 31) // 32}], got {mask.dtype} "
                         f"{tuple(mask.shape)}")
    return mask.shape[1]


def _logits_out(out: torch.Tensor | None, logits: torch.Tensor) -> torch.Tensor:
    """Where the gradient goes: `out` (logits itself, say), or new memory."""
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if out.dtype != logits.dtype or out.shape != logits.shape or out.device != logits.device:
        raise ValueError("out must be as the logits are")
    _check_rows(out)
    return out


@lru_cache(maxsize=256)
def token_scores_workspace(R: int, V: int, top: int) -> int:
    """Bytes of workspace that token_scores takes."""
    need = N.lib().strim_token_scores_workspace(R, V, top)
    if need < 0:
        raise N.StrimError(need, "strim_token_scores_workspace")
    return need


def token_scores(logits: torch.Tensor, tokens: torch.Tensor | None = None, top: int = 0,
                 temperature: float = 1.0, mask: torch.Tensor | None = None,
                 ignore_index: int = -100, workspace: torch.Tensor | None = None,
                 stream=None) -> TokenScores:
    """Log-probabilities of the given tokens (int32 [R] or [R, S]) under softmax(logits /
    temperature) over the ids that `mask` (int32 words as Context.sample takes them) allows, its
    entropy and log-sum-exp, and its `top` most probable ids (the lower id first where logits are
    equal; past the last one -1 and -inf). logits bf16 or float32 [R, V]. Status per row: OK, EINVAL
    (a token outside [0, V) that is not ignore_index: log-probability 0, as an ignored one's), EEMPTY
    or ENONFINITE. strim_amd.loss has the differentiable form."""
    code = _check_logits(logits, temperature)
    check_ignore_index(ignore_index)
    R, V = logits.shape
    dev = logits.device
    S = 0 if tokens is None else _check_list("tokens", tokens, torch.int32, R)
    words = _check_mask(mask, R, V)
    if not 0 <= top <= N.SCORE_MAX_LIST:
        raise ValueError(f"top must be in [0, {N.SCORE_MAX_LIST}], got {top}")
    _check_with(dev, tokens, mask)
    if _elsewhere(stream, dev):
        return _there(token_scores, stream, dev, logits, tokens, top, temperature, mask, ignore_index,
                      workspace)
    lp = None if tokens is None else torch.empty(tokens.shape, dtype=torch.float32, device=dev)
    entropy = torch.empty(R, dtype=torch.float32, device=dev)
    lse = torch.empty(R, dtype=torch.float32, device=dev)
    ids = torch.empty(R, top, dtype=torch.int32, device=dev) if top else None
    ilp = torch.empty(R, top, dtype=torch.float32, device=dev) if top else None
    status = torch.empty(R, dtype=torch.int32, device=dev)
    ws = _workspace(workspace, token_scores_workspace(R, V, top), dev)
    N.check(N.lib().strim_token_scores(_stream_of(dev), _ptr(logits), code, R, V, _row_stride(logits),
                                       temperature, _ptr(mask), words, _ptr(tokens), S, ignore_index,
                                       top, _ptr(ws), _bytes(ws), _ptr(lp), _ptr(entropy), _ptr(lse),
                                       _ptr(ids), _ptr(ilp), _ptr(status)), "strim_token_scores")
    return TokenScores(lp, entropy, lse, ids, ilp, status)


def token_scores_grad(logits: torch.Tensor, tokens: torch.Tensor | None, lse: torch.Tensor,
                      entropy: torch.Tensor | None = None, grad_logprobs: torch.Tensor | None = None,
                      grad_entropy: torch.Tensor | None = None, grad_lse: torch.Tensor | None = None,
                      temperature: float = 1.0, mask: torch.Tensor | None = None,
                      ignore_index: int = -100, out: torch.Tensor | None = None,
                      stream=None) -> torch.Tensor:
    """The logits' gradient [R, V] (of their type) from lse and entropy as token_scores gave them and
    the float32 gradients of its log-probabilities (shaped as tokens), entropy and lse; each may be
    None. out: where it goes, the logits themselves included."""
    code = _check_logits(logits, temperature)
    check_ignore_index(ignore_index)
    R, V = logits.shape
    dev = logits.device
    S = 0
    if grad_logprobs is not None:
        if tokens is None or grad_logprobs.shape != tokens.shape:
            raise ValueError("grad_logprobs must be shaped as the tokens are")
        S = _check_list("tokens", tokens, torch.int32, R)
        _check_list("grad_logprobs", grad_logprobs, torch.float32, R)
    if grad_entropy is not None and entropy is None:
        raise ValueError("grad_entropy needs the entropy")
    for t in (lse, entropy, grad_entropy, grad_lse):
        if t is not None and (t.dtype != torch.float32 or t.shape != (R,)):
            raise ValueError(f"lse, entropy and their gradients must be float32 [{R}]")
    words = _check_mask(mask, R, V)
    _check_with(dev, tokens, mask, lse, entropy, grad_logprobs, grad_entropy, grad_lse)
    if _elsewhere(stream, dev):
        return _there(token_scores_grad, stream, dev, logits, tokens, lse, entropy, grad_logprobs,
                      grad_entropy, grad_lse, temperature, mask, ignore_index, out)
    d = _logits_out(out, logits)
    N.check(N.lib().strim_token_scores_grad(
        _stream_of(dev), _ptr(logits), code, R, V, _row_stride(logits), temperature, _ptr(mask), words,
        _ptr(tokens), S, ignore_index, _ptr(lse), _ptr(entropy), _ptr(grad_logprobs), _ptr(grad_entropy),
        _ptr(grad_lse), _ptr(d), _row_stride(d)), "strim_token_scores_grad")
    return d


def _distill_args(logits, ids, logprobs, temperature):
    """Checks of the distillation calls; (dtype code, N, V, M)."""
    code = _check_logits(logits, temperature)
    R, V = logits.shape
    for t, dt, name in ((ids, torch.int32, "ids"), (logprobs, torch.float32, "logprobs")):
        if t.dtype != dt or t.dim() != 2 or t.shape[0] != R or t.shape != ids.shape:
            raise ValueError(f"{name} must be {dt} [{R}, M], got {t.dtype} {tuple(t.shape)}")
    M = ids.shape[1]
    if not 0 < M <= N.SCORE_MAX_LIST:
        raise ValueError(f"a row has 1 to {N.SCORE_MAX_LIST} alternatives, got {M}")
    _check_with(logits.device, ids, logprobs)
    return code, R, V, M


@lru_cache(maxsize=256)
def distill_workspace(rows: int, V: int, M: int, step: bool = False) -> int:
    """Bytes of workspace that distill (or distill_step) takes."""
    need = N.lib().strim_distill_workspace(rows, V, M, int(step))
    if need < 0:
        raise N.StrimError(need, "strim_distill_workspace")
    return need


def distill(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float = 1.0,
            tail: bool = False, workspace: torch.Tensor | None = None, stream=None):
    """Divergence of softmax(logits / temperature) from a teacher's alternatives: ids int32 and
    logprobs float32 [N, M] as token_scores gives them (at the same temperature), a negative id or a
    log-probability of -inf being padding. tail: the teacher's remaining mass is one more alternative,
    against the student's mass outside the ids; else the alternatives are renormalised. Returns (loss
    [N], lse [N], log_rest [N], status [N]); a row without alternatives has loss 0, one with an id of V
    or more 0 and EINVAL. strim_amd.loss has the differentiable form."""
    code, R, V, M = _distill_args(logits, ids, logprobs, temperature)
    dev = logits.device
    if _elsewhere(stream, dev):
        return _there(distill, stream, dev, logits, ids, logprobs, temperature, tail, workspace)
    loss = torch.empty(R, dtype=torch.float32, device=dev)
    lse = torch.empty(R, dtype=torch.float32, device=dev)
    rest = torch.empty(R, dtype=torch.float32, device=dev)
    status = torch.empty(R, dtype=torch.int32, device=dev)
    ws = _workspace(workspace, distill_workspace(R, V, M), dev)
    N.check(N.lib().strim_distill(_stream_of(dev), _ptr(logits), code, R, V, _row_stride(logits),
                                  temperature, _ptr(ids), _ptr(logprobs), M, int(tail), _ptr(ws),
                                  _bytes(ws), _ptr(loss), _ptr(lse), _ptr(rest), _ptr(status)),
            "strim_distill")
    return loss, lse, rest, status


def distill_grad(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, lse: torch.Tensor,
                 log_rest: torch.Tensor, grad_loss: torch.Tensor, temperature: float = 1.0,
                 tail: bool = False, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The logits' gradient [N, V] (of their type) from lse and log_rest as distill gave them and the
    float32 [N] gradient of its loss. out: where it goes, the logits themselves included. (Probabilities
    are off by the rounding of lse and log_rest, 2^-24 of either: small unless the largest logit over the
    temperature is large, or the rest is all but excluded. distill_step's are not.)"""
    code, R, V, M = _distill_args(logits, ids, logprobs, temperature)
    dev = logits.device
    for t in (lse, log_rest, grad_loss):
        if t.dtype != torch.float32 or t.shape != (R,):
            raise ValueError(f"lse, log_rest and grad_loss must be float32 [{R}]")
    _check_with(dev, lse, log_rest, grad_loss)
    if _elsewhere(stream, dev):
        return _there(distill_grad, stream, dev, logits, ids, logprobs, lse, log_rest, grad_loss,
                      temperature, tail, out)
    d = _logits_out(out, logits)
    N.check(N.lib().strim_distill_grad(_stream_of(dev), _ptr(logits), code, R, V, _row_stride(logits),
                                       temperature, _ptr(ids), _ptr(logprobs), M, int(tail), _ptr(lse),
                                       _ptr(log_rest), _ptr(grad_loss), _ptr(d), _row_stride(d)),
            "strim_distill_grad")
    return d


def distill_step(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                 weights: torch.Tensor, temperature: float = 1.0, tail: bool = False,
                 out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None):
    """distill and distill_grad in one call, for rows whose weights float32 [N] are known beforehand
    (a mean's 1 / count): (loss [N], d_logits [N, V], status [N]). What a workgroup holds of a row is
    read once; few rows over a long vocabulary are read twice."""
    code, R, V, M = _distill_args(logits, ids, logprobs, temperature)
    dev = logits.device
    if weights.dtype != torch.float32 or weights.shape != (R,):
        raise ValueError(f"weights must be float32 [{R}]")
    _check_with(dev, weights)
    if _elsewhere(stream, dev):
        return _there(distill_step, stream, dev, logits, ids, logprobs, weights, temperature, tail, out,
                      workspace)
    loss = torch.empty(R, dtype=torch.float32, device=dev)
    status = torch.empty(R, dtype=torch.int32, device=dev)
    d = _logits_out(out, logits)
    ws = _workspace(workspace, distill_workspace(R, V, M, True), dev)
    N.check(N.lib().strim_distill_step(_stream_of(dev), _ptr(logits), code, R, V, _row_stride(logits),
                                       temperature, _ptr(ids), _ptr(logprobs), M, int(tail),
                                       _ptr(weights), _ptr(ws), _bytes(ws), _ptr(loss), _ptr(d),
                                       _row_stride(d), _ptr(status)), "strim_distill_step")
    return loss, d, status


def distill_scale(data: torch.Tensor, factor: torch.Tensor, stream=None) -> torch.Tensor:
    """data *= factor (one float32 on the device), in place; nothing is written where it is 1."""
    code = _dtype_code(data)
    if factor.dtype != torch.float32 or factor.numel() != 1:
        raise ValueError("factor must be one float32 number")
    if not data.is_cuda:
        raise ValueError("every tensor argument must be on the GPU")
    _check_with(data.device, data, factor)
    if _elsewhere(stream, data.device):
        return _there(distill_scale, stream, data.device, data, factor)
    N.check(N.lib().strim_distill_scale(_stream_of(data.device), _ptr(data), code, data.numel(),
                                        _ptr(factor)), "strim_distill_scale")
    return data


def _norm_args(x, weight, bias):
    """Checks of the norm calls; (dtype code, weight dtype code, N, K)."""
    code = _dtype_code(x)
    if not x.is_cuda:
        raise ValueError("every tensor argument must be on the GPU")
    _check_norm_rows("x", x)
    R, K = x.shape
    if R > N.NORM_MAX_ROWS or not 0 < K <= N.NORM_MAX_WIDTH:
        raise ValueError(f"x must be at most [{N.NORM_MAX_ROWS}, {N.NORM_MAX_WIDTH}], got [{R}, {K}]")
    wcode = N.DTYPE_F32
    for t in (weight, bias):
        if t is None:
            continue
        wcode = _dtype_code(t)
        if t.shape != (K,):
            raise ValueError(f"weight and bias must be [{K}], got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must be of one type")
    _check_with(x.device, weight, bias)
    return code, wcode, R, K


def _check_norm_rows(name: str, t: torch.Tensor) -> None:
    if t.dim() != 2 or (not t.is_contiguous() and
                        (t.stride(1) != 1 or _row_stride(t) < t.shape[1])):
        raise ValueError(f"{name} must be [N, K] with contiguous rows (row stride >= K)")


def norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
         eps: float = 1e-6, center: bool = False, stream=None):
    """Rows of x (bf16 or float32 [N, K]) over their root mean square, or (center) less their mean over
    their standard deviation, times weight plus bias ([K], both of one type or None). Returns (y of x's
    type, rstd float32 [N], mean float32 [N] or None without center). strim_amd.norm has the
    differentiable forms."""
    code, wcode, R, K = _norm_args(x, weight, bias)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    dev = x.device
    if _elsewhere(stream, dev):
        return _there(norm, stream, dev, x, weight, bias, eps, center)
    y = torch.empty(R, K, dtype=x.dtype, device=dev)
    rstd = torch.empty(R, dtype=torch.float32, device=dev)
    mean = torch.empty(R, dtype=torch.float32, device=dev) if center else None
    N.check(N.lib().strim_norm(_stream_of(dev), _ptr(x), code, R, K, _row_stride(x), _ptr(weight),
                               _ptr(bias), wcode, eps, int(center), _ptr(y), K, _ptr(rstd), _ptr(mean)),
            "strim_norm")
    return y, rstd, mean


@lru_cache(maxsize=256)
def norm_workspace(rows: int, K: int, want_weight: bool = False, want_bias: bool = False) -> int:
    """Bytes of workspace that norm_grad takes."""
    need = N.lib().strim_norm_workspace(rows, K, int(want_weight), int(want_bias))
    if need < 0:
        raise N.StrimError(need, "strim_norm_workspace")
    return need


def norm_grad(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
              grad_y: torch.Tensor, rstd: torch.Tensor, mean: torch.Tensor | None = None,
              want_x: bool = True, want_weight: bool = True, want_bias: bool = True,
              workspace: torch.Tensor | None = None, stream=None):
    """Gradients of norm: (d_x of x's type or None, d_weight, d_bias of their types, or None where there
    is no weight, no bias, or none wanted) from rstd and mean as norm gave them and grad_y of x's type
    and shape."""
    code, wcode, R, K = _norm_args(x, weight, bias)
    dev = x.device
    if grad_y.dtype != x.dtype or grad_y.shape != x.shape or grad_y.device != dev:
        raise ValueError("grad_y must be as x is")
    _check_norm_rows("grad_y", grad_y)
    for t in (rstd, mean):
        if t is not None and (t.dtype != torch.float32 or t.shape != (R,)):
            raise ValueError(f"rstd and mean must be float32 [{R}]")
    _check_with(dev, rstd, mean)
    want_weight, want_bias = want_weight and weight is not None, want_bias and bias is not None
    if not (want_x or want_weight or want_bias):
        return None, None, None
    if _elsewhere(stream, dev):
        return _there(norm_grad, stream, dev, x, weight, bias, grad_y, rstd, mean, want_x, want_weight,
                      want_bias, workspace)
    dx = torch.empty(R, K, dtype=x.dtype, device=dev) if want_x else None
    dw = torch.empty(K, dtype=weight.dtype, device=dev) if want_weight else None
    db = torch.empty(K, dtype=bias.dtype, device=dev) if want_bias else None
    ws = _workspace(workspace, norm_workspace(R, K, want_weight, want_bias), dev)
    N.check(N.lib().strim_norm_grad(_stream_of(dev), _ptr(x), code, R, K, _row_stride(x), _ptr(grad_y),
                                    _row_stride(grad_y), _ptr(weight), wcode, _ptr(rstd), _ptr(mean),
                                    _ptr(ws), _bytes(ws), _ptr(dx), K, _ptr(dw), _ptr(db)),
            "strim_norm_grad")
    return dx, dw, db


def draft_argmax(draft_logits: torch.Tensor, draft_to_full: torch.Tensor | None = None,
                 stream=None):
    """MTP.nextTokenIndex (MTP.swift:104-111): table[argmax(draft logits)] per row."""
    if draft_logits.dim() == 1:
        draft_logits = draft_logits.unsqueeze(0)
    R, Vd = draft_logits.shape
    _check_rows(draft_logits)
    _check_cuda(draft_to_full)
    out = torch.empty(R, dtype=torch.int32, device=draft_logits.device)
    N.check(N.lib().strim_draft_argmax(_stream(stream), _ptr(draft_logits),
                                       _dtype_code(draft_logits), R, Vd, _row_stride(draft_logits),
                                       _ptr(draft_to_full), _ptr(out)), "strim_draft_argmax")
    return out


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool [..., V] -> int32 words [..., ceil(V/32)], bit (i & 31) of word (i >> 5)
    (the byte layout of the reference's UInt64 bitset, GrammarVocab.swift:77-86)."""
    V = allowed.shape[-1]
    W = (V + 31) // 32
    pad = torch.zeros(allowed.shape[:-1] + (W * 32,), dtype=torch.int64, device=allowed.device)
    pad[..., :V] = allowed.to(torch.int64)
    bits = pad.reshape(allowed.shape[:-1] + (W, 32))
    words = (bits << torch.arange(32, device=allowed.device, dtype=torch.int64)).sum(-1)
    return _to_i32(words)


def _to_i32(words: torch.Tensor) -> torch.Tensor:
    w = words & 0xFFFFFFFF
    w = torch.where(w >= (1 << 31), w - (1 << 32), w)
    return w.to(torch.int32)


class BoundCall:
    """A strim_sample call with its ctypes arguments prepared (see Context.bind_sample).
    It launches on the given stream, or on the current stream at call time (so a graph
    capture records it)."""

    def __init__(self, fn, args, keep, out_ids, out_status, stream=None, name="strim_sample"):
        self._fn = fn
        self._args = args
        self._keep = keep
        self._stream = stream
        self._name = name
        self.out_ids = out_ids
        self.out_status = out_status

    def __call__(self) -> None:
        self._args[1] = _stream(self._stream)
        rc = self._fn(*self._args)
        if rc != N.OK:
            raise N.StrimError(rc, self._name)
