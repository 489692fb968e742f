"""Stand-alone ops on torch tensors: the gated delta rule (one token, ragged prompts) and filtered sampling.

Thin checked wrappers of the C ABI's dfssm_gated_delta_step, dfssm_gated_delta_prefill and
dfssm_sample_filtered (include/dfssm.h has the formulas): they take CUDA tensors, run on the tensors'
device and its current stream, neither synchronise nor keep anything between calls, and raise ValueError
for arguments that do not fit.  A gated delta state [slots, v_heads, dv, dk] is the layout of
DFSSMModel.h_states; logits come from DFSSMModel.forward or dfssm_lm_head_argmax.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _need(ok, what: str):
    if not ok:
        raise ValueError(what)


def _on(t, name: str, device=None):
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.is_cuda, f"{name} must be on a CUDA device (there is no CPU fallback)")
    _need(device is None or t.device == device, f"{name} is on {t.device}, not {device}")


def _vector(t, name: str, n: int, dtype, device):
    _on(t, name, device)
    _need(t.dtype == dtype and t.dim() == 1 and t.shape[0] == n and (n < 2 or t.stride(0) == 1),
          f"{name} must be a contiguous {dtype} tensor of {n} elements")
    return t.data_ptr()


def _rows(t, name: str, n: int, inner, dtype, device):
    """Pointer and row stride of [n, *inner] whose rows are contiguous."""
    _on(t, name, device)
    _need(t.dtype == dtype and tuple(t.shape) == (n, *inner),
          f"{name} must be a {dtype} tensor of shape {(n, *inner)}, not {t.dtype} {tuple(t.shape)}")
    width = 1
    for d, s in zip(reversed(inner), reversed(t.stride()[1:])):
        _need(d == 1 or s == width, f"{name} must be contiguous within a row")
        width *= d
    ld = t.stride(0) if n > 1 else width
    _need(width <= ld < 2**31, f"{name}: row stride {ld} of rows of {width}")
    return t.data_ptr(), ld


def _call(device, fn, *args):
    """Runs a C entry on `device`, on its current stream (the last argument)."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))


def _delta(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out, scale):
    _on(q, "q")
    dev, dtype = q.device, q.dtype
    _need(dtype in (torch.float16, torch.bfloat16), f"q must be fp16 or bf16, not {dtype}")
    _need(q.dim() == 3 and isinstance(v, torch.Tensor) and v.dim() == 3, "q and v must be [tokens, heads, width]")
    n, hk, dk = q.shape
    hv, dv = v.shape[1], v.shape[2]
    _on(state, "state", dev)
    _need(state.dtype == torch.float32 and state.dim() == 4 and tuple(state.shape[1:]) == (hv, dv, dk) and
          state.is_contiguous(), f"state must be contiguous fp32 [slots, {hv}, {dv}, {dk}]")
    qp = _rows(q, "q", n, (hk, dk), dtype, dev)
    kp = _rows(k, "k", n, (hk, dk), dtype, dev)
    vp = _rows(v, "v", n, (hv, dv), dtype, dev)
    ap = _rows(a, "a", n, (hv,), dtype, dev)
    bp = _rows(b, "b", n, (hv,), dtype, dev)
    if out is None:
        out = torch.empty(n, hv, dv, dtype=dtype, device=dev)
    op = _rows(out, "out", n, (hv, dv), dtype, dev)
    al, db = _vector(A_log, "A_log", hv, torch.float32, dev), _vector(dt_bias, "dt_bias", hv, torch.float32, dev)
    sl = None if slots is None else _vector(slots, "slots", n_seq, torch.int32, dev)
    head = (*qp, *kp, *vp, *ap, *bp, al, db, state.data_ptr(), state.shape[0], sl)
    tail = (*op, hk, hv, dk, dv, dk ** -0.5 if scale is None else float(scale))
    return dev, head, tail, out, (n, hk, hv, dk, dv, _DTYPES[dtype])


def gated_delta_step(q, k, v, a, b, A_log, dt_bias, state, *, slots=None, scale: Optional[float] = None,
                     qk_norm: bool = True, out=None):
    """One token of every sequence through the gated delta rule (dfssm_gated_delta_step).

    q, k [B, k_heads, dk], v [B, v_heads, dv], a, b [B, v_heads] in fp16 or bf16 (rows may be strided views,
    as slices of one projection are); A_log, dt_bias fp32 [v_heads]; state fp32 [slots, v_heads, dv, dk],
    updated in place; slots int32 [B] on the device (None: sequence i is in slot i).  scale defaults to
    dk ** -0.5.  Returns o [B, v_heads, dv] (`out` if given)."""
    n_seq = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    dev, head, tail, out, dims = _delta(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out, scale)
    _call(dev, _lib.load().dfssm_gated_delta_step, *head, n_seq, *tail, int(bool(qk_norm)), dims[-1])
    return out


def gated_delta_workspace(tokens: int, n_seq: int, k_heads: int, v_heads: int, dk: int, dv: int,
                          dtype=torch.float16) -> int:
    """Bytes of scratch that gated_delta_prefill uses for these sizes."""
    return _lib.load().dfssm_gated_delta_workspace(tokens, n_seq, k_heads, v_heads, dk, dv, _DTYPES[dtype])


def gated_delta_prefill(q, k, v, a, b, A_log, dt_bias, state, cu_seqlens, *, slots=None, scale: Optional[float] = None,
                        qk_norm: bool = True, out=None, workspace=None):
    """Ragged prompts through the gated delta rule (dfssm_gated_delta_prefill): sequence i owns the rows
    cu_seqlens[i] .. cu_seqlens[i + 1] (int32 [n_seq + 1] on the device) of q, k, v, a, b and of the returned
    o, starts from its slot's state and leaves its final state there.  The other arguments are those of
    gated_delta_step.  `workspace`: a uint8 tensor of gated_delta_workspace() bytes for a caller that keeps
    one; else it comes from torch's allocator for the length of the call.  Rows of a new o that no sequence
    owns are undefined."""
    _on(q, "q")
    _need(isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1,
          "cu_seqlens must hold one offset more than there are sequences")
    n_seq = cu_seqlens.shape[0] - 1
    cu = _vector(cu_seqlens, "cu_seqlens", n_seq + 1, torch.int32, q.device)
    dev, head, tail, out, dims = _delta(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out, scale)
    lib = _lib.load()
    need = lib.dfssm_gated_delta_workspace(dims[0], n_seq, *dims[1:])
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    _on(workspace, "workspace", dev)
    _need(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need,
          f"workspace must be a contiguous uint8 tensor of at least {need} bytes")
    _call(dev, lib.dfssm_gated_delta_prefill, *head, cu, n_seq, dims[0], *tail, int(bool(qk_norm)), dims[-1],
          workspace.data_ptr(), workspace.numel())
    return out


def _per_row(x, name: str, rows: int, dtype, device):
    """A per-row setting as a device vector: None, a number for all rows, or a tensor [rows]."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor):
        x = torch.full((rows,), x, dtype=dtype, device=device)
    _vector(x, name, rows, dtype, device)
    return x


def sample_filtered(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None, seen_bits=None,
                    rep_penalty: float = 1.0, out=None):
    """The next token of every row of logits [B, vocab] (fp32, fp16 or bf16) from uniform fp32 [B]
    (dfssm_sample_filtered): temperature, then the first top_k tokens, then the top_p nucleus of these, then
    min_p, then the draw in vocabulary order.  temperature, top_p, min_p (fp32) and top_k (int32) are each
    None, one number, or a device tensor [B]; temperature <= 0 takes the most likely token.  seen_bits int32
    [B, ceil(vocab / 32)] and rep_penalty as in dfssm_sample.  Returns (tokens int32 [B], kept int32 [B],
    prob fp32 [B]): the token, how many tokens the filters kept, and the token's share of their weight;
    -1, 0, 0 for a row without a finite logit.  `out`: that triple to write into."""
    _on(logits, "logits")
    _need(logits.dtype in _DTYPES and logits.dim() == 2 and logits.shape[1] > 0, "logits must be [rows, vocab] in fp32, fp16 or bf16")
    dev = logits.device
    B, V = logits.shape
    _need(V == 1 or logits.stride(1) == 1, "logits must be contiguous within a row")
    ld = logits.stride(0) if B > 1 else V
    _need(ld >= V, "the rows of logits overlap")
    u = _vector(uniform, "uniform", B, torch.float32, dev)
    temperature = _per_row(temperature, "temperature", B, torch.float32, dev)
    top_k = _per_row(top_k, "top_k", B, torch.int32, dev)
    top_p = _per_row(top_p, "top_p", B, torch.float32, dev)
    min_p = _per_row(min_p, "min_p", B, torch.float32, dev)
    if seen_bits is not None:
        _on(seen_bits, "seen_bits", dev)
        _need(seen_bits.dtype == torch.int32 and tuple(seen_bits.shape) == (B, (V + 31) // 32) and seen_bits.is_contiguous(),
              f"seen_bits must be contiguous int32 [{B}, {(V + 31) // 32}]")
    if out is None:
        out = (torch.empty(B, dtype=torch.int32, device=dev), torch.empty(B, dtype=torch.int32, device=dev),
               torch.empty(B, dtype=torch.float32, device=dev))
    token, kept, prob = out
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _call(dev, _lib.load().dfssm_sample_filtered, logits.data_ptr(), ld, _DTYPES[logits.dtype], B, V, ptr(temperature),
          ptr(top_k), ptr(top_p), ptr(min_p), ptr(seen_bits), float(rep_penalty), u,
          _vector(token, "out[0]", B, torch.int32, dev), _vector(kept, "out[1]", B, torch.int32, dev),
          _vector(prob, "out[2]", B, torch.float32, dev))
    return out
