"""Stand-alone ops on torch tensors: the gated delta rule (one token, ragged prompts) and filtered sampling.

Thin checked wrappers of the C ABI's dfssm_gated_delta_step, dfssm_gated_delta_prefill and
dfssm_sample_filtered (include/dfssm.h has the formulas): they take CUDA tensors, run on the tensors'
device and its current stream, neither synchronise nor keep anything between calls, record no gradients, and
raise ValueError for arguments that do not fit.  Outputs must not overlap inputs.  A gated delta state
[slots, v_heads, dv, dk] is the layout of DFSSMModel.h_states; logits come from DFSSMModel.forward or
dfssm_lm_head_argmax.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

# The handle of a device's current stream; torch.cuda.current_stream() also makes a Stream object, 2 us a call.
_stream_of = torch._C._cuda_getCurrentRawStream

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


# The checks run before every launch, which a one-token op waits for: messages are only put together on failure.


def _refuse(t, name: str, what: str, device=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device (there is no CPU fallback)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")
    raise ValueError(f"{name} must be {what}, not {t.dtype} {tuple(t.shape)} with strides {t.stride()}")


def _on(t, name: str, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or (device is not None and t.device != device):
        _refuse(t, name, "a tensor", device)


def _vector(t, name: str, n: int, dtype, device):
    """Pointer of a contiguous [n]."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and t.shape == (n,) and t.is_contiguous():
        return t.data_ptr()
    _refuse(t, name, f"a contiguous {dtype} vector of {n}", device)


def _call(index, fn, *args):
    """Runs a C entry on that device, on its current stream (the last argument)."""
    if index == torch.cuda.current_device():
        rc = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream_of(index))
    if rc:
        _lib.check(rc)


def _explain(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out):
    """Finds out what _delta's checks did not like, and says so."""
    _on(q, "q")
    dev, dtype = q.device, q.dtype
    if dtype not in (torch.float16, torch.bfloat16) or q.dim() != 3:
        _refuse(q, "q", "fp16 or bf16 [tokens, k_heads, dk]")
    if not isinstance(v, torch.Tensor) or v.dim() != 3:
        _refuse(v, "v", "[tokens, v_heads, dv]", dev)
    (n, hk, dk), (hv, dv) = q.shape, v.shape[1:]
    if (not isinstance(state, torch.Tensor) or state.dtype is not torch.float32 or state.device != dev or state.dim() != 4
            or state.shape[1:] != (hv, dv, dk) or not state.is_contiguous()):
        _refuse(state, "state", f"contiguous fp32 [slots, {hv}, {dv}, {dk}]", dev)
    for t, name, shape in ((q, "q", (n, hk, dk)), (k, "k", (n, hk, dk)), (v, "v", (n, hv, dv)), (out, "out", (n, hv, dv)),
                           (a, "a", (n, hv)), (b, "b", (n, hv))):
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != dev or t.shape != shape or _row(t) is None:
            _refuse(t, name, f"{dtype} {shape} with contiguous rows", dev)
    _vector(A_log, "A_log", hv, torch.float32, dev)
    _vector(dt_bias, "dt_bias", hv, torch.float32, dev)
    if slots is not None:
        _vector(slots, "slots", n_seq, torch.int32, dev)
    raise ValueError("arguments do not fit together")


def _row(t):
    """Row stride of [rows, heads, width] or [rows, heads] whose rows are contiguous, else None."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        n, h, d = shape
        ld, sh, sd = stride
        width, ok = h * d, (sd == 1 or d == 1) and (sh == d or h == 1)
    else:
        n, width = shape
        ld, sh = stride
        ok = sh == 1 or width == 1
    if n < 2:
        ld = width
    return ld if ok and width <= ld < 2**31 else None


def _delta(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out, scale):
    # One straight run of checks: a one-token call is over in less time than they take.
    try:
        dtype, index = q.dtype, q.get_device()
        keys, values, heads = q.shape, v.shape, a.shape
        n, hk, dk = keys
        hv, dv = values[1:]
        if out is None:
            out = torch.empty_like(v) if v.is_contiguous() else v.new_empty(values)
        f32, outputs = torch.float32, out.shape
        ok = (index >= 0 and (dtype is torch.float16 or dtype is torch.bfloat16) and k.shape == keys and outputs == values
              and values[0] == n and heads == (n, hv) and b.shape == heads and state.shape[1:] == (hv, dv, dk)
              and k.dtype is dtype and v.dtype is dtype and a.dtype is dtype and b.dtype is dtype and out.dtype is dtype
              and state.dtype is f32 and A_log.dtype is f32 and dt_bias.dtype is f32
              and A_log.shape == (hv,) and dt_bias.shape == (hv,)
              and k.get_device() == index and v.get_device() == index and a.get_device() == index
              and b.get_device() == index and state.get_device() == index and out.get_device() == index
              and A_log.get_device() == index and dt_bias.get_device() == index
              and state.is_contiguous() and A_log.is_contiguous() and dt_bias.is_contiguous())
        if slots is None:
            slot = None
        else:
            slot = slots.data_ptr()
            ok = (ok and slots.dtype is torch.int32 and slots.shape == (n_seq,) and slots.get_device() == index
                  and slots.is_contiguous())
        if ok:
            wide, deep = hk * dk, hv * dv
            lq = wide if q.is_contiguous() else _row(q)
            lk = wide if k.is_contiguous() else _row(k)
            lv = deep if v.is_contiguous() else _row(v)
            lo = deep if out.is_contiguous() else _row(out)
            la = hv if a.is_contiguous() else _row(a)
            lb = hv if b.is_contiguous() else _row(b)
            if None not in (lq, lk, lv, la, lb, lo):
                return (index, (q.data_ptr(), lq, k.data_ptr(), lk, v.data_ptr(), lv, a.data_ptr(), la, b.data_ptr(), lb,
                                A_log.data_ptr(), dt_bias.data_ptr(), state.data_ptr(), state.shape[0], slot),
                        (out.data_ptr(), lo, hk, hv, dk, dv, dk ** -0.5 if scale is None else float(scale)),
                        out, (n, hk, hv, dk, dv, _DTYPES[dtype]))
    except (AttributeError, TypeError, ValueError):  # not a tensor, or not of that rank
        pass
    _explain(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, v if out is None else out)


def gated_delta_step(q, k, v, a, b, A_log, dt_bias, state, *, slots=None, scale: Optional[float] = None,
                     qk_norm: bool = True, out=None):
    """One token of every sequence through the gated delta rule (dfssm_gated_delta_step).

    q, k [B, k_heads, dk], v [B, v_heads, dv], a, b [B, v_heads] in fp16 or bf16 (rows may be strided views,
    as slices of one projection are); A_log, dt_bias fp32 [v_heads]; state fp32 [slots, v_heads, dv, dk],
    updated in place; slots int32 [B] on the device (None: sequence i is in slot i).  scale defaults to
    dk ** -0.5.  Returns o [B, v_heads, dv] (`out` if given).  A row whose slot does not exist (-1 for the padding of a
    batch) or is taken by an earlier row is left out: its row of a new o is undefined."""
    n_seq = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    index, head, tail, out, dims = _delta(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out, scale)
    _call(index, _lib.load().dfssm_gated_delta_step, *head, n_seq, *tail, int(bool(qk_norm)), dims[-1])
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
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        _refuse(cu_seqlens, "cu_seqlens", "int32 [sequences + 1]")
    n_seq = cu_seqlens.shape[0] - 1
    cu = _vector(cu_seqlens, "cu_seqlens", n_seq + 1, torch.int32, q.device)
    index, head, tail, out, dims = _delta(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out, scale)
    lib = _lib.load()
    need = lib.dfssm_gated_delta_workspace(dims[0], n_seq, *dims[1:])
    if workspace is None:
        workspace = v.new_empty(need, dtype=torch.uint8)
    elif (not isinstance(workspace, torch.Tensor) or workspace.dtype is not torch.uint8 or workspace.get_device() != index
          or not workspace.is_contiguous() or workspace.numel() < need):
        _refuse(workspace, "workspace", f"contiguous uint8 of at least {need} bytes", q.device)
    _call(index, lib.dfssm_gated_delta_prefill, *head, cu, n_seq, dims[0], *tail, int(bool(qk_norm)), dims[-1],
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
    if logits.dtype not in _DTYPES or logits.dim() != 2 or logits.shape[1] < 1:
        _refuse(logits, "logits", "[rows, vocab] in fp32, fp16 or bf16")
    dev = logits.device
    B, V = logits.shape
    ld, step = logits.stride()
    if B < 2:
        ld = V
    if (V > 1 and step != 1) or ld < V:
        _refuse(logits, "logits", "contiguous within a row, rows apart")
    u = _vector(uniform, "uniform", B, torch.float32, dev)
    temperature = _per_row(temperature, "temperature", B, torch.float32, dev)
    top_k = _per_row(top_k, "top_k", B, torch.int32, dev)
    top_p = _per_row(top_p, "top_p", B, torch.float32, dev)
    min_p = _per_row(min_p, "min_p", B, torch.float32, dev)
    if seen_bits is not None:
        if (not isinstance(seen_bits, torch.Tensor) or seen_bits.dtype is not torch.int32 or seen_bits.device != dev
                or seen_bits.shape != (B, (V + 31) // 32) or not seen_bits.is_contiguous()):
            _refuse(seen_bits, "seen_bits", f"contiguous int32 [{B}, {(V + 31) // 32}]", dev)
    if out is None:
        out = (torch.empty_like(uniform, dtype=torch.int32), torch.empty_like(uniform, dtype=torch.int32), torch.empty_like(uniform))
        tp, kp, pp = (t.data_ptr() for t in out)
    else:
        token, kept, prob = out
        tp, kp = _vector(token, "out[0]", B, torch.int32, dev), _vector(kept, "out[1]", B, torch.int32, dev)
        pp = _vector(prob, "out[2]", B, torch.float32, dev)
    _call(dev.index, _lib.load().dfssm_sample_filtered, logits.data_ptr(), ld, _DTYPES[logits.dtype], B, V,
          None if temperature is None else temperature.data_ptr(), None if top_k is None else top_k.data_ptr(),
          None if top_p is None else top_p.data_ptr(), None if min_p is None else min_p.data_ptr(),
          None if seen_bits is None else seen_bits.data_ptr(), float(rep_penalty), u, tp, kp, pp)
    return out
