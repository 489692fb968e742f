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

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _run(name: str, anchor, args, explain):
    """One call of the native host path (csrc/pycalls.cpp), which looks at the arguments, allocates and launches: a
    one-token op is over in less time than checks in Python take.  `explain` says what it did not like."""
    native = getattr(_lib.pycalls(), name)
    result = native(*args)
    if result is NotImplemented:  # the tensors are on another device than the current one
        with torch.cuda.device(anchor.device):
            result = native(*args)
    if result is None:
        explain()
        raise ValueError("arguments do not fit together")
    if type(result) is int:
        _lib.check(result)
    return result


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
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != (n,)
            or not t.is_contiguous()):
        _refuse(t, name, f"a contiguous {dtype} vector of {n}", device)


def _rows_fit(t, most: int) -> bool:
    """Whether [rows, heads, width] or [rows, heads] has contiguous rows that do not overlap and start at most `most` elements
    apart."""
    if t.is_contiguous():
        return True
    width = t[0].numel() if t.shape[0] else 0
    return t[:1].is_contiguous() and (t.shape[0] < 2 or width <= t.stride(0) <= most)


def _explain(q, k, v, a, b, A_log, dt_bias, state, n_seq, slots, out):
    """Finds out which argument of a gated delta op does not fit, and says so."""
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
        if t is None and name == "out":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != dev or t.shape != shape or not _rows_fit(t, 2 ** 31 - 1):
            _refuse(t, name, f"{dtype} {shape} with contiguous rows, less than 2^31 elements apart", dev)
    _vector(A_log, "A_log", hv, torch.float32, dev)
    _vector(dt_bias, "dt_bias", hv, torch.float32, dev)
    if slots is not None:
        _vector(slots, "slots", n_seq, torch.int32, dev)


def gated_delta_step(q, k, v, a, b, A_log, dt_bias, state, *, slots=None, scale: Optional[float] = None,
                     qk_norm: bool = True, out=None):
    """One token of every sequence through the gated delta rule (dfssm_gated_delta_step).

    q, k [B, k_heads, dk], v [B, v_heads, dv], a, b [B, v_heads] in fp16 or bf16 (rows may be strided views,
    as slices of one projection are); A_log, dt_bias fp32 [v_heads]; state fp32 [slots, v_heads, dv, dk],
    updated in place; slots int32 [B] on the device (None: sequence i is in slot i).  scale defaults to
    dk ** -0.5.  Returns o [B, v_heads, dv] (`out` if given).  A row whose slot does not exist (-1 for the padding of a
    batch) or is taken by an earlier row is left out: its row of a new o is undefined."""
    x = (q, k, v, a, b, A_log, dt_bias, state)
    return _run("gated_delta_step", q, (*x, slots, scale, qk_norm, out),
                lambda: _explain(*x, q.shape[0] if isinstance(q, torch.Tensor) and q.dim() else 0, slots, out))


def gated_delta_workspace(tokens: int, n_seq: int, k_heads: int, v_heads: int, dk: int, dv: int,
                          dtype=torch.float16) -> int:
    """Bytes of scratch that gated_delta_prefill uses for these sizes; never less for more tokens or sequences, so that a
    workspace of the largest call's size serves every one."""
    return _lib.load().dfssm_gated_delta_workspace(tokens, n_seq, k_heads, v_heads, dk, dv, _DTYPES[dtype])


def gated_delta_prefill(q, k, v, a, b, A_log, dt_bias, state, cu_seqlens, *, slots=None, scale: Optional[float] = None,
                        qk_norm: bool = True, out=None, workspace=None):
    """Ragged prompts through the gated delta rule (dfssm_gated_delta_prefill): sequence i owns the rows
    cu_seqlens[i] .. cu_seqlens[i + 1] (int32 [n_seq + 1] on the device) of q, k, v, a, b and of the returned
    o, starts from its slot's state and leaves its final state there.  The other arguments are those of
    gated_delta_step.  `workspace`: a uint8 tensor of gated_delta_workspace() bytes for a caller that keeps
    one; else it comes from torch's allocator for the length of the call.  Rows of a new o that no sequence
    owns are undefined."""
    x = (q, k, v, a, b, A_log, dt_bias, state)

    def explain():
        _on(q, "q")
        if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            _refuse(cu_seqlens, "cu_seqlens", "int32 [sequences + 1]")
        n_seq = cu_seqlens.shape[0] - 1
        _vector(cu_seqlens, "cu_seqlens", n_seq + 1, torch.int32, q.device)
        _explain(*x, n_seq, slots, out)
        need = gated_delta_workspace(q.shape[0], n_seq, q.shape[1], v.shape[1], q.shape[2], v.shape[2], q.dtype)
        if workspace is not None:
            _refuse(workspace, "workspace", f"contiguous uint8 of at least {need} bytes", q.device)

    return _run("gated_delta_prefill", q, (*x, cu_seqlens, slots, scale, qk_norm, out, workspace), explain)


def sample_filtered(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None, seen_bits=None,
                    rep_penalty: float = 1.0, out=None):
    """The next token of every row of logits [B, vocab] (fp32, fp16 or bf16) from uniform fp32 [B]
    (dfssm_sample_filtered): temperature, then the first top_k tokens, then the top_p nucleus of these, then
    min_p, then the draw in vocabulary order.  temperature, top_p, min_p (fp32) and top_k (int32) are each
    None, one number, or a device tensor [B]; temperature <= 0 takes the most likely token.  seen_bits int32
    [B, ceil(vocab / 32)] and rep_penalty as in dfssm_sample.  Returns (tokens int32 [B], kept int32 [B],
    prob fp32 [B]): the token, how many tokens the filters kept, and the token's share of their weight;
    -1, 0, 0 for a row without a finite logit.  `out`: that triple to write into."""
    if temperature is None or top_k is None or top_p is None or min_p is None or not (
            type(temperature) is type(top_k) is type(top_p) is type(min_p) is torch.Tensor):
        _on(logits, "logits")
        if logits.dim() != 2:
            _refuse(logits, "logits", "[rows, vocab] in fp32, fp16 or bf16")
        of_rows = lambda x, dtype: (x if x is None or isinstance(x, torch.Tensor) else  # noqa: E731
                                    torch.full((logits.shape[0],), x, dtype=dtype, device=logits.device))
        temperature, top_k = of_rows(temperature, torch.float32), of_rows(top_k, torch.int32)
        top_p, min_p = of_rows(top_p, torch.float32), of_rows(min_p, torch.float32)

    try:
        triple = None if out is None else tuple(out)
    except TypeError:
        triple = ()

    def explain():
        _on(logits, "logits")
        if logits.dtype not in _DTYPES or logits.dim() != 2 or logits.shape[1] < 1:
            _refuse(logits, "logits", "[rows, vocab] in fp32, fp16 or bf16")
        dev, (B, V) = logits.device, logits.shape
        if not _rows_fit(logits, 2 ** 63 - 1):
            _refuse(logits, "logits", "contiguous within a row, rows apart")
        _vector(uniform, "uniform", B, torch.float32, dev)
        for t, name, dtype in ((temperature, "temperature", torch.float32), (top_k, "top_k", torch.int32),
                               (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32)):
            if t is not None:
                _vector(t, name, B, dtype, dev)
        words = (V + 31) // 32
        if seen_bits is not None and (not isinstance(seen_bits, torch.Tensor) or seen_bits.dtype is not torch.int32
                                      or seen_bits.device != dev or seen_bits.shape != (B, words) or not seen_bits.is_contiguous()):
            _refuse(seen_bits, "seen_bits", f"contiguous int32 [{B}, {words}]", dev)
        if out is not None:
            if len(triple) != 3:
                raise ValueError("out must be three tensors: tokens, kept counts and probabilities")
            token, kept, prob = triple
            _vector(token, "out[0]", B, torch.int32, dev)
            _vector(kept, "out[1]", B, torch.int32, dev)
            _vector(prob, "out[2]", B, torch.float32, dev)

    return _run("sample_filtered", logits, (logits, uniform, temperature, top_k, top_p, min_p, seen_bits, rep_penalty,
                                            triple), explain)
