"""CPU tests: what the gated delta rule and filtered sampling entry points refuse, before they touch a GPU."""
import pytest

from dfssm_b200 import _lib

P = 0x10000  # an aligned address that is never read: every call below is refused on the host
OK = dict(q=P, ld_q=128, k=P, ld_k=128, v=P, ld_v=128, a=P, ld_a=2, b=P, ld_b=2, A_log=P, dt_bias=P, state=P, n_slots=4,
          slots=None, batch=3, o=P, ld_o=128, k_heads=1, v_heads=2, dk=128, dv=64, scale=0.1, qk_norm=1, dtype=0, stream=None)
BAD = [dict(q=None), dict(k=None), dict(v=None), dict(a=None), dict(b=None), dict(A_log=None), dict(dt_bias=None),
       dict(state=None), dict(o=None), dict(dk=96), dict(dk=256, ld_q=256, ld_k=256), dict(dv=24), dict(dv=0), dict(dv=272, ld_v=544, ld_o=544),
       dict(dtype=2), dict(dtype=-1), dict(k_heads=0), dict(v_heads=0), dict(k_heads=2, v_heads=3, ld_q=256, ld_k=256, ld_v=192, ld_o=192, ld_a=3, ld_b=3),
       dict(batch=-1), dict(n_slots=0), dict(batch=5), dict(ld_q=120), dict(ld_k=64), dict(ld_v=120), dict(ld_o=64), dict(ld_a=1), dict(ld_b=1),
       dict(ld_q=132), dict(ld_o=130), dict(q=P + 2), dict(v=P + 8), dict(state=P + 4), dict(o=P + 2),
       dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("bad", BAD, ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_gated_delta_refusals(lib, bad):
    x = {**OK, **bad}
    rc = lib.dfssm_gated_delta_step(*x.values())
    assert rc in (1, 3) and lib.dfssm_last_error()
    order = list(x)
    at = order.index("batch")
    vals = [x[n] for n in order]
    tail = vals[at + 1:-1] + [P, 1 << 40, None]
    assert lib.dfssm_gated_delta_prefill(*vals[:at], P, x["batch"], 10, *tail) in (1, 3)


def test_prefill_refusals(lib):
    x = list(OK.values())
    at = list(OK).index("batch")
    head, tail = x[:at], x[at + 1:-1]
    call = lambda cu, n, t, w, nb: lib.dfssm_gated_delta_prefill(*head, cu, n, t, *tail, w, nb, None)  # noqa: E731
    assert call(None, 3, 10, P, 1 << 40) == 1
    assert call(P, -1, 10, P, 1 << 40) == 1
    assert call(P, 3, -1, P, 1 << 40) == 1
    need = lib.dfssm_gated_delta_workspace(100000, 3, 1, 2, 128, 64, 0)
    if need:
        assert call(P, 3, 100000, None, need) == 1 and call(P, 3, 100000, P, need - 1) == 1
        assert call(P, 3, 100000, P + 64, need) == 1
    assert call(P, 0, 10, P, 1 << 40) == 0 and call(P, 3, 0, P, 1 << 40) == 0  # nothing to do: no launch
    assert lib.dfssm_gated_delta_workspace(-1, 3, 1, 2, 128, 64, 0) == 0


def test_sample_filtered_refusals(lib):
    ok = dict(logits=P, ld=1000, dtype=2, batch=2, vocab=1000, t=None, k=None, p=None, m=None, seen=None, rep=1.0, u=P, next=P,
              kept=None, prob=None, stream=None)
    call = lambda **kw: lib.dfssm_sample_filtered(*{**ok, **kw}.values())  # noqa: E731
    for bad in (dict(logits=None), dict(u=None), dict(next=None), dict(dtype=3), dict(batch=-1), dict(vocab=0), dict(ld=999),
                dict(vocab=(1 << 24) + 1, ld=1 << 25), dict(seen=P, rep=0.0), dict(seen=P, rep=float("nan"))):
        assert call(**bad) in (1, 3) and lib.dfssm_last_error(), bad
    assert call(batch=0) == 0


def test_wrappers_refuse_what_they_cannot_run():
    torch = pytest.importorskip("torch")
    from dfssm_b200 import ops
    x = torch.zeros(2, 1, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_delta_step(x, x, x, x[:, :, 0], x[:, :, 0], torch.zeros(1), torch.zeros(1), torch.zeros(2, 1, 128, 128))
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_filtered(torch.zeros(2, 10), torch.zeros(2))
    assert ops.gated_delta_workspace(0, 0, 1, 1, 128, 64) == 0


@pytest.mark.gpu
def test_wrappers_check_shapes_types_and_devices():
    import torch
    from dfssm_b200 import ops
    mk = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    ok = dict(q=mk(3, 1, 128), k=mk(3, 1, 128), v=mk(3, 2, 64), a=mk(3, 2), b=mk(3, 2), A_log=mk(2, t=torch.float32),
              dt_bias=mk(2, t=torch.float32), state=mk(4, 2, 64, 128, t=torch.float32))
    ops.gated_delta_step(*ok.values())
    bad = [dict(q=mk(3, 1, 128, t=torch.float32)), dict(k=mk(3, 1, 128, t=torch.bfloat16)), dict(k=mk(2, 1, 128)), dict(v=mk(3, 2, 64).cpu()),
           dict(v=mk(3, 64, 2).transpose(1, 2)), dict(a=mk(3, 3)), dict(A_log=mk(2)), dict(dt_bias=mk(3, t=torch.float32)),
           dict(state=mk(4, 2, 128, 64, t=torch.float32)), dict(state=mk(4, 2, 64, 128)), dict(state=mk(4, 4, 64, 128, t=torch.float32)[:, ::2]),
           dict(q=mk(1, 1, 128).expand(3, 1, 128)), dict(state=None)]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.gated_delta_step(*{**ok, **kw}.values())
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for kw in (dict(slots=i32(0, 1)), dict(slots=torch.tensor([0, 1, 2], device="cuda")), dict(out=mk(3, 2, 32))):
        with pytest.raises(ValueError):
            ops.gated_delta_step(*ok.values(), **kw)
    for cu in (torch.tensor([0, 3], device="cuda"), i32(0, 3).cpu(), i32(), None):
        with pytest.raises(ValueError):
            ops.gated_delta_prefill(*ok.values(), cu)
    with pytest.raises(_lib.DFSSMError):  # five sequences, four slots
        ops.gated_delta_prefill(*ok.values(), i32(0, 1, 1, 2, 2, 3))
    lg, u = mk(3, 50, t=torch.float32), mk(3, t=torch.float32)
    for a, kw in (((lg[0], u), {}), ((lg, u[:2]), {}), ((lg.t(), mk(50, t=torch.float32)), {}), ((lg.double(), u), {}), ((lg, u.cpu()), {}),
                  ((lg, u), dict(top_k=mk(3, t=torch.float32))), ((lg, u), dict(top_p=mk(2, t=torch.float32))),
                  ((lg, u), dict(seen_bits=mk(3, 1, t=torch.int32)))):
        with pytest.raises(ValueError):
            ops.sample_filtered(*a, **kw)


def test_wrappers_refuse_what_is_no_tensor():
    """Wrong kinds of arguments are a ValueError that names one, wherever they stand."""
    torch = pytest.importorskip("torch")
    from dfssm_b200 import ops
    x = [torch.zeros(2, 1, 128, dtype=torch.float16)] * 3 + [torch.zeros(2, 1, dtype=torch.float16)] * 2
    x += [torch.zeros(1), torch.zeros(1), torch.zeros(2, 1, 128, 128)]
    for bad in (None, 3, "q", torch.zeros(()), torch.zeros(1, 1, 1, 1, 1)):
        for at in range(8):
            with pytest.raises(ValueError):
                ops.gated_delta_step(*x[:at], bad, *x[at + 1:])
        with pytest.raises(ValueError):
            ops.gated_delta_prefill(*x, bad)
        for kw in (dict(logits=bad, uniform=torch.zeros(2)), dict(logits=torch.zeros(2, 9), uniform=bad),
                   dict(logits=bad, uniform=torch.zeros(2), top_p=0.9)):
            with pytest.raises(ValueError):
                ops.sample_filtered(**kw)


@pytest.mark.gpu
def test_wrappers_leak_nothing_and_name_what_is_wrong():
    import gc
    import sys
    import torch
    from dfssm_b200 import ops
    mk = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    f32, i32 = torch.float32, torch.int32
    x = [mk(3, 1, 128), mk(3, 1, 128), mk(3, 2, 64), mk(3, 2), mk(3, 2), mk(2, t=f32), mk(2, t=f32), mk(4, 2, 64, 128, t=f32)]
    cu, slots = torch.tensor([0, 3], dtype=i32, device="cuda"), torch.tensor([2, 1, 0], dtype=i32, device="cuda")
    lg, u, p = mk(3, 50, t=f32), mk(3, t=f32), torch.full((3,), 0.9, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    held = [*x, cu, slots, lg, u, p, ws]

    def calls():
        out = mk(3, 2, 64)
        assert ops.gated_delta_step(*x, slots=slots, out=out) is out
        wide = mk(3, 400)
        ops.gated_delta_step(wide[:, :128].unflatten(1, (1, 128)), *x[1:], scale=0.5)
        ops.gated_delta_step(*x[:2], wide[:, 128:256].unflatten(1, (2, 64)), *x[3:])
        ops.gated_delta_prefill(*x, cu, out=out)
        ops.gated_delta_prefill(*x, cu, workspace=ws)
        ops.sample_filtered(lg, u, top_p=p, out=(mk(3, t=i32), mk(3, t=i32), mk(3, t=f32)))
        ops.sample_filtered(lg, u, temperature=0.7, top_k=5)
        for fn, a, kw, name in ((ops.gated_delta_step, x, dict(out=mk(3, 2, 32)), "out"), (ops.gated_delta_step, x, dict(slots=cu), "slots"),
                                (ops.gated_delta_prefill, (*x, slots.long()), {}, "cu_seqlens"),
                                (ops.gated_delta_prefill, (*x, cu), dict(workspace=ws[:8]), "workspace"),
                                (ops.gated_delta_step, (*x[:7], mk(4, 2, 64, 64, t=f32)), {}, "state"),
                                (ops.sample_filtered, (lg, u[:2]), {}, "uniform"), (ops.sample_filtered, (lg.t(), u), {}, "logits"),
                                (ops.sample_filtered, (lg, u), dict(min_p=slots), "min_p"), (ops.sample_filtered, (lg, u), dict(out=(u, u, u)), "out")):
            with pytest.raises(ValueError, match=name):
                fn(*a, **kw)

    calls()
    gc.collect()
    torch.cuda.synchronize()
    before, memory = [sys.getrefcount(t) for t in held], torch.cuda.memory_allocated()
    for _ in range(20):
        calls()
    gc.collect()
    assert [sys.getrefcount(t) for t in held] == before and torch.cuda.memory_allocated() == memory


@pytest.mark.gpu
def test_tensors_on_another_device_than_the_current_one():
    """The host path steps aside when another device is current; here it is told so once, with the one device there is."""
    import torch
    from dfssm_b200 import ops
    g = torch.Generator("cuda").manual_seed(3)
    x = [torch.randn(*s, device="cuda", generator=g).half() for s in ((3, 1, 64), (3, 1, 64), (3, 2, 32), (3, 2), (3, 2))]
    x += [torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")]
    lg, u, cu = torch.randn(3, 99, device="cuda", generator=g), torch.rand(3, device="cuda", generator=g), torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    calls = (lambda s: ops.gated_delta_step(*x, s), lambda s: ops.gated_delta_prefill(*x, s, cu), lambda s: ops.sample_filtered(lg, u, top_p=0.9)[0])
    state = lambda: torch.ones(3, 2, 32, 64, device="cuda")  # noqa: E731
    want = [f(state()) for f in calls]
    native = _lib.pycalls()
    at = [getattr(_lib.load(), "dfssm_" + n) for n in ("gated_delta_step", "gated_delta_workspace", "gated_delta_prefill", "sample_filtered")]
    asked = []

    def current():
        asked.append(1)
        return 7 if len(asked) % 2 else torch.cuda.current_device()

    import ctypes
    try:
        native.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in at), torch.Tensor, torch.float16, torch.bfloat16, torch.float32, torch.int32,
                    torch.uint8, torch.empty_like, torch._C._cuda_getCurrentRawStream, current)
        got = [f(state()) for f in calls]
    finally:
        _lib._pycalls = None
        _lib.pycalls()
    assert len(asked) == 6 and all(torch.equal(a, b) for a, b in zip(got, want))
