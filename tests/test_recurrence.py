"""Gated linear recurrence: the HIP kernels against the float64 oracle, element by element within running error bounds
(oracle/sequence_oracle.py), and what the entry points refuse."""
import os

import numpy as np
import pytest
import torch

from oracle import megacrn_oracle as MO
from oracle import sequence_oracle as O

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# without a GPU
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["tanh", "none"])
@pytest.mark.parametrize("G", [6, 2, 1])
def test_oracle_gradient_matches_differences(act, G):
    """The oracle's gradients against central differences in float64: truncation h^2 and cancellation 1e-16 / h at h = 1e-5 leave
    1e-9 of values around 1."""
    rng = np.random.default_rng(0)
    B, T, N, H = 2, 5, 3, 6
    gate, cand, state = rng.normal(1, 1, (B, T, N, G)), rng.normal(0, 1, (B, T, N, H)), rng.normal(0, 1, (B, N, H))
    mask = rng.random((B, T, N)) > 0.3
    mask[0, :, 1] = False
    dout, dlast = rng.normal(0, 1, (B, T, N, H)), rng.normal(0, 1, (B, N, H))

    def loss(*a):
        out, last, _, _ = O.glr_fwd(*a, mask=mask, act=act)
        return (out * dout).sum() + (last * dlast).sum()

    got = O.glr_bwd(O.glr_fwd(gate, cand, state, mask, act)[3], dout, dlast)[:3]
    for k, x in enumerate((gate, cand, state)):
        for _ in range(6):
            d = rng.normal(0, 1, x.shape)
            args = [gate, cand, state]
            args[k] = x + 1e-5 * d
            hi = loss(*args)
            args[k] = x - 1e-5 * d
            assert abs((hi - loss(*args)) / 2e-5 - (got[k] * d).sum()) < 1e-7
    assert not got[0][0, :, 1].any() and not got[1][0, :, 1].any()


def _cpu(**over):
    a = {"gate": torch.zeros(2, 3, 4, 8), "cand": torch.zeros(2, 3, 4, 8), "state": torch.zeros(2, 4, 8), "mask": torch.ones(2, 3, 4, dtype=torch.bool)}
    a.update(over)
    return a


@pytest.mark.parametrize("over,kind", [
    (dict(gate=torch.zeros(2, 3, 4, 3)), ValueError),                      # 3 gates for 8 channels
    (dict(gate=torch.zeros(2, 3, 4, 0)), ValueError),
    (dict(gate=torch.zeros(2, 2, 4, 8)), ValueError),
    (dict(gate=torch.zeros(2, 3, 32)), ValueError),
    (dict(gate=torch.zeros(2, 3, 4, 8, dtype=torch.bfloat16)), ValueError),
    (dict(gate=torch.zeros(2, 3, 4, 8, dtype=torch.float64), cand=torch.zeros(2, 3, 4, 8, dtype=torch.float64)), TypeError),
    (dict(gate=torch.zeros(2, 3, 4, 8, dtype=torch.int32)), TypeError),
    (dict(cand=[1.0]), TypeError),
    (dict(state=torch.zeros(2, 4, 8, dtype=torch.bfloat16)), ValueError),
    (dict(state=torch.zeros(1, 4, 8)), ValueError),
    (dict(mask=torch.ones(2, 3, 4)), ValueError),                          # not bool
    (dict(mask=torch.ones(2, 4, 4, dtype=torch.bool)), ValueError),
    (dict(mask=torch.ones(3, dtype=torch.bool)), ValueError),
    (dict(activation="relu"), ValueError),
    (dict(), RuntimeError),                                                # all in order, but on the CPU
])
def test_refusals(over, kind):
    import megacrn_amd
    with pytest.raises(kind):
        megacrn_amd.gated_linear_recurrence(**_cpu(**over))


@pytest.mark.parametrize("over,kind", [
    (dict(state=None), ValueError), (dict(state=torch.zeros(8, 4, 2).permute(2, 1, 0)), ValueError), (dict(), RuntimeError)])
def test_step_refusals(over, kind):
    import megacrn_amd
    a = _cpu(gate=torch.zeros(2, 4, 8), cand=torch.zeros(2, 4, 8), mask=None)
    a.update(over)
    with pytest.raises(kind):
        megacrn_amd.gated_linear_recurrence_step(**a)


@pytest.mark.parametrize("which", ["gate", "cand", "state"])
@pytest.mark.parametrize("where", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_dual_tensors_are_refused(which, where):
    """A forward-mode tangent is not dropped: the sequence and the step raise, and the step leaves its state alone."""
    import megacrn_amd
    from torch.autograd import forward_ad
    for f, a in ((megacrn_amd.gated_linear_recurrence, _cpu(mask=None)),
                 (megacrn_amd.gated_linear_recurrence_step, dict(gate=torch.zeros(2, 4, 8), cand=torch.ones(2, 4, 8), state=torch.ones(2, 4, 8)))):
        a = {k: None if t is None else t.to(where) for k, t in a.items()}
        with forward_ad.dual_level():
            a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
            with pytest.raises(RuntimeError, match="forward gradient"):
                f(**a)
        assert f is megacrn_amd.gated_linear_recurrence or (a["state"] == 1).all()


def test_c_sizes():
    """Checkpoints: one state in fp32 before every 8th step (every 4th of up to 4 and of 9 to 12 steps) but the first, 16-bit types only; a
    workspace for long sequences with few channels."""
    import ctypes as C
    from megacrn_amd._lib import lib

    class Glr(C.Structure):                                # mcrn_glr_t
        _fields_ = [("i", C.c_int * 8), ("s", C.c_longlong * 12)]

    def ck(*a):
        f = lib.mcrn_glr_checkpoint_floats
        f.restype, f.argtypes = C.c_size_t, [C.POINTER(Glr)]
        return f(C.byref(Glr((C.c_int * 8)(*a, 1, 0))))

    def ws(*a, backward=0):
        f = lib.mcrn_glr_workspace_bytes
        f.restype, f.argtypes = C.c_size_t, [C.POINTER(Glr), C.c_int]
        return f(C.byref(Glr((C.c_int * 8)(*a, 1, 0))), backward)
    assert ck(2, 8, 3, 4, 4, 1) == 0
    assert ck(2, 9, 3, 4, 4, 1) == 48
    assert ck(2, 13, 3, 4, 4, 1) == 24
    assert ck(2, 17, 3, 4, 4, 2) == 48
    assert ck(2, 17, 3, 4, 4, 0) == 0
    assert ck(2, 0, 3, 4, 4, 1) == 0
    assert ws(1, 1, 207, 64, 64, 0, backward=1) == 0
    assert ws(1, 20000, 1, 33, 33, 0) > 0
    for bad in ((-1, 8, 3, 4, 4, 1), (2, 8, 3, 4, 3, 1), (2, 8, 3, 4, 4, 3), (2, 8, 3, 0, 1, 0)):
        assert ws(*bad) == 0


@pytest.mark.parametrize("where", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tracing_is_refused(where):
    """torch.jit.trace would record that outputs are allocated, and nothing else."""
    import warnings
    import megacrn_amd
    a = [torch.zeros(2, 3, 4, 8, device=where) for _ in range(2)]
    b = [t[:, 0].contiguous() for t in (*a, a[0])]
    for f, args in ((lambda x, y: megacrn_amd.gated_linear_recurrence(x, y)[0], a), (lambda x, y, s: megacrn_amd.gated_linear_recurrence_step(x, y, s), b)):
        with warnings.catch_warnings(), pytest.raises(RuntimeError, match="cannot be traced"):
            warnings.simplefilter("ignore")
            torch.jit.trace(f, tuple(args), check_trace=False)


@pytest.mark.gpu
def test_transforms_are_refused():
    """Tensors that stand for others (vmap, functional gradients, fake ones) have no memory that a kernel could read: an error, no numbers."""
    import megacrn_amd
    from torch._subclasses.fake_tensor import FakeTensorMode
    x = torch.zeros(2, 2, 3, 4, 8, device="cuda")
    f = megacrn_amd.gated_linear_recurrence
    with pytest.raises(Exception):
        torch.vmap(lambda t: f(t, t)[0])(x)
    with pytest.raises(Exception):
        torch.func.grad(lambda t: f(t, t)[0].sum())(x[0])
    with pytest.raises(Exception):
        torch.func.jvp(lambda t: f(t, t)[0], (x[0],), (x[0],))
    one = x[0].clone()
    with FakeTensorMode() as mode:
        t = mode.from_tensor(one)
        with pytest.raises(Exception):
            f(t, t)


def test_package_without_its_host_nodes():
    """_host.so missing: the package imports, its recurrence and optimizer say what to build."""
    import subprocess
    import sys
    code = ("import sys; sys.modules['megacrn_amd._host'] = None\n"
            "import torch, megacrn_amd\n"
            "megacrn_amd.AGCN(1, 2, 3)\n"
            "x = torch.zeros(1, 1, 1, 1)\n"
            "for f in (lambda: megacrn_amd.gated_linear_recurrence(x, x), lambda: megacrn_amd.gated_linear_recurrence_step(x[0], x[0], x[0]),\n"
            "          lambda: megacrn_amd.AdamW([x])):\n"
            "    try:\n"
            "        f()\n"
            "    except ImportError as e:\n"
            "        assert 'make -C megacrn_amd/csrc host' in str(e)\n"
            "    else:\n"
            "        raise SystemExit('no error')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_c_sizes_of_many_chunks():
    """300 sequences of 2^23 steps and one channel: chained chunks of 128 steps would be 300 x 2^16 blocks, more than a launch holds (2^24 - 1), so
    they are split (at most 256 chunks, two floats each); half as long they are chained."""
    import ctypes as C
    from megacrn_amd._lib import lib

    class Glr(C.Structure):                                # mcrn_glr_t
        _fields_ = [("i", C.c_int * 8), ("s", C.c_longlong * 12)]
    f = lib.mcrn_glr_workspace_bytes
    f.restype, f.argtypes = C.c_size_t, [C.POINTER(Glr), C.c_int]
    ws = [f(C.byref(Glr((C.c_int * 8)(300, T, 1, 1, 1, 0, 1, 0))), back) for T in (2 ** 23, 2 ** 22) for back in (0, 1)]
    assert max(ws[:2]) <= 256 * 300 * 2 * 4 + 256 and min(ws[2:]) >= 300 * 2 ** 15 * 4


# ---------------------------------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------------------------------
def _inputs(B, T, N, H, G, dt, mask, seed, state=True):
    g = torch.Generator().manual_seed(seed)
    gate = (torch.randn(B, T, N, G, generator=g) * 1.5 + 1.5).to(TORCH[dt])
    cand = torch.randn(B, T, N, H, generator=g).to(TORCH[dt])
    st = torch.randn(B, N, H, generator=g) if state else None
    keep = None
    if mask:
        keep = torch.rand(B, T, N, generator=g) > 0.25
        keep[:, :, N // 2] = False                       # a row that nothing is left of
        for bad in (float("nan"), float("inf"), torch.finfo(TORCH[dt]).min):
            hit = (torch.rand(B, T, N, generator=g) < 0.3) & ~keep
            gate[hit], cand[hit] = bad, -bad
    return gate, cand, st, keep, torch.randn(B, T, N, H, generator=g).to(TORCH[dt]), torch.randn(B, N, H, generator=g)


def _np(t):
    return None if t is None else t.double().numpy()


def _close(got, want, bound, what):
    """The bounds are relative to what the operations make of normal numbers.  Below 2^-126 an exponential, a reciprocal or a product may be
    flushed to 0 or rounded to 2^-149, and is then off by at most 2^-126 absolutely; what multiplies it afterwards (states, candidates,
    gradients and sums over the steps that it passes) stays below 2^6 in these tests: 2^-120 in all."""
    got = got.detach().cpu().double().numpy()
    assert got.shape == want.shape, what
    over = np.abs(got - want) - bound - 2.0 ** -120
    assert not (over > 0).any() and np.isfinite(got).all(), f"{what}: {(over > 0).sum()} of {over.size} beyond the bound, worst {over.max():.3g}"


def _against_oracle(gate, cand, st, keep, dout, dlast, act, dt, lay=lambda t: t.cuda(), want_grad=True):
    import megacrn_amd
    m = None if keep is None else keep.numpy()
    out, last, eh, cache = O.glr_fwd(_np(gate), _np(cand), _np(st), m, act, dt)
    leaves = [lay(t).detach().requires_grad_() if t is not None else None for t in (gate, cand, st)]
    got, glast = megacrn_amd.gated_linear_recurrence(leaves[0], leaves[1], leaves[2], None if keep is None else keep.cuda(), activation=act)
    _close(got, out, eh + O.half_step(out, dt), "out")
    e_last = eh[:, -1] if cand.shape[1] else 0 * last
    _close(glast, last, e_last + O.half_step(last, "f32"), "last")
    if not want_grad:
        return
    have = [t for t in leaves if t is not None]
    grads = torch.autograd.grad((got, glast), have, (lay(dout), dlast.cuda()))
    dg, dc, ds, eg, ec, es = O.glr_bwd(cache, _np(dout), _np(dlast))
    _close(grads[0], dg, eg + O.half_step(dg, dt), "dgate")
    _close(grads[1], dc, ec + O.half_step(dc, dt), "dcand")
    if st is not None:
        _close(grads[2], ds, es + O.half_step(ds, "f32"), "dstate")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["tanh", "none"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,N,H,G", [
    (1, 1, 1, 1, 1), (2, 1, 3, 8, 8), (1, 2, 5, 4, 1), (3, 7, 2, 12, 12), (1, 8, 3, 33, 33), (2, 9, 3, 64, 64), (1, 16, 29, 16, 4),
    (2, 17, 7, 20, 5), (1, 40, 3, 48, 1), (1, 127, 5, 64, 64), (1, 128, 2, 64, 16), (2, 129, 3, 32, 32), (1, 300, 1, 7, 7),
    (1, 257, 2, 300, 1), (1, 70, 1, 70, 1), (1, 33, 2, 70, 7), (1, 20, 1, 1100, 1),
])
def test_against_oracle(B, T, N, H, G, dt, act):
    _against_oracle(*_inputs(B, T, N, H, G, dt, True, B * 1000 + T * 10 + H), act, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,N,H,G,dt,family", [
    (1, 2100, 1, 33, 33, "f32", "split"), (2, 2051, 3, 16, 4, "bf16", "split"), (1, 4100, 2, 8, 1, "f16", "split"), (1, 1025, 1, 260, 1, "f32", "split"),
    (32, 20, 64, 63, 63, "f32", "tile"), (64, 13, 130, 63, 63, "f32", "stream"), (33, 20, 64, 65, 5, "bf16", "stream"), (64, 1, 17, 64, 64, "f16", "stream"),
    (8, 12, 100, 64, 64, "f32", "stream"), (8, 14, 100, 64, 64, "f32", "tile"), (1, 500, 30, 64, 64, "f32", "split"), (8, 150, 100, 64, 1, "bf16", "chain"), (16, 200, 64, 64, 64, "f32", "chain"),
    (16, 200, 104, 64, 1, "bf16", "tile"), (17, 99, 100, 64, 64, "f32", "tile"),
    (8, 120, 100, 64, 16, "f16", "tile"), (2, 1000, 300, 63, 63, "f32", "chain"), (1, 1280, 300, 65, 13, "bf16", "chain"),
])
def test_every_variant(B, T, N, H, G, dt, family):
    """The plans' variants by name: one thread walks all steps, segments of a block, chunks of several blocks."""
    from megacrn_amd import _lib
    _lib.launch_histogram(reset=True)
    _against_oracle(*_inputs(B, T, N, H, G, dt, T % 2 == 1, T + H, state=T % 3 != 0), "tanh", dt)
    seen = {k for k, v in _lib.launch_histogram().items() if k.startswith("glr:") and v}
    assert seen == {f"glr:fwd_{family}", f"glr:bwd_{family}"}, seen


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,N,H", [(1, 1, 2, 3), (2, 5, 2, 3), (2, 40, 1, 5), (3, 9, 7, 37), (1, 17, 1, 6), (1, 300, 5, 42), (2, 2100, 3, 9), (2, 260, 150, 33), (1, 700, 130, 106)])
def test_vectors_over_the_ends_of_nodes(B, T, N, H, dt):
    """Channels that 4 does not divide: four neighbours may belong to two nodes, whose masks differ."""
    _against_oracle(*_inputs(B, T, N, H, H, dt, True, B + T + H), "tanh", dt)


@pytest.mark.gpu
def test_vectors_over_the_ends_of_nodes_past_the_caches():
    import megacrn_amd
    T, N, H = 4200, 484, 33
    g = torch.Generator(device="cuda").manual_seed(1)
    gate, cand = (torch.randn(1, T, N, H, generator=g, device="cuda") for _ in range(2))
    keep = torch.rand(1, T, N, generator=g, device="cuda") > 0.2
    out, last = megacrn_amd.gated_linear_recurrence(gate, cand, None, keep)
    pick = [0, 1, 241, N - 1]
    want, wlast, eh, _ = O.glr_fwd(*(t[:, :, pick].double().cpu().numpy() for t in (gate, cand)), None, keep[:, :, pick].cpu().numpy())
    _close(out[:, :, pick], want, eh + O.half_step(want, "f32"), "out")
    _close(last[:, pick], wlast, eh[:, -1] + O.half_step(wlast, "f32"), "last")


@pytest.mark.gpu
@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("B,T,N,H,G,dt", [(4, 640, 207, 64, 64, "f32"), (4, 1300, 400, 64, 1, "bf16"), (1, 700, 3000, 33, 33, "f16"), (64, 13, 650, 64, 64, "f32")])
def test_gradients_past_the_caches(B, T, N, H, G, dt, mask):
    """Gradients that are more than 256 MB: some nodes (the channels of others do not reach them) against the oracle."""
    import megacrn_amd
    g = torch.Generator(device="cuda").manual_seed(T)
    gate, cand, dout = ((torch.randn(B, T, N, w, generator=g, device="cuda") + m).to(TORCH[dt]) for w, m in ((G, 1.5), (H, 0.0), (H, 0.0)))
    st, dlast = (torch.randn(B, N, H, generator=g, device="cuda") for _ in range(2))
    keep = torch.rand(B, T, N, generator=g, device="cuda") > 0.2 if mask else None
    leaves = [t.requires_grad_() for t in (gate, cand, st)]
    out, last = megacrn_amd.gated_linear_recurrence(*leaves, keep)
    grads = torch.autograd.grad((out, last), leaves, (dout, dlast))
    assert all(torch.isfinite(t).all() for t in grads)
    pick = [0, 1, N // 2, N - 1]
    host = [t[..., pick, :].detach().double().cpu().numpy() for t in (gate, cand, st, dout, dlast)]
    want, wlast, eh, cache = O.glr_fwd(*host[:3], None if keep is None else keep[:, :, pick].cpu().numpy(), "tanh", dt)
    dg, dc, ds, eg, ec, es = O.glr_bwd(cache, *host[3:])
    for got, w, e, t, what in ((out, want, eh, dt, "out"), (last, wlast, eh[:, -1], "f32", "last"), (grads[0], dg, eg, dt, "dgate"), (grads[1], dc, ec, dt, "dcand"),
                               (grads[2], ds, es, "f32", "dstate")):
        _close(got[..., pick, :], w, e + O.half_step(w, t), what)


@pytest.mark.gpu
def test_long_memory():
    """Gates that hardly forget (1 - a down to e^-12) over 3000 steps: 1 - a has to keep its own relative precision."""
    gate, cand, st, keep, dout, dlast = _inputs(1, 3000, 2, 12, 12, "f32", False, 5)
    gate = gate * 2 + 6
    _against_oracle(gate, cand, st, None, dout, dlast, "tanh", "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("G", [12, 3, 1])
@pytest.mark.parametrize("B,T,N", [(2, 1, 3), (1, 3, 2), (1, 8, 2), (2, 40, 3), (1, 130, 3), (1, 2100, 1), (4, 200, 130)])
def test_closed_gates_keep_their_share(B, T, N, G):
    """Gates of -25 .. -4 among open ones, states of 1e6: a = sigmoid(gate) has to keep its own relative precision (1 - a rounds to 1 below -17), in
    outputs, state gradients and gradients that cross a reset."""
    gate, cand, st, _, dout, dlast = _inputs(B, T, N, 12, G, "f32", False, T + G)
    g = torch.Generator().manual_seed(T)
    closed = torch.rand(gate.shape, generator=g) < (1.0 if T < 4 else 0.3)
    gate = torch.where(closed, -4 - 21 * torch.rand(gate.shape, generator=g), gate)
    _against_oracle(gate, cand, st * 1e6, None, dout, dlast, "tanh", "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,T,N,G", [(2, 1, 3, 12), (1, 8, 2, 3), (2, 40, 3, 12), (1, 2100, 1, 1), (4, 200, 130, 12)])
def test_16_bit_inputs_have_fp32_states(B, T, N, G, dt):
    """Small candidates (tanh near 0) and gates far from 0 of 16-bit types: the fp32 state is as exact as that of fp32 inputs."""
    gate, cand, st, _, dout, dlast = _inputs(B, T, N, 12, G, dt, False, T + G)
    g = torch.Generator().manual_seed(T)
    cand = (cand.float() * 10.0 ** (-3 * torch.rand(cand.shape, generator=g))).to(TORCH[dt])
    gate = torch.where(torch.rand(gate.shape, generator=g) < 0.3, -25 + 50 * torch.rand(gate.shape, generator=g), gate.float()).to(TORCH[dt])
    _against_oracle(gate, cand, st * 1e-3, None, dout, dlast, "tanh", dt)


@pytest.mark.gpu
def test_extreme_gates_and_small_candidates():
    """Gates of +-100 and +-inf hold or replace the state exactly; tanh of 1e-6 .. 1e-2 keeps its relative precision."""
    import megacrn_amd
    gate = torch.tensor([100.0, -100.0, float("inf"), float("-inf"), 80.0, -80.0, 0.0, -0.0]).view(1, 1, 1, 8).expand(1, 40, 1, 8).contiguous()
    cand = torch.full((1, 40, 1, 8), 0.5)
    st = torch.arange(1.0, 9.0).view(1, 1, 8)
    out, last = megacrn_amd.gated_linear_recurrence(gate.cuda(), cand.cuda(), st.cuda(), activation="none")
    want = torch.tensor([1.0, 0.5, 3.0, 0.5, 5.0, 0.5])
    assert torch.equal(out[0, 0, 0, :6].cpu(), want) and torch.equal(last[0, 0, :6].cpu(), want)
    small = torch.logspace(-6, -0.2, 64).view(1, 1, 1, 64)
    out, _ = megacrn_amd.gated_linear_recurrence(torch.full_like(small, -100.0).cuda(), torch.cat([small, -small], 1).cuda()[:, :1])
    rel = (out.cpu().double() / torch.tanh(small.double()) - 1).abs().max().item()
    assert rel <= (O.KC + 2) * O.U, rel


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strided_inputs(dt):
    """Gate and candidate as halves of one product, transposed batches, rows of odd stride, masks shared over nodes or time."""
    import megacrn_amd
    torch.manual_seed(0)
    B, T, N, H = 3, 21, 5, 16
    both = torch.randn(B, T, N, 2 * H).to(TORCH[dt])
    gate, cand, st, _, dout, dlast = _inputs(B, T, N, H, H, dt, False, 3)
    views = [lambda t: torch.cat([t, t], -1).cuda()[..., t.shape[-1]:] if t.dim() == 4 else t.cuda(),
             lambda t: t.transpose(0, 1).contiguous().cuda().transpose(0, 1),
             lambda t: torch.nn.functional.pad(t, (0, 3)).cuda()[..., :-3] if t.dim() == 4 else t.cuda(),
             lambda t: torch.nn.functional.pad(t, (1, 0)).cuda()[..., 1:] if t.dim() == 4 else t.cuda(),
             lambda t: t.transpose(2, 3).contiguous().cuda().transpose(2, 3) if t.dim() == 4 else t.cuda()]
    for lay in views:
        _against_oracle(gate, cand, st, None, dout, dlast, "tanh", dt, lay)
    halves = both.cuda().chunk(2, -1)
    a, _ = megacrn_amd.gated_linear_recurrence(*halves, st.cuda())
    b, _ = megacrn_amd.gated_linear_recurrence(*[t.contiguous() for t in halves], st.cuda())
    assert torch.equal(a, b)
    rows = torch.rand(B, T) > 0.3
    for mask in (rows, rows.unsqueeze(-1), rows[:1].unsqueeze(-1), rows[:, :1, None]):
        full = (mask if mask.dim() == 3 else mask.unsqueeze(-1)).expand(B, T, N)
        a, _ = megacrn_amd.gated_linear_recurrence(*halves, st.cuda(), mask.cuda())
        b, _ = megacrn_amd.gated_linear_recurrence(*halves, st.cuda(), full.contiguous().cuda())
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,H", [(30, 3, 8), (300, 40, 64), (700, 3, 8)])
def test_gradient_of_expanded_and_partial_outputs(T, N, H):
    """dout that is expanded (a sum), missing (only `last` used) or reaches one step only; a gate broadcast by its user."""
    import megacrn_amd
    gate, cand, st, _, _, _ = _inputs(2, T, N, H, H, "f32", False, 9)
    out, last, eh, cache = O.glr_fwd(_np(gate), _np(cand), _np(st))
    one = np.zeros_like(out)
    one[:, 11] = 1.0
    for pick, dout, dlast in ((lambda o, l: o.sum(), np.ones_like(out), None), (lambda o, l: l.sum(), None, np.ones_like(last)),
                              (lambda o, l: o[:, 11].sum(), one, None)):
        leaves = [t.cuda().requires_grad_() for t in (gate, cand, st)]
        grads = torch.autograd.grad(pick(*megacrn_amd.gated_linear_recurrence(*leaves)), leaves)
        dg, dc, ds, eg, ec, es = O.glr_bwd(cache, dout, dlast)
        _close(grads[0], dg, eg + O.half_step(dg, "f32"), "dgate")
        _close(grads[1], dc, ec + O.half_step(dc, "f32"), "dcand")
        _close(grads[2], ds, es + O.half_step(ds, "f32"), "dstate")
    row = gate[:1, :1].cuda().requires_grad_()                             # one gate row for all batch entries and steps
    o, _ = megacrn_amd.gated_linear_recurrence(row.expand(2, T, N, H), cand.cuda())
    (g,) = torch.autograd.grad(o.sum(), row)
    _, _, _, cache = O.glr_fwd(np.broadcast_to(_np(gate[:1, :1]), gate.shape).copy(), _np(cand))
    dg, _, _, eg, _, _ = O.glr_bwd(cache, np.ones_like(out), None)
    # the sum over 2 T rows is torch's: at most 2 T roundings of partial sums
    _close(g, dg.sum((0, 1), keepdims=True), (eg + O.half_step(dg, "f32")).sum((0, 1), keepdims=True) + 2 * T * O.U * np.abs(dg).sum((0, 1), keepdims=True), "shared row")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 0, 3, 8), (0, 5, 3, 8), (2, 5, 0, 8)])
def test_empty(shape):
    import megacrn_amd
    B, T, N, H = shape
    st = torch.randn(B, N, H, device="cuda", requires_grad=True)
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    out, last = megacrn_amd.gated_linear_recurrence(x, x, st)
    assert out.shape == shape and torch.equal(last, st)
    (g,) = torch.autograd.grad(last.sum(), st)
    assert torch.equal(g, torch.ones_like(st))
    assert megacrn_amd.gated_linear_recurrence_step(torch.zeros(0, 3, 8, device="cuda"), torch.zeros(0, 3, 8, device="cuda"), torch.zeros(0, 3, 8, device="cuda")).shape == (0, 3, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 0, 3, 8), (0, 5, 3, 8), (2, 5, 0, 8)])
def test_backward_of_empty_sequences(shape, dt, state):
    """No batch, no step or no node: a loss over the outputs still has a backward pass, with gradients of no elements."""
    import megacrn_amd
    B, T, N, H = shape
    gate, cand = (torch.zeros(B, T, N, w, dtype=TORCH[dt], device="cuda", requires_grad=True) for w in (2, H))
    st = torch.randn(B, N, H, device="cuda", requires_grad=True) if state else None
    out, last = megacrn_amd.gated_linear_recurrence(gate, cand, st)
    assert out.shape == shape and out.dtype == TORCH[dt] and last.dtype == torch.float32 and torch.equal(last, torch.zeros(B, N, H, device="cuda") if st is None else st)
    for loss in (out.float().sum(), last.sum(), out.float().sum() + last.sum()):
        grads = torch.autograd.grad(loss, [gate, cand], retain_graph=True)
        assert grads[0].shape == gate.shape and grads[1].shape == cand.shape
    if state:
        assert torch.equal(torch.autograd.grad(last.sum(), st)[0], torch.ones_like(st))


@pytest.mark.gpu
def test_agl_cell_without_batch_or_steps():
    import megacrn_amd
    cell = megacrn_amd.AGLRCell(5, 3, 8, 3).cuda()
    sup = [torch.eye(5, device="cuda")] * 2
    for B, T in ((0, 4), (2, 0)):
        st = torch.randn(B, 5, 8, device="cuda")
        out, last = cell(torch.zeros(B, T, 5, 3, device="cuda"), st, sup)
        assert out.shape == (B, T, 5, 8) and torch.equal(last, st)
    assert cell.step(torch.zeros(0, 5, 3, device="cuda"), torch.zeros(0, 5, 8, device="cuda"), sup).shape == (0, 5, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("G", [24, 3, 1])
def test_steps_are_the_sequence(dt, G):
    """Steps taken one by one give the states of the whole sequence."""
    import megacrn_amd
    gate, cand, st, keep, _, _ = (None if t is None else t.cuda() for t in _inputs(4, 13, 6, 24, G, dt, True, 1))
    out, last = megacrn_amd.gated_linear_recurrence(gate, cand, st, keep)
    now = st.clone()
    for t in range(13):
        o = megacrn_amd.gated_linear_recurrence_step(gate[:, t], cand[:, t], now, keep[:, t])
        assert o.dtype == TORCH[dt]
        want = O.glr_fwd(_np(gate[:, :t + 1].cpu()), _np(cand[:, :t + 1].cpu()), _np(st.cpu()), keep[:, :t + 1].cpu().numpy(), dt=dt)
        _close(o, want[0][:, -1], want[2][:, -1] + O.half_step(want[0][:, -1], dt), f"step {t}")
    _close(now, want[1], want[2][:, -1] + O.half_step(want[1], "f32"), "state")
    _close(last, want[1], want[2][:, -1] + O.half_step(want[1], "f32"), "last")
    with pytest.raises(RuntimeError):
        megacrn_amd.gated_linear_recurrence_step(gate[:, 0].requires_grad_(), cand[:, 0], now)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [8, 1])
def test_views_that_are_negative_by_a_bit(H):
    """The imaginary part of a conjugate holds its numbers with the other sign in memory; a last dimension of 1 is read in place whatever its stride."""
    import megacrn_amd
    torch.manual_seed(1)
    z = torch.randn(5, 2, 7, 3, H, dtype=torch.complex64, device="cuda")
    neg = z.conj().imag
    assert neg.is_neg()
    real = neg.resolve_neg()
    grads = []
    for t in (neg, real):
        leaves = [t[0].detach().requires_grad_(), t[1].detach(), t[2, :, 0].detach()]
        out, last = megacrn_amd.gated_linear_recurrence(*leaves)
        (g,) = torch.autograd.grad((out, last), leaves[:1], (t[3], t[4, :, 0]))
        now = real[2, :, 0].contiguous()
        with torch.no_grad():
            grads.append((out, last, g, megacrn_amd.gated_linear_recurrence_step(t[0, :, 0], t[1, :, 0], now), now, megacrn_amd.gated_linear_recurrence(*leaves)[0]))
        p = torch.ones(2, 7, 3, H, device="cuda")
        megacrn_amd.AdamW([p]).step(grads=[t[0]])
        grads[-1] += (p,)
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    with pytest.raises(ValueError):
        megacrn_amd.gated_linear_recurrence_step(real[0, :, 0], real[1, :, 0], torch._neg_view(torch.empty(2, 3, H, device="cuda")))


@pytest.mark.gpu
def test_step_whose_inputs_lie_in_its_state():
    """A gate or a candidate that is a view of the state, or of memory that overlaps it, is what it was before the step."""
    import megacrn_amd
    N, H = 20000, 1100
    buf = torch.randn(1, N + 1, H, device="cuda")
    for pick in (lambda b: (b[:, :N, :1], b[:, 1:]), lambda b: (b[:, 1:], b[:, :N]), lambda b: (b[:, 1:], b[:, 1:]), lambda b: (b[:, 1:], b[:, 1:2].expand(1, N, H)),
                 lambda b: (b[:, 1:2].expand(1, N, H), b[:, -1:].expand(1, N, H))):
        a, want = buf.clone(), buf.clone()
        ref = want[:, 1:].clone()
        out_ref = megacrn_amd.gated_linear_recurrence_step(*(t.clone() for t in pick(want)), ref)
        out = megacrn_amd.gated_linear_recurrence_step(*pick(a), a[:, 1:])
        assert torch.equal(out, out_ref) and torch.equal(a[:, 1:], ref) and torch.equal(a[:, :1], buf[:, :1])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,N,H", [(2, 1, 3, 8), (2, 5, 3, 8), (2, 30, 3, 8), (2, 300, 3, 8), (1, 300, 40, 64), (64, 20, 40, 256)])
def test_state_of_a_masked_row_is_kept_whatever_it_is(B, T, N, H, dt):
    """Infinities and NaN among the states that no step writes; the gradients of masked steps are 0 there too."""
    import megacrn_amd
    gate, cand, st, _, _, _ = (None if t is None else t.cuda() for t in _inputs(B, T, N, H, H, dt, False, 3))
    keep = torch.ones(B, T, N, dtype=torch.bool, device="cuda")
    keep[-1, :, 1] = False
    st[-1, 1, :4] = torch.tensor([float("inf"), -float("inf"), 3e38, float("nan")], device="cuda")
    gate[-1, :, 1], cand[-1, :, 1] = float("nan"), float("inf")
    gate.requires_grad_(), cand.requires_grad_()
    out, last = megacrn_amd.gated_linear_recurrence(gate, cand, st, keep)
    want = st[-1, 1]
    assert torch.equal(torch.nan_to_num(last[-1, 1], 7.0), torch.nan_to_num(want, 7.0)) and torch.isnan(last).sum() == 1
    rows = want.to(TORCH[dt]).expand(T, H)
    assert torch.equal(torch.nan_to_num(out[-1, :, 1], 7.0), torch.nan_to_num(rows, 7.0)) and torch.isnan(out).sum() == T
    dgate, dcand = torch.autograd.grad(out, (gate, cand), torch.ones_like(out))
    assert not dgate[-1, :, 1].any() and not dcand[-1, :, 1].any() and torch.isfinite(dcand).all() and torch.isfinite(dgate).all()
    now = st.clone()
    with torch.no_grad():
        step = megacrn_amd.gated_linear_recurrence_step(gate[:, 0], cand[:, 0], now, keep[:, 0])
    assert torch.equal(torch.nan_to_num(now[-1, 1], 7.0), torch.nan_to_num(want, 7.0)) and torch.isnan(now).sum() == 1
    assert torch.equal(torch.nan_to_num(step[-1, 1], 7.0), torch.nan_to_num(rows[0], 7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,N,H,G", [(2, 1, 3, 8, 8), (2, 5, 3, 8, 4), (2, 8, 3, 7, 7), (2, 30, 3, 8, 8), (2, 33, 5, 12, 1), (2, 300, 3, 8, 2), (2, 2100, 3, 9, 9),
                                       (2, 300, 40, 64, 64), (2, 300, 100, 64, 1), (2, 300, 150, 33, 33), (64, 20, 40, 256, 256), (33, 20, 64, 65, 5)])
def test_infinite_gradients_of_masked_steps(B, T, N, H, G, dt):
    """Gradients that are not finite pass a masked step as they are and leave its own gradients 0, in every variant and whether T fills its tiles
    or not; every other row is what it is without them."""
    import megacrn_amd
    gate, cand, st, _, dout, dlast = (None if t is None else t.cuda() for t in _inputs(B, T, N, H, G, dt, False, 3))
    keep = torch.rand(B, T, N, generator=torch.Generator().manual_seed(T)).cuda() > 0.2
    keep[-1, :, 1] = False                                                 # never moved
    keep[0, T // 2:, 2] = False                                            # masked towards the end
    gate[-1, :, 1], cand[-1, :, 1] = float("nan"), -float("inf")

    def run(dout, dlast):
        leaves = [t.detach().requires_grad_() for t in (gate, cand, st)]
        out, last = megacrn_amd.gated_linear_recurrence(*leaves, keep)
        return torch.autograd.grad((out, last), leaves, (dout, dlast))
    want = run(dout, dlast)
    assert all(torch.isfinite(t).all() for t in want)
    bad = torch.tensor([float("inf"), -float("inf"), float("nan")], device="cuda").repeat((H + 2) // 3)[:H]
    dlast2, dout2 = dlast.clone(), dout.clone()
    dlast2[-1, 1] = bad
    dout2[0, -1, 2] = bad.to(dout.dtype)
    got = run(dout2, dlast2)
    assert torch.equal(torch.nan_to_num(got[2][-1, 1], 7.0), torch.nan_to_num(bad, 7.0))
    for g, w in zip(got[:2], want[:2]):
        assert not g[-1, :, 1].any() and not g[0, T // 2:, 2].any()
        g[0, :, 2] = w[0, :, 2]
    got[2][0, 2], got[2][-1, 1] = want[2][0, 2], want[2][-1, 1]
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_nan_stays_in_its_row():
    """A NaN that is not masked reaches its own channel's later steps and nothing else."""
    import megacrn_amd
    gate, cand, st, _, _, _ = (None if t is None else t.cuda() for t in _inputs(2, 300, 3, 8, 8, "f32", False, 2))
    want, _ = megacrn_amd.gated_linear_recurrence(gate, cand, st)
    cand[1, 150, 2, 5] = float("nan")
    got, last = megacrn_amd.gated_linear_recurrence(gate, cand, st)
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[1, 150:, 2, 5] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit]) and torch.isnan(last).sum() == 1


@pytest.mark.gpu
def test_graph_replay_and_other_stream():
    """Forward, backward and a serving step captured once and replayed on new inputs, with eager work between; then the same
    calls on a stream of their own.  One plan and one order of sums: bit for bit."""
    import megacrn_amd
    shapes = [(2, 24, 5, 16), (1, 2100, 1, 12), (2, 400, 40, 64)]
    for B, T, N, H in shapes:
        def fresh(seed):
            return [None if t is None else t.cuda() for t in _inputs(B, T, N, H, H, "f32", True, seed)]

        def run(gate, cand, st, keep, dout, dlast):
            leaves = [t.detach().requires_grad_() for t in (gate, cand, st)]
            out, last = megacrn_amd.gated_linear_recurrence(*leaves, keep)
            return (out.detach(), last.detach()) + torch.autograd.grad((out, last), leaves, (dout, dlast))

        static = fresh(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        now = static[2].clone()
        with torch.cuda.graph(graph):
            held = run(*static)
            megacrn_amd.gated_linear_recurrence_step(static[0][:, 0], static[1][:, 0], now, static[3][:, 0])
        for seed in (1, 2, 3):
            new = fresh(seed)
            for s, t in zip(static, new):
                s.copy_(t)
            now.copy_(new[2])
            graph.replay()
            want = run(*new)
            torch.cuda.synchronize()
            for a, b in zip(held, want):
                assert torch.equal(a, b)
            first = new[2].clone()
            megacrn_amd.gated_linear_recurrence_step(new[0][:, 0], new[1][:, 0], first, new[3][:, 0])
            assert torch.equal(now, first)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            other = run(*new)
        torch.cuda.synchronize()
        for a, b in zip(other, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_second_derivative_is_refused():
    import megacrn_amd
    gate, cand, st, _, _, _ = (None if t is None else t.cuda() for t in _inputs(1, 20, 2, 4, 4, "f32", False, 2))
    out, _ = megacrn_amd.gated_linear_recurrence(gate.requires_grad_(), cand, st)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out.sum(), gate, create_graph=True)


@pytest.mark.gpu
def test_output_changed_before_backward_is_noticed():
    import megacrn_amd
    gate, cand, st, _, _, _ = (None if t is None else t.cuda() for t in _inputs(1, 20, 2, 4, 4, "f32", False, 2))
    out, last = megacrn_amd.gated_linear_recurrence(gate.requires_grad_(), cand, st)
    loss = out.sum()
    with torch.no_grad():
        out.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_many_elements():
    """More than 2^31 elements of gate and cand (bf16): offsets past 32 bits.  Gates of -100 make every step its candidate."""
    import megacrn_amd
    B, T, N, H = 3, 4200, 2700, 64
    gate = torch.full((1, 1, 1, 1), -100.0, dtype=torch.bfloat16, device="cuda").expand(B, T, N, 1)
    cand = torch.empty(B, T, N, H, dtype=torch.bfloat16, device="cuda")
    cand.copy_((torch.arange(T, device="cuda").view(1, T, 1, 1) % 100 + torch.arange(B, device="cuda").view(B, 1, 1, 1)).to(torch.bfloat16))
    assert cand.numel() > 2 ** 31
    with torch.no_grad():
        out, last = megacrn_amd.gated_linear_recurrence(gate, cand, None, activation="none")
    for b in range(B):
        assert torch.equal(out[b], cand[b])
    assert torch.equal(last, cand[:, -1].float())


@pytest.mark.gpu
def test_masks_that_lie_far_apart():
    """A mask whose nodes are 4 GB from each other is copied as the inputs are."""
    import megacrn_amd
    far = torch.zeros(2 ** 32 + 64, dtype=torch.bool, device="cuda").as_strided((1, 3, 2), (64, 8, 2 ** 32))
    near = torch.tensor([[[True, False], [False, True], [True, True]]], device="cuda")
    far.copy_(near)
    x = torch.randn(1, 3, 2, 4, device="cuda", requires_grad=True)
    a, b = (megacrn_amd.gated_linear_recurrence(x, x, None, m) for m in (far, near))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert all(torch.equal(p, q) for p, q in zip(*(torch.autograd.grad(t[0].sum(), x) for t in (a, b))))
    states = [torch.ones(1, 2, 4, device="cuda") for _ in range(2)]
    with torch.no_grad():
        for st, m in zip(states, (far, near)):
            megacrn_amd.gated_linear_recurrence_step(x[:, 1], x[:, 1], st, m[:, 1])
    assert torch.equal(*states)


@pytest.mark.gpu
def test_as_many_sequences_as_a_launch_holds():
    """2^24 - 1 sequences of one channel are one launch; one more is refused before it."""
    import megacrn_amd
    B = 2 ** 24 - 1
    cand = torch.arange(B, device="cuda", dtype=torch.float32).view(B, 1, 1, 1)
    gate = torch.full((1, 1, 1, 1), -200.0, device="cuda")
    out, last = megacrn_amd.gated_linear_recurrence(gate.expand(B, 1, 1, 1), cand, activation="none")
    assert torch.equal(out, cand) and torch.equal(last, cand[:, 0])
    many = torch.zeros(1, 1, 1, 1, device="cuda").expand(B + 1, 1, 1, 1)
    with pytest.raises(RuntimeError, match="too many sequences"):
        megacrn_amd.gated_linear_recurrence(many, many)


@pytest.mark.gpu
def test_rows_that_lie_far_apart():
    """Nodes 4 GB from each other: beyond the 32 bits that a lane has, so the node copies them first; the C entry refuses them."""
    import megacrn_amd
    buf = torch.zeros(2 ** 31 + 64, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((1, 3, 2, 4), (64, 8, 2 ** 31, 1))
    near = torch.randn(1, 3, 2, 4, device="cuda").to(torch.bfloat16)
    far.copy_(near)
    a, la = megacrn_amd.gated_linear_recurrence(far, far)
    b, lb = megacrn_amd.gated_linear_recurrence(near, near)
    assert torch.equal(a, b) and torch.equal(la, lb)


def _c_forward(gate, cand, state, out, last, ws=0, **over):
    """The C entry itself on contiguous tensors."""
    import ctypes as C
    from megacrn_amd._lib import lib
    B, T, N, H = cand.shape
    G = gate.shape[3]

    class Glr(C.Structure):
        _fields_ = [("i", C.c_int * 8), ("s", C.c_longlong * 12)]
    v = dict(B=B, T=T, N=N, H=H, G=G, dtype=0, act=1, reserved=0)
    v.update(over)
    d = Glr((C.c_int * 8)(*v.values()), (C.c_longlong * 12)(T * N * G, N * G, G, T * N * H, N * H, H, 0, 0, 0, 0, 0, 0))
    lib.mcrn_glr_workspace_bytes.restype, lib.mcrn_glr_workspace_bytes.argtypes = C.c_size_t, [C.POINTER(Glr), C.c_int]
    nb = lib.mcrn_glr_workspace_bytes(C.byref(d), 0)
    space = torch.empty(max(nb, 256), dtype=torch.uint8, device="cuda")
    f = lib.mcrn_glr_forward
    f.restype, f.argtypes = C.c_int, [C.POINTER(Glr)] + [C.c_void_p] * 5 + [C.c_size_t] + [C.c_void_p] * 4
    p = [None if t is None else t.data_ptr() for t in (gate, cand, state, out, last)]
    return f(C.byref(d), p[0], p[1], None, p[2], space.data_ptr(), nb + ws, p[3], p[4], None, torch.cuda.current_stream().cuda_stream), nb


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,N,H", [(2, 0, 3, 8), (1, 3000, 1, 12), (1, 700, 80, 64), (3, 5, 2, 8), (1, 100, 3, 8),
                                     (1, 1, 9, 33), (2, 5, 3, 7), (1, 100, 3, 9), (1, 3000, 1, 13)])
def test_c_entry_in_place_and_without_outputs(B, T, N, H):
    """The state advanced in place over a whole sequence, with no `out`, in every variant (a split would read what it overwrites: not planned)."""
    import megacrn_amd
    gate, cand, st, _, _, _ = (None if t is None else t.cuda() for t in _inputs(B, T, N, H, H, "f32", False, 4))
    _, want = megacrn_amd.gated_linear_recurrence(gate, cand, st)
    for _ in range(3):
        now = st.clone()
        assert _c_forward(gate, cand, now, None, now)[0] == 0
        assert (now - want).abs().max().item() <= 1e-5 if T else torch.equal(now, want)


@pytest.mark.gpu
def test_c_entry_refusals():
    """Sizes, types, alignment and a workspace that is too small come back as an error code before anything is launched."""
    from megacrn_amd._lib import lib
    gate, cand, st, _, _, _ = (None if t is None else t.cuda() for t in _inputs(1, 2100, 1, 12, 12, "f32", False, 4))
    out, last = torch.empty_like(cand), torch.empty_like(st)
    rc, nb = _c_forward(gate, cand, st, out, last)
    assert rc == 0 and nb > 0
    assert _c_forward(gate, cand, st, out, last, ws=-nb)[0] == -1 and b"workspace" in lib.mcrn_last_error()
    for over in (dict(B=-1), dict(H=0), dict(G=5), dict(dtype=3), dict(act=2), dict(reserved=1), dict(T=2 ** 30 + 1)):
        assert _c_forward(gate, cand, st, out, last, **over)[0] == -1
    assert _c_forward(gate, cand, torch.empty(64, device="cuda", dtype=torch.uint8)[1:], out, last)[0] == -1
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_sequences_at_once():
    """Two chained sequences on two streams: each waits for its own blocks only, both give what they give alone."""
    import megacrn_amd
    data = [[None if t is None else t.cuda() for t in _inputs(1, 3000, 80, 64, 64, "bf16", True, k)] for k in (1, 2)]
    want = [megacrn_amd.gated_linear_recurrence(d[0], d[1], d[2], d[3]) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, (d, s) in enumerate(zip(data, streams)):
            with torch.cuda.stream(s):
                got[k].append(megacrn_amd.gated_linear_recurrence(d[0], d[1], d[2], d[3]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for out, last in got[k]:
            assert torch.equal(out, want[k][0]) and torch.equal(last, want[k][1])


@pytest.mark.gpu
def test_two_threads():
    """One thread trains (its backward passes run on autograd's thread, without the interpreter lock), another one serves and updates:
    each gets what it gets alone."""
    import threading
    import megacrn_amd
    gate, cand, st, keep, dout, _ = (t.cuda() for t in _inputs(2, 300, 5, 8, 8, "f32", True, 6))
    gate.requires_grad_(), cand.requires_grad_()
    w, g = torch.randn(500, device="cuda"), torch.randn(500, device="cuda")

    def train(got):
        for _ in range(100):
            out, _ = megacrn_amd.gated_linear_recurrence(gate, cand, st, keep)
            got[:] = torch.autograd.grad(out, (gate, cand), dout)

    def serve(got):
        now, p = st.clone(), w.clone()
        opt = megacrn_amd.AdamW([p], max_grad_norm=1.0, state_bits=8)
        for t in range(300):
            with torch.no_grad():
                megacrn_amd.gated_linear_recurrence_step(gate[:, t], cand[:, t], now, keep[:, t])
            opt.step(grads=[g])
        got[:] = [now, p]
    alone, both, errors = [[], []], [[], []], []
    train(alone[0]), serve(alone[1])

    def guarded(f, got):
        try:
            f(got)
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(f, got)) for f, got in zip((train, serve), both)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert len(b) == 2 and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_cells_on_two_threads_and_streams():
    """A cell trains on one thread and stream while another one serves on its own: the graph convolution's calls and workspaces are part of it."""
    import threading
    import megacrn_amd
    torch.manual_seed(5)
    B, T, N, C, H, K = 2, 12, 20, 3, 16, 3
    cells = [megacrn_amd.AGLRCell(N, C, H, K).cuda() for _ in range(2)]
    sup = [torch.softmax(torch.randn(N, N, device="cuda"), -1) for _ in range(2)]
    x, st = torch.randn(B, T, N, C, device="cuda"), torch.randn(B, N, H, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def train(got):
        with torch.cuda.stream(streams[0]):
            for _ in range(60):
                out, last = cells[0](x, st, sup)
                got[:] = [out.detach(), *torch.autograd.grad(out.sum() + last.sum(), list(cells[0].parameters()))]

    def serve(got):
        with torch.cuda.stream(streams[1]):
            for _ in range(20):
                now = st.clone()
                for t in range(T):
                    cells[1].step(x[:, t], now, sup)
                out, _ = cells[1](x, st, sup)              # the training thread's sizes, its own workspace
                got[:] = [now, out.detach()]
    alone, both, errors = [[], []], [[], []], []
    train(alone[0]), serve(alone[1])
    torch.cuda.synchronize()

    def guarded(f, got):
        try:
            f(got)
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(f, got)) for f, got in zip((train, serve), both)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert len(a) == len(b) and all(torch.allclose(p, q, rtol=1e-5, atol=1e-6 * p.abs().max().item()) for p, q in zip(a, b))


@pytest.mark.gpu
def test_agl_cell_training_run():
    """The module as it is used: supports -> graph convolution of all steps -> recurrence -> loss -> gradients, against float64; then
    its steps in place against the sequence, and an AdamW update of all its parameters."""
    import megacrn_amd
    torch.manual_seed(3)
    B, T, N, C, H, K = 2, 11, 9, 3, 8, 3
    cell = megacrn_amd.AGLRCell(N, C, H, K).cuda()
    assert set(cell.state_dict()) == {"gate_cand.weights", "gate_cand.bias"}
    S = [torch.softmax(torch.randn(N, N), -1) for _ in range(2)]
    x, st, mask = torch.randn(B, T, N, C), torch.randn(B, N, H), torch.rand(B, T, N) > 0.2
    d = torch.randn(B, T, N, H)
    sup = [s.cuda() for s in S]
    out, last = cell(x.cuda(), st.cuda(), sup, mask.cuda())
    (out * d.cuda()).sum().backward()
    W, b = (p.detach().cpu().double().numpy() for p in (cell.gate_cand.weights, cell.gate_cand.bias))
    y, cache = MO.agcn_fwd(_np(x).reshape(B * T, N, C), [_np(s) for s in S], W, b, K)
    y = y.reshape(B, T, N, 2 * H)
    want, wlast, _, gc = O.glr_fwd(y[..., :H].copy(), y[..., H:].copy(), _np(st), mask.numpy())
    dg, dc, _, _, _, _ = O.glr_bwd(gc, _np(d), None)
    back = MO.agcn_bwd(np.concatenate([dg, dc], -1).reshape(B * T, N, 2 * H), cache)
    grads = [g for g in back if isinstance(g, np.ndarray) and g.shape in (W.shape, b.shape)]
    # the convolution's own contract is 1e-4 of a tensor's scale; the recurrence's step is no steeper than 1 in gate and candidate
    for got, ref in ((out, want), (last, wlast), (cell.gate_cand.weights.grad, grads[0]), (cell.gate_cand.bias.grad, grads[1])):
        assert np.abs(got.detach().cpu().double().numpy() - ref).max() <= 2e-4 * np.abs(ref).max()
    now = st.cuda().clone()
    for t in range(T):
        o = cell.step(x[:, t].cuda(), now, sup, mask[:, t].cuda())
        assert np.abs(o.cpu().double().numpy() - want[:, t]).max() <= 2e-4 * np.abs(want).max()
    opt = megacrn_amd.AdamW(cell.parameters(), lr=1e-2, max_grad_norm=1.0, state_bits=8)
    before = [p.detach().clone() for p in cell.parameters()]
    opt.step()
    for p, q in zip(cell.parameters(), before):
        assert torch.isfinite(p).all() and 0 < (p - q).abs().max() <= 1.1e-2 * (1 + q.abs().max())
