"""AdamW over many tensors: 32-bit moments against float64 within running error bounds, 8-bit moments code by code against the
oracle's own formats (oracle/sequence_oracle.py), and what the optimizer refuses."""
import numpy as np
import pytest
import torch

from helpers import SC_MEAN, SC_STD
from oracle import megacrn_oracle as MO
from oracle import sequence_oracle as O

F = np.float32


# ---------------------------------------------------------------------------------------------------------------------
# without a GPU
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("second", [False, True])
def test_formats(second):
    """Every code stands for the number that its exponent and mantissa say, codes rise with their numbers, and a code's own value
    comes back as that code whatever the random bits are."""
    t = O.table(second)
    assert (np.diff(t) > 0).all() and t[0] == 0
    for s in (1, 60, 127, 200):
        top = 15 if second else 7
        codes = np.array([c for c in range(len(t) - 1) if 0 < t[c] < 2.0 ** (top + 1)], np.uint8)
        codes = np.concatenate([codes, np.full((-len(codes)) % 64, codes[-1], np.uint8)]).reshape(-1, 64)
        for blk in codes:
            blk[0] = max(c for c in range(len(t)) if t[c] < 2.0 ** (top + 1))           # a value that fixes the scale
            x = (t[blk.astype(int)] * 2.0 ** (s - 127)).astype(F)
            if (x == 0).any() or not np.isfinite(x).all():
                continue
            for r in (0, 0xFFFF):
                got, sc = O.encode(x, np.full(64, r), second)
                assert sc[0] == s and (got == blk).all()


@pytest.mark.parametrize("second", [False, True])
def test_rounding_is_unbiased(second):
    """The mean over the random bits is the value: 4096 copies of 60 values, off by at most 6 standard errors of a rounding between
    neighbours (each at most half their distance)."""
    rng = np.random.default_rng(1)
    vals = (np.abs(rng.normal(1, 0.4, 60)) * 10.0 ** rng.uniform(-3, 0, 60)).astype(F)
    bits = O.random_bits(7, 3, 11, 64 * 64 * 64).reshape(64 * 64, 64)
    acc = np.zeros(60)
    for row in bits:
        blk = np.concatenate([[F(1.9)], vals, np.zeros(3, F)])
        c, s = O.encode(blk, (row >> 16) if second else (row & 0xFFFF), second)
        acc += O.decode(c, s, second)[1:61]
    gap = np.maximum(vals / 8, 2.0 ** (s[0] - 127.0) * O.table(second)[1])
    assert (np.abs(acc / len(bits) - vals) <= 6 * gap / 2 / np.sqrt(len(bits))).all()


def test_random_bits_are_spread():
    """Means, lags and both halves of the 32 bits over 2^16 elements within 5 standard errors."""
    n = 1 << 16
    for key in ((0, 0, 1), (0, 0, 2), (5, 7, 1000)):
        b = O.random_bits(*key, n)
        lo, hi = (b & 0xFFFF) / 65536.0 - 0.5, (b >> 16) / 65536.0 - 0.5
        for x, y in ((lo, np.ones(n) / np.sqrt(12)), (hi, np.ones(n) / np.sqrt(12)), (lo, hi), (lo, np.roll(lo, 1)), (hi, np.roll(hi, 64))):
            assert abs((x * y).mean()) * 12 <= 5 / np.sqrt(n)


def test_arena_and_workspace_sizes():
    import ctypes as C
    from megacrn_amd._lib import lib, Adamw
    n = (C.c_longlong * 4)(1, 64, 65, 0)

    def cfg(k=4, dtype=0, bits=32):
        return C.byref(Adamw(k, dtype, bits, 0, 0, 0, 0.9, 0.999, 1e-8, 0.0, 1.0))
    assert lib.mcrn_adamw_arena_elements(cfg(), n) == 64 + 64 + 128
    assert lib.mcrn_adamw_workspace_bytes(cfg(), n) > 0
    for bad in (cfg(k=0), cfg(dtype=2), cfg(bits=4)):
        assert lib.mcrn_adamw_arena_elements(bad, n) == -1 and lib.mcrn_adamw_workspace_bytes(bad, n) == 0
    assert lib.mcrn_adamw_arena_elements(cfg(), (C.c_longlong * 4)(1, -1, 65, 0)) == -1


def test_sizes_that_no_launch_holds():
    """A launch has fewer than 2^32 work items, 2^24 blocks of 256 threads and 1024 elements: what lies beyond is refused with the sizes, not by a
    launch after others have updated their tensors."""
    import ctypes as C
    from megacrn_amd._lib import lib, Adamw
    cfg = C.byref(Adamw(2, 1, 8, 0, 0, 0, 0.9, 0.999, 1e-8, 1.0, 1.0))
    most = 2 ** 34 - 1024
    for n, ok in ((most, True), (most + 1, False), (2 ** 40, False)):
        sizes = (C.c_longlong * 2)(100, n)
        assert lib.mcrn_adamw_arena_elements(cfg, sizes) == ((128 + most) if ok else -1)
        assert (lib.mcrn_adamw_workspace_bytes(cfg, sizes) > 0) == ok


P = torch.nn.Parameter


@pytest.mark.parametrize("params,kw,kind", [
    ([], {}, ValueError), ([torch.zeros(3)], dict(state_bits=16), ValueError), ([torch.zeros(3)], dict(betas=(0.9, 1.0)), ValueError),
    ([torch.zeros(3)], dict(eps=0.0), ValueError), ([torch.zeros(3)], dict(lr=-1.0), ValueError), ([torch.zeros(3)], dict(weight_decay=-1.0), ValueError),
    ([torch.zeros(3)], dict(max_grad_norm=float("nan")), ValueError),
    ([torch.zeros(3, dtype=torch.float16)], {}, TypeError), ([torch.zeros(3), torch.zeros(3, dtype=torch.bfloat16)], {}, TypeError),
    ([torch.zeros(3, 4).t()], {}, ValueError), (["x"], {}, TypeError), ([torch.zeros(3)], {}, RuntimeError),
])
def test_refusals(params, kw, kind):
    import megacrn_amd
    with pytest.raises(kind):
        megacrn_amd.AdamW(params, **kw)


def test_refuses_a_parameter_twice():
    import megacrn_amd
    p = torch.zeros(3)
    with pytest.raises(ValueError, match="twice"):
        megacrn_amd.AdamW([{"params": [p]}, {"params": [p]}])


def test_refuses_shared_memory_and_unknown_group_keys():
    import megacrn_amd
    base = torch.zeros(9)
    for pair in ([base[:5], base[4:]], [base, base.view(3, 3)], [base[4:5], base]):
        with pytest.raises(ValueError, match="share memory"):
            megacrn_amd.AdamW(pair)
    with pytest.raises(RuntimeError, match="MI355X"):                     # neighbours, and an empty one in between: only the device is wrong
        megacrn_amd.AdamW([base[:4], base[4:], base[2:2]])
    with pytest.raises(ValueError, match="lr and weight_decay"):
        megacrn_amd.AdamW([{"params": [torch.zeros(3)], "betas": (0.8, 0.9)}])


def test_trainer_and_command_options():
    from megacrn_amd.train import build_parser
    from megacrn_amd.trainer import FlatTrainer
    a = build_parser().parse_args([])
    assert (a.optimizer, a.state_bits) == ("adam", 32)
    with pytest.raises(ValueError):
        FlatTrainer(None, optimizer="sgd")
    with pytest.raises(ValueError):
        FlatTrainer(None, optimizer="adam", state_bits=8)


# ---------------------------------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------------------------------
SHAPES = [(1,), (63,), (64,), (65, 3), (), (0, 4), (1024,), (33, 77), (4100,), (2, 3, 5)]


def _make(shapes, dt, seed, off=0):
    """Parameters (views that start `off` elements behind an aligned address) and gradients of several magnitudes."""
    g = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for i, s in enumerate(shapes):
        n = int(np.prod(s))
        for out, scale in ((ps, 1.0), (gs, 10.0 ** (i % 4 - 3))):
            base = torch.empty(n + off, dtype=dt, device="cuda")
            v = base[off:].view(s)
            v.copy_((torch.randn(s, generator=g) * scale).to(dt))
            out.append(v)
    return ps, gs


def _piece(arena, opt, i):
    n = opt.params[i].numel()
    return arena[opt.offsets[i]:opt.offsets[i] + n].double().cpu().numpy()


def _padding_is_zero(opt):
    real = torch.zeros(opt.moments()[0].numel(), dtype=torch.bool, device="cuda")
    for p, o in zip(opt.params, opt.offsets):
        real[o:o + p.numel()] = True
    for t in (*opt.moments(), opt.master):
        assert t is None or not t[~real].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("clip", [0.0, 1.0, 1e9])
def test_32_bit_steps(dt, off, clip):
    """Five steps, each from the moments and parameters that the last one left, element by element within the bounds of the fp32 operations."""
    import megacrn_amd
    ps, gs = _make(SHAPES, dt, 3, off)
    opt = megacrn_amd.AdamW(ps, lr=3e-2, weight_decay=0.1, max_grad_norm=clip)
    for step in range(1, 6):
        if step == 3:
            gs = [None if i in (1, 6) else g * 0.5 for i, g in enumerate(gs)]
        before = [[_piece(a, opt, i) for a in opt.moments()] for i in range(len(ps))]
        pb = [(_piece(opt.master, opt, i) if opt.master is not None else p.detach().double().cpu().numpy().reshape(-1)) for i, p in enumerate(ps)]
        kept = [p.detach().clone() for p in ps]
        opt.step(grads=gs, grad_scale=0.5)
        factor = 0.5
        if clip:
            norm = 0.5 * np.sqrt(sum(float(g.double().pow(2).sum()) for g in gs if g is not None))
            assert abs(opt.total_norm.item() - norm) <= 1.01 * O.U * norm          # 64-bit sums, one rounding to fp32
            factor = 0.5 * min(1.0, clip / (norm + 1e-6))
        for i, (p, g) in enumerate(zip(ps, gs)):
            if g is None or g.numel() == 0:
                assert torch.equal(p, kept[i])
                assert all((a == b).all() for a, b in zip([_piece(a, opt, i) for a in opt.moments()], before[i]))
                continue
            s = opt.steps()[i]
            assert s == (step if i not in (1, 6) else min(step, 2))
            want = O.adamw_step(pb[i], g.double().cpu().numpy().reshape(-1), *before[i], s, 3e-2, 0.1, factor=factor)
            got = _piece(opt.master, opt, i) if opt.master is not None else p.detach().double().cpu().numpy().reshape(-1)
            for a, w, e in ((got, want[0], want[3]), (_piece(opt.moments()[0], opt, i), want[1], want[4]), (_piece(opt.moments()[1], opt, i), want[2], want[5])):
                assert (np.abs(a - w) <= e).all(), (step, i, np.max(np.abs(a - w) - e))
            if opt.master is not None:
                assert torch.equal(p.reshape(-1), opt.master[opt.offsets[i]:opt.offsets[i] + p.numel()].to(dt))
        _padding_is_zero(opt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip", [0.0, 1.0])
def test_8_bit_steps_code_by_code(dt, clip):
    """Three steps whose moments are the oracle's, code by code: the fp32 operations are the same ones, the rounding is exact."""
    import megacrn_amd
    ps, gs = _make(SHAPES, dt, 4, 1)
    opt = megacrn_amd.AdamW(ps, lr=1e-2, max_grad_norm=clip, state_bits=8, seed=123)
    for step in range(1, 4):
        old = [[_piece(a, opt, i) for a in opt.moments()] for i in range(len(ps))]
        opt.step(grads=gs)
        factor = F(1.0)
        if clip:
            norm = F(opt.total_norm.item())
            factor = min(F(1.0), F(clip) / (norm + F(1e-6)))
        d = opt.state_dict()
        for i, (p, g) in enumerate(zip(ps, gs)):
            n = g.numel()
            if not n:
                continue
            m, v = O.moments_f32(g.float().cpu().numpy().reshape(-1), old[i][0], old[i][1], factor)
            bits = O.random_bits(123, i, step, n)
            o, nb = opt.offsets[i], (n + 63) // 64
            for second, x, r in ((False, m, bits & 0xFFFF), (True, v, bits >> 16)):
                codes, scales = O.encode(x, r, second)
                key = "v" if second else "m"
                assert (d[key][o:o + n].cpu().numpy() == codes).all()
                assert (d[key + "_scale"][o // 64:o // 64 + nb].cpu().numpy() == scales).all()
                assert (_piece(opt.moments()[second], opt, i) == O.decode(codes, scales, second).astype(F)).all()
        _padding_is_zero(opt)


@pytest.mark.gpu
def test_8_bit_tracks_32_bit():
    """400 steps of gradients of constant variance, then 4000 of a tenth of it: v in 8 bits stays unbiased and decays as v in 32 bits
    does.  A step moves v by a share 1e-3 |g^2 / v - 1| (mean < 1e-3), between codes at most v / 8 apart, so its variance grows by at most
    1e-3 v^2 / 8 a step and forgets itself over 500: a spread of 25 % of v for an element, 25 % / 128 for the mean of 16384."""
    import megacrn_amd
    torch.manual_seed(0)
    n = 16384
    a, b = (torch.zeros(n, device="cuda") for _ in range(2))
    o32, o8 = megacrn_amd.AdamW([a], lr=0.0), megacrn_amd.AdamW([b], lr=0.0, state_bits=8, seed=1)
    for step in range(4400):
        g = torch.randn(n, device="cuda") * (1.0 if step < 400 else 0.1)
        o32.step(grads=[g])
        o8.step(grads=[g])
        if step in (399, 4399):
            v32, v8 = o32.moments()[1].double(), o8.moments()[1].double()
            assert abs((v8.sum() / v32.sum()).item() - 1) <= 6 * 0.25 / 128
            m32, m8 = o32.moments()[0].double(), o8.moments()[0].double()
            assert ((m8 - m32).norm() / m32.norm()).item() <= 0.25       # m forgets over 10 steps, each rounding spread by v's argument < 5 %


@pytest.mark.gpu
@pytest.mark.parametrize("count", [61, 150])
def test_more_tensors_than_a_launch_carries(count):
    import megacrn_amd
    shapes = [(1 + (7 * i) % 90,) for i in range(count)]
    ps, gs = _make(shapes, torch.float32, 5)
    qs = [p.clone() for p in ps]
    gs[60] = None
    opt = megacrn_amd.AdamW(ps, lr=1e-2, max_grad_norm=0.5)
    opt.step(grads=gs)
    norm = np.sqrt(sum(float(g.double().pow(2).sum()) for g in gs if g is not None))
    assert abs(opt.total_norm.item() - norm) <= 1.01 * O.U * norm
    for i, (p, q, g) in enumerate(zip(ps, qs, gs)):
        if g is None:
            assert torch.equal(p, q)
            continue
        z = np.zeros(g.numel())
        want = O.adamw_step(q.double().cpu().numpy(), g.double().cpu().numpy(), z, z, 1, 1e-2, 1e-2, factor=min(1.0, 0.5 / (norm + 1e-6)))
        assert (np.abs(p.double().cpu().numpy() - want[0]) <= want[3]).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count", [701, 900, 1500])
def test_many_small_tensors(count, dt):
    """As many sums as tensors, added by every block or (from 702 on) once: one norm, one factor for all."""
    import megacrn_amd
    shapes = [(1 + (7 * i) % 20,) for i in range(count)]
    ps, gs = _make(shapes, dt, 5)
    opt = megacrn_amd.AdamW(ps, lr=1e-2, max_grad_norm=0.5)
    before = torch.cat([p.double() for p in ps])
    opt.step(grads=gs)
    g = torch.cat([x.double() for x in gs])
    norm = g.norm().item()
    assert abs(opt.total_norm.item() - norm) <= 1.01 * O.U * norm
    z = np.zeros(g.numel())
    want = O.adamw_step(before.cpu().numpy(), g.cpu().numpy(), z, z, 1, 1e-2, 1e-2, factor=min(1.0, 0.5 / (norm + 1e-6)))
    got = ps if opt.master is None else [opt.master[o:o + p.numel()] for o, p in zip(opt.offsets, ps)]
    assert (np.abs(torch.cat([p.double() for p in got]).cpu().numpy() - want[0]) <= want[3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,bits,n", [(torch.float32, 32, 66_000_321), (torch.float32, 8, 27_000_321), (torch.bfloat16, 32, 9_000_321), (torch.bfloat16, 8, 130_000_321)])
def test_steps_that_stream_past_the_caches(dt, bits, n):
    """Steps that move more than 256 MB (the norm's gradients with the first and the last), an aligned tensor and one that is not: every element of two
    steps' parameters from zero moments against float64 on the device, the moments too; 8-bit codes of blocks all over the tensors against the
    oracle's.  Bounds: those of the oracle's step, which are elementwise in its operations."""
    import megacrn_amd
    gen = torch.Generator(device="cuda").manual_seed(n)
    ps, gs = [], []
    for k, off in ((n, 0), (n // 9, 1)):
        for lst, std in ((ps, 1.0), (gs, 1e-3)):
            lst.append((torch.randn(k + off, generator=gen, device="cuda") * std).to(dt)[off:])
    opt = megacrn_amd.AdamW(ps, lr=1e-2, max_grad_norm=1.0, state_bits=bits, seed=3)
    for step in (1, 2):
        old = [[a[o:o + p.numel()].double() for a in opt.moments()] for p, o in zip(ps, opt.offsets)]
        before = [(p if opt.master is None else opt.master[o:o + p.numel()]).double() for p, o in zip(ps, opt.offsets)]
        opt.step(grads=gs)
        norm = sum(g.double().pow(2).sum().item() for g in gs) ** 0.5
        assert norm > 1 and abs(opt.total_norm.item() - norm) <= 1.01 * O.U * norm
        f = 1.0 / (norm + 1e-6)
        for i, (p, g, o) in enumerate(zip(ps, gs, opt.offsets)):
            # O.adamw_step, its operations on device tensors
            x, k = g.double() * f, p.numel()
            big_m, v = 0.9 * old[i][0].abs() + 0.1 * x.abs(), 0.999 * old[i][1] + 0.001 * x * x
            m = 0.9 * old[i][0] + 0.1 * x
            em, ev = 5 * O.U * big_m + 2.0 ** -148, 7 * O.U * v + 2.0 ** -148
            c = (1 - 0.999 ** step) ** 0.5
            denom, size = v.sqrt() / c + 1e-8, 1e-2 / (1 - 0.9 ** step)
            upd = size * m / denom
            ed = torch.where(v > 2.0 ** -120, 0.5 * ev / v.clamp(min=2.0 ** -120).sqrt(), ev.sqrt()) / c + 4 * O.U * denom
            ep = size / denom * em + upd.abs() * ed / denom + 4 * O.U * upd.abs() + 3 * O.U * before[i].abs()
            got = (p if opt.master is None else opt.master[o:o + k]).double()
            assert not ((got - (before[i] * (1 - 1e-4) - upd)).abs() > ep).any(), (step, i)
            if opt.master is not None:
                assert torch.equal(p, opt.master[o:o + k].to(dt))
            if bits == 32:
                for a, w, e in zip(opt.moments(), (m, v), (em, ev)):
                    assert not ((a[o:o + k].double() - w).abs() > e).any(), (step, i)
                continue
            d, values = opt.state_dict(), opt.moments()
            F1 = F(opt.total_norm.item()) + F(1e-6)
            for b in [0, 1, k // 128, (k - 1) // 64 - 1, (k - 1) // 64] + list(range(7, k // 64, k // 64 // 20)):
                at, to = b * 64, min(b * 64 + 64, k)
                mm, vv = O.moments_f32(g[at:to].float().cpu().numpy(), old[i][0][at:to].cpu().numpy(), old[i][1][at:to].cpu().numpy(), F(1.0) / F1)
                key = O.mix(3 + 0x9E3779B9 * (i + 1) + O.mix(step))
                r = np.array([O.mix(q * 0x9E3779B9 + key) for q in range(at, to)], dtype=np.int64)
                for second, q, bits16 in ((False, mm, r & 0xFFFF), (True, vv, r >> 16)):
                    codes, scales = O.encode(q, bits16, second)
                    name = "v" if second else "m"
                    assert (d[name][o + at:o + to].cpu().numpy() == codes).all() and d[name + "_scale"][(o + at) // 64].item() == scales[0], (step, i, b)
                    assert (values[second][o + at:o + to].cpu().numpy() == O.decode(codes, scales, second).astype(F)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_large_tensor_and_groups(bits):
    """Blocks of several runs (over 4 M elements), two groups with rates and decays of their own, and the same numbers whichever way
    the elements are cut into tensors of whole blocks."""
    import megacrn_amd
    torch.manual_seed(1)
    n = 5 * 1024 * 1024 + 321
    w, g = torch.randn(n, device="cuda"), torch.randn(n, device="cuda") * 0.01
    small, gs = torch.randn(100, device="cuda"), torch.randn(100, device="cuda")
    p, q = w.clone(), small.clone()
    opt = megacrn_amd.AdamW([{"params": [p], "lr": 1e-3, "weight_decay": 0.0}, {"params": [q], "lr": 1e-1}], weight_decay=0.5,
                            max_grad_norm=1.0, state_bits=bits)
    opt.step(grads=[g, gs])
    norm = torch.cat([g, gs]).double().norm().item()
    assert abs(opt.total_norm.item() - norm) <= 1.01 * O.U * norm
    f = min(1.0, 1.0 / (norm + 1e-6))
    for got, x, gr, lr, wd in ((p, w, g, 1e-3, 0.0), (q, small, gs, 1e-1, 0.5)):
        z = np.zeros(x.numel())
        want = O.adamw_step(x.double().cpu().numpy(), gr.double().cpu().numpy(), z, z, 1, lr, wd, factor=f)
        assert (np.abs(got.double().cpu().numpy() - want[0]) <= want[3]).all()
    if bits == 32:
        cut = [w.clone()[a:b] for a, b in ((0, 4096), (4096, n))]
        other = megacrn_amd.AdamW(cut + [small.clone()], lr=1e-3, weight_decay=0.0, max_grad_norm=1.0)
        other.step(grads=[g[:4096], g[4096:], gs])
        assert torch.allclose(torch.cat(cut), p, rtol=0, atol=2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1.2e-38, 1e-30, 1e-20, 1e-12, 1e-10, 1e-8])
def test_small_eps_and_subnormal_moments(eps):
    """Gradients down to 1e-21, whose v is subnormal: its root is no 0 that the update would be divided by.  Three steps in 32 bits within the oracle's
    bounds."""
    import megacrn_amd
    g = torch.cat([torch.tensor([10.0 ** -(k / 4) for k in range(85)]), torch.zeros(3)]).cuda()
    w = torch.randn(g.numel(), device="cuda")
    opt = megacrn_amd.AdamW([w], lr=1e-2, eps=eps)
    for step in range(1, 4):
        before, mv = w.double().cpu().numpy(), [_piece(a, opt, 0) for a in opt.moments()]
        opt.step(grads=[g])
        want = O.adamw_step(before, g.double().cpu().numpy(), *mv, step, 1e-2, 1e-2, eps=eps)
        assert (np.abs(w.double().cpu().numpy() - want[0]) <= want[3]).all(), (step, (np.abs(w.double().cpu().numpy() - want[0]) / want[3]).max())


@pytest.mark.gpu
def test_not_finite_gradients():
    """Unclipped, a NaN or infinite gradient spoils its own element and, in 8 bits, no other of its block; clipped, the norm is not
    finite: NaN reaches every element, infinity its own (the others' factor is 0)."""
    import megacrn_amd
    for bits in (32, 8):
        ps, gs = _make([(200,)], torch.float32, 6)
        gs[0][70], gs[0][71] = float("nan"), float("inf")
        ref, rg = ps[0].clone(), gs[0].clone()
        rg[70:72] = 0
        opt, clean = megacrn_amd.AdamW(ps, state_bits=bits), megacrn_amd.AdamW([ref], state_bits=bits)
        opt.step(grads=gs)
        clean.step(grads=[rg])
        bad = torch.zeros(200, dtype=torch.bool, device="cuda")
        bad[70:72] = True
        assert torch.equal(~torch.isfinite(ps[0]), bad) and torch.equal(ps[0][~bad], ref[~bad])
        for x, y in zip(opt.moments(), clean.moments()):
            assert torch.equal(x[:200][~bad], y[:200][~bad]) and not torch.isfinite(x[:200][bad]).any()
        ps, gs = _make([(200,), (5,)], torch.float32, 6)
        gs[0][70] = float("nan")
        opt = megacrn_amd.AdamW(ps, state_bits=bits, max_grad_norm=1.0)
        opt.step(grads=gs)
        assert torch.isnan(opt.total_norm) and all(torch.isnan(p).all() for p in ps)
        _padding_is_zero(opt)


@pytest.mark.gpu
def test_grad_attribute_views_and_errors():
    import megacrn_amd
    p = [torch.nn.Parameter(torch.randn(8, 6, device="cuda")) for _ in range(3)]
    opt = megacrn_amd.AdamW(p, lr=1e-2)
    ref = [q.detach().clone() for q in p]
    p[0].grad = torch.randn(6, 8, device="cuda").t()                     # not contiguous
    p[2].grad = torch.randn(8, 6, device="cuda")
    opt.step()
    assert opt.steps() == [1, 0, 1] and torch.equal(p[1], ref[1])
    z = np.zeros(48)
    for i in (0, 2):
        want = O.adamw_step(ref[i].double().cpu().numpy().reshape(-1), p[i].grad.double().cpu().numpy().reshape(-1), z, z, 1, 1e-2, 1e-2)
        assert (np.abs(p[i].detach().double().cpu().numpy().reshape(-1) - want[0]) <= want[3]).all()
    opt.zero_grad()
    assert all(q.grad is None for q in p)
    opt.step()                                                            # nothing to do
    assert opt.steps() == [1, 0, 1]
    with pytest.raises(ValueError):
        opt.step(grads=[None])
    for bad in (torch.randn(8, 5, device="cuda"), torch.randn(8, 6), torch.randn(8, 6, device="cuda", dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            opt.step(grads=[bad, None, None])
    with pytest.raises(RuntimeError):
        opt.step(grads=[p[0].detach(), None, None], grad_scale=0.0)
    assert opt.steps() == [1, 0, 1]
    d = opt.state_dict()
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step(grads=[None, None, p[2].detach().clone()])
    opt.param_groups[0]["lr"] = 1e-2
    for broken in (dict(d, state_bits=8), dict(d, m=d["m"][:-1]), dict(d, steps=[1]), dict(d, groups=[]), dict(d, steps=[1, -1, 1])):
        with pytest.raises(ValueError):
            opt.load_state_dict(broken)


@pytest.mark.gpu
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_elements(bits, capturable):
    """Alone they make a step that does nothing; beside others they have no updates, whoever counts."""
    import megacrn_amd
    e, p = torch.zeros(0, 4, device="cuda"), torch.ones(5, device="cuda")
    opt = megacrn_amd.AdamW([e], state_bits=bits, max_grad_norm=1.0, capturable=capturable)
    opt.step(grads=[torch.zeros_like(e)])
    assert opt.steps() == [0] and all(t.numel() == 0 for t in opt.moments())
    opt.load_state_dict(opt.state_dict())
    opt = megacrn_amd.AdamW([e, p], state_bits=bits, max_grad_norm=1.0, capturable=capturable)
    for _ in range(2):
        opt.step(grads=[torch.zeros_like(e), torch.ones_like(p)])
    assert opt.steps() == [0, 2] and (p < 1).all()


@pytest.mark.gpu
def test_rates_that_change_in_place_and_fixed_constants():
    """A rate held in a tensor is read at each step, whatever happened to it in place; betas and eps cannot be set without effect."""
    import megacrn_amd
    p, q = torch.ones(70, device="cuda"), torch.ones(70, device="cuda")
    g = torch.full_like(p, 0.5)
    a, b = megacrn_amd.AdamW([p], lr=1e-2), megacrn_amd.AdamW([q], lr=1e-2)
    rate = torch.tensor(1e-2, dtype=torch.float64)
    a.param_groups[0]["lr"] = rate
    for lr in (1e-2, 3e-3, 0.0):
        rate.fill_(lr)
        b.param_groups[0]["lr"] = lr
        a.step(grads=[g]), b.step(grads=[g])
        assert torch.equal(p, q)
    for name, value in (("betas", (0.5, 0.9)), ("eps", 1e-3)):
        with pytest.raises(AttributeError):
            setattr(a, name, value)
    assert a.betas == (0.9, 0.999) and a.eps == 1e-8


@pytest.mark.gpu
def test_a_norm_that_is_no_number_is_refused():
    """Set later, it would switch the clipping off."""
    import megacrn_amd
    p = torch.ones(5, device="cuda")
    opt = megacrn_amd.AdamW([p], max_grad_norm=1.0)
    opt.max_grad_norm = float("nan")
    with pytest.raises(RuntimeError, match="max_norm"):
        opt.step(grads=[torch.ones_like(p)])
    assert opt.steps() == [0] and (p == 1).all()


@pytest.mark.gpu
def test_dual_tensors_are_refused():
    import megacrn_amd
    from torch.autograd import forward_ad
    p, g = torch.ones(5, device="cuda"), torch.ones(5, device="cuda")
    opt = megacrn_amd.AdamW([p])
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward gradient"):
            opt.step(grads=[forward_ad.make_dual(g, torch.ones_like(g))])
    assert opt.steps() == [0] and (p == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_resumed_and_captured_runs(bits, dt):
    """A run that is saved and resumed, and one whose step is captured and replayed, give the numbers of the uninterrupted eager run bit for bit."""
    import megacrn_amd
    kw = dict(lr=1e-2, max_grad_norm=1.0, state_bits=bits, seed=9)
    shapes = [(100, 7), (3,), (2000,)]
    ps, _ = _make(shapes, dt, 8)
    grads = [_make(shapes, dt, 100 + k)[1] for k in range(6)]
    qs, rs = [p.clone() for p in ps], [p.clone() for p in ps]
    opt = megacrn_amd.AdamW(ps, **kw)
    for g in grads:
        opt.step(grads=g)
    first = megacrn_amd.AdamW(qs, **kw)
    for g in grads[:3]:
        first.step(grads=g)
    second = megacrn_amd.AdamW(qs, **dict(kw, lr=5.0, seed=77))
    second.load_state_dict(first.state_dict())
    for g in grads[3:]:
        second.step(grads=g)
    cap = megacrn_amd.AdamW(rs, capturable=True, **kw)
    static = [g.clone() for g in grads[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cap.step(grads=static)                                            # the first step, eager
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap.step(grads=static)
    for g in grads[1:]:
        for s, t in zip(static, g):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
    assert cap.steps() == opt.steps() == second.steps() == [6] * 3
    for a, b, c in zip(ps, qs, rs):
        assert torch.equal(a, b) and torch.equal(a, c)
    for a, b, c in zip(opt.moments(), second.moments(), cap.moments()):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert torch.equal(opt.total_norm, cap.total_norm)
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(grads=grads[0])
    torch.cuda.synchronize()
    opt.step(grads=grads[0])                                              # eager work goes on


@pytest.mark.gpu
@pytest.mark.parametrize("capturable", [False, True])
def test_copied_optimizer(capturable):
    """A deep copy (parameters included) goes on by itself: its steps are the original's, and leave the original alone."""
    import copy
    import megacrn_amd
    ps, gs = _make([(65, 3), (4100,)], torch.bfloat16, 9)
    opt = megacrn_amd.AdamW(ps, lr=1e-2, state_bits=8, max_grad_norm=1.0, capturable=capturable)
    opt.step(grads=gs)
    twin = copy.deepcopy(opt)
    assert all(a is b for a, b in zip(twin.params, twin.param_groups[0]["params"]))
    before = [p.clone() for p in ps]
    twin.step(grads=gs)
    assert opt.steps() == [1, 1] and twin.steps() == [2, 2] and all(torch.equal(p, q) for p, q in zip(ps, before))
    opt.step(grads=gs)
    assert opt.steps() == [2, 2] and all(torch.equal(p, q) for p, q in zip(ps, twin.params))
    assert all(torch.equal(x, y) for x, y in zip(opt.moments(), twin.moments()))


@pytest.mark.gpu
def test_masters_follow_a_loaded_model():
    import megacrn_amd
    p = torch.randn(100, device="cuda").to(torch.bfloat16)
    opt = megacrn_amd.AdamW([p], lr=1e-3, weight_decay=0.0)
    p.copy_(torch.ones(100, device="cuda"))
    opt.sync_masters()
    opt.step(grads=[torch.ones_like(p)])
    assert (opt.master[:100] - (1 - 1e-3)).abs().max() <= 4 * O.U and opt.master[100:].abs().max() == 0


@pytest.mark.gpu
def test_wide_range_of_moments_in_8_bits():
    """Gradients of one block over 36 octaves, the smallest and largest that fp32 squares hold, and zeros: codes against the oracle."""
    import megacrn_amd
    g = torch.cat([torch.tensor([2.0 ** (k - 30) for k in range(36)]), torch.zeros(28), torch.tensor([1e-30, 1e-23, 1e-19, 0.0] * 16),
                   torch.tensor([1e18, 3e18, 1.0, 1e-3] * 16), torch.full((64,), 1e-38)]).cuda()
    opt = megacrn_amd.AdamW([torch.zeros_like(g)], state_bits=8, seed=5)
    for step in (1, 2, 3):
        old = [_piece(a, opt, 0) for a in opt.moments()]
        opt.step(grads=[g])
        m, v = O.moments_f32(g.cpu().numpy(), *old, F(1.0))
        bits = O.random_bits(5, 0, step, g.numel())
        d = opt.state_dict()
        for key, x, r, second in (("m", m, bits & 0xFFFF, False), ("v", v, bits >> 16, True)):
            codes, scales = O.encode(x, r, second)
            assert (d[key].cpu().numpy() == codes).all() and (d[key + "_scale"].cpu().numpy() == scales).all()
            assert ((codes > 0) | (x == 0)).all() or not second                # a v above 0 never gets code 0
    assert torch.isfinite(opt.params[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_flat_trainer_with_adamw(bits):
    """FlatTrainer(optimizer="adamw"): two steps; the second's parameters against float64 AdamW on the trainer's own gradients and moments."""
    import megacrn_amd
    from megacrn_amd.trainer import FlatTrainer
    N, T, H, M, D, B = 17, 3, 16, 5, 8, 4
    model = megacrn_amd.MegaCRN(N, 1, 1, T, H, mem_num=M, mem_dim=D)
    model.load_state_dict({k: torch.from_numpy(v) for k, v in MO.init_params(N, rnn_units=H, mem_num=M, mem_dim=D, seed=2).items()})
    model = model.cuda().train()
    model._teacher_flags = lambda labels, bs: [False] * T
    tr = FlatTrainer(model, lr=0.01, eps=1e-3, max_grad_norm=0.1, scaler_mean=SC_MEAN, scaler_std=SC_STD, autotune=False,
                     optimizer="adamw", weight_decay=0.2, state_bits=bits)
    torch.manual_seed(4)
    x, yc, y = (torch.randn(B, T, N, 1, device="cuda") for _ in range(3))
    tr.train_step(x, yc, y)
    before = [p.detach().double().cpu().numpy().reshape(-1) for p in tr.params]
    mv = [[_piece(a, tr.opt, i) for a in tr.opt.moments()] for i in range(len(tr.params))]
    tr.lr = 0.02
    loss = tr.train_step(x, yc, y)
    assert torch.isfinite(loss)
    norm = np.sqrt(sum(float(g.double().pow(2).sum()) for g in tr._gviews))
    assert abs(tr.total_norm.item() - norm) <= 1.01 * O.U * norm and norm > 0.1
    for i, (p, g) in enumerate(zip(tr.params, tr._gviews)):
        want = O.adamw_step(before[i], g.double().cpu().numpy().reshape(-1), *mv[i], 2, 0.02, 0.2, eps=1e-3, factor=0.1 / (norm + 1e-6))
        assert (np.abs(p.detach().double().cpu().numpy().reshape(-1) - want[0]) <= want[3]).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("bits", ["32", "8"])
def test_train_command_with_adamw(bits, tmp_path):
    from megacrn_amd import train
    np.random.seed(0); torch.manual_seed(0)
    hist = train.main(["--synthetic", "48", "--num_nodes", "13", "--rnn_units", "16", "--mem_num", "6", "--mem_dim", "8", "--batch_size", "16",
                       "--epochs", "2", "--seed", "0", "--save_dir", str(tmp_path), "--seq_len", "4", "--horizon", "4",
                       "--optimizer", "adamw", "--state_bits", bits, "--weight_decay", "0.05"])
    assert len(hist) == 2 and all(np.isfinite(v) for row in hist for v in row)
    assert list(tmp_path.glob("*/MegaCRN.pt"))
