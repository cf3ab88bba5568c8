"""AdamW (pin_adamw_step) against the formula in 64 bits, step by step from the state the kernel left.

Tolerances of one step from given parameters, moments and gradients, u = 2^-24 (half a step of f32):
  m: each product and the sum round once and the factors are rounded once: 3 u (|b1 m| + |c1 g|); v: 4 u of its size.
  p: with d = lr/(1 - b1^t) m / (sqrt v / sqrt(1 - b2^t) + eps), m is off by 3 u (|b1 m| + |c1 g|), sqrt v by 2 u, the
  square root, two divisions, a sum, a product and the three rounded scalars add 8 u: 10 u |d| and m's part.  With 8 bits
  v's and m's own rounding to f32 is u / 2 and u, the square root and the reciprocal of one unit in the last place are 2 u
  each, the fma, its factor, eps and two products u each, the three scalars 3 u (the second is inverted: u more): 13.5 u.
  14 u |d| covers both; p (1 - lr wd) adds 2 u |p|, the difference u |p'|.  A 16-bit parameter adds half its step.
  Averages that 32 bits cannot hold (a square beyond 3.4e38) are infinite with 32 bits and themselves with 8.
The 8-bit codes are whole numbers and have to be equal: the averages are formed in 64 bits, and a last-bit difference there
reaches a code with a probability of 2^-32 per element."""
import copy
import math

import numpy as np
import pytest
import torch

import pin_slam_amd as P
from tests.adamw_codes import BLOCK, decode, dither, encode

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HYPER = dict(lr=0.02, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return "cuda"


def np64(t):
    return t.detach().double().cpu().numpy()


def snapshot(opt, gi=0):
    """Parameters, moments and copies of a group in 64 bits, tensor by tensor."""
    group = opt.param_groups[gi]
    opt._arena(gi)
    m, v = (np64(x) for x in opt.moments(gi))
    w = opt.master(gi)
    out = []
    for p, a in zip(group["params"], opt.offsets(gi)):
        n = p.numel()
        base = np64(p).reshape(-1) if w is None or p.dtype == torch.float32 else np64(w[a:a + n])
        out.append((base, m[a:a + n], v[a:a + n]))
    return out


def check_step(opt, t, gi=0, grads=None):
    """One step of a group against the formula; t: the step's number for each of its parameters."""
    group = opt.param_groups[gi]
    (b1, b2), lr, eps, wd = group["betas"], float(group["lr"]), group["eps"], group["weight_decay"]
    before = snapshot(opt, gi)
    codes = [{k: s.clone() for k, s in opt.state[p].items()} for p in group["params"]]
    opt.step()
    torch.cuda.synchronize()
    after = snapshot(opt, gi)
    t = t if isinstance(t, (list, tuple)) else [t] * len(before)
    for i, (p, (p0, m0, v0), (p1, m1, v1)) in enumerate(zip(group["params"], before, after)):
        if p.grad is None:
            assert np.array_equal(p0, p1) and np.array_equal(m0, m1) and np.array_equal(v0, v1)
            continue
        g = np64(p.grad).reshape(-1)
        if group["state_bits"] == 8:   # from the codes: the moments in 64 bits, not their f32 values
            m0, v0 = decode(codes[i]["exp_avg"].cpu().numpy().reshape(-1), codes[i]["exp_avg_sq"].cpu().numpy().reshape(-1),
                            codes[i]["exponents"].cpu().numpy())
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        if group["state_bits"] == 32:
            tol_m = 3 * U * (np.abs(b1 * m0) + np.abs((1 - b1) * g)) + 1e-44
            assert (np.abs(m1 - m) <= tol_m).all(), float(np.max(np.abs(m1 - m) - tol_m))
            over = v >= float(np.finfo(np.float32).max)   # more than the state can hold: infinite
            assert np.isinf(v1[over]).all() and (np.abs(v1[~over] - v[~over]) <= 4 * U * v[~over] + 1e-44).all()
        else:
            a = opt.offsets(gi)[i]
            dm, dv = dither(a + np.arange(g.size), t[i], opt.seed, gi)
            em, ev, exps = encode(m, v, dm, dv)
            st = opt.state[p]
            np.testing.assert_array_equal(st["exponents"].cpu().numpy(), exps)
            np.testing.assert_array_equal(st["exp_avg"].cpu().numpy().reshape(-1), em)
            np.testing.assert_array_equal(st["exp_avg_sq"].cpu().numpy().reshape(-1), ev)
        with np.errstate(over="ignore"):
            m32, v32 = m.astype(np.float32).astype(np.float64), v.astype(np.float32).astype(np.float64)
            if group["state_bits"] == 8:
                m32, v32 = m, v
        den = np.sqrt(v32 / (1 - b2 ** t[i])) + eps
        with np.errstate(all="ignore"):
            d = lr / (1 - b1 ** t[i]) * np.where(m32 == 0, 0.0, m32 / den)
            off = lr / (1 - b1 ** t[i]) * 3 * U * (np.abs(b1 * m0) + np.abs((1 - b1) * g)) / den
        want = p0 * (1 - lr * wd) - d
        tol = 14 * U * np.abs(d) + np.nan_to_num(off) + 2 * U * np.abs(p0) + U * np.abs(want) + 1e-44
        if p.dtype == torch.float32 or group["master_weights"]:
            bad = np.abs(p1 - want) > tol
            assert not bad.any(), (i, float(np.max(np.abs(p1 - want) - tol)), int(bad.sum()))
        if p.dtype != torch.float32:
            half, least = torch.finfo(p.dtype).eps / 2, {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[p.dtype]
            got = np64(p).reshape(-1)
            if group["master_weights"]:
                assert np.array_equal(got, np64(opt.state[p]["master"].to(p.dtype)).reshape(-1))
            else:
                assert (np.abs(got - want) <= tol * (1 + half) + half * np.abs(want) + least).all()


def tensors(sizes, kind, dev, seed=0, shift=0):
    """Parameters of these sizes; shift: each lies that many elements behind an aligned place."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        buf = torch.randn((n + shift,), generator=g).to(kind).to(dev)
        out.append(torch.nn.Parameter(buf[shift:]))
    return out


def set_grads(params, seed, scale=1.0, some=None, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    for i, p in enumerate(params):
        x = torch.randn(p.shape, generator=g) * torch.exp(2 * torch.randn(p.shape, generator=g)) * scale
        p.grad = None if some is not None and i not in some else x.to(p.dtype).to(p.device)


SIZES = [1, 3, 4, 5, 64, 255, 256, 257, 833, 1000, 1023, 1024, 1025, 2049, 5000, 70001]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,master", [("f32", False), ("f16", False), ("bf16", False), ("f16", True), ("bf16", True)])
def test_steps_match_the_formula(dev, bits, kind, master):
    params = tensors(SIZES, TYPES[kind], dev)
    opt = P.AdamW(params, state_bits=bits, master_weights=master, **HYPER)
    for t in range(1, 5):
        set_grads(params, t)
        check_step(opt, t)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_alignments(dev, bits, shift):
    for kind in TYPES.values():
        params = tensors([7, 256, 1030, 4097], kind, dev, shift=shift)
        opt = P.AdamW(params, state_bits=bits, **HYPER)
        for t in (1, 2):
            set_grads(params, t)
            for p in params:   # gradients at other alignments still
                buf = torch.zeros((p.numel() + 5 - shift,), dtype=kind, device=dev)
                buf[5 - shift:] = p.grad
                p.grad = buf[5 - shift:]
            check_step(opt, t)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_lies_around_stays(dev, bits):
    """Elements before and behind a parameter, and the state behind a tensor, are left as they were."""
    buf = torch.full((5000,), 7.0, device=dev)
    p = torch.nn.Parameter(buf[1001:2004])
    opt = P.AdamW([p], state_bits=bits, **HYPER)
    for t in (1, 2):
        p.grad = torch.ones_like(p)
        opt.step()
    assert bool((buf[:1001] == 7).all()) and bool((buf[2004:] == 7).all()) and not bool((buf[1001:2004] == 7).any())
    arena = opt._arena(0)
    assert not bool(arena.m[1003:].any()) and not bool(arena.v[1003:].any())


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_shapes(dev, bits):
    """More tensors than one launch takes, empty ones among them, gradients that come and go."""
    sizes = [(i * 37) % 700 for i in range(260)]
    params = tensors(sizes, torch.float32, dev)
    params[3] = torch.nn.Parameter(params[3].detach().clone().view(3, -1))
    opt = P.AdamW(params, state_bits=bits, **HYPER)
    count = [0] * len(params)
    for t in range(3):
        some = {i for i in range(len(params)) if t == 0 or i % (t + 1) == 0}
        set_grads(params, t, some=some)
        count = [c + (i in some) for i, c in enumerate(count)]
        check_step(opt, count)


def test_groups(dev):
    """Groups of other rates, types and widths of state step as each would alone."""
    def build():
        return [tensors([500, 33], torch.float32, dev, 1), tensors([1000], torch.bfloat16, dev, 2),
                tensors([300, 7], torch.float32, dev, 3) + tensors([300], torch.float16, dev, 4)]

    kinds = [dict(lr=0.1, weight_decay=0.5), dict(betas=(0.8, 0.999), state_bits=8, master_weights=True),
             dict(eps=1e-3, master_weights=True)]
    together, alone = build(), build()
    opt = P.AdamW([dict(params=p, **k) for p, k in zip(together, kinds)], **HYPER)
    single = [P.AdamW([dict(params=p, **k)], **HYPER) for p, k in zip(alone, kinds)]
    for t in range(1, 4):
        for i, (a, b) in enumerate(zip(together, alone)):
            set_grads(a, 10 * t + i)
            set_grads(b, 10 * t + i)
        opt.step()
        for s in single:
            s.step()
    for i in (0, 2):   # the 8-bit group's rounding goes by its place among the groups
        for a, b in zip(together[i], alone[i]):
            assert torch.equal(a, b)
    for a, b in zip(together[1], alone[1]):
        torch.testing.assert_close(a.float(), b.float(), rtol=0.05, atol=0.02)


def test_like_torch(dev):
    """torch.optim.AdamW on the same run: the same formula, other roundings (2e-6 of the parameters after 20 steps)."""
    mine, theirs = tensors([4097, 64, 1], torch.float32, dev), tensors([4097, 64, 1], torch.float32, dev)
    a = P.AdamW(mine, **HYPER)
    b = torch.optim.AdamW(theirs, foreach=False, **HYPER)
    sched = [torch.optim.lr_scheduler.ExponentialLR(o, 0.9) for o in (a, b)]
    for t in range(20):
        set_grads(mine, t)
        set_grads(theirs, t)
        for o, s in ((a, sched[0]), (b, sched[1])):
            o.step()
            s.step()
    for p, q in zip(mine, theirs):
        torch.testing.assert_close(p, q, rtol=2e-6, atol=2e-6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e-4, 1e10, 1e18])
def test_gradients_of_any_size(dev, bits, scale):
    """Down to where squares underflow f32, up to where they nearly overflow it."""
    params = tensors([2049], torch.float32, dev)
    opt = P.AdamW(params, state_bits=bits, lr=0.01, betas=(0.9, 0.99), eps=1e-15)
    for t in (1, 2, 3):
        set_grads(params, t, scale)
        params[0].grad[::5] = 0
        check_step(opt, t)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients(dev, bits):
    """Moments of zero leave the parameter to its decay alone, also with eps 0 elsewhere in the block."""
    p = tensors([1000], torch.float32, dev)[0]
    opt = P.AdamW([p], state_bits=bits, **HYPER)
    p0 = p.detach().clone()
    p.grad = torch.zeros_like(p)
    p.grad[700:] = 1.0
    for _ in range(3):
        opt.step()
    decay = np.float32(1 - HYPER["lr"] * HYPER["weight_decay"])
    want = p0[:700].cpu().numpy()
    for _ in range(3):
        want = want * decay
    assert np.array_equal(p.detach()[:700].cpu().numpy(), want)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,master", [("f32", False), ("bf16", True)])
@pytest.mark.parametrize("betas,eps,steps", [((0.9, 0.0), 1e-8, 3), ((0.9, 0.0), 1e-15, 3), ((0.9, 0.5), 1e-8, 420),
                                             ((0.99, 0.9), 1e-8, 2300), ((0.9, 0.5), 1e-15, 420)])
def test_gradients_that_stop(dev, bits, kind, master, betas, eps, steps):
    """Steps without a gradient after one with: the second moment goes faster than the first, to zero at once where
    beta2 is 0, and what is left of the step goes by eps."""
    params = tensors([1000, 300], TYPES[kind], dev)
    opt = P.AdamW(params, state_bits=bits, master_weights=master, lr=1e-12, betas=betas, eps=eps, weight_decay=0.1)
    set_grads(params, 1)
    check_step(opt, 1)
    for p in params:
        p.grad.zero_()
    t = 1
    while t < steps:
        at = min(steps, t + 1 if t < 3 else 2 * t)
        for _ in range(at - t - 1):
            opt.step()
        t = at
        check_step(opt, t)
    assert all(bool(torch.isfinite(p).all()) for p in params)


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-15, 1.0])
@pytest.mark.parametrize("small", [1e-9, 1e-20, 1e-25, 1e-30])
def test_tiny_gradients_beside_large_ones(dev, eps, small):
    """One block, gradients far apart: with 8 bits the averages are formed in 64 bits, and so is the step where 32 would
    not hold what it is made of."""
    p = tensors([700], torch.float32, dev)[0]
    opt = P.AdamW([p], state_bits=8, lr=0.01, betas=(0.9, 0.99), eps=eps)
    for t in (1, 2):
        p.grad = torch.full_like(p, small) * (1 + torch.arange(700, device=dev) % 7)
        p.grad[17], p.grad[300], p.grad[301] = 1e6, 1e12, -1e-3
        check_step(opt, t)


def test_untouched_elements_without_eps(dev):
    """eps 0 and moments of zero: 0/0, not a number, as the formula has it; elements with a gradient step as ever."""
    for bits in (32, 8):
        p = tensors([600], torch.float32, dev)[0]
        opt = P.AdamW([p], state_bits=bits, lr=0.01, betas=(0.9, 0.99), eps=0.0)
        p.grad = torch.ones_like(p)
        p.grad[::3] = 0
        p0 = p.detach().clone()
        opt.step()
        zero = torch.zeros_like(p, dtype=torch.bool)
        zero[::3] = True
        assert torch.equal(torch.isnan(p), zero)
        torch.testing.assert_close(p.detach()[~zero], p0[~zero] - 0.01, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_not_a_number_stays_in_its_place(dev, bits):
    p = tensors([1500], torch.float32, dev)[0]
    opt = P.AdamW([p], state_bits=bits, **HYPER)
    set_grads([p], 1)
    p.grad[10], p.grad[300], p.grad[301] = math.nan, math.inf, -math.inf
    opt.step()
    for t in range(2):
        set_grads([p], 2 + t)
        opt.step()
    bad = torch.isnan(p.detach()).nonzero()[:, 0].tolist()
    assert bad == [10, 300, 301]
    m, v = opt.moments()
    for x in (m, v):
        assert (~torch.isfinite(x)).nonzero()[:, 0].tolist() == [10, 300, 301]


def test_positive_second_moment_never_zero(dev):
    """One huge gradient in the block, tiny ones beside it: nothing divides by zero, no step is out of measure."""
    p = torch.nn.Parameter(torch.zeros(256, device=dev))
    opt = P.AdamW([p], state_bits=8, lr=0.01, betas=(0.9, 0.99), eps=0.0)
    p.grad = torch.full_like(p, 1e-9)
    p.grad[17] = 1e6
    for t in range(50):
        before = p.detach().clone()
        opt.step()
        assert bool((opt.state[p]["exp_avg_sq"] > 0).all())
        # |m| is at most 2^(E_m+1) and one code's step more, sqrt v at least 2^(E_v/2-15): with both from one element of
        # 1e6 a step is below lr * 4
        assert float((p.detach() - before).abs().max()) <= 0.04


def test_rounding_keeps_the_average(dev):
    """Gradients that stay the same: the moments go to them (to nearest they would not move at all).  Codes are at most
    1/8 apart; the rounding's error of a step has a standard deviation of sqrt(f (1 - f)) / 8 of the value, f the place
    between two codes, and the average over 32768 elements of a stationary error of at most 0.25 of the value is within
    0.25 / sqrt(32768) * 5 = 0.7 %."""
    n = 32768
    p = torch.nn.Parameter(torch.zeros(n, device=dev))
    opt = P.AdamW([p], state_bits=8, lr=0.0, betas=(0.9, 0.99), eps=1e-8, seed=3)
    g = torch.full((n,), 0.7, device=dev)
    p.grad = g
    for t in range(400):
        opt.step()
        if t + 1 in (20, 100, 400):
            m, v = opt.moments()
            assert float(m.double().mean()) == pytest.approx(0.7 * (1 - 0.9 ** (t + 1)), rel=0.007)
            assert float(v.double().mean()) == pytest.approx(0.49 * (1 - 0.99 ** (t + 1)), rel=0.007)


def test_same_bits_every_time(dev):
    for bits in (32, 8):
        runs = []
        for seed in (1, 1, 2):
            params = tensors([5000, 77], torch.float32, dev)
            opt = P.AdamW(params, state_bits=bits, seed=seed, **HYPER)
            for t in range(5):
                set_grads(params, t)
                opt.step()
            runs.append([p.detach() for p in params] + list(opt.moments()))
        assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
        assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[2])) == (bits == 32)


@pytest.mark.parametrize("bits,master", [(32, False), (32, True), (8, False), (8, True)])
def test_saved_and_loaded(dev, bits, master, tmp_path):
    """A run that goes on from a checkpoint makes the steps of the one that was not interrupted."""
    kind = torch.bfloat16 if master else torch.float32
    a = tensors([1000, 33, 4], kind, dev)
    opt = P.AdamW(a, state_bits=bits, master_weights=master, **HYPER)
    for t in range(3):
        set_grads(a, t, some={0, 1} if t == 1 else None)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = P.AdamW(b, state_bits=bits, master_weights=master, lr=0.5)
    other.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    assert other.param_groups[0]["lr"] == HYPER["lr"] and other.state_dict()["state"][2]["step"] == 2
    for t in range(3, 6):
        for params, o in ((a, opt), (b, other)):
            set_grads(params, t)
            o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    for x, y in zip(opt.moments(), other.moments()):
        assert torch.equal(x, y)


def test_load_refuses_what_does_not_fit(dev):
    p = tensors([300], torch.float32, dev)
    opt = P.AdamW(p, state_bits=8, **HYPER)
    set_grads(p, 1)
    opt.step()
    saved = opt.state_dict()
    with pytest.raises(ValueError, match="state_bits"):
        P.AdamW(tensors([300], torch.float32, dev), **HYPER).load_state_dict(saved)
    with pytest.raises(ValueError, match="groups"):
        P.AdamW(tensors([300, 2], torch.float32, dev), state_bits=8).load_state_dict(saved)
    with pytest.raises(ValueError, match="exp_avg"):
        P.AdamW(tensors([301], torch.float32, dev), state_bits=8).load_state_dict(saved)
    worse = {**saved, "param_groups": [{**saved["param_groups"][0], "betas": (0.9, 1.0)}]}
    with pytest.raises(ValueError, match="betas"):
        opt.load_state_dict(worse)
    assert opt.param_groups[0]["betas"] == HYPER["betas"] and opt.state_dict()["state"][0]["step"] == 1   # as it was
    bad = copy.copy(saved)
    bad["state"] = {0: {**saved["state"][0], "exponents": saved["state"][0]["exponents"][:1]}}
    with pytest.raises(ValueError, match="exponents"):
        P.AdamW(tensors([300], torch.float32, dev), state_bits=8).load_state_dict(bad)


def test_hooks_of_saving_and_loading(dev):
    """torch's hooks see what they see of its own optimisers: the whole saved state, the state to load before it is taken
    (and may put another in its place), the optimiser after."""
    def build():
        p = tensors([300, 20], torch.float32, dev)
        return p, P.AdamW(p, state_bits=8, **HYPER)

    a, opt = build()
    set_grads(a, 1)
    opt.step()
    seen = []
    opt.register_state_dict_pre_hook(lambda o: seen.append(("save", o)))

    def after(o, saved):
        seen.append(("saved", [s["step"] for s in saved["state"].values()]))
        return {**saved, "extra": 7}

    opt.register_state_dict_post_hook(after)
    saved = opt.state_dict()
    assert seen == [("save", opt), ("saved", [1, 1])] and saved["extra"] == 7
    assert all("step" not in opt.state[p] for p in a)
    b, other = build()
    calls = []

    def before(o, d):
        calls.append(o)
        assert d is not saved and d["extra"] == 7
        groups = [{**g, "lr": 0.5} for g in d["param_groups"]]
        return {**d, "param_groups": groups}

    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(lambda o: calls.append(o.param_groups[0]["lr"]))
    other.load_state_dict(saved)
    assert calls == [other, 0.5] and saved["param_groups"][0]["lr"] == HYPER["lr"]
    assert all(torch.equal(x, y) for x, y in zip(opt.moments(), other.moments()))
    copied = copy.deepcopy(other)
    copied.load_state_dict(copied.state_dict())   # (a copy has no hooks)
    assert len(calls) == 2


def test_load_names_what_another_optimisers_state_lacks(dev):
    p = tensors([300], torch.float32, dev)
    set_grads(p, 1)
    opt = P.AdamW(p, **HYPER)
    theirs = torch.optim.AdamW(tensors([300], torch.float32, dev), foreach=False)
    theirs.param_groups[0]["params"][0].grad = torch.ones(300, device=dev)
    theirs.step()
    with pytest.raises(ValueError, match="state_bits"):
        opt.load_state_dict(theirs.state_dict())
    opt.step()
    saved = opt.state_dict()
    for bad in ({}, {"state": {}}, {"param_groups": saved["param_groups"]}):
        with pytest.raises(ValueError, match="param_groups"):
            opt.load_state_dict(bad)
    with pytest.raises(ValueError, match="betas"):
        opt.load_state_dict({**saved, "param_groups": [{k: v for k, v in saved["param_groups"][0].items() if k != "betas"}]})
    with pytest.raises(ValueError, match="step"):
        opt.load_state_dict({**saved, "state": {0: {k: v for k, v in saved["state"][0].items() if k != "step"}}})
    assert opt.state_dict()["state"][0]["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(dev, bits):
    """A captured step counts on: replays with new gradients and a new lr equal eager steps of another optimiser."""
    a, b = tensors([5000, 257], torch.float32, dev), tensors([5000, 257], torch.float32, dev)
    lr = torch.tensor([0.02], device=dev)
    hyper = {**HYPER, "lr": lr}
    opt = P.AdamW(a, state_bits=bits, capturable=True, **hyper)
    ref = P.AdamW(b, state_bits=bits, **{**HYPER, "lr": float(lr)})
    for params in (a, b):
        set_grads(params, 0)
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for t in range(1, 5):
        for params in (a, b):
            kept = [p.grad for p in params]
            set_grads(params, t)
            for p, g in zip(params, kept):
                g.copy_(p.grad)
                p.grad = g
        lr.fill_(0.02 / t)
        ref.param_groups[0]["lr"] = float(lr)
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            torch.testing.assert_close(p, q, rtol=1e-6, atol=1e-6)
        for x, y in zip(opt.moments(), ref.moments()):
            assert torch.equal(x, y)
    assert opt.state_dict()["state"][0]["step"] == 5
    saved = copy.deepcopy(opt.state_dict())
    graph.replay()
    opt.load_state_dict(saved)   # the lr's value goes to where the graph reads it
    assert opt.param_groups[0]["lr"] is lr and opt.state_dict()["state"][0]["step"] == 5


@pytest.mark.parametrize("bits,kind", [(32, torch.bfloat16), (8, torch.float32)])
def test_a_captured_step_goes_on_from_what_was_loaded(dev, bits, kind):
    """Loading writes the state where it lies: replays after it equal steps of an optimiser that loaded the same."""
    a, b = tensors([5000, 257], kind, dev), tensors([5000, 257], kind, dev)
    new = lambda p: P.AdamW(p, state_bits=bits, master_weights=True, capturable=True, **HYPER)   # noqa: E731
    opt, ref = new(a), new(b)
    set_grads(a, 0)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    saved, at = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in a]
    graph.replay()
    spare = [torch.full((5000,), float("nan"), device=dev) for _ in range(8)]   # (what a freed state would become)
    for own in (False, True):
        opt.load_state_dict(opt.state_dict() if own else saved)   # its own, views of its state, changes nothing
        if own:
            graph.replay()
            ref.step()
        else:
            ref.load_state_dict(saved)
            with torch.no_grad():
                for p, q, x in zip(a, b, at):
                    p.copy_(x)
                    q.copy_(x)
            set_grads(b, 0)
            graph.replay()
            ref.step()
        torch.cuda.synchronize()
        for p, q in zip([*a, *opt.moments()], [*b, *ref.moments()]):
            assert torch.equal(p, q)
    assert opt.state_dict()["state"][1]["step"] == ref.state_dict()["state"][1]["step"] == 4
    assert all(bool(x.isnan().all()) for x in spare)
    opt.load_state_dict(new(tensors([5000, 257], kind, dev)).state_dict())   # one that never stepped
    assert not any(bool(x.any()) for x in opt.moments()) and opt.state_dict()["state"][0]["step"] == 0


def test_a_parameter_laid_out_anew_is_refused(dev):
    p = tensors([64 * 64], torch.float32, dev)[0]
    p.data = p.data.view(64, 64)
    opt = P.AdamW([p], **HYPER)
    for _ in range(2):
        p.grad = torch.ones(64, 64, device=dev)
        opt.step()
    p.data = p.data.t()   # the same address and size, the gradient as before
    with pytest.raises(RuntimeError, match="reshaped"):
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_copied_with_its_parameters(dev, bits):
    a = tensors([1000, 33], torch.float32, dev)
    opt = P.AdamW(a, state_bits=bits, seed=5, **HYPER)
    set_grads(a, 1)
    opt.step()
    b, other = copy.deepcopy((a, opt))
    for t in (2, 3):
        for params, o in ((a, opt), (b, other)):
            set_grads(params, t)
            o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and p.data_ptr() != q.data_ptr()


def test_a_tensor_lr_is_checked_at_each_step(dev):
    p = tensors([100], torch.float32, dev)
    set_grads(p, 1)
    plain = P.AdamW(p, **HYPER)
    plain.param_groups[0]["lr"] = torch.tensor([0.1], device=dev)
    with pytest.raises(ValueError, match="tensor lr"):
        plain.step()
    opt = P.AdamW(p, capturable=True, **{**HYPER, "lr": torch.tensor([0.1], device=dev)})
    opt.step()
    for bad in (torch.tensor([0.1]), torch.tensor([0.1], device=dev, dtype=torch.float64), torch.zeros(2, device=dev)):
        opt.param_groups[0]["lr"] = bad
        with pytest.raises(ValueError, match="tensor lr"):
            opt.step()


def test_capture_refusals(dev):
    p = tensors([100], torch.float32, dev)
    set_grads(p, 1)
    opt = P.AdamW(p, **HYPER)
    opt.step()
    fresh = P.AdamW(tensors([100], torch.float32, dev), capturable=True, **HYPER)
    set_grads(fresh.param_groups[0]["params"], 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for o, what in ((opt, "capturable=True"), (fresh, "run one step")):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=what):
            with torch.cuda.graph(graph):
                o.step()
    fresh.param_groups[0]["params"][0].grad = None
    with pytest.raises(RuntimeError, match="needs a gradient"):
        fresh.step()


def test_on_another_stream(dev):
    a, b = tensors([70001], torch.float32, dev), tensors([70001], torch.float32, dev)
    set_grads(a, 1)
    set_grads(b, 1)
    P.AdamW(a, **HYPER).step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b[0].grad.mul_(2).mul_(0.5)
        P.AdamW(b, **HYPER).step()
    s.synchronize()
    assert torch.equal(a[0], b[0])


def test_gradients_in_other_layouts(dev):
    p = torch.nn.Parameter(torch.randn((64, 48), device=dev))
    q = torch.nn.Parameter(p.detach().clone())
    g = torch.randn((48, 64), device=dev)
    p.grad, q.grad = g.t(), g.t().contiguous()
    for x in (p, q):
        P.AdamW([x], **HYPER).step()
    assert torch.equal(p, q)


def test_a_negated_view_as_gradient(dev):
    a, b = tensors([1000], torch.float32, dev), tensors([1000], torch.float32, dev)
    set_grads(a, 3)
    b[0].grad = torch._neg_view(-a[0].grad)
    for p in (a, b):
        P.AdamW(p, **HYPER).step()
    assert b[0].grad.is_neg() and torch.equal(a[0], b[0])


def test_more_elements_than_32_bits_count(dev):
    """2^31 + 300 elements with moments in 8 bits: the first and last blocks as a small tensor's at the same places."""
    n = (1 << 31) + 300
    p = torch.nn.Parameter(torch.zeros((n,), dtype=torch.bfloat16, device=dev))
    p.grad = torch.zeros_like(p)
    g = torch.randn((600,), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    p.grad[-600:] = g
    p.grad[:600] = g
    opt = P.AdamW([p], state_bits=8, **HYPER)
    opt.step()
    small = torch.nn.Parameter(torch.zeros((600,), dtype=torch.bfloat16, device=dev))
    small.grad = g
    one = P.AdamW([small], state_bits=8, **HYPER)
    one.step()
    assert torch.equal(p.detach()[:600], small.detach())
    assert torch.equal(p.detach()[-600:], small.detach())   # the step itself does not depend on the place
    st = opt.state[p]
    assert torch.equal(st["exp_avg"][:600], one.state[small]["exp_avg"])
    place = np.arange(n - 300, n)   # the last two blocks, the second partly behind the tensor
    d = np64(p.grad[-300:])
    m, v = (1 - 0.9) * d, (1 - 0.99) * d * d
    em, ev, exps = encode(m, v, *dither(place, 1, 0, 0))
    np.testing.assert_array_equal(st["exp_avg"][-300:].cpu().numpy(), em)
    np.testing.assert_array_equal(st["exp_avg_sq"][-300:].cpu().numpy(), ev)
    np.testing.assert_array_equal(st["exponents"][-2:].cpu().numpy(), exps)
    assert not bool(p.detach()[600:-600].any())


def test_a_training_step_of_the_class_head(dev):
    """The two operators as they are used together: the class head's loss with its gradient, then the step, against the
    same run through torch's own operators in f32."""
    cfg = P.Config(device=dev)

    def run(ours):
        torch.manual_seed(11)
        dec = P.Decoder(cfg, cfg.geo_mlp_hidden_dim, cfg.geo_mlp_level, 20)
        feats = torch.nn.Parameter(torch.randn((4000, 11), device=dev))
        y = torch.randint(0, 20, (4000,), device=dev)
        y[::7] = -100
        params = [feats, *dec.parameters()]
        hyper = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.01)
        opt = P.AdamW(params, **hyper) if ours else torch.optim.AdamW(params, foreach=False, **hyper)
        kept = (y != -100).sum()
        for _ in range(5):
            opt.zero_grad()
            if ours:
                r = dec.sem_label_log_prob(feats, y, top_k=3)
                loss = -r.log_prob.sum() / kept + 0.1 * r.entropy.mean()
            else:
                logp = dec.sem_label_prob(feats)
                loss = torch.nn.functional.nll_loss(logp, y, ignore_index=-100) - 0.1 * (logp.exp() * logp).sum(1).mean()
            loss.backward()
            opt.step()
        return [p.detach() for p in params], [p.grad for p in params]

    (a, ga), (b, gb) = run(True), run(False)
    for x, y in zip(ga, gb):   # gradients: f32 sums in another order
        torch.testing.assert_close(x, y, rtol=2e-3, atol=2e-3 * float(y.abs().max()))
    for x, y in zip(a, b):     # five steps of at most lr each
        assert float((x - y).abs().max()) <= 0.1 * 5 * 0.01


def test_each_step_of_the_class_heads_training(dev):
    """Loss, gradient and step of the two operators: torch's AdamW, fed the gradients that this run's loss gave, goes the
    same way parameter by parameter.  A step is off by 14 u of its update (at most lr) and 3 u of the parameter on either
    side, and five of them add up: 30 u |p| + 140 u lr, 1.8e-6 |p| + 8.4e-8.  (A bias correction or decay that is wrong
    by a thousandth moves a parameter by 1e-5.)"""
    cfg = P.Config(device=dev)
    torch.manual_seed(12)
    dec = P.Decoder(cfg, cfg.geo_mlp_hidden_dim, cfg.geo_mlp_level, 20)
    feats = torch.nn.Parameter(torch.randn((4000, 11), device=dev))
    y = torch.randint(0, 20, (4000,), device=dev)
    y[::7] = -100
    mine = [feats, *dec.parameters()]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    hyper = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    opt, ref = P.AdamW(mine, **hyper), torch.optim.AdamW(theirs, foreach=False, **hyper)
    kept = (y != -100).sum()
    losses = []
    for _ in range(5):
        opt.zero_grad()
        r = dec.sem_label_log_prob(feats, y, top_k=3)
        loss = -r.log_prob.sum() / kept + 0.1 * r.entropy.mean()
        loss.backward()
        before = [p.detach().clone() for p in mine]
        for p, q in zip(mine, theirs):
            q.grad = p.grad.clone()
        opt.step()
        ref.step()
        losses.append(float(loss))
        for p, q, b in zip(mine, theirs, before):
            torch.testing.assert_close(p.detach(), q.detach(), rtol=1.8e-6, atol=8.4e-8)
            assert float((p.detach() - b).abs().max()) > 1e-3   # it moved
    assert all(math.isfinite(x) for x in losses)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_training_step(dev, bits):
    """Loss, gradient into the leaf's own .grad and step in one graph, replayed between eager work, against the same calls
    made eagerly."""
    n, c = 300, 700
    labels = [torch.randint(0, c, (n,), generator=torch.Generator().manual_seed(t)).to(dev) for t in range(5)]
    up = torch.full((n,), -1.0 / n, device=dev)

    def start():
        x = torch.nn.Parameter(torch.randn((n, c), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(dev))
        return x, P.AdamW([x], state_bits=bits, master_weights=True, capturable=True, **HYPER)

    def turn(x, opt, y):
        x.grad = None
        r = P.label_log_probs(x, y, top_k=2)
        torch.autograd.backward([r.log_prob, r.entropy], [up, up])
        opt.step()
        return r.log_prob.detach(), r.top_index

    (x, opt), (q, ref) = start(), start()
    y = labels[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn(x, opt, y)
    torch.cuda.current_stream().wait_stream(side)
    turn(q, ref, labels[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = turn(x, opt, y)
    for t in range(1, 5):
        y.copy_(labels[t])
        want = turn(q, ref, labels[t])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*out, x, x.grad, *opt.moments(), opt.master()],
                                                     [*want, q, q.grad, *ref.moments(), ref.master()]))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_query_after_a_step_sees_it(dev, bits):
    """A map's queries read views of its features and decoder that are kept until those are modified: after a step they
    are made anew, as a decoder and a map with the same values and no views give."""
    from pin_slam_amd.synthetic import surface_map, surface_pool
    nm, dec, pts = surface_map(200, device=dev, buffer_size=1 << 22, query_backend="grid")
    q = surface_pool(pts, 5000, seed=3, device=dev)[0]
    ask = lambda d: P.query_sdf(nm, d, q, query_locally=True, want_grad=True)[:2]   # noqa: E731
    feats = nm.local_geo_features
    for params in ([*dec.parameters()], [feats], [feats, *dec.parameters()]):
        for p in params:
            p.grad = torch.full_like(p, 0.1)
        if len(params) > 1:
            params[-1].grad = torch._neg_view(-params[-1].grad)   # one that is copied first
        opt = P.AdamW(params, lr=0.05, state_bits=bits)
        for _ in range(2):
            before = ask(dec)
            opt.step()
            after = ask(dec)
            nm._cache = {}
            copied = P.Decoder(nm.config, 64, 1, 1)
            copied.load_state_dict(dec.state_dict())
            fresh = ask(copied)
            assert not torch.equal(before[0], after[0])
            assert all(torch.equal(a, b) for a, b in zip(after, fresh))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_between_forward_and_backward_is_seen(dev, bits):
    """A graph that saved a parameter refuses to go back through it after a step, as with torch's optimisers."""
    for way in ("fast", "some", "copied"):
        params = tensors([500, 20], torch.float32, dev)
        set_grads(params, 1)
        if way == "copied":
            params[0].grad = torch._neg_view(-params[0].grad)
        opt = P.AdamW(params, state_bits=bits, **HYPER)
        if way == "some":
            opt.step()
            params[1].grad = None
        out = [(p * p).sum() for p in params]
        versions = [p._version for p in params]
        opt.step()
        assert params[0]._version > versions[0] and (params[1]._version > versions[1]) == (way != "some")
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out[0].backward()
        if way == "some":
            out[1].backward()
        st = opt.state[params[0]]
        before = {k: t._version for k, t in st.items()}
        opt.step()
        assert all(t._version > before[k] for k, t in st.items())
    logits = torch.nn.Parameter(torch.randn((30, 20), device=dev))
    r = P.label_log_probs(logits, torch.zeros((30,), dtype=torch.int64, device=dev))
    logits.grad = torch.ones_like(logits)
    P.AdamW([logits], state_bits=bits, **HYPER).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.log_prob.sum().backward()


def test_queries_between_replays(dev):
    """A replayed step marks nothing: increment_version does, as documented."""
    from pin_slam_amd.synthetic import surface_map, surface_pool
    nm, dec, pts = surface_map(200, device=dev, buffer_size=1 << 22, query_backend="grid")
    q = surface_pool(pts, 3000, seed=3, device=dev)[0]
    params = [nm.local_geo_features, *dec.parameters()]
    for p in params:
        p.grad = torch.full_like(p, 0.1)
    opt = P.AdamW(params, lr=0.05, capturable=True)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        torch.autograd.graph.increment_version(params)
        after = P.query_sdf(nm, dec, q, query_locally=True, want_grad=True)[:2]
        nm._cache = {}
        copied = P.Decoder(nm.config, 64, 1, 1)
        copied.load_state_dict(dec.state_dict())
        fresh = P.query_sdf(nm, copied, q, query_locally=True, want_grad=True)[:2]
        assert all(torch.equal(a, b) for a, b in zip(after, fresh))


@pytest.mark.parametrize("capturable", [False, True])
def test_rates_changed_later_are_checked_before_any_group_steps(dev, capturable):
    """A group that is refused leaves the others as they were, and the next good step goes on from there."""
    def build():
        a, b = tensors([500, 20], torch.bfloat16, dev), tensors([300], torch.float32, dev, 1)
        for ps in (a, b):
            set_grads(ps, 3)
        return a + b, P.AdamW([dict(params=a, master_weights=True), dict(params=b, state_bits=8)], capturable=capturable,
                              **HYPER)

    (params, opt), (others, ref) = build(), build()
    opt.step()
    ref.step()
    for gi, key, bad in ((1, "lr", -1.0), (1, "lr", math.nan), (1, "betas", (0.9, 1.0)), (1, "betas", (-0.1, 0.9)),
                         (1, "eps", -1e-3), (1, "weight_decay", math.inf), (1, "state_bits", 16), (1, "state_bits", 32),
                         (0, "master_weights", False)):
        group = opt.param_groups[gi]
        kept, group[key] = group[key], bad
        versions = [p._version for p in params]
        with pytest.raises((ValueError, RuntimeError)):
            opt.step()
        group[key] = kept
        assert [p._version for p in params] == versions
        assert all(torch.equal(p, q) for p, q in zip(params, others))
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [1, 1, 1]
    opt.param_groups[1]["master_weights"] = True   # of parameters in 32 bits: nothing changes
    opt.step()
    ref.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others))
    assert all(torch.equal(x, y) for gi in (0, 1) for x, y in zip(opt.moments(gi), ref.moments(gi)))


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_counted_from_the_end(dev, bits):
    """moments(-1) is the last group's, and asking changes nothing."""
    a, b = tensors([500], torch.float32, dev), tensors([300, 20], torch.bfloat16, dev, 1)
    opt = P.AdamW([dict(params=a), dict(params=b, master_weights=True)], state_bits=bits, **HYPER)
    for t in (1, 2):
        set_grads(a + b, t)
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    for gi in (1, 0):
        assert all(torch.equal(x, y) and bool(x.any()) for x, y in zip(opt.moments(gi), opt.moments(gi - 2)))
        assert opt.offsets(gi) == opt.offsets(gi - 2)
    assert torch.equal(opt.master(1), opt.master(-1)) and opt.master(0) is None and opt.master(-2) is None
    again = opt.state_dict()
    for k, one in saved["state"].items():
        assert one["step"] == again["state"][k]["step"] == 2
        assert all(torch.equal(one[key], again["state"][k][key]) for key in one if key != "step")
    for bad in (2, -3):
        with pytest.raises(IndexError):
            opt.moments(bad)


@pytest.mark.parametrize("bits,capturable", [(32, False), (8, False), (8, True)])
def test_emptied_state_begins_anew(dev, bits, capturable):
    """Emptying or replacing opt.state, as programs do with torch's optimisers: the next step is a first step, and a
    parameter that takes another's place in a group is refused."""
    from collections import defaultdict
    a, b = tensors([500, 20], torch.bfloat16, dev), None
    opt = P.AdamW(a, state_bits=bits, master_weights=True, capturable=capturable, **HYPER)
    for way in ("clear", "replace"):
        for t in (1, 2):
            set_grads(a, t)
            opt.step()
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        ref = P.AdamW(b, state_bits=bits, master_weights=True, capturable=capturable, **HYPER)
        if way == "clear":
            opt.state.clear()
        else:
            opt.state = defaultdict(dict)
        assert opt.state_dict()["state"] == {}
        for t in (1, 2):
            set_grads(a, 5 + t)
            set_grads(b, 5 + t)
            opt.step()
            ref.step()
            assert all(torch.equal(p, q) for p, q in zip([*a, *opt.moments(), opt.master()], [*b, *ref.moments(), ref.master()]))
        assert [s["step"] for s in opt.state_dict()["state"].values()] == [2, 2]
    opt.param_groups[0]["params"][0] = b[0]
    with pytest.raises(RuntimeError, match="added to or taken from"):
        opt.step()


@pytest.mark.parametrize("first,then", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_a_parameter_that_changes_its_width_beside_its_copy_is_refused(dev, first, then):
    """master_weights: a parameter that became 16 bits wide has no copy, or one of its first value, and one that became 32
    bits wide would leave its copy behind; loading starts from what it is now.  Without copies the type may change."""
    for alone in (True, False):
        p = tensors([300] if alone else [300, 20], first, dev)
        if not alone:
            p[1].data = p[1].data.to(torch.float16)
        opt = P.AdamW(p, master_weights=True, **HYPER)
        set_grads(p, 1)
        opt.step()
        p[0].grad, p[0].data = None, p[0].data.to(then)
        set_grads(p, 2)
        before = [q.detach().clone() for q in p]
        with pytest.raises(RuntimeError, match="copy in 32 bits became"):
            opt.step()
        assert all(torch.equal(x, q) for x, q in zip(before, p))
        b = [torch.nn.Parameter(x.clone()) for x in before]
        other = P.AdamW(b, master_weights=True, **HYPER)
        opt.load_state_dict(other.state_dict())
        set_grads(b, 2)
        opt.step()
        other.step()
        assert all(torch.equal(x, y) for x, y in zip(p, b))
    q = tensors([300], first, dev)
    opt = P.AdamW(q, **HYPER)
    set_grads(q, 1)
    opt.step()
    q[0].grad, q[0].data = None, q[0].data.to(then)
    set_grads(q, 2)
    check_step(opt, 2)


def test_a_copy_serves_either_type_of_16_bits(dev):
    p = tensors([300], torch.bfloat16, dev)
    opt = P.AdamW(p, master_weights=True, **HYPER)
    set_grads(p, 1)
    opt.step()
    p[0].grad, p[0].data = None, p[0].data.to(torch.float16)
    set_grads(p, 2)
    check_step(opt, 2)


@pytest.mark.parametrize("bits", [32, 8])
def test_asking_before_the_first_step_keeps_nothing(dev, bits):
    """moments(), master() and offsets() of a group that has not stepped: zeros, the parameters as they are, places; weights
    that are loaded afterwards are those that the first step goes on from."""
    a, b = tensors([300, 20], torch.bfloat16, dev), tensors([300, 20], torch.bfloat16, dev, 1)
    opt = P.AdamW(a, state_bits=bits, master_weights=True, **HYPER)
    ref = P.AdamW(b, state_bits=bits, master_weights=True, **HYPER)
    assert opt.offsets() == [0, 512] and not any(bool(x.any()) for x in opt.moments())
    assert torch.equal(opt.master()[:300], a[0].detach().float()) and opt.state_dict()["state"] == {}
    with torch.no_grad():
        for p, q in zip(a, b):
            p.copy_(q)
    assert torch.equal(opt.master()[512:532], b[1].detach().float())
    for t in (1, 2):
        set_grads(a, t)
        set_grads(b, t)
        opt.step()
        ref.step()
        assert all(torch.equal(p, q) for p, q in zip([*a, *opt.moments(), opt.master()], [*b, *ref.moments(), ref.master()]))
    assert opt.master() is opt.master() and opt.offsets() == [0, 512]


def test_refusals(dev):
    ok = lambda: torch.nn.Parameter(torch.zeros(8, device=dev))   # noqa: E731
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(state_bits=16),
                dict(lr=math.nan)):
        with pytest.raises(ValueError):
            P.AdamW([ok()], **bad)
    with pytest.raises(ValueError, match="contiguous"):
        P.AdamW([torch.nn.Parameter(torch.zeros((4, 6), device=dev).t())])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        P.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64, device=dev))])
    buf = torch.zeros(20, device=dev)
    with pytest.raises(ValueError, match="share memory"):
        P.AdamW([torch.nn.Parameter(buf[:10]), torch.nn.Parameter(buf[9:])])
    with pytest.raises(ValueError):
        P.AdamW([ok()], lr=torch.tensor([0.1], device=dev))
    p = ok()
    opt = P.AdamW([p], **HYPER)
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]], device=dev), torch.ones(1, device=dev), (8,))
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    p.grad = torch.ones_like(p)
    opt.step()
    p.data = torch.zeros(9, device=dev)
    p.grad = torch.ones(9, device=dev)
    with pytest.raises(RuntimeError, match="reshaped or moved"):
        opt.step()
