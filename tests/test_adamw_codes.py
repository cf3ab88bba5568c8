"""CPU: the 8-bit codes of AdamW's moments, and the refusals that need no device."""
import ctypes

import numpy as np
import pytest
import torch

import pin_slam_amd as P
from pin_slam_amd import _lib
from tests.adamw_codes import BLOCK, decode, dither, encode


def test_codes_of_their_own_values():
    """A code's value is coded as itself, whatever the dither, where the block's exponent is the same."""
    n = BLOCK
    m = np.full(n, 0x70, np.uint8)   # 2^E itself is there: the exponent stays E
    m[:240] = np.concatenate([np.arange(0x78), 0x80 + np.arange(0x78)])
    v = np.full(n, 0xF0, np.uint8)
    v[:248] = np.arange(248)
    exps = np.array([[5, -40]], np.int16)
    a, b = decode(m, v, exps)
    for d in (0.0, 65536.0, 131071.0):
        em, ev, e = encode(a, b, np.full(n, d), np.full(n, d))
        assert np.array_equal(em, m) and np.array_equal(ev, v) and np.array_equal(e, exps)


def test_rounding_error_and_expectation():
    """Every value lies within one code of itself, and the mean over all dithers is the value (to 2^-17 of a code)."""
    rng = np.random.default_rng(1)
    x = rng.normal(size=BLOCK) * np.exp(2 * rng.normal(size=BLOCK))
    y = x * x
    dithers = np.linspace(0, 131071, 512).astype(int)
    total_m, total_v = np.zeros(BLOCK), np.zeros(BLOCK)
    for d in dithers:
        cm, cv, e = encode(x, y, np.full(BLOCK, float(d)), np.full(BLOCK, float(d)))
        m, v = decode(cm, cv, e)
        top = np.ldexp(1.0, int(e[0, 0]))
        assert (np.abs(m - x) <= np.maximum(np.abs(x) / 8, top * 2.0 ** -16)).all()
        assert (np.abs(v - y) <= y / 8 + np.ldexp(1.2, int(e[0, 1]) - 30)).all() and (v > 0).all()
        total_m += m
        total_v += v
    step = np.abs(x) / 8 + top * 2.0 ** -16
    assert (np.abs(total_m / 512 - x) <= step / 256).all()
    assert (np.abs(total_v / 512 - y) <= y / 8 / 256 + np.ldexp(1.2, int(e[0, 1]) - 30)).all()


def test_dither_is_spread_evenly():
    """Mean 1/2 and no correlation between the two numbers, neighbours or steps (5 standard deviations of 2^18 draws)."""
    n = 1 << 18
    a, b = (x / 2 ** 17 for x in dither(np.arange(n), 1, 0, 0))
    c = dither(np.arange(n), 2, 0, 0)[0] / 2 ** 17
    for x in (a, b, c):
        assert abs(x.mean() - 0.5) < 5 * (1 / 12 / n) ** 0.5
        assert np.abs(np.histogram(x, 16, (0, 1))[0] - n / 16).max() < 5 * (n / 16) ** 0.5
    for x, y in ((a, b), (a, c), (a[1:], a[:-1]), (a[64:], a[:-64])):
        assert abs(np.corrcoef(x, y)[0, 1]) < 5 / n ** 0.5


def test_refusals_without_a_device():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = P.AdamW([p])
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        opt.step()
    with pytest.raises(ValueError, match="state_bits"):
        P.AdamW([p], state_bits=4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        P.label_log_probs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))


def test_argument_errors_before_any_device_work():
    lib = _lib.load()
    ok = ctypes.c_void_p(4096)   # never read: every call below is refused on the host

    def logprob(logits=ok, dtype=0, n=4, c=10, stride=10, labels=ok, k=2, lp=ok, ent=ok, top=ok, idx=ok):
        return lib.pin_label_logprob(logits, dtype, n, c, stride, labels, -100, k, lp, ent, None, top, idx, None, None)

    assert logprob(n=0) == 0
    for bad in (dict(logits=None), dict(dtype=3), dict(dtype=-1), dict(n=-1), dict(c=0), dict(c=524281),
                dict(stride=-1), dict(labels=None), dict(k=11), dict(k=33, c=100), dict(k=-1), dict(lp=None),
                dict(ent=None), dict(top=None), dict(idx=None), dict(logits=ctypes.c_void_p(4098))):
        assert logprob(**bad) == -1, bad
    assert lib.pin_label_logprob_bwd(ok, 0, 4, 10, 10, ok, -100, 2, ok, None, ok, ok, ok, ok, None) == -1
    assert lib.pin_label_logprob_bwd(ok, 0, 4, 10, 10, ok, -100, 2, None, ok, ok, ok, ok, ok, None) == -1
    assert lib.pin_label_logprob_bwd(ok, 0, 4, 10, 10, ok, -100, 2, ok, ok, ok, ok, ok, None, None) == -1

    def adamw(ps=(4096, 8192), gs=(4096, 8192), sizes=(300, 5), offsets=(0, 512), dtype=0, bits=8, m=ok, v=ok, e=ok, w=None,
              total=768, lr=0.1, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, step=1, scalars=None):
        n = len(sizes)
        arr = lambda t, x: (t * n)(*x)   # noqa: E731
        return lib.pin_adamw_step(arr(ctypes.c_void_p, ps), arr(ctypes.c_void_p, gs), arr(ctypes.c_int64, sizes),
                                  arr(ctypes.c_int64, offsets), n, dtype, bits, m, v, e, w, total, lr, b1, b2, eps, wd,
                                  step, 0, scalars, None)

    for bad in (dict(ps=(4096, None)), dict(gs=(None, 4096)), dict(sizes=(-1, 5)), dict(sizes=(300, 400)),
                dict(offsets=(0, 256)), dict(offsets=(0, 500)), dict(offsets=(512, 0)), dict(dtype=5), dict(bits=16),
                dict(m=None), dict(v=None), dict(e=None), dict(m=ctypes.c_void_p(4097)), dict(e=ctypes.c_void_p(4098)),
                dict(w=ctypes.c_void_p(4100)), dict(total=700), dict(total=-256), dict(lr=-1.0), dict(lr=float("nan")),
                dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(eps=float("nan")), dict(wd=-1.0), dict(step=0),
                dict(ps=(4098, 8192)), dict(scalars=ctypes.c_void_p(4100))):
        assert adamw(**bad) == -1, bad
    assert adamw(sizes=(0, 0), offsets=(0, 0), ps=(None, None), gs=(None, None)) == 0   # nothing to step
    assert lib.pin_adamw_scalars(None, None, 0.1, 0.9, 0.99, 0.0, 0, ok, None) == -1
    assert lib.pin_adamw_scalars(ok, None, -0.1, 0.9, 0.99, 0.0, 0, ok, None) == -1
    assert lib.pin_adamw_moments(ok, ok, ok, 100, ok, ok, None) == -1
    assert lib.pin_adamw_moments(ok, ok, None, 256, ok, ok, None) == -1
    assert lib.pin_adamw_moments(ok, ok, ok, 0, None, None, None) == 0


def test_what_is_no_tensor_is_refused():
    fns = [_lib.address(n) for n in ("pin_label_logprob_workspace_bytes", "pin_label_logprob", "pin_label_logprob_bwd")]
    with pytest.raises(TypeError, match="two tensors"):
        _lib.torch_fn("pin_torch_label")(*fns, 3, torch.zeros(2, dtype=torch.int64), 0, -100, 1)


def test_addresses_of_many_tensors():
    """pin_torch_gather: addresses of what is as the kernel takes it, refusal of anything else (host tensors, device -1)."""
    import weakref
    from array import array

    gather = _lib.torch_fn("pin_torch_gather")

    def make(kind=torch.float32, shapes=((7,), (3, 4), (), (0,))):
        out = [torch.nn.Parameter(torch.ones(s, dtype=kind)) for s in shapes]
        for p in out:
            p.grad = torch.zeros_like(p)
        return out

    def ask(params, sizes=None, device=-1):
        sizes = array("q", [p.numel() for p in params] if sizes is None else sizes)
        n = len(sizes)
        ps, gs = array("Q", bytes(8 * n)), array("Q", bytes(8 * n))
        return gather(params, n, *(x if isinstance(x, int) else x.buffer_info()[0] for x in (sizes, device, ps, gs))), ps, gs

    for kind, code in _lib.TYPES.items():
        params = make(kind)
        rc, ps, gs = ask(params)
        assert rc == code
        assert list(ps) == [p.data_ptr() for p in params] and list(gs) == [p.grad.data_ptr() for p in params]
    assert ask(make(torch.float64))[0] == -1
    assert ask(make(), device=0)[0] == -1
    assert ask(make(), sizes=[7, 12, 1, 1])[0] == -1 and ask(make(), sizes=[7, 12, 1])[0] == -1
    assert ask([])[0] == -1 and ask(tuple(make()), sizes=[7, 12, 1, 0])[0] == -1
    assert ask([*make(), 3], sizes=[7, 12, 1, 0, 1])[0] == -1

    def changed(i, f):
        params = make(shapes=((7,), (4, 4)))
        f(params[i])
        return ask(params, sizes=[7, 16])[0]

    assert changed(0, lambda p: None) == 0
    assert changed(0, lambda p: setattr(p, "grad", None)) == -1
    assert changed(1, lambda p: setattr(p, "data", p.data.t())) == -1
    assert changed(1, lambda p: setattr(p, "grad", torch.zeros(4, 4).t())) == -1
    assert changed(1, lambda p: setattr(p, "data", torch.ones(4, 4, dtype=torch.float16))) == -1
    assert changed(1, lambda p: setattr(p, "grad", torch.zeros(4, 4).to_sparse())) == -1
    m = torch.nn.Parameter(torch.ones(7, device="meta"))
    m.grad = torch.zeros(7, device="meta")
    assert ask([m])[0] == -1   # no addresses
    assert ask([*make(torch.float32), *make(torch.float16)])[0] == -1
    p = make()[0]
    assert ask([p * 1], sizes=[7])[0] == -1   # not a leaf

    class Other(torch.Tensor):
        pass

    q = torch.nn.Parameter(torch.ones(7).as_subclass(Other))
    q.grad = torch.zeros(7)
    assert ask([q], sizes=[7])[0] == -1
    gone = weakref.ref(p)   # no reference is kept
    del p
    assert gone() is None


def test_versions_of_what_is_written():
    """pin_torch_touched raises the versions that torch's check of saved tensors goes by (of tensors that have one)."""
    touched = _lib.torch_fn("pin_torch_touched")
    p = torch.nn.Parameter(torch.ones(4))
    flat = torch.zeros(8)
    view = flat[2:4]
    with torch.inference_mode():
        free = torch.ones(3)
    out = (p * p).sum()
    before = p._version
    assert touched([p, flat, free]) == 0
    assert p._version == before + 1 and flat._version == view._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()
    assert touched([]) == 0 and touched([p, 3]) == -1 and touched((p,)) == -1


def test_workspace_of_many_split_rows():
    """Rows that are split come in batches of fewer than 2^24 parts, which share one workspace."""
    ws = _lib.load().pin_label_logprob_workspace_bytes
    for kind, size, c in [(0, 4, 524280), (2, 2, 524280), (2, 2, 300001), (0, 4, 140001)]:
        one = ws(1 << 12, c, kind, 4) // (1 << 12)
        assert one > 0 and one % 272 == 0 and ws(1 << 12, c, kind, 0) * 17 == one << 12
        parts = one // 272
        assert 1 < parts <= 64
        for n in ((1 << 24) // parts, (1 << 24) // parts + 1, 1 << 40):
            assert ws(n, c, kind, 4) == ((1 << 24) - 1) // parts * one
