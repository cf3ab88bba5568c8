"""label_log_probs (log probability of given labels, entropy, most probable classes, and the gradient)
against the definition in 64 bits.

Tolerances.  u = 2^-24 is half a step of f32.  A term e^d (d = z - max) carries the rounding of d
(|d| u), of its product with log2 e (as much again) and of the exponential (2 u): (2|d| + 4) u of
itself.  A sum of positive terms in chains of at most 160 (the longest in a thread, then the tree)
adds 160 u.  With D = sum p|d| and Q = sum p d^2 that gives for s = sum e^d a relative error
  A = u (2 D + 164),
for log_prob = d_y - log s: A + u (2|d_y| + 4|log s| + 2|log_prob|) and for the entropy
log s - (sum e^d d)/s: A (1 + D) + u (2 Q + 164 D + 4|log s| + 2 H).
The gradient -p (G + g_H (log p + H)) + (the given terms): the factor's own errors times p, and
(2|d| + 8) u + A for p itself, 4 u for its products, (k + 1) u for the sum G, and 4 u of the sizes of the given terms, which
may cancel, for their sums.  An output of fewer
bits adds half its step, and where it underflows half its least positive value."""
import math

import numpy as np
import pytest
import torch

import pin_slam_amd as P

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return "cuda"


def reference(z, y, k, g_lp=None, g_ent=None, g_top=None, ignore=IGNORE):
    """The definition in 64 bits (z [n, C] of any type, on the CPU), and the tolerances above."""
    zt = z.to(torch.float64)
    n, c = zt.shape
    z = zt.numpy()
    y = np.asarray(y)
    sick = ~(z < np.inf).all(1)                      # a NaN or +inf
    m = np.where(sick, 0.0, np.where(np.isnan(z), -np.inf, z).max(1))
    dead = m == -np.inf
    with np.errstate(all="ignore"):
        d = np.where((sick | dead)[:, None], 0.0, z - np.where(dead, 0.0, m)[:, None])
        e = np.exp(d)
        s = e.sum(1)
        ls = np.log(s)
        logp = d - ls[:, None]
        p = e / s[:, None]
        pd = np.where(p > 0, p * np.abs(np.where(p > 0, d, 0)), 0.0)
        D = pd.sum(1)
        Q = np.where(p > 0, pd * np.abs(np.where(p > 0, d, 0)), 0.0).sum(1)
        ent = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0.0).sum(1)
    logp[dead] = -np.inf
    p[dead] = 0.0
    ent[dead] = 0.0
    logp[sick], p[sick], ent[sick] = np.nan, np.nan, np.nan
    has = y != ignore
    inside = (y >= 0) & (y < c)
    at = np.where(inside, y, 0)
    lp = np.where(has, np.where(inside, logp[np.arange(n), at], np.nan), 0.0)
    # value descending, class ascending; both zeros are the same value
    order = np.argsort(-np.where(sick[:, None], 0.0, z), axis=1, kind="stable")[:, :k]
    tlp = np.take_along_axis(logp, order, 1)
    idx = np.where(sick[:, None], -1, order)
    A = U * (2 * D + 164)
    fin = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)   # noqa: E731
    dy = fin(d[np.arange(n), at])
    tol = {"lp": A + U * (2 * dy + 4 * fin(ls) + 2 * fin(lp)),
           "ent": A * (1 + D) + U * (2 * Q + 164 * D + 4 * fin(ls) + 2 * fin(ent)),
           "top": A[:, None] + U * (2 * fin(np.take_along_axis(d, order, 1)) + 4 * fin(ls)[:, None] + 2 * fin(tlp))}
    out = {"lp": lp, "ent": ent, "top": tlp, "idx": idx}
    if g_lp is not None or g_ent is not None or g_top is not None:
        zero = np.zeros(n)
        gl = np.where(has, np.where(inside, g_lp, np.nan), 0.0) if g_lp is not None else zero
        ge = g_ent if g_ent is not None else zero
        gt = g_top if g_top is not None else np.zeros((n, k))
        G = gl + gt.sum(1)
        hit = np.zeros((n, c))
        hit[np.arange(n), at] += np.where(has, gl, 0.0)
        np.add.at(hit, (np.arange(n)[:, None], order), gt)
        given = np.zeros((n, c))
        given[np.arange(n), at] += np.where(has, np.abs(gl), 0.0)
        np.add.at(given, (np.arange(n)[:, None], order), np.abs(gt))
        with np.errstate(all="ignore"):
            spread = np.where(p > 0, np.where(p > 0, logp, 0) + ent[:, None], 0.0)
            dz = -p * (G[:, None] + ge[:, None] * spread) + hit
            size = p * (np.abs(gl) + np.abs(gt).sum(1) + 0.0)[:, None] + p * np.abs(ge)[:, None] * np.where(
                p > 0, np.abs(np.where(p > 0, logp, 0)) + ent[:, None], 0.0)
            rel = U * (2 * fin(d) + 12 + k) + A[:, None]
            t = size * rel + p * np.abs(ge)[:, None] * ((tol["ent"] + A + 4 * U * fin(ls))[:, None] + 2 * U * fin(d)) \
                + 4 * U * (given + np.abs(dz)) + 1e-37
        dz[dead] = 0.0
        dz[sick] = np.nan
        t[dead] = 0.0
        out["dz"], tol["dz"] = dz, t
    return out, tol


def near(got, want, tol, what):
    got, tol = got.detach().double().cpu().numpy(), np.broadcast_to(tol, want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf], err_msg=what)
    ok = np.isfinite(want)
    over = np.abs(got[ok] - want[ok]) - tol[ok]
    assert over.size == 0 or over.max() <= 0, (what, float(over.max()), int((over > 0).sum()))


def grad_tol(tol, dz, kind):
    """The f32 value's tolerance and its rounding to the logits' type."""
    if kind == torch.float32:
        return tol
    least = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[kind]
    half = torch.finfo(kind).eps / 2
    return tol * (1 + half) + half * np.abs(np.nan_to_num(dz)) + least / 2


def check(logits, labels, k, grads=True, seed=0):
    """One call (and its gradient) on the device against the reference; returns the outputs."""
    kind = logits.dtype
    n = logits.shape[0]
    rng = np.random.default_rng(seed)
    up = [rng.normal(size=n).astype(np.float32), rng.normal(size=n).astype(np.float32),
          rng.normal(size=(n, k)).astype(np.float32)]
    want, tol = reference(logits.cpu(), labels.cpu().numpy(), k, *[u.astype(np.float64) for u in up])
    x = logits.detach()
    x = x.requires_grad_(True) if grads else x
    r = P.label_log_probs(x, labels, top_k=k, ignore_index=IGNORE)
    assert r.log_prob.dtype == r.entropy.dtype == r.top_log_prob.dtype == torch.float32
    assert r.top_index.dtype == torch.int64
    near(r.log_prob, want["lp"], tol["lp"], "log_prob")
    near(r.entropy, want["ent"], tol["ent"], "entropy")
    np.testing.assert_array_equal(r.top_index.cpu().numpy(), want["idx"], err_msg="top_index")
    near(r.top_log_prob, want["top"], tol["top"], "top_log_prob")
    if grads:
        outs = [r.log_prob, r.entropy] + ([r.top_log_prob] if k else [])
        dz, = torch.autograd.grad(outs, x, [torch.from_numpy(u).to(x.device) for u in up[:len(outs)]])
        assert dz.dtype == kind and dz.shape == x.shape
        near(dz, want["dz"], grad_tol(tol["dz"], want["dz"], kind), "gradient")
    return r


def make(n, c, kind, dev, pad=0, seed=0, ignore_some=True):
    g = torch.Generator().manual_seed(1000 * n + c + seed)
    wide = torch.full((n, c + pad), math.nan)         # what lies between the rows takes no part
    z = torch.randn((n, c), generator=g) * (0.2 + 4 * torch.rand((n, 1), generator=g)) + 5 * torch.randn((n, 1), generator=g)
    wide[:, :c] = z
    y = torch.randint(0, c, (n,), generator=g)
    if ignore_some and n > 2:
        y[::3] = IGNORE
    return wide.to(kind).to(dev)[:, :c], y.to(dev)


SIZES = [(1, 1), (1, 2), (2, 3), (300, 20), (1025, 19), (9, 31), (70, 32), (5, 33), (7, 63), (130, 64), (4, 65), (3, 127),
         (11, 255), (6, 257), (513, 500), (3, 1003), (2, 2047), (5, 4097), (3, 8191), (2, 8192), (3, 16385), (2, 32769),
         (1, 50021), (3, 65537), (1, 131072), (2, 140001), (2, 300001), (1, 524280), (5000, 70), (4099, 130), (4100, 301),
         (4096, 1000), (260, 20003)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,c", SIZES)
def test_sizes(dev, n, c, kind):
    for k in sorted({0, 1, min(c, 5), min(c, 32)}):
        logits, y = make(n, c, TYPES[kind], dev, pad=(n + c) % 3, seed=k)
        check(logits, y, k)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("pad,first", [(1, 0), (7, 3), (64, 1)])
@pytest.mark.parametrize("c", [20, 1001, 20003])
def test_strides_and_alignments(dev, kind, pad, first, c):
    """Rows that begin at any element, with what is not theirs between them."""
    n = 6
    logits, y = make(n, c, TYPES[kind], dev)
    wide = torch.full((n, first + c + pad), math.inf, dtype=TYPES[kind], device=dev)
    wide[:, first:first + c] = logits
    a = check(wide[:, first:first + c], y, 4)
    b = P.label_log_probs(logits.contiguous(), y, top_k=4)
    for p, q in zip(a, b):   # where a row lies does not change its values
        torch.testing.assert_close(p.detach(), q, rtol=1e-5, atol=1e-5)
    # classes that are not adjacent, rows that are the same, more dimensions
    t = P.label_log_probs(logits.t().contiguous().t(), y, top_k=4)
    assert all(torch.equal(p, q) for p, q in zip(t, b))
    row = logits[1].expand(n, c)
    r = P.label_log_probs(row, y, top_k=4)
    assert torch.equal(r.entropy, r.entropy[:1].expand(n)) and torch.equal(r.top_index, r.top_index[:1].expand(n, 4))
    v = P.label_log_probs(logits.reshape(2, 3, c), y.reshape(2, 3), top_k=4)
    assert v.log_prob.shape == (2, 3) and v.top_index.shape == (2, 3, 4)
    assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(v, P.label_log_probs(logits.reshape(6, c), y, top_k=4)))
    o = P.label_log_probs(logits[2], y[2], top_k=2)
    assert o.log_prob.shape == () and o.top_index.shape == (2,)


def special_rows(c, kind, seed=0):
    """Rows whose mask or values are where a softmax goes wrong, with labels for them."""
    g = torch.Generator().manual_seed(seed + c)
    base = torch.randn((c,), generator=g)
    low = torch.finfo(kind).min
    rows, labels = [], []

    def add(r, y):
        rows.append(r.clone())
        labels.append(y)

    add(torch.full((c,), -math.inf), 0)                       # nothing left
    add(torch.full((c,), -math.inf), IGNORE)
    add(torch.full((c,), low), c - 1)                         # masked by the type's lowest value only
    add(torch.full((c,), torch.finfo(kind).max), 0)           # the type's largest
    one = torch.full((c,), -math.inf)
    one[c // 2] = 1.5
    add(one, c // 2)                                          # one class left, and it is the label
    add(one, 0)                                               # ... or it is not
    few = torch.full((c,), -math.inf)
    few[::max(1, c // 3)] = base[::max(1, c // 3)]
    add(few, 0)                                               # fewer classes left than alternatives
    lows = torch.full((c,), low)
    lows[::max(1, c // 3)] = base[::max(1, c // 3)]
    add(lows, 0)
    add(torch.zeros(c), c // 3)                               # all equal
    two = torch.where(base > 0, 1.0, -1.0)
    add(two, 0)                                               # two values: many ties
    add(torch.where(base > 0, 0.0, -0.0), 0)                  # both zeros are the same
    add(torch.linspace(6.0, -6.0, c), 0)                      # sorted
    add(torch.linspace(-6.0, 6.0, c), 0)
    add(torch.linspace(-6.0, 6.0, c) * 1e-3, c - 1)
    sharp = base.clone()
    sharp[c - 1] = 60.0
    add(sharp, c - 1)                                         # a sure label
    add(sharp, 0)                                             # a hopeless one
    add(base * 2.0 ** 10, 0)                                  # far apart
    nan = base.clone()
    nan[c // 2] = math.nan
    add(nan, 0)
    neg = torch.full((c,), -math.inf)
    neg[0] = math.nan
    add(neg, 0)
    inf = base.clone()
    inf[0] = math.inf
    add(inf, 0)
    add(base, -1)                                             # labels that are no class
    add(base, c)
    add(base, 2 ** 40)
    add(base, IGNORE)
    return torch.stack(rows).to(kind), torch.tensor(labels)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", [1, 2, 20, 64, 100, 700, 2500, 9001, 40000, 131073])
def test_masks_ties_and_values(dev, c, kind):
    z, y = special_rows(c, TYPES[kind])
    for k in sorted({0, min(c, 3), min(c, 32)}):
        check(z.to(dev), y.to(dev), k)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("c,times", [(100, 171), (700, 171), (20003, 11)])
def test_masks_ties_and_values_of_many_rows(dev, c, times, kind):
    """The same rows where so many are laid out otherwise on the chip."""
    z, y = special_rows(c, TYPES[kind])
    for k in (0, 2, 5, 32):
        check(z.repeat(times, 1).to(dev), y.repeat(times).to(dev), k)


FILLS = [1e6, 5e7, 5e9, 1e10, 1e12, 1e20, 1e30]


def finite_mask_rows(c, kind, seed=0):
    """Rows in which a large finite value stands in all classes, in most, or in a range beside ordinary ones, below
    them (a mask that programs write in -inf's place) or above."""
    g = torch.Generator().manual_seed(seed + 7 * c)
    base = torch.randn((c,), generator=g)
    rows, labels = [], []
    off = torch.rand((c,), generator=g) < 0.9
    off[c // 3] = False
    part = torch.zeros((c,), dtype=torch.bool)
    part[c // 8:c // 8 + (c + 1) // 2] = True
    for i, size in enumerate(FILLS):
        for fill in (-size, size):
            rows.append(torch.full((c,), fill))
            labels.append(IGNORE if i % 2 else c // 2)
            if fill < 0 or i in (0, 3, 6):
                rows += [torch.where(off, fill, base), torch.where(part, fill, base)]
                labels += [c // 3, 0 if i % 2 else c // 8]
    spread = base * 1e10
    rows += [spread, spread - 1e12, torch.where(part, -1e30, -1e10 + 1e4 * base), torch.where(part, 1e6, 1e6 + 1e5 * base),
             torch.where(part, -1e12, (1 << 20) + base)]
    labels += [0, c - 1, c // 3, 0, c // 3]
    return torch.stack(rows).to(kind), torch.tensor(labels)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("c", [1, 2, 20, 64, 100, 700, 2500, 9001, 40000, 131073])
def test_large_finite_masks(dev, c, kind):
    """Every layout of few rows: no result and no gradient is lost to the size of a mask."""
    z, y = finite_mask_rows(c, TYPES[kind])
    for k in sorted({0, min(c, 3), min(c, 32)}):
        check(z.to(dev), y.to(dev), k)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("c,times", [(100, 120), (700, 120), (20003, 8)])
def test_large_finite_masks_of_many_rows(dev, c, times, kind):
    z, y = finite_mask_rows(c, TYPES[kind])
    for k in (0, 2, 32):
        check(z.repeat(times, 1).to(dev), y.repeat(times).to(dev), k)


@pytest.mark.parametrize("c,times", [(20, 1), (100, 1), (700, 1), (700, 700), (9001, 1), (20003, 43), (131073, 1)])
def test_maxima_about_the_size_beyond_which_they_are_subtracted_first(dev, c, times):
    """Rows whose classes, threads and parts lie on both sides of 2^20, in either sign."""
    g = torch.Generator().manual_seed(c)
    base = torch.randn((c,), generator=g)
    at, half = float(1 << 20), torch.arange(c) < c // 2
    rows = [s * at + d + w * base for s in (-1, 1) for d in (-3.0, 0.0, 3.0) for w in (0.0, 1.0)]
    rows += [torch.where(half, s * at - 2.0 + 0.5 * base, s * at + 2.0 + 0.5 * base) for s in (-1, 1)]
    z, y = torch.stack(rows), torch.randint(0, c, (len(rows),), generator=g)
    for k in (0, 2):
        check(z.repeat(times, 1).to(dev), y.repeat(times).to(dev), k)


def test_an_ignored_row_masked_by_a_finite_value_passes_no_gradient(dev):
    """What a padded row leaves in the gradient of the layer before it: nothing."""
    for c in (20, 700, 9001, 131073):
        for fill in (-5e9, -1e10, -1e12, -1e30):
            z = torch.randn((3, c), generator=torch.Generator().manual_seed(c)).to(dev)
            z[1] = fill
            x = z.requires_grad_(True)
            r = P.label_log_probs(x, torch.tensor([0, IGNORE, c - 1], device=dev))
            dz, = torch.autograd.grad(r.log_prob.sum(), x)
            assert not bool(dz[1].any()) and bool(torch.isfinite(dz).all())


@pytest.mark.parametrize("kind,c", [("f32", 131000), ("f16", 131072), ("bf16", 131072), ("bf16", 262000)])
def test_longest_rows_of_one_workgroup(dev, c, kind):
    """A workgroup's longest rows, many of them: nearly flat ones, whose sums take the most
    terms of one size, at several heights (the f32 values of the terms go by it: at 1360, 2736 and 3408 they are 1 and
    nearly 2^-15 more or less, which a chain of a thousand terms rounds off or up each time, 254 u in all), a range held
    by a finite mask."""
    g = torch.Generator().manual_seed(c)
    base = torch.randn((c,), generator=g)
    rows = [base * 0.0, base * 0.0 + 1360.0, base * 0.0 + 2736.0, base * 0.0 + 3408.0, base * 1e-3, 0.1 + base * 0.05, 37.7 + torch.linspace(0.0, 0.4, c), -911.3 - torch.linspace(0.0, 0.3, c),
            base, 3 * base, torch.where(torch.arange(c) < c // 2, -1e10, base), -3e7 + 0.3 * base, 5e6 + torch.linspace(0.0, 2.0, c)]
    z = torch.stack(rows).to(TYPES[kind]) if kind != "f16" else torch.stack(rows[:10]).to(TYPES[kind])
    n = z.shape[0]
    y = torch.randint(0, c, (n,), generator=g)
    for k in (0, 3):
        want, tol = reference(z, y.numpy(), k)
        got = P.label_log_probs(z.to(dev)[:, None].expand(n, 300, c), y.to(dev)[:, None].expand(n, 300), top_k=k)
        assert all(torch.equal(t, t[:, :1].expand(t.shape)) for t in got)
        near(got.log_prob[:, 0], want["lp"], tol["lp"], "log_prob")
        near(got.entropy[:, 0], want["ent"], tol["ent"], "entropy")
        np.testing.assert_array_equal(got.top_index[:, 0].cpu().numpy(), want["idx"])
        near(got.top_log_prob[:, 0], want["top"], tol["top"], "top_log_prob")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("times", [1, 33])
def test_large_values_in_one_place(dev, kind, times):
    """All of the largest values next to one another (one lane's, one wave's, one workgroup's): the alternatives
    come from one place, in order."""
    c = 70001
    z = torch.randn((8, c), generator=torch.Generator().manual_seed(7))
    for r, a in enumerate([0, 8, 64, 500, 4096, 16000, 32768, c - 3000]):
        z[r, a:a + 3000] = torch.linspace(50.0, 20.0, 3000) if r % 2 else torch.linspace(20.0, 50.0, 3000)
    check(z.repeat(times, 1).to(TYPES[kind]).to(dev), (torch.arange(8, device=dev) * 5000).repeat(times), 32, grads=times == 1)


def test_more_rows_than_one_launch_takes(dev):
    """2^23 + 3 rows (one row's memory): the last rows' values and gradients are the first's."""
    n, c = (1 << 23) + 3, 300
    row, y = make(1, c, torch.bfloat16, dev, ignore_some=False)
    got = P.label_log_probs(row.expand(n, c), y.expand(n), top_k=8)
    for t in got:
        assert torch.equal(t[-5:], t[:1].expand(5, *t.shape[1:]))
    check(row.expand(4097, c), y.expand(4097), 8)
    x = row[:, :5].expand(n, 5).requires_grad_(True)
    r = P.label_log_probs(x, y.expand(n) % 5, top_k=2)
    dz, = torch.autograd.grad([r.log_prob, r.top_log_prob], x, [torch.ones_like(r.log_prob), torch.ones_like(r.top_log_prob)])
    assert torch.equal(dz[-5:], dz[:1].expand(5, 5)) and bool(dz.any())


@pytest.mark.parametrize("n,k", [(1 << 18, 0), ((1 << 18) + 5, 0), ((1 << 18) + 5, 3)])
def test_more_split_rows_than_one_launch_takes(dev, n, k):
    """Rows of 64 parts each (one row's memory), 2^24 parts and more: every row as the first, and as alone."""
    c = 524280
    row, y = make(1, c, torch.bfloat16, dev, ignore_some=False)
    got = P.label_log_probs(row.expand(n, c), y.expand(n), top_k=k)
    for t in got:
        assert torch.equal(t, t[:1].expand(n, *t.shape[1:]))
    want, tol = reference(row.cpu(), y.cpu().numpy(), k)
    near(got.log_prob[:1], want["lp"], tol["lp"], "log_prob")
    near(got.entropy[-1:], want["ent"], tol["ent"], "entropy")
    np.testing.assert_array_equal(got.top_index[-1:].cpu().numpy(), want["idx"])


def test_gradient_through_other_layouts(dev):
    """Logits that are a transposed, sliced or expanded leaf: the gradient comes back in the leaf's layout."""
    logits, y = make(6, 40, torch.float32, dev, ignore_some=False)
    x = logits.detach().clone().requires_grad_(True)
    want, = torch.autograd.grad(P.label_log_probs(x, y).log_prob.sum(), x)
    t = logits.t().contiguous().requires_grad_(True)
    got, = torch.autograd.grad(P.label_log_probs(t.t(), y).log_prob.sum(), t)
    torch.testing.assert_close(got.t(), want)
    w = torch.zeros((6, 50), device=dev)
    w[:, 3:43] = logits
    w.requires_grad_(True)
    got, = torch.autograd.grad(P.label_log_probs(w[:, 3:43], y).log_prob.sum(), w)
    torch.testing.assert_close(got[:, 3:43], want)
    assert not bool(got[:, :3].any()) and not bool(got[:, 43:].any())
    one = logits[:1].clone().requires_grad_(True)
    got, = torch.autograd.grad(P.label_log_probs(one.expand(6, 40), y).log_prob.sum(), one)
    each = [torch.autograd.grad(P.label_log_probs(one, y[i:i + 1]).log_prob.sum(), one)[0] for i in range(6)]
    torch.testing.assert_close(got, sum(each))


def test_partial_gradients(dev):
    """Each output alone, and expanded upstream gradients."""
    logits, y = make(37, 257, torch.float32, dev)
    full = []
    for part in range(3):
        x = logits.detach().clone().requires_grad_(True)
        r = P.label_log_probs(x, y, top_k=3)
        out = [r.log_prob, r.entropy, r.top_log_prob][part]
        dz, = torch.autograd.grad(out.sum(), x)
        up = [None, None, None]
        up[part] = np.ones((37, 3) if part == 2 else 37)
        want, tol = reference(logits.cpu(), y.cpu().numpy(), 3, *up)
        near(dz, want["dz"], tol["dz"], f"part {part}")
        full.append(dz)
    x = logits.detach().clone().requires_grad_(True)
    r = P.label_log_probs(x, y, top_k=3)
    dz, = torch.autograd.grad(r.log_prob.sum() + r.entropy.sum() + r.top_log_prob.sum(), x)
    torch.testing.assert_close(dz, sum(full), rtol=1e-4, atol=1e-5)


def test_gradient_against_differences(dev):
    """Central differences of the definition in 64 bits: error h^2/6 f''' + 2^-53 f / h, about 1e-9 at h = 1e-4
    for logits of order 1, far below the f32 tolerance of 2e-6."""
    n, c, k = 3, 23, 2
    logits, y = make(n, c, torch.float32, dev, ignore_some=False)
    logits = logits * 0.2
    rng = np.random.default_rng(3)
    up = [rng.normal(size=n), rng.normal(size=n), rng.normal(size=(n, k))]
    x = logits.detach().requires_grad_(True)
    r = P.label_log_probs(x, y, top_k=k)
    dz, = torch.autograd.grad(list(r[:3]), x, [torch.tensor(u, dtype=torch.float32, device=dev) for u in up])
    z0 = logits.double().cpu()
    idx = r.top_index.cpu()

    def value(z):
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        ent = -(logp.exp() * logp).sum(1)
        lp = logp.gather(1, y.cpu()[:, None])[:, 0]
        return float((lp * torch.tensor(up[0])).sum() + (ent * torch.tensor(up[1])).sum()
                     + (logp.gather(1, idx) * torch.tensor(up[2])).sum())

    h = 1e-4
    for i in range(n):
        for j in range(c):
            a, b = z0.clone(), z0.clone()
            a[i, j] += h
            b[i, j] -= h
            assert abs((value(a) - value(b)) / (2 * h) - float(dz[i, j])) <= 2e-6 * (1 + abs(float(dz[i, j])))


def test_same_bits_every_time(dev):
    for n, c in [(2000, 20), (64, 1003), (3, 140001)]:
        logits, y = make(n, c, torch.bfloat16, dev)
        runs = []
        for _ in range(3):
            x = logits.detach().clone().requires_grad_(True)
            r = P.label_log_probs(x, y, top_k=5)
            dz, = torch.autograd.grad([r.log_prob, r.entropy], x, [torch.ones_like(r.log_prob)] * 2)
            runs.append([*r, dz])
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_rows_do_not_depend_on_their_number(dev):
    """Few long rows are split over the chip, many are not: the values stay within the tolerances either way, the
    classes are the same."""
    logits, y = make(700, 9001, torch.float32, dev)
    whole = P.label_log_probs(logits, y, top_k=6)
    want, tol = reference(logits[:4].cpu(), y[:4].cpu().numpy(), 6)
    for m in (1, 2, 4):
        part = P.label_log_probs(logits[:m], y[:m], top_k=6)
        assert torch.equal(part.top_index, whole.top_index[:m])
        for r in (part, P.LabelLogProbs(*[t[:m] for t in whole])):
            near(r.log_prob, want["lp"][:m], tol["lp"][:m], "log_prob")
            near(r.entropy, want["ent"][:m], tol["ent"][:m], "entropy")


def test_places_past_32_bits(dev):
    """Rows more than 2^32 bytes and 2^31 elements apart."""
    c, far = 1003, (1 << 31) + 24
    buf = torch.empty((far + c,), dtype=torch.bfloat16, device=dev)
    z = buf.as_strided((2, c), (far, 1))
    logits, y = make(2, c, torch.bfloat16, dev)
    z.copy_(logits)
    # (a row's vectors begin where its address does, so the sums' order, and their last bits, go by the place)
    check(z, y, 5, grads=False)


def test_gradient_past_32_bits(dev):
    """A gradient of more than 2^31 elements: the last rows are the same as alone."""
    n, c = 4400, 500003
    z = torch.zeros((1, c), dtype=torch.bfloat16, device=dev)
    z[0, :1000] = torch.randn((1000,), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    x = z.expand(n, c).requires_grad_(True)
    y = torch.arange(n, device=dev)
    r = P.label_log_probs(x, y)
    dz, = torch.autograd.grad(r.log_prob, x, torch.ones((n,), device=dev))
    last = z.clone().requires_grad_(True)
    one, = torch.autograd.grad(P.label_log_probs(last, y[-1:]).log_prob, last, torch.ones((1,), device=dev))
    assert torch.equal(dz[-1], one[0])
    assert float(r.log_prob[-1]) == pytest.approx(float(P.label_log_probs(z, y[-1:]).log_prob), rel=1e-5)


def test_no_rows_and_other_label_types(dev):
    x = torch.empty((0, 50), device=dev, requires_grad=True)
    r = P.label_log_probs(x, torch.empty((0,), dtype=torch.int64, device=dev), top_k=2)
    assert r.log_prob.shape == (0,) and r.top_index.shape == (0, 2)
    dz, = torch.autograd.grad(r.log_prob.sum(), x)
    assert dz.shape == (0, 50)
    logits, y = make(9, 40, torch.float32, dev)
    a = P.label_log_probs(logits, y, top_k=1)
    b = P.label_log_probs(logits, y.to(torch.int32), top_k=1)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    other = torch.where(y == IGNORE, 39, y)
    c = P.label_log_probs(logits, other, ignore_index=39)
    assert torch.equal(c.log_prob[::3], torch.zeros_like(c.log_prob[::3]))


def test_on_another_stream(dev):
    s = torch.cuda.Stream()
    logits, y = make(40, 5003, torch.bfloat16, dev)
    want = P.label_log_probs(logits, y, top_k=5)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        x = (logits.float() * 1.0).to(torch.bfloat16)
        got = P.label_log_probs(x, y, top_k=5)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed(dev):
    """Two graphs of forward and gradient, replayed in turn with new inputs between eager calls."""
    graphs = []
    for n, c in [(5, 40001), (64, 1003), (300, 20)]:
        logits, y = make(n, c, torch.bfloat16, dev)
        x = logits.detach().clone().requires_grad_(True)
        up = torch.randn((n,), generator=torch.Generator().manual_seed(n)).to(dev)

        def run(x=x, y=y, up=up):
            r = P.label_log_probs(x, y, top_k=4)
            return [t.detach() for t in r] + list(torch.autograd.grad([r.log_prob, r.entropy], x, [up, up]))

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out, x, run))
    for turn in range(4):
        for g, out, x, run in graphs:
            with torch.no_grad():
                x.copy_(torch.roll(x, turn + 1, 1))
            want = [t.clone() for t in run()]
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_decoder_head_uses_it(dev):
    """Decoder.sem_label_log_prob against the head's own log_softmax, argmax and gradient."""
    cfg = P.Config(device=dev)
    torch.manual_seed(5)
    dec = P.Decoder(cfg, cfg.geo_mlp_hidden_dim, cfg.geo_mlp_level, 20)
    x = torch.randn((500, 11), device=dev)
    y = torch.randint(0, 20, (500,), device=dev)
    r = dec.sem_label_log_prob(x, y, top_k=1)
    logp = dec.sem_label_prob(x)
    torch.testing.assert_close(r.log_prob, logp.gather(1, y[:, None])[:, 0], rtol=1e-5, atol=1e-5)
    assert torch.equal(r.top_index[:, 0], dec.sem_label(x))
    (-r.log_prob.mean()).backward()
    mine = [p.grad.clone() for p in dec.parameters()]
    dec.zero_grad()
    torch.nn.functional.nll_loss(dec.sem_label_prob(x), y).backward()
    for a, p in zip(mine, dec.parameters()):
        torch.testing.assert_close(a, p.grad, rtol=1e-4, atol=1e-6)


def test_refusals(dev):
    z = torch.zeros((4, 10), device=dev)
    y = torch.zeros((4,), dtype=torch.int64, device=dev)
    for bad in (dict(top_k=11), dict(top_k=-1), dict(top_k=33)):
        with pytest.raises(ValueError, match="top_k"):
            P.label_log_probs(z, y, **bad)
    with pytest.raises(ValueError, match="labels"):
        P.label_log_probs(z, y[:3])
    with pytest.raises(ValueError, match="whole numbers"):
        P.label_log_probs(z, y.float())
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        P.label_log_probs(z.double(), y)
    with pytest.raises(ValueError, match="labels on"):
        P.label_log_probs(z, y.cpu())
    with pytest.raises(ValueError, match="classes"):
        P.label_log_probs(z[:, :0], y)
    x = z.clone().requires_grad_(True)
    r = P.label_log_probs(x, y)
    g, = torch.autograd.grad(r.log_prob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()
    r = P.label_log_probs(x, y)
    r.log_prob.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        r.entropy.sum().backward()
    r = P.label_log_probs(x, y)
    with torch.no_grad():
        x += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.log_prob.sum().backward()


def test_views_that_negate_and_forward_mode(dev):
    logits, y = make(9, 100, torch.float32, dev, ignore_some=False)
    x = logits.detach().clone().requires_grad_(True)
    r = P.label_log_probs(x, y, top_k=2)
    up = torch.randn((9,), generator=torch.Generator().manual_seed(1)).to(dev)
    want, = torch.autograd.grad(r.log_prob, x, up)
    n = torch._neg_view(-x)
    got = P.label_log_probs(n, y, top_k=2)
    assert n.is_neg() and all(torch.equal(a, b) for a, b in zip(got, r))
    g, = torch.autograd.grad(got.log_prob, x, torch._neg_view(-up))
    assert torch.equal(g, want)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        P.label_log_probs(fwd.make_dual(logits, torch.ones_like(logits)), y)


def test_unsigned_labels(dev):
    """Labels of 64 bits without a sign: those beyond int64 are no class, whatever ignore_index is."""
    logits, _ = make(6, 40, torch.float32, dev)
    y = torch.tensor([3, 39, 40, 0, 5, 7], device=dev)
    want = P.label_log_probs(logits, y, ignore_index=5)
    for kind in (torch.uint8, torch.uint16, torch.uint32, torch.uint64):
        got = P.label_log_probs(logits, y.to(kind), ignore_index=5)
        assert torch.equal(torch.nan_to_num(got.log_prob, nan=7.0), torch.nan_to_num(want.log_prob, nan=7.0))
    far = torch.from_numpy(np.array([2 ** 64 - 100, 2 ** 64 - 1, 2 ** 63, 2 ** 63 - 1, 2, 39], dtype=np.uint64)).to(dev)
    for ignore in (IGNORE, -1, -2 ** 63):
        got = P.label_log_probs(logits, far, ignore_index=ignore).log_prob
        assert torch.isnan(got).tolist() == [True] * 4 + [False] * 2
    got = P.label_log_probs(logits, far, ignore_index=2 ** 63 - 1).log_prob
    assert torch.isnan(got).tolist() == [True] * 3 + [False] * 3 and float(got[3]) == 0.0
    for ignore in (2 ** 63, 2 ** 64 - 100, -2 ** 63 - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            P.label_log_probs(logits, far, ignore_index=ignore)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.int16, torch.int8])
def test_labels_that_are_a_negating_view(dev, kind):
    logits, y = make(9, 100, torch.float32, dev)
    n = torch._neg_view((-y).to(kind))
    x = logits.detach().clone().requires_grad_(True)
    want, got = P.label_log_probs(x, y, top_k=2), P.label_log_probs(x, n, top_k=2)
    assert n.is_neg() and all(torch.equal(a, b) for a, b in zip(got, want))
    a, = torch.autograd.grad(want.log_prob.sum(), x)
    b, = torch.autograd.grad(got.log_prob.sum(), x)
    assert torch.equal(a, b)


def test_transforms_are_refused(dev):
    """torch.func's transforms and tensors without memory: an error before any launch, and nothing is left behind."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    logits, y = make(6, 70, torch.float32, dev, ignore_some=False)
    many, ys = logits.view(2, 3, 70), y.view(2, 3)
    loss = lambda z: P.label_log_probs(z, y).log_prob.sum()   # noqa: E731
    whole = lambda _: loss(logits)   # noqa: E731  (what it reads is no argument of the transform)
    calls = [lambda: torch.func.grad(loss)(logits), lambda: torch.func.vjp(loss, logits), lambda: torch.func.grad(lambda z: loss(logits) + z.sum())(logits),
             lambda: torch.func.vmap(lambda z, t: P.label_log_probs(z, t).log_prob)(many, ys),
             lambda: torch.func.vmap(lambda t: P.label_log_probs(logits[:3], t).log_prob)(ys),
             lambda: torch.func.vmap(lambda z: P.label_log_probs(z, ys[0], top_k=2).top_log_prob)(many),
             lambda: torch.func.vmap(whole)(many), lambda: torch.func.jvp(loss, (logits,), (torch.ones_like(logits),)),
             lambda: torch.func.functionalize(loss)(logits), lambda: torch.func.hessian(loss)(logits)]
    for call in calls:
        with pytest.raises(NotImplementedError, match="torch.func|forward-mode"):
            call()
    x = logits.detach().clone().requires_grad_(True)
    r = P.label_log_probs(x, y, top_k=2)
    for out, up in ((r.log_prob, torch.ones((3, 6), device=dev)), (r.top_log_prob, torch.ones((3, 6, 2), device=dev))):
        with pytest.raises(NotImplementedError, match="batched gradients"):
            torch.autograd.grad(out, x, up, is_grads_batched=True, retain_graph=True)
    dz, = torch.autograd.grad(r.log_prob.sum(), x)   # the graph is as it was
    assert bool(dz.any())
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = mode.from_tensor(logits)
        with pytest.raises(NotImplementedError, match="without memory"):
            P.label_log_probs(fake, mode.from_tensor(y))
    want, tol = reference(logits.cpu(), y.cpu().numpy(), 2)
    near(P.label_log_probs(logits, y, top_k=2).log_prob, want["lp"], tol["lp"], "log_prob")


def test_under_torch_compile(dev):
    """The graph breaks there: values and gradients are the eager call's."""
    logits, y = make(30, 70, torch.float32, dev)

    def loss(z, t):
        r = P.label_log_probs(z * 2.0, t, top_k=2)
        return -r.log_prob.sum() + 0.1 * r.entropy.sum() + r.top_log_prob[:, 1].sum()

    for backend in ("eager", "aot_eager"):
        torch._dynamo.reset()
        fast = torch.compile(loss, backend=backend)
        for turn in range(3):
            x, q = (logits.detach().clone().add_(turn).requires_grad_(True) for _ in range(2))
            a, b = loss(x, y), fast(q, y)
            a.backward()
            b.backward()
            assert torch.equal(a, b) and torch.equal(x.grad, q.grad)
    torch._dynamo.reset()


def test_the_node_in_torchs_graph(dev):
    """What torch does with any operator's results: kept graphs, results changed in place, hooks, checkpoints, anomaly
    checks, results and graphs that go without a backward pass."""
    logits, y = make(12, 100, torch.float32, dev, ignore_some=False)
    x = logits.detach().clone().requires_grad_(True)
    r = P.label_log_probs(x, y, top_k=2)
    assert r.log_prob.grad_fn is not None and r.top_index.grad_fn is None and not r.top_index.requires_grad
    want, = torch.autograd.grad(r.log_prob.sum(), x, retain_graph=True)
    again, = torch.autograd.grad(r.log_prob.sum(), x)
    assert torch.equal(want, again)
    r = P.label_log_probs(x, y, top_k=2)
    r.log_prob.mul_(2.0)   # its own result: nothing of the node's
    got, = torch.autograd.grad(r.log_prob.sum(), x)
    torch.testing.assert_close(got, 2 * want, rtol=1e-6, atol=1e-6)
    seen = []
    r = P.label_log_probs(x, y)
    r.log_prob.register_hook(lambda g: seen.append(g) or 3 * g)
    got, = torch.autograd.grad(r.log_prob.sum(), x)
    torch.testing.assert_close(got, 3 * want, rtol=1e-6, atol=1e-6)
    assert len(seen) == 1
    from torch.utils.checkpoint import checkpoint
    for reentrant in (False, True):
        out = checkpoint(lambda t: P.label_log_probs(t * 1.0, y, top_k=2).log_prob, x, use_reentrant=reentrant)
        out.sum().backward()
        assert torch.equal(x.grad, want)
        x.grad = None
    with torch.autograd.graph.save_on_cpu():
        out = P.label_log_probs((x.t() * 1.0).t(), y, top_k=2).log_prob.sum()
    got, = torch.autograd.grad(out, x)
    assert torch.equal(got, want)
    with torch.autograd.detect_anomaly(check_nan=True):
        got, = torch.autograd.grad(P.label_log_probs(x, y).log_prob.sum(), x)
    assert torch.equal(got, want)
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        P.label_log_probs(x, y, top_k=2)
    assert torch.cuda.memory_allocated() == before
    with torch.inference_mode():
        assert not P.label_log_probs(x, y).log_prob.requires_grad
