"""Softmax read-out on the GPU against its definition in 64 bits.

Tolerances.  u = 2^-53 (float64 scores) or 2^-24.  A difference to the row's maximum times the scale is rounded twice (the
scale once more), so log p carries 3 u |d| from its own difference; a term exp(d) carries |d| u (its argument) + 2 u, in the
mean over p at most log V u, and a serial sum of L = V / 256 + 64 terms of one sign (L + 10) u.  log1p and the last
subtraction add 2 u of |log p| and of log1p.  Together  u (4 |log p| + L + 128)  for a log probability,
u (L + 128) (2 + log V)  for an entropy (a sum of terms p |log p| over as many partial sums), and for a gradient the
same relative error of p and of log p + H, plus half a step of the type it is stored in."""
import math

import numpy as np
import pytest

import vqa_amd
from vqa_amd import _lib

pytestmark = pytest.mark.gpu

TYPES = ["float64", "float32", "bfloat16", "float16"]


def unit(t):
    return 2.0 ** -53 if t == "float64" else 2.0 ** -24


def half_step(t):
    import torch

    return torch.finfo(getattr(torch, t)).eps / 2


def scores(rng, rows, width, t, masked=0.1, spread=2.5):
    import torch

    z = spread * rng.standard_normal((rows, width))
    z[rng.random((rows, width)) < masked] = -np.inf
    return torch.from_numpy(z).to(getattr(torch, t)).cuda()


def reference(z, targets, scale, k):
    """numpy, 64 bits; a row at a time in the plainest words"""
    z = z.double().cpu().numpy()
    R, V = z.shape
    lp, ent = np.zeros(R), np.zeros(R)
    top, ix = np.full((R, k), -np.inf), np.full((R, k), -1, np.int64)
    logs = np.full((R, V), -np.inf)
    for r in range(R):
        t = None if targets is None else int(targets[r])
        if np.isnan(z[r]).any() or (z[r] == np.inf).any() or (t is not None and t >= V):
            lp[r] = ent[r] = np.nan
            top[r], logs[r] = np.nan, np.nan
            continue
        live = z[r] > -np.inf
        if live.any():
            x = scale * z[r][live]
            m = x.max()
            ls = math.log(math.fsum(np.exp(x - m)))
            logs[r, live] = x - m - ls
            p = np.exp(logs[r, live])
            ent[r] = -math.fsum(p[p > 0] * logs[r, live][p > 0])
        if t is not None and t >= 0:
            lp[r] = logs[r, t]
        order = np.argsort(-z[r], kind="stable")
        order = order[z[r][order] > -np.inf][:k]
        ix[r, :len(order)], top[r, :len(order)] = order, logs[r, order]
    return lp, ent, top, ix, logs


def near(got, want, tol):
    """finite values within tol, NaN and infinities in the same places"""
    got, want, tol = np.asarray(got, float), np.asarray(want, float), np.broadcast_to(tol, np.shape(want))
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(got[fine] - want[fine])
    assert (off <= tol[fine]).all(), (off - tol[fine]).max()


def tolerances(t, V, lp):
    u, L = unit(t), V / 256 + 64
    with np.errstate(invalid="ignore"):
        a = np.where(np.isfinite(lp), u * (4 * np.abs(lp) + L + 128), 0.0)
    return a, u * (L + 128) * (2 + math.log(V))


WIDTHS = [1, 2, 3, 4, 5, 12, 16, 17, 63, 64, 65, 200, 256, 257, 1000, 1024, 1025, 2049, 5000, 8191, 20011]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", WIDTHS)
def test_score_matches_the_definition(t, V):
    rng = np.random.default_rng(V)
    R = 9 if V < 5000 else 4
    z = scores(rng, R, V, t)
    tg = rng.integers(-1, V, R)
    k = min(V, 20, 64)
    import torch

    r = vqa_amd.log_probs(z, torch.from_numpy(tg).cuda(), top_k=k, scale=1.7)
    lp, ent, top, ix, _ = reference(z, tg, 1.7, k)
    a, b = tolerances(t, V, lp)
    near(r.log_prob.cpu(), lp, a)
    near(r.entropy.cpu(), ent, b)
    assert np.array_equal(r.top_index.cpu().numpy(), ix)
    near(r.top_log_prob.cpu(), top, tolerances(t, V, top)[0])
    assert r.entropy.dtype == (torch.float64 if t == "float64" else torch.float32) and r.top_index.dtype == torch.int32


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [1, 3, 16, 65, 1000, 1025, 4099, 20011])
def test_gradient_matches_the_formula(t, V):
    import torch

    rng = np.random.default_rng(V + 1)
    R = 7 if V < 5000 else 3
    z = scores(rng, R, V, t)
    tg = rng.integers(-1, V, R)
    g, h = rng.standard_normal(R), rng.standard_normal(R)
    scale = 0.8
    wide = torch.float64 if t == "float64" else torch.float32
    gt, ht = (torch.from_numpy(v).to(wide).cuda() for v in (g, h))
    r = vqa_amd.log_probs_grad(z, torch.from_numpy(tg.astype(np.int32)).cuda(), gt, ht, scale=scale)
    lp, ent, _, _, logs = reference(z, tg, scale, 0)
    near(r.log_prob.cpu(), lp, tolerances(t, V, lp)[0])
    near(r.entropy.cpu(), ent, tolerances(t, V, lp)[1])
    g, h = gt.double().cpu().numpy(), ht.double().cpu().numpy()
    p = np.exp(logs)
    want, tol = np.zeros_like(p), np.zeros_like(p)
    u, L = unit(t), V / 256 + 64
    for i in range(R):
        live = logs[i] > -np.inf
        gi = g[i] if tg[i] >= 0 else 0.0
        want[i, live] = -gi * p[i, live] - h[i] * p[i, live] * (logs[i, live] + ent[i])
        size = np.zeros(V)
        size[live] = (abs(gi) * p[i, live] + abs(h[i]) * p[i, live] * (np.abs(logs[i, live]) + ent[i] + 1)) * (4 * np.abs(logs[i, live]) + L + 128)
        size *= 2 + math.log(V)              # the entropy's error
        if tg[i] >= 0 and live.any():        # (a row with everything masked has gradient 0)
            want[i, tg[i]] += gi
            size[tg[i]] += 4 * abs(gi)
        tol[i] = u * scale * size
    want *= scale
    # stored: half a step of the value, or of the smallest normal number below it
    f = torch.finfo(getattr(torch, t))
    tol += half_step(t) * (np.abs(want) + tol) + f.smallest_normal * f.eps + 1e-38
    near(r.d_logits.double().cpu(), want, tol)
    assert r.d_logits.dtype == z.dtype


def special_rows(z, V):
    z[0] = -np.inf
    z[1] = -np.inf
    z[1, V - 1] = 2.0
    z[2, V // 2] = float("nan")
    z[3, 0] = float("inf")
    z[4] = 1.5
    z[5, V - 1] = float("nan")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("R,V", [(600, 1031), (513, 4100), (520, 8192), (512, 8193), (130, 2047), (129, 16001), (140, 33333), (130, 70001),
                                 (128, 131075), (1100, 20011)])
def test_many_rows(t, R, V):
    """the forms that take a row a wave and a row a workgroup, on every eighth row and the special ones"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(R + V)
    z = torch.randn(R, V, device="cuda", generator=gen, dtype=torch.float64) * 2.5
    z[torch.rand(R, V, device="cuda", generator=gen) < 0.1] = -np.inf
    z = z.to(getattr(torch, t))
    special_rows(z, V)
    tg = torch.randint(-1, V, (R,), device="cuda", generator=gen)
    rows = torch.cat([torch.arange(6), torch.arange(6, R, max(8, R // 12))]).tolist()
    k = 17
    scale = 0.9
    g, h = 0.7, -0.4
    r = vqa_amd.log_probs(z, tg, top_k=k, scale=scale)
    d = vqa_amd.log_probs_grad(z, tg, g, h, scale=scale)
    tgn = tg.cpu().numpy()[rows]
    lp, ent, top, ix, logs = reference(z[rows], tgn, scale, k)
    a, b = tolerances(t, V, lp)
    for o in (r, d):
        near(o.log_prob.cpu()[rows], lp, a)
        near(o.entropy.cpu()[rows], ent, b)
    assert np.array_equal(r.top_index.cpu().numpy()[rows], ix)
    near(r.top_log_prob.cpu()[rows], top, tolerances(t, V, top)[0])
    p = np.exp(logs)
    u, L = unit(t), V / 256 + 64
    f = torch.finfo(z.dtype)
    gw, hw = (float(torch.tensor(x, dtype=r.entropy.dtype)) for x in (g, h))
    for n, i in enumerate(rows):
        got = d.d_logits[i].double().cpu().numpy()
        if np.isnan(ent[n]):
            assert np.isnan(got).all()
            continue
        live = logs[n] > -np.inf
        gi = gw if tgn[n] >= 0 else 0.0
        want, size = np.zeros(V), np.zeros(V)
        want[live] = -gi * p[n, live] - hw * p[n, live] * (logs[n, live] + ent[n])
        size[live] = (abs(gi) * p[n, live] + abs(hw) * p[n, live] * (np.abs(logs[n, live]) + ent[n] + 1)) * (4 * np.abs(logs[n, live]) + L + 128)
        size *= 2 + math.log(V)
        if tgn[n] >= 0 and live.any():
            want[tgn[n]] += gi
            size[tgn[n]] += 4 * abs(gi)
        tol = u * scale * size
        tol += half_step(t) * (np.abs(scale * want) + tol) + f.smallest_normal * f.eps + 1e-38
        near(got, scale * want, tol)


@pytest.mark.parametrize("V", [5, 700, 6000])
def test_gradient_matches_differences(V):
    """central differences of the loss, float64: the third derivative is below 4 scale^3, so a step of 1e-4 leaves 1e-8, and
    the loss's own rounding 2^-52 * 10 / 1e-4 = 2e-11"""
    import torch

    rng = np.random.default_rng(3)
    R = 2
    z = scores(rng, R, V, "float64", masked=0.0, spread=1.0)
    tg = torch.tensor([1, V - 1], dtype=torch.int32).cuda()
    g, h = torch.tensor([0.7, -1.1], dtype=torch.float64).cuda(), torch.tensor([0.4, 0.9], dtype=torch.float64).cuda()

    def value(zz):
        r = vqa_amd.log_probs(zz, tg, scale=1.3)
        return float((g * r.log_prob + h * r.entropy).sum())

    d = vqa_amd.log_probs_grad(z, tg, g, h, scale=1.3).d_logits
    for r in range(R):
        for c in {0, 1, V // 2, V - 1}:
            e = torch.zeros_like(z)
            e[r, c] = 1e-4
            assert abs((value(z + e) - value(z - e)) / 2e-4 - float(d[r, c])) < 4e-8


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [4, 100, 1000, 3000, 9000])
def test_rows_that_are_special(t, V):
    import torch

    rng = np.random.default_rng(5)
    z = scores(rng, 12, V, t, masked=0.0)
    z[0] = -np.inf                       # nothing left
    z[1] = -np.inf
    z[1, V - 1] = 2.0                    # one outcome left
    z[2, V // 2] = float("nan")
    z[3, 0] = float("inf")
    z[4] = 1.5                           # all equal: the lowest indices
    z[5] = -np.inf
    z[5, 1], z[5, 3] = -3.0, -3.0
    z[6, :] = float("nan")
    z[7, V - 1] = float("inf")
    z[7, V - 2] = float("inf")
    z[8] = -torch.finfo(z.dtype).max     # the type's lowest value is a score like any other
    z[9, 1:] = -torch.finfo(z.dtype).max
    z[9, 0] = torch.finfo(z.dtype).max
    tg = np.array([1, 0, 0, 0, V - 1, 3, 0, 1, 2, 0, V, 2 ** 31 - 1])
    k = 4
    for targets in (torch.from_numpy(tg).cuda(), torch.from_numpy(tg.astype(np.int32)).cuda()):
        r = vqa_amd.log_probs(z, targets, top_k=k)
        lp, ent, top, ix, logs = reference(z, tg, 1.0, k)
        a, b = tolerances(t, V, lp)
        near(r.log_prob.cpu(), lp, a)
        near(r.entropy.cpu(), ent, b)
        assert np.array_equal(r.top_index.cpu().numpy(), ix)
        rows = [i for i in range(12) if i != 9]
        near(r.top_log_prob.cpu()[rows], top[rows], tolerances(t, V, top)[0][rows])
        assert float(r.top_log_prob[9, 0]) == 0.0
        d = vqa_amd.log_probs_grad(z, targets, 1.0, 0.5)
        dz = d.d_logits.double().cpu().numpy()
        assert (dz[0, [c for c in range(V) if c != 1]] == 0).all() and dz[0, 1] == 0      # nothing left: no gradient
        for i in (2, 3, 6, 7, 10, 11):
            assert np.isnan(dz[i]).all()
        assert np.isfinite(dz[[1, 4, 5, 8, 9]]).all()
        assert (dz[1, 1:V - 1] == 0).all() and dz[1, 0] == 1.0 and dz[1, V - 1] == -1.0   # target is masked: its delta alone


def test_one_outcome_far_ahead_keeps_its_small_log_probability():
    """log p = -log1p(s) with s = 2^-40 (V - 1) e-fold parts: relative accuracy, not absolute"""
    import torch

    for V in (3, 500, 5000):
        for t in ("float64", "float32"):
            z = torch.zeros(1, V, dtype=getattr(torch, t)).cuda()
            z[0, V - 1] = 30.0
            r = vqa_amd.log_probs(z, torch.tensor([V - 1]).cuda(), top_k=1)
            want = -math.log1p((V - 1) * math.exp(-30.0))
            # exp(-30) from a rounded argument: 30 u; a sum of V terms of one sign
            assert abs(float(r.log_prob[0]) - want) <= unit(t) * (64 + V / 256 + 64) * abs(want)
            assert abs(float(r.entropy[0]) - (-want + (V - 1) * math.exp(-30.0) * 30 / (1 + (V - 1) * math.exp(-30.0)))) <= 2 * unit(t) * (64 + V / 256 + 64) * 31 * abs(want) + 1e-25


@pytest.mark.parametrize("V", [13, 600, 4100, 30000])
@pytest.mark.parametrize("t", TYPES)
def test_top_outcomes_with_many_ties(t, V):
    import torch

    rng = np.random.default_rng(V)
    z = torch.from_numpy(rng.integers(0, 6, (5, V)).astype(np.float64)).to(getattr(torch, t)).cuda()
    z[1] = torch.arange(V).to(z.dtype).cuda().clamp(max=2048)        # ascending: every element is a new best one
    z[2] = -z[1]
    for k in {1, 2, min(13, V), min(64, V)}:
        r = vqa_amd.log_probs(z, top_k=k)
        assert r.log_prob is None
        _, _, _, ix, _ = reference(z, None, 1.0, k)
        assert np.array_equal(r.top_index.cpu().numpy(), ix), k


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("copies,V", [(1, 1100), (1, 9000), (1, 140000), (40, 3000), (2, 8192), (64, 5001)])
@pytest.mark.parametrize("k", [1, 7, 33, 64])
def test_top_outcomes_of_rows_in_any_order(t, copies, V, k):
    """rows in order, in reverse, all alike, of two or a few values, with everything but a few masked, close together beside
    one far away: the same outcomes as a stable sort, however many candidates there are at once"""
    import torch

    rng = np.random.default_rng(V + k)
    up = np.arange(V) / 64.0
    rows = [up, up[::-1], np.zeros(V), np.full(V, -3.0), (np.arange(V) % 2).astype(float), (np.arange(V) // 700).astype(float),
            rng.integers(0, 3, V).astype(float), np.where(rng.random(V) < 20 / V, 1.0, -np.inf), np.full(V, -np.inf),
            np.where(np.arange(V) == V // 2, 6e4, 1.0 + np.arange(V) * 2.0 ** -17), rng.standard_normal(V), np.sort(rng.standard_normal(V))]
    z = torch.from_numpy(np.stack(rows)).to(getattr(torch, t)).cuda().repeat(copies, 1)
    r = vqa_amd.log_probs(z, top_k=k)
    first = z[:len(rows)].double().cpu().numpy()
    want = np.argsort(-first, axis=1, kind="stable")[:, :k]
    want = np.where(np.take_along_axis(first, want, 1) == -np.inf, -1, want)
    assert np.array_equal(r.top_index.cpu().numpy(), np.tile(want, (copies, 1)))


@pytest.mark.parametrize("t", ["float64", "bfloat16"])
@pytest.mark.parametrize("V,stride,first", [(3, 7, 1), (100, 105, 3), (1500, 1507, 5), (9001, 9100, 7)])
def test_strided_rows_and_unaligned_starts(t, V, stride, first):
    import torch

    rng = np.random.default_rng(1)
    big = scores(rng, 6, stride, t)
    big[:, first + V:] = float("nan")              # padding may hold anything
    big[:, :first] = float("nan")
    z = big[:, first:first + V]
    keep = z.clone()
    tg = torch.from_numpy(rng.integers(0, V, 6)).cuda()
    out = torch.full((6, stride), 7.0, dtype=z.dtype).cuda()
    a = vqa_amd.log_probs_grad(z, tg, 1.0, 0.3, out=out[:, 1:1 + V])
    b = vqa_amd.log_probs_grad(keep.contiguous(), tg, 1.0, 0.3)
    # the same sums: a part of a row begins at another piece of memory, so the order may differ by an element or two
    u = unit(t) * (V / 256 + 200) * (2 + math.log(V)) * 20
    near(a.log_prob.cpu(), b.log_prob.double().cpu(), u)
    near(a.entropy.cpu(), b.entropy.double().cpu(), u)
    assert (a.d_logits.double() - b.d_logits.double()).abs().max() <= u + 2 * half_step(t)
    left = torch.ones(stride, dtype=torch.bool)
    left[1:1 + V] = False
    assert (out[:, left.cuda()] == 7.0).all()       # what lies between the rows is as it was
    for zz in (z.t().contiguous().t(), z[::2]):     # columns apart, rows skipped
        r = vqa_amd.log_probs(zz, top_k=2)
        s = vqa_amd.log_probs(zz.contiguous(), top_k=2)
        assert torch.equal(r.top_index, s.top_index)


@pytest.mark.parametrize("t", ["float64", "float16"])
@pytest.mark.parametrize("R,V", [(5, 7), (130, 1500), (3, 5000)])
def test_scores_and_gradient_in_one_array(t, R, V):
    """columns of one array hold the scores, others take the gradient; the columns between stay"""
    import torch

    big = torch.full((R, 2 * V + 5), 3.0, dtype=getattr(torch, t)).cuda()
    big[:, 1:V + 1] = scores(np.random.default_rng(V), R, V, t)
    z, out = big[:, 1:V + 1], big[:, V + 3:2 * V + 3]
    tg = torch.zeros(R, dtype=torch.int32).cuda()
    want = vqa_amd.log_probs_grad(z, tg, -1.0, 0.2)     # (the same addresses: where a row begins decides which lane adds what)
    got = vqa_amd.log_probs_grad(z, tg, -1.0, 0.2, out=out)
    assert torch.equal(got.d_logits, want.d_logits) and torch.equal(got.log_prob, want.log_prob)
    assert (big[:, 0] == 3).all() and (big[:, V + 1:V + 3] == 3).all() and (big[:, 2 * V + 3:] == 3).all()
    with pytest.raises(_lib.VqaError):
        vqa_amd.log_probs_grad(z, tg, -1.0, 0.2, out=big[:, 2:V + 2])


def test_expanded_rows_and_one_number_weights():
    import torch

    z = torch.randn(1, 50, dtype=torch.float64).cuda().expand(4, 50)
    r = vqa_amd.log_probs_grad(z, torch.tensor([0, 1, 2, -1]).cuda(), -0.25)
    s = vqa_amd.log_probs_grad(z.contiguous(), torch.tensor([0, 1, 2, -1]).cuda(), torch.full((4,), -0.25, dtype=torch.float64).cuda())
    assert torch.equal(r.d_logits, s.d_logits) and (r.d_logits[3] == 0).all()


@pytest.mark.parametrize("R,V", [(0, 10), (1, 1), (3000, 3), (1, 300000), (70, 4096 * 3), (20000, 40)])
def test_counts_of_rows(R, V):
    import torch

    rng = np.random.default_rng(R + V)
    z = scores(rng, R, V, "float32")
    tg = torch.from_numpy(rng.integers(-1, V, R)).cuda()
    r = vqa_amd.log_probs(z, tg, top_k=min(3, V))
    d = vqa_amd.log_probs_grad(z, tg, 1.0, 0.1)
    assert r.log_prob.shape == (R,) and d.d_logits.shape == (R, V)
    if R:
        x = z.double()
        want = torch.log_softmax(x, 1).nan_to_num(nan=-np.inf, neginf=-np.inf)      # (rows with everything masked)
        got = r.log_prob.double()
        t = tg.clamp(min=0)
        ref = torch.where(tg < 0, torch.zeros_like(got), want.gather(1, t[:, None])[:, 0])
        lp = ref.cpu().numpy()
        near(got.cpu(), lp, tolerances("float32", V, lp)[0])
        # the same sums in the same order (the loss reads the row as the scoring call does), up to the top list
        near(d.log_prob.cpu(), lp, tolerances("float32", V, lp)[0])


@pytest.mark.parametrize("dt", [np.float64, np.float32, np.float16])
def test_host_pointer_path_equals_the_device_path(dt):
    import torch

    rng = np.random.default_rng(2)
    for V in (3, 2000):
        z = rng.standard_normal((11, V)).astype(dt)
        tg = rng.integers(-1, V, 11)
        a = vqa_amd.log_probs(z, tg, top_k=3, scale=2.0)
        b = vqa_amd.log_probs(torch.from_numpy(z).cuda(), torch.from_numpy(tg).cuda(), top_k=3, scale=2.0)
        assert all(np.array_equal(x, y.cpu().numpy()) for x, y in zip(a, b))
        a = vqa_amd.log_probs_grad(z, tg, -1 / 11, 0.5)
        b = vqa_amd.log_probs_grad(torch.from_numpy(z).cuda(), torch.from_numpy(tg).cuda(), -1 / 11, 0.5)
        assert all(np.array_equal(x, y.cpu().numpy()) for x, y in zip(a, b))
        assert a.d_logits.dtype == dt
    got = vqa_amd.log_probs(np.arange(6).reshape(2, 3))         # whole numbers are taken as float64
    assert got.entropy.dtype == np.float64
    assert vqa_amd.log_probs(np.zeros((0, 3))).entropy.shape == (0,)


def test_the_same_call_gives_the_same_bits_on_any_stream():
    import torch

    z = scores(np.random.default_rng(0), 3, 150000, "bfloat16")
    tg = torch.tensor([1, 2, 3]).cuda()
    a = vqa_amd.log_probs(z, tg, top_k=30)
    a2 = vqa_amd.log_probs_grad(z, tg, 1.0, 1.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = vqa_amd.log_probs(z, tg, top_k=30)
        b2 = vqa_amd.log_probs_grad(z, tg, 1.0, 1.0)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(a2, b2))


@pytest.mark.parametrize("R,V", [(1, 131072), (7, 40000), (600, 3000)])
def test_calls_at_the_same_time(R, V):
    """queued on three streams without waiting, each call's workspace is its own"""
    import torch

    zs = [scores(np.random.default_rng(k), R, V, "float32") for k in range(3)]
    tg = torch.zeros(R, dtype=torch.int32).cuda()
    want = [(vqa_amd.log_probs(z, tg, top_k=20), vqa_amd.log_probs_grad(z, tg, -1.0, 0.1)) for z in zs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in zs]
    got = [[], [], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append((vqa_amd.log_probs(zs[k], tg, top_k=20), vqa_amd.log_probs_grad(zs[k], tg, -1.0, 0.1)))
    torch.cuda.synchronize()
    for k in range(3):
        for a, b in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(a, want[k][0])) and all(torch.equal(x, y) for x, y in zip(b, want[k][1]))


@pytest.mark.parametrize("V", [12, 40000])
def test_captured_calls_replay_with_new_scores(V):
    """two graphs of the same call, each with its own memory, replayed in turn with eager work between"""
    import torch

    rng = np.random.default_rng(8)
    data = [scores(rng, 5, V, "float32") for _ in range(4)]
    tg = torch.from_numpy(rng.integers(0, V, 5).astype(np.int32)).cuda()
    g = torch.full((5,), -0.2).cuda()
    z = data[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        vqa_amd.log_probs(z, tg, top_k=5)
        vqa_amd.log_probs_grad(z, tg, g)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append((vqa_amd.log_probs(z, tg, top_k=5), vqa_amd.log_probs_grad(z, tg, g)))
        graphs.append(gr)
    for n in range(6):
        z.copy_(data[n % 4])
        graphs[n % 2].replay()
        want = vqa_amd.log_probs(data[n % 4], tg, top_k=5), vqa_amd.log_probs_grad(data[n % 4], tg, g)
        torch.cuda.synchronize()
        got = outs[n % 2]
        assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b)), n


def test_the_current_device_and_bad_devices():
    import torch

    assert torch.cuda.current_device() == 0
    L = _lib.lib()
    z = torch.zeros(2, 3, dtype=torch.float64).cuda()
    ent = torch.zeros(2, dtype=torch.float64).cuda()
    assert L.vqa_log_probs_dev(99, None, 0, z.data_ptr(), 2, 3, 3, 1.0, None, 0, None, None, ent.data_ptr(), None, None) == _lib.ENODEVICE
    assert L.vqa_log_probs_dev(-1, None, 0, z.data_ptr(), 2, 3, 3, 1.0, None, 0, None, None, ent.data_ptr(), None, None) == _lib.ENODEVICE
    assert torch.cuda.current_device() == 0
    with pytest.raises(ValueError):
        vqa_amd.log_probs(z, torch.zeros(2, dtype=torch.int32))          # targets on the host
    with pytest.raises(ValueError):
        vqa_amd.log_probs(z.to(torch.int32))
    with pytest.raises(_lib.VqaError):
        vqa_amd.log_probs_grad(z, torch.zeros(2, dtype=torch.int32).cuda(), 1.0, out=z)


def test_large_offsets():
    """rows that start beyond 2^31 elements: 40 rows 2^26 elements apart, 16-bit (5.4 GB)"""
    import torch

    if torch.cuda.mem_get_info()[0] < 8e9:
        pytest.skip("needs 8 GB")
    big = torch.empty(40 * 2 ** 26, dtype=torch.float16, device="cuda")
    z = big.view(40, 2 ** 26)[:, :5000]
    z.copy_(torch.randn(40, 5000, device="cuda"))
    tg = torch.arange(40, device="cuda")
    a = vqa_amd.log_probs(z, tg, top_k=4)
    b = vqa_amd.log_probs(z.contiguous(), tg, top_k=4)
    assert torch.equal(a.top_index, b.top_index)
    assert (a.log_prob - b.log_prob).abs().max() < 1e-5
    c = vqa_amd.log_probs_grad(z.contiguous(), tg, 1.0, 0.0, out=z)
    # written to the rows of `out`: every row of a softmax's gradient sums to 0 up to its 5000 roundings
    assert c.d_logits.data_ptr() == z.data_ptr() and c.d_logits.double().sum(1).abs().max() < 0.05


# ---- the chain into circuit parameters, and the classifier's loss -------------------------------------------------


@pytest.mark.parametrize("B,P,n_obs", [(1, 1, 1), (3, 5, 3), (64, 64, 2), (65, 65, 12), (1000, 37, 3), (9000, 20, 3), (0, 4, 2)])
def test_chain_matches_numpy(B, P, n_obs):
    import torch

    rng = np.random.default_rng(B + P)
    E, d = rng.standard_normal((B, 2 * P + 1, n_obs)), rng.standard_normal((B, n_obs))
    got = vqa_amd.psr_chain(torch.from_numpy(E).cuda(), torch.from_numpy(d).cuda()).cpu().numpy()
    want = 0.5 * np.einsum("bo,bio->i", d, E[:, 1::2] - E[:, 2::2])
    # B * n_obs terms of size up to |d| |E| * 2, in any order
    size = 0.5 * np.einsum("bo,bio->i", np.abs(d), np.abs(E[:, 1::2]) + np.abs(E[:, 2::2]))
    assert (np.abs(got - want) <= 2.0 ** -52 * (B * n_obs + 4) * size + 1e-300).all()


def classifier(n_train=24, **kw):
    from vqa_amd.qml_utils import create_ibm_HEA_ansatz
    from vqa_amd.qnn_classifier import myQNN_classifier

    rng = np.random.default_rng(4)
    c = create_ibm_HEA_ansatz(4, 2, seed=1)
    x, y = rng.uniform(0, 1, (n_train + 6, 4)), rng.integers(0, 3, n_train + 6)
    q = myQNN_classifier(4, c, x[:n_train], y[:n_train], x[n_train:], y[n_train:], **kw)
    return q, rng.uniform(-3, 3, q.n_params)


def test_softmax_loss_of_the_classifier():
    """loss and gradient against the class probabilities' own softmax in numpy, and against differences of the loss"""
    q, p = classifier()
    q.softmax_scale, q.entropy_weight = 3.0, 0.05
    pr = q._exact_probs(p, which="train")
    x = 3.0 * pr
    lg = x - x.max(1, keepdims=True)
    lg -= np.log(np.exp(lg).sum(1, keepdims=True))
    ent = -(np.exp(lg) * lg).sum(1)
    want = -lg[np.arange(len(lg)), q.y_train].mean() - 0.05 * ent.mean()
    assert abs(q._softmax_CE(p, "train") - want) < 1e-13
    assert set(q.exact_softmax_CE_to_track(p)) == {"test", "train"}
    g = q.softmax_CE_grad_eval(p, mini_batch_size=len(q.x_train))
    assert q.shots_counter[0] == 0 and q.circuit_counter[0] == 24 * (2 * len(p) + 1)
    for i in range(0, len(p), 5):
        e = np.zeros_like(p)
        e[i] = 1e-4
        # the loss is a trigonometric polynomial through a softmax of scale 3: third derivative below 3^3 * 4
        assert abs((q._softmax_CE(p + e, "train") - q._softmax_CE(p - e, "train")) / 2e-4 - g[i]) < 2e-7
    r = q.softmax_log_probs(q.x_test, p, labels=q.y_test, top_k=2)
    pt = q._exact_probs(p, which="test")
    assert np.array_equal(r.top_index, np.argsort(-pt, axis=1, kind="stable")[:, :2])


def test_fit_with_the_softmax_loss_and_an_orthogonalised_optimizer():
    """compile / fit reach the read-out, its gradient and the orthogonalised step; the trajectory is the one of the same
    formulas written out here"""
    q, p = classifier()
    n_steps = 4
    q.compile(optimizer="Muon", loss="softmax_cross_entropy", hpara=dict(LR_rule=0.05, batch_size_rule=24, s_list_rule=1), init_params=p,
              softmax_scale=2.0, entropy_weight=0.01)
    res = q.fit(options=dict(max_iter=n_steps), auto_save=False)
    path = np.array(res["para_evol"])
    assert path.shape == (n_steps + 1, len(p)) and np.isfinite(path).all()
    assert q.shots_counter[0] == 0 and isinstance(res["func_evol"][-1], dict)
    from vqa_amd.optimizers import map_to_pi_range

    m, w = np.zeros((3, 12)), p.copy()
    for n in range(n_steps):
        g = q.softmax_CE_grad_eval(w, mini_batch_size=24).reshape(3, 12)
        m = 0.95 * m + g
        u = g + 0.95 * m
        U, S, Vt = np.linalg.svd(u / (np.linalg.norm(u) + 1e-7), full_matrices=False)
        for _ in range(5):
            S = S * (3.4445 + S * S * (-4.7750 + 2.0315 * S * S))
        w = map_to_pi_range(w - 0.05 * ((U * S) @ Vt).reshape(-1), np.arange(len(p)))
        # small singular values of a gradient grow by up to 3.4445^5 = 485 in a step, and with them its rounding errors
        assert np.max(np.abs(path[n + 1] - w)) < 1e-8


def test_strided_scores_of_a_sweep_are_read_in_place():
    """the unshifted rows of a sweep [B, 2P+1, n_obs] are rows (2P+1) n_obs elements apart"""
    import torch

    E = torch.randn(10, 7, 3, dtype=torch.float64).cuda()
    a = vqa_amd.log_probs_grad(E[:, 0], torch.zeros(10, dtype=torch.int32).cuda(), 1.0)
    b = vqa_amd.log_probs_grad(E[:, 0].contiguous(), torch.zeros(10, dtype=torch.int32).cuda(), 1.0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dt", ["uint8", "int8", "int16", "int64", "uint16", "uint32", "uint64"])
@pytest.mark.parametrize("V", [3, 100, 200, 1000, 40000])
def test_targets_of_every_integer_type(dt, V):
    """narrow types that hold neither -1 nor the width give what int32 targets give, on the GPU and from the host"""
    import torch

    z = scores(np.random.default_rng(V), 40, V, "float32", masked=0.0)
    most = min(V, np.iinfo(dt).max + 1)
    tg = np.arange(40) * (most - 1) // 39
    if dt[0] == "i":
        tg[::7] = -1
    want = vqa_amd.log_probs(z, torch.from_numpy(tg.astype(np.int32)).cuda(), top_k=2)
    assert torch.isfinite(want.log_prob).all()
    t = torch.from_numpy(tg.astype(dt)).cuda()
    got, host = vqa_amd.log_probs(z, t, top_k=2), vqa_amd.log_probs(z.cpu().numpy(), tg.astype(dt), top_k=2)
    assert all(torch.equal(a, b) and np.array_equal(a.cpu().numpy(), c) for a, b, c in zip(want, got, host))
    a, b = vqa_amd.log_probs_grad(z, torch.from_numpy(tg.astype(np.int32)).cuda(), -1.0), vqa_amd.log_probs_grad(z, t, -1.0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    if dt == "uint64":
        tg = np.full(40, 2 ** 63 + 5, np.uint64)
        far = vqa_amd.log_probs(z, torch.from_numpy(tg).cuda())
        assert torch.isnan(far.log_prob).all() and np.isnan(vqa_amd.log_probs(z.cpu().numpy(), tg).log_prob).all()


def test_softmax_loss_takes_the_penalty():
    """L2_reg_lmd, which cross_entropy beside it applies, reaches loss and gradient, also through fit()"""
    q, p = classifier()
    n, lmd = len(q.x_train), 0.3
    g0, g1 = q.softmax_CE_grad_eval(p, mini_batch_size=n), q.softmax_CE_grad_eval(p, mini_batch_size=n, L2_reg_lmd=lmd)
    # the two batches hold the samples in different orders: 72 terms of the sum in another one, together below 3 (24 samples of
    # weight 1 / 24, three class values whose differences are at most 1), each addition 2^-53 of what it gives
    assert np.abs(g1 - (lmd * p + g0)).max() <= 2.0 ** -53 * 2 * (72 + 8) * (3 + lmd * 4)
    loss = lambda w: q.softmax_CE_loss_eval(w, mini_batch_size=n, L2_reg_lmd=lmd)
    assert abs(loss(p) - q._softmax_CE(p, "train") - 0.15 * np.sum(p * p)) < 1e-13
    for i in (0, 7, len(p) - 1):
        e = np.zeros_like(p)
        e[i] = 1e-4
        assert abs((loss(p + e) - loss(p - e)) / 2e-4 - g1[i]) < 2e-7          # third derivative of the penalty: 0
    q.compile(optimizer="SGD", loss="softmax_cross_entropy", hpara=dict(LR_rule=0.05, batch_size_rule=n, s_list_rule=1), init_params=p)
    path = np.array(q.fit(options=dict(max_iter=1), auto_save=False, L2_reg_lmd=lmd)["para_evol"])
    from vqa_amd.optimizers import map_to_pi_range

    assert np.max(np.abs(path[1] - map_to_pi_range(p - 0.05 * g1, np.arange(len(p))))) < 1e-12


def test_tensors_that_torch_holds_negated():
    """a view whose sign is not yet applied in memory (of a conjugate's imaginary part) is read as what it stands for, and is
    no place for results; complex weights are refused"""
    import torch

    z, g = torch.randn(6, 40, device="cuda"), torch.randn(6, device="cuda")
    neg = lambda t: torch._neg_view(-t)
    tg = torch.arange(6, device="cuda")
    assert neg(z).is_neg() and torch.equal(neg(z), z)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    assert same(vqa_amd.log_probs(neg(z), tg, top_k=3), vqa_amd.log_probs(z, tg, top_k=3))
    assert same(vqa_amd.log_probs_grad(neg(z), tg, neg(g), neg(g)), vqa_amd.log_probs_grad(z, tg, g, g))
    E, d = torch.randn(4, 5, 2, dtype=torch.float64, device="cuda"), torch.randn(4, 2, dtype=torch.float64, device="cuda")
    assert torch.equal(vqa_amd.psr_chain(neg(E), neg(d)), vqa_amd.psr_chain(E, d))
    assert torch.equal(vqa_amd.orthogonalize(neg(z)), vqa_amd.orthogonalize(z))
    w, m = torch.ones_like(z), torch.zeros_like(z)
    vqa_amd.muon_step(w, neg(z), m, 0.1)
    v, n = torch.ones_like(z), torch.zeros_like(z)
    vqa_amd.muon_step(v, z, n, 0.1)
    assert torch.equal(w, v) and torch.equal(m, n)
    for call in (lambda: vqa_amd.orthogonalize(z, out=neg(w)), lambda: vqa_amd.muon_step(neg(w), z, m, 0.1), lambda: vqa_amd.muon_step(w, z, neg(m), 0.1),
                 lambda: vqa_amd.log_probs_grad(z, tg, g, out=neg(w)), lambda: vqa_amd.log_probs_grad(z, tg, g.to(torch.complex64))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("V", [12, 3000, 60000])
def test_numbers_as_weights_in_a_captured_call(V):
    """one number for all rows needs no copy from the host, so the call can be captured; the same as a tensor of it"""
    import torch

    data = [scores(np.random.default_rng(k), 7, V, "float32") for k in range(2)]
    z, tg = data[0].clone(), torch.arange(7, device="cuda")
    full = lambda v: torch.full((7,), v, device="cuda")
    a, b = vqa_amd.log_probs_grad(z, tg, -1.0 / 7, 0.3), vqa_amd.log_probs_grad(z, tg, full(-1.0 / 7), full(0.3))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = vqa_amd.log_probs_grad(z, tg, -1.0 / 7, np.float32(0.3))
    for n in range(4):
        z.copy_(data[n % 2])
        graph.replay()
        want = vqa_amd.log_probs_grad(data[n % 2], tg, full(-1.0 / 7), full(0.3))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), n


def test_a_rank_without_samples():
    """a batch of fewer samples than ranks: the rank that gets none adds zeros"""
    q, p = classifier()

    class Shard:
        lo = hi = 0

        def reduce(self, sums, per_item=None):
            return sums.cpu().numpy(), None

        def bcast_ints(self, ind):
            return ind

    q._shard = lambda n: Shard()
    assert np.array_equal(q.softmax_CE_grad_eval(p, mini_batch_size=1), np.zeros(len(p)))
