"""Newton-Schulz products and the optimizer step on the GPU against the definition on singular values, in 64 bits.

Tolerances.  With u = 2^-53 or 2^-24, a product over K terms is off by about u sqrt(K) of its factors' sizes (independent
roundings), a step of the iteration by that times |a| + |b| + |c| = 10.3 (X in norm at most 1.3), and what a step adds in the
direction of a small singular value grows by at most |a| = 3.4445 a step after it: in Frobenius norm, with r rows of norm
about 1,  u sqrt(K) 10.3 (3.4445^steps - 1) / 2.4445 sqrt(r).  That bound is loose where many roundings cancel, so matrices of
32 bits are also held to four times what a plain 32-bit run of the same formulas is off: values in 16-bit pairs and their
left-out product round at 2^-22 to 2^-23, a quarter of a 32-bit step.  A result of 16 bits adds half a step of each value."""
import math

import numpy as np
import pytest

import vqa_amd
from vqa_amd.orthogonal import COEFS

pytestmark = pytest.mark.gpu

UNIT = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "bfloat16": 2.0 ** -24, "float16": 2.0 ** -24}


def defined(g, steps=5, coefs=COEFS, eps=1e-7):
    """U p(S) V^T in numpy, 64 bits"""
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = s / (np.sqrt((g ** 2).sum(axis=(-2, -1)))[..., None] + eps)
    for _ in range(steps):
        s = s * (coefs[0] + s * s * (coefs[1] + coefs[2] * s * s))
    return (u * s[..., None, :]) @ vt


def plain(g, dtype, steps=5, coefs=COEFS, eps=1e-7):
    """the products in `dtype` on the GPU"""
    import torch

    x = (g.double() / (torch.linalg.vector_norm(g.double(), dim=(1, 2), keepdim=True) + eps)).to(dtype)
    turned = x.shape[1] > x.shape[2]
    if turned:
        x = x.transpose(1, 2).contiguous()
    for _ in range(steps):
        a = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = coefs[0] * x + torch.matmul(coefs[1] * a + coefs[2] * torch.matmul(a, a), x)
    return x.transpose(1, 2).contiguous() if turned else x


def bound(t, r, c, steps=5):
    return UNIT[t] * math.sqrt(c + 2 * r) * 10.3 * (3.4445 ** steps - 1) / 2.4445 * math.sqrt(r)


def matrices(rng, batch, rows, cols, t, noise=0.5):
    import torch

    k = max(1, min(rows, cols) // 8)
    g = rng.standard_normal((batch, rows, k)) @ rng.standard_normal((batch, k, cols)) / math.sqrt(k) + noise * rng.standard_normal((batch, rows, cols))
    return torch.from_numpy(g * 1e-2).to(getattr(torch, t)).cuda()


def check(got, g, t, steps=5, coefs=COEFS, eps=1e-7):
    import torch

    rows, cols = g.shape[-2:]
    r, c = min(rows, cols), max(rows, cols)
    g64 = g.double().reshape(-1, rows, cols)
    want = defined(g64.cpu().numpy(), steps, coefs, eps)
    o = got.double().cpu().numpy().reshape(want.shape)
    assert np.isfinite(o).all()
    off = np.sqrt(((o - want) ** 2).sum(axis=(1, 2)))
    half = 0.0 if t in ("float64", "float32") else torch.finfo(getattr(torch, t)).eps / 2
    stored = half * np.sqrt((want ** 2).sum(axis=(1, 2))) + (2.0 ** -25 * math.sqrt(r * c) if t == "float16" else 0.0)
    assert (off <= bound(t, r, c, steps) + stored).all(), (off.max(), bound(t, r, c, steps))
    wide = torch.float64 if t == "float64" else torch.float32
    p = plain(g64, wide, steps, coefs, eps).double().cpu().numpy()
    poff = np.sqrt(((p - want) ** 2).sum(axis=(1, 2)))
    # (a few elements' roundings say little: at least those of a single product of K terms)
    floor = UNIT[t] * math.sqrt(c + 2 * r) * np.sqrt((want ** 2).sum(axis=(1, 2))) * 4
    assert (off <= 4 * poff + floor + stored).all(), (off.max(), poff.max())


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 5), (11, 36), (36, 11), (9, 60), (16, 16), (17, 33), (64, 64), (64, 200), (200, 64),
          (65, 65), (64, 513), (63, 130), (1, 700), (2, 5000), (100, 100), (128, 128), (129, 257), (300, 100), (257, 640)]


@pytest.mark.parametrize("t", list(UNIT))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize_matches_the_definition(t, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    g = matrices(rng, 2, rows, cols, t)
    check(vqa_amd.orthogonalize(g), g, t)


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float64"])
def test_larger_matrices(t):
    rng = np.random.default_rng(1)
    for rows, cols in [(777, 1000), (1000, 520)]:
        g = matrices(rng, 1, rows, cols, t)[0]
        o = vqa_amd.orthogonalize(g)
        assert o.shape == g.shape and o.dtype == g.dtype
        check(o, g, t)


@pytest.mark.parametrize("t", list(UNIT))
@pytest.mark.parametrize("batch,rows,cols", [(1, 11, 300), (2, 16, 1500), (1, 1700, 15), (1, 16, 2048), (33, 16, 2048), (40, 1500, 3), (2, 3, 4000), (1, 16, 4096), (1, 16, 4099),
                                             (2, 17, 2000), (1, 64, 5000), (5, 33, 777), (1, 1, 65536), (3, 1300, 64), (2, 48, 512), (1, 3000, 12), (300, 9, 530),
                                             (3, 20, 100), (1, 32, 700), (2, 33, 50), (1, 48, 400), (1, 270, 47), (3, 49, 64), (1, 64, 300)])
def test_forms_of_small_matrices(t, batch, rows, cols):
    """strips of one, four and eight a wave, blocks of two to four tiles, long rows in one part and several, at their ends"""
    g = matrices(np.random.default_rng(rows + cols), batch, rows, cols, t)
    check(vqa_amd.orthogonalize(g), g, t)


@pytest.mark.parametrize("t", list(UNIT))
@pytest.mark.parametrize("rows,cols", [(20, 600), (2100, 50), (9, 3000)])
def test_long_rows(t, rows, cols):
    """special matrices, in place, more steps than one round holds, momentum, replayed graphs"""
    import torch

    g = matrices(np.random.default_rng(30), 6, rows, cols, t)
    g[1] = 0
    g[2, 0, 0] = float("nan")
    g[3, rows - 1, cols - 1] = float("inf")
    g[4] = 0
    g[4, 1, 2] = 3.0
    o = vqa_amd.orthogonalize(g)
    assert (o[1] == 0).all() and torch.isnan(o[2]).all() and torch.isnan(o[3]).all()
    check(torch.stack([o[0], o[4], o[5]]), torch.stack([g[0], g[4], g[5]]), t)
    assert torch.equal(vqa_amd.orthogonalize(g[5]), vqa_amd.orthogonalize(g[5:])[0])
    h = g[[0, 5]].contiguous()
    want = vqa_amd.orthogonalize(h.clone())
    assert vqa_amd.orthogonalize(h, out=h).data_ptr() == h.data_ptr() and torch.equal(h, want)
    g = g[[0, 5]].contiguous()
    for steps in (1, 7, 8, 12):
        check(vqa_amd.orthogonalize(g, steps=steps), g, t, steps=steps)
    wide = torch.float64 if t == "float64" else torch.float32
    w, m = torch.ones(2, rows, cols, dtype=wide).cuda(), 1e-2 * torch.ones(2, rows, cols, dtype=wide).cuda()
    w0, m64 = w.double().clone(), 0.9 * m.double() + g.double()
    ew, em = w.clone(), m.clone()
    vqa_amd.muon_step(w, g, m, 0.1, 0.9, 0.2)
    u = UNIT[t]
    assert ((m.double() - m64).abs() <= u * (3 * m64.abs() + 3 * g.double().abs() + 3 * (m64 - g.double()).abs())).all()
    rate = 0.1 * math.sqrt(max(1.0, rows / cols))
    w64 = 0.98 * w0.cpu().numpy() - rate * defined((g.double() + 0.9 * m64).cpu().numpy())
    off = np.sqrt(((w.double().cpu().numpy() - w64) ** 2).sum(axis=(1, 2)))
    r, c = sorted((rows, cols))
    assert (off <= rate * bound(t, r, c) * 2 + 4 * u * np.sqrt((w64 ** 2).sum(axis=(1, 2)))).all()
    graph = torch.cuda.CUDAGraph()
    cw, cm = ew.clone(), em.clone()
    with torch.cuda.graph(graph):
        vqa_amd.muon_step(cw, g, cm, 0.1, 0.9, 0.2)
    for _ in range(4):
        graph.replay()
        vqa_amd.muon_step(ew, g, em, 0.1, 0.9, 0.2)
        torch.cuda.synchronize()
        assert torch.equal(cw, ew) and torch.equal(cm, em)


@pytest.mark.parametrize("batch,rows,cols,t", [(1, 100, 4000, "float32"), (3, 200, 1111, "float32"), (2, 4100, 70, "bfloat16"), (1, 80, 3000, "float64"),
                                               (1, 500, 4096, "float16"), (5, 66, 600, "float64"), (120, 65, 300, "float32")])
def test_split_sums_are_repeatable(batch, rows, cols, t):
    """the parts of a split sum are added in their order, whichever comes last, also in a replayed graph"""
    import torch

    g = matrices(np.random.default_rng(rows), batch, rows, cols, t)
    a = vqa_amd.orthogonalize(g)
    check(a, g, t)
    out = torch.empty_like(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        vqa_amd.orthogonalize(g, out=out)
    for n in range(4):
        out.zero_()
        graph.replay()
        b = vqa_amd.orthogonalize(g)
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(b, a), n


def check_large(got, g, t, extra=0.0):
    """against the same products in 64 bits on the GPU, matrix by matrix; as check() without the singular values"""
    import torch

    r, c = sorted(g.shape[-2:])
    want = plain(g, torch.float64)
    norm = torch.linalg.vector_norm(want, dim=(1, 2))
    off = torch.linalg.vector_norm(got.double() - want, dim=(1, 2))
    poff = torch.linalg.vector_norm(plain(g, torch.float32).double() - want, dim=(1, 2))
    half = 0.0 if t == "float32" else torch.finfo(getattr(torch, t)).eps / 2
    tol = torch.minimum(torch.full_like(norm, bound(t, r, c)), 4 * poff + UNIT[t] * math.sqrt(c + 2 * r) * norm * 4) + half * norm + extra
    assert torch.isfinite(got).all() and (off <= tol).all(), (off, tol)


@pytest.mark.parametrize("batch,rows,cols,t", [(1, 2048, 2048, "float32"), (1, 2000, 2111, "bfloat16"), (1, 1024, 4096, "bfloat16"), (1, 1500, 3001, "float32"),
                                               (2, 1300, 1290, "float32"), (40, 130, 150, "bfloat16"), (1, 2500, 1100, "float16"), (300, 65, 70, "float32"),
                                               (1, 4096, 4096, "float32"), (1, 4096, 4000, "bfloat16"), (1, 3900, 4032, "float16")])
def test_tiles_of_all_sizes(batch, rows, cols, t):
    """matrices whose products take tiles of 128 and 256, and different ones for X X^T and the update"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    k = min(rows, cols) // 8
    g = torch.stack([torch.randn(rows, k, generator=gen, device="cuda") @ torch.randn(k, cols, generator=gen, device="cuda") / math.sqrt(k)
                     + 0.5 * torch.randn(rows, cols, generator=gen, device="cuda") for _ in range(batch)]).to(getattr(torch, t))
    check_large(vqa_amd.orthogonalize(g), g, t)


@pytest.mark.parametrize("batch,rows,cols", [(8, 1024, 1024), (3, 981, 614), (29, 276, 160), (2, 97, 1001), (1, 1500, 1490)])
def test_tiles_of_all_sizes_in_64_bits(batch, rows, cols):
    """tiles of 32 and 64 and both in one matrix; against the same products by the library, each within the bound"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    g = torch.randn(batch, rows, cols, generator=gen, device="cuda", dtype=torch.float64)
    want = plain(g, torch.float64)
    off = torch.linalg.vector_norm(vqa_amd.orthogonalize(g) - want, dim=(1, 2))
    r, c = sorted((rows, cols))
    assert (off <= 2 * bound("float64", r, c)).all(), off


@pytest.mark.parametrize("batch,rows,cols", [(1, 2048, 1500), (1, 4000, 4096), (1, 150, 3000), (20, 200, 130)])
def test_optimizer_step_of_large_matrices(batch, rows, cols):
    """bfloat16 gradients, weights and momentum of 32 bits: the update keeps 32 bits' accuracy"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(cols)
    g = (1e-2 * torch.randn(batch, rows, cols, generator=gen, device="cuda")).bfloat16()
    w, m = torch.randn(batch, rows, cols, generator=gen, device="cuda"), 1e-2 * torch.randn(batch, rows, cols, generator=gen, device="cuda")
    w0, m64 = w.clone(), 0.9 * m.double() + g.double()
    vqa_amd.muon_step(w, g, m, 0.5, 0.9, 0.0, True)
    assert ((m.double() - m64).abs() <= 2.0 ** -24 * (3 * m64.abs() + 3 * g.double().abs() + 3 * (m64 - g.double()).abs())).all()
    u = g.double() + 0.9 * m64
    rate = 0.5 * math.sqrt(max(1.0, rows / cols))
    # W's own rounding, and that of its difference here, half a step each of a value of W's size; the entering matrix is off
    # by 3 roundings of its norm, which grow as those of a product of 9 terms do
    half = 2.0 ** -24 * float(torch.linalg.vector_norm(w0.double())) * 2 / rate
    check_large((w0.double() - w.double()) / rate, u, "float32", half + bound("float32", min(rows, cols), 9 - 2 * min(rows, cols)))


@pytest.mark.parametrize("t", ["float64", "float32"])
@pytest.mark.parametrize("rows,cols", [(11, 36), (150, 70)])
@pytest.mark.parametrize("steps,coefs", [(1, COEFS), (2, COEFS), (3, (15 / 8, -10 / 8, 3 / 8)), (12, (1.5, -0.5, 0.0)), (5, (3.0, -3.2, 1.2))])
def test_steps_and_coefficients(t, rows, cols, steps, coefs):
    g = matrices(np.random.default_rng(2), 1, rows, cols, t)[0]
    import torch

    o = vqa_amd.orthogonalize(g, steps=steps, coefs=coefs)
    want = defined(g.double().cpu().numpy(), steps, coefs)
    r, c = min(rows, cols), max(rows, cols)
    # |a| a step in the direction of small singular values, the sum of the coefficients' sizes in a step
    a, all3 = max(abs(coefs[0]), 1.01), sum(abs(v) for v in coefs)
    tol = UNIT[t] * math.sqrt(c + 2 * r) * (all3 + 1) * (a ** steps - 1) / (a - 1) * math.sqrt(r)
    assert np.sqrt(((o.double().cpu().numpy() - want) ** 2).sum()) <= tol
    assert isinstance(o, torch.Tensor)


@pytest.mark.parametrize("t", list(UNIT))
@pytest.mark.parametrize("rows,cols", [(5, 9), (70, 90)])
def test_matrices_that_are_special(t, rows, cols):
    import torch

    g = matrices(np.random.default_rng(3), 6, rows, cols, t)
    g[1] = 0
    g[2, 0, 0] = float("nan")
    g[3, rows - 1, cols - 1] = float("inf")
    g[4] = 0
    g[4, 1, 2] = 3.0                                     # rank one
    o = vqa_amd.orthogonalize(g)
    assert (o[1] == 0).all() and torch.isnan(o[2]).all() and torch.isnan(o[3]).all()
    keep = torch.stack([g[0], g[4], g[5]])
    check(torch.stack([o[0], o[4], o[5]]), keep, t)
    # one matrix of a batch does not touch another
    assert torch.equal(vqa_amd.orthogonalize(g[5]), o[5])


@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_sizes_of_entries(size):
    """the norm is taken in 64 bits: squares of 1e30 do not overflow; entries far below eps give a result near 0"""
    import torch

    for rows, cols in [(6, 10), (80, 70)]:
        g = (matrices(np.random.default_rng(4), 1, rows, cols, "float64")[0] * size).float()
        o = vqa_amd.orthogonalize(g)
        if size > 1:
            check(o, g, "float32")
        else:
            assert o.abs().max() < 1e-18


@pytest.mark.parametrize("t", list(UNIT))
@pytest.mark.parametrize("rows,cols", [(11, 36), (40, 60), (20, 600), (96, 128), (128, 96), (97, 130), (2000, 2048)])
def test_results_that_begin_anywhere(t, rows, cols):
    """out, weight and momentum an element behind an aligned address: the same values, and nothing written around them"""
    import torch

    g = matrices(np.random.default_rng(8), 1, rows, cols, t)[0]
    want = vqa_amd.orthogonalize(g)
    wide = torch.float64 if t == "float64" else torch.float32
    n = rows * cols
    buf = torch.full((n + 2,), 7.0, dtype=g.dtype).cuda()
    o = vqa_amd.orthogonalize(g, out=buf[1:n + 1].view(rows, cols))
    assert torch.equal(o, want) and buf[0] == 7 and buf[n + 1] == 7
    w, m = torch.ones(rows, cols, dtype=wide).cuda(), torch.ones(rows, cols, dtype=wide).cuda()
    wb, mb = torch.ones(n + 2, dtype=wide).cuda(), torch.ones(n + 2, dtype=wide).cuda()
    vqa_amd.muon_step(w, g, m, 0.1)
    vqa_amd.muon_step(wb[1:n + 1].view(rows, cols), g, mb[1:n + 1].view(rows, cols), 0.1)
    assert torch.equal(wb[1:n + 1].view(rows, cols), w) and torch.equal(mb[1:n + 1].view(rows, cols), m)
    assert wb[0] == 1 and wb[n + 1] == 1 and mb[0] == 1 and mb[n + 1] == 1


@pytest.mark.parametrize("rows,cols", [(6, 10), (40, 60), (5, 3000), (80, 70)])
def test_squares_beyond_64_bits_give_nan(rows, cols):
    """and a zero matrix stays zero with the smallest eps"""
    import torch

    g = matrices(np.random.default_rng(4), 2, rows, cols, "float64")
    big = g * 1e180
    assert torch.isnan(vqa_amd.orthogonalize(big)).all()
    assert (vqa_amd.orthogonalize(torch.zeros_like(g), eps=1e-300) == 0).all()
    check(vqa_amd.orthogonalize(g * 1e-100, eps=1e-300), g * 1e-100, "float64", eps=1e-300)


@pytest.mark.parametrize("t", ["float64", "bfloat16"])
def test_strides_out_and_in_place(t):
    import torch

    for rows, cols in [(11, 36), (90, 100)]:
        big = matrices(np.random.default_rng(5), 3, rows + 2, cols + 5, t)
        g = big[:, 1:rows + 1, 3:cols + 3]
        want = vqa_amd.orthogonalize(g.contiguous())
        assert torch.equal(vqa_amd.orthogonalize(g), want)
        tr = g.transpose(1, 2)                                  # columns apart: taken through a copy
        assert torch.equal(vqa_amd.orthogonalize(tr), vqa_amd.orthogonalize(tr.contiguous()))
        h = g.contiguous()
        assert vqa_amd.orthogonalize(h, out=h).data_ptr() == h.data_ptr() and torch.equal(h, want)
        e = g[:1].expand(3, rows, cols)
        assert torch.equal(vqa_amd.orthogonalize(e)[2], want[0])
        with pytest.raises(ValueError):
            vqa_amd.orthogonalize(h, out=big[:, 1:rows + 1, 3:cols + 3])
    assert vqa_amd.orthogonalize(torch.zeros(0, 3, 4, dtype=torch.float64).cuda()).shape == (0, 3, 4)


@pytest.mark.parametrize("t", list(UNIT))
@pytest.mark.parametrize("rows,cols", [(11, 36), (36, 11), (1, 1), (130, 70), (70, 300)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_matches_the_formulas(t, rows, cols, nesterov):
    import torch

    rng = np.random.default_rng(6)
    wide = torch.float64 if t == "float64" else torch.float32
    g = matrices(rng, 2, rows, cols, t)
    w = torch.from_numpy(rng.standard_normal((2, rows, cols))).to(wide).cuda()
    m = torch.from_numpy(1e-2 * rng.standard_normal((2, rows, cols))).to(wide).cuda()
    lr, mu, wd = 0.03, 0.9, 0.1
    w64, m64, g64 = (x.double().cpu().numpy() for x in (w, m, g))
    m64 = mu * m64 + g64
    u64 = g64 + mu * m64 if nesterov else m64
    rate = lr * math.sqrt(max(1.0, rows / cols))
    w64 = (1 - lr * wd) * w64 - rate * defined(u64)
    assert vqa_amd.muon_step(w, g, m, lr, mu, wd, nesterov) is w
    u = UNIT[t]
    # mu is rounded to the type, then a product and a sum
    assert (np.abs(m.double().cpu().numpy() - m64) <= u * (3 * np.abs(m64) + 3 * np.abs(g64) + 3 * np.abs(m64 - g64))).all()
    off = np.sqrt(((w.double().cpu().numpy() - w64) ** 2).sum(axis=(1, 2)))
    r, c = min(rows, cols), max(rows, cols)
    # the entering matrix is off by a few u of its norm: the same bound again, K = 1
    tol = rate * bound(t, r, c) * 2 + 4 * u * np.sqrt((w64 ** 2).sum(axis=(1, 2)))
    assert (off <= tol).all(), (off, tol)


@pytest.mark.parametrize("dt", [np.float64, np.float32])
def test_host_pointer_paths(dt):
    import torch

    rng = np.random.default_rng(7)
    for shape in ((11, 36), (2, 70, 66)):
        g = rng.standard_normal(shape).astype(dt)
        dev = torch.from_numpy(g).cuda()
        assert np.array_equal(vqa_amd.orthogonalize(g), vqa_amd.orthogonalize(dev).cpu().numpy())
        w, m = rng.standard_normal(shape).astype(dt), np.zeros(shape, dt)
        wt, mt = torch.from_numpy(w.copy()).cuda(), torch.from_numpy(m.copy()).cuda()
        vqa_amd.muon_step(w, g, m, 0.1)
        vqa_amd.muon_step(wt, dev, mt, 0.1)
        assert np.array_equal(w, wt.cpu().numpy()) and np.array_equal(m, mt.cpu().numpy())


@pytest.mark.parametrize("rows,cols", [(11, 36), (200, 300)])
def test_streams_and_captured_steps(rows, cols):
    """a captured optimizer step is replayed; eager steps on copies run beside it and agree bit for bit"""
    import torch

    rng = np.random.default_rng(9)
    grads = [matrices(rng, 1, rows, cols, "float32") for _ in range(3)]
    w = torch.from_numpy(rng.standard_normal((1, rows, cols))).float().cuda()
    m, g = torch.zeros_like(w), grads[0].clone()
    ew, em = w.clone(), m.clone()
    a = vqa_amd.orthogonalize(g)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = vqa_amd.orthogonalize(g)
        vqa_amd.muon_step(w.clone(), g, m.clone(), 0.01)       # loads the kernels before the capture
    s.synchronize()
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        vqa_amd.muon_step(w, g, m, 0.01)
    for n in range(5):
        g.copy_(grads[n % 3])
        graph.replay()
        vqa_amd.muon_step(ew, grads[n % 3], em, 0.01)
        torch.cuda.synchronize()
        assert torch.equal(w, ew) and torch.equal(m, em), n


@pytest.mark.parametrize("rows,cols,t", [(100, 4000, "float32"), (20, 3000, "float32"), (300, 300, "float64"), (700, 800, "bfloat16"), (30, 80, "float64")])
def test_calls_at_the_same_time(rows, cols, t):
    """queued on three streams without waiting, each call's workspace is its own"""
    import torch

    gs = [matrices(np.random.default_rng(k), 1, rows, cols, t)[0] for k in range(3)]
    want = [vqa_amd.orthogonalize(g) for g in gs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in gs]
    got = [[], [], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(vqa_amd.orthogonalize(gs[k]))
    torch.cuda.synchronize()
    for k in range(3):
        assert all(torch.equal(o, want[k]) for o in got[k])


def test_refusals_on_the_gpu():
    import torch

    w = torch.zeros(4, 6).cuda()
    g = torch.zeros(4, 6, dtype=torch.bfloat16).cuda()
    m = torch.zeros(4, 6).cuda()
    with pytest.raises(ValueError):
        vqa_amd.muon_step(w.double(), g, m, 0.1)
    with pytest.raises(ValueError):
        vqa_amd.muon_step(w.t().contiguous().t(), g, m, 0.1)
    with pytest.raises(ValueError):
        vqa_amd.muon_step(w, g, torch.zeros(4, 6), 0.1)
    from vqa_amd import _lib
    with pytest.raises(_lib.VqaError):
        vqa_amd.muon_step(w, g, w, 0.1)
    with pytest.raises(_lib.VqaError):
        vqa_amd.orthogonalize(w, coefs=(9.0, 0.0, 0.0))
    with pytest.raises(ValueError):
        vqa_amd.orthogonalize(w.to(torch.int32))


def test_muon_optimizer_trains_the_regressor():
    """compile / fit with optimizer="Muon": the matrix part takes the orthogonalised step, the scale parameter SGDM's"""
    from vqa_amd.qml_utils import create_ibm_HEA_ansatz
    from vqa_amd.qnn_base import myQNN_base

    rng = np.random.default_rng(0)
    x = rng.uniform(0, 1, (16, 4))
    q = myQNN_base(4, create_ibm_HEA_ansatz(4, 1, seed=2), x, np.sin(x.sum(1)), x, np.sin(x.sum(1)), min_approx_shots=-10)
    p = np.concatenate([rng.uniform(-3, 3, q.n_c_params), [0.9]])
    q.compile(optimizer="Muon", hpara=dict(LR_rule=0.02, batch_size_rule=16, s_list_rule=100), init_params=p, min_approx_shots=-10)
    res = q.fit(options=dict(max_iter=2), auto_save=False)
    path = np.array(res["para_evol"])
    g = q.MSE_grad_eval(p, np.full(len(p), 100), mini_batch_size=16, option_min_approx=-10)
    o = defined((g + 0.95 * g)[:24].reshape(2, 12))
    from vqa_amd.optimizers import map_to_pi_range

    want = p - 0.02 * np.concatenate([o.reshape(-1), g[24:]])
    want = map_to_pi_range(want, q.optimizer.periodic_para_inds)
    assert np.max(np.abs(path[1] - want)) < 1e-9


def before_rounding(got, want):
    """The Frobenius norm of the least error that takes `want` into what rounds to `got` (16 bits): a result is off by its
    rounding and by what it was off before, and only the second counts here."""
    import torch

    bits = got.contiguous().view(torch.int16)
    mag = bits & 0x7fff
    value = lambda m: m.view(got.dtype).double()
    x, up, down = value(mag), value(mag + 1), value((mag - 1).clamp(min=0))
    w = torch.where(bits < 0, -want, want)
    high = (x + up) / 2
    low = torch.where(mag == 0, -high, (x + down) / 2)
    return torch.linalg.vector_norm(torch.maximum(w - high, low - w).clamp(min=0), dim=(-2, -1))


@pytest.mark.parametrize("t", ["bfloat16", "float16"])
@pytest.mark.parametrize("batch,rows,cols", [(2, 11, 36), (2, 40, 60), (2, 20, 600), (3, 80, 70), (1, 300, 300), (1, 100, 4000), (1, 1024, 4096), (1, 2048, 1500),
                                             (1, 2000, 2111), (1, 4096, 4096)])
def test_results_of_16_bits_are_rounded_once(t, batch, rows, cols):
    """what a 16-bit result is off before its rounding is held to what a 32-bit result may be off, whatever its size and tiles"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    k = max(1, min(rows, cols) // 8)
    g = (torch.randn(batch, rows, k, generator=gen, device="cuda") @ torch.randn(batch, k, cols, generator=gen, device="cuda") / math.sqrt(k)
         + 0.5 * torch.randn(batch, rows, cols, generator=gen, device="cuda")).to(getattr(torch, t))
    o = vqa_amd.orthogonalize(g)
    want = plain(g, torch.float64)
    r, c = sorted((rows, cols))
    norm = torch.linalg.vector_norm(want, dim=(1, 2))
    poff = torch.linalg.vector_norm(plain(g, torch.float32).double() - want, dim=(1, 2))
    tol = torch.minimum(torch.full_like(norm, bound(t, r, c)), 4 * poff + UNIT[t] * math.sqrt(c + 2 * r) * norm * 4)
    off = before_rounding(o, want)
    assert torch.isfinite(o).all() and (off <= tol).all(), (off / norm, tol / norm)
    for _ in range(3):
        assert torch.equal(vqa_amd.orthogonalize(g), o)


def of_norm(gen, batch, rows, cols, norm):
    import torch

    k = max(1, min(rows, cols) // 8)
    g = (torch.randn(batch, rows, k, generator=gen, device="cuda", dtype=torch.float64) @ torch.randn(batch, k, cols, generator=gen, device="cuda", dtype=torch.float64)
         / math.sqrt(k) + 0.5 * torch.randn(batch, rows, cols, generator=gen, device="cuda", dtype=torch.float64))
    return g / torch.linalg.vector_norm(g, dim=(1, 2), keepdim=True) * norm


@pytest.mark.parametrize("rows,cols", [(11, 36), (40, 60), (20, 600), (80, 70), (300, 300), (100, 4000), (2000, 1500)])
@pytest.mark.parametrize("steps", [1, 5, 16])
def test_norms_far_below_eps(rows, cols, steps):
    """X = G / (|G| + eps) is then small itself, and stays so for many steps: relative to the result's own norm it is as exact as
    32-bit products are (a batch of all sizes of norm, each matrix for itself)"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows + cols + steps)
    norms = [1.0, 3e-7, 1e-7, 1e-9, 1e-11, 1e-13, 1e-16, 1e-22, 1e-27]
    g64 = of_norm(gen, len(norms), rows, cols, torch.tensor(norms, device="cuda", dtype=torch.float64)[:, None, None])
    for t in ("float32", "bfloat16"):
        g = g64.to(getattr(torch, t))
        o = vqa_amd.orthogonalize(g, steps=steps)
        want, p = plain(g, torch.float64, steps), plain(g, torch.float32, steps)
        r, c = sorted((rows, cols))
        norm = torch.linalg.vector_norm(want, dim=(1, 2))
        off = torch.linalg.vector_norm(o.double() - want, dim=(1, 2)) if t == "float32" else before_rounding(o, want)
        tol = 4 * torch.linalg.vector_norm(p.double() - want, dim=(1, 2)) + UNIT[t] * math.sqrt(c + 2 * r) * norm * 4
        assert torch.isfinite(o).all() and (off <= tol).all(), (t, off / norm, tol / norm)
        for b in range(len(norms)):
            assert (off[b] <= tol[b]) and norm[b] > 0


@pytest.mark.parametrize("rows,cols,eps", [(80, 70, 1.0), (80, 70, 1e4), (300, 200, 1e9), (1100, 1000, 1e30)])
def test_eps_far_above_the_norm(rows, cols, eps):
    """the same by way of eps, with float16 as well; weights that take the step, and a matrix of zeros"""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(rows)
    g64 = of_norm(gen, 3, rows, cols, 1.0)
    g64[1] = 0
    r, c = sorted((rows, cols))
    for t in ("float32", "float16"):
        g = g64.to(getattr(torch, t))
        m, w = torch.zeros(3, rows, cols, device="cuda"), torch.zeros(3, rows, cols, device="cuda")
        vqa_amd.muon_step(w, g, m, 1.0, 0.0, eps=eps)        # momentum and update are g itself, w becomes -rate * result
        want, p = plain(g, torch.float64, eps=eps), plain(g, torch.float32, eps=eps)
        rate = math.sqrt(max(1.0, rows / cols))
        off = torch.linalg.vector_norm(-w.double() / rate - want, dim=(1, 2))
        norm = torch.linalg.vector_norm(want, dim=(1, 2))
        # (the rate is rounded and multiplied: a step of each value)
        tol = 4 * torch.linalg.vector_norm(p.double() - want, dim=(1, 2)) + UNIT[t] * (math.sqrt(c + 2 * r) * 4 + 2) * norm
        assert (w[1] == 0).all() and (off <= tol).all(), (t, off / norm, tol / norm)


def test_autograd_sees_what_was_overwritten():
    """weight, momentum and out= move torch's version counters: a backward pass that saved them raises, as after torch's own
    in-place operations, and does not take the new values for the old; tensors of inference mode have no counters"""
    import torch

    for rows, cols in ((4, 6), (80, 70)):
        g = torch.randn(rows, cols, device="cuda")
        w, m, out = torch.ones_like(g), torch.zeros_like(g), torch.empty_like(g)
        a = torch.ones_like(g, requires_grad=True)
        for write, written in ((lambda: vqa_amd.muon_step(w, g, m, 0.1), (w, m)), (lambda: vqa_amd.orthogonalize(g, out=out), (out,)),
                               (lambda: vqa_amd.log_probs_grad(g, torch.zeros(rows, dtype=torch.int32, device="cuda"), 1.0, out=out), (out,))):
            read = g._version
            losses = [(a * t).sum() for t in written]
            before = [t._version for t in written]
            write()
            assert all(t._version > v for t, v in zip(written, before)) and g._version == read
            for y in losses:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.backward()
        y = (a * g).sum()
        vqa_amd.orthogonalize(g)                     # a result of its own: nothing that was there has changed
        y.backward()
        y = (a * g).sum()
        vqa_amd.orthogonalize(g, out=g)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():
            w, m = torch.ones(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
            vqa_amd.muon_step(w, torch.ones_like(w), m, 0.1)
            vqa_amd.orthogonalize(w, out=w)
            assert torch.isfinite(w).all() and (m == 1).all()


@pytest.mark.parametrize("rows,cols", [(11, 36), (40, 60), (60, 200), (20, 600), (64, 5000), (3000, 12), (150, 70), (300, 290)])
@pytest.mark.parametrize("steps,coefs", [(3, (15 / 8, -10 / 8, 3 / 8)), (20, (15 / 8, -10 / 8, 3 / 8)), (12, (1.5, -0.5, 0.0)), (30, (1.5, -0.5, 0.0)),
                                         (5, (3.0, -3.2, 1.2)), (9, (3.0, -3.2, 1.2)), (6, (2.0, -1.5, 0.5)), (4, (0.5, 3.0, -2.9)), (7, (-1.2, 0.9, -0.4)),
                                         (5, (0.7, 0.0, 0.0)), (3, (0.0, 1.5, -0.9)), (12, (1.0, -0.9, 0.0)), (40, (1.0, -0.3, 0.0)), (10, (-1.0, 2.5, -1.6)),
                                         (3, (1.0, 0.0, 0.0))])
def test_other_coefficients_in_every_form(rows, cols, steps, coefs):
    """strips, blocks, the steps on X X^T (several rounds of them, for small and large first coefficients) and tiles: as exact as
    four runs of the products in the type's own precision, with the size of one product's roundings beside"""
    import torch

    for t in UNIT:
        g = matrices(np.random.default_rng(rows + steps), 2, rows, cols, t)
        if t != "float64" and min(rows, cols) > 64 and abs(coefs[0]) < 1:
            from vqa_amd import _lib

            with pytest.raises(_lib.VqaError, match="shrink"):
                vqa_amd.orthogonalize(g, steps=steps, coefs=coefs)
            continue
        want = torch.from_numpy(defined(g.double().cpu().numpy(), steps, coefs)).cuda()
        p = plain(g.double(), torch.float64 if t == "float64" else torch.float32, steps, coefs)
        r, c = sorted((rows, cols))
        norm = torch.linalg.vector_norm(want, dim=(1, 2))
        o = vqa_amd.orthogonalize(g, steps=steps, coefs=coefs)
        off = before_rounding(o, want) if t in ("bfloat16", "float16") else torch.linalg.vector_norm(o.double() - want, dim=(1, 2))
        tol = 4 * torch.linalg.vector_norm(p.double() - want, dim=(1, 2)) + UNIT[t] * math.sqrt(c + 2 * r) * norm * 4
        assert torch.isfinite(o).all() and (off <= tol).all(), (t, off / norm, tol / norm)
