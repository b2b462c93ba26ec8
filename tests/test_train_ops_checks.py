"""Refusals of the softmax read-out and of the orthogonalised updates (C ABI and Python): no GPU is needed, every check comes
before the device is touched.  The pointers are host memory that no call reads."""
import ctypes as C

import numpy as np
import pytest

import vqa_amd
from vqa_amd import _lib

MEM = np.zeros(1 << 16, np.float64)
P = MEM.ctypes.data


def refused(rc, code, *words):
    assert rc == code
    msg = _lib.lib().vqa_last_error().decode()
    for w in words:
        assert w in msg, msg


def score(dtype=0, z=P, rows=4, width=8, stride=8, scale=1.0, t=P + 4096, k=2, ws=None, lp=P + 8192, ent=P + 12288, tl=P + 16384,
          ti=P + 20480):
    return _lib.lib().vqa_log_probs_dev(0, None, dtype, z, rows, width, stride, scale, t, k, ws, lp, ent, tl, ti)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=4), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(width=0), "width"),
    (dict(width=2 ** 31, stride=2 ** 31), "width"), (dict(stride=7), "row stride"), (dict(stride=2 ** 41), "row stride"),
    (dict(z=None), "NULL"), (dict(z=P + 4), "aligned"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(k=-1), "top_k"), (dict(k=9), "top_k"),
    (dict(width=100, stride=100, k=65), "top_k"), (dict(tl=None), "top_log_prob"), (dict(ti=None), "top_log_prob"),
    (dict(t=None), "targets"), (dict(width=5000, stride=5000, rows=1), "workspace"),
    (dict(rows=2 ** 40, width=2 ** 30, stride=2 ** 30), "too large"),
])
def test_score_refusals(kw, word):
    refused(score(**kw), _lib.EINVAL, word)


def test_score_of_nothing():
    assert score(rows=0, z=None, t=None, lp=None, ent=None, tl=None, ti=None) == 0


def loss(dtype=0, z=P, rows=4, width=8, stride=8, scale=1.0, t=P + 4096, g=P + 4096, h=None, ws=None, lp=P + 8192, ent=None,
         dz=P + 16384, dz_stride=8):
    return _lib.lib().vqa_log_probs_grad_dev(0, None, dtype, z, rows, width, stride, scale, t, g, h, ws, lp, ent, dz, dz_stride)


@pytest.mark.parametrize("kw,word", [
    (dict(dz=None), "dscores"), (dict(dz_stride=7), "dscores"), (dict(dz=P), "overlap"), (dict(dz=P + 8 * 31), "overlap"),
    (dict(z=P + 8 * 31, dz=P), "overlap"), (dict(t=None), "targets"), (dict(t=None, lp=None), "targets"), (dict(scale=-2.0), "scale"),
    (dict(dtype=9), "dtype"), (dict(width=3000, stride=3000, dz_stride=3000, rows=1, dz=P + 32768), "workspace"),
])
def test_loss_refusals(kw, word):
    refused(loss(**kw), _lib.EINVAL, word)


K = (C.c_double * 3)(*vqa_amd.orthogonal.COEFS)


def ortho(dtype=0, g=P, batch=2, rows=4, cols=8, sr=8, sb=32, steps=5, k=K, eps=1e-7, ws=None, out=P + 8192):
    return _lib.lib().vqa_orthogonalize_dev(0, None, dtype, g, batch, rows, cols, sr, sb, steps, k, eps, ws, out)


def k3(*v):
    return (C.c_double * 3)(*v)


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=7), _lib.EINVAL, "dtype"), (dict(batch=-1), _lib.EINVAL, "batch"), (dict(batch=65536), _lib.EINVAL, "batch"),
    (dict(rows=0), _lib.EINVAL, "rows"), (dict(cols=65537, sr=65537), _lib.EINVAL, "rows"), (dict(sr=7), _lib.EINVAL, "row_stride"),
    (dict(sb=31), _lib.EINVAL, "batch_stride"), (dict(steps=0), _lib.EINVAL, "steps"), (dict(steps=101), _lib.EINVAL, "steps"),
    (dict(k=None), _lib.EINVAL, "coefs"), (dict(k=k3(1, float("nan"), 0)), _lib.EINVAL, "finite"),
    (dict(k=k3(5.0, 0, 0)), _lib.EUNSUPPORTED, "singular value"), (dict(k=k3(1.5, 0, 0)), _lib.EUNSUPPORTED, "singular value"),
    (dict(k=k3(0.0, 0.0, 40.0)), _lib.EUNSUPPORTED, "polynomial"), (dict(eps=0.0), _lib.EINVAL, "eps"), (dict(eps=1e-301), _lib.EINVAL, "eps"),
    (dict(eps=float("inf")), _lib.EINVAL, "eps"), (dict(g=None), _lib.EINVAL, "g is NULL"), (dict(g=P + 2), _lib.EINVAL, "aligned"),
    (dict(out=None), _lib.EINVAL, "out"), (dict(out=P + 8), _lib.EINVAL, "overlap"), (dict(out=P, sr=9, sb=36), _lib.EINVAL, "overlap"),
    (dict(rows=100, cols=100, sr=100, sb=10000, batch=1, out=P + 80000), _lib.EINVAL, "workspace"),
])
def test_orthogonalize_refusals(kw, code, word):
    refused(ortho(**kw), code, word)


def test_ordinary_coefficients_pass_the_range_check():
    # (3, -3.2, 1.2) and (15/8, -10/8, 3/8) stay within range for many steps; the check is the last before the batch of 0 returns
    for k in (vqa_amd.orthogonal.COEFS, (3.0, -3.2, 1.2), (15 / 8, -10 / 8, 3 / 8), (1.5, -0.5, 0.0)):
        assert ortho(batch=0, g=None, out=None, k=k3(*k), steps=100) == 0


def step(dtype=0, w=P, g=P + 8192, m=P + 16384, batch=2, rows=4, cols=8, sr=8, sb=32, lr=0.1, mu=0.9, wd=0.0):
    return _lib.lib().vqa_muon_step_dev(0, None, dtype, w, g, m, batch, rows, cols, sr, sb, lr, mu, wd, 1, 5, K, 1e-7, None)


@pytest.mark.parametrize("kw,word", [
    (dict(w=None), "weight"), (dict(m=None), "weight"), (dict(m=P + 8), "overlap"), (dict(g=P + 8), "overlap"),
    (dict(g=P + 16384), "overlap"), (dict(lr=float("nan")), "finite"), (dict(mu=float("inf")), "finite"), (dict(wd=float("nan")), "finite"),
])
def test_step_refusals(kw, word):
    refused(step(**kw), _lib.EINVAL, word)


def test_chain_refusals():
    L = _lib.lib()
    call = lambda e=P, B=2, n=3, o=1, d=P, ws=P, out=P: L.vqa_psr_chain_dev(0, None, e, B, n, o, 0.5, d, ws, out)
    refused(call(B=-1), _lib.EINVAL, "n_samples")
    refused(call(B=2 ** 22 + 1), _lib.EINVAL, "n_samples")
    refused(call(o=0), _lib.EINVAL, "n_obs")
    refused(call(out=None), _lib.EINVAL, "out")
    refused(call(e=None), _lib.EINVAL, "NULL")
    assert call(n=0) == 0


def test_workspace_of_bad_arguments_is_zero():
    L = _lib.lib()
    assert L.vqa_log_probs_workspace(9, 1, 1, 0) == 0 and L.vqa_log_probs_workspace(0, -1, 1, 0) == 0
    assert L.vqa_orthogonalize_workspace(0, 1, 0, 5) == 0
    assert L.vqa_log_probs_workspace(0, 5, 3, 3) == 0
    assert L.vqa_log_probs_workspace(0, 5, 10 ** 6, 3) > 0 and L.vqa_orthogonalize_workspace(2, 3, 500, 600) > 0


def test_python_refusals():
    z = np.zeros((3, 4))
    for bad in (np.zeros(4), np.zeros((2, 3, 4))):
        with pytest.raises(ValueError):
            vqa_amd.log_probs(bad)
    with pytest.raises(ValueError):
        vqa_amd.log_probs(z, top_k=5)
    with pytest.raises(ValueError):
        vqa_amd.log_probs(z, targets=np.zeros(4, int))
    with pytest.raises(ValueError):
        vqa_amd.log_probs(z, targets=np.zeros(3))
    with pytest.raises(ValueError):
        vqa_amd.log_probs_grad(z, None, d_log_prob=1.0)
    with pytest.raises(ValueError):
        vqa_amd.log_probs_grad(z, np.zeros(3, int), 1.0, out=np.zeros((3, 5)))
    with pytest.raises(ValueError):
        vqa_amd.orthogonalize(np.zeros(4))
    with pytest.raises(ValueError):
        vqa_amd.orthogonalize(z, coefs=(1.0, 2.0))
    with pytest.raises(ValueError):
        vqa_amd.orthogonalize(z, out=np.zeros((4, 3)))
    w = np.zeros((3, 4))
    with pytest.raises(ValueError):
        vqa_amd.muon_step(w.T, w.T, w.T, 0.1)          # not C-contiguous: an in-place step would go to a copy
    with pytest.raises(ValueError):
        vqa_amd.muon_step(w, w, np.zeros((4, 3)), 0.1)
    import torch
    with pytest.raises(ValueError):
        vqa_amd.log_probs(torch.zeros(3, 4))           # a tensor on the host: numpy is the host path
    with pytest.raises(ValueError):
        vqa_amd.orthogonalize(torch.zeros(3, 4))


def test_muon_needs_a_matrix():
    class Target:
        n_c_params, n_qubits = 14, 4
        shots_counter = call_counter = circuit_counter = epoch_counter = [0]
        methods_for_optimization = {}

    with pytest.raises(ValueError, match="matrix_shape"):
        vqa_amd.optimizers.Muon({}, dict(target_obj=Target(), init_params=np.zeros(14)))
    with pytest.raises(ValueError, match="matrix_shape"):
        vqa_amd.optimizers.Muon(dict(matrix_shape=(4, 4)), dict(target_obj=Target(), init_params=np.zeros(14)))
    o = vqa_amd.optimizers.Muon(dict(matrix_shape=(2, 7)), dict(target_obj=Target(), init_params=np.zeros(14)))
    assert o._shape() == (2, 7)
    Target.n_c_params = 24
    o = vqa_amd.optimizers.get_optimizer_class("Muon")({}, dict(target_obj=Target(), init_params=np.zeros(25)))
    assert o._shape() == (2, 12)


@pytest.mark.parametrize("builder,angles", [("create_jerbi_ansatz", 3), ("create_ibm_HEA_ansatz", 3), ("create_ry_rz_cz_ansatz", 2), ("create_ry_cz_ansatz", 1)])
@pytest.mark.parametrize("n_qubits", [2, 3, 4])
def test_the_default_matrix_has_a_row_a_layer(builder, angles, n_qubits):
    """for every shipped builder and depth, also where the number of angles would go into layers of three a qubit"""
    from vqa_amd import qml_utils

    class Target:
        shots_counter = call_counter = circuit_counter = epoch_counter = [0]
        methods_for_optimization = {}

    for depth in range(9):
        Target.n_qubits, Target.circuit = n_qubits, getattr(qml_utils, builder)(n_qubits, depth)
        Target.n_c_params = Target.circuit.n_theta
        for more in (0, 1):                      # the regressor's scale stands behind them
            o = vqa_amd.optimizers.Muon({}, dict(target_obj=Target(), init_params=np.zeros(Target.n_c_params + more)))
            assert o._shape() == (depth + 1, angles * n_qubits), depth


def test_a_circuit_without_layers_needs_matrix_shape():
    """gates that repeat nothing form no matrix, whatever their number; a shared angle counts where it first turns"""
    from vqa_amd.circuit import GateList

    class Target:
        n_qubits = 2
        shots_counter = call_counter = circuit_counter = epoch_counter = [0]
        methods_for_optimization = {}

    def made(gates, shared=()):
        c = GateList(2)
        for kind, q in gates:
            getattr(c, f"add_parametric_R{kind}_gate")(q, 0.1)
        for p in shared:
            c.add_parametric_RX_gate(0, 0.0, share_with=p)
        Target.circuit, Target.n_c_params = c, c.n_theta
        return vqa_amd.optimizers.Muon({}, dict(target_obj=Target(), init_params=np.zeros(c.n_theta)))._shape()

    with pytest.raises(ValueError, match="matrix_shape"):
        made([("X", 0), ("Y", 0), ("Z", 0), ("X", 1), ("Y", 0), ("Z", 0)])       # 6 angles on 2 qubits
    with pytest.raises(ValueError, match="matrix_shape"):
        made([("X", 0)] * 6)                                                     # one qubit of two
    assert made([("X", 0), ("X", 1)] * 3) == (3, 2)
    assert made([("X", 0), ("X", 1)] * 3, shared=[0, 2]) == (3, 2)
    assert made([(k, q) for q in (0, 1) for k in "YZY"]) == (1, 6)               # one layer, every qubit turned as often
    assert made([(k, q) for q in (0, 1) for k in "YZY"] * 2) == (2, 6)

    class Other:                                                                 # a circuit whose gates cannot be read
        pass

    Target.circuit, Target.n_c_params = Other(), 6
    with pytest.raises(ValueError, match="matrix_shape"):
        vqa_amd.optimizers.Muon({}, dict(target_obj=Target(), init_params=np.zeros(6)))


def test_softmax_loss_refuses_what_it_does_not_know():
    """a keyword that would change nothing without saying so"""
    from vqa_amd.qnn_classifier import myQNN_classifier as Q

    q = Q.__new__(Q)
    for f in (Q.softmax_CE_grad_eval, Q.softmax_CE_loss_eval):
        for kw in (dict(partial_MSE=True), dict(L2_reg=0.1)):
            with pytest.raises(TypeError, match=next(iter(kw))):
                f(q, np.zeros(3), **kw)


def test_softmax_gradient_runs_on_the_circuits_gpu(monkeypatch):
    """a sweep that comes back as numpy goes to the GPU that the circuit names, not to the current one"""
    import torch

    from vqa_amd import qnn_classifier, softmax

    went = []

    class Circuit:
        device = 3

        def psr_full(self, theta, handle, sel, **kw):
            return np.zeros((len(sel), 2 * len(theta) + 1, 3)), None

    q = qnn_classifier.myQNN_classifier.__new__(qnn_classifier.myQNN_classifier)
    q.circuit, q.n_c_params = Circuit(), 4
    q.circuit_counter, q.call_counter = [0], [0]
    q._setup = lambda *a: (None, np.arange(5), np.zeros(5, int), None)
    q._shard = lambda n: None
    q._handle = lambda which: None
    q.class_observables = lambda: []
    monkeypatch.setattr(torch.Tensor, "cuda", lambda t, *a, **k: went.append(("current", a)) or t)
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a, **k: went.append(a[0] if a else k) or t)
    monkeypatch.setattr(softmax, "log_probs_grad", lambda z, *a, **k: softmax.LogProbsGrad(None, None, z))
    monkeypatch.setattr(softmax, "psr_chain", lambda E, d: torch.zeros(4, dtype=torch.float64))
    assert np.array_equal(q.softmax_CE_grad_eval(np.ones(4)), np.zeros(4))
    assert went == ["cuda:3"]
    del Circuit.device                       # a circuit that names none: the first, as its other calls take it
    went.clear()
    q.softmax_CE_grad_eval(np.ones(4))
    assert went == ["cuda:0"]


def read_only(a):
    a = a.copy()
    a.flags.writeable = False
    return a


@pytest.mark.parametrize("out", [read_only(np.zeros((3, 4))), np.frombuffer(bytes(96)).reshape(3, 4)])
def test_results_do_not_go_to_read_only_arrays(out):
    z = np.zeros((3, 4))
    with pytest.raises(ValueError, match="writable"):
        vqa_amd.orthogonalize(z, out=out)
    with pytest.raises(ValueError, match="writable"):
        vqa_amd.log_probs_grad(z, np.zeros(3, int), 1.0, out=out)
    with pytest.raises(ValueError, match="writable"):
        vqa_amd.muon_step(out, z, np.zeros((3, 4)), 0.1)
    assert not out.any()


def test_arrays_in_the_other_byte_order_and_complex_ones():
    """numpy arrays reach the library in the machine's byte order; an imaginary part is not dropped"""
    from vqa_amd import orthogonal, softmax

    a = np.arange(12.0).reshape(3, 4) - 5
    for kind in ("f8", "f4", "f2"):
        for take in (softmax._np_rows, orthogonal._np_matrices):
            got = take(a.astype(">" + kind), "it")
            assert got.dtype.isnative and got.dtype == np.dtype(kind) and np.array_equal(got, a)
    for take in (softmax._np_rows, orthogonal._np_matrices):
        assert take(a.astype(">i4"), "it").dtype == np.float64
        with pytest.raises(ValueError, match="real"):
            take(a + 1j, "it")
    assert softmax._np_targets(np.array([2, 0, 1], ">i8"), 3, 4).tolist() == [2, 0, 1]
    with pytest.raises(ValueError):
        vqa_amd.orthogonalize(a, out=np.empty((3, 4), ">f8"))
    w = np.zeros((3, 4))
    with pytest.raises(ValueError):
        vqa_amd.muon_step(w.astype(">f8"), w, w.copy(), 0.1)
    for bad in (a + 1j, "abcd"):
        with pytest.raises(ValueError):
            vqa_amd.muon_step(w, bad, w.copy(), 0.1)
    for kw in (dict(d_log_prob=1j), dict(d_entropy=np.full(3, 1j))):
        with pytest.raises(ValueError):
            vqa_amd.log_probs_grad(a, np.zeros(3, int), **kw)


@pytest.mark.parametrize("kw", [
    dict(t=P + 4098), dict(lp=P + 8196), dict(ent=P + 12292), dict(tl=P + 16388), dict(ti=P + 20482), dict(dtype=1, lp=P + 8194),
    dict(rows=1, width=5000, stride=5000, ws=P + 131080)])
def test_score_pointers_are_aligned(kw):
    refused(score(**kw), _lib.EINVAL, "aligned")


@pytest.mark.parametrize("kw", [
    dict(t=P + 4097), dict(g=P + 4100), dict(h=P + 4100), dict(lp=P + 8196), dict(ent=P + 8196), dict(dz=P + 16388), dict(dtype=2, g=P + 4098),
    dict(rows=1, width=3000, stride=3000, dz_stride=3000, dz=P + 32768, ws=P + 131080)])
def test_loss_pointers_are_aligned(kw):
    refused(loss(**kw), _lib.EINVAL, "aligned")


def test_matrix_and_chain_pointers_are_aligned():
    refused(ortho(out=P + 8196), _lib.EINVAL, "aligned")
    refused(ortho(dtype=2, out=P + 8193), _lib.EINVAL, "aligned")
    refused(ortho(dtype=1, rows=100, cols=100, sr=100, sb=10000, batch=1, out=P + 80000, ws=P + 131080), _lib.EINVAL, "aligned")
    refused(step(w=P + 4), _lib.EINVAL, "aligned")
    refused(step(m=P + 16388), _lib.EINVAL, "aligned")
    refused(step(dtype=3, w=P + 2), _lib.EINVAL, "aligned")
    L = _lib.lib()
    ok = dict(e=P, d=P + 1024, ws=P + 2048, out=P + 4096)
    for k in ok:
        a = dict(ok)
        a[k] += 4
        refused(L.vqa_psr_chain_dev(0, None, a["e"], 2, 3, 1, 0.5, a["d"], a["ws"], a["out"]), _lib.EINVAL, "aligned")


def test_refused_pointers_were_the_only_fault():
    """the calls of the alignment tests with their ordinary pointers reach the device (or find none here)"""
    if _lib.lib().vqa_device_count() > 0:
        pytest.skip("the pointers are host memory")
    for rc in (score(), loss(), ortho(), step(), _lib.lib().vqa_psr_chain_dev(0, None, P, 2, 3, 1, 0.5, P, P, P),
               score(rows=1, width=5000, stride=5000, ws=P + 131072), ortho(dtype=1, rows=100, cols=100, sr=100, sb=10000, batch=1, out=P + 80000, ws=P + 131072)):
        assert rc == _lib.ENODEVICE
    # the host-pointer forms copy: their outputs may lie anywhere
    L = _lib.lib()
    for rc in (L.vqa_muon_step(0, 0, P + 4, P + 8192, P + 16388, 2, 4, 8, 8, 32, 0.1, 0.9, 0.0, 1, 5, K, 1e-7),
               L.vqa_orthogonalize(0, 0, P, 2, 4, 8, 8, 32, 5, K, 1e-7, P + 8196),
               L.vqa_log_probs(0, 0, P, 4, 8, 8, 1.0, P + 4097, 2, P + 8196, P + 12292, P + 16388, P + 20482)):
        assert rc == _lib.ENODEVICE


def test_a_workspace_is_asked_for_where_it_is_used():
    """its size and the launches go by one rule: without one a call is refused or needs none; one sized for outcomes does for a
    gradient too"""
    L = _lib.lib()
    if L.vqa_device_count() > 0:
        pytest.skip("the pointers are host memory")
    for rows in (1, 2, 100, 127, 128, 200, 511, 512, 1023, 1024, 5000):
        for width in (3, 64, 256, 257, 1024, 1025, 4095, 8191, 8192, 8193, 20000, 500000):
            for k in (0, 3):
                n = L.vqa_log_probs_workspace(1, rows, width, k)
                rc = score(dtype=1, rows=rows, width=width, stride=width, k=k)
                assert (rc == _lib.EINVAL) if n else (rc == _lib.ENODEVICE), (rows, width, k)
                assert n >= L.vqa_log_probs_workspace(1, rows, width, 0)
            rc = loss(dtype=1, rows=rows, width=width, stride=2 * width, dz_stride=2 * width, dz=P + 4 * width)
            assert (rc == _lib.EINVAL) if L.vqa_log_probs_workspace(1, rows, width, 0) else (rc == _lib.ENODEVICE), (rows, width)
    assert L.vqa_log_probs_workspace(1, 5000, 2000, 8) == 0       # a wave a row: nothing is kept between kernels
    assert L.vqa_log_probs_workspace(1, 4, 10 ** 6, 8) > L.vqa_log_probs_workspace(1, 4, 10 ** 6, 0) > 0


def test_the_build_refuses_cut_literals(tmp_path):
    """every object of the library is made by the rule that searches its assembly, and the rule stops at a wide literal"""
    import os
    import subprocess

    csrc = os.path.join(os.path.dirname(os.path.abspath(vqa_amd.__file__)), "csrc")
    make = open(os.path.join(csrc, "Makefile")).read()
    body = make[make.index("define compile"):make.index("endef")]
    pattern = make[make.index("WIDE_MOVE :="):].splitlines()[0].split(":= ")[1]
    for rule in ("%.o:", "kern_hbm.o:", "kern_hbm_t11.o:"):
        assert make[make.index("\n" + rule):].split("\n")[2].startswith("\t$(call compile,")
    # a compiler that writes the assembly at hand in place of its own
    for move, fine in (("s_mov_b64 s[90:91], 0xfff0000000000000", False), ("s_mov_b64 s[0:1], 0x1000", True), ("s_mov_b64 s[0:1], 1.0", True),
                       ("s_mov_b64 s[0:1], -1 ; 0xfff0000000000000", True)):
        (tmp_path / "x.hip").write_text(move)
        (tmp_path / "cc").write_text('#!/bin/sh\nfor o; do :; done\ncp x.hip $(dirname $o)/x-gfx950.s && touch $o\n')
        (tmp_path / "cc").chmod(0o755)
        (tmp_path / "Makefile").write_text(f"HIPCC := ./cc\nARCH := gfx950\nWIDE_MOVE := {pattern}\n{body}endef\n\nx.o: x.hip\n\t$(call compile,)\n")
        run = subprocess.run(["make", "-B", "x.o"], cwd=tmp_path, capture_output=True, text=True)
        assert (run.returncode == 0) == fine and (tmp_path / "x.o").exists() == fine, run.stdout + run.stderr
        (tmp_path / "x.o").unlink(missing_ok=True)


def test_coefficients_that_shrink_small_singular_values():
    """refused where values are held as pairs of 16-bit floats, before anything else happens; not in the other forms"""
    call = lambda dtype, n, a: ortho(dtype=dtype, rows=n, cols=n + 9, sr=n + 9, sb=n * (n + 9), batch=0, g=None, out=None, k=k3(a, 0.5, -0.3))
    for dtype in (1, 2, 3):
        refused(call(dtype, 65, 0.99), _lib.EUNSUPPORTED, "shrink")
        refused(call(dtype, 65, -0.5), _lib.EUNSUPPORTED, "shrink")
        assert call(dtype, 65, 1.0) == 0 and call(dtype, 65, -1.1) == 0 and call(dtype, 64, 0.5) == 0
    assert call(0, 65, 0.5) == 0
