"""8-bit state stores on a machine without a GPU: the numpy twin the GPU tests compare with, the layout, the refusals of the
C entry points (all of them come before anything touches a device)."""
import ctypes as C

import numpy as np
import pytest

from quake_amd import _lib, build
from tests import _states8 as S8


@pytest.fixture(scope="module")
def lib():
    if build.needs_build():
        build.build_library(verbose=False)
    return _lib.load()


def test_twin_encodes_every_value_and_tie():
    assert np.array_equal(S8.encode(S8.GRID), np.arange(127)) and np.array_equal(S8.encode(-S8.GRID[1:]), np.arange(1, 127) + 128)
    mid = S8.encode(S8.HALF)
    assert (mid % 2 == 0).all()
    eps = np.spacing(S8.HALF)
    assert np.array_equal(S8.encode(S8.HALF - eps), np.arange(126)) and np.array_equal(S8.encode(S8.HALF + eps), np.arange(1, 127))
    assert S8.GRID[126] == 448.0 and S8.GRID[1] == 2.0 ** -9


@pytest.mark.parametrize("kind", ["spread", "product"])
@pytest.mark.parametrize("D", [2, 16, 100, 1024])
def test_stored_states_keep_norm_and_angle(kind, D):
    rng = np.random.default_rng(D)
    psi = S8.states(rng, 20, D, kind)
    codes, scales, gains = S8.write(psi)
    q = S8.rows(codes, scales, D)
    # a component is off by 2^-4 of itself at most, or by half the smallest step
    assert (np.abs((q - psi).real) <= np.maximum(2.0 ** -4 * np.abs(psi.real), 2.0 ** -10 * np.exp2(scales.max() - 127.0))).all()
    K, _, _ = S8.kernel(q, gains, q, gains)
    assert np.abs(np.diag(K) - 1).max() < 1e-12
    assert np.linalg.eigvalsh(K).min() > -1e-12
    ref = np.abs(psi.conj() @ psi.T) ** 2
    assert np.abs(K - ref).max() <= 0.13          # two angles of asin(2^-4): |dK| <= sin(2 asin(2^-4)) = 0.1247


def test_layout(lib):
    c, s = C.c_int64(), C.c_int64()
    for D, want in [(1, (128, 4)), (64, (128, 4)), (65, (256, 4)), (512, (1024, 4)), (513, (1152, 8)), (65536, (131072, 512))]:
        assert lib.qk_states8_layout(D, C.byref(c), C.byref(s)) == 0 and (c.value, s.value) == want
    for D in (0, -1, (1 << 26) + 1):
        assert lib.qk_states8_layout(D, C.byref(c), C.byref(s)) == _lib.QK_ERR_INVALID
    assert lib.qk_states8_layout(8, None, C.byref(s)) == _lib.QK_ERR_INVALID


def _store(rows, base=1 << 20):
    return _lib.qk_states8(base, base + 4096, base + 8192, rows)


def test_gram8_refusals(lib):
    def call(ws=None, nbytes=0, n=1, **kw):
        j = _lib.qk_gram8_job()
        j.A, j.B, j.D, j.K, j.KT, j.ldk, j.ldkt, j.flags = _store(8), _store(8, 1 << 21), 256, 1 << 22, None, 8, 8, 0
        for k, v in kw.items():
            setattr(j, k, v)
        return lib.qk_gram8_jobs_dev(C.byref(j), n, ws, nbytes, None)
    bad = _lib.QK_ERR_INVALID
    assert call(D=0) == bad and call(D=1 << 27) == bad
    assert call(ldk=7) == bad and "leading dimension" in _lib.last_error()
    assert call(KT=1 << 23, ldkt=7) == bad
    assert call(K=None) == bad
    assert call(flags=2 | 4) == bad and call(flags=64) == bad
    assert call(flags=1) == bad and "same store" in _lib.last_error()
    assert call(A=_store(8, (1 << 20) + 8)) == bad and "alignment" in _lib.last_error()
    assert call(A=_lib.qk_states8(None, None, None, 3)) == bad
    assert call(A=_store(-1)) == bad and call(A=_store(1 << 31)) == _lib.QK_ERR_UNSUPPORTED
    assert call(n=-1) == bad
    same = dict(A=_store(8), B=_store(8), flags=1)
    assert call(KT=1 << 23, **same) == bad and "mirror" in _lib.last_error()
    assert call(D=65536, A=_store(1)) == bad and "workspace" in _lib.last_error()      # one long row: sums in slices
    need = C.c_size_t(7)
    assert lib.qk_gram8_workspace(None, 0, C.byref(need)) == 0 and need.value == 0
    assert lib.qk_gram8_workspace(None, 1, C.byref(need)) == bad
    assert lib.qk_gram8_jobs_dev(None, 0, None, 0, None) == 0
    assert call(A=_lib.qk_states8(None, None, None, 0), K=None) == 0                    # an empty block: nothing to do


def test_states8_refusals(lib):
    bad = _lib.QK_ERR_INVALID
    to = _store(4)
    w = lambda psi=1 << 24, f32=0, ld=256, D=256, to=to: lib.qk_states8_write_dev(psi, f32, ld, D, C.byref(to), None)
    assert w(psi=None) == bad and w(ld=255) == bad and w(D=0) == bad and w(psi=(1 << 24) + 8) == bad
    assert w(psi=(1 << 24) + 4, f32=1) == bad and w(to=_store(-2)) == bad
    assert lib.qk_states8_write_dev(1 << 24, 0, 256, 256, None, None) == bad
    assert w(psi=None, to=_lib.qk_states8(None, None, None, 0)) == 0
    r = lambda index=None, N=4, psi=1 << 24, f32=1, ld=256, D=256: lib.qk_states8_read_dev(C.byref(to), D, index, N, psi, f32, ld, None)
    assert r(N=5) == bad and r(N=-1) == bad and r(psi=None) == bad and r(ld=3) == bad and r(psi=(1 << 24) + 8, f32=0) == bad
    assert r(N=0) == 0


def test_decision8_refusals(lib):
    bad = _lib.QK_ERR_INVALID
    need = C.c_size_t()
    assert lib.qk_decision8_workspace(5, 5, 16, 0, C.byref(need)) == _lib.QK_ERR_UNSUPPORTED
    assert lib.qk_decision8_workspace(5, 5, 16, 65, C.byref(need)) == _lib.QK_ERR_UNSUPPORTED
    assert lib.qk_decision8_workspace(-1, 5, 16, 1, C.byref(need)) == bad
    assert lib.qk_decision8_workspace(1, 100000, 16, 1, C.byref(need)) == 0 and need.value > 0
    x, y = _store(8), _store(9, 1 << 21)

    def call(x=x, y=y, D=16, coef=1 << 22, ldc=2, C_=2, b=None, out=1 << 23, ldo=2, ws=1 << 25, nbytes=1 << 30):
        return lib.qk_decision8_dev(C.byref(x), C.byref(y), D, coef, ldc, C_, b, out, ldo, ws, nbytes, None)
    assert call(coef=None) == bad and call(out=None) == bad and call(ldc=1) == bad and call(ldo=1) == bad
    assert call(x=_store(1), y=_store(100000), nbytes=0) == bad and "workspace" in _lib.last_error()
    assert call(x=_lib.qk_states8(None, None, None, 0)) == 0
    assert lib.qk_decision8_dev(None, C.byref(y), 16, 1, 2, 2, None, 1, 2, None, 0, None) == bad


def test_python_entry_points_refuse_cpu_tensors():
    import torch
    from quake_amd import device as qdev
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    with pytest.raises(ValueError):
        qdev.States8.from_arrays(u8(3, 128), u8(3, 4), torch.zeros(3), 16)
    with pytest.raises(ValueError):
        qdev.States8(4, 16, device="cpu")
    for dim in (0, (1 << 26) + 1):
        with pytest.raises(ValueError):
            qdev.States8(4, dim)


@pytest.mark.parametrize("classes", [2, 3, 5])
def test_pair_coefficients_are_sklearns_decision(classes):
    from sklearn.svm import SVC
    from quake_amd.serving import pair_coefficients
    rng = np.random.default_rng(classes)
    psi = S8.states(rng, 60, 16, "product")
    K = np.abs(psi.conj() @ psi.T) ** 2
    y = rng.integers(0, classes, size=60)
    svc = SVC(kernel="precomputed", C=10, decision_function_shape="ovo").fit(K, y)
    coef, b = pair_coefficients(svc)
    want = svc.decision_function(K).reshape(60, -1)
    got = K[:, svc.support_] @ coef + b
    assert coef.shape == (len(svc.support_), classes * (classes - 1) // 2)
    assert np.abs(got - want).max() < 1e-9 * np.abs(want).max()


def test_served_svc_refusals():
    from sklearn.svm import SVC
    from quake_amd import circuit as qc, featuremaps as fm
    from quake_amd.kernels import HipFidelityKernel
    from quake_amd.serving import ServedSVC
    k = HipFidelityKernel(fm.zz_featuremap(qc.ParameterVector("x", 3), 3, 1))
    X, y = np.random.default_rng(0).uniform(size=(20, 3)), np.arange(20) % 2
    with pytest.raises(ValueError):
        ServedSVC(k, SVC(kernel="rbf").fit(X, y), X)
    with pytest.raises(ValueError):
        ServedSVC(k, SVC(kernel="precomputed"), X)
    svc = SVC(kernel="precomputed").fit(X @ X.T, y)
    with pytest.raises(ValueError):
        ServedSVC(k, svc, X[:19])
    with pytest.raises(ValueError):
        ServedSVC(k, svc, X[:, :2])
    many = SVC(kernel="precomputed").fit(np.eye(24), np.arange(24) % 12)
    with pytest.raises(ValueError, match="classes"):
        ServedSVC(k, many, np.zeros((24, 3)))


def test_precision_names():
    from quake_amd import circuit as qc, featuremaps as fm, ga
    from quake_amd.kernels import HipFidelityKernel, evaluate_population, make_kernels
    fmap = fm.z_featuremap(qc.ParameterVector("x", 2), 2)
    assert make_kernels([fmap], precision="fp8")[0]._precision == "fp8"
    with pytest.raises(ValueError):
        HipFidelityKernel(fmap, precision="half")
    with pytest.raises(ValueError):
        evaluate_population([fmap], [np.zeros((3, 2))], precision="single")
    with pytest.raises(ValueError, match="projected"):
        ga.generation_fitness([], np.zeros((3, 2)), np.zeros(3), {}, 2, 1, 2, lambda accuracy: 0, projected=True, precision="fp8")


def test_evaluate8_and_batch_refusals(lib):
    from quake_amd import circuit as qc, featuremaps as fm
    h = _lib.CircuitHandle(fm.z_featuremap(qc.ParameterVector("x", 2), 2).compile())
    X, K = np.zeros((3, 2)), np.zeros((3, 3))
    call = lambda x=X.ctypes.data, n=3, f=2, mode=0, k=K.ctypes.data: lib.qk_evaluate8(h.handle, x, n, None, 0, f, mode, 0.0, 0, k)
    bad = _lib.QK_ERR_INVALID
    assert call(f=3) == bad and call(n=-1) == bad and call(x=None) == bad and call(mode=9) == bad and call(k=None) == bad
    assert call(n=0) == 0
    opts = _lib.qk_batch_opts(0, 2, 0.0, 0)
    P = C.c_void_p
    assert lib.qk_evaluate_batch(1, (P * 1)(h.handle), (P * 1)(X.ctypes.data), (C.c_int64 * 1)(3), None, C.byref(opts),
                                 (P * 1)(K.ctypes.data), None) == bad and "flag" in _lib.last_error()
