"""Values of the 8-bit stores' operators held to the arithmetic that the header states, against tests/_states8.py."""
import ctypes as C

import numpy as np
import pytest
import torch

from quake_amd import _lib, device as qdev
from tests import _states8 as S8
from tests.test_gpu_states8 import check_decision, fill, path, put  # noqa: F401  (path is a fixture)

pytestmark = pytest.mark.gpu


def half_step(v):
    """Half the distance of float16 numbers at v >= 0."""
    return np.exp2(np.maximum(np.frexp(np.maximum(v, 1e-30))[1] - 1, -14) - 11.0)


def close_states(rng, N, D):
    """States near one another: every K is near 1, where a sum that is cut shows most."""
    one = S8.states(rng, 1, D, "product")
    psi = one + 0.1 * S8.states(rng, N, D)
    return psi / np.linalg.norm(psi, axis=1, keepdims=True)


# ---- float16 K: FP32 sums, rounded once ------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,N,D,kind", [(130, 131, 256, "close"), (700, 500, 128, "close"), (300, 300, 16, "product"), (1100, 1000, 512, "close"),
                                        (257, 129, 300, "spread"), (64, 300, 64, "product"), (5, 400, 200, "close"), (1500, 1200, 65, "spread")])
def test_half_kernel_is_rounded_once(M, N, D, kind, path):
    """Off by FP32's bound and half a step of float16, whatever kernel takes the product."""
    rng = np.random.default_rng(M + N + D)
    make = close_states if kind == "close" else lambda r, n, d: S8.states(r, n, d, kind)
    states = make(rng, M + N, D)
    x, a, ga = fill(states[:M])
    y, b, gb = fill(states[M:])
    ref, t32, _ = S8.kernel(a, ga, b, gb)
    off = np.abs(qdev.gram8(x, y, dtype=torch.float16).cpu().numpy().astype(np.float64) - ref) - (t32 + half_step(ref + t32))
    assert (off <= 0).all(), (off.max(), (off > 0).sum())
    ref, t32, _ = S8.kernel(a, ga, a, ga)
    np.fill_diagonal(ref, 1.0)
    off = np.abs(qdev.gram8(x, dtype=torch.float16).cpu().numpy().astype(np.float64) - ref) - (t32 + half_step(ref + t32))
    assert (off <= 0).all(), (off.max(), (off > 0).sum())


@pytest.mark.parametrize("M,N,D", [(130, 131, 256), (700, 900, 4096), (33, 2000, 2048), (1, 5000, 1024), (20, 300, 16384), (200, 0, 16384), (700, 0, 512),
                                   (1200, 0, 8192), (4090, 0, 256), (3000, 2000, 64)])
def test_half_and_double_kernel_are_the_single_one_converted(M, N, D, path):
    """One arithmetic for all types of K: FP32 sums, converted once."""
    rng = np.random.default_rng(M + N + D)
    x = fill(S8.states(rng, M, D, "product"))[0]
    y = fill(S8.states(rng, N, D, "product"))[0] if N else None
    K = qdev.gram8(x, y)
    assert torch.equal(qdev.gram8(x, y, dtype=torch.float16), K.half())
    assert torch.equal(qdev.gram8(x, y, dtype=torch.float64), K.double())


# ---- decision values --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,N,D,C", [(1, 33, 16, 64), (8, 200, 448, 64), (20, 40, 64, 64), (32, 129, 100, 1), (3, 4, 2, 63)])
def test_short_rows_many_columns_every_run(M, N, D, C):
    """Rows of fewer than 8 chunks against few others: every wave's sums start from its own zeros, run after run."""
    rng = np.random.default_rng(M + N + D + C)
    x, y = fill(S8.states(rng, M, D, "spread")), fill(S8.states(rng, N, D, "spread"))
    coef = rng.normal(size=(N, C)).astype(np.float32)
    cd = torch.from_numpy(coef).cuda()
    first = qdev.decision8(x[0], y[0], cd)
    check_decision(first, x, y, coef, None)
    for _ in range(50):
        assert torch.equal(qdev.decision8(x[0], y[0], cd), first)


# ---- copies of a store ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("again", ["deepcopy", "pickle"])
def test_a_copy_has_memory_of_its_own(again):
    import copy
    import pickle
    psi = S8.states(np.random.default_rng(3), 9, 200)
    x, a, ga = fill(psi)
    before = x.codes.clone()
    t = copy.deepcopy(x) if again == "deepcopy" else pickle.loads(pickle.dumps(x))
    t.write(put(psi[::-1]), at=0)
    assert torch.equal(x.codes, before) and torch.equal(t.codes, before.flip(0))
    del x
    K, t32, _ = S8.kernel(a[::-1], ga[::-1], a[::-1], ga[::-1])
    np.fill_diagonal(K, 1.0)
    assert (np.abs(qdev.gram8(t).cpu().numpy() - K) <= t32 + S8.U32 * K).all()


# ---- served models ----------------------------------------------------------------------------------------------------------
def test_served_svc_answers_at_once_on_another_stream():
    """A model whose simulation takes a while, asked on a side stream as soon as it is there."""
    from sklearn.svm import SVC
    from quake_amd import featuremaps as fm
    from quake_amd.circuit import ParameterVector
    from quake_amd.kernels import HipFidelityKernel
    from quake_amd.serving import ServedSVC
    rng = np.random.default_rng(2)
    n, N = 4, 60
    X, Q = rng.uniform(-1.5, 1.5, size=(N, n)), rng.uniform(-1.5, 1.5, size=(7, n))
    kernel = HipFidelityKernel(fm.zz_featuremap(ParameterVector("x", n), n, 1), precision="fp8")
    svc = SVC(kernel="precomputed").fit(kernel.evaluate(X), (X[:, 0] > 0).astype(int))
    want = ServedSVC(kernel, svc, X).decision_function(Q)
    q = torch.from_numpy(Q).cuda()
    slow, plain = qdev.DeviceCircuit.simulate, torch.cuda._sleep
    try:
        qdev.DeviceCircuit.simulate = lambda self, x, **k: (plain(100_000_000), slow(self, x, **k))[1]
        served = ServedSVC(kernel, svc, X)
    finally:
        qdev.DeviceCircuit.simulate = slow
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = served.decide(q)
    side.synchronize()
    assert np.array_equal(got.cpu().numpy()[:, 0], want)


# ---- the host path's own account ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("N", [40, 3000])
def test_profile_of_the_last_call_is_the_fp8_one(N):
    """The itemised time of a call starts from zero and ends with the call's own total."""
    import time
    from quake_amd import featuremaps as fm
    from quake_amd.circuit import ParameterVector
    from quake_amd.kernels import HipFidelityKernel
    fn = _lib.load().qk_evaluate_profile
    fn.restype, fn.argtypes = C.c_int, [C.POINTER(C.c_double), C.c_int]
    t = (C.c_double * 8)()
    circ = fm.zz_featuremap(ParameterVector("x", 4), 4, 1)
    X = np.random.default_rng(1).uniform(-1, 1, size=(N, 4))
    HipFidelityKernel(circ).evaluate(np.random.default_rng(2).uniform(-1, 1, size=(6000, 4)))       # a longer call before
    kernel = HipFidelityKernel(circ, precision="fp8")
    for _ in range(3):
        begin = time.perf_counter()
        kernel.evaluate(X)
        wall = time.perf_counter() - begin
        assert fn(t, 8) == 0
        total, parts = t[6], sum(t[:6])
        assert 0 < parts <= total * (1 + 1e-9) and total <= wall and t[0] > 0 and t[2] > 0


# ---- gains --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("single", [False, True])
def test_gains_are_rounded_once(single):
    """Sums of squares in FP64: what is left is the quotient's rounding to float32 (and FP64's, 300 times 2^-53 at most).  Four
    amplitudes of one lane, one of them large and the others in the lower half of the format."""
    rng = np.random.default_rng(6)
    psi = np.zeros((2000, 128), dtype=np.complex128)
    for k, at in enumerate((9, 41, 73, 105)):
        scale = 1.0 if k == 0 else 2.0 ** -10
        psi[:, at] = scale * (rng.uniform(0.3, 1, 2000) + 1j * rng.uniform(0.3, 1, 2000))
    psi[:1000] = S8.states(rng, 1000, 128)
    if single:
        psi = psi.astype(np.complex64).astype(np.complex128)
    store = qdev.States8(2000, 128)
    store.write(put(psi, single))
    gains = S8.write(psi)[2]
    off = np.abs(store.gains.cpu().numpy() - gains) / gains
    assert (off <= S8.U32 * (1 + 1e-6) + 300 * 2.0 ** -53).all(), ((off > S8.U32 * (1 + 1e-6)).sum(), off.max() / S8.U32)


# ---- rows that are not finite -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("N,D", [(1, 4), (3, 100), (40, 300), (200, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_diagonal_of_a_symmetric_kernel_is_one_for_every_row(N, D, dtype, path):
    """As of every symmetric job: also for a row of zeros and for one with a NaN, whose other entries are 0 and NaN."""
    psi = S8.states(np.random.default_rng(N), N, D)
    psi[0, 0] = np.nan
    if N > 2:
        psi[2] = 0
    x, _, _ = fill(psi)
    K = qdev.gram8(x, dtype=dtype).cpu().numpy()
    assert (np.diag(K) == 1).all() and np.isnan(K[0, 1:]).all() and np.isnan(K[1:, 0]).all()
    if N > 2:
        assert (np.delete(K[2], [0, 2]) == 0).all()
    cross = qdev.gram8(x, x.rows(0, N), dtype=dtype).cpu().numpy()
    assert np.isnan(cross[0]).all()
