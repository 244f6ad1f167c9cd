"""8-bit state stores on the GPU against tests/_states8.py (float64 numpy)."""
import ctypes as C

import numpy as np
import pytest
import torch

from quake_amd import _lib, device as qdev
from tests import _states8 as S8

pytestmark = pytest.mark.gpu
NP = {torch.float32: S8.U32, torch.float16: S8.U16, torch.float64: 0.0}


@pytest.fixture(params=["auto", "wave", "tile", "thin"])
def path(request):
    """The kernel that takes the products: by the library's rule, always 32 x 32 tiles, always 128 x 128, the ones for few rows."""
    fn = _lib.load().qk_gram8_set_path
    fn.restype, fn.argtypes = C.c_int, [C.c_char_p]
    _lib.check(fn(request.param.encode()))
    yield request.param
    fn(b"auto")


def put(psi, single=False):
    t = torch.from_numpy(np.ascontiguousarray(psi)).cuda()
    return t.to(torch.complex64) if single else t


def fill(psi):
    """A store with these states, and what it holds: (store, q, gains)."""
    store = qdev.States8(max(len(psi), 1), psi.shape[1])
    if len(psi):
        store.write(put(psi))
    q = S8.rows(store.codes.cpu().numpy(), store.scales.cpu().numpy(), psi.shape[1])
    return store, q[:len(psi)], store.gains.cpu().numpy().astype(np.float64)[:len(psi)]


def check_k(K, a, ga, b, gb, symmetric=False):
    ref, t32, t8 = S8.kernel(a, ga, b, gb)
    if symmetric:
        np.fill_diagonal(ref, 1.0)
    got = K.cpu().numpy().astype(np.float64)
    # rounding K to its type: half a step, and half the smallest number of float16
    tol = (t8 if K.dtype == torch.float16 else t32) + NP[K.dtype] * np.abs(ref) + (2.0 ** -25 if K.dtype == torch.float16 else 0)
    off = np.abs(got - ref) - tol
    assert got.shape == ref.shape and (off <= 0).all(), (off.max(), np.unravel_index(off.argmax(), off.shape))
    if symmetric:
        assert np.array_equal(got, got.T) and (np.diag(got) == 1.0).all()


# ---- write / read ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("N,D,kind", [(1, 1, "spread"), (3, 2, "spread"), (100, 16, "product"), (7, 63, "spread"), (5, 64, "spread"),
                                      (9, 65, "product"), (33, 127, "spread"), (4, 129, "spread"), (6, 512, "product"),
                                      (2, 1000, "spread"), (1, 1024, "product"), (5, 1025, "spread"), (17, 4096, "product"),
                                      (2, 8193, "spread"), (3, 65536, "product")])
def test_write_and_read(N, D, kind, single):
    psi = S8.states(np.random.default_rng(N * 100003 + D), N, D, kind)
    if single:
        psi = psi.astype(np.complex64).astype(np.complex128)
    store = qdev.States8(N + 3, D)
    store.codes.fill_(0xEE), store.scales.fill_(0xEE), store.gains.fill_(-1)
    store.write(put(psi, single))
    codes, scales, gains = S8.write(psi)
    assert len(store) == N
    assert np.array_equal(store.codes.cpu().numpy()[:N], codes)
    assert np.array_equal(store.scales.cpu().numpy()[:N], scales)
    assert (np.abs(store.gains.cpu().numpy()[:N] - gains) <= 2 * S8.U32 * gains).all()      # one rounding of an FP64 quotient
    for rest, was in ((store.codes, 0xEE), (store.scales, 0xEE), (store.gains, -1)):        # rows behind the last stay
        assert (rest[N:] == was).all()
    q = S8.rows(codes, scales, D)
    assert np.array_equal(store.read().cpu().numpy().astype(np.complex128), q)
    assert np.array_equal(store.read(dtype=torch.complex128).cpu().numpy(), q)
    index = torch.tensor([N - 1, 0, 0, N, -1, 1 << 40, N // 2], device="cuda")
    got = store.read(index).cpu().numpy()
    assert np.array_equal(got[[0, 1, 2, 6]], q[[N - 1, 0, 0, N // 2]].astype(np.complex64))
    assert np.isnan(got[3:6].real).all() and np.isnan(got[3:6].imag).all()


def test_every_code_and_tie():
    """All e4m3 values, all midpoints between them and their FP64 neighbours, both signs, under the scale 448 fixes."""
    v = np.concatenate([S8.GRID, S8.HALF, np.nextafter(S8.HALF, 0), np.nextafter(S8.HALF, 1e3)])
    v = np.concatenate([v, -v])
    psi = np.zeros((len(v), 128), dtype=np.complex128)
    psi[:, 5], psi[:, 77] = v + 448j, -448.0 + 1j * v
    store, q, _ = fill(psi * 2.0 ** -60)
    codes, scales, _ = S8.write(psi)
    assert np.array_equal(store.codes.cpu().numpy(), codes) and (store.scales.cpu().numpy()[:, 0] == 127 - 60).all()


def test_scale_borders_and_tiny_blocks():
    """448 is the largest value that stays under a scale; blocks of 2^-100 and less; a block of zeros between others."""
    tops = [448.0, np.nextafter(448.0, 1e3), np.nextafter(448.0, 0), 256.0, 1.0, 2.0 ** -90, 1.75 * 2.0 ** -92, 2.0 ** -105, 2.0 ** -140, 0.0, 2.0 ** 60]
    psi = np.zeros((len(tops), 384), dtype=np.complex128)
    for k, t in enumerate(tops):
        psi[k, 3], psi[k, 300] = t, 0.3j * t
    store, _, g = fill(psi)
    codes, scales, gains = S8.write(psi)
    assert np.array_equal(store.codes.cpu().numpy(), codes) and np.array_equal(store.scales.cpu().numpy(), scales)
    assert (np.abs(g - gains) <= 2 * S8.U32 * gains).all() and g[9] == 0 and (scales[:, 1] == 127).all()


def test_values_that_are_not_finite(path):
    psi = S8.states(np.random.default_rng(4), 6, 300)
    psi[1, 10], psi[2, 200], psi[3, 299], psi[4, 0] = np.nan, np.inf, 1j * -np.inf, 1e39
    store, q, g = fill(psi)
    codes, scales, gains = S8.write(psi)
    assert np.array_equal(store.codes.cpu().numpy(), codes) and np.array_equal(store.scales.cpu().numpy(), scales)
    bad = [1, 2, 3, 4]
    assert np.isnan(g[bad]).all() and np.isfinite(g[[0, 5]]).all()
    for dtype in NP:
        K = qdev.gram8(store, dtype=dtype).cpu().numpy()
        assert np.isnan(K[bad][:, [0, 5]]).all() and np.isnan(K[0][bad]).all() and np.isfinite(K[[0, 5]][:, [0, 5]]).all()
    out = qdev.decision8(store, store.rows(5, 6), torch.ones(1, device="cuda")).cpu().numpy()
    assert np.isnan(out[bad]).all() and np.isfinite(out[[0, 5]]).all()


def test_write_appends_overwrites_and_takes_strides():
    rng = np.random.default_rng(1)
    D = 200
    psi = S8.states(rng, 12, D)
    wide = torch.zeros((12, D + 37), dtype=torch.complex128, device="cuda")
    wide[:, 7:7 + D] = put(psi)
    store = qdev.States8(12, D)
    store.write(wide[:5, 7:7 + D])
    store.write(wide[5:6, 7:7 + D])
    store.write(put(np.zeros((0, D), dtype=np.complex128)))
    store.write(wide[6:, 7:7 + D])
    codes, scales, gains = S8.write(psi)
    assert len(store) == 12 and np.array_equal(store.codes.cpu().numpy(), codes)
    store.write(put(psi[:2]), at=9)
    assert len(store) == 12
    got = store.codes.cpu().numpy()
    assert np.array_equal(got[9:11], codes[:2]) and np.array_equal(got[[8, 11]], codes[[8, 11]])
    every = wide[::3, 7:7 + D]                                   # a row stride that is a multiple
    store.clear()
    store.write(every)
    assert len(store) == 4 and np.array_equal(store.codes.cpu().numpy()[:4], codes[::3])


def test_more_rows_than_one_launch_takes():
    """2^26 rows and some: more threads than a launch may have, and code offsets far beyond 32 bits."""
    N = (1 << 26) + 70
    angle = torch.arange(N, device="cuda", dtype=torch.float32) * 0.37
    psi = torch.polar(0.5 + 0.5 * torch.sin(angle).abs(), angle).view(N, 1)
    store = qdev.States8(N, 1)
    store.write(psi)
    some = torch.tensor([0, 1, (1 << 26) - 5, (1 << 26) - 4, (1 << 26) - 1, 1 << 26, N - 2, N - 1], device="cuda")
    codes, scales, gains = S8.write(psi[some].cpu().numpy())
    assert np.array_equal(store.codes[some].cpu().numpy(), codes) and np.array_equal(store.scales[some].cpu().numpy(), scales)
    assert (np.abs(store.gains[some].cpu().numpy() - gains) <= 2 * S8.U32 * gains).all()
    q = S8.rows(codes, scales, 1)
    assert np.array_equal(store.read(some).cpu().numpy(), q.astype(np.complex64))
    K = qdev.gram8(store.rows(N - 2, N), store)
    check_k(K[:, some], q[-2:], gains[-2:], q, gains)
    check_k(qdev.gram8(store.rows(N - 2, N)), q[-2:], gains[-2:], q[-2:], gains[-2:], symmetric=True)
    few = qdev.gram8(store.rows(N - 260, N), store, dtype=torch.float16)      # 9 x 2^21 tiles of 32 x 32
    check_k(few[-2:, some], q[-2:], gains[-2:], q, gains)
    assert torch.equal(few[:, -260:], few[:, -260:].T)
    del few
    out = qdev.decision8(store.rows(N - 2, N), store.rows(N - 1, N), torch.full((1, 1), 2.0, device="cuda"))
    check_k(out / 2, q[-2:], gains[-2:], q[-1:], gains[-1:])


# ---- kernels -------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (2, 3, 2), (31, 33, 16), (100, 64, 16), (1, 500, 64), (32, 129, 65), (257, 1, 100), (65, 70, 128), (130, 131, 256),
          (200, 257, 1000), (3, 129, 4096), (129, 260, 2048), (1, 40, 65536), (70, 30, 16384), (40, 300, 8192), (8, 70, 300), (9, 33, 1025), (300, 2, 640), (65, 32, 100), (500, 5, 2048)]


@pytest.mark.parametrize("dtype", list(NP))
@pytest.mark.parametrize("M,N,D", SHAPES)
def test_gram8_cross(M, N, D, dtype, path):
    rng = np.random.default_rng(M * 7 + N * 13 + D)
    x, a, ga = fill(S8.states(rng, M, D, "product" if D > 1 else "spread"))
    y, b, gb = fill(S8.states(rng, N, D, "product" if M % 2 else "spread"))
    check_k(qdev.gram8(x, y, dtype=dtype), a, ga, b, gb)


@pytest.mark.parametrize("dtype", list(NP))
@pytest.mark.parametrize("N,D", [(1, 2), (2, 16), (31, 64), (100, 16), (129, 32), (64, 300), (257, 128), (300, 1024), (513, 256), (40, 65536), (200, 4096)])
def test_gram8_symmetric(N, D, dtype, path):
    x, a, ga = fill(S8.states(np.random.default_rng(N + D), N, D, "product"))
    check_k(qdev.gram8(x, dtype=dtype), a, ga, a, ga, symmetric=True)


@pytest.mark.parametrize("M,N,D", [(1500, 1100, 512), (1, 5000, 1024), (2, 3000, 4096), (33, 2000, 2048), (700, 700, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gram8_larger(M, N, D, dtype, path):
    rng = np.random.default_rng(D + M)
    x, a, ga = fill(S8.states(rng, M, D, "product"))
    y, b, gb = fill(S8.states(rng, N, D, "spread"))
    check_k(qdev.gram8(x, y, dtype=dtype), a, ga, b, gb)
    if M >= 700:
        check_k(qdev.gram8(x, dtype=dtype), a, ga, a, ga, symmetric=True)


@pytest.mark.parametrize("dtype", list(NP))
@pytest.mark.parametrize("N,M,D", [(4001, 0, 64), (4090, 0, 200), (4096, 0, 300), (2011, 4195, 60), (4195, 2011, 130), (16, 4096, 16)])
def test_gram8_a_full_round_and_a_few_tiles(N, M, D, dtype):
    """Up to 32 tiles of 128 x 128 behind the first 512 (another shape of the last tiles); beside a job that comes first too."""
    rng = np.random.default_rng(N + D)
    x, a, ga = fill(S8.states(rng, N, D, "product"))
    if not M:
        check_k(qdev.gram8(x, dtype=dtype), a, ga, a, ga, symmetric=True)
        return
    y, b, gb = fill(S8.states(rng, M, D, "spread"))
    z, c, gc = fill(S8.states(rng, 140, 256))
    KT = torch.full((M, N), -3.0, dtype=dtype, device="cuda")
    KZ, K = qdev.gram8_jobs([dict(A=z), dict(A=x, B=y, KT=KT)], dtype=dtype)
    check_k(KZ, c, gc, c, gc, symmetric=True)
    check_k(K, a, ga, b, gb)
    assert torch.equal(KT, K.T)
    check_k(qdev.gram8(x, y, dtype=dtype), a, ga, b, gb)


@pytest.mark.parametrize("dtype", list(NP))
def test_gram8_writes_its_block_only(dtype, path):
    rng = np.random.default_rng(8)
    x, a, ga = fill(S8.states(rng, 150, 256))
    y, b, gb = fill(S8.states(rng, 141, 256))
    for off, ld in ((0, 160), (3, 149), (5, 151)):                # aligned and odd rows
        big = torch.full((152, ld), -3.0, dtype=dtype, device="cuda")
        big_t = torch.full((143, 155), -3.0, dtype=dtype, device="cuda")
        K, KT = big[1:151, off:off + 141], big_t[1:142, 2:152]
        got = qdev.gram8_jobs([dict(A=x, B=y, K=K, KT=KT)])[0]
        assert got is K
        check_k(K, a, ga, b, gb)
        assert torch.equal(KT, K.T)
        keep, keep_t = torch.ones_like(big, dtype=torch.bool), torch.ones_like(big_t, dtype=torch.bool)
        keep[1:151, off:off + 141], keep_t[1:142, 2:152] = False, False
        assert (big[keep] == -3).all() and (big_t[keep_t] == -3).all()
    sym = torch.full((152, 161), -3.0, dtype=dtype, device="cuda")
    check_k(qdev.gram8(x, out=sym[1:151, 3:153]), a, ga, a, ga, symmetric=True)
    assert (sym[0] == -3).all() and (sym[151] == -3).all() and (sym[:, :3] == -3).all() and (sym[:, 153:] == -3).all()


def test_gram8_empty_sides_and_row_views():
    x, a, ga = fill(S8.states(np.random.default_rng(3), 90, 100))
    none = x.rows(40, 40)
    assert qdev.gram8(none, x).shape == (0, 90) and qdev.gram8(x, none).shape == (90, 0) and qdev.gram8(none).shape == (0, 0)
    check_k(qdev.gram8(x.rows(13, 60), x.rows(7, 8)), a[13:60], ga[13:60], a[7:8], ga[7:8])
    # a selection with repeats (the support vectors of a model)
    pick = torch.tensor([5, 5, 89, 0, 17], device="cuda")
    sel = qdev.States8.from_arrays(x.codes[pick], x.scales[pick], x.gains[pick], 100)
    p = pick.cpu().numpy()
    check_k(qdev.gram8(sel, x), a[p], ga[p], a, ga)


def test_gram8_zero_rows_and_unnormalised_rows():
    psi = S8.states(np.random.default_rng(6), 40, 256)
    psi[3] = 0
    psi[7] *= 1e-6
    psi[9] *= 1e5
    x, a, ga = fill(psi)
    y, b, gb = fill(S8.states(np.random.default_rng(7), 33, 256))
    K = qdev.gram8(x, y)
    check_k(K, a, ga, b, gb)
    assert (K[3] == 0).all()
    assert ga[3] == 0 and abs(ga[7] * np.sum(np.abs(a[7]) ** 2) - 1e-12) < 1e-18      # the gain keeps ||psi||^2


def test_population_of_ragged_sizes(path):
    rng = np.random.default_rng(12)
    shapes = [(1, 2), (100, 16), (33, 1024), (257, 64), (2, 65536), (500, 200), (64, 32), (31, 8), (129, 4096), (100, 512), (3, 3)] * 3
    held = [fill(S8.states(rng, n, d, "product")) for n, d in shapes]
    cross = [(fill(S8.states(rng, 17, d)), k) for k, (n, d) in enumerate(shapes) if k % 5 == 0]
    jobs = [dict(A=h[0]) for h in held] + [dict(A=c[0], B=held[k][0]) for c, k in cross] + [dict(A=held[0][0].rows(0, 0))]
    for dtype in (torch.float32, torch.float16):
        Ks = qdev.gram8_jobs(jobs, dtype=dtype)                   # more jobs than one launch takes
        for K, (_, q, g) in zip(Ks, held):
            check_k(K, q, g, q, g, symmetric=True)
        for K, (c, k) in zip(Ks[len(held):], cross):
            check_k(K, c[1], c[2], held[k][1], held[k][2])
        assert Ks[-1].shape == (0, 0)
    assert qdev.gram8_jobs([]) == []


# ---- decision values ---------------------------------------------------------------------------------------------------------
def check_decision(out, x, y, coef, intercept):
    (_, a, ga), (_, b, gb) = x, y
    K, tol, _ = S8.kernel(a, ga, b, gb)
    w = coef.astype(np.float64)
    ref = K @ w + (0 if intercept is None else intercept.astype(np.float64))
    # K's own error, one rounding of each product, and a sum whose partial sums stay below sum |K w|
    size = K @ np.abs(w)
    bound = tol @ np.abs(w) + (2 + 8 * np.sqrt(max(len(b), 1))) * S8.U32 * size + 2 * S8.U32 * np.abs(ref) + 1e-37
    off = np.abs(out.cpu().numpy().astype(np.float64) - ref) - bound
    assert out.shape == ref.shape and (off <= 0).all(), off.max()


@pytest.mark.parametrize("M,N,D,C", [(1, 1, 2, 1), (1, 1000, 1024, 1), (1, 33, 65536, 3), (33, 31, 16, 2), (100, 100, 16, 1), (257, 300, 200, 45),
                                     (129, 1000, 64, 64), (500, 700, 1024, 1), (1, 5000, 256, 10), (64, 128, 128, 33), (1300, 400, 512, 7),
                                     (2, 257, 4096, 5), (40, 2000, 100, 16), (8, 40, 1000, 64), (9, 300, 513, 2), (30, 65, 64, 64), (3, 2000, 16384, 4)])
def test_decision8(M, N, D, C, path):
    rng = np.random.default_rng(M + N + D + C)
    x, y = fill(S8.states(rng, M, D, "product")), fill(S8.states(rng, N, D, "spread"))
    coef = (rng.normal(size=(N, C)) * rng.choice([0, 1, 100], size=(N, 1))).astype(np.float32)
    b = rng.normal(size=C).astype(np.float32)
    cd, bd = torch.from_numpy(coef).cuda(), torch.from_numpy(b).cuda()
    check_decision(qdev.decision8(x[0], y[0], cd, bd), x, y, coef, b)
    check_decision(qdev.decision8(x[0], y[0], cd), x, y, coef, None)
    if C == 1:
        check_decision(qdev.decision8(x[0], y[0], cd[:, 0]), x, y, coef, None)
    wide = torch.zeros((N, C + 3), device="cuda")
    wide[:, 1:1 + C] = cd
    out = torch.full((M + 2, C + 5), -3.0, device="cuda")
    check_decision(qdev.decision8(x[0], y[0], wide[:, 1:1 + C], bd, out=out[1:M + 1, 2:2 + C]), x, y, coef, b)
    assert (out[0] == -3).all() and (out[M + 1] == -3).all() and (out[:, :2] == -3).all() and (out[:, 2 + C:] == -3).all()


@pytest.mark.parametrize("M,N,D,C", [(32, 4096, 4160, 3), (33, 100, 8192, 2), (7, 4097, 4200, 1), (31, 5, 20000, 64), (1, 1, 65536, 1)])
def test_decision8_few_long_rows(M, N, D, C):
    """Both sides of the sizes that go through K in memory; twice on one workspace, with an infinite coefficient in one column."""
    rng = np.random.default_rng(D)
    x, y = fill(S8.states(rng, M, D, "spread")), fill(S8.states(rng, N, D, "spread"))
    coef, b = rng.normal(size=(N, C)).astype(np.float32), rng.normal(size=C).astype(np.float32)
    cd, bd = torch.from_numpy(coef).cuda(), torch.from_numpy(b).cuda()
    out = qdev.decision8(x[0], y[0], cd, bd)
    check_decision(out, x, y, coef, b)
    assert torch.equal(qdev.decision8(x[0], y[0], cd, bd), out)
    cd[-1, 0] = float("inf")
    last = qdev.decision8(x[0], y[0], cd, bd)
    assert torch.isposinf(last[:, 0]).all() and torch.equal(last[:, 1:], out[:, 1:])


@pytest.mark.parametrize("C", [1, 8, 9, 32, 33, 45, 50])
def test_decision8_several_tiles_per_workgroup(C):
    """Sums that are carried from tile to tile, the last of them ragged."""
    rng = np.random.default_rng(C)
    x, y = fill(S8.states(rng, 6500, 20, "product")), fill(S8.states(rng, 2570, 20, "spread"))
    coef = rng.normal(size=(2570, C)).astype(np.float32)
    check_decision(qdev.decision8(x[0], y[0], torch.from_numpy(coef).cuda()), x, y, coef, None)


@pytest.mark.parametrize("M,N,D,C", [(70, 200, 64, 1), (70, 200, 64, 3), (70, 193, 64, 45), (3, 33, 1024, 2)])
def test_decision8_infinite_coefficients(M, N, D, C, path):
    """An infinite coefficient of the last row, whose place behind the end of a tile must not meet a zero."""
    rng = np.random.default_rng(M + C)
    x, y = fill(S8.states(rng, M, D, "product")), fill(S8.states(rng, N, D, "spread"))
    coef = rng.normal(size=(N, C)).astype(np.float32)
    coef[-1, 0] = np.inf
    out = qdev.decision8(x[0], y[0], torch.from_numpy(coef).cuda())
    assert (S8.kernel(x[1], x[2], y[1], y[2])[0][:, -1] > 0).all()
    assert torch.isposinf(out[:, 0]).all()
    if C > 1:
        check_decision(out[:, 1:], x, y, coef[:, 1:], None)


def test_decision8_empty_sides():
    x, y = fill(S8.states(np.random.default_rng(1), 9, 32)), fill(S8.states(np.random.default_rng(2), 4, 32))
    b = torch.tensor([1.5, -2.0], device="cuda")
    out = qdev.decision8(x[0], y[0].rows(0, 0), torch.zeros((0, 2), device="cuda"), b)
    assert torch.equal(out, b.expand(9, 2))
    assert (qdev.decision8(x[0], y[0].rows(0, 0), torch.zeros((0, 2), device="cuda")) == 0).all()
    assert qdev.decision8(x[0].rows(3, 3), y[0], torch.zeros((4, 2), device="cuda"), b).shape == (0, 2)


def test_decision8_gradient_by_coef():
    """The gradient of a loss by coef and intercept: the formula's, the swapped call's and central differences'."""
    rng = np.random.default_rng(21)
    x, y = fill(S8.states(rng, 150, 64)), fill(S8.states(rng, 90, 64))
    coef = rng.normal(size=(90, 3)).astype(np.float32)
    up = rng.normal(size=(150, 3)).astype(np.float32)                 # dloss / dout of loss = sum(up * out)
    grad = qdev.decision8(y[0], x[0], torch.from_numpy(up).cuda())
    check_decision(grad, y, x, up, None)
    g = grad.cpu().numpy().astype(np.float64)
    loss = lambda c: float((qdev.decision8(x[0], y[0], torch.from_numpy(c).cuda()).double() * torch.from_numpy(up).cuda()).sum())
    K, tol, _ = S8.kernel(x[1], x[2], y[1], y[2])
    for j, c in ((0, 0), (41, 1), (89, 2)):
        d = np.zeros_like(coef)
        d[j, c] = 0.5                                                 # the loss is linear in coef: the step needs no limit
        fd = loss(coef + d) - loss(coef - d)
        noise = 2 * (np.abs(up) * (K @ np.abs(coef))).sum() * 90 * S8.U32 + 2 * (tol[:, j] * np.abs(up[:, c])).sum()
        assert abs(fd - g[j, c]) < noise + 1e-5 * abs(g[j, c])


# ---- together, streams, graphs -----------------------------------------------------------------------------------------------
def test_results_do_not_depend_on_the_run():
    rng = np.random.default_rng(5)
    x, _, _ = fill(S8.states(rng, 300, 2048))
    y, _, _ = fill(S8.states(rng, 100, 2048))
    w = torch.from_numpy(rng.normal(size=(100, 4)).astype(np.float32)).cuda()
    K, Ky, o = qdev.gram8(x), qdev.gram8(x, y), qdev.decision8(x, y, w)
    for _ in range(3):
        assert torch.equal(qdev.gram8(x), K) and torch.equal(qdev.gram8(x, y), Ky) and torch.equal(qdev.decision8(x, y, w), o)


def test_train_then_serve_on_a_side_stream():
    """A training set written in pieces, its kernel, a ridge fit, and answers for single samples, on a stream of their own."""
    rng = np.random.default_rng(30)
    D, N = 256, 200
    train, test = S8.states(rng, N, D, "product"), S8.states(rng, 5, D, "product")
    target = np.sign(rng.normal(size=N))
    stream = torch.cuda.Stream()
    td, qd = put(train), put(test)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        store = qdev.States8(N, D)
        for a in range(0, N, 64):
            store.write(td[a:a + 64])
        K = qdev.gram8(store, dtype=torch.float64)
        coef = torch.linalg.solve(K + 0.1 * torch.eye(N, dtype=torch.float64, device="cuda"), torch.from_numpy(target).cuda())
        one = qdev.States8(1, D)
        outs = []
        for k in range(5):
            one.clear()
            one.write(qd[k:k + 1])
            outs.append(qdev.decision8(one, store, coef.float()))
    stream.synchronize()
    _, q, g = fill(train)
    _, t, gt = fill(test)
    Kt, tol, _ = S8.kernel(t, gt, q, g)
    w = coef.cpu().numpy()
    got = torch.cat(outs).cpu().numpy()[:, 0]
    bound = (tol + (3 + 8 * np.sqrt(N)) * S8.U32 * Kt) @ np.abs(w)      # + coef's rounding to FP32, in the 3
    assert (np.abs(got - Kt @ w) <= bound).all()


def test_captured_graphs_replay_beside_eager_work():
    rng = np.random.default_rng(31)
    D = 8192
    psi = [put(S8.states(rng, 3, D)) for _ in range(3)]
    x, y = qdev.States8(3, D), qdev.States8(200, D)
    y.write(put(S8.states(rng, 200, D, "product")))
    w = torch.from_numpy(rng.normal(size=(200, 2)).astype(np.float32)).cuda()
    inp = psi[0].clone()
    def step():
        x.clear()
        x.write(inp)
        return qdev.gram8(x, y), qdev.decision8(x, y, w), qdev.gram8(y)
    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step()
            graphs.append((g, out))
    torch.cuda.synchronize()
    for k in (1, 2, 0, 1):
        inp.copy_(psi[k])
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for g, out in graphs:
            for t in out:
                t.fill_(-1)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_refusals():
    x, y = qdev.States8(4, 64), qdev.States8(4, 65)
    psi = torch.zeros((4, 64), dtype=torch.complex128, device="cuda")
    bad = [lambda: x.write(psi.real), lambda: x.write(psi[:, :63]), lambda: x.write(psi.cpu()), lambda: x.write(psi.T.contiguous().T),
           lambda: x.write(psi.conj()), lambda: x.write(psi, at=1), lambda: x.write(torch.cat([psi, psi])), lambda: x.write(psi[0:1].expand(4, 64)),
           lambda: x.rows(0, 1), lambda: x.read(torch.zeros(1, dtype=torch.int32, device="cuda")), lambda: x.read(dtype=torch.float32),
           lambda: qdev.gram8(x, y), lambda: qdev.gram8(x, dtype=torch.bfloat16), lambda: qdev.gram8(psi),
           lambda: qdev.gram8(x, out=torch.zeros((1, 1), device="cuda")), lambda: qdev.decision8(x, y, torch.zeros((4, 1), device="cuda")),
           lambda: qdev.States8.from_arrays(x.codes, x.scales[:, :2], x.gains, 64), lambda: qdev.States8(-1, 64)]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {k} was taken")
    x.write(psi)
    assert len(x) == 4
    more = [lambda: qdev.gram8(x, out=torch.zeros((4, 4), device="cuda").T[:, ::2]), lambda: qdev.gram8(x, out=torch.zeros((4, 4))),
            lambda: qdev.gram8_jobs([dict(A=x, KT=torch.zeros((4, 4), device="cuda"))]),
            lambda: qdev.decision8(x, x, torch.zeros((4, 65), device="cuda")), lambda: qdev.decision8(x, x, torch.zeros((4, 0), device="cuda")),
            lambda: qdev.decision8(x, x, torch.zeros((3, 1), device="cuda")), lambda: qdev.decision8(x, x, torch.zeros((4, 1), dtype=torch.float64, device="cuda")),
            lambda: qdev.decision8(x, x, torch.zeros((4, 2), device="cuda"), torch.zeros(1, device="cuda")),
            lambda: qdev.decision8(x, x, torch.zeros((2, 4), device="cuda").T)]
    for k, f in enumerate(more):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {k} was taken")


# ---- the framework's own paths ---------------------------------------------------------------------------------------------
def fp8_kernel(circ, X, Y=None):
    """K of HipFidelityKernel(precision="fp8") in float64 from the library's own FP64 states, with its error bound."""
    from quake_amd.kernels import HipFidelityKernel
    exact = HipFidelityKernel(circ)
    def side(v):
        codes, scales, gains = S8.write(exact.statevectors(v))
        return S8.rows(codes, scales, 1 << circ.num_qubits), gains.astype(np.float32).astype(np.float64)
    a, ga = side(X)
    b, gb = (a, ga) if Y is None else side(Y)
    K, tol, _ = S8.kernel(a, ga, b, gb)
    if Y is None:
        np.fill_diagonal(K, 1.0)
    return K, tol


@pytest.mark.parametrize("n,N,M", [(1, 5, 3), (4, 100, 17), (6, 33, 70), (8, 300, 1), (12, 40, 65), (14, 5, 9)])
def test_kernel_object_fp8(n, N, M):
    from quake_amd import featuremaps as fm
    from quake_amd.circuit import ParameterVector
    from quake_amd.kernels import HipFidelityKernel
    rng = np.random.default_rng(n)
    X, Y = rng.uniform(-1.5, 1.5, size=(N, n)), rng.uniform(-1.5, 1.5, size=(M, n))
    circ = fm.zz_featuremap(ParameterVector("x", n), n, 2) if n > 1 else fm.z_featuremap(ParameterVector("x", n), n, 2)
    k8 = HipFidelityKernel(circ, precision="fp8")
    K = k8.evaluate(X)
    ref, tol = fp8_kernel(circ, X)
    assert K.dtype == np.float64 and np.array_equal(K, K.T) and (np.diag(K) == 1).all() and (np.abs(K - ref) <= tol).all()
    assert np.linalg.eigvalsh(K).min() > -(tol.max() + 1e-12) * N            # positive semidefinite up to its rounding
    ref, tol = fp8_kernel(circ, X, Y)
    assert (np.abs(k8.evaluate(X, Y) - ref) <= tol).all()
    out = np.empty((N, N))
    assert k8.evaluate(X, out=out) is out and np.array_equal(out, K)
    full = HipFidelityKernel(circ).evaluate(X)
    assert np.abs(K - full).max() <= 0.13
    shots = HipFidelityKernel(circ, precision="fp8", shots=1000, seed=3)
    S = shots.evaluate(X)
    assert np.array_equal(S, S.T) and (S * 1000 == np.round(S * 1000)).all() and np.abs(S - K).max() < 6 * 0.5 / np.sqrt(1000)


def test_kernel_object_fp8_in_bands():
    """Enough rows for the host path's bands (symmetric blocks, mirrored blocks) and for several batches of states."""
    from quake_amd import featuremaps as fm
    from quake_amd.circuit import ParameterVector
    from quake_amd.kernels import HipFidelityKernel
    rng = np.random.default_rng(0)
    X = rng.uniform(-1.5, 1.5, size=(4500, 6))
    circ = fm.zz_featuremap(ParameterVector("x", 6), 6, 1)
    K = HipFidelityKernel(circ, precision="fp8").evaluate(X)
    assert np.array_equal(K, K.T) and (np.diag(K) == 1).all()
    pick = np.concatenate([np.arange(0, 4500, 271), [1023, 1024, 1151, 1152, 4499]])
    ref, tol = fp8_kernel(circ, X[pick], X)
    got = K[pick]
    own = np.zeros(got.shape, dtype=bool)
    own[np.arange(len(pick)), pick] = True
    assert (np.abs(got - ref)[~own] <= tol[~own]).all()
    Kx = HipFidelityKernel(circ, precision="fp8").evaluate(X, X[:77])
    ref, tol = fp8_kernel(circ, X[pick], X[:77])
    same = pick[:, None] == np.arange(77)[None, :]                  # equal rows: exactly one, as in every precision
    assert (np.abs(Kx[pick] - ref)[~same] <= tol[~same]).all() and (Kx[pick][same] == 1).all()


def test_population_fp8():
    from quake_amd import featuremaps as fm
    from quake_amd.circuit import ParameterVector
    from quake_amd.kernels import evaluate_population
    rng = np.random.default_rng(5)
    sizes = [(2, 30), (4, 100), (10, 129), (3, 64), (11, 20), (4, 7)] * 5          # wave-resident circuits and one that is not
    maps = [fm.zz_featuremap(ParameterVector("x", n), n, 1) for n, _ in sizes]
    xs = [rng.uniform(-1.5, 1.5, size=(N, n)) for n, N in sizes]
    labels = [rng.integers(0, 2, size=N) for _, N in sizes]
    Ks, stats = evaluate_population(maps, xs, labels=labels, precision="fp8")
    _, exact = evaluate_population(maps, xs, labels=labels)
    for circ, x, K, st, ex in zip(maps, xs, Ks, stats, exact):
        ref, tol = fp8_kernel(circ, x)
        assert np.array_equal(K, K.T) and (np.diag(K) == 1).all() and (np.abs(K - ref) <= tol).all()
        assert abs(st["offdiagonal_mean"] - np.triu(K, 1).mean()) < 1e-12
        assert abs(st["offdiagonal_mean"] - ex["offdiagonal_mean"]) < 0.13
    big, _ = evaluate_population(maps[1:2], [rng.uniform(-1.5, 1.5, size=(1100, 4))], precision="fp8")     # one by one above 1024 rows
    assert (np.diag(big[0]) == 1).all() and np.linalg.eigvalsh(big[0]).min() > -1e-4
    noisy, _ = evaluate_population(maps[:2], xs[:2], noise=("gaussian", 0.01), seed=4, precision="fp8")
    assert 0.001 < np.abs(noisy[1] - Ks[1]).max() < 0.1


@pytest.mark.parametrize("classes", [2, 3, 10])
def test_served_svc(classes):
    from sklearn.svm import SVC
    from quake_amd import featuremaps as fm
    from quake_amd.circuit import ParameterVector
    from quake_amd.kernels import HipFidelityKernel
    from quake_amd.serving import ServedSVC
    rng = np.random.default_rng(classes)
    n, N = 6, 300
    X, Q = rng.uniform(-1.5, 1.5, size=(N, n)), rng.uniform(-1.5, 1.5, size=(41, n))
    y = (X[:, 0] * 2 + X[:, 1] > np.linspace(-3, 3, classes + 1)[1:-1, None]).sum(axis=0)
    circ = fm.custom2_featuremap(ParameterVector("x", n), n, 1)
    kernel = HipFidelityKernel(circ, precision="fp8")
    svc = SVC(kernel="precomputed", C=5, decision_function_shape="ovo").fit(kernel.evaluate(X), y)
    served = ServedSVC(kernel, svc, X)
    Kq = kernel.evaluate(Q, X)
    want = svc.decision_function(Kq).reshape(41, -1)
    coef = np.abs(svc.dual_coef_).sum()
    got = served.decision_function(Q).reshape(41, -1)
    # every entry of K is at most 1: FP32's rounding of the coefficients, the products and their sum; and two computations of K,
    # each off by 2 sqrt(2) sqrt(K) 8 sqrt(2 D) U32 S (tests/_states8.py) with S <= sqrt(2) (1 + 2^-4)^2
    k_error = 2 * np.sqrt(2) * 8 * np.sqrt(2.0 ** (n + 1)) * S8.U32 * np.sqrt(2) * 1.13
    assert np.abs(got - want).max() <= ((3 + 8 * np.sqrt(N)) * S8.U32 + 2 * k_error) * coef
    assert np.array_equal(served.decision_function(Q[3]).ravel(), served.decision_function(Q[3:4]).ravel())
    clear = np.abs(want).min(axis=1) > 1e-3
    assert np.array_equal(served.predict(Q)[clear], svc.predict(Kq)[clear]) and clear.sum() > 20
