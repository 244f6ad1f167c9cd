"""The 8-bit state store and its products in float64 numpy, from their formulas, with the error bounds that the tests use."""
import numpy as np

U32 = 2.0 ** -24      # half a step of FP32, relative
U16 = 2.0 ** -11      # half a step of FP16, relative


def e4m3_grid():
    """The finite non-negative e4m3 values in the order of their codes 0 .. 126."""
    sub = [f * 2.0 ** -9 for f in range(8)]
    return np.array((sub + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8)])[:127])


GRID = e4m3_grid()
HALF = (GRID[1:] + GRID[:-1]) / 2


def encode(v):
    """float64 |v| <= 448 (or NaN) -> code bytes, nearest, ties to the even code."""
    a = np.abs(v)
    i = np.searchsorted(HALF, a, side="left")                       # a on a midpoint: the lower code ...
    tie = (i < 126) & (a == HALF[np.minimum(i, 125)]) & (i % 2 == 1)
    code = (i + tie).astype(np.int64)                               # ... unless that is odd
    code = np.where(np.isnan(v), 127, code)
    return np.where(np.signbit(v) & ~np.isnan(v), code + 128, code).astype(np.uint8)


def decode(c):
    c = c.astype(np.int64)
    v = np.append(GRID, np.nan)[c & 127]
    return np.where(c >= 128, -v, v)


def write(psi):
    """codes [N, 128 ceil(D/64)], scales [N, 4 ceil(D/512)], gains float64 [N] of complex rows."""
    psi = np.asarray(psi, dtype=np.complex128)
    N, D = psi.shape
    chunks, blocks = -(-D // 64), -(-D // 128)
    part = np.zeros((N, blocks * 128, 2))
    part[:, :D, 0], part[:, :D, 1] = psi.real, psi.imag
    part = np.where(np.abs(part) < 2.0 ** 128, part, np.nan)         # not finite in FP32
    part = part.reshape(N, blocks, 128, 2)
    top = np.nan_to_num(np.abs(part), nan=0.0).max(axis=(2, 3))
    m, x = np.frexp(top)
    e = np.where(top > 0, np.maximum(x - np.where(m <= 0.875, 9, 8), -100), 0)
    code = encode(part * np.exp2(-e.astype(np.float64))[:, :, None, None])
    q = decode(code) * np.exp2(e.astype(np.float64))[:, :, None, None]
    norm, kept = (part ** 2).sum(axis=(1, 2, 3)), (q ** 2).sum(axis=(1, 2, 3))
    with np.errstate(invalid="ignore", divide="ignore"):
        gains = np.where(kept == 0, 0.0, norm / kept)
    codes = code.reshape(N, 2 * blocks, 64, 2).transpose(0, 1, 3, 2)[:, :chunks].reshape(N, -1)
    scales = np.full((N, 4 * (-(-blocks // 4))), 127, dtype=np.uint8)
    scales[:, :blocks] = e + 127
    return np.ascontiguousarray(codes), scales, gains


def rows(codes, scales, D):
    """The rows q that a store holds, complex128 [N, D]."""
    N = codes.shape[0]
    q = decode(codes).reshape(N, -1, 2, 64)
    q = q * np.exp2(scales.astype(np.float64) - 127)[:, np.arange(q.shape[1]) // 2, None, None]
    return (q[:, :, 0] + 1j * q[:, :, 1]).reshape(N, -1)[:, :D]


def kernel(a, ga, b, gb):
    """(K, bound on its error in FP32 arithmetic, bound with the matrix unit's 8-bit products).

    FP32: re and im are sums of 2 D exact products whose partial sums stay below S = sum |a||b| in size; every one of the
    2 D roundings is off by at most U32 S, and they are independent: 8 standard deviations, 8 sqrt(2 D) U32 S.
    8-bit products: the matrix unit aligns 8 products to the largest of them and keeps 13 bits: a group of 8 is off by at
    most 8 * 2^-13 of its largest product, all groups together by 2^-10 S."""
    ov = np.conj(a) @ b.T
    S = np.abs(a) @ np.abs(b).T * np.sqrt(2)
    g = np.outer(ga, gb)
    K = g * np.abs(ov) ** 2
    D = a.shape[1]
    out = []
    for d in (8 * np.sqrt(2 * D) * U32 * S, 2.0 ** -10 * S):
        out.append(g * (2 * np.sqrt(2) * np.abs(ov) * d + 2 * d ** 2) + 8 * U32 * K + 1e-37)
    return K, out[0], out[1]


def states(rng, N, D, kind="spread"):
    """Normalised states: spread over all amplitudes, or products of rotated qubits (a wide range of sizes)."""
    if kind == "spread":
        psi = rng.normal(size=(N, D)) + 1j * rng.normal(size=(N, D))
    else:
        psi = np.ones((N, 1), dtype=np.complex128)
        while psi.shape[1] < D:
            t, p = rng.uniform(0, np.pi / 2, size=(N, 1)), rng.uniform(0, 2 * np.pi, size=(N, 1))
            psi = np.concatenate([np.cos(t) * psi, np.sin(t) * np.exp(1j * p) * psi], axis=1)
        psi = psi[:, :D]
    return psi / np.linalg.norm(psi, axis=1, keepdims=True)
