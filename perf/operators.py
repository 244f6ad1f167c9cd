"""The 8-bit operators of the quantum-kernel engine: their cases, their plain forms and their 64-bit values.

A kernel model keeps the statevectors of its training samples.  ``States8`` holds them in 8 bits: e4m3 codes with one
power-of-two scale for each block of 128 amplitudes, and one float per row that restores the row's norm.  On such stores
work the fidelity kernel of two sets of states (``gram8``), the kernels of a population of circuits of ragged sizes
(``gram8_jobs``) and the decision values of a kernel machine (``decision8``).

Layout of a row of D amplitudes: chunks of 64 amplitudes, each 64 real codes and then 64 imaginary ones (the last chunk
padded with zeros); scales: one exponent byte (value 2^(byte - 127)) per 128 amplitudes, rows padded to whole 4 bytes with 127.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 128          # amplitudes that share one scale
CHUNK = 64           # amplitudes whose codes lie together
LARGEST = 8.0 * 12000 * 12001 / 2 * 65536       # flops of the largest listed case


def listed():
    return [
        # a sample that has just been simulated joins the cache (10 qubits, one row): latency
        dict(name="write one row", op="write", rows=1, dim=1024, single=False),
        # the training states of a 16-qubit model as the simulator leaves them: the widest rows the benchmark has
        dict(name="write 16 qubits", op="write", rows=4096, dim=65536, single=False),
        # the states of the support vectors of a 12-qubit model, read back by their row numbers
        dict(name="read 12 qubits", op="read", rows=20001, of=40000, dim=4096, single=True),
        # the bundled cross-validation set through a 4-qubit circuit: 100 rows, what a search evaluates all day
        dict(name="gram 4 qubits", op="gram", rows=100, cols=0, dim=16, half=False),
        # 8 qubits, 4096 rows, train x train, K in half precision: what it writes is most of its traffic
        dict(name="gram 8 qubits", op="gram", rows=4096, cols=0, dim=256, half=True),
        # 16 qubits, train x train, K in half precision: the matrix product at its longest
        dict(name="gram 16 qubits", op="gram", rows=12000, cols=0, dim=65536, half=True),
        # one new sample against 65536 cached ones of 12 qubits: the kernel row of a served prediction
        dict(name="gram one row", op="gram", rows=1, cols=65536, dim=4096, half=False),
        # one generation of a search at the bundled data's size: 50 genomes of 4 to 10 qubits over 100 rows
        dict(name="population", op="group", groups=50, rows_lo=100, rows_hi=100, dim_lo=16, dim_hi=1024, sizes=1, half=False),
        # a population whose genomes bring their own rows: a few large kernels among small ones
        dict(name="population ragged", op="group", groups=12, rows_lo=33, rows_hi=4097, dim_lo=16, dim_hi=4096, sizes=2, half=False),
        # the answer for one sample from 8192 support vectors of 10 qubits: latency
        dict(name="decide one", op="decide", rows=1, cols=8192, dim=1024, outs=1),
        # 16384 test rows against 16384 cached rows of 10 qubits, two classes
        dict(name="decide batch", op="decide", rows=16384, cols=16384, dim=1024, outs=1),
        # odd sizes, ten classes one against one
        dict(name="decide classes", op="decide", rows=3001, cols=10007, dim=256, outs=45),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _dim(rng, lo=2, hi=65536):
    """Mostly whole registers, now and then the dimension of a subspace."""
    if rng.random() < 0.8:
        return 1 << rng.randint(int(math.log2(lo)), int(math.log2(hi)))
    return _log(rng, lo, hi)


def draw(rng: random.Random):
    op = rng.choice(["write", "read", "gram", "gram", "group", "decide", "decide"])
    if op == "write":
        dim = _dim(rng)
        return dict(op=op, rows=_log(rng, 1, min(1 << 20, (1 << 27) // dim)), dim=dim, single=rng.random() < 0.5)
    if op == "read":
        dim = _dim(rng)
        of = _log(rng, 1, min(1 << 20, (1 << 27) // dim))
        return dict(op=op, rows=_log(rng, 1, of), of=of, dim=dim, single=rng.random() < 0.5)
    if op == "group":
        lo = _log(rng, 1, 300)
        return dict(op=op, groups=rng.randint(2, 60), rows_lo=lo, rows_hi=_log(rng, lo, 2000), dim_lo=4,
                    dim_hi=1 << rng.randint(3, 11), sizes=rng.randint(0, 1 << 20), half=rng.random() < 0.4)
    dim = _dim(rng)
    most = 1 << 28                                  # amplitudes of one side, and entries of the kernel matrix
    cols = _log(rng, 1, min(65536, most // dim))
    if op == "gram" and rng.random() < 0.4:
        rows, cols = min(cols, 16384), 0
    else:
        rows = _log(rng, 1, min(16384, most // dim, most // cols))
    case = dict(op=op, rows=rows, cols=cols, dim=dim)
    if op == "decide":
        case["outs"] = rng.choice([1, 1, 1, 2, 3, 10, 45, 64])
    else:
        case["half"] = rng.random() < 0.5
    return case


def sizes(case):
    """(rows, dim) of every genome of a population."""
    r = random.Random(case["sizes"])
    got = []
    for _ in range(case["groups"]):
        dim = 1 << r.randint(int(math.log2(case["dim_lo"])), int(math.log2(case["dim_hi"])))
        got.append((_log(r, case["rows_lo"], case["rows_hi"]), dim))
    return got


def _row_bytes(dim):
    return 2 * CHUNK * -(-dim // CHUNK) + -(-dim // BLOCK) + 4


def work(case):
    op, dim = case["op"], case.get("dim", 0)
    if op in ("write", "read"):
        plain = case["rows"] * dim * (8 if case["single"] else 16)
        return {"bytes": plain + case["rows"] * (_row_bytes(dim) + (8 if op == "read" else 0)), "flops": 8.0 * case["rows"] * dim}
    entry = 2 if case.get("half") else 4
    if op == "group":
        return {"bytes": float(sum(n * _row_bytes(d) + entry * n * n for n, d in sizes(case))),
                "flops": float(sum(8 * d * n * (n + 1) // 2 for n, d in sizes(case)))}
    m, n = case["rows"], case["cols"]
    if op == "gram" and n == 0:
        return {"bytes": float(m * _row_bytes(dim) + entry * m * m), "flops": 8.0 * dim * m * (m + 1) / 2}
    bytes_ = (m + n) * _row_bytes(dim)
    if op == "gram":
        return {"bytes": float(bytes_ + entry * m * n), "flops": 8.0 * dim * m * n}
    c = case["outs"]
    return {"bytes": float(bytes_ + 4 * (n * c + c + m * c)), "flops": 8.0 * dim * m * n + 2.0 * m * n * c}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _states(gen, rows, dim, dtype):
    """Encoded samples as a feature map makes them: product states of rotated qubits with their phases, then a quadratic
    phase; a dimension that is no power of two keeps that many amplitudes.  Normalised to rounding."""
    n = max(1, math.ceil(math.log2(dim)))
    real = torch.float64 if dtype == torch.complex128 else torch.float32
    out = torch.empty((rows, dim), dtype=dtype, device=DEV)
    step = max(1, (1 << 27) >> n)
    for a in range(0, rows, step):
        r = min(step, rows - a)
        x = torch.rand((r, n), generator=gen, device=DEV, dtype=real) * (math.pi - 2e-5) - math.pi / 2 + 1e-5
        phase = torch.rand((r, n), generator=gen, device=DEV, dtype=real) * (2 * math.pi)
        psi = torch.ones((r, 1), dtype=dtype, device=DEV)
        for q in range(n):
            one = torch.polar(torch.sin(x[:, q] / 2 + math.pi / 4), phase[:, q]).unsqueeze(1)
            zero = torch.cos(x[:, q] / 2 + math.pi / 4).to(dtype).unsqueeze(1)
            psi = torch.cat([psi * zero, psi * one], dim=1)
        psi = psi[:, :dim]
        out[a:a + r] = psi / psi.abs().square().sum(dim=1, keepdim=True).sqrt()
    return out


def _store(gen, rows, dim):
    """(codes, scales, gains) of `rows` random states, in the layout at the top of this file."""
    codes, scales, gains = [], [], []
    step = max(1, (1 << 26) // dim)
    for a in range(0, rows, step):
        c, s, g = _quantise(_states(gen, min(step, rows - a), dim, torch.complex64))
        codes.append(c), scales.append(s), gains.append(g)
    return torch.cat(codes), torch.cat(scales), torch.cat(gains)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 7919 + 17)
    op, dim = case["op"], case.get("dim", 0)
    if op == "write":
        psi = _states(gen, case["rows"], dim, torch.complex64 if case["single"] else torch.complex128)
        return dict(case=case, psi=psi)
    if op == "read":
        codes, scales, gains = _store(gen, case["of"], dim)
        index = torch.randint(0, case["of"], (case["rows"],), generator=gen, device=DEV)
        return dict(case=case, codes=codes, scales=scales, gains=gains, index=index)
    if op == "group":
        return dict(case=case, stores=[(*_store(gen, n, d), d) for n, d in sizes(case)])
    state = dict(case=case, x=_store(gen, case["rows"], dim), y=_store(gen, case["cols"], dim) if case["cols"] else None)
    if op == "decide":
        # dual coefficients: signed, most of them small, as a soft-margin fit leaves them
        coef = torch.randn((case["cols"], case["outs"]), generator=gen, device=DEV)
        state["coef"] = coef * coef.abs()
        state["intercept"] = torch.randn((case["outs"],), generator=gen, device=DEV)
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _e4m3(v):
    """Nearest e4m3 value of |v| <= 448, ties to even: the grid's step around v is 2^(floor(log2 |v|) - 3), at least 2^-9."""
    shift = 4 - torch.clamp(torch.frexp(v).exponent, min=-5)
    return torch.ldexp(torch.round(torch.ldexp(v, shift)), -shift)


def _quantise(psi):
    rows, dim = psi.shape
    chunks, blocks = -(-dim // CHUNK), -(-dim // BLOCK)
    parts = torch.view_as_real(psi)
    parts = torch.nn.functional.pad(parts, (0, 0, 0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK, 2)
    most = parts.abs().amax(dim=(2, 3))
    m, x = torch.frexp(most)
    e = torch.where(most > 0, torch.clamp(x - torch.where(m <= 0.875, 9, 8), -127, 127), 0)
    q = _e4m3(torch.ldexp(parts, -e[:, :, None, None]))
    value = torch.ldexp(q, e[:, :, None, None])
    norm = parts.double().square().sum(dim=(1, 2, 3))
    kept = value.double().square().sum(dim=(1, 2, 3))
    gains = torch.where(kept > 0, norm / kept, torch.zeros_like(norm)).float()
    codes = q.view(rows, 2 * blocks, CHUNK, 2).transpose(2, 3)[:, :chunks].float().to(torch.float8_e4m3fn)
    scales = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device=psi.device)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return codes.reshape(rows, chunks * 2 * CHUNK).view(torch.uint8), scales, gains


def _parts(codes, scales, dim):
    """Real and imaginary parts in float32, without the padding."""
    rows, chunks = codes.shape[0], -(-dim // CHUNK)
    q = codes.view(torch.float8_e4m3fn).float().view(rows, chunks, 2, CHUNK)
    e = (scales.int() - 127).repeat_interleave(2, dim=1)[:, :chunks]
    q = torch.ldexp(q, e[:, :, None, None])
    return q[:, :, 0].reshape(rows, -1)[:, :dim], q[:, :, 1].reshape(rows, -1)[:, :dim]


def _kernel(x, y, dim, dtype=torch.float32):
    """K = gain gain |<x|y>|^2; y is None: the rows with themselves, with a unit diagonal."""
    ar, ai = _parts(x[0], x[1], dim)
    br, bi = (ar, ai) if y is None else _parts(y[0], y[1], dim)
    re = ar @ br.T + ai @ bi.T
    im = ar @ bi.T - ai @ br.T
    K = (re.square() + im.square()) * x[2][:, None] * (x if y is None else y)[2][None, :]
    if y is None:
        K.fill_diagonal_(1.0)
    return K.to(dtype)


def run(state):
    case = state["case"]
    op, dim = case["op"], case.get("dim", 0)
    dtype = torch.float16 if case.get("half") else torch.float32          # of K
    if own:
        from quake_amd import device as qdev
        if op == "write":
            store = qdev.States8(case["rows"], dim)
            store.write(state["psi"])
            return dict(codes=store.codes.view(torch.float8_e4m3fn), scales=store.scales, gains=store.gains)
        if op == "read":
            store = qdev.States8.from_arrays(state["codes"], state["scales"], state["gains"], dim)
            return store.read(state["index"], dtype=torch.complex64 if case["single"] else torch.complex128)
        if op == "group":
            stores = [qdev.States8.from_arrays(*s) for s in state["stores"]]
            return qdev.gram8_jobs([dict(A=s) for s in stores], dtype=dtype)
        x = qdev.States8.from_arrays(*state["x"], dim)
        y = qdev.States8.from_arrays(*state["y"], dim) if state["y"] else None
        if op == "gram":
            return qdev.gram8(x, y, dtype=dtype)
        return qdev.decision8(x, y, state["coef"], state["intercept"])
    if op == "write":
        codes, scales, gains = _quantise(state["psi"])
        return dict(codes=codes.view(torch.float8_e4m3fn), scales=scales, gains=gains)
    if op == "read":
        re, im = _parts(state["codes"][state["index"]], state["scales"][state["index"]], dim)
        return torch.complex(re, im) if case["single"] else torch.complex(re.double(), im.double())
    if op == "group":
        return [_kernel((c, s, g), None, d, dtype) for c, s, g, d in state["stores"]]
    K = _kernel(state["x"], state["y"], dim, dtype)
    return K if op == "gram" else K @ state["coef"] + state["intercept"]


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _grid():
    """The 127 finite e4m3 values >= 0 in order, from the format: 4 exponent bits of bias 7, 3 fraction bits."""
    vals = [f / 8 * 2.0 ** -6 for f in range(8)]
    vals += [(1 + f / 8) * 2.0 ** (e - 7) for e in range(1, 16) for f in range(8)]
    return torch.tensor(vals[:127], dtype=torch.float64, device=DEV)


def _exact_write(psi):
    rows, dim = psi.shape
    grid = _grid()
    half = (grid[1:] + grid[:-1]) / 2
    chunks, blocks = -(-dim // CHUNK), -(-dim // BLOCK)
    codes = torch.zeros((rows, chunks, 2, CHUNK), dtype=torch.float64, device=DEV)
    scales = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device=DEV)
    norm = torch.zeros(rows, dtype=torch.float64, device=DEV)
    kept = torch.zeros(rows, dtype=torch.float64, device=DEV)
    for b in range(blocks):
        for k, plane in enumerate((psi.real, psi.imag)):
            v = plane[:, b * BLOCK:(b + 1) * BLOCK].double()
            if k == 0:
                top = torch.maximum(v.abs().amax(1), psi.imag[:, b * BLOCK:(b + 1) * BLOCK].double().abs().amax(1))
                e = torch.ceil(torch.log2(top / 448.0))          # the least e with top <= 448 * 2^e
                e = torch.where(top > torch.exp2(e) * 448.0, e + 1, e)
                e = torch.where(top <= torch.exp2(e - 1) * 448.0, e - 1, e)
                e = torch.where(top > 0, torch.clamp(e, -127, 127), torch.zeros_like(e))
                scales[:, b] = (e + 127).to(torch.uint8)
                unit = torch.exp2(e)[:, None]
            w = v / unit
            i = torch.bucketize(w.abs(), half)
            tie = (i < 126) & (w.abs() == half[torch.clamp(i, max=125)]) & (i % 2 == 1)
            q = grid[i + tie.long()] * torch.sign(w)
            norm += v.square().sum(1)
            kept += (q * unit).square().sum(1)
            for c in range(2):
                piece = q[:, c * CHUNK:(c + 1) * CHUNK]
                if piece.shape[1]:
                    codes[:, 2 * b + c, k, :piece.shape[1]] = piece
    gains = torch.where(kept > 0, norm / kept, torch.zeros_like(norm))
    return codes.view(rows, -1), scales, gains


def _wide(codes, scales, dim):
    """The rows that a store stands for, complex128."""
    byte = codes.long()
    mag, low = (byte >> 3) & 15, byte & 7
    val = torch.where(mag > 0, (8 + low).double() * torch.exp2((mag - 10).double()), low.double() * 2.0 ** -9)
    val = torch.where(byte >= 128, -val, val).view(codes.shape[0], -1, 2, CHUNK)
    unit = torch.exp2(scales.double() - 127)
    at = torch.arange(val.shape[1], device=DEV) // 2
    val = val * unit[:, at][:, :, None, None]
    return torch.complex(val[:, :, 0].reshape(codes.shape[0], -1), val[:, :, 1].reshape(codes.shape[0], -1))[:, :dim].contiguous()


def _exact_kernel(x, y, dim):
    a = _wide(x[0], x[1], dim)
    b = a if y is None else _wide(y[0], y[1], dim)
    K = torch.matmul(a, b.conj().resolve_conj().transpose(0, 1).contiguous()).abs().square()
    K = K * torch.outer(x[2].double(), (x if y is None else y)[2].double())
    if y is None:
        K.fill_diagonal_(1.0)
    return K


def exact(case, seed):
    op, dim = case["op"], case.get("dim", 0)
    if work(case)["flops"] > 0.2 * LARGEST:
        return None                                    # 64-bit products of that size take too long
    state = prepare(case, seed)
    if op == "write":
        codes, scales, gains = _exact_write(state["psi"])
        return dict(codes=codes, scales=scales, gains=gains)
    if op == "read":
        return _wide(state["codes"][state["index"]], state["scales"][state["index"]], dim)
    if op == "group":
        return [_exact_kernel((c, s, g), None, d) for c, s, g, d in state["stores"]]
    K = _exact_kernel(state["x"], state["y"], dim)
    return K if op == "gram" else torch.matmul(K, state["coef"].double()) + state["intercept"].double()
