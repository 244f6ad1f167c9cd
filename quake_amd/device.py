"""Device-resident entry points: torch tensors in HBM in, torch tensors out.

torch is plumbing here (device memory, the current HIP stream, torch.distributed);
every kernel is launched through the ``*_dev`` functions of libquake_hip.so on
torch's current stream.  Used by ``bench.py`` and :mod:`quake_amd.sharded`.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import List, Optional, Sequence

import torch

from . import _lib
from .circuit import QuantumCircuit


def _stream_ptr() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dp(t: Optional[torch.Tensor]) -> Optional[C.c_void_p]:
    return None if t is None else C.c_void_p(t.data_ptr())


def from_dlpack(x) -> Optional[torch.Tensor]:
    """DLPack hand-off at the device boundary ("DLPack/numpy hand-off"): anything that
    implements ``__dlpack__`` (a cupy / jax / numba array, another framework's tensor) or a raw DLPack capsule is
    viewed -- zero copy -- as the torch tensor the launchers work on; torch tensors pass through.  Every tensor
    this module returns implements ``__dlpack__`` itself, so results travel back the same way
    (``consumer.from_dlpack(K)``)."""
    if x is None or isinstance(x, torch.Tensor):
        return x
    if hasattr(x, "__dlpack__"):
        return torch.from_dlpack(x)
    if type(x).__name__ == "PyCapsule":
        return torch.utils.dlpack.from_dlpack(x)
    raise TypeError(f"expected a torch tensor, an object with __dlpack__ or a DLPack capsule, got {type(x).__name__}")


def to_dlpack(t: torch.Tensor):
    """A DLPack capsule of a result tensor (for consumers that take capsules rather than ``__dlpack__`` objects)."""
    return torch.utils.dlpack.to_dlpack(t)


def _require_gpu(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("device entry points need tensors in GPU memory")


class DeviceCircuit:
    """A feature map compiled once and kept as a ``qk_circuit`` handle."""

    def __init__(self, feature_map: QuantumCircuit):
        self.feature_map = feature_map
        self.compiled = feature_map.compile()
        self.handle = _lib.CircuitHandle(self.compiled)
        self.n_qubits = self.compiled.n_qubits
        self.n_params = self.compiled.n_params
        self.dim = 1 << self.n_qubits

    def simulate(self, X: torch.Tensor, out: Optional[torch.Tensor] = None, dtype=torch.complex128) -> torch.Tensor:
        """X float64 [N, n_params] (row stride free) -> Psi [N, 2^n], complex128 or (FP32 mode:
        evolved in FP64, rounded at the store) complex64 -- the dtype of ``out`` if given."""
        X, out = from_dlpack(X), from_dlpack(out)
        _require_gpu(X, out)
        if X.dtype != torch.float64 or X.dim() != 2 or X.stride(1) != 1:
            raise ValueError("X must be a float64 [N, F] tensor with unit column stride")
        if X.shape[1] != self.n_params:
            raise ValueError(
                f"x_vec and class feature map have incompatible dimensions.\n"
                f"x_vec has {X.shape[1]} dimensions, but feature map has {self.n_params}.")
        N = X.shape[0]
        if out is None:
            out = torch.empty((N, self.dim), dtype=dtype, device=X.device)
        elif out.dtype not in (torch.complex128, torch.complex64) or tuple(out.shape) != (N, self.dim) \
                or not out.is_contiguous():
            raise ValueError("out must be a contiguous complex128 / complex64 [N, 2^n] tensor")
        ldx = X.stride(0) if N > 1 else max(self.n_params, 1)
        lib = _lib.load()
        if out.dtype == torch.complex128:
            _lib.check(lib.qk_simulate_dev(self.handle.handle, _dp(X), N, ldx, _dp(out), _stream_ptr()))
        else:
            ws = None
            if self.handle.num_passes > 1:     # earlier passes go through a complex128 workspace
                ws = torch.empty((N, self.dim), dtype=torch.complex128, device=X.device)
            _lib.check(lib.qk_simulate_c64_dev(self.handle.handle, _dp(X), N, ldx, _dp(out), _dp(ws), _stream_ptr()))
        return out


def simulate_rdm1(circuit: "DeviceCircuit", X: torch.Tensor) -> torch.Tensor:
    """Per-qubit reduced density matrices of the encoded states, float64 [N, n, 4], without writing
    the statevectors when the circuit fits one LDS-resident pass (``qk_simulate_rdm1_dev``)."""
    X = from_dlpack(X)
    _require_gpu(X)
    lib = _lib.load()
    if X.dtype != torch.float64 or X.dim() != 2 or X.shape[1] != circuit.n_params or (X.numel() and X.stride(1) != 1):
        raise ValueError("X must be float64 [N, n_params] with unit column stride")
    N, n = X.shape[0], circuit.n_qubits
    out = torch.empty((N, n, 4), dtype=torch.float64, device=X.device)
    ws = None
    if lib.qk_simulate_rdm1_wants_workspace(circuit.handle.handle, N):      # not fused, or the two-step route is the faster one
        ws = torch.empty((N, 1 << n), dtype=torch.complex128, device=X.device)
    ldx = X.stride(0) if (N > 1 and X.shape[1]) else max(X.shape[1], 1)
    _lib.check(lib.qk_simulate_rdm1_dev(circuit.handle.handle, _dp(X) if X.numel() else None, N, ldx, _dp(out), _dp(ws),
                                        _stream_ptr()))
    return out


def gram_jobs(jobs: Sequence[dict], D: int) -> None:
    """Run several block jobs in one launch.  Each job: dict(A=, B=, K=, KT=None, symmetric=False);
    A, B complex128 (or, for the FP32 Gram stage, complex64) [rows, D] contiguous; K (and KT) float64
    2-D views with unit column stride."""
    jobs = [dict(j, A=from_dlpack(j["A"]), B=from_dlpack(j["B"]), K=from_dlpack(j["K"]), KT=from_dlpack(j.get("KT")))
            for j in jobs]
    arr = (_lib.qk_gram_job * len(jobs))()
    dtype = jobs[0]["A"].dtype if jobs else torch.complex128
    if dtype not in (torch.complex128, torch.complex64):
        raise ValueError("statevectors must be complex128 or complex64")
    for k, j in enumerate(jobs):
        A, B, K, KT = j["A"], j["B"], j["K"], j.get("KT")
        _require_gpu(A, B, K, KT)
        for t in (A, B):
            if t.dtype != dtype or t.dim() != 2 or t.shape[1] != D or not t.is_contiguous():
                raise ValueError("A and B must be contiguous [rows, D] of one complex dtype")
        if K.dtype != torch.float64 or K.stride(1) != 1 or tuple(K.shape) != (A.shape[0], B.shape[0]):
            raise ValueError("K must be float64 [rows(A), rows(B)] with unit column stride")
        if KT is not None and (KT.dtype != torch.float64 or KT.stride(1) != 1
                               or tuple(KT.shape) != (B.shape[0], A.shape[0])):
            raise ValueError("KT must be float64 [rows(B), rows(A)] with unit column stride")
        arr[k].A, arr[k].B = A.data_ptr(), B.data_ptr()
        arr[k].K = K.data_ptr()
        arr[k].KT = KT.data_ptr() if KT is not None else None
        arr[k].ma, arr[k].nb = A.shape[0], B.shape[0]
        arr[k].ldk = K.stride(0) if K.shape[0] > 1 else max(K.shape[1], 1)
        arr[k].ldkt = (KT.stride(0) if KT.shape[0] > 1 else max(KT.shape[1], 1)) if KT is not None else 0
        arr[k].flags = _lib.QK_GRAM_SYMMETRIC if j.get("symmetric") else 0
    fn = _lib.load().qk_gram_jobs_dev if dtype == torch.complex128 else _lib.load().qk_gram32_jobs_dev
    _lib.check(fn(arr, len(jobs), D, _stream_ptr()))


def gram(psi_x: torch.Tensor, psi_y: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """K = |Psi_x Psi_y^H|^2; ``psi_y is None`` -> symmetric block with exact unit diagonal."""
    psi_x, psi_y, out = from_dlpack(psi_x), from_dlpack(psi_y), from_dlpack(out)
    _require_gpu(psi_x, psi_y, out)
    N, D = psi_x.shape
    M = N if psi_y is None else psi_y.shape[0]
    if out is None:
        out = torch.empty((N, M), dtype=torch.float64, device=psi_x.device)
    gram_jobs([dict(A=psi_x, B=psi_x if psi_y is None else psi_y, K=out, symmetric=psi_y is None)], D)
    return out


def block_to_host(K_dev: torch.Tensor, K_host: torch.Tensor, stream: Optional["torch.cuda.Stream"] = None) -> None:
    """Enqueue the copy of a 2-D float64 device view (unit column stride) into a host view of the same
    shape (page-locked memory for a copy that overlaps other streams) on ``stream`` (default: torch's
    current stream): ``qk_block_to_host_async``, one strided copy, no temporaries."""
    _require_gpu(K_dev)
    if K_host.is_cuda or K_dev.dtype != torch.float64 or K_host.dtype != torch.float64:
        raise ValueError("block_to_host copies a float64 device view into a float64 host view")
    if K_dev.dim() != 2 or tuple(K_dev.shape) != tuple(K_host.shape):
        raise ValueError("device and host views must be 2-D and of one shape")
    rows, cols = K_dev.shape
    if rows == 0 or cols == 0:
        return
    if K_dev.stride(1) != 1 or K_host.stride(1) != 1:
        raise ValueError("both views need unit column stride")
    s = C.c_void_p((stream or torch.cuda.current_stream()).cuda_stream)
    _lib.check(_lib.load().qk_block_to_host_async(
        _dp(K_dev), K_dev.stride(0) if rows > 1 else cols, rows, cols,
        C.c_void_p(K_host.data_ptr()), K_host.stride(0) if rows > 1 else cols, s))


def rdm1(psi: torch.Tensor, n_qubits: int) -> torch.Tensor:
    """Per-qubit reduced density matrices, float64 [N, n, 4] = (rho00, rho11, Re rho01, Im rho01)."""
    psi = from_dlpack(psi)
    _require_gpu(psi)
    if psi.dtype != torch.complex128 or not psi.is_contiguous() or psi.shape[1] != (1 << n_qubits):
        raise ValueError("psi must be contiguous complex128 [N, 2^n]")
    out = torch.empty((psi.shape[0], n_qubits, 4), dtype=torch.float64, device=psi.device)
    _lib.check(_lib.load().qk_rdm1_dev(_dp(psi), psi.shape[0], n_qubits, _dp(out), _stream_ptr()))
    return out


def pqk(rdm_x: torch.Tensor, rdm_y: Optional[torch.Tensor], gamma: float,
        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Projected kernel block from RDM tables; ``rdm_y is None`` -> symmetric with unit diagonal."""
    rdm_x, rdm_y, out = from_dlpack(rdm_x), from_dlpack(rdm_y), from_dlpack(out)
    _require_gpu(rdm_x, rdm_y, out)
    N, n, _ = rdm_x.shape
    M = N if rdm_y is None else rdm_y.shape[0]
    if out is None:
        out = torch.empty((N, M), dtype=torch.float64, device=rdm_x.device)
    ldk = out.stride(0) if N > 1 else max(M, 1)
    _lib.check(_lib.load().qk_pqk_dev(_dp(rdm_x.contiguous()), N, _dp(rdm_y.contiguous()) if rdm_y is not None else None,
                                      M, n, float(gamma), _dp(out), ldk, _stream_ptr()))
    return out


# --------------------------------------------------------------------------- #
# 8-bit state stores
# --------------------------------------------------------------------------- #
_NO_GUARD = contextlib.nullcontext()


def _on(gpu: int):
    """Makes a GPU the current one for a launch (kernels run on that GPU's current stream)."""
    return _NO_GUARD if gpu == torch.cuda.current_device() else torch.cuda.device(gpu)


def _stream_on(gpu: int) -> int:
    return torch._C._cuda_getCurrentRawStream(gpu)


def _same_gpu(gpu: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != gpu:
            raise ValueError("device entry points need tensors in GPU memory, all on one GPU")


def _plain(*tensors) -> None:
    """The library reads and writes memory: a lazily negated or conjugated view holds other values there than it shows.  And
    nothing is recorded for autograd: an output without a graph would drop a gradient without a word."""
    for t in tensors:
        if t is None:
            continue
        if t.is_neg() or t.is_conj():
            raise ValueError("lazily negated or conjugated tensors are not taken: call resolve_neg() / resolve_conj() first")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("no gradient is recorded through 8-bit stores: detach() the tensor or call under torch.no_grad() "
                             "(the gradient of decision8 by coef is decision8(y, x, dloss/dout))")


class States8:
    """Statevectors kept in 8 bits: e4m3 codes, one power-of-two scale for each block of 128 amplitudes, and one float per row
    that restores the row's norm -- 2 bytes per amplitude instead of complex128's 16.  The training states of a kernel model:
    written once (``write`` appends), read by every prediction (:func:`gram8`, :func:`decision8`).

    ``codes`` uint8 [capacity, 128 * ceil(dim / 64)], ``scales`` uint8 [capacity, 4 * ceil(dim / 512)] and ``gains`` float32
    [capacity] are plain tensors (layout and formulas: ``qk_states8`` in quake_hip.h); ``len(store)`` rows are written.  A
    component is off by at most 2^-4 of itself (or, where that is more, 2^-17 of the largest in its block), the fidelity of two
    states by up to 0.13 in the worst case and by about 0.07 sqrt(K / dim) for states spread over their ``dim`` amplitudes."""

    def __init__(self, capacity: int, dim: int, device=None):
        code, scale = self._layout(dim)
        if capacity < 0:
            raise ValueError("capacity must not be negative")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("device entry points need tensors in GPU memory")
        self._set(torch.empty((capacity, code), dtype=torch.uint8, device=device),
                  torch.empty((capacity, scale), dtype=torch.uint8, device=device),
                  torch.empty((capacity,), dtype=torch.float32, device=device), dim, 0)

    @staticmethod
    def _layout(dim: int):
        if not 1 <= dim <= 1 << 26:
            raise ValueError("dim must be in 1..2^26")
        return 128 * (-(-dim // 64)), 4 * (-(-dim // 512))

    def _set(self, codes, scales, gains, dim, rows):
        self.codes, self.scales, self.gains, self.dim, self._rows = codes, scales, gains, dim, rows
        self._gpu = gpu = codes.get_device()
        if gpu < 0 or scales.get_device() != gpu or gains.get_device() != gpu:
            raise ValueError("device entry points need tensors in GPU memory, all on one GPU")

    @property
    def _at(self):      # at every call: a copy of a store (copy.deepcopy, pickle) has arrays of its own
        return self.codes.data_ptr(), self.scales.data_ptr(), self.gains.data_ptr()

    def __setstate__(self, state) -> None:
        self._set(state["codes"], state["scales"], state["gains"], state["dim"], state["_rows"])

    @classmethod
    def from_arrays(cls, codes: torch.Tensor, scales: torch.Tensor, gains: torch.Tensor, dim: int) -> "States8":
        """A store over arrays that hold written rows already (a saved store, a selection ``codes[rows], scales[rows],
        gains[rows]`` of another one's); the arrays are used, not copied."""
        code, scale = cls._layout(dim)
        rows = gains.numel()
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or gains.dtype is not torch.float32 \
                or gains.dim() != 1 or codes.shape != (rows, code) or scales.shape != (rows, scale) \
                or not (codes.is_contiguous() and scales.is_contiguous() and gains.is_contiguous()):
            raise ValueError("need contiguous codes uint8 [rows, 128 ceil(dim / 64)], scales uint8 [rows, 4 ceil(dim / 512)], "
                             "gains float32 [rows]")
        _plain(gains)
        store = cls.__new__(cls)
        store._set(codes, scales, gains, dim, rows)
        return store

    def __len__(self) -> int:
        return self._rows

    @property
    def capacity(self) -> int:
        return self.gains.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def rows(self, start: int, stop: int) -> "States8":
        """The written rows start .. stop - 1 as a store of their own (a view: nothing is copied)."""
        if not 0 <= start <= stop <= self._rows:
            raise ValueError(f"rows {start}..{stop} of a store that holds {self._rows}")
        store = States8.__new__(States8)
        store._set(self.codes[start:stop], self.scales[start:stop], self.gains[start:stop], self.dim, stop - start)
        return store

    def clear(self) -> None:
        """Forgets the written rows; the memory stays."""
        self._rows = 0

    def _struct(self, start: int = 0, rows: Optional[int] = None) -> "_lib.qk_states8":
        codes, scales, gains = self._at
        if start:
            codes, scales, gains = codes + start * self.codes.shape[1], scales + start * self.scales.shape[1], gains + 4 * start
        return _lib.qk_states8(codes, scales, gains, self._rows if rows is None else rows)

    def write(self, psi: torch.Tensor, at: Optional[int] = None) -> None:
        """Quantises psi [rows, dim] (complex128 or complex64, unit column stride) behind the rows written so far, or from row
        ``at`` on (overwriting; ``at`` may be at most the number of rows written so far)."""
        psi = from_dlpack(psi)
        _same_gpu(self._gpu, psi)
        if psi.dtype not in (torch.complex128, torch.complex64) or psi.dim() != 2 or psi.shape[1] != self.dim \
                or (psi.shape[0] and self.dim > 1 and psi.stride(1) != 1):
            raise ValueError("psi must be a complex128 / complex64 [rows, dim] tensor with unit column stride")
        _plain(psi)
        n, at = psi.shape[0], self._rows if at is None else at
        if not 0 <= at <= self._rows:
            raise ValueError(f"at = {at}: the store holds {self._rows} rows")
        if at + n > self.capacity:
            raise ValueError(f"{n} rows from row {at} on do not fit a capacity of {self.capacity}")
        ld = psi.stride(0) if n > 1 else self.dim
        if ld < self.dim:
            raise ValueError("the rows of psi overlap")
        to = self._struct(at, n)
        with _on(self._gpu):
            _lib.check(_lib.load().qk_states8_write_dev(_dp(psi), int(psi.dtype == torch.complex64), ld, self.dim, C.byref(to),
                                                        _stream_on(self._gpu)))
        self._rows = max(self._rows, at + n)

    def read(self, index: Optional[torch.Tensor] = None, dtype=torch.complex64, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The stored states q (code * scale, exact in complex64; the gain is not applied): all written rows, or the rows
        ``index`` (int64 on the GPU, any order, repeats allowed; a number outside the store gives a row of NaN)."""
        index, out = from_dlpack(index), from_dlpack(out)
        _same_gpu(self._gpu, index, out)
        _plain(index, out)
        if index is not None and (index.dtype != torch.int64 or index.dim() != 1 or not index.is_contiguous()):
            raise ValueError("index must be a contiguous int64 vector")
        n = self._rows if index is None else index.shape[0]
        if out is None:
            if dtype not in (torch.complex64, torch.complex128):
                raise ValueError("dtype must be complex64 or complex128")
            out = torch.empty((n, self.dim), dtype=dtype, device=self.device)
        elif out.dtype not in (torch.complex64, torch.complex128) or out.shape != (n, self.dim) or not out.is_contiguous():
            raise ValueError("out must be a contiguous complex64 / complex128 [rows, dim] tensor")
        of = self._struct()
        with _on(self._gpu):
            _lib.check(_lib.load().qk_states8_read_dev(C.byref(of), self.dim, _dp(index), n, _dp(out),
                                                       int(out.dtype == torch.complex64), self.dim, _stream_on(self._gpu)))
        return out


_K8_FLAGS = {torch.float32: 0, torch.float16: _lib.QK_GRAM8_F16, torch.float64: _lib.QK_GRAM8_F64}


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def gram8_jobs(jobs: Sequence[dict], dtype=torch.float32) -> List[torch.Tensor]:
    """Fidelity kernels of several pairs of 8-bit stores in one call (one launch for up to 24 of them), every job with its
    own rows and its own dim: the kernels of a population.  Each job: dict(A=, B=None, K=None, KT=None) with A, B
    :class:`States8`; B is None: the symmetric kernel of A with an exact unit diagonal.  K (allocated as ``dtype`` if not
    given, several of them in one allocation) and KT, the transposed copy (not for symmetric jobs): float32, float16 or
    float64 [len(A), len(B)] views with unit column stride, converted once from FP32 sums.  Returns the Ks."""
    if not jobs:
        return []
    if dtype not in _K8_FLAGS:
        raise ValueError("K must be float32, float16 or float64")
    several, pairs, gpu, entries = len(jobs) > 1, [], None, 0
    for j in jobs:
        A, B, K = j["A"], j.get("B"), j.get("K")
        sym = B is None
        if sym:
            B = A
        if not isinstance(A, States8) or not (sym or isinstance(B, States8)):
            raise ValueError("A and B must be States8 stores")
        if not sym and A.dim != B.dim:
            raise ValueError(f"stores of different dim: {A.dim} and {B.dim}")
        if gpu is None:
            gpu, device = A._gpu, A.codes.device
        if A._gpu != gpu or B._gpu != gpu:
            raise ValueError("stores on different GPUs")
        if K is None:
            entries += (A._rows * B._rows + 127) & ~127
        pairs.append((A, B, sym, K, j.get("KT")))
    flat, used = torch.empty(entries, dtype=dtype, device=device) if several and entries else None, 0
    packed, Ks = [], []
    for A, B, sym, K, KT in pairs:
        m, n = A._rows, B._rows
        if K is None:
            if flat is None:
                K = torch.empty((m, n), dtype=dtype, device=device)
            else:                       # views of one allocation, which lives as long as any of them
                K = flat.as_strided((m, n), (n or 1, 1), used)
                used += (m * n + 127) & ~127
            ldk = n or 1
        else:
            K = from_dlpack(K)
            if K.dtype not in _K8_FLAGS or K.shape != (m, n) or (K.numel() and ((n > 1 and K.stride(1) != 1) or (m > 1 and K.stride(0) < n))):
                raise ValueError("K must be float32, float16 or float64 [len(A), len(B)] with unit column stride")
            _same_gpu(gpu, K)
            _plain(K)
            ldk = K.stride(0) if m > 1 and n else max(n, 1)
        kt = ldkt = 0
        if KT is not None:
            KT = from_dlpack(KT)
            if sym or KT.dtype != K.dtype or KT.shape != (n, m) \
                    or (KT.numel() and ((m > 1 and KT.stride(1) != 1) or (n > 1 and KT.stride(0) < m))):
                raise ValueError("KT must be of K's type, [len(B), len(A)] with unit column stride, and not for a symmetric job")
            _same_gpu(gpu, KT)
            _plain(KT)
            kt, ldkt = KT.data_ptr(), (KT.stride(0) if n > 1 and m else max(m, 1))
        at = A._at
        packed.append(_lib.GRAM8_JOB.pack(*at, m, *(at if sym else B._at), n, A.dim, K.data_ptr(), kt, ldk, ldkt,
                                          _K8_FLAGS[K.dtype] | (_lib.QK_GRAM_SYMMETRIC if sym else 0), 0))
        Ks.append(K)
    lib, arr = _lib.load(), b"".join(packed)
    need = C.c_size_t()
    _lib.check(lib.qk_gram8_workspace(arr, len(jobs), C.byref(need)))
    with _on(gpu):
        ws = _workspace(need.value, device)
        _lib.check(lib.qk_gram8_jobs_dev(arr, len(jobs), _dp(ws), need.value, _stream_on(gpu)))
    return Ks


def gram8(x: States8, y: Optional[States8] = None, out: Optional[torch.Tensor] = None, dtype=torch.float32) -> torch.Tensor:
    """K = gain gain |<x|y>|^2 of two 8-bit stores; ``y is None`` -> the symmetric kernel of x with an exact unit diagonal.
    ``dtype`` (or the type of ``out``): float32, float16 or float64.  From one row (a kernel row for one sample) up."""
    return gram8_jobs([dict(A=x, B=y, K=out)], dtype)[0]


def decision8(x: States8, y: States8, coef: torch.Tensor, intercept: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What a kernel machine answers, out[m, c] = sum_j K(x_m, y_j) coef[j, c] + intercept[c], float32 [len(x), C], without K
    in memory (a small K for up to 32 rows of x against up to 4096 of y with more than 4096 amplitudes): ``SVC.decision_function`` on a precomputed kernel (``coef = dual_coef_.T``, y the support vectors), kernel
    ridge predictions, or K times a vector inside an iterative solver.  coef: float32 [len(y), C] (or [len(y)] for C = 1) with
    unit column stride, C up to 64.  Nothing is recorded for autograd (a tensor that requires a gradient is refused): the gradient of
    a loss by coef is ``decision8(y, x, dloss/dout)``, the one by the intercept the sum over dloss/dout's rows."""
    coef, intercept, out = from_dlpack(coef), from_dlpack(intercept), from_dlpack(out)
    if not isinstance(x, States8) or not isinstance(y, States8):
        raise ValueError("x and y must be States8 stores")
    _same_gpu(x._gpu, y.codes, coef, intercept, out)
    _plain(coef, intercept, out)
    if x.dim != y.dim:
        raise ValueError(f"stores of different dim: {x.dim} and {y.dim}")
    if coef.dim() == 1:
        coef = coef.unsqueeze(1)
    m, n, c = x._rows, y._rows, coef.shape[1] if coef.dim() == 2 else 0
    if coef.dtype != torch.float32 or coef.shape != (n, c) or not 1 <= c <= _lib.QK_DECISION8_MAX_C or (n and c > 1 and coef.stride(1) != 1):
        raise ValueError("coef must be float32 [len(y), C] with unit column stride and 1 <= C <= 64")
    if intercept is not None and (intercept.dtype != torch.float32 or intercept.shape != (c,) or not intercept.is_contiguous()):
        raise ValueError("intercept must be a contiguous float32 vector of C entries")
    if out is None:
        out = torch.empty((m, c), dtype=torch.float32, device=x.device)
    elif out.dtype != torch.float32 or out.shape != (m, c) or (m and c > 1 and out.stride(1) != 1):
        raise ValueError("out must be float32 [len(x), C] with unit column stride")
    ldc, ldo = (coef.stride(0) if n > 1 else c), (out.stride(0) if m > 1 else c)
    if ldc < c or ldo < c:
        raise ValueError("the rows of coef or out overlap")
    lib = _lib.load()
    need = C.c_size_t()
    _lib.check(lib.qk_decision8_workspace(m, n, x.dim, c, C.byref(need)))
    sx, sy = x._struct(), y._struct()
    with _on(x._gpu):
        ws = _workspace(need.value, x.device)
        _lib.check(lib.qk_decision8_dev(C.byref(sx), C.byref(sy), x.dim, _dp(coef), ldc, c, _dp(intercept), _dp(out), ldo, _dp(ws),
                                        need.value, _stream_on(x._gpu)))
    return out


def kernel_stats(K: torch.Tensor, labels: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Raw sums of the GA's kernel statistics over the strict upper triangle of a symmetric device
    K (see ``qk_kernel_stats_dev``): float64 [8] on the device."""
    K, labels = from_dlpack(K), from_dlpack(labels)
    _require_gpu(K, labels)
    if K.dtype != torch.float64 or K.dim() != 2 or K.shape[0] != K.shape[1] or K.stride(1) != 1:
        raise ValueError("K must be a square float64 matrix with unit column stride")
    if labels is not None:
        labels = labels.to(device=K.device, dtype=torch.int32).contiguous()
        if labels.numel() != K.shape[0]:
            raise ValueError("labels must have one entry per row of K")
    out = torch.empty(_lib.STATS_LEN, dtype=torch.float64, device=K.device)
    ws = torch.empty(_lib.STATS_WS, dtype=torch.float64, device=K.device)
    N = K.shape[0]
    _lib.check(_lib.load().qk_kernel_stats_dev(_dp(K), N, K.stride(0) if N > 1 else N, _dp(labels), _dp(out), _dp(ws),
                                               _stream_ptr()))
    return out


def kernel_noise_(K: torch.Tensor, mode: str, param: float, seed: int = 0, symmetric: bool = True) -> torch.Tensor:
    """In-place noise on a device K: ``mode`` = "gaussian" (param = std, reference genetic_v3.py:620-627) or "shots"
    (param = shots, the QPU-style P(0...0) estimate).  ``symmetric`` (a square train kernel): the entries right of
    the diagonal are drawn and mirrored, the diagonal stays exact; otherwise (a test-versus-train block of any
    shape) every entry is drawn."""
    K = from_dlpack(K)
    _require_gpu(K)
    if K.dtype != torch.float64 or K.dim() != 2 or K.stride(1) != 1 or K.shape[0] < 1 or K.shape[1] < 1:
        raise ValueError("K must be a float64 matrix with unit column stride")
    if symmetric and K.shape[0] != K.shape[1]:
        raise ValueError("a symmetric K must be square")
    code = {"gaussian": _lib.NOISE_GAUSSIAN, "shots": _lib.NOISE_SHOTS}[mode]
    rows, cols = K.shape
    ldk = K.stride(0) if rows > 1 else cols
    if symmetric:
        _lib.check(_lib.load().qk_kernel_noise_dev(_dp(K), rows, ldk, code, float(param), int(seed) & (2**64 - 1),
                                                   _stream_ptr()))
    else:
        _lib.check(_lib.load().qk_kernel_noise_rect_dev(_dp(K), rows, cols, ldk, code, float(param),
                                                        int(seed) & (2**64 - 1), _stream_ptr()))
    return K
