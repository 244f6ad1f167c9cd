"""8-bit stores and served models as Python objects, on a machine without a GPU: what reaches the library, and what is refused
before it.  Tensors in host memory pass for GPU tensors here, and a recorder stands in for the library."""
import contextlib
import copy
import ctypes as C
import io
import pickle

import numpy as np
import pytest
import torch

from quake_amd import _lib, device as qdev


class Recorder:
    """Takes the entry points' calls, runs nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def host(monkeypatch):
    """Host tensors pass for tensors on GPU 0."""
    lib = Recorder()
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(qdev, "_on", lambda gpu: contextlib.nullcontext())
    monkeypatch.setattr(qdev, "_stream_on", lambda gpu: 0)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    return lib


def store(rows=5, dim=100):
    code, scale = 128 * -(-dim // 64), 4 * -(-dim // 512)
    return qdev.States8.from_arrays(torch.zeros((rows, code), dtype=torch.uint8), torch.full((rows, scale), 127, dtype=torch.uint8),
                                    torch.ones(rows), dim)


def addresses(s):
    return s.codes.data_ptr(), s.scales.data_ptr(), s.gains.data_ptr()


def saved(s):
    f = io.BytesIO()
    torch.save(s, f)
    f.seek(0)
    return torch.load(f, weights_only=False)          # (a file that this test wrote itself)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda s: pickle.loads(pickle.dumps(s)), saved],
                         ids=["copy", "deepcopy", "pickle", "torch.save"])
def test_copies_bring_their_own_addresses(host, again):
    first = store()
    t = again(first)
    assert len(t) == 5 and t.dim == 100 and t.capacity == 5 and torch.equal(t.codes, first.codes)
    if again is not copy.copy:
        assert not set(addresses(t)) & set(addresses(first))
    s = t._struct(2, 1)
    assert (s.codes, s.scales, s.gains) == (t.codes[2].data_ptr(), t.scales[2].data_ptr(), t.gains[2:].data_ptr()) and s.rows == 1
    qdev.gram8(t, out=torch.zeros((5, 5)))
    name, args = host.calls[-1]
    assert name == "qk_gram8_jobs_dev" and _lib.GRAM8_JOB.unpack(args[0])[:3] == addresses(t)


def test_arrays_that_moved_are_found(host):
    s = store()
    s.gains = s.gains.clone()
    s.codes.data = s.codes.data.clone()
    at = s._struct()
    assert (at.codes, at.scales, at.gains) == addresses(s)


def test_a_copy_in_host_memory_is_refused(host, monkeypatch):
    raw = pickle.dumps(store())
    monkeypatch.undo()                                # host tensors are host tensors again
    with pytest.raises(ValueError, match="GPU memory"):
        pickle.loads(raw)


def test_views_whose_values_are_not_in_memory_are_refused(host):
    """A lazily negated or conjugated tensor: its memory holds other values than it shows."""
    x, y = store(4), store(5)
    full = lambda *s, **k: torch.zeros(s, **k)
    z = torch.zeros((5, 1), dtype=torch.complex64).conj()
    assert z.imag.is_neg()
    neg = torch._neg_view
    psi, out = full(2, 100, dtype=torch.complex64), full(5, 100, dtype=torch.complex64)
    coef, b = full(5, 1), full(1)
    index = torch.zeros(5, dtype=torch.int64)
    calls = [lambda: qdev.decision8(x, y, z.imag), lambda: qdev.decision8(x, y, z.imag[:, 0]), lambda: qdev.decision8(x, y, neg(coef)),
             lambda: qdev.decision8(x, y, coef, neg(b)), lambda: qdev.decision8(x, y, coef, b, out=neg(full(4, 1))),
             lambda: x.write(psi.conj(), at=0), lambda: x.write(neg(psi), at=0), lambda: y.read(out=out.conj()), lambda: y.read(out=neg(out)),
             lambda: y.read(neg(index)), lambda: qdev.gram8(x, y, out=neg(full(4, 5))),
             lambda: qdev.gram8_jobs([dict(A=x, B=y, KT=neg(full(5, 4)))]),
             lambda: qdev.States8.from_arrays(y.codes, y.scales, neg(y.gains), 100)]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError, match="conjugated"):
            call()
            pytest.fail(f"case {k} was taken")
    assert not host.calls
    qdev.decision8(x, y, z.imag.resolve_neg(), b, out=full(4, 1)), x.write(psi.conj().resolve_conj(), at=0), y.read(index, out=out)
    assert [name for name, _ in host.calls if name.endswith("dev")] == ["qk_decision8_dev", "qk_states8_write_dev", "qk_states8_read_dev"]


def test_tensors_that_want_a_gradient_are_refused(host):
    """No graph is recorded: an output without one would drop the gradient without a word."""
    x, y = store(4), store(5)
    leaf = lambda *s, **k: torch.zeros(s, requires_grad=True, **k)
    coef, b = torch.zeros(5, 2), torch.zeros(2)
    calls = [lambda: qdev.decision8(x, y, leaf(5, 2)), lambda: qdev.decision8(x, y, leaf(5)), lambda: qdev.decision8(x, y, 2 * leaf(5, 2)),
             lambda: qdev.decision8(x, y, coef, leaf(2)), lambda: qdev.decision8(x, y, coef, b, out=leaf(4, 2)),
             lambda: x.write(leaf(2, 100, dtype=torch.complex64), at=0), lambda: y.read(out=leaf(5, 100, dtype=torch.complex64)),
             lambda: qdev.gram8(x, y, out=leaf(4, 5)), lambda: qdev.gram8_jobs([dict(A=x, B=y, KT=leaf(5, 4))])]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError, match="detach"):
            call()
            pytest.fail(f"case {k} was taken")
    assert not host.calls
    out = torch.zeros(4, 2)
    with torch.no_grad():
        qdev.decision8(x, y, leaf(5, 2), leaf(2), out=out)
    qdev.decision8(x, y, leaf(5, 2).detach(), out=out)
    assert [name for name, _ in host.calls].count("qk_decision8_dev") == 2


# ---- served models ---------------------------------------------------------------------------------------------------------
def served(classes, decisions):
    """A model that answers these decision values."""
    from quake_amd.serving import ServedSVC
    m = ServedSVC.__new__(ServedSVC)
    m.classes = np.asarray(classes)
    m.decision_function = lambda x: np.asarray(decisions, dtype=np.float32)
    return m


def test_served_svc_refuses_to_break_ties():
    """break_ties takes the argmax of the ovr values: other answers than the votes of the pairs."""
    from sklearn.svm import SVC
    from quake_amd import circuit as qc, featuremaps as fm
    from quake_amd.kernels import HipFidelityKernel
    from quake_amd.serving import ServedSVC
    k = HipFidelityKernel(fm.zz_featuremap(qc.ParameterVector("x", 3), 3, 1))
    X = np.random.default_rng(0).uniform(size=(21, 3))
    three = SVC(kernel="precomputed", break_ties=True, decision_function_shape="ovr").fit(np.eye(21), np.arange(21) % 3)
    with pytest.raises(ValueError, match="break_ties"):
        ServedSVC(k, three, X)


def test_a_decision_of_exactly_zero_goes_where_sklearn_sends_it():
    from sklearn.svm import SVC
    svc = SVC(kernel="precomputed").fit(np.eye(4), [3, 5, 3, 5])
    rows = np.array([[0, 0, 0, 0], [1, 0, 0, 0], [0, 1, 0, 0]], dtype=float)        # nothing in common with any support vector; one; the other
    d = svc.decision_function(rows)
    assert d[0] == 0 and d[1] < 0 < d[2]
    assert np.array_equal(served([3, 5], d).predict(rows), svc.predict(rows))
    three = SVC(kernel="precomputed", decision_function_shape="ovo").fit(np.eye(6), [0, 1, 2, 0, 1, 2])
    rows = np.zeros((1, 6))
    d = three.decision_function(rows)
    assert (d == 0).all()
    assert np.array_equal(served([0, 1, 2], d).predict(rows), three.predict(rows))


def test_a_sample_without_an_answer_gets_no_label():
    """sklearn refuses a kernel row with NaN; the votes would name a class for it."""
    for classes, d in (([0, 1], [0.5, np.nan]), ([0, 1, 2], [[1, 1, 1], [np.nan, 1, -1]])):
        with pytest.raises(ValueError, match="NaN"):
            served(classes, d).predict(np.zeros((2, 1)))
    assert list(served([4, 9], [np.inf, -np.inf]).predict(np.zeros((2, 1)))) == [9, 4]


@pytest.fixture
def model(monkeypatch):
    """A served model whose store says that it lies on GPU 2, while another is current; nothing runs."""
    from sklearn.svm import SVC
    from quake_amd import circuit as qc, featuremaps as fm
    from quake_amd.kernels import HipFidelityKernel
    from quake_amd.serving import ServedSVC
    entered, synced = [], []

    class Store:
        def __init__(self, capacity, dim, device=None):
            wanted = torch.device("cuda" if device is None else device)
            self.device = torch.device("cuda", 2 if wanted.index is None else wanted.index)

        def write(self, psi):
            synced.clear()                             # work that nobody has waited for

    class Stream:
        def __init__(self, device):
            self.device = device

        def synchronize(self):
            synced.append(self.device)

    monkeypatch.setattr(qdev, "States8", Store)
    monkeypatch.setattr(qdev, "decision8", lambda x, y, coef, b: torch.zeros(1, 1))
    monkeypatch.setattr(qdev.DeviceCircuit, "simulate", lambda self, x: x)
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a: self)
    monkeypatch.setattr(torch.cuda, "device", lambda d: entered.append(d) or contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream(d))
    k = HipFidelityKernel(fm.zz_featuremap(qc.ParameterVector("x", 3), 3, 1))
    X = np.random.default_rng(0).uniform(size=(20, 3))
    m = ServedSVC(k, SVC(kernel="precomputed").fit(X @ X.T, np.arange(20) % 2), X)
    m.entered, m.synced = entered, synced
    return m


def test_a_served_model_stays_on_its_gpu(model):
    here = torch.device("cuda", 2)
    assert model.device == here and all(d == here for d in model.entered) and model.entered


def test_samples_on_another_device_are_refused(model):
    del model.entered[:]
    with pytest.raises(ValueError, match="cuda:2"):
        model.decide(torch.zeros((1, 3), dtype=torch.float64))
    with pytest.raises(ValueError, match="cuda:2"):
        model.decide(torch.utils.dlpack.to_dlpack(torch.zeros((1, 3), dtype=torch.float64)))      # by DLPack, like every device entry point
    assert not model.entered


def test_a_served_model_is_finished_when_it_is_there(model):
    """It may be asked on any stream at once: its constructor has waited for the store's writes."""
    assert model.synced == [torch.device("cuda", 2)]


# ---- the C entry points ------------------------------------------------------------------------------------------------------
def test_no_memory_on_the_host_is_an_error_code():
    """A call of two million jobs in a process that may not grow: an error, no exception across the C boundary."""
    import subprocess
    import sys
    from pathlib import Path
    child = """
import ctypes as C, resource
from quake_amd import _lib
lib, n = _lib.load(), 1 << 21
job = _lib.GRAM8_JOB.pack(1 << 20, 1 << 21, 1 << 22, 1, 1 << 20, 1 << 21, 1 << 22, 1, 64, 1 << 23, 0, 1, 0, 0, 0)
jobs, need = C.create_string_buffer(job * n, len(job) * n), C.c_size_t()
assert lib.qk_gram8_workspace(jobs, 100, C.byref(need)) == 0
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (size + (1 << 20), resource.RLIM_INFINITY))
print(lib.qk_gram8_workspace(jobs, n, C.byref(need)), lib.qk_gram8_jobs_dev(jobs, n, None, 0, None), _lib.last_error())
"""
    done = subprocess.run([sys.executable, "-c", child], capture_output=True, text=True, cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0, done.stderr[-500:]
    assert done.stdout.split()[:2] == [str(_lib.QK_ERR_INVALID)] * 2 and "out of memory" in done.stdout
