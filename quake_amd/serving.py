"""Answers of a fitted QSVM from the statevectors of its support vectors, kept on the GPU in 8 bits.

The reference answers a new sample by evaluating its kernel row against the whole training set and handing that to
sklearn (``qsvm/train.py:152-160``), which simulates every training sample again.  Here the support vectors' states are
simulated and stored once (:class:`quake_amd.device.States8`), and a sample costs its own simulation and one pass over
the store (:func:`quake_amd.device.decision8`); no kernel matrix reaches the host.
"""
from __future__ import annotations

from typing import Tuple

import numpy as np

from . import _lib
from .kernels import HipFidelityKernel, _as_2d

PSI_BYTES = 1 << 30     # statevectors of one batch


def pair_coefficients(svc) -> Tuple[np.ndarray, np.ndarray]:
    """``(coef [n_SV, pairs], intercept [pairs])`` with ``decision = K[:, svc.support_] @ coef + intercept``: one column for
    two classes (positive: ``classes_[1]``), else one per pair of classes i < j in sklearn's "ovo" order (positive: class i)."""
    classes = len(svc.classes_)
    if classes == 2:
        return np.asarray(svc.dual_coef_).T.copy(), np.asarray(svc.intercept_, dtype=np.float64).copy()
    ends = np.cumsum(svc.n_support_)
    of = [slice(e - n, e) for n, e in zip(svc.n_support_, ends)]          # support vectors are grouped by class
    pairs = [(i, j) for i in range(classes) for j in range(i + 1, classes)]
    coef = np.zeros((ends[-1], len(pairs)))
    for p, (i, j) in enumerate(pairs):
        coef[of[i], p] = svc.dual_coef_[j - 1, of[i]]
        coef[of[j], p] = svc.dual_coef_[i, of[j]]
    return coef, np.asarray(svc.intercept_, dtype=np.float64).copy()


class ServedSVC:
    """An ``SVC(kernel="precomputed")`` fitted on ``kernel.evaluate(x_train)``, ready to answer.

    kernel:   the :class:`quake_amd.kernels.HipFidelityKernel` (its feature map and bound training parameters are used; the
              answers come from 8-bit states whatever its precision).
    svc:      the fitted model; up to 11 classes, not with ``break_ties``.
    x_train:  the rows it was fitted on, in their order."""

    def __init__(self, kernel: HipFidelityKernel, svc, x_train, device=None):
        if getattr(svc, "kernel", None) != "precomputed" or not hasattr(svc, "support_"):
            raise ValueError("svc must be a fitted SVC(kernel='precomputed')")
        x, _ = kernel._validate(x_train, None)
        if x.shape[0] != svc.shape_fit_[0]:
            raise ValueError(f"the model was fitted on {svc.shape_fit_[0]} rows, x_train has {x.shape[0]}")
        if getattr(svc, "break_ties", False) and getattr(svc, "decision_function_shape", "ovr") == "ovr" and len(svc.classes_) > 2:
            raise ValueError("svc.break_ties is not supported: classes are decided by the votes of their pairs")
        coef, intercept = pair_coefficients(svc)
        if coef.shape[1] > _lib.QK_DECISION8_MAX_C:
            raise ValueError(f"{len(svc.classes_)} classes need {coef.shape[1]} columns, at most {_lib.QK_DECISION8_MAX_C} are possible")
        import torch

        from . import device as qdev
        self._torch, self._qdev = torch, qdev
        self.classes = np.asarray(svc.classes_)
        self._n_features = x.shape[1]
        self._circuit = qdev.DeviceCircuit(kernel._bound)
        self._rows = max(1, PSI_BYTES // (16 * self._circuit.dim))
        self.store = qdev.States8(coef.shape[0], self._circuit.dim, device=device)
        self.device = self.store.device      # with its index: another GPU may be the current one when the model is asked
        self._coef = torch.as_tensor(coef, dtype=torch.float32).to(self.device).contiguous()
        self._intercept = torch.as_tensor(intercept, dtype=torch.float32).to(self.device)
        self._fill(self.store, torch.as_tensor(x[svc.support_]).to(self.device))
        torch.cuda.current_stream(self.device).synchronize()      # whoever asks may do so on another stream

    def _fill(self, store, x) -> None:
        with self._torch.cuda.device(self.device):
            for a in range(0, x.shape[0], self._rows):
                store.write(self._circuit.simulate(x[a:a + self._rows]))

    def decide(self, x):
        """Decision values of device rows: float64 [M, features] tensor on the model's GPU -> float32 [M, pairs] tensor, enqueued
        on that GPU's current stream."""
        x = self._qdev.from_dlpack(x)
        if x.device != self.device:
            raise ValueError(f"x is on {x.device}, the model on {self.device}")
        queries = self._qdev.States8(x.shape[0], self._circuit.dim, device=self.device)
        self._fill(queries, x)
        return self._qdev.decision8(queries, self.store, self._coef, self._intercept)

    def decision_function(self, x_vec) -> np.ndarray:
        """float32 [M] for two classes, else [M, pairs] in "ovo" order."""
        x = _as_2d(x_vec, "x_vec")
        if x.shape[1] != self._n_features:
            raise ValueError(f"x_vec has {x.shape[1]} columns, the model {self._n_features}")
        out = self.decide(self._torch.as_tensor(x).to(self.device)).cpu().numpy()
        return out[:, 0] if len(self.classes) == 2 else out

    def predict(self, x_vec) -> np.ndarray:
        """Class labels: the sign for two classes (zero goes to ``classes[1]``), else most pairs won (a tie goes to the class that
        comes first).  A sample whose decision values are NaN (one whose features are not finite) is refused."""
        d = self.decision_function(x_vec)
        if np.isnan(d).any():
            raise ValueError(f"{int(np.isnan(d.reshape(len(d), -1)).any(axis=1).sum())} of {len(d)} samples have NaN decision values")
        if len(self.classes) == 2:
            return self.classes[(d >= 0).astype(int)]
        votes = np.zeros((d.shape[0], len(self.classes)), dtype=int)
        rows, p = np.arange(d.shape[0]), 0
        for i in range(len(self.classes)):
            for j in range(i + 1, len(self.classes)):
                np.add.at(votes, (rows, np.where(d[:, p] > 0, i, j)), 1)
                p += 1
        return self.classes[votes.argmax(axis=1)]
