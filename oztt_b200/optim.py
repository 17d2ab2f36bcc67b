"""AdamW over many CUDA tensors of torch in one launch, with moments in 32 bits or in 8 (oztt_adamw_step of the
C ABI). No counterpart in the reference."""

from __future__ import annotations

import struct

import numpy as np
import torch

from . import _binding

__all__ = ["AdamW"]

BLOCK = 256  # OZTT_ADAMW_BLOCK: elements of the moments that share an exponent
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # OZTT_TYPE_*

# oztt_adamw_tensor and oztt_adamw_hyper
_TENSOR = np.dtype([("param", np.uint64), ("grad", np.uint64), ("master", np.uint64), ("count", np.uint64),
                    ("param_type", np.int32), ("grad_type", np.int32)])
_HYPER = struct.Struct("=5dQQI4x")

_torch = _binding()  # csrc/torch_binding.cpp: the tensors' checks and addresses, the current stream


class AdamW:
    """The AdamW optimiser of a list of tensors (Adam with decoupled weight decay), one launch a step.

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

    params: contiguous BF16, FP16 or FP32 tensors of one CUDA device that do not overlap; they are updated in place.
    state_bits: 32, or 8 for moments of one byte an element, blocks of 256 elements sharing an exponent, rounded
    stochastically (by `seed` and the step's number, so that a run can be repeated).
    masters: FP32 copies of the parameters that the steps are taken on (a list as long as params, with None for
    those without), or True to make them; without, the step is taken on the parameter's own value and rounded to
    its type to nearest, which loses steps smaller than half its spacing.
    """

    def __init__(self, params, *, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32, masters=None, seed: int = 0):
        params = list(params)
        if not params:
            raise ValueError("AdamW: no parameters")
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits must be 8 or 32")
        device = params[0].device
        if device.type != "cuda":
            raise ValueError("AdamW: the parameters must be on a CUDA device")
        if masters is True:
            masters = [None if p.dtype == torch.float32 else p.detach().float() for p in params]
        masters = [None] * len(params) if masters is None or masters is False else list(masters)
        if len(masters) != len(params):
            raise ValueError("AdamW: masters must be as many as params")
        spans = []
        for i, (p, w) in enumerate(zip(params, masters)):
            if p.dtype not in _TYPES or p.device != device or not p.is_contiguous() or not _torch.has_memory(p):
                raise ValueError(f"AdamW: parameter {i} must be a contiguous BF16, FP16 or FP32 tensor on {device}")
            spans.append((p.data_ptr(), p.numel() * p.element_size()))
            if w is not None:
                if (w.dtype != torch.float32 or w.device != device or not w.is_contiguous() or w.shape != p.shape
                        or not _torch.has_memory(w)):
                    raise ValueError(f"AdamW: master {i} must be a contiguous FP32 tensor like its parameter")
                spans.append((w.data_ptr(), w.numel() * 4))
        end = 0
        for at, size in sorted(s for s in spans if s[1]):
            if at < end:
                raise ValueError("AdamW: parameters overlap")
            end = at + size
        self.params, self.masters, self.state_bits, self.device, self.seed = params, masters, state_bits, device, seed
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.t = 0
        self._counts = [p.numel() for p in params]
        blocks = [-(-n // BLOCK) for n in self._counts]
        self.blocks = sum(blocks)
        # where each tensor's part of the flat moments starts
        self.offsets = [BLOCK * (sum_ - b) for b, sum_ in zip(blocks, np.cumsum(blocks).tolist())]
        kind = torch.uint8 if state_bits == 8 else torch.float32
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=device)  # noqa: E731
        self._m, self._v = zeros(self.blocks * BLOCK, kind), zeros(self.blocks * BLOCK, kind)
        self._m_exp = self._v_exp = None
        if state_bits == 8:
            self._m_exp, self._v_exp = zeros(self.blocks, kind), zeros(self.blocks, kind)
        self._table = np.zeros(len(params), _TENSOR)
        self._table["count"] = self._counts
        self._table["param_type"] = [_TYPES[p.dtype] for p in params]

    def step(self, grads=None, *, grad_scale: torch.Tensor | None = None, lr: float | None = None,
             seed: int | None = None) -> None:
        """One step on the current stream, without waiting for it. grads: a gradient for each parameter (contiguous,
        of the parameter's size, BF16, FP16 or FP32), None for one that stays as it is; by default the parameters'
        .grad. grad_scale: one FP32 number on the device that every gradient is multiplied by (a clipping
        coefficient). lr: this step's learning rate. seed: of this step's rounding, by default from the optimiser's
        seed and the step's number. The step's number and rates are numbers of the launch: a CUDA graph of it
        repeats the same step. The versions of what is stepped are raised, as by torch's own operations in place."""
        if grads is None:
            grads = [p.grad for p in self.params]
        t = self.t + 1
        if seed is None:
            seed = self.seed + 0x632BE5AB * t
        hyper = _HYPER.pack(self.lr if lr is None else lr, *self.betas, self.eps, self.weight_decay, t,
                            0, seed & 0xFFFFFFFF)
        _torch.adamw_step(self._table, self.params, self.masters, grads, grad_scale,
                          (self._m, self._v, self._m_exp, self._v_exp), hyper, self.device.index)
        self.t = t

    # The moments as they are kept: FP32, or bytes with the blocks' exponents.
    m = property(lambda self: self._m)
    v = property(lambda self: self._v)
    m_exp = property(lambda self: self._m_exp)
    v_exp = property(lambda self: self._v_exp)

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The flat moments (m, v), tensor i's from offsets[i] on: the FP32 buffers themselves with 32 bits, new
        BF16 tensors with 8, which hold the values of the codes exactly."""
        if self.state_bits == 32:
            return self._m, self._v
        return _torch.adamw_values((self._m, self._v, self._m_exp, self._v_exp), self.blocks, self.device.index)

    def state_dict(self) -> dict:
        """What load_state_dict needs to go on from here: the number of steps, the moments as they are kept, and the
        masters. The tensors are the optimiser's own."""
        d = {"t": self.t, "state_bits": self.state_bits, "seed": self.seed, "counts": tuple(self._counts), "m": self._m,
             "v": self._v, "masters": self.masters}
        if self.state_bits == 8:
            d["m_exp"], d["v_exp"] = self._m_exp, self._v_exp
        return d

    def load_state_dict(self, d: dict) -> None:
        """Copies a state_dict of an optimiser of like tensors and bits; ValueError, with nothing copied, for another."""
        names = ["m", "v"] + (["m_exp", "v_exp"] if self.state_bits == 8 else [])
        missing = [n for n in (*names, "masters", "t", "seed") if n not in d]
        if missing:
            raise ValueError(f"AdamW: the state has no {', '.join(missing)}")
        like = lambda x, y: x is None if y is None else (  # noqa: E731
            torch.is_tensor(x) and x.shape == y.shape and x.dtype == y.dtype)
        # (a state without counts was saved before they were part of one)
        if (d.get("state_bits") != self.state_bits or list(d.get("counts", self._counts)) != self._counts
                or not all(like(d[n], getattr(self, "_" + n)) for n in names)):
            raise ValueError("AdamW: the state is of other tensors or bits")
        if len(d["masters"]) != len(self.masters) or not all(map(like, d["masters"], self.masters)):
            raise ValueError("AdamW: the state has other masters")
        for n in names:
            getattr(self, "_" + n).copy_(d[n])
        for w, s in zip(self.masters, d["masters"]):
            if w is not None:
                w.copy_(s)
        self.t, self.seed = int(d["t"]), int(d["seed"])
