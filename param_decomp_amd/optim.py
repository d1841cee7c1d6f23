"""AdamW over many tensors at once, on the GPU.

The optimizer of the components and CI functions (`param_decomp/param_decomp/core/optimizer.py`,
there optax's adamw): master parameters in fp32, moments in fp32 or in 8 bits, and the bf16 casts
that the next step computes with, all tensors in one launch.
"""

from __future__ import annotations

import ctypes
import operator

import torch

from param_decomp_amd import _lib as L
from param_decomp_amd.prng import Key

QBLOCK = 256  # values of an 8-bit state that share a scale
FP8 = torch.float8_e4m3fn
_ADDRESS, _NUMEL = torch.Tensor.data_ptr, torch.Tensor.numel


def _plain(name: str, label: str, t: torch.Tensor, numel: int, dtypes, device) -> torch.Tensor:
    if t is None:
        raise L.PDError(f"{name}: {label} is missing")
    if t.dtype not in dtypes or t.numel() != numel or t.device != device or not t.is_contiguous():
        raise L.PDError(f"{name}: {label} is a dense {' or '.join(str(d)[6:] for d in dtypes)} tensor of {numel} values "
                        f"on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t


class AdamW:
    """`p -= lr (weight_decay p + m_hat / (sqrt(v_hat) + eps))` for every tensor of `params` (fp32,
    dense, one GPU), as `torch.optim.AdamW`. `state_bits` 8 keeps m and sqrt(v) as
    `float8_e4m3fn` with one fp32 scale for 256 values, rounded stochastically with draws of
    `key`; tensors of fewer than `min_8bit_size` values keep fp32 states then. `copies`: bf16
    tensors of the parameters' sizes (or None in their places) that receive the new values with
    the step.

    `state`: {"step" int32 [1], "m", "v": lists} and with 8 bits {"m_scale", "v_scale": lists},
    where a tensor of fp32 states has None; used in place. Default: zeros. `v` holds sqrt(v)
    where it has 8 bits. The step count is in device memory: a captured `step` goes on counting
    when it is replayed. Tensors exchanged in `params`, `state` and `copies` (of the same sizes and types: checked) are those that
    the next `step` uses; a captured one keeps those that it was captured with."""

    def __init__(self, params, *, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32, key: Key = (0, 0), min_8bit_size: int = 0,
                 copies=None, state: dict | None = None):
        name = "AdamW"
        self.params = [p for p in params]
        if not self.params:
            raise L.PDError(f"{name}: no parameters")
        if state_bits not in (8, 32):
            raise L.PDError(f"{name}: states have 8 or 32 bits, got {state_bits}")
        device = self.params[0].device
        if device.type != "cuda":
            raise L.PDError("pd kernels take GPU tensors")
        self.device, self.lr, self.betas, self.eps, self.weight_decay = device, lr, betas, eps, weight_decay
        self.key = (int(key[0]), int(key[1]))
        self._sizes = [p.numel() for p in self.params]
        self._small = [state_bits == 32 or n < min_8bit_size for n in self._sizes]  # states of 32 bits
        self.state = self._zeros(self._sizes, self._small) if state is None else state
        self.copies = None if copies is None else list(copies)
        self._ticket = torch.zeros(1, dtype=torch.int32, device=device)
        self._c_sizes = L.host_array(ctypes.c_int64, self._sizes)
        self._held: list = []
        self._pointers()

    def _pointers(self) -> None:
        """The arrays of addresses, checked and formed again where a tensor is another one than before or its memory has been
        exchanged (`p.data = ...`): the steps use what `params`, `state` and `copies` hold when they run."""
        n, st = len(self._sizes), self.state
        none = [None] * n
        # the tensors of each argument, in the entry point's order
        held = [*self.params, *st["m"], *st["v"], *(st.get("m_scale") or none), *(st.get("v_scale") or none),
                *(none if self.copies is None else self.copies), st["step"]]
        live = [t for t in held if t is not None]
        at, sizes = list(map(_ADDRESS, live)), list(map(_NUMEL, live))
        if len(held) == len(self._held) and all(map(operator.is_, held, self._held)) and at == self._at and sizes == self._at_sizes:
            return
        self._check()
        where = [None if t is None else t.data_ptr() or None for t in held]
        arrays = [L.host_array(ctypes.c_void_p, where[k * n:(k + 1) * n]) for k in range(6)]
        self._p, self._m, self._v, self._ms, self._vs, self._c = arrays
        self._shapes = [p.shape for p in self.params]
        self._written = [*self.params, *(c for c in self.copies or () if c is not None)]
        self._held, self._at, self._at_sizes = held, at, sizes
        # the memory is kept, so that nothing else can come to lie at an address that was checked
        self._memory = [t.detach() for t in live]

    def _check(self) -> None:
        name, st, sizes = "AdamW", self.state, self._sizes
        if len(self.params) != len(sizes):
            raise L.PDError(f"{name}: {len(self.params)} parameters, {len(sizes)} when it was made")
        for i, (p, n) in enumerate(zip(self.params, sizes)):
            _plain(name, f"parameter {i}", p, n, (torch.float32,), self.device)
        self._check_state(sizes, self._small)
        copies = [None] * len(sizes) if self.copies is None else self.copies
        if len(copies) != len(sizes):
            raise L.PDError(f"{name}: {len(copies)} copies for {len(sizes)} parameters")
        for i, (c, n) in enumerate(zip(copies, sizes)):
            if c is not None:
                _plain(name, f"copy {i}", c, n, (torch.bfloat16,), self.device)
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                       for ts in (self.params, st["m"], st["v"], st.get("m_scale") or (), st.get("v_scale") or (), copies, [st["step"]])
                       for t in ts if t is not None and t.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise L.PDError(f"{name}: two of the parameters, states and copies share memory")

    def _zeros(self, sizes, small) -> dict:
        dev = self.device
        one = lambda n, s: torch.zeros(n, dtype=torch.float32 if s else FP8, device=dev)  # noqa: E731
        state = {"step": torch.zeros(1, dtype=torch.int32, device=dev)}
        for name in ("m", "v"):
            state[name] = [one(n, s) for n, s in zip(sizes, small)]
            state[name + "_scale"] = [None if s else torch.zeros(-(-n // QBLOCK), dtype=torch.float32, device=dev)
                                      for n, s in zip(sizes, small)]
        return state

    def _check_state(self, sizes, small) -> None:
        st, name = self.state, "AdamW"
        _plain(name, "step", st["step"], 1, (torch.int32,), self.device)
        for key in ("m", "v"):
            scales = st.get(key + "_scale") or [None] * len(sizes)
            if len(st[key]) != len(sizes) or len(scales) != len(sizes):
                raise L.PDError(f"{name}: state {key} has {len(st[key])} tensors for {len(sizes)} parameters")
            for i, (n, s) in enumerate(zip(sizes, small)):
                _plain(name, f"{key}[{i}]", st[key][i], n, (torch.float32 if s else FP8,), self.device)
                if s != (scales[i] is None):
                    raise L.PDError(f"{name}: {key}_scale[{i}] goes with a state of 8 bits")
                if not s:
                    _plain(name, f"{key}_scale[{i}]", scales[i], -(-n // QBLOCK), (torch.float32,), self.device)

    def _scalar(self, label: str, t: torch.Tensor) -> int:
        return _plain("AdamW.step", label, t, 1, (torch.float32,), self.device).data_ptr()

    def step(self, grads=None, *, lr: float | torch.Tensor | None = None,
             grad_scale: torch.Tensor | None = None) -> None:
        """One step from `grads` (fp32 or bf16, one for each parameter; None: their `.grad`); a
        parameter whose gradient is None stays as it is. `lr`: this step's, a number or an fp32
        tensor of one value on the GPU, and `grad_scale` such a tensor that gradients are
        multiplied with: both are read when the step runs, also in a replayed graph."""
        name, n = "AdamW.step", len(self._sizes)
        self._pointers()
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != n:
            raise L.PDError(f"{name}: {len(grads)} gradients for {n} parameters")
        ptrs, types, dense = [], [], []
        for i, g in enumerate(grads):
            if g is None:
                ptrs.append(None)
                types.append(L.F32)
                continue
            if g.shape != self._shapes[i] or g.device != self.device or g.dtype not in (torch.float32, torch.bfloat16):
                raise L.PDError(f"{name}: gradient {i} is float32 or bfloat16 {tuple(self._shapes[i])} on {self.device}, "
                                f"got {g.dtype} {tuple(g.shape)} on {g.device}")
            if not g.is_contiguous():
                g = g.contiguous()
                dense.append(g)
            ptrs.append(g.data_ptr())
            types.append(L.F32 if g.dtype == torch.float32 else L.BF16)
        lr = self.lr if lr is None else lr
        lr_dev = self._scalar("lr", lr) if isinstance(lr, torch.Tensor) else None
        scale = None if grad_scale is None else self._scalar("grad_scale", grad_scale)
        L.launch("pd_adamw_step", self.device, n, self._c_sizes, self._p, (ctypes.c_void_p * n)(*ptrs),
                 (ctypes.c_int32 * n)(*types), self._m, self._v, self._ms, self._vs, self._c,
                 self.state["step"].data_ptr(), self._ticket.data_ptr(), 0.0 if lr_dev else float(lr), lr_dev, scale,
                 self.betas[0], self.betas[1], self.eps, self.weight_decay, self.key[0], self.key[1])
        torch.autograd.graph.increment_version(self._written)

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    def state_dict(self) -> dict:
        """The state's tensors themselves (clone what has to outlive the next step)."""
        return dict(self.state)

    def load_state_dict(self, state: dict) -> None:
        """Copies `state`, of an optimizer over parameters of the same sizes and bits, into this one's."""
        pairs, none = [], [None] * len(self._sizes)
        for name in ("step", "m", "v", "m_scale", "v_scale"):
            mine, theirs = self.state.get(name), state.get(name)
            mine, theirs = ([x] if isinstance(x, torch.Tensor) else list(x or none) for x in (mine, theirs))
            if len(mine) != len(theirs) or any((a is None) != (b is None) or
                                               (a is not None and (a.dtype != b.dtype or a.numel() != b.numel()))
                                               for a, b in zip(mine, theirs)):
                raise L.PDError(f"AdamW.load_state_dict: {name} is of other sizes or bits")
            pairs += [(a, b) for a, b in zip(mine, theirs) if a is not None]
        for a, b in pairs:
            a.copy_(b.reshape(a.shape))
