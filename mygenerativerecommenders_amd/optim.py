"""AdamW as one launch per parameter group (``gr_adamw_step``).

torch.optim.AdamW(fused=True, capturable=True) -- the reference's optimizer
(``configs/model/*.yaml``: AdamW, betas (0.9, 0.98), weight decay 1e-3) -- costs two
launches per step on the GPU: the step counters' ``_foreach_add_`` and the fused
multi-tensor kernel.  ``FlatAdamW`` keeps the moments in two flat fp32 buffers and runs
the same update, the counter advanced inside the same launch; the tensors' pointers
travel in the kernel arguments (up to 48 tensors per launch), as torch's tensor lists
do, so graph capture and fresh gradient tensors each step both work.  The
per-parameter state (``exp_avg`` / ``exp_avg_sq`` views into the flat buffers, ``step``)
has torch's names.  Dense fp32 CUDA tensors only; ``amsgrad`` and ``maximize`` raise.

``state_bits=8`` holds both moments in 8 bits (``gr_adamw8_step``): 2.1 bytes of state an
element instead of 8.  ``exp_avg`` / ``exp_avg_sq`` are then ``torch.float8_e4m3fn`` and
``exp_avg_scale`` / ``exp_avg_sq_scale`` hold a power of two for each 64 consecutive elements:
a moment is code times scale.  Codes are rounded at random from a hash of (element, step), so
equal gradients give equal bits on every replica and in every run.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib


_BLOCK = 64  # elements that share a scale of an 8-bit moment


class FlatAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, amsgrad: bool = False, maximize: bool = False,
                 state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"FlatAdamW: state_bits must be 8 or 32 (got {state_bits})")
        if amsgrad or maximize:
            raise NotImplementedError("FlatAdamW: amsgrad / maximize are not supported")
        if not 0.0 <= lr or not 0.0 <= eps or not 0.0 <= weight_decay:
            raise ValueError(f"FlatAdamW: invalid lr / eps / weight_decay ({lr}, {eps}, {weight_decay})")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"FlatAdamW: invalid betas {betas}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self._flat: dict = {}
        self._bits = state_bits

    def _group_state(self, gi: int, group: dict) -> dict:
        fs = self._flat.get(gi)
        if fs is not None:
            return fs
        params = group["params"]
        if not self._takes(params):
            raise TypeError("FlatAdamW: contiguous fp32 CUDA parameters on one device expected")
        fs = self._buffers8(params) if self._bits == 8 else self._buffers32(params)
        self._fill(fs, params)
        self._flat[gi] = fs
        return fs

    def _takes(self, params: list) -> bool:
        return all(p.device == params[0].device and p.dtype == torch.float32 and p.is_contiguous() and p.is_cuda
                   for p in params)

    def _buffers32(self, params: list) -> dict:
        offs = np.zeros(len(params), np.int64)
        o = 0
        for i, p in enumerate(params):
            offs[i] = o
            o += (p.numel() + 3) // 4 * 4  # 16-byte aligned moments (float4 path)
        new = {"dtype": torch.float32, "device": params[0].device}
        return {"m": torch.zeros(o, **new), "v": torch.zeros(o, **new), "step": torch.zeros(1, **new),
                "done": torch.zeros(1, dtype=torch.int32, device=params[0].device), "offs": offs}

    def _buffers8(self, params: list) -> dict:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FlatAdamW: take a step (or load a state) before capturing one, or the "
                               "captured graph would clear the moments on every replay")
        offs = np.zeros(len(params), np.int64)
        o = 0
        for i, p in enumerate(params):
            offs[i] = o
            o += -(-p.numel() // _BLOCK) * _BLOCK  # scales belong to one tensor each
        dev = params[0].device
        return {"exp_avg": torch.zeros(o, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                "exp_avg_scale": torch.zeros(o // _BLOCK, dtype=torch.float32, device=dev),
                "exp_avg_sq": torch.zeros(o, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                "exp_avg_sq_scale": torch.zeros(o // _BLOCK, dtype=torch.float32, device=dev),
                "step": torch.zeros(1, dtype=torch.float32, device=dev),
                "done": torch.zeros(1040, dtype=torch.int32, device=dev),  # 65 counters, 64 bytes apart
                "offs": offs}

    def _names(self) -> tuple:
        return ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if self._bits == 8 else ())

    def _views(self, fs: dict, p, off: int) -> dict:
        """The per-parameter state of p, whose moments start at element ``off`` of the buffers."""
        n = p.numel()
        if self._bits == 8:
            blocks = slice(off // _BLOCK, (off + n + _BLOCK - 1) // _BLOCK)
            return {"step": fs["step"], "exp_avg": fs["exp_avg"][off:off + n].view_as(p),
                    "exp_avg_scale": fs["exp_avg_scale"][blocks],
                    "exp_avg_sq": fs["exp_avg_sq"][off:off + n].view_as(p),
                    "exp_avg_sq_scale": fs["exp_avg_sq_scale"][blocks]}
        return {"step": fs["step"], "exp_avg": fs["m"][off:off + n].view_as(p),
                "exp_avg_sq": fs["v"][off:off + n].view_as(p)}

    @torch.no_grad()
    def _fill(self, fs: dict, params: list) -> None:
        """Moves what ``self.state`` holds for the parameters (a loaded state, checked) into a group's
        buffers, zeros where they hold nothing yet, and makes the state views of them."""
        step = None
        for p, off in zip(params, fs["offs"].tolist()):
            loaded, self.state[p] = self.state.get(p), self._views(fs, p, off)
            if loaded:
                for n in self._names():
                    self.state[p][n].copy_(loaded[n])
                step = loaded["step"]
        if step is not None:
            fs["step"].copy_(torch.as_tensor(step, dtype=torch.float32).reshape(1))

    def flat_state(self, group: int = 0) -> dict:
        """The flat buffers behind a parameter group's per-parameter state, by torch's names
        (``exp_avg``, ``exp_avg_sq``, ``step``; with ``state_bits=8`` the two scales too).
        Tensor i's entries start at its offset: sizes rounded up to 4 elements (32 bits) or
        64 (8 bits), in the order of the group's parameters."""
        fs = self._group_state(group, self.param_groups[group])
        if self._bits == 8:
            return {n: t for n, t in fs.items() if n not in ("done", "offs")}
        return {"exp_avg": fs["m"], "exp_avg_sq": fs["v"], "step": fs["step"]}

    def load_state_dict(self, state_dict: dict) -> None:
        """torch's, with the loaded moments copied into the flat buffers that the step reads: those
        that are there, so that a captured step goes on from them.  A state of the other
        ``state_bits`` raises ValueError, and so do parameters of one group that have taken
        different numbers of steps (the group has one counter); the optimizer is then as it was.
        With parameters on the CPU the state waits for the first step on the GPU."""
        kept, fresh = (self.state, self.param_groups), {}
        try:
            super().load_state_dict(state_dict)
            self._check_loaded()
            for gi, group in enumerate(self.param_groups):
                params = group["params"]
                if params and self._takes(params) and (gi in self._flat or any(self.state.get(p) for p in params)):
                    fresh[gi] = self._buffers8(params) if self._bits == 8 else self._buffers32(params)
                    self._fill(fresh[gi], params)
                else:  # waits, on its own: what was loaded may be another optimizer's buffers
                    for p in params:
                        if self.state.get(p):
                            self.state[p] = {n: t.clone() if torch.is_tensor(t) else t for n, t in self.state[p].items()}
        except BaseException:
            self.state, self.param_groups = kept
            raise
        for gi in [i for i in self._flat if i not in fresh]:
            del self._flat[gi]
        for gi, new in fresh.items():
            old = self._flat.setdefault(gi, new)
            if old is new:
                continue
            if old["step"].device != new["step"].device or not np.array_equal(old["offs"], new["offs"]):
                self._flat[gi] = new
                continue
            for n in old:  # the loaded tensors may be views of these: through the fresh ones
                if n not in ("done", "offs"):
                    old[n].copy_(new[n])
            for p, off in zip(self.param_groups[gi]["params"], old["offs"].tolist()):
                self.state[p] = self._views(old, p, off)

    def _check_loaded(self) -> None:
        """Raises ValueError unless ``self.state``, as torch has loaded it, fits."""
        names, groups, steps, there = self._names(), [], {}, []
        for group in self.param_groups:
            groups.append([])
            for p in group["params"]:
                st = self.state.get(p)
                if not st:
                    continue
                if any(n not in st for n in (*names, "step")) or ("exp_avg_scale" in st) != (self._bits == 8):
                    raise ValueError(f"FlatAdamW: the loaded state does not hold {self._bits}-bit moments")
                for n in names:
                    want = (-(-p.numel() // _BLOCK),) if n.endswith("scale") else tuple(p.shape)
                    if tuple(st[n].shape) != want:
                        raise ValueError(f"FlatAdamW: loaded {n} has shape {tuple(st[n].shape)}, expected {want}")
                step = st["step"]
                groups[-1].append(step)
                if torch.is_tensor(step) and step.numel() != 1:
                    raise ValueError(f"FlatAdamW: loaded step has shape {tuple(step.shape)}")
                if id(step) not in steps:
                    steps[id(step)] = step
                    if torch.is_tensor(step) and step.is_cuda:
                        there.append(step)
        if there:  # one copy to the host for all
            dev = there[0].device
            values = torch.stack([t.detach().reshape(()).to(dev, torch.float32) for t in there]).tolist()
            steps.update((id(t), v) for t, v in zip(there, values))
        for group in groups:
            taken = {float(steps[id(step)]) for step in group}
            if len(taken) > 1:
                raise ValueError(f"FlatAdamW: parameters of one group have taken {sorted(taken)} steps")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            params = group["params"]
            if self._bits == 8 and params:
                fs = self._flat.get(gi) or self._group_state(gi, group)
                _lib.nodes().adamw8_step.default(
                    params, fs["exp_avg"], fs["exp_avg_scale"], fs["exp_avg_sq"], fs["exp_avg_sq_scale"],
                    fs["step"], fs["done"], float(group["lr"]), float(group["betas"][0]),
                    float(group["betas"][1]), float(group["eps"]), float(group["weight_decay"]))
                continue
            if not params or all(p.grad is None for p in params):
                continue
            fs = self._group_state(gi, group)
            n = len(params)
            pp = np.zeros(n, np.uint64)
            gp = np.zeros(n, np.uint64)
            ne = np.zeros(n, np.int64)
            for i, p in enumerate(params):
                g = p.grad
                if g is None:
                    continue
                if (g.dtype != torch.float32 or g.is_sparse or not g.is_contiguous()
                        or g.shape != p.shape or g.device != p.device):
                    raise TypeError("FlatAdamW: dense contiguous fp32 gradients expected")
                pp[i], gp[i], ne[i] = p.data_ptr(), g.data_ptr(), p.numel()
            b1, b2 = group["betas"]
            _lib.call("gr_adamw_step", pp.ctypes.data, gp.ctypes.data, fs["offs"].ctypes.data,
                      ne.ctypes.data, n, fs["m"].data_ptr(), fs["v"].data_ptr(),
                      fs["step"].data_ptr(), fs["done"].data_ptr(), float(group["lr"]), float(b1),
                      float(b2), float(group["eps"]), float(group["weight_decay"]),
                      _lib.stream_handle())
        return loss
