"""AdamW over many tensors at once, next to the Newton-Schulz step of the matrices (zmoe.muon): the reference trains what
Muon leaves (gates, norms, embeddings) with an auxiliary Adam (optimizer/muon.py:574-653), inside a captured graph
(optimizer/hybrid.py:95-117).

``AdamW`` is a ``torch.optim.Optimizer``. A step is one launch over all tensors of a type (forty-eight a launch), a small
one in front for the step counts, and two more for the grads' norm where it clips. Everything that a step needs is on the
device, so a step can be captured into a graph and replayed (after one eager step, which makes the state).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import library, ops, profiling

_STATE_DTYPES = {32: (torch.float32, torch.float32), 8: (torch.int8, torch.uint8)}


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill its memory without gaps or overlaps, in any order of its dims."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != step:
            return False
        step *= size
    return True


def _alike(t: torch.Tensor, p: torch.Tensor) -> bool:
    """Whether t's elements lie in memory as p's do."""
    return t.shape == p.shape and all(a == b for a, b, n in zip(t.stride(), p.stride(), p.shape) if n != 1)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, p <- p - lr wd p - lr mhat / (sqrt(vhat) + eps), for float32 and bfloat16
    parameters on the GPU (float32 arithmetic, one rounding of a bfloat16 parameter; parameters must not share memory).

    ``state_bits`` (also a group's): 32, moments in float32; 8, a byte for each element and a float32 scale for each 256 of
    them (``zmoe.h``, zmoe_adamw). ``max_grad_norm``: the grads of all groups are multiplied by
    min(1, max_grad_norm / (norm + 1e-6)), norm their common 2-norm, which ``grad_norm`` holds after a step. ``lr``: a number
    or a float32 tensor of one element on the device, which a captured step reads anew."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, max_grad_norm: Optional[float] = None):
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        if self.max_grad_norm is not None and not self.max_grad_norm > 0.0:
            raise ValueError(f"AdamW: max_grad_norm must be positive, got {max_grad_norm}")
        self.grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    @staticmethod
    def _check_group(g) -> None:
        """Whether a group's numbers are a step's."""
        lr, betas = g["lr"], tuple(g["betas"])
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or (lr.is_cuda and lr.dtype != torch.float32):
                raise ValueError("AdamW: lr must be a number or a float32 tensor of one element")
        elif not lr >= 0.0:
            raise ValueError(f"AdamW: lr must not be negative, got {lr}")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas}")
        if not g["eps"] >= 0.0 or not g["weight_decay"] >= 0.0:
            raise ValueError(f"AdamW: eps and weight_decay must not be negative, got {g['eps']} and {g['weight_decay']}")
        if g["state_bits"] not in _STATE_DTYPES:
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {g['state_bits']}")

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            self._check_group(g)
            if len({id(p) for p in g["params"]}) != len(g["params"]):
                raise ValueError("AdamW: a parameter is given twice")  # (one launch would write it from two places)
            for p in g["params"]:
                if type(p).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__:
                    raise ValueError(f"AdamW: a parameter of {type(p).__name__}, whose memory is not its own (sharded and other "
                                     "wrapped tensors: give what they hold)")
                if p.dtype not in (torch.float32, torch.bfloat16):
                    raise ValueError(f"AdamW: parameters must be float32 or bfloat16, got {p.dtype}")
                if not _dense(p):
                    raise ValueError("AdamW: a parameter's elements must lie in memory without gaps or overlaps "
                                     f"(shape {tuple(p.shape)}, strides {p.stride()})")
        except ValueError:
            self.param_groups.pop()
            raise

    def __getstate__(self) -> dict:  # (copies and pickles keep the clipping; a state_dict leaves it to the constructor)
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "grad_norm": None}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        for g in self.param_groups:
            g.setdefault("state_bits", 32)

    @torch.inference_mode(False)  # (a state made under inference mode could not be changed after it)
    def _state_of(self, p: torch.Tensor, bits: int) -> dict:
        st = self.state[p]
        if not st:
            if not p.is_cuda:
                raise ValueError("zmoe ops need tensors on a HIP device")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: take a step before capturing one (its state must not be made in the graph)")
            m, v = _STATE_DTYPES[bits]
            st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            st["exp_avg"] = torch.zeros_like(p, dtype=m)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=v)
            if bits == 8:
                n = -(-p.numel() // ops.ADAMW_BLOCK)
                st["exp_avg_scale"] = torch.zeros(n, dtype=torch.float32, device=p.device)
                st["exp_avg_sq_scale"] = torch.zeros(n, dtype=torch.float32, device=p.device)
        return st

    def step(self, closure=None):
        return (self._uncompiled if torch.compiler.is_compiling() else self._step)(closure)

    @torch.no_grad()
    def _step(self, closure):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, all_grads = [], []
        for group in self.param_groups:
            bits = group["state_bits"]
            lists = [], [], [], [], [], [], []  # params, grads, m, v, m scales, v scales, steps
            ps, gs, ms, vs, sms, svs, ts = lists
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                st = self.state.get(p) or self._state_of(p, bits)
                if bits == 8 and "exp_avg_scale" not in st:
                    raise ValueError("AdamW: moments in 32 bits in a group of state_bits 8")
                ps.append(p)
                gs.append(g)
                ms.append(st["exp_avg"])
                vs.append(st["exp_avg_sq"])
                ts.append(st["step"])
                if bits == 8:
                    sms.append(st["exp_avg_scale"])
                    svs.append(st["exp_avg_sq_scale"])
            if ps:
                work.append((group, lists))
                all_grads += gs
        if not work:
            return loss
        native = None if profiling.active() else library.native_node("adamw_step", ())
        clip = None
        if self.max_grad_norm is not None:
            norm = None if native is None else library.native_node("grad_norm", ())(all_grads, self.max_grad_norm)
            if norm is None:
                for _, lists in work:
                    self._in_order(lists)
                norm = ops.grad_norm([g for _, lists in work for g in lists[1]], self.max_grad_norm)
            self.grad_norm, clip = norm[0], norm[1]
        for group, lists in work:
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and not lr.is_cuda:
                lr = float(lr)
            lr_t, lr = (lr, 0.0) if isinstance(lr, torch.Tensor) else (None, float(lr))
            b1, b2 = group["betas"]
            if native is not None and native(*lists, group["state_bits"], lr_t, lr, b1, b2, group["eps"],
                                             group["weight_decay"], clip):
                continue
            self._in_order(lists)
            if not torch.is_inference_mode_enabled() and any(t.is_inference() for some in (lists[0], *lists[2:]) for t in some):
                raise RuntimeError("AdamW: a parameter or state made under inference mode is changed under it only")
            for p, m, v in zip(lists[0], lists[2], lists[3]):
                if not _alike(m, p) or not _alike(v, p):
                    raise RuntimeError("AdamW: a parameter's shape or order in memory is not its moments'")
            by: dict = {}  # one call for each device and type
            for i, p in enumerate(lists[0]):
                for to, of in zip(by.setdefault((p.device, p.dtype), ([], [], [], [], [], [], [])), lists):
                    if of:
                        to.append(of[i])
            for to in by.values():
                ops.adamw_(*to, group["state_bits"], lr if lr_t is None else lr_t, b1, b2, group["eps"],
                           group["weight_decay"], clip)
                torch.autograd.graph.increment_version([t for some in (to[0], *to[2:]) for t in some])
        return loss

    _uncompiled = torch._disable_dynamo(_step)  # a compiled function calls the step as it is

    @staticmethod
    def _in_order(lists) -> None:
        """The grads as the kernels take them: dense, of the parameter's type and order in memory."""
        for i, (p, g) in enumerate(zip(lists[0], lists[1])):
            if g.layout != torch.strided:
                raise RuntimeError("AdamW: sparse grads are not supported")
            if g.dtype != p.dtype:
                raise RuntimeError(f"AdamW: a grad of {g.dtype} for a parameter of {p.dtype}")
            if not _alike(g, p):
                lists[1][i] = torch.empty_like(p).copy_(g)

    @torch.no_grad()
    def moments(self) -> list:
        """(first, second) moment of every parameter, in the groups' order, as float32 values of its shape: the state itself
        where it has 32 bits, what the bytes stand for where it has 8, zeros before a first step."""
        out, codes, scales, second, at = [], [], [], [], []
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p)
                if not st:
                    out.append(tuple(torch.zeros_like(p, dtype=torch.float32) for _ in range(2)))
                elif st["exp_avg"].dtype == torch.float32:
                    out.append((st["exp_avg"], st["exp_avg_sq"]))
                else:
                    at.append(len(out))
                    out.append(None)
                    codes += [st["exp_avg"], st["exp_avg_sq"]]
                    scales += [st["exp_avg_scale"], st["exp_avg_sq_scale"]]
                    second += [False, True]
        values = ops.adamw_moments(codes, scales, second) if codes else []
        for i, k in enumerate(at):
            out[k] = values[2 * i], values[2 * i + 1]
        return out

    def load_state_dict(self, state_dict) -> None:
        """As torch's, with the state's own types kept (torch casts a state to its parameter's); a torch AdamW's state
        loads too, its moments in float32, but for forms of the step that this one does not have. A state that is refused
        leaves the optimizer as it was: the new state is made, and checked, before torch takes the groups over."""
        made: dict = {}
        before = self.register_load_state_dict_pre_hook(lambda opt, d: made.update(opt._state_made_of(d)))
        after = self.register_load_state_dict_post_hook(lambda opt: opt.state.update(made), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            before.remove()
            after.remove()

    @torch.inference_mode(False)
    def _state_made_of(self, state_dict) -> dict:
        """Each parameter's state from a state dict, or ValueError."""
        saved, new = state_dict["param_groups"], {}
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            return new  # (which torch refuses)
        for g, group in zip(saved, self.param_groups):
            for name in ("amsgrad", "maximize"):
                if g.get(name):
                    raise ValueError(f"AdamW: the state of a step with {name}")
            missing = {"lr", "betas", "eps", "weight_decay"} - g.keys()
            if missing:
                raise ValueError(f"AdamW: a group without {', '.join(sorted(missing))}")
            g = {"state_bits": 32, **g}
            self._check_group(g)
            if g.get("decoupled_weight_decay") is False and g["weight_decay"] != 0.0:
                raise ValueError("AdamW: the state of a step whose decay goes through its moments")
            for i, p in zip(g["params"], group["params"]):
                if state_dict["state"].get(i):  # (reading opt.state of a parameter before its first step leaves an empty one)
                    new[p] = self._one_state_made_of(state_dict["state"][i], p, g["state_bits"])
        return new

    @staticmethod
    def _one_state_made_of(src, p: torch.Tensor, bits: int) -> dict:
        moments = dict(zip(("exp_avg", "exp_avg_sq"), _STATE_DTYPES[bits]))
        scales = ("exp_avg_scale", "exp_avg_sq_scale") if bits == 8 else ()
        for name in (*moments, *scales):
            if not isinstance(src.get(name), torch.Tensor):
                raise ValueError(f"AdamW: a state without {name}")
        if "step" not in src or torch.as_tensor(src["step"]).numel() != 1:
            raise ValueError("AdamW: a state without its step count")
        st = {"step": torch.as_tensor(src["step"]).to(dtype=torch.float32, device=p.device, copy=True).reshape(())}
        for name, dtype in moments.items():
            t = src[name]
            if t.shape != p.shape or t.is_floating_point() != (dtype == torch.float32) \
                    or (dtype != torch.float32 and t.dtype != dtype):
                raise ValueError(f"AdamW: {name} of {t.dtype} and shape {tuple(t.shape)} does not fit a parameter of "
                                 f"shape {tuple(p.shape)} with moments in {bits} bits")
            st[name] = torch.empty_like(p, dtype=dtype, requires_grad=False)
            if bits == 8 and not (t.is_contiguous() and p.is_contiguous()) \
                    and t.stride() != st[name].stride():  # blocks are of elements next to each other in memory
                raise ValueError(f"AdamW: 8-bit {name} of strides {t.stride()} for a parameter of strides {p.stride()}")
            st[name].copy_(t)
        blocks = -(-p.numel() // ops.ADAMW_BLOCK)
        for name in scales:
            if src[name].shape != (blocks,) or not src[name].is_floating_point():
                raise ValueError(f"AdamW: {name} of {src[name].dtype} and shape {tuple(src[name].shape)}, not a scale for each "
                                 f"of {blocks} blocks")
            st[name] = src[name].to(dtype=torch.float32, device=p.device, copy=True)
        return st
