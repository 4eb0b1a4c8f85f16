"""AdamW over all tensors of a parameter group in one launch, with moments in 32 or in 8 bits.

Takes the place of torch.optim.Adam / AdamW (the reference: src/train.py:104-105) where parameters are many separate
tensors, as on the drop-in module route; the fused TrainStep has its own update over one flat buffer.
"""
from __future__ import annotations

from array import array
from copy import deepcopy
from operator import is_
from typing import Dict, List, Optional, Tuple

import torch

from . import ops
from ._lib import direct

__all__ = ["AdamW"]

F32 = torch.float32
BLOCK = 256           # elements that share a scale of the 8-bit moments; every tensor starts on a block of its own
CHUNK = 4096          # elements per workgroup
CODES = torch.float8_e4m3fn


class _Bank:
    """The tensors of one group that share an element type: their moments in flat buffers, the kernel's job table."""

    def __init__(self, params: List[torch.Tensor], bits: int):
        self.params, self.bits = params, bits
        self.dtype, self.device = params[0].dtype, params[0].device
        self.sizes = [p.numel() for p in params]
        self.starts, blocks, first = [], 0, [0]
        for n in self.sizes:
            self.starts.append(blocks * BLOCK)
            blocks += -(-n // BLOCK)
            first.append(first[-1] + -(-n // CHUNK))
        self.first = array("i", first)
        begin = torch.tensor(first)
        tensor = torch.repeat_interleave(torch.arange(len(params)), begin.diff())
        chunks = torch.stack((tensor, torch.arange(first[-1]) - begin[tensor]), 1)          # of a workgroup: (tensor, chunk of it)
        with torch.cuda.device(self.device):
            self.map = (chunks if first[-1] else torch.zeros(1, 2)).to(torch.int32).to(self.device)
            self.steps = torch.zeros(len(params), dtype=torch.int32, device=self.device)
            self.coef = torch.zeros(len(params), 2, dtype=F32, device=self.device)
            many = max(blocks, 1) * BLOCK
            self.flat: Dict[str, torch.Tensor] = {}
            if bits == 32:
                for name in ("exp_avg", "exp_avg_sq"):
                    self.flat[name] = torch.zeros(many, dtype=F32, device=self.device)
            else:
                for name in ("exp_avg", "exp_avg_sq_root"):
                    self.flat[name] = torch.zeros(many, dtype=torch.uint8, device=self.device).view(CODES)
                    self.flat[name + "_scale"] = torch.zeros(many // BLOCK, dtype=F32, device=self.device)
        self.table: Optional[torch.Tensor] = None
        self.captured = False                         # whether a captured step reads the table
        self.kept: List[torch.Tensor] = []            # earlier tables that one reads
        self.at = array("q")
        self.elements = array("q", self.sizes)
        self.grads = array("q", bytes(8 * len(params)))

    def views(self) -> List[Dict[str, torch.Tensor]]:
        """The state of each tensor, as views of the flat buffers."""
        blocks = [-(-n // BLOCK) for n in self.sizes]
        pieces = [m for n, b in zip(self.sizes, blocks) for m in (n, b * BLOCK - n)]        # tensors and what lies between
        out = [{"step": t} for t in self.steps.unbind()]
        for name, buf in self.flat.items():
            if name.endswith("_scale"):
                parts = buf[:sum(blocks)].split(blocks)
            else:
                parts = [t.view(p.shape) for t, p in zip(buf[:sum(pieces)].split(pieces)[::2], self.params)]
            for state, t in zip(out, parts):
                state[name] = t
        return out

    def bind(self, at):
        """Build the job table for parameters at these addresses."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the parameters moved (or this is the first step); run a step before the capture")
        for p, n in zip(self.params, self.sizes):
            _check_param(p)
            if p.numel() != n or p.dtype is not self.dtype or p.device != self.device:
                raise RuntimeError("AdamW: a parameter changed its size, type or device after the optimizer's first step")
        width = self.params[0].element_size()
        spans = sorted((p, p + n * width) for p, n in zip(at, self.sizes) if n)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters share memory")
        one = 4 if self.bits == 32 else 1                     # bytes of a moment
        m, v = (self.flat[k].data_ptr() for k in self.flat if not k.endswith("_scale"))
        ms, vs = (self.flat[k].data_ptr() for k in self.flat if k.endswith("_scale")) if self.bits == 8 else (0, 0)
        rows = [(p, m + s * one, v + s * one, ms and ms + s // BLOCK * 4, vs and vs + s // BLOCK * 4, n)
                for p, s, n in zip(at, self.starts, self.sizes)]
        rows = torch.tensor(rows, dtype=torch.int64)
        if self.table is None or self.captured:
            if self.captured:
                self.kept.append(self.table)
            self.table, self.captured = rows.to(self.device), False
        else:                                                     # (on the stream of this step, so behind the one before it)
            self.table.copy_(rows)
        self.at = at

    def gradients(self):
        """Addresses of the gradients in self.grads (0: none); returns the copies that stand in for those that are not
        contiguous.  Follows parameters that moved."""
        if direct().gradients(self.params, self.at, self.elements, self.grads):
            return ()
        at = array("q", [p.data_ptr() for p in self.params])
        if at != self.at or any(p.numel() != n or not p.is_contiguous() or p.is_neg() for p, n in zip(self.params, self.sizes)):
            self.bind(at)                                         # (which refuses a parameter that lies there otherwise)
        kept = []
        for i, (p, n) in enumerate(zip(self.params, self.sizes)):
            g = p.grad
            if g is None:
                self.grads[i] = 0
                continue
            if g.dtype is not self.dtype or g.layout is not torch.strided:
                raise TypeError(f"AdamW: gradients are dense and of their parameter's type, not {g.layout} {g.dtype}")
            if g.numel() != n or g.device != self.device:
                raise ValueError(f"AdamW: a gradient of {g.numel()} elements on {g.device} for a parameter of {n} on {self.device}")
            if not g.is_contiguous() or g.is_neg():
                g = g.contiguous().resolve_neg()
                kept.append(g)
            self.grads[i] = g.data_ptr()
        torch.autograd.graph.increment_version([p for p in self.params if p.grad is not None])
        return kept


def _check_param(p: torch.Tensor):
    if p.device.type != "cuda":
        raise RuntimeError("AdamW: parameters must be on a ROCm device (call .cuda()); there is no CPU path")
    if p.dtype not in (F32, torch.bfloat16):
        raise TypeError(f"AdamW: parameters are fp32 or bf16, not {p.dtype}")
    if not p.is_contiguous() or p.is_neg():
        raise ValueError("AdamW: parameters must be contiguous")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay), one launch per parameter group and element type.

    params: tensors or groups of fp32 or bf16 parameters on a ROCm device, contiguous.  state_bits: 32 keeps both moments
    in fp32; 8 keeps them in e4m3 codes with an fp32 scale per 256 elements - the first moment, and the square root of
    the second - a quarter of the memory and of the state's traffic.  Sums are fp32 either way; bf16 parameters are
    rounded once per step.

    Step counts live on the device and only tensors with a gradient are counted and updated, so a step may be captured
    into a HIP graph once one step has run eagerly (the replays read the gradients where they were at the capture, and
    the learning rate is captured by value).  State dicts hold per tensor `step` and `exp_avg`, `exp_avg_sq` (as
    torch.optim.AdamW's), or the codes `exp_avg`, `exp_avg_sq_root` and their `..._scale`: value = code * scale."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32):
        if state_bits not in (32, 8):
            raise ValueError(f"AdamW: moments have 32 or 8 bits, not {state_bits}")
        self._check_values(lr, betas, eps, weight_decay)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))
        for group in self.param_groups:
            self._check_values(group["lr"], group["betas"], group["eps"], group["weight_decay"])
        self._banks: Dict[int, Tuple[List[torch.Tensor], List[_Bank]]] = {}      # of a group: its parameters and their banks

    @staticmethod
    def _check_values(lr, betas, eps, weight_decay):
        if isinstance(lr, torch.Tensor):
            raise TypeError("AdamW: lr is a number, not a tensor")
        AdamW._check_numbers(lr, betas, eps, weight_decay)

    @staticmethod
    def _check_numbers(lr, betas, eps, weight_decay):
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("AdamW: lr, eps and weight_decay are not negative, betas lie in [0, 1)")

    def __setstate__(self, state):
        super().__setstate__(state)
        self._banks = {}

    def _group_banks(self, gi: int, group) -> List[_Bank]:
        if gi in self._banks:
            known, banks = self._banks[gi]
            if len(known) != len(group["params"]) or not all(map(is_, known, group["params"])):
                if len(known) != len(group["params"]) or set(map(id, known)) != set(map(id, group["params"])):
                    raise RuntimeError("AdamW: a group's parameters changed after its first step; use add_param_group")
                self._banks[gi] = list(group["params"]), banks              # (the same ones in another order)
            return banks
        if len({id(p) for p in group["params"]}) != len(group["params"]):
            raise ValueError("AdamW: the same parameter twice in one group")
        if group["state_bits"] not in (32, 8):
            raise ValueError(f"AdamW: moments have 32 or 8 bits, not {group['state_bits']}")
        kinds: Dict[tuple, List[torch.Tensor]] = {}
        for p in group["params"]:
            _check_param(p)
            kinds.setdefault((p.dtype, p.device), []).append(p)
        if kinds and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: run a step before the capture")
        banks = [_Bank(ps, group["state_bits"]) for ps in kinds.values()]
        states = [(p, views) for bank in banks for p, views in zip(bank.params, bank.views())]
        for p, views in states:
            if self.state.get(p):
                self._check_state(self.state[p], views)
                self._take(self.state[p], views)
        self.state.update(states)
        self._banks[gi] = list(group["params"]), banks
        return banks

    @staticmethod
    def _check_state(saved, views):
        if set(saved) != set(views):
            raise ValueError(f"AdamW: state with {sorted(saved)}, wanted {sorted(views)} (moments of another number of bits?)")
        for name, dst in views.items():
            src = torch.as_tensor(saved[name])
            if src.numel() != dst.numel() or (name != "step" and src.shape != dst.shape):
                raise ValueError(f"AdamW: state `{name}` has shape {tuple(src.shape)}, not {tuple(dst.shape)}")
            if name != "step" and (src.dtype is CODES) != (dst.dtype is CODES):
                raise ValueError(f"AdamW: state `{name}` is {src.dtype}, not {dst.dtype}")

    @staticmethod
    def _take(saved, views):
        for name, dst in views.items():
            dst.copy_(torch.as_tensor(saved[name]).reshape(dst.shape))

    def flat_state(self) -> List[Dict[str, torch.Tensor]]:
        """The moments of all tensors in one buffer per kind - one dict per group and element type, in the order of the
        groups.  Tensors follow one another, each from a multiple of 256 elements on; what lies between is zero."""
        return [bank.flat for gi, group in enumerate(self.param_groups) for bank in self._group_banks(gi, group)]

    def load_state_dict(self, state_dict):
        """Copies the saved moments into this optimizer's buffers (so a captured step goes on with them), and all entries of the
        groups but their parameters; registered hooks run before and after.  A state that does not fit changes nothing."""
        state_dict = dict(state_dict)                             # (a hook may change its own)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            if changed is not None:
                state_dict = changed
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("AdamW: the state dict has other parameter groups")
        for mine, theirs in zip(self.param_groups, groups):
            if theirs.get("state_bits", 32) != mine["state_bits"]:
                raise ValueError(f"AdamW: a state of {theirs.get('state_bits', 32)} bits for an optimizer of {mine['state_bits']}")
            self._check_values(theirs["lr"], theirs["betas"], theirs["eps"], theirs["weight_decay"])
            if theirs.get("maximize") or theirs.get("amsgrad"):
                raise ValueError("AdamW: there is no maximize and no amsgrad")
        for gi, mine in enumerate(self.param_groups):
            self._group_banks(gi, mine)
        states = [(state_dict["state"].get(index), self.state[p])
                  for mine, theirs in zip(self.param_groups, groups) for index, p in zip(theirs["params"], mine["params"])]
        for saved, views in states:                               # (everything is looked at before anything is written)
            if saved:
                self._check_state(saved, views)
        for mine, theirs in zip(self.param_groups, groups):
            mine.update((key, deepcopy(value)) for key, value in theirs.items() if key not in ("params", "state_bits"))
            mine["betas"] = tuple(mine["betas"])
        for saved, views in states:
            if saved:
                self._take(saved, views)
            else:
                for t in views.values():
                    (t.view(torch.uint8) if t.dtype is CODES else t).zero_()
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            self._check_numbers(group["lr"], group["betas"], group["eps"], group["weight_decay"])
        work = [(group, bank) for gi, group in enumerate(self.param_groups) for bank in self._group_banks(gi, group)]
        kept = [bank.gradients() for _, bank in work]              # noqa: F841  (alive until the launches; all refusals come first)
        for group, bank in work:
            bank.captured |= torch.cuda.is_current_stream_capturing()
            ops.adamw_jobs(bank.table, bank.map, bank.grads, bank.first, bank.steps, bank.coef, float(group["lr"]),
                           group["betas"][0], group["betas"][1], group["eps"], group["weight_decay"], bank.dtype, bank.bits)
        return loss
