"""Fused optimizer tail of step_batch (/root/reference/utils/train_step.py:56-63):

    scaler.unscale_(opt); clip_grad_norm_(model.parameters(), grad_clip); scaler.step(opt)

with the AdamW that /root/reference/utils/builders.py:143-146 builds.  `FusedAdamW` IS a
`torch.optim.AdamW` (same constructor, param_groups, state and state_dict layout, LR schedulers and step
hooks work unchanged); only `step()` differs: one multi-tensor HIP kernel per 40 tensors updates
parameter, exp_avg and exp_avg_sq in a single pass (28 B/parameter instead of torch's ~10 foreach
passes), and `clip_and_step()` folds clip_grad_norm_ into it: one pass for the global L2 norm, the
clip coefficient stays on the device (no host sync) and is applied while the update reads the gradient.

Anything the kernels do not cover (amsgrad, maximize, capturable, tensor lr, non-fp32 / CPU / sparse /
non-contiguous tensors) takes torch's own path, so behaviour never silently differs.

`state_bits=8` holds both moments in 8 bits (64 elements share an exponent, stochastic rounding; ops.adamw8_step): 2.03
bytes of state per parameter instead of 8 and 16 bytes of traffic per parameter and step instead of 28.  The state then is
uint8 (`exp_avg`, `exp_avg_sq` in the parameter's shape, `exp_avg_e`, `exp_avg_sq_e` one per 64 elements); checkpoints of
either kind load into an optimizer of either kind, and no other optimizer loads 8-bit ones (a group without parameters at
the end of the state_dict's param_groups keeps them out).  There is no torch path behind it: what the kernel does not cover raises.
"""
from typing import Iterable, Optional

import torch

from . import ops
from ._lib import UNetHipError

_STATE8 = ("exp_avg", "exp_avg_sq", "exp_avg_e", "exp_avg_sq_e")
_MARK8 = {"params": [], "state_bits": 8}         # last entry of param_groups in a state_dict that holds 8-bit state


class FusedAdamW(torch.optim.AdamW):
    def __init__(self, params, *args, state_bits: int = 32, state_seed: int = 0, **kwargs):
        """state_bits: 32 or 8; state_seed: seed of the 8-bit moments' stochastic rounding."""
        if state_bits not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits must be 8 or 32 (got {state_bits!r})")
        super().__init__(params, *args, **kwargs)
        self.state_bits, self.state_seed = state_bits, int(state_seed)
        self._slot8 = {}            # parameter -> (its arena: the four flat buffers, first block, its views)
        self._loaded8 = False       # 32 bits: the state may hold 8-bit entries
        if state_bits == 8:
            for g in self.param_groups:
                if not self._group_ok(g):
                    raise ValueError("FusedAdamW: state_bits=8 serves plain AdamW only (no amsgrad, maximize, capturable, "
                                     "differentiable, fused, tensor lr)")
                if not self._betas8_ok(g):
                    raise ValueError("FusedAdamW: 8-bit moments follow betas up to 1 - 2^-17")
        self._mt_ws = {}            # device -> (partials fp64, norm_out fp32[2])
        self._pending_clip = None
        self._clip_norm = None
        self._vetoable = []         # parameters whose step count the last fused step() advanced under a device-side veto

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "state_seed": self.state_seed}

    def __setstate__(self, state):
        """Of a copy or a pickle, and of load_state_dict: workspaces and flat buffers are not part of the state."""
        super().__setstate__(state)
        for k, v in (("state_bits", 32), ("state_seed", 0), ("_mt_ws", {}), ("_pending_clip", None), ("_clip_norm", None), ("_vetoable", [])):
            self.__dict__.setdefault(k, v)
        self._slot8 = {}
        self._loaded8 = any("exp_avg_e" in st for st in self.state.values())

    # ------------------------------------------------------------------ helpers
    @staticmethod
    def _tensor_ok(t: torch.Tensor) -> bool:
        return t.is_cuda and t.dtype == torch.float32 and not t.is_sparse and t.is_contiguous()

    @staticmethod
    def _group_ok(g) -> bool:
        return not (g.get("amsgrad") or g.get("maximize") or g.get("capturable") or g.get("differentiable") or g.get("fused")
                    or isinstance(g["lr"], torch.Tensor))

    @staticmethod
    def _betas8_ok(g) -> bool:
        return all(0 <= b and 1 - b >= ops.MOMENT8_LEAST for b in g["betas"])

    def _ws(self, device, nblocks):
        ws = self._mt_ws.get(device)
        if ws is None or ws[0].numel() < nblocks:
            ws = (torch.empty(max(nblocks, 1024), dtype=torch.float64, device=device),
                  torch.empty(2, dtype=torch.float32, device=device))
            self._mt_ws[device] = ws
        return ws

    def _init_states(self, params):
        """Adam's lazy state (torch.optim.Adam._init_group) for every parameter of the group that has a gradient and no
        state yet: the moments are views of ONE zeroed buffer per moment (each on a 256-byte boundary) instead of two
        zeros_like launches per parameter (164 fills in the first step of the 4-level U-Net)."""
        todo = [p for p in params if p.grad is not None and len(self.state[p]) == 0 and self._tensor_ok(p)]
        offs, total = [], 0
        for p in todo:
            offs.append(total)
            total += (p.numel() + 63) // 64 * 64
        flats = {}
        for p, off in zip(todo, offs):
            if p.device not in flats:
                flats[p.device] = (torch.zeros(total, dtype=torch.float32, device=p.device),
                                   torch.zeros(total, dtype=torch.float32, device=p.device))
            m, v = flats[p.device]
            st = self.state[p]
            st["step"] = torch.tensor(0.0, dtype=torch.get_default_dtype())
            st["exp_avg"] = m[off:off + p.numel()].view_as(p)
            st["exp_avg_sq"] = v[off:off + p.numel()].view_as(p)
        for p in params:                                    # anything the fused path will refuse anyway: torch's own layout
            if p.grad is not None and len(self.state[p]) == 0:
                st = self.state[p]
                st["step"] = torch.tensor(0.0, dtype=torch.get_default_dtype())
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)

    def _in_arena(self, p) -> bool:
        slot, st = self._slot8.get(p), self.state[p]
        return slot is not None and all(st.get(k) is v for k, v in zip(_STATE8, slot[2]))

    def _adopt8(self, params):
        """Moves the state of `params` into one set of flat buffers in which every tensor starts on a block: empty state becomes
        zeros, 8-bit state (of a checkpoint) is copied, 32-bit state is rounded to nearest."""
        first, total = [], 0
        for p in params:
            first.append(total)
            total += ops.moment8_blocks(p.numel())
        dev = params[0].device
        arena = tuple(torch.zeros(total * w, dtype=torch.uint8, device=dev) for w in (64, 64, 1, 1))
        for p, f in zip(params, first):
            st, n, b = self.state[p], p.numel(), ops.moment8_blocks(p.numel())
            new = {k: a[f * w:f * w + (n if w == 64 else b)] for k, a, w in zip(_STATE8, arena, (64, 64, 1, 1))}
            if len(st) == 0:
                st["step"] = torch.tensor(0.0, dtype=torch.get_default_dtype())
            elif "exp_avg_e" in st:
                for k in _STATE8:
                    new[k].copy_(st[k].reshape(-1))
            else:
                for k, signed in (("exp_avg", True), ("exp_avg_sq", False)):
                    ops.moment8_encode(st[k].to(device=dev, dtype=torch.float32).contiguous().view(-1), signed, new[k], new[k + "_e"])
            for k in _STATE8:
                st[k] = new[k].view(p.shape) if k in ("exp_avg", "exp_avg_sq") else new[k]
            self._slot8[p] = (arena, f, tuple(st[k] for k in _STATE8))

    def _to_32_bits(self, params):
        """State of an 8-bit checkpoint in a 32-bit optimizer: the values it stands for."""
        for p in params:
            st = self.state[p]
            for k, signed in (("exp_avg", True), ("exp_avg_sq", False)):
                codes, e = (st[x].to(device=p.device, dtype=torch.uint8).contiguous().view(-1) for x in (k, k + "_e"))
                st[k] = ops.moment8_decode(codes, e, signed).view(p.shape)
            for k in ("exp_avg_e", "exp_avg_sq_e"):
                del st[k]

    def state_dict(self):
        """As torch's.  8-bit state comes with one more group, without parameters, that says so: other optimizers then refuse the
        state (another number of groups) instead of taking the codes for moments."""
        sd = super().state_dict()
        if any("exp_avg_e" in st for st in self.state.values()):
            sd["param_groups"] = sd["param_groups"] + [dict(_MARK8)]
        return sd

    def load_state_dict(self, state_dict):
        groups = [g for g in state_dict["param_groups"] if dict(g) != _MARK8]
        super().load_state_dict({**state_dict, "param_groups": groups})
        if self.state_bits == 8:                            # (a checkpoint read straight to the GPU has its step counts there)
            for st in self.state.values():
                if isinstance(st.get("step"), torch.Tensor):
                    st["step"] = st["step"].cpu()
        for st in self.state.values():                      # torch casts every entry to the parameter's dtype: whole numbers survive
            if "exp_avg_e" in st:
                for k in _STATE8:
                    st[k] = st[k].to(torch.uint8)

    def _prepare8(self, params):
        """Checks that the 8-bit kernel covers these parameters and brings their state into flat buffers."""
        if not params:
            return
        for p in params:
            if not (self._tensor_ok(p) and self._tensor_ok(p.grad)):
                raise UNetHipError("FusedAdamW(state_bits=8) needs contiguous fp32 parameters and gradients on the GPU")
        if len({p.device for p in params}) > 1:
            raise UNetHipError("FusedAdamW(state_bits=8): parameters on more than one device")
        if torch.cuda.is_current_stream_capturing():        # (before step counts and gradients have changed)
            raise UNetHipError("FusedAdamW(state_bits=8): a step cannot be captured into a graph, its step number is a host value")
        todo = [p for p in params if not self._in_arena(p)]
        if todo:
            self._adopt8(todo)

    def _collect(self):
        """-> [(group, step, params, grads, exp_avg, exp_avg_sq)] with the state initialised as
        torch.optim.Adam._init_group does, or None when some tensor needs torch's own path."""
        work = []
        device = None
        if self.state_bits == 8:
            self._prepare8([p for group in self.param_groups for p in group["params"] if p.grad is not None])
        elif self._loaded8:
            self._to_32_bits([p for group in self.param_groups for p in group["params"] if "exp_avg_e" in self.state.get(p, ())])
            self._loaded8 = False
        for group in self.param_groups:
            if not self._group_ok(group):
                if self.state_bits == 8:
                    raise UNetHipError("FusedAdamW(state_bits=8) serves plain AdamW only")
                return None
            if self.state_bits == 8 and not (group["lr"] >= 0 and group["eps"] >= 0 and self._betas8_ok(group)):
                raise UNetHipError("FusedAdamW(state_bits=8): bad hyper-parameters")        # (before another group is stepped)
            by_step = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not (self._tensor_ok(p) and self._tensor_ok(p.grad)):
                    return None
                if device is None:
                    device = p.device
                elif p.device != device:
                    return None
                st = self.state[p]
                if len(st) == 0:
                    self._init_states(group["params"])
                if self.state_bits == 32 and not (self._tensor_ok(st["exp_avg"]) and self._tensor_ok(st["exp_avg_sq"])):
                    if "exp_avg_e" not in st:
                        return None
                    self._to_32_bits([p])               # (8-bit state that did not come by load_state_dict)
                step_t = st["step"]
                if not isinstance(step_t, torch.Tensor) or step_t.is_cuda:
                    if self.state_bits == 8:
                        raise UNetHipError("FusedAdamW(state_bits=8): the step count must be a host tensor")
                    return None
                by_step.setdefault(int(step_t.item()), []).append(p)
            for step, plist in by_step.items():
                work.append((group, step, plist))
        return work

    def _by_arena(self, plist):
        """-> [(the four buffers, the parameters whose state they hold)]; one entry unless parameters joined later."""
        groups = {}
        for p in plist:
            arena = self._slot8[p][0]
            groups.setdefault(id(arena), (arena, []))[1].append(p)
        return list(groups.values())

    # ------------------------------------------------------------------ API
    def clip_and_step(self, parameters: Iterable[torch.Tensor], max_norm: float, grad_scale: float = 1.0,
                      veto: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """clip_grad_norm_(parameters, max_norm) followed by step(), without a host sync.
        Returns the total gradient norm (0-dim device tensor), as clip_grad_norm_ does.
        grad_scale: the .grad tensors hold 1/grad_scale times the gradients (data parallel hands over the all-reduced
        SUM with grad_scale = 1/world); norm, clipping and update are those of grad_scale*grad, and the clipped
        gradients written back are the averaged ones.
        veto: one fp32 device element; if it is > 0 when the update kernel runs, parameters, moments and gradients are left
        untouched (step_batch passes the loss kernel's illegal-label counter; only the fused path honours it)."""
        if isinstance(parameters, torch.Tensor):
            parameters = [parameters]
        self._pending_clip = ([p for p in parameters if p.grad is not None], float(max_norm), float(grad_scale))
        self._clip_norm = None
        self._veto = veto
        try:
            self.step()
        finally:
            self._pending_clip = None
            self._veto = None
        return self._clip_norm

    def undo_vetoed_step(self):
        """The veto element was > 0 when the last clip_and_step() ran, i.e. its update kernels did nothing: take back the
        host-side step counts they were launched with.  The caller (step_batch) learns the flag at its host sync."""
        for p in self._vetoable:
            self.state[p]["step"] -= 1
        self._vetoable = []

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        clip = self._pending_clip
        self._pending_clip = None
        clip_ok = clip is None or all(self._tensor_ok(p.grad) for p in clip[0])
        if self.state_bits == 8 and not clip_ok:        # (also gradients that this optimizer does not own; before anything changes)
            raise UNetHipError("FusedAdamW(state_bits=8) clips contiguous fp32 gradients on the GPU only")
        work = self._collect()
        if clip is not None and clip[2] != 1.0 and (work is None or not clip_ok or len({p.grad.device for p in clip[0]}) > 1
                                                    or {id(p) for p in clip[0]} != {id(p) for _, _, pl in (work or []) for p in pl}):
            for p in clip[0]:                           # a path below that cannot fold the scale: apply it first
                p.grad.mul_(clip[2])
            clip = (clip[0], clip[1], 1.0)
        if work is None or not clip_ok:
            if clip is not None and clip[0]:
                self._clip_norm = torch.nn.utils.clip_grad_norm_(clip[0], clip[1])
            super().step()
            return loss
        norm_out = None
        if clip is not None and clip[0]:
            grads = [p.grad for p in clip[0]]
            dev = grads[0].device
            if any(g.device != dev for g in grads):
                self._clip_norm = torch.nn.utils.clip_grad_norm_(clip[0], clip[1])
            else:
                partials, norm_out = self._ws(dev, ops.mt_blocks([g.numel() for g in grads]))
                ops.grad_norm(grads, clip[1], partials, norm_out, clip[2])
                self._clip_norm = norm_out[0].clone()
                stepped = {id(p) for _, _, plist in work for p in plist}
                for p in clip[0]:                       # clipped but not stepped by this optimizer
                    if id(p) not in stepped:
                        p.grad.mul_(norm_out[1])
                if work and work[0][2][0].device != dev:
                    for _, _, plist in work:            # norm lives on another device than the parameters
                        for p in plist:
                            p.grad.mul_(norm_out[1].to(p.device))
                    norm_out = None
        veto = getattr(self, "_veto", None)
        self._vetoable = []
        for group, step, plist in work:
            beta1, beta2 = group["betas"]
            if self.state_bits == 8:
                for arena, pl in self._by_arena(plist):
                    ops.adamw8_step(pl, [p.grad for p in pl], *arena, norm_out, norm_out is not None,
                                    group["lr"], beta1, beta2, group["eps"], group["weight_decay"], step + 1,
                                    seed=self.state_seed, veto=veto, first_block=[self._slot8[p][1] for p in pl])
            else:
                ops.adamw_step(plist, [p.grad for p in plist], [self.state[p]["exp_avg"] for p in plist],
                               [self.state[p]["exp_avg_sq"] for p in plist], norm_out, norm_out is not None,
                               group["lr"], beta1, beta2, group["eps"], group["weight_decay"], step + 1,
                               veto=veto)
            for p in plist:                     # (behind the call: one that is refused leaves the counts alone)
                self.state[p]["step"] += 1
            if veto is not None:
                self._vetoable += plist
            # the kernels write through raw pointers: tell autograd (and the engines' packed-weight caches)
            touched = plist + [self.state[p][k] for k in (_STATE8 if self.state_bits == 8 else _STATE8[:2]) for p in plist]
            if norm_out is not None:
                touched += [p.grad for p in plist]
            torch.autograd.graph.increment_version(touched)
        return loss
