"""AdamW + gradient clipping of the training step as two HIP launches (csrc/optim.hip).

The reference trains with `torch.optim.AdamW(lr=1e-3, weight_decay=0.1)` behind Lightning's `gradient_clip_val: 5.0` (config yaml:117-120,
train.py:135-146).  Over RTFS-Net's 403 parameter tensors that pair is ~15 multi-tensor launches and a host-bound 2 ms at the end of every step;
`FusedAdamW.step(max_norm=5.0)` does the same arithmetic - total gradient norm, clip coefficient, in-place gradient scaling, decoupled weight decay,
moment updates, bias-corrected update, in torch.optim.AdamW's own operation order - with the clip coefficient formed on the device.

`FusedAdamW` is a `torch.optim.Optimizer`: param groups, `zero_grad`, `state_dict` / `load_state_dict` behave as usual and the per-parameter state
(`step`, `exp_avg`, `exp_avg_sq`) has torch.optim.AdamW's keys, so optimizer checkpoints interchange with it.  One group's hyper-parameters apply per
launch pair; parameters must be contiguous fp32 CUDA tensors (RTFS-Net's are).  `amsgrad`, `maximize`, sparse gradients: not supported (raise).

`clip_grad_norm_` is the clip alone (csrc/clip.hip), for any other optimizer and for fp32, bf16 and fp16 gradients.
"""
from __future__ import annotations

import array
import math
import operator

import torch

from . import lib

_CHUNK = 1024  # kOptChunk in csrc/optim.hip


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        if lr < 0.0 or eps < 0.0 or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or weight_decay < 0.0:
            raise ValueError("invalid AdamW hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._plans = {}

    # ---- per-group launch plan: static tables (parameters, state, sizes, chunk map) + a pinned row for the gradient pointers of the step ----
    def _plan(self, gi, ps):
        # the tables hold raw device addresses: a plan is valid for exactly these parameter objects AT these addresses (p.data = ..., module.to() and
        # re-sharding keep the Parameter object and move its storage) with these moment tensors
        key = tuple((id(p), p.data_ptr(), p.numel()) for p in ps)
        plan = self._plans.get(gi)
        if plan is not None and plan["key"] == key and all(self.state[p]["exp_avg"].data_ptr() == a and self.state[p]["exp_avg_sq"].data_ptr() == b
                                                           for p, a, b in zip(ps, plan["m_ptrs"], plan["v_ptrs"])):
            return plan
        dev = ps[0].device
        for p in ps:
            if p.dtype != torch.float32 or not p.is_cuda or p.device != dev or not p.is_contiguous():
                raise ValueError("FusedAdamW needs contiguous fp32 parameters on one HIP device")
            st = self.state[p]
            if len(st) == 0:
                st["step"] = torch.zeros((), dtype=torch.float32)  # host scalar per parameter, as torch.optim.AdamW's non-capturable path keeps it (a
                # tensor shared by all parameters would be incremented once per parameter by torch.optim.AdamW after a state_dict interchange)
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        sizes = [p.numel() for p in ps]
        chunks = [(i, s) for i, n in enumerate(sizes) for s in range(0, n, _CHUNK)]
        host = torch.zeros(5, len(ps), dtype=torch.int64)
        host[0] = torch.tensor([p.data_ptr() for p in ps], dtype=torch.int64)
        host[2] = torch.tensor([self.state[p]["exp_avg"].data_ptr() for p in ps], dtype=torch.int64)
        host[3] = torch.tensor([self.state[p]["exp_avg_sq"].data_ptr() for p in ps], dtype=torch.int64)
        host[4] = torch.tensor(sizes, dtype=torch.int64)
        plan = {"key": key, "dev": host.to(dev), "n_chunks": len(chunks), "n": len(ps),
                "chunks": torch.tensor(chunks, dtype=torch.int32).reshape(-1, 2).to(dev), "sqnorm": torch.zeros(1, dtype=torch.float64, device=dev),
                "m_ptrs": [self.state[p]["exp_avg"].data_ptr() for p in ps], "v_ptrs": [self.state[p]["exp_avg_sq"].data_ptr() for p in ps]}
        self._plans[gi] = plan
        return plan

    @torch.no_grad()
    def step(self, closure=None, max_norm=None):
        """One AdamW step.  `max_norm`: clip the total 2-norm of ALL gradients handed to this optimizer to it first (torch.nn.utils.clip_grad_norm_'s
        arithmetic, the gradients are left scaled in place); None: no clipping.  With several param groups the norm is taken over all of them."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for gi, group in enumerate(self.param_groups):
            if group.get("amsgrad") or group.get("maximize"):
                raise NotImplementedError("FusedAdamW: amsgrad / maximize are not implemented")
            with_grad = [p for p in group["params"] if p.grad is not None]
            if not with_grad:
                continue
            # one launch applies ONE pair of bias corrections: parameters whose step counts differ (a parameter that first received a gradient later, one
            # skipped under DDP's find_unused_parameters, interchanged optimizer states) go in separate launches, as torch.optim.AdamW corrects per parameter
            by_step = {}
            for p in with_grad:
                st = self.state[p]
                by_step.setdefault(float(st["step"]) if len(st) else 0.0, []).append(p)
            for si, (_, ps) in enumerate(sorted(by_step.items())):
                work.append(self._stage(group, (gi, si, len(by_step)), ps))
        if not work:
            return loss
        clip = max_norm is not None
        if clip:
            if len(work) == 1:
                group, ps, plan = work[0]
                d = plan["dev"]
                lib.call("rtfs_grad_sqnorm", d[0], d[1], d[2], d[3], d[4], plan["chunks"], plan["n_chunks"], plan["sqnorm"])
                sq = plan["sqnorm"]
            else:  # several launches: one norm over all of them (the kernel zeroes its output, so the partial sums are added here on the device)
                sq = None
                for group, ps, plan in work:
                    d = plan["dev"]
                    lib.call("rtfs_grad_sqnorm", d[0], d[1], d[2], d[3], d[4], plan["chunks"], plan["n_chunks"], plan["sqnorm"])
                    sq = plan["sqnorm"].clone() if sq is None else sq + plan["sqnorm"]
        for group, ps, plan in work:
            torch._foreach_add_([self.state[p]["step"] for p in ps], 1)
            k = float(self.state[ps[0]]["step"])
            b1, b2 = group["betas"]
            d = plan["dev"]
            lib.call("rtfs_adamw_clip_step", d[0], d[1], d[2], d[3], d[4], plan["chunks"], plan["n_chunks"], sq if clip else plan["sqnorm"],
                     float(max_norm) if clip else 0.0, float(group["lr"]), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"]),
                     1.0 - b1 ** k, math.sqrt(1.0 - b2 ** k))
            # the kernel wrote the parameters, moments and gradients through raw pointers: tell autograd (and everything keyed on version counters -
            # the kernel-layout weight copies of rtfs_net_amd.models are rebuilt when a parameter's counter moves) that these tensors changed
            torch.autograd.graph.increment_version(ps)
            torch.autograd.graph.increment_version([p.grad for p in ps])
            torch.autograd.graph.increment_version([self.state[p]["exp_avg"] for p in ps] + [self.state[p]["exp_avg_sq"] for p in ps])
        return loss

    def _stage(self, group, slot, ps):
        """plan + this step's gradient-pointer row of one launch (the parameters of `group` that share a step count)"""
        plan = self._plan(slot, ps)
        # the gradient tensors are new objects every step: their pointers go up in a FRESH pinned row (the caching host allocator keeps a block until
        # the copy that reads it has run - the host may be several steps ahead of the device, a reused staging row would be overwritten under it)
        row = torch.empty(plan["n"], dtype=torch.int64, pin_memory=True)
        g_np = row.numpy()
        for i, p in enumerate(ps):
            g = p.grad
            if g.is_sparse or g.dtype != torch.float32 or not g.is_contiguous() or g.device != p.device:
                raise ValueError("FusedAdamW needs dense contiguous fp32 gradients on the parameters' device")
            g_np[i] = g.data_ptr()
        plan["dev"][1].copy_(row, non_blocking=True)
        return group, ps, plan


_CLIP_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0):
    """torch.nn.utils.clip_grad_norm_ as HIP launches: the norm of all gradients of `parameters` (a tensor or an iterable of them; those without a gradient are
    passed over) taken as one vector, and every gradient scaled in place by min(1, max_norm / (norm + 1e-6)).

    norm_type 2 or inf.  fp32, bf16 and fp16 gradients in any mix, dense in any order of their dimensions, without memory in common (refused), on one device; the
    same tensor listed twice counts once.  The norm's squares are summed in fp64 in a fixed order.  -> the norm before clipping, a 0-dim fp32 tensor on the gradients'
    device (nothing is copied to the host; a norm that is not finite is not an error: a NaN goes through to every gradient).  Every gradient is written, also where
    the factor is 1."""
    max_norm, norm_type = float(max_norm), float(norm_type)
    if not max_norm >= 0.0:
        raise ValueError("clip_grad_norm_: max_norm must not be negative")
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"clip_grad_norm_: norm_type 2 or inf, got {norm_type}")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros(())
    # one pass per question over all tensors: a small model's hundreds of them are host time, not device time
    kinds, devices = set(map(operator.attrgetter("dtype"), grads)), set(map(torch.Tensor.get_device, grads))
    if not kinds <= _CLIP_TYPES.keys() or -1 in devices or set(map(operator.attrgetter("layout"), grads)) != {torch.strided}:
        raise ValueError("clip_grad_norm_: gradients must be dense fp32, bf16 or fp16 HIP tensors")
    if len(devices) > 1:
        raise ValueError(f"clip_grad_norm_: gradients on devices {sorted(devices)}")
    if not all(map(torch.Tensor.is_contiguous, grads)) and not all(g.is_contiguous() or _fills_its_span(g) for g in grads):
        raise ValueError("clip_grad_norm_: a gradient has gaps or overlaps in memory")
    device = grads[0].device
    at = array.array("q", map(torch.Tensor.data_ptr, grads))
    if len(set(at)) != len(at):  # the same tensor more than once, or empty ones
        grads = [g for g in {id(g): g for g in grads}.values() if g.numel()]
        at = array.array("q", map(torch.Tensor.data_ptr, grads))
        if len(set(at)) != len(at):
            raise ValueError("clip_grad_norm_: two gradients start at the same address")
    sizes = array.array("q", map(torch.Tensor.numel, grads))
    if not any(sizes):
        return torch.zeros((), device=device)
    types = [_CLIP_TYPES[g.dtype] for g in grads] if len(kinds) > 1 else [_CLIP_TYPES[grads[0].dtype]] * len(grads)
    types = array.array("i", types)
    norm = torch.empty((), device=device)
    listed = len(grads) + (sum(sizes) >> 30)  # a tensor of over 2^30 elements is listed in pieces
    parts = torch.empty(2561 + 512 * (listed // 240), dtype=torch.float64, device=device)
    try:
        lib.call("rtfs_clip_grad_norm", at.buffer_info()[0], sizes.buffer_info()[0], types.buffer_info()[0], len(grads), max_norm, 2 if norm_type == 2.0 else 0, parts,
                 parts.numel(), norm)
    except RuntimeError:
        spans = sorted((a, a + g.nbytes) for a, g in zip(at, grads) if g.numel())
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("clip_grad_norm_: two gradients have memory in common") from None
        raise
    torch.autograd.graph.increment_version(grads)  # written through their addresses
    return norm


def _fills_its_span(t):
    """whether t's elements are a gap-free stretch of memory, in whatever order of its dimensions"""
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True
