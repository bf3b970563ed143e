"""Data-parallel step for LoRA fine-tuning: one process per GPU, frames sharded by rank, and ONE
exchange step per iteration -- a mean all-reduce of the LoRA gradients only (28,672 fp32 values at
r=4).  This replaces DistributedDataParallel's reducer (train_lora_sam.py:126,172; SURVEY.md
section 2b): with every non-LoRA parameter frozen the reducer's traffic is exactly these tensors.

The gradients travel in buckets of one LoRA block each (4 tensors, 56 KiB at r=4), in the order the
backward produces them.  `attach(trunk)` registers a hook with the trunk so that a block's bucket is
all-reduced (RCCL, backend "nccl" on ROCm, on its own stream) as soon as that block's backward is
enqueued, overlapping the rest of the backward; `reduce()` then only waits, scales by 1/world and
writes the result to `.grad`.  Without `attach` (or for gradients the hook never saw) `reduce()`
all-reduces the buckets itself.  At this size the collective is latency-bound, not link-bound, so
the buckets are not split further.  On CPU the same code runs over gloo (tests/test_dp_cpu.py).

Whenever a process group exists the exchange step RUNS, whatever the group's size: a one-rank group (a 1-GPU box under
torch.distributed.run, tests/test_dp_gpu.py) still builds the RCCL communicator, broadcasts, and all-reduces every bucket
from inside the backward -- the mean over one rank is the identity, so results stay bit-equal to the plain step.  Only
without any process group (plain `python bench.py`) are the calls no-ops.  `stats` counts the collectives issued."""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence, Union

import torch
import torch.distributed as dist

from . import ops


@torch.no_grad()
def clip_grads_(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, out: Optional[Sequence[torch.Tensor]] = None,
                grad_scale: float = 1.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """The global norm of `grad_scale * grads` (fp32, 0-d, on the device) and the gradients scaled by grad_scale * min(1, max_norm /
    (norm + 1e-6)), in place or into `out`.

    fp32 / bf16 tensors of any mix on one GPU; `out` may have other types than `grads` (bf16 gradients into fp32 buffers).  norm_type
    2 or inf.  Squares are summed in fp64.  A norm that is not finite makes the factor what torch.nn.utils.clip_grad_norm_ makes it
    (NaN, or 0 for an infinite one); error_if_nonfinite looks at the norm on the host first and raises, with nothing changed.
    max_norm = inf: the norm alone, of tensors of any layout, and nothing is written.  Contiguous tensors that share memory are refused
    where anything would be written, and so are others that begin at one address or repeat their elements (expanded ones)."""
    grads = list(grads)
    inf_norm = float(norm_type) == float("inf")
    if not inf_norm and float(norm_type) != 2.0:
        raise ops._C.LsamError(f"clip_grads_: norm_type {norm_type}; 2 and inf are built")
    max_norm, grad_scale = float(max_norm), float(grad_scale)
    if not max_norm >= 0.0 or grad_scale != grad_scale:
        raise ValueError(f"clip_grads_: max_norm {max_norm}, grad_scale {grad_scale}")
    if not grads:
        return torch.tensor(0.0)
    if out is None:
        into = grads
    else:
        into = list(out)
        if list(map(torch.Tensor.size, into)) != list(map(torch.Tensor.size, grads)):
            raise ops._C.LsamError("clip_grads_: out must hold one tensor of the same shape for each gradient")
    dense = torch.Tensor.is_contiguous
    src = grads if all(map(dense, grads)) else [g.contiguous() for g in grads]   # another layout goes through a contiguous copy
    dst = src if out is None else into if all(map(dense, into)) else [t.contiguous() for t in into]
    writes = out is not None or max_norm != float("inf") or grad_scale != 1.0
    if writes and dst is not into:                             # copies hide what the kernel's check sees
        starts = [t.data_ptr() for t in into if t.numel()]
        if len(set(starts)) != len(starts) or any(n > 1 and s == 0 for t in into for n, s in zip(t.shape, t.stride())):
            raise ops._C.LsamError("clip_grads_: tensors that share memory, or repeat their elements")
    if error_if_nonfinite:
        norm = ops._clip_grads(src, src, float("inf"), inf_norm, 1.0)[0] * abs(grad_scale)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it cannot be clipped.")
    norm = ops._clip_grads(src, dst, max_norm, inf_norm, grad_scale)[0]
    if writes and dst is not into:
        for t, d in zip(into, dst):
            if t is not d:
                t.copy_(d)
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ on liblsam: clips the gradients of `parameters` in place by their global norm and returns it.
    A parameter that is listed twice counts once."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(dict.fromkeys(parameters))
    return clip_grads_([p.grad for p in params if p.grad is not None], max_norm, norm_type, error_if_nonfinite=error_if_nonfinite)


class _Bucket:
    def __init__(self, params, flat):
        self.params = params
        self.flat = flat
        self.views = []
        o = 0
        for p in params:
            self.views.append(flat[o:o + p.numel()].view_as(p))
            o += p.numel()
        self.work = None      # in-flight all-reduce started by the hook
        self.filled = False   # flat holds this step's local gradients
        self.pending = []     # (increment buffer, work) of further backwards before reduce()


class LoRAGradReducer:
    def __init__(self, params: Iterable[torch.nn.Parameter], group: Optional[dist.ProcessGroup] = None,
                 tensors_per_bucket: int = 4):
        self.params: List[torch.nn.Parameter] = [p for p in params if p.requires_grad]
        if not self.params:
            raise ValueError("LoRAGradReducer: no trainable parameters")
        if tensors_per_bucket < 1:
            raise ValueError("LoRAGradReducer: tensors_per_bucket must be positive")
        self.group = group
        self.numel = sum(p.numel() for p in self.params)
        p0 = self.params[0]
        self.flat = torch.zeros(self.numel, dtype=torch.float32, device=p0.device)
        self.buckets: List[_Bucket] = []
        o = 0
        for i in range(0, len(self.params), tensors_per_bucket):
            ps = self.params[i:i + tensors_per_bucket]
            n = sum(p.numel() for p in ps)
            self.buckets.append(_Bucket(ps, self.flat[o:o + n]))
            o += n
        self.views = [v for b in self.buckets for v in b.views]
        self._by_first = {id(b.params[0]): b for b in self.buckets}
        self._invalidate = []   # trunks whose packed weights must be refreshed after parameters change through .data
        self.stats = {"broadcast": 0, "all_reduce": 0, "all_reduce_from_backward": 0}

    def active(self) -> bool:
        """A process group exists: collectives are issued (also on a one-rank group)."""
        return dist.is_available() and dist.is_initialized()

    def world_size(self) -> int:
        return dist.get_world_size(self.group) if self.active() else 1

    def _all_reduce(self, t, from_backward=False):
        self.stats["all_reduce"] += 1
        if from_backward:
            self.stats["all_reduce_from_backward"] += 1
        return dist.all_reduce(t, op=dist.ReduceOp.SUM, group=self.group, async_op=True)

    def attach(self, trunk) -> "LoRAGradReducer":
        """Overlap mode: the trunk's backward hands each LoRA block's gradients to on_bucket()."""
        trunk.set_grad_bucket_hook(self.on_bucket)
        inv = getattr(trunk, "invalidate_packed", None)
        if inv is not None:
            self._invalidate.append(inv)
        return self

    @torch.no_grad()
    def broadcast_params(self, src: int = 0):
        """DDP's constructor broadcast, restricted to the trainable tensors (frozen ones are built
        from the same checkpoint / seed on every rank)."""
        if not self.active():
            return
        torch._foreach_copy_(self.views, [p.data for p in self.params])
        dist.broadcast(self.flat, src=src, group=self.group)
        self.stats["broadcast"] += 1
        torch._foreach_copy_([p.data for p in self.params], self.views)
        for inv in self._invalidate:
            inv()

    @torch.no_grad()
    def on_bucket(self, params, grads):
        """Called from the backward (autograd thread) once the gradients of `params` are enqueued on
        the current stream: stage them in the bucket and start its all-reduce without waiting."""
        b = self._by_first.get(id(params[0]))
        if b is None or len(params) != len(b.params) or any(p is not q for p, q in zip(params, b.params)):
            return   # not one of our buckets: reduce() falls back to .grad
        if not self.active():
            return
        if b.filled:
            # a second backward before reduce() (gradient accumulation, two views per step): DDP sums the micro-batches.
            # The first all-reduce may still be in flight on b.flat, so the increment gets a staging buffer of its own
            # and is reduced separately: sum_r(g1_r) + sum_r(g2_r) = sum_r(g1_r + g2_r); reduce() adds them up.
            inc = torch.empty_like(b.flat)
            o = 0
            views = []
            for p in b.params:
                views.append(inc[o:o + p.numel()].view_as(p))
                o += p.numel()
            torch._foreach_copy_(views, list(grads))
            b.pending.append((inc, self._all_reduce(inc, True)))
            return
        torch._foreach_copy_(b.views, list(grads))
        b.filled = True
        b.work = self._all_reduce(b.flat, True)

    @torch.no_grad()
    def reduce(self, max_norm: Optional[float] = None):
        """grads <- mean over ranks.  Missing grads count as zero (DDP semantics).  With `max_norm` the mean is clipped to that global
        norm as it is written (one pass with the division by the ranks: clip_grads_), and the norm before clipping is returned; every
        rank clips the same sums, so the ranks stay alike without another exchange."""
        if max_norm is not None and not (float(max_norm) >= 0.0 and self.flat.is_cuda):   # before any exchange, on every rank alike
            raise ops._C.LsamError(f"LoRAGradReducer.reduce: max_norm {max_norm} on {self.flat.device}; a norm >= 0 on the MI355X (there is "
                                   "no CPU fallback)")
        if max_norm is not None:
            for p in self.params:
                if p.dtype not in (torch.float32, torch.bfloat16):
                    raise ops._C.LsamError(f"LoRAGradReducer.reduce: max_norm with a parameter of {p.dtype}; float32 and bfloat16 are built")
        if not self.active():
            return None if max_norm is None else clip_grad_norm_(self.params, max_norm)
        ws = self.world_size()
        for b in reversed(self.buckets):   # the order the backward produced (and launched) them
            if not b.filled:
                grads = [p.grad if p.grad is not None else torch.zeros_like(p) for p in b.params]
                torch._foreach_copy_(b.views, grads)
                b.work = self._all_reduce(b.flat)
        for b in reversed(self.buckets):
            b.work.wait()
            for inc, work in b.pending:
                work.wait()
                b.flat.add_(inc)
            b.pending = []
            b.work, b.filled = None, False
        if max_norm is not None:
            out = [torch.empty_like(p) if p.grad is None else p.grad for p in self.params]
            norm = clip_grads_(self.views, max_norm, out=out, grad_scale=1.0 / ws)
            for p, g in zip(self.params, out):
                if p.grad is None:
                    p.grad = g
            return norm
        if ws > 1:
            self.flat.mul_(1.0 / ws)
        for p, v in zip(self.params, self.views):
            if p.grad is None:
                p.grad = v.clone()
            else:
                p.grad.copy_(v)
