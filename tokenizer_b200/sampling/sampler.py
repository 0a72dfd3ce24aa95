"""Greedy, temperature and nucleus sampling on the device, one row of float32
logits per request (reference: qwen-infer/src/sample.rs:43-137).  temperature 0
is argmax with ties to the lower id and ignores top_p; otherwise weights
exp((l - max)/T), candidates by logit descending, the shortest prefix whose
share reaches top_p, and one draw u scaled by the kept weight.  Beyond the reference's two, a request may
filter with top_k (the first k candidates of that order; top_p is then a share of what they weigh) and min_p
(candidates that weigh at least min_p times the best one)."""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import torch

from ..kernels import ops


def validate_sampling(temperature: float, top_p: float, top_k: int = 0, min_p: float = 0.0) -> None:
    """sample.rs:77-88 and generate.rs:409-424; top_k is a whole number (0: no limit), min_p a share."""
    if not math.isfinite(temperature):
        raise ValueError(f"temperature {temperature} is not finite")
    if temperature < 0:
        raise ValueError(f"temperature {temperature} is negative")
    if not math.isfinite(top_p):
        raise ValueError(f"top_p {top_p} is not finite")
    if top_p < 0:
        raise ValueError(f"top_p {top_p} is negative")
    if isinstance(top_k, bool) or not isinstance(top_k, int):
        raise ValueError(f"top_k {top_k!r} is not a whole number")
    if not 0 <= top_k < 1 << 31:
        raise ValueError(f"top_k {top_k} is negative or beyond 32 bits")
    if not 0.0 <= min_p <= 1.0:      # NaN too
        raise ValueError(f"min_p {min_p} is not between 0 and 1")


class PendingIds:
    """Ids on their way from the device; one outstanding draw per sampler at a time.
    `device_ids` (int32, one a row) can feed the next step before the host has read them."""

    def __init__(self, host, done, device_ids=None):
        self._host, self._done = host, done
        self.device_ids = device_ids

    def result(self) -> List[int]:
        if self._host is None:
            return []
        self._done.synchronize()
        # the step that made these logits has finished: had one of its bounded waits run out,
        # the ids would come from wrong logits
        ops.raise_if_error("found when a draw's ids were read")
        return self._host.tolist()


class Sampler:
    def __init__(self, device):
        self.device = torch.device(device)
        self._pinned = None
        self.scratch = ops.ScratchSpace()       # the greedy choice's partial results and counters

    def sample(self, logits: torch.Tensor, temperature: Sequence[float], top_p: Sequence[float],
               uniform: Sequence[float], top_k: Optional[Sequence[int]] = None,
               min_p: Optional[Sequence[float]] = None) -> List[int]:
        """One id per row.  All-greedy batches skip the parameter upload.  `top_k` (0: off) and `min_p` (0.0: off) may be None."""
        return self.sample_launch(logits, temperature, top_p, uniform, top_k, min_p).result()

    def sample_launch(self, logits: torch.Tensor, temperature: Sequence[float],
                      top_p: Sequence[float], uniform: Sequence[float], top_k: Optional[Sequence[int]] = None,
                      min_p: Optional[Sequence[float]] = None) -> "PendingIds":
        """Start the draw and the copy of the ids to pinned host memory; `result()` waits for
        them.  What the host does in between runs beside the device.  A row with top_k or min_p is drawn by
        `ops.sample_filtered`, any other by `ops.sample`, whatever else is in the batch."""
        n = logits.shape[0]
        if n == 0:
            return PendingIds(None, None)
        if logits.shape[1] == 0:
            raise ValueError("no logits to sample")
        out = torch.empty(n, dtype=torch.int32, device=self.device)
        with ops.scratch_scope(self.scratch):
            filtered = [t != 0 and (k > 0 or m > 0) for t, k, m in zip(temperature, top_k or [0] * n, min_p or [0.0] * n)]
            if any(filtered):
                self._sample_filtered(logits, filtered, temperature, top_p, uniform, top_k or [0] * n, min_p or [0.0] * n, out)
            elif all(t == 0 for t in temperature):
                ops.sample(logits, None, None, None, out)
            else:
                params = torch.tensor([list(temperature), list(top_p), list(uniform)],
                                      dtype=torch.float32).to(self.device, non_blocking=True)
                ops.sample(logits, params[0], params[1], params[2], out)
        if self._pinned is None or self._pinned.numel() < n:
            self._pinned = torch.empty(max(n, 256), dtype=torch.int32, pin_memory=True)
        host = self._pinned[:n]
        host.copy_(out, non_blocking=True)
        done = torch.cuda.Event()
        done.record()
        return PendingIds(host, done, out)

    def _sample_filtered(self, logits, filtered, temperature, top_p, uniform, top_k, min_p, out) -> None:
        """Rows that are not `filtered` but sampled go to the kernel that takes them when they are alone."""
        params = torch.tensor([[t if f else 0.0 for t, f in zip(temperature, filtered)], list(top_p), list(uniform), list(min_p),
                               [0.0 if f else t for t, f in zip(temperature, filtered)], [float(f) for f in filtered]],
                              dtype=torch.float32).to(self.device, non_blocking=True)
        ks = torch.tensor(list(top_k), dtype=torch.int32).to(self.device, non_blocking=True)
        ops.sample_filtered(logits, params[0], ks, params[1], params[3], params[2], out)
        if any(t != 0 and not f for t, f in zip(temperature, filtered)):
            others = torch.empty_like(out)
            ops.sample(logits, params[4], params[1], params[2], others)
            out.copy_(torch.where(params[5] != 0, out, others))

    def greedy(self, logits: torch.Tensor) -> torch.Tensor:
        out = torch.empty(logits.shape[0], dtype=torch.int32, device=self.device)
        with ops.scratch_scope(self.scratch):
            ops.sample(logits, None, None, None, out)
        return out
