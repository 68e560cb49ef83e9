"""Next-token choice on the device for a batch of logits rows.

Greedy is the reference's argmax (crates/core-types/src/model.rs:44-62: lowest index wins a
tie, NaN is skipped).  With a temperature the kernel draws from softmax(logits / T) by the
Gumbel-max trick with a counter-based hash keyed by (seed, tokens generated so far,
vocabulary index): a request's draw does not depend on the batch it shares a step with.  Rows with
filters (top-k, top-p, which the reference's `SamplingParams` carries and accepts only as 1,
crates/core-types/src/schedule.rs:16-40, and min-p) are drawn by a kernel of their own from one random number each, a hash of (seed, tokens
generated so far) again.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from ..errors import InvalidRequest
from ..ops import lib as ops


_MASK = (1 << 64) - 1


def _mix64(x):
    """The finaliser of the splitmix64 generator (Steele, Lea and Flood 2014)."""
    x = (x + 0x9E3779B97F4A7C15) & _MASK
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & _MASK
    return x ^ (x >> 31)


def uniform(seed, counter):
    """The random number in [0, 1) of a request's draw number `counter`: 53 bits that depend on (seed, counter) alone."""
    return (_mix64(_mix64(int(seed) & _MASK) ^ int(counter)) >> 11) * 2.0 ** -53


def _float32(v):
    """A filter's value as the kernel gets it, where one below 2^-149 is 0; NaN for what is no number."""
    try:
        with np.errstate(over="ignore"):
            return float("nan") if isinstance(v, (str, bytes, list, tuple)) else float(np.float32(v))
    except (TypeError, ValueError, OverflowError):
        return float("nan")


@dataclass(frozen=True)
class Filters:
    """What a draw leaves out (in this order; `ops.sample_filtered` has the definition): all but the top_k largest logits (0:
    off), what lies beyond the top_p part of their mass (1: off), what is less likely than min_p times the likeliest (0: off)."""
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self):
        try:
            whole = not isinstance(self.top_k, bool) and int(self.top_k) == self.top_k
        except (TypeError, ValueError, OverflowError):      # (what is no number, a NaN, an infinity)
            whole = False
        if not whole or not 0 <= self.top_k < 1 << 31:
            raise InvalidRequest("top_k must be a whole number, 0 (off) or more")
        if not 0 < _float32(self.top_p) <= 1:
            raise InvalidRequest("top_p must be in (0, 1]")
        if not 0 <= _float32(self.min_p) <= 1:
            raise InvalidRequest("min_p must be in [0, 1]")

    @property
    def on(self):
        return self.top_k > 0 or self.top_p < 1 or self.min_p > 0


class Ticket:
    """A launched sampling whose ids have not been read yet."""
    __slots__ = ("n", "host", "event")

    def __init__(self, n, host, event):
        self.n, self.host, self.event = n, host, event


class DeviceSampler:
    """Owns the small pinned and device buffers a step's sampling needs; one instance per engine.

    `launch` enqueues the kernel and the copy of its ids to the host and returns at once;
    `collect` waits for that copy.  Two samplings may be in flight (the engine queues the next
    step before it reads this one), so the pinned buffers are rings.  The kernel can write the
    ids to a second place on the device as well (`also_to`): the token buffer of a step that is
    queued behind this one.  The kernels' error flag lives behind the ids (`err`)."""

    DEPTH = 4

    def __init__(self, max_rows: int, device="cuda"):
        from ..engine.batch import PinnedRing
        n = int(max_rows)
        self.device = device
        dev = lambda dt: torch.empty(n + 1, dtype=dt, device=device)
        self._inv_t = (PinnedRing(n + 1, torch.float32, device, self.DEPTH), dev(torch.float32))
        self._seeds = (PinnedRing(n + 1, torch.int64, device, self.DEPTH), dev(torch.int64))
        self._counters = (PinnedRing(n + 1, torch.int32, device, self.DEPTH), dev(torch.int32))
        # rows with filters: uniform (float64), then temperature, top_p, min_p (float32), then row, top_k (int32)
        self._filtered = (PinnedRing(28 * (n + 1), torch.uint8, device, self.DEPTH), torch.empty(28 * (n + 1), dtype=torch.uint8, device=device))
        self._ids_host = [torch.empty(n + 1, dtype=torch.int32).pin_memory() for _ in range(self.DEPTH)]
        self._events = [torch.cuda.Event() for _ in range(self.DEPTH)]
        self._turn = 0
        self.max_rows = n
        self.ids_device = dev(torch.int32)
        self.ids_device.zero_()
        # the kernels' error flag sits behind the ids, so that one copy brings both to the host
        self.err = self.ids_device[n:n + 1]
        self.d2h_bytes = 0

    def _launch_filtered(self, logits, rows, filters, picked, also_to):
        """Draws the rows `picked` (indices) with their filters."""
        ring, dev = self._filtered
        m = len(picked)
        host = ring.next()
        h = host.numpy()[:28 * m]
        h[:8 * m].view(np.float64)[:] = [uniform(rows[i].seed, rows[i].counter) for i in picked]
        f = h[8 * m:20 * m].view(np.float32)
        f[:m] = [rows[i].temperature for i in picked]
        f[m:2 * m] = [filters[i].top_p for i in picked]
        f[2 * m:] = [filters[i].min_p for i in picked]
        k = h[20 * m:].view(np.int32)
        k[:m], k[m:] = picked, [filters[i].top_k for i in picked]
        dev[:28 * m].copy_(host[:28 * m], non_blocking=True)
        ring.sent()
        u, f, k = dev[:8 * m].view(torch.float64), dev[8 * m:20 * m].view(torch.float32), dev[20 * m:28 * m].view(torch.int32)
        ops.sample_filtered(logits, m, self.ids_device, self.err, f[:m], k[m:], f[m:2 * m], f[2 * m:], u, rows=k[:m], also_to=also_to)

    def launch(self, logits, rows, also_to=None, filters=None) -> Ticket:
        """rows: objects with `temperature`, `seed`, `counter`, one per row of `logits`; filters: `Filters` or None per row
        (they act on rows with a temperature).  The ids
        and the error flag (`self.err`, which the step's kernels must have been given) travel to
        the host in one copy.  also_to: an int32 device tensor that receives the ids as well."""
        n, err = len(rows), self.err
        if n > self.max_rows:
            raise ValueError(f"{n} rows to sample, the sampler was made for {self.max_rows}")
        ids_d = self.ids_device
        picked = [i for i, (r, f) in enumerate(zip(rows, filters)) if f is not None and f.on and r.temperature > 0] if filters else []
        if len(picked) == n and n:
            pass                       # no row is left for the kernel of plain draws
        elif any(r.temperature > 0 for r in rows):
            (it_r, it_d), (sd_r, sd_d), (ct_r, ct_d) = self._inv_t, self._seeds, self._counters
            it_h, sd_h, ct_h = it_r.next(), sd_r.next(), ct_r.next()
            for i, r in enumerate(rows):
                it_h[i] = float(np.float32(1.0 / r.temperature)) if r.temperature > 0 else 0.0
                sd_h[i] = int(np.uint64(r.seed).astype(np.int64))
                ct_h[i] = r.counter
            for ring, h, d in ((it_r, it_h, it_d), (sd_r, sd_h, sd_d), (ct_r, ct_h, ct_d)):
                d[:n].copy_(h[:n], non_blocking=True)
                ring.sent()
            ops.sample(logits, n, ids_d, err, it_d[:n], sd_d[:n], ct_d[:n], also_to=also_to)
        else:
            ops.sample(logits, n, ids_d, err, also_to=also_to)
        if picked:
            self._launch_filtered(logits, rows, filters, picked, also_to)
        self._turn = (self._turn + 1) % self.DEPTH
        host, event = self._ids_host[self._turn], self._events[self._turn]
        host.copy_(ids_d, non_blocking=True)
        event.record(ops.current_stream())
        self.d2h_bytes = 4 * (self.max_rows + 1)
        return Ticket(n, host, event)

    @staticmethod
    def collect(ticket: Ticket):
        """(ids, device error code) of a launch; the wait for its copy is the step's only
        synchronisation."""
        ticket.event.synchronize()
        out = ticket.host.tolist()
        return out[:ticket.n], out[-1]

    def sample(self, logits, rows, filters=None):
        """launch + collect."""
        return self.collect(self.launch(logits, rows, filters=filters))
