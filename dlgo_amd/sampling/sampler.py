"""Next tokens from logits on the device: argmax when every row is greedy, else
the sampling kernel with each row's own options."""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops
from .options import SamplerConfig

RECENT = 64   # tokens the repetition penalty looks back on (models/llm/generate.go:361-365)


def _below_one(uniforms: Sequence[Sequence[float]], n: int) -> np.ndarray:
    """n numbers of [0, 1) as float32 of [0, 1): what would round up to one (1 - 2^-25 and more) is the largest below it, for
    a draft that is sure of its token (u * 1 < 1) and a draw (the first sum above u times the whole) need u < 1."""
    u = np.fromiter((v for row in uniforms for v in row), dtype=np.float32, count=n)
    return np.minimum(u, np.float32(1 - 2.0 ** -24))


class Sampler:
    #: the tokens a request has been given are also kept on the device (start(), and keys= of the choose calls), so
    #: that the repetition penalty does not need them back from the host before the next choice
    keeps_recent = True

    def __init__(self, vocab: int, device, max_rows: int = 256):
        self.vocab = vocab
        self.device = torch.device(device)
        self.max_rows = max_rows
        self._out = torch.empty(max_rows, dtype=torch.int32, device=self.device)
        self._pinned = [torch.empty(max_rows, dtype=torch.int32, pin_memory=True) for _ in range(4)]
        self._pin_next = 0
        self._work: Optional[torch.Tensor] = None
        # the rows' options go up in one copy from pinned memory that does not wait for the device: a copy from
        # ordinary memory would hold the host until the step queued before it is done, and the step after it with it
        self._staging: List[tuple] = []                 # (pinned int32 buffer, event of the copy that last read it)
        self._staging_next = 0
        self._options: Optional[torch.Tensor] = None    # the device's copy: 7 rows of int32/float32 bits
        self._verify_dev: Optional[torch.Tensor] = None    # verify()'s arrays and scratch on the device
        self._verify_work: Optional[torch.Tensor] = None
        self._rings: Optional[torch.Tensor] = None      # [keys, RECENT] last tokens chosen per key
        self._counts: Optional[torch.Tensor] = None     # [keys] tokens chosen so far per key

    def start(self, keys: Sequence[int]) -> None:
        """Requests begin under these keys (any small integers that stay with a request, such as its slot): what the
        device remembers of earlier requests under them is forgotten."""
        need = max(keys) + 1 if len(keys) else 0
        if self._counts is None or self._counts.shape[0] < need:
            size = max(need, 2 * (self._counts.shape[0] if self._counts is not None else 0), self.max_rows)
            counts = torch.zeros(size, dtype=torch.int32, device=self.device)
            rings = torch.full((size, RECENT), -1, dtype=torch.int32, device=self.device)
            if self._counts is not None:
                counts[:self._counts.shape[0]] = self._counts
                rings[:self._rings.shape[0]] = self._rings
            self._counts, self._rings = counts, rings
        if len(keys):
            self._counts[torch.as_tensor(list(keys), dtype=torch.long)] = 0

    def _upload(self, f: np.ndarray, k: np.ndarray):
        """f [5, n] float32 and k [2, n] int32 -> their device copies, through one pinned buffer and one copy that the
        host does not wait for."""
        n = f.shape[1]
        if not self._staging:
            self._staging = [(torch.empty(7 * max(n, self.max_rows), dtype=torch.int32, pin_memory=True), None) for _ in range(4)]
        i = self._staging_next
        self._staging_next = (i + 1) % len(self._staging)
        buf, ev = self._staging[i]
        if ev is not None:
            ev.synchronize()
        if buf.numel() < 7 * n:
            buf = torch.empty(14 * n, dtype=torch.int32, pin_memory=True)
        hv = buf.numpy()
        hv[:5 * n] = f.reshape(-1).view(np.int32)
        hv[5 * n:7 * n] = k.reshape(-1)
        if self._options is None or self._options.numel() < 7 * n:
            self._options = torch.empty(14 * n, dtype=torch.int32, device=self.device)
        dev = self._options[:7 * n]
        dev.copy_(buf[:7 * n], non_blocking=True)
        ev = torch.cuda.Event()
        ev.record()
        self._staging[i] = (buf, ev)
        return dev[:5 * n].view(torch.float32).view(5, n), dev[5 * n:].view(2, n)

    def _grow(self, rows: int) -> None:
        if rows > self._out.shape[0]:
            self._out = torch.empty(rows, dtype=torch.int32, device=self.device)
            self._work = None

    def choose(self, logits: torch.Tensor, configs: Sequence[SamplerConfig], uniforms: Sequence[float],
               recent: Optional[Sequence[Sequence[int]]] = None) -> List[int]:
        """logits [rows, vocab] float32 on the device -> one token id per row (host list)."""
        return self.choose_device(logits, configs, uniforms, recent).tolist()

    def choose_async(self, logits: torch.Tensor, configs: Sequence[SamplerConfig], uniforms: Sequence[float],
                     recent: Optional[Sequence[Sequence[int]]] = None, keys: Optional[Sequence[int]] = None):
        """The ids as a device tensor (valid until the next call) and a function that waits for them and
        returns them as a host list; work can be queued behind the choice before the ids are awaited.
        keys (instead of recent): each row's key as given to start(); the recent tokens are the device's own record."""
        out = self.choose_device(logits, configs, uniforms, recent, keys)
        n = out.shape[0]
        i = self._pin_next
        self._pin_next = (i + 1) % len(self._pinned)
        host = self._pinned[i]
        if host.shape[0] < n:
            host = self._pinned[i] = torch.empty(max(n, 2 * host.shape[0]), dtype=torch.int32, pin_memory=True)
        host[:n].copy_(out, non_blocking=True)
        event = torch.cuda.Event()
        event.record()

        def wait() -> List[int]:
            event.synchronize()
            return host[:n].tolist()
        return out, wait

    def needs_recent(self, configs: Sequence[SamplerConfig]) -> bool:
        """True if a row's choice depends on the tokens generated so far (the repetition penalty)."""
        return any(c.repetition_penalty > 1.0 and not c.greedy for c in configs)

    def choose_device(self, logits: torch.Tensor, configs: Sequence[SamplerConfig], uniforms: Sequence[float],
                      recent: Optional[Sequence[Sequence[int]]] = None, keys: Optional[Sequence[int]] = None) -> torch.Tensor:
        """logits [rows, vocab] float32 on the device -> int32 ids on the device (overwritten by the next call)."""
        n = logits.shape[0]
        if n != len(configs) or n != len(uniforms):
            raise ValueError("sampler: one configuration and one uniform number per row")
        self._grow(n)
        out = self._out[:n]
        if all(c.greedy for c in configs):
            ops.argmax(logits, out)
            return out
        if self._work is None:
            rows = self._out.shape[0]
            self._work = torch.empty((rows, self.vocab), dtype=torch.float32, device=self.device)
        f = np.zeros((5, n), dtype=np.float32)
        k = np.zeros((2, n), dtype=np.int32)        # top-k, and the row's key if the device keeps the recent tokens
        for i, c in enumerate(configs):
            f[0, i], f[1, i], f[2, i], f[3, i], f[4, i] = c.temperature, c.top_p, c.min_p, c.repetition_penalty, uniforms[i]
            k[0, i] = c.top_k
        penalised = any(c.repetition_penalty > 1.0 and not c.greedy for c in configs)
        rings = keys is not None and recent is None
        if rings:
            if self._counts is None or max(keys) >= self._counts.shape[0]:
                raise ValueError("sampler: keys that start() was never given")
            k[1] = np.asarray(keys, dtype=np.int32)
        fd, kd = self._upload(f, k)
        # rows that several blocks share: a top-k of up to 1,024, or neither top-k nor top-p; without one, two kernels need not be
        # launched (a hint only: which rows those kernels take they decide themselves, from the options on the device)
        dealt_rows = any(not c.greedy and (1 <= c.top_k <= 1024 or (not 0 < c.top_k < self.vocab and c.top_p >= 1.0))
                         for c in configs)
        if rings:       # every choice is recorded, penalty or not: a later row of the request may have one
            ops.sample(logits, self._work, fd[0], kd[0], fd[1], fd[2], fd[3], self._rings, fd[4], out,
                       recent_rows=kd[1], counts=self._counts, dealt_rows=dealt_rows)
            return out
        rec = None
        if recent is not None and penalised:
            r = np.full((n, RECENT), -1, dtype=np.int32)
            for i, toks in enumerate(recent):
                toks = list(toks)[-RECENT:]
                r[i, :len(toks)] = toks
            rec = torch.from_numpy(r).to(self.device)
        ops.sample(logits, self._work, fd[0], kd[0], fd[1], fd[2], fd[3], rec, fd[4], out, dealt_rows=dealt_rows)
        return out

    def verify(self, logits: torch.Tensor, drafts: Sequence[Sequence[int]], configs: Sequence[SamplerConfig],
               uniforms: Sequence[Sequence[float]], draft_logits: Optional[torch.Tensor] = None):
        """Sequence i drafted the tokens drafts[i] (perhaps none) and logits holds, for sequence after sequence, the target
        model's rows for the place of each draft and the place after them ([sum(len + 1), vocab] float32 on the device).
        Returns (kept, tokens) as host lists: how many of each sequence's drafts are kept, and the token that follows
        them; both are then distributed as if the target had chosen every token itself.  uniforms[i]: a number in [0, 1)
        for each draft and one for the token after.  draft_logits [sum(len), vocab]: what a draft model drew the drafts
        from, at the same temperature; None where they are certain (looked up).  Greedy rows keep what is the maximum."""
        n, d = len(drafts), sum(len(x) for x in drafts)
        if len(configs) != n or len(uniforms) != n or any(len(u) != len(x) + 1 for u, x in zip(uniforms, drafts)):
            raise ValueError("sampler: one configuration per sequence, and a uniform number for each draft and one more")
        if logits.shape[0] != n + d:
            raise ValueError(f"sampler: {n} sequences with {d} drafts need {n + d} rows of logits, not {logits.shape[0]}")
        for c in configs:
            if not c.temperature_alone:
                raise ValueError("sampler: drafts are verified greedily or at a temperature alone (no top-k, top-p, min-p or repetition penalty)")
        if n == 0:
            return [], []
        lens = np.array([len(x) for x in drafts], dtype=np.int64)
        # one copy up (drafts, their offsets, temperatures, uniform numbers), one down (kept counts and tokens)
        parts = (np.fromiter((t for x in drafts for t in x), dtype=np.int32, count=d),
                 np.concatenate([[0], np.cumsum(lens)]).astype(np.int32),
                 np.array([max(0.0, c.temperature) for c in configs], dtype=np.float32).view(np.int32),
                 _below_one(uniforms, n + d).view(np.int32))
        offs, total = [], 0
        for a in parts:
            offs.append(total)
            total += (len(a) + 3) // 4 * 4
        if self._verify_dev is None or self._verify_dev.numel() < total + 2 * n:
            self._verify_dev = torch.empty(2 * (total + 2 * n), dtype=torch.int32, device=self.device)
        i = self._pin_next
        self._pin_next = (i + 1) % len(self._pinned)
        if self._pinned[i].shape[0] < max(total, 2 * n):
            self._pinned[i] = torch.empty(2 * max(total, 2 * n), dtype=torch.int32, pin_memory=True)
        host = self._pinned[i]
        for a, o in zip(parts, offs):
            host.numpy()[o:o + len(a)] = a
        dev = self._verify_dev
        dev[:total].copy_(host[:total], non_blocking=True)
        at = [dev[o:o + len(a)] for a, o in zip(parts, offs)]
        out = dev[total:total + 2 * n]

        def scratch(size):
            if self._verify_work is None or self._verify_work.numel() < size:
                self._verify_work = torch.empty(size, dtype=torch.uint8, device=self.device)
            return self._verify_work
        ops.verify_drafts(logits, at[0], at[1], at[2].view(torch.float32), at[3].view(torch.float32), out[:n], out[n:], int(lens.max()),
                          draft_logits=draft_logits, scratch=scratch)
        host[:2 * n].copy_(out, non_blocking=True)         # behind the copy up, in the same stream
        event = torch.cuda.Event()
        event.record()
        event.synchronize()
        got = host[:2 * n].tolist()
        return got[:n], got[n:]
