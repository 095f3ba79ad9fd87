"""Turns logits rows into token ids on the device.

Same interface idea as the reference's `Sampler.sample(logits, params, token_histories)`
(somi_inference/core/sampler.py:31-55), but the whole pipeline (repetition
penalty, temperature, top-k, top-p, argmax or draw) is one kernel launch for
all rows, and each row carries (seed, counter) for its random number.  Rows with `min_p`, and draws
from numbers that the caller brings (`draw`), go to the kernel that cuts exactly k tokens and makes any number of draws
a row (`CudaOps.draw_tokens`).
"""

from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

from .params import SamplingParams

_LIKELIEST = SamplingParams(temperature=0.0)


class Sampler:
    def __init__(self, ops, device: torch.device | str) -> None:
        self.ops = ops
        self.device = torch.device(device)
        self.h2d_bytes_last = 0
        self._greedy: dict = {}

    def sample(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               counters: Sequence[int], seeds: Sequence[int],
               histories: Sequence[Sequence[int]] | None = None) -> torch.Tensor:
        """logits [rows, vocab] float32 on the device -> int32 [rows] on the device.

        `counters[i]` is how many tokens row i's request has sampled so far;
        `seeds[i]` its seed; `histories[i]` its prompt and output tokens (only
        read where the row's repetition penalty is not 1).
        """
        rows = logits.shape[0]
        if logits.dim() != 2:
            raise ValueError(f"logits must be 2D, got shape {tuple(logits.shape)}")
        if not (len(params) == len(counters) == len(seeds) == rows):
            raise ValueError("one SamplingParams, counter and seed per logits row is needed")
        if all(p.temperature == 0.0 and p.repetition_penalty == 1.0 for p in params):
            # argmax rows need neither seeds, counters nor histories: one cached parameter block
            cached = self._greedy.get(rows)
            if cached is None:
                cached = self._pack(params, [0] * rows, [0] * rows, None)
                self._greedy[rows] = cached
            self.h2d_bytes_last = 0
            return self._launch(logits, rows, *cached)
        cut = [i for i, p in enumerate(params) if p.min_p > 0.0 and p.temperature > 0.0]
        if not cut:
            return self._launch(logits, rows, *self._pack(params, counters, seeds, histories))
        # Rows with min-p by themselves, so that the other rows' tokens do not depend on them, with the numbers that the rows
        # would have drawn in the other kernel.  All arguments go up at once and nothing waits: the stream may hold a whole
        # step in front of this one, whose tokens the caller is still to read.
        numbers = [self.ops.uniform(int(seeds[i]) % (1 << 64), int(counters[i]) % (1 << 32)) for i in cut]
        some = [params[i] for i in cut]
        drawn = self._fill(some, [0] * len(cut), [0] * len(cut), None if histories is None else [histories[i] for i in cut])
        floats = np.array([numbers, [p.min_p for p in some]], dtype=np.float32)
        if len(cut) == rows:
            views, (number, min_p) = self._upload([drawn], floats)
            return self._draw(logits, some, *views, number, min_p)[0]
        # (the other kernel leaves something for every row: for these the token that costs it least)
        rest = list(params)
        for i in cut:
            rest[i] = _LIKELIEST
        usual = self._fill(rest, counters, seeds, histories)
        views, (number, min_p), at = self._upload([usual, drawn], floats, np.array(cut, dtype=np.int64))
        out = self._launch(logits, rows, *views[:8])
        out[at] = self._draw(logits[at], some, *views[8:], number, min_p)[0]
        return out

    def draw(self, logits: torch.Tensor, params: Sequence[SamplingParams], uniforms: torch.Tensor,
             histories: Sequence[Sequence[int]] | None = None, probabilities: bool = True):
        """Tokens by numbers that the caller brings: logits [rows, vocab], `uniforms` float32 [rows], or [rows, n] for n
        draws of every row (the first tokens of n continuations of one prompt, say), in [0, 1), on the
        device.  Returns (int32 tokens, float32 probabilities that they were drawn with, or None), shaped as `uniforms`."""
        rows = logits.shape[0]
        if not (len(params) == rows == uniforms.shape[0]):
            raise ValueError("one SamplingParams and one row of numbers per logits row is needed")
        views, (min_p,) = self._upload([self._fill(params, [0] * rows, [0] * rows, histories)],
                                       np.array([[p.min_p for p in params]], dtype=np.float32))
        return self._draw(logits, params, *views, uniforms, min_p, probabilities)

    def _draw(self, logits, params, temperature, top_k, top_p, penalty, _seed, _counter, hist_off, hist_tok, uniforms, min_p,
              probabilities=False):
        out = torch.empty(uniforms.shape, dtype=torch.int32, device=self.device)
        prob = torch.empty_like(uniforms) if probabilities else None
        penalised = any(p.repetition_penalty != 1.0 for p in params)
        self.ops.draw_tokens(logits, uniforms, temperature, top_k, top_p, min_p, out, prob=prob,
                             **(dict(penalty=penalty, hist_off=hist_off, hist_tok=hist_tok) if penalised else {}))
        return out, prob

    def _pack(self, params, counters, seeds, histories):
        """The kernel's arguments as views of one uploaded buffer (the block of an all-greedy step is cached with them)."""
        return self._upload([self._fill(params, counters, seeds, histories)])[0]

    def _upload(self, blocks, floats=None, index=None):
        """One copy to the device of blocks from `_fill`, rows of float32 numbers and an index: (the blocks' views, one
        behind the other; the rows; the index)."""
        arrays = [buf for buf, _ in blocks]
        if index is not None:
            arrays.append(index.view(np.int32))              # (8-byte integers: the blocks have even lengths)
        if floats is not None:
            arrays.append(floats.reshape(-1).view(np.int32))
        buf = arrays[0] if len(arrays) == 1 else np.concatenate(arrays)
        self.h2d_bytes_last = buf.nbytes
        dev = torch.from_numpy(buf).to(self.device, non_blocking=True)
        views, at = [], 0
        for block, views_of in blocks:
            views += views_of(dev[at:at + len(block)])
            at += len(block)
        result = [views]
        if floats is not None:
            n, m = floats.shape
            first = len(buf) - n * m
            result.append([dev[first + j * m:first + (j + 1) * m].view(torch.float32) for j in range(n)])
        if index is not None:
            result.append(dev[at:at + 2 * len(index)].view(torch.int64))
        return result

    @staticmethod
    def _fill(params, counters, seeds, histories):
        """Parameters, seeds, counters and histories of rows as int32 numbers, an even number of them, and the function that
        makes the kernel's arguments of their copy on the device."""
        rows = len(params)
        # 4 float/int arrays of `rows`, seeds as two int32 each, offsets, tokens
        hist_off = np.zeros(rows + 1, dtype=np.int64)
        toks: list[np.ndarray] = []
        for i, p in enumerate(params):
            n = 0
            if p.repetition_penalty != 1.0 and histories is not None and len(histories[i]):
                h = np.unique(np.asarray(histories[i], dtype=np.int64))
                toks.append(h)
                n = len(h)
            hist_off[i + 1] = hist_off[i] + n
        n_hist = int(hist_off[-1])
        r8 = -(-rows // 2) * 2
        size = 7 * r8 + 2 + rows + 1 + max(n_hist, 1)
        buf = np.zeros(size + size % 2, dtype=np.int32)
        buf[0:rows].view(np.float32)[:] = [p.temperature for p in params]
        buf[r8:r8 + rows] = [p.top_k for p in params]
        buf[2 * r8:2 * r8 + rows].view(np.float32)[:] = [p.top_p for p in params]
        buf[3 * r8:3 * r8 + rows].view(np.float32)[:] = [p.repetition_penalty for p in params]
        buf[4 * r8:4 * r8 + 2 * rows].view(np.uint64)[:] = np.asarray(
            [int(s) % (1 << 64) for s in seeds], dtype=np.uint64)
        buf[6 * r8:6 * r8 + rows].view(np.uint32)[:] = np.asarray(counters, dtype=np.uint32)
        o = 7 * r8
        buf[o:o + rows + 1] = hist_off
        h = o + rows + 1
        h += h % 2
        if n_hist:
            buf[h:h + n_hist] = np.concatenate(toks)

        def views(dev):
            return (dev[0:rows].view(torch.float32), dev[r8:r8 + rows],
                    dev[2 * r8:2 * r8 + rows].view(torch.float32),
                    dev[3 * r8:3 * r8 + rows].view(torch.float32),
                    dev[4 * r8:4 * r8 + 2 * rows], dev[6 * r8:6 * r8 + rows],
                    dev[o:o + rows + 1], dev[h:h + max(n_hist, 1)])
        return buf, views

    def _launch(self, logits, rows, *views):
        out = torch.empty(rows, dtype=torch.int32, device=self.device)
        self.ops.sample(logits, *views, out)
        return out
