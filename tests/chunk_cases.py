"""What the tests of a layer's forward over a bounded cache share: caches in pages or not, in the model dtype or in 8 bits, with their values in 64 bits."""

from __future__ import annotations

import numpy as np
import torch

from oracle import rows as O

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 0.0}  # half a step, relative
U = 2.0**-24


def normal(gen: torch.Generator, shape: tuple, model: str, scale: float = 1.0) -> torch.Tensor:
    loud = torch.where(torch.rand(shape[-1:], generator=gen) < 0.06, 5.0, 0.8)
    return (torch.randn(shape, generator=gen) * loud * scale).to(TYPES[model])


class Cache:
    """`seqs` sequences with room for `n` rows each, filled: in pages of `page` rows in any order with pages of nobody's between them, or (page 0)
    one after the other. `values[0 or 1][b, h, i]` is what row i stands for, in 64 bits. What is nobody's holds NaN."""

    def __init__(self, gen: torch.Generator, seqs: int, h: int, n: int, d: int, model: str, *, eight: bool = False, page: int = 0, room: int = 0) -> None:
        from lazykv_amd import kernels

        self.model, self.eight, self.page, self.shape = model, eight, page, (seqs, h, n, d)
        each = -(-max(n, 1) // page) if page else 0
        if page:
            order = torch.randperm(seqs * each + 2, generator=gen)[: seqs * each]
            self.table = order.view(seqs, each)
            store = (seqs * each + 2, h, page, d)
        else:
            self.table = None
            store = (seqs, h, n + room, d)
        self.pages = None if self.table is None else self.table.int().cuda()
        kv = [normal(gen, (seqs, h, n, d), model), torch.randn((seqs, h, n, d), generator=gen).to(TYPES[model])]
        if eight:
            coded = [O.mx_encode(x.double().numpy(), model) for x in kv]
            self.values = [O.mx_decode(*c) for c in coded]
            codes = torch.full((2, *store), 0x7F, dtype=torch.uint8)
            scales = torch.full((2, *store[:-1], d // 32), 0xFF, dtype=torch.uint8)
            for i, (c, s) in enumerate(coded):
                self._put(codes[i], torch.from_numpy(c).to(torch.float8_e4m3fn).view(torch.uint8))
                self._put(scales[i], torch.from_numpy(s))
            self.held = [codes.cuda(), scales.cuda()]
            self.rows = kernels.mx_rows(*self.held, TYPES[model])
        else:
            self.values = [x.double().numpy() for x in kv]
            both = torch.full((2, *store), float("nan"), dtype=TYPES[model])
            for i, x in enumerate(kv):
                self._put(both[i], x)
            self.held = [both.cuda()]
            self.rows = kernels.dense_rows(self.held[0][0], self.held[0][1])

    def _put(self, store: torch.Tensor, x: torch.Tensor) -> None:
        for b in range(x.shape[0]):
            for i in range(x.shape[2]):
                where, at = self.place(b, i)
                store[where, :, at] = x[b, :, i]

    def place(self, b: int, i: int) -> tuple[int, int]:
        return (b, i) if self.table is None else (int(self.table[b, i // self.page]), i % self.page)

    def read(self, of: list[torch.Tensor] | None = None) -> list[np.ndarray]:
        """What the rows hold now, keys and values [seqs, h, n, d] in 64 bits."""
        held = [x.cpu() for x in (of or self.held)]
        if self.eight:
            codes = held[0].view(torch.float8_e4m3fn).double()
            f = torch.exp2(held[1].double() - 127).repeat_interleave(32, -1)
            store = codes * f
        else:
            store = held[0].double()
        seqs, h, n, d = self.shape
        got = [np.empty((seqs, h, n, d)) for _ in range(2)]
        for b in range(seqs):
            for i in range(n):
                where, at = self.place(b, i)
                for j in range(2):
                    got[j][b, :, i] = store[j, where, :, at].numpy()
        return got


def int32(x: list) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device="cuda")
