"""Low-rank adapters of many requests at once beside a shared projection (moe_adapter_add): the
projection (ops.affine_linear, TokenHead.logits) runs once for all rows, and each row gets its own
request's correction."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from ._lib import call
from .ops import QMatrix, _launch_on, _need, _stream

MAX_RANK = 128


@dataclass
class AdapterBank:
    """The adapters of one projection of K inputs and N outputs, all of one rank (a smaller one is
    padded with zeros): a bf16 [adapters, rank, K], b bf16 [adapters, N, rank], scale fp32
    [adapters]. rank and K are multiples of 8, rank at most 128."""

    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor

    def __post_init__(self):
        _need(self.a, "a", (torch.bfloat16,))
        _need(self.b, "b", (torch.bfloat16,), self.a.device)
        _need(self.scale, "scale", (torch.float32,), self.a.device)
        if self.a.dim() != 3 or self.b.dim() != 3 or self.scale.dim() != 1:
            raise ValueError("an adapter bank is a [adapters, rank, K], b [adapters, N, rank], scale [adapters]")
        n, r, _ = self.a.shape
        if n < 1 or self.b.shape[0] != n or self.b.shape[2] != r or self.scale.shape[0] != n:
            raise ValueError(f"a {tuple(self.a.shape)}, b {tuple(self.b.shape)} and scale "
                             f"{tuple(self.scale.shape)} do not belong together")
        if r % 8 or not 8 <= r <= MAX_RANK:
            raise ValueError(f"rank {r}: a multiple of 8 up to {MAX_RANK} is needed")

    @property
    def adapters(self) -> int:
        return self.a.shape[0]

    @property
    def rank(self) -> int:
        return self.a.shape[1]

    @property
    def K(self) -> int:
        return self.a.shape[2]

    @property
    def N(self) -> int:
        return self.b.shape[1]

    @property
    def device(self) -> torch.device:
        return self.a.device

    @classmethod
    def synthetic(cls, adapters: int, rank: int, K: int, N: int, device, seed: int = 11,
                  scale: float = 1.0) -> "AdapterBank":
        """Seeded N(0, 1/K) a and N(0, 1/rank) b rows, bf16."""
        dev = torch.device(device)
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        a = (torch.randn((adapters, rank, K), generator=g, device=dev) * K ** -0.5).to(torch.bfloat16)
        b = (torch.randn((adapters, N, rank), generator=g, device=dev) * rank ** -0.5).to(torch.bfloat16)
        return cls(a, b, torch.full((adapters,), float(scale), dtype=torch.float32, device=dev))

    def add(self, y: torch.Tensor, x: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None,
            stream=None) -> torch.Tensor:
        """out[t] = y[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T with a = ids[t]; -1 keeps y[t]. x bf16
        [T, K], y bf16 or fp32 [T, N], ids int32 [T] (device). out may be y."""
        dev = self.device
        _need(x, "x", (torch.bfloat16,), dev)
        _need(y, "y", (torch.bfloat16, torch.float32), dev)
        _need(ids, "ids", (torch.int32,), dev)
        if x.dim() != 2 or x.shape[1] != self.K:
            raise ValueError(f"x has shape {tuple(x.shape)}, expected [T, {self.K}]")
        T = x.shape[0]
        if tuple(y.shape) != (T, self.N) or ids.numel() != T:
            raise ValueError(f"y {tuple(y.shape)} and ids {tuple(ids.shape)} do not fit x [{T}, {self.K}] and "
                             f"N = {self.N}")
        if out is not None:
            _need(out, "out", (y.dtype,), dev)
            if out.shape != y.shape:
                raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(y.shape)}")
        with _launch_on(dev, stream):
            if out is None:
                out = torch.empty_like(y)
            if T:
                call("moe_adapter_add", x.data_ptr(), T, self.K, self.N, self.a.data_ptr(), self.b.data_ptr(),
                     self.scale.data_ptr(), self.adapters, self.rank, ids.data_ptr(), y.data_ptr(),
                     int(y.dtype == torch.float32), out.data_ptr(), _stream(stream, dev))
        return out


def adapter_linear(x: torch.Tensor, w: QMatrix, bank: AdapterBank, ids: torch.Tensor, *, y=None,
                   stream=None) -> torch.Tensor:
    """affine_linear(x, w) with each row's adapter of `bank` added: y [T, N] for x [T, K]."""
    with _launch_on(x.device, stream):
        y = ops.affine_linear(x, w, y=y, stream=stream)
        return bank.add(y, x, ids, out=y, stream=stream)
