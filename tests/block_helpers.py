"""Device buffers with red zones and small tools for the expert block's tests."""
from __future__ import annotations

import torch

import raggedroute_amd as rr

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": int(rr.ScalarType.kFp32), "f16": int(rr.ScalarType.kFp16), "bf16": int(rr.ScalarType.kBf16)}
# half a unit in the last place, relative, and absolutely below the normal numbers
ROUNDING = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -140, "f16": 2.0 ** -25, "bf16": 2.0 ** -130}

ZONE = 256
CANARY = 0xA5


class Buf:
    """A tensor `offset` elements past a 256-byte boundary between two red zones."""

    def __init__(self, value=None, shape=None, dtype=None, device="cuda:0", offset=0):
        if value is not None:
            shape, dtype = value.shape, value.dtype
        size = torch.empty(0, dtype=dtype).element_size()
        count = 1
        for n in shape:
            count *= n
        self.begin = ZONE + offset * size
        self.end = self.begin + count * size
        self.raw = torch.full((self.end + ZONE,), CANARY, dtype=torch.uint8, device=device)
        # (a copy where the payload's start is not aligned for a view of the raw bytes)
        self.shape, self.dtype, self.size = tuple(shape), dtype, size
        if value is not None:
            flat = value.contiguous().reshape(-1).view(torch.uint8) if count else value.new_empty(0, dtype=torch.uint8)
            self.raw[self.begin:self.end] = flat
        self.ptr = self.raw.data_ptr() + self.begin

    @property
    def t(self) -> torch.Tensor:
        torch.cuda.synchronize()
        return self.raw[self.begin:self.end].clone().view(self.dtype).reshape(self.shape)

    def intact(self) -> bool:
        torch.cuda.synchronize()
        return bool((self.raw[:self.begin] == CANARY).all() and (self.raw[self.end:] == CANARY).all())

    def untouched(self, rows: slice) -> bool:
        """Whether rows of an output still hold the fill."""
        t = self.t[rows].contiguous().view(torch.uint8)
        return bool((t == CANARY).all())


def context(workspace_bytes=0, stream=None):
    """A runtime context with a workspace of exactly that size between red zones; (context, buffer)."""
    ws = Buf(shape=(max(16, workspace_bytes),), dtype=torch.uint8)
    stream = stream if stream is not None else torch.cuda.current_stream()
    return rr.RuntimeContext(stream=stream.cuda_stream, workspace=ws.ptr, workspace_bytes=workspace_bytes,
                             architecture=int(rr.DeviceArchitecture.kGfx950)), ws


def offsets_of(counts, device="cuda:0"):
    total, out = 0, [0]
    for c in counts:
        total += c
        out.append(total)
    return torch.tensor(out, dtype=torch.int32, device=device), total


def segments(counts):
    row = 0
    for e, c in enumerate(counts):
        yield e, slice(row, row + c)
        row += c


def assert_within(got, want, bound, what):
    """Every value within its own error bound (64 bits)."""
    got = got.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    if worst > 0:
        at = over.argmax().item()
        raise AssertionError(f"{what}: {got.reshape(-1)[at].item()} for {want.reshape(-1)[at].item()}, "
                             f"{worst:.3g} past its bound {bound.reshape(-1)[at].item():.3g}")


def silu(g):
    return g * torch.sigmoid(g)


def gelu(g):
    return g * torch.sigmoid(2.0 * (2.0 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))


ACTIVATIONS = {"silu": (rr.Activation.kSilu, silu), "gelu": (rr.Activation.kGeluTanh, gelu)}
