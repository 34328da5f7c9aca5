"""Offsets that do not rise from 0 to the number of rows: bounds are cut to [0, rows], one that
falls counts as the largest before it, so that every row belongs to one expert at most; rows of
none are left alone. Results against 64 bits in every kernel that reads offsets."""
from __future__ import annotations

import pytest
import torch

import raggedroute_amd as rr
from block_helpers import ACTIVATIONS, Buf, assert_within
from test_gpu_block_ffn import backward, check_forward, forward, grads, make
from test_gpu_block_int8 import FAMILIES, context

pytestmark = pytest.mark.gpu

# offsets in units of a size, to be cut to 10 of them
OFFSETS = {
    "start": [3, 5, 5, 8],
    "end": [0, 2, 4, 7],
    "falls": [0, 5, 1, 3, 8, 2],
    "falls last": [0, 4, 9, 6],
    "falls and rises again": [0, 6, 0, 6, 0, 9],
    "outside": [-4, 3, 40, 2],
    "many falls": [2, 6] + [0, 6] * 40 + [0, 7],
}


def bounds(offsets, rows):
    """First row and one past the last of every expert."""
    most, out = 0, []
    for o in offsets:
        most = max(most, min(max(o, 0), rows))
        out.append(most)
    return out


class Rows:
    """The rows of an output from `first` on."""

    def __init__(self, buf, first):
        self.buf, self.first = buf, first

    @property
    def t(self):
        return self.buf.t[self.first:]


# (unit, k, f, n): split sums and few rows; few rows; short tiles; tiles of 128 and of 256 rows; through registers
SIZES = [(1, 2048, 2048, 48), (1, 256, 96, 264), (14, 96, 136, 72), (40, 64, 264, 128), (300, 72, 40, 64), (33, 45, 67, 31)]


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("unit,k,f,n", SIZES)
@pytest.mark.parametrize("name", list(OFFSETS))
def test_ffn(device, name, unit, k, f, n, family):
    rows = 10 * unit
    offsets = [unit * o for o in OFFSETS[name]]
    counts = [rows] + [0] * (len(offsets) - 2)
    v, b, _ = make(counts, k, f, n, "bf16", seed=len(offsets) + unit)
    b["offsets"] = Buf(torch.tensor(offsets, dtype=torch.int32, device="cuda:0"))
    m = bounds(offsets, rows)
    experts = [to - at for at, to in zip(m, m[1:])]
    out = forward(b, experts, rows, k, f, n, "bf16", family=family)
    ofmine = {**v, "x": v["x"][m[0]:]}
    check_forward(ofmine, {key: Rows(buf, m[0]) for key, buf in out.items()}, experts, "bf16", "silu")
    grad = backward(b, experts, rows, k, f, n, "bf16", family=family)
    for e, (at, to) in enumerate(zip(m, m[1:])):
        want, bound = grads(v, experts, e, slice(at, to), "bf16", "silu")
        for key in want:
            got = grad[key].t[at:to] if key == "dx" else grad[key].t[e]
            assert_within(got, want[key], bound[key], f"{key} of expert {e}")
    for buf in (out["act"], out["y"], out["gate"], grad["dx"]):
        assert buf.untouched(slice(0, m[0])) and buf.untouched(slice(m[-1], None))


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("unit,k,n", [(1, 256, 72), (40, 144, 136), (300, 64, 72), (33, 45, 67)])
@pytest.mark.parametrize("name", list(OFFSETS))
def test_int8(device, name, unit, k, n, family):
    """Sums of at most 100 products of one: exact in FP32."""
    rows = 10 * unit
    offsets = [unit * o for o in OFFSETS[name]]
    m = bounds(offsets, rows)
    e = len(m) - 1
    q = Buf(torch.ones(rows, k, dtype=torch.int8, device="cuda:0"))
    w = Buf((torch.arange(e, device="cuda:0") + 1).to(torch.int8)[:, None, None].expand(e, n, k).contiguous())
    qs, ws = Buf(torch.ones(rows, device="cuda:0")), Buf(torch.ones(e, n, device="cuda:0"))
    offs, y = Buf(torch.tensor(offsets, dtype=torch.int32, device="cuda:0")), Buf(shape=(rows, n), dtype=torch.float32)
    args = rr.Int8GroupedGemmArgs(q=q.ptr, q_scale=qs.ptr, w=w.ptr, w_scale=ws.ptr, offsets=offs.ptr, y=y.ptr, rows=rows,
                                  experts=e, hidden=k, output=n, dtype=int(rr.ScalarType.kFp32),
                                  activation=int(ACTIVATIONS["silu"][0]), kernel=FAMILIES[family])
    ctx, _ = context(rr.get_int8_grouped_gemm_workspace_size(args))
    status = rr.int8_grouped_gemm(args, ctx)
    assert status.ok(), status.message
    assert y.intact()
    for i, (at, to) in enumerate(zip(m, m[1:])):
        assert (y.t[at:to] == k * (i + 1)).all(), i
    assert y.untouched(slice(0, m[0])) and y.untouched(slice(m[-1], None))
