"""GPU: a layer of experts as it is used: routing, the gated product with the gather, the
second product, the weighted sum onto the residual stream, with 16-bit and 4-bit weights,
eager, captured and on another stream. The bound of a run: each operator's own (moe_util),
carried on by the next one's weights."""
import math

import pytest

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, GATE

pytestmark = pytest.mark.gpu
E, K, H, F = 12, 3, 128, 96


class Layer:
    def __init__(self, torch, t, dtype, bits, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.torch, self.t, self.bits = torch, t, bits
        self.x = torch.randn((t, H), generator=g).to(DT[dtype])
        self.logits = torch.randn((t, E), generator=g)
        self.logits[t // 2] = -math.inf  # a padded token
        if bits == 16:
            self.w1 = (torch.randn((E, 2 * F, H), generator=g) / math.sqrt(H)).to(DT[dtype])
            self.w2 = (torch.randn((E, H, F), generator=g) / math.sqrt(F)).to(DT[dtype])
        else:
            self.w1 = moe_util.random_w4(E, 2 * F, H, 64, dtype, seed + 1, True)
            self.w2 = moe_util.random_w4(E, H, F, 32, dtype, seed + 2, False)
        i = dict(dtype=torch.int32, device="cuda")
        self.route = [torch.empty((t, K), **i), torch.empty((t, K), device="cuda"), torch.empty(E + 1, **i),
                      torch.empty(t * K, **i), torch.empty(t * K, **i)]
        h = dict(dtype=DT[dtype], device="cuda")
        self.h, self.y, self.out = torch.empty((t * K, F), **h), torch.empty((t * K, H), **h), torch.empty((t, H), **h)
        self.h.fill_(float("nan"))  # rows without an expert are never read
        self.y.fill_(float("nan"))
        self.ws = pyc_amd.moe_route_workspace(t, E, K)
        on = lambda w: w.cuda() if bits == 16 else [None if v is None else v.cuda() for v in w]  # noqa: E731
        self.dev = self.x.cuda(), self.logits.cuda(), on(self.w1), on(self.w2)

    def run(self):
        x, logits, w1, w2 = self.dev
        _, weights, offsets, rows, places = self.route
        pyc_amd.moe_route(logits, *self.route, workspace=self.ws)
        if self.bits == 16:
            pyc_amd.grouped_gemm(x, w1, offsets, self.h, rows=rows, fan=K, epilogue=GATE)
            pyc_amd.grouped_gemm(self.h, w2, offsets, self.y)
        else:
            pyc_amd.w4a16_grouped_gemm(x, w1[0], w1[1], offsets, self.h, zeros=w1[2], rows=rows, fan=K, epilogue=GATE)
            pyc_amd.w4a16_grouped_gemm(self.h, w2[0], w2[1], offsets, self.y)
        pyc_amd.moe_combine(self.y, weights, places, self.out, base=x)

    def reference(self):
        """(out, bound) in 64 bits."""
        torch = self.torch
        values = lambda w: (w.double(), None) if self.bits == 16 else (  # noqa: E731
            lambda v: (v[0] * v[1], (80 if self.x.dtype == torch.bfloat16 else 288) * v[1].abs()))(moe_util.w4_values(*w))
        (w1, s1), (w2, s2) = values(self.w1), values(self.w2)
        r = moe_util.route_ref(self.logits, K, True)
        like = lambda n: torch.zeros((self.t * K, n), dtype=self.x.dtype)  # noqa: E731
        h, dh = moe_util.product_ref(self.x, w1, r["offsets"], like(F), r["rows"], K, epi=GATE, spread=s1)
        out, bound = self.x.double().clone(), torch.zeros((self.t, H), dtype=torch.float64)
        for e in range(E):
            for p in range(r["offsets"][e], r["offsets"][e + 1]):
                t, j = divmod(int(r["rows"][p]), K)
                y = w2[e] @ h[p]
                s = (w2[e].abs() if s2 is None else s2[e]) @ (h[p].abs() + dh[p])
                dy = w2[e].abs() @ dh[p] + (F + 4) * moe_util.U * s
                dy = moe_util.rounded(y, dy, self.x.dtype)
                a = float(r["weights"][t, j])
                out[t] += a * y
                bound[t] += a * (dy + 64 * moe_util.U * (y.abs() + dy))  # the weight's and the sum's roundings
        bound = bound + (K + 1) * moe_util.U * (out.abs() + self.x.double().abs())
        return out, moe_util.rounded(out, bound, self.x.dtype)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t", [1, 2, 40, 130])
def test_layer(gpu, t, dtype, bits):
    layer = Layer(gpu, t, dtype, bits, seed=t)
    layer.run()
    moe_util.check(layer.out, *layer.reference())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("t", [3, 150])
def test_captured(gpu, t, bits):
    """One capture, other inputs on every replay, the program's own eager work in between."""
    torch = gpu
    layer = Layer(torch, t, "bf16", bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run()
    for seed in range(4):
        other = Layer(torch, t, "bf16", bits, seed=seed + 50)
        layer.dev[0].copy_(other.dev[0])
        layer.dev[1].copy_(other.dev[1])
        for mine, new in zip(layer.dev[2:], other.dev[2:]):
            for a, b in zip([mine] if bits == 16 else mine, [new] if bits == 16 else new):
                if a is not None:
                    a.copy_(b)
        layer.out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        other.run()
        torch.cuda.synchronize()
        assert torch.equal(layer.out, other.out), seed
        assert torch.equal(layer.route[3], other.route[3]), seed


def test_two_streams(gpu):
    """Two layers on two streams at once, each with its own workspace, against the same calls one after the other."""
    torch = gpu
    a, b = Layer(torch, 150, "bf16", 16, 1), Layer(torch, 90, "bf16", 4, 2)
    ref = []
    for layer in (a, b):
        layer.run()
        torch.cuda.synchronize()
        ref.append(layer.out.clone())
        layer.out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for layer, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                layer.run()
    torch.cuda.synchronize()
    assert torch.equal(a.out, ref[0]) and torch.equal(b.out, ref[1])
