"""GPU: plan, append and attention together, as a serving loop uses them: prompts,
then decoding with requests that come and go, eagerly and as one captured graph
whose lengths, tables and queries live on the device."""
import numpy as np
import pytest

import pyc_amd
from tests import kv_util
from tests.kv_util import DT, HALF

pytestmark = pytest.mark.gpu


class Server:
    """A cache, its tables and one step's buffers on the device."""

    def __init__(self, torch, requests, tokens, blocks, bs, hq, hk, d, dtype, width, max_q, seed):
        i32 = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.torch, self.bs, self.dtype, self.max_q = torch, bs, dtype, max_q
        c = kv_util.random_cache(blocks, hk, bs, d, seed)
        self.c = {k: v.cuda() for k, v in c.items()}
        self.cache = pyc_amd.KvCache(self.c["k"], self.c["v"], self.c["k_scale"], self.c["v_scale"])
        self.cached, self.fresh, self.table = i32(requests), i32(requests), i32(requests, width)
        self.free = torch.from_numpy(np.random.default_rng(seed).permutation(blocks).astype(np.int32)).cuda()
        self.count = i32(1)
        self.count[0] = blocks
        self.offsets, self.slots, self.pos = i32(requests + 1), i32(tokens), i32(tokens)
        self.k, self.v, self.q, self.o = (torch.zeros((tokens, h, d), dtype=DT[dtype], device="cuda")
                                          for h in (hk, hk, hq, hq))
        self.ws = pyc_amd.kv_attention_workspace(requests, hq, hk, d, max_q)
        self.scale = d ** -0.5

    def fill(self, fresh, seed):
        torch = self.torch
        self.fresh.copy_(torch.tensor(fresh, dtype=torch.int32))
        g = torch.Generator().manual_seed(seed)
        for x in (self.k, self.v, self.q):
            x.copy_(torch.randn(x.shape, generator=g))
        self.o.fill_(7.0)

    def step(self):
        pyc_amd.kv_plan(self.cached, self.fresh, self.table, self.free, self.count, self.bs, self.cached, self.offsets,
                        self.slots, self.pos, self.count)
        pyc_amd.kv_append(self.k, self.v, self.slots, self.cache)
        pyc_amd.kv_attention(self.q, self.cache, self.table, self.cached, self.offsets, self.o, self.scale, self.max_q,
                             workspace=self.ws)

    def host(self):
        return {n: getattr(self, n).cpu().numpy().copy() for n in ("cached", "fresh", "table", "free", "count")}

    def check(self, before, old):
        """One step's results from the state before it."""
        torch = self.torch
        torch.cuda.synchronize()
        p = kv_util.plan_ref(before["cached"], before["fresh"], before["table"], before["free"], int(before["count"][0]),
                             self.bs, self.slots.numel())
        for name, x in (("table", self.table), ("free", self.free), ("lens", self.cached), ("q_offsets", self.offsets),
                        ("slots", self.slots), ("positions", self.pos), ("free_after", self.count)):
            assert np.array_equal(x.cpu().numpy(), p[name]), name
        ref = kv_util.values(old)
        kv_util.append_ref(ref, self.k.cpu(), self.v.cpu(), p["slots"].tolist())
        now = {k: v.cpu() for k, v in self.c.items()}
        got = kv_util.values(now)
        for name in ref:
            same = torch.equal(got[name], ref[name])
            assert same, name
        o, bound, done = kv_util.attention_ref(self.q.cpu(), now, torch.from_numpy(p["table"]), p["lens"], p["q_offsets"],
                                               self.scale, self.max_q, torch.full(self.q.shape, 7.0))
        g = self.o.cpu().double()
        off = (g - o).abs() - bound * 1.01 - HALF[self.dtype] * o.abs() - 2.0 ** -24
        assert bool((off <= 0).all()), float(off.max())
        assert int(done.sum()) == int(p["q_offsets"][-1])


def _old(s):
    # the two odd scales of random_cache would make code values ambiguous at ties
    return {k: v.cpu().clone() for k, v in s.c.items()}


STEPS = [[20, 33, 0, 1], [1, 1, 47, 1], [1, 5, 1, -1], [-1, 1, 1, 30], [16, 1, -1, 1], [1, 40, 3, 1]]


@pytest.mark.parametrize("dtype,d,bs", [("bf16", 128, 16), ("f16", 64, 32)])
def test_loop(gpu, dtype, d, bs):
    s = Server(gpu, 4, 70, 24, bs, 4, 2, d, dtype, 8, 48, 1)
    s.c["k_scale"][0, 0] = s.c["v_scale"][0, 0] = 0.5
    for i, fresh in enumerate(STEPS):
        s.fill(fresh, i)
        before, old = s.host(), _old(s)
        s.step()
        s.check(before, old)


def test_captured_step(gpu):
    """The whole step captured once: every replay takes the lengths, tables and
    rows that are on the device then, with eager work in between, and equals the
    64-bit step."""
    torch = gpu
    s = Server(torch, 4, 70, 24, 16, 8, 2, 128, "bf16", 8, 48, 2)
    s.c["k_scale"][0, 0] = s.c["v_scale"][0, 0] = 0.5
    s.fill([0, 0, 0, 0], 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.step()
    for i, fresh in enumerate(STEPS):
        s.fill(fresh, i)
        before, old = s.host(), _old(s)
        g.replay()
        s.check(before, old)
        torch.randn(1000, device="cuda").sum().item()


def test_two_captured_steps_in_turn(gpu):
    """Two servers, a graph each with workspaces of their own, replayed on two
    streams at once."""
    torch = gpu
    servers, graphs = [], []
    for i in range(2):
        s = Server(torch, 4, 70, 24, 16, 8, 2, 64, "bf16", 8, 48, 3 + i)
        s.c["k_scale"][0, 0] = s.c["v_scale"][0, 0] = 0.5
        s.fill([0] * 4, 0)
        s.step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.step()
        servers.append(s)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, fresh in enumerate(STEPS):
        states = []
        for j, s in enumerate(servers):
            s.fill(fresh, 10 * i + j)
            states.append((s.host(), _old(s)))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, (before, old) in zip(servers, states):
            s.check(before, old)


def test_decode_alone_as_in_a_batch(gpu):
    """A request's output does not depend on who else is in the batch, beyond the
    order of sums: two results within twice the derived bound of each other."""
    torch = gpu
    s = Server(torch, 4, 70, 24, 16, 4, 2, 64, "bf16", 8, 48, 5)
    s.fill([40, 3, 0, 20], 1)
    s.step()
    torch.cuda.synchronize()
    o = torch.empty_like(s.q[40:43])
    pyc_amd.kv_attention(s.q[40:43], s.cache, s.table[1:2], s.cached[1:2],
                         torch.tensor([0, 3], dtype=torch.int32, device="cuda"), o, s.scale, 3)
    torch.cuda.synchronize()
    ref, bound, _ = kv_util.attention_ref(s.q[40:43].cpu(), {k: v.cpu() for k, v in s.c.items()}, s.table[1:2].cpu(),
                                          [3], [0, 3], s.scale)
    for x in (o, s.o[40:43]):
        off = (x.cpu().double() - ref).abs() - bound * 1.01 - HALF["bf16"] * ref.abs()
        assert bool((off <= 0).all())
