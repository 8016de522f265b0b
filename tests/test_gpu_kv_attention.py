"""GPU: attention over the paged 8-bit cache (pyc_hip_kv_attention_dispatch)
against kv_util.attention_ref in 64 bits. An output may be off by what
attention_ref derives (scores, sums and the rounding of P) plus half a step of the
output's type; f16's step does not go below 2^-24."""
import numpy as np
import pytest

import pyc_amd
from tests import kv_util
from tests.kv_util import DT, HALF

pytestmark = pytest.mark.gpu


def _tables(lens, bs, blocks, seed, width=None):
    r = np.random.default_rng(seed)
    ids = r.permutation(blocks)
    need = [kv_util.ceil_div(n, bs) for n in lens]
    width = width or max(max(need), 1)
    t = np.full((len(lens), width), -1, np.int64)  # what is not a request's is no block
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return t


class Call:
    """A batch: lens (the step's tokens among them), counts of tokens."""

    def __init__(self, torch, dtype, hq, hk, d, bs, lens, counts, seed=0, gain=1.0, blocks=None, width=None):
        self.torch, self.dtype, self.d = torch, dtype, d
        need = sum(kv_util.ceil_div(n, bs) for n in lens)
        self.blocks = blocks or need + 1
        self.cache = kv_util.random_cache(self.blocks, hk, bs, d, seed + 1)
        self.table = torch.from_numpy(_tables(lens, bs, self.blocks, seed, width)).to(torch.int32)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.offsets = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32)
        self.max_q = max(max(counts), 1)
        g = torch.Generator().manual_seed(seed + 2)
        self.q = (torch.randn((max(int(sum(counts)), 1), hq, d), generator=g) * gain).to(DT[dtype])
        self.scale = d ** -0.5

    def handle(self):
        return pyc_amd.KvCache(*(self.cache[n].cuda() for n in ("k", "v", "k_scale", "v_scale")))

    def run(self, max_len=0, max_q=None, fill=7.0, workspace=None):
        torch = self.torch
        o = torch.full(self.q.shape, fill, dtype=self.q.dtype, device="cuda")
        pyc_amd.kv_attention(self.q.cuda(), self.handle(), self.table.cuda(), self.lens.cuda(), self.offsets.cuda(), o,
                             self.scale, max_q or self.max_q, max_len=max_len, workspace=workspace)
        torch.cuda.synchronize()
        return o.cpu()

    def check(self, got, max_q=1 << 30, fill=7.0, only=None):
        torch = self.torch
        ref, bound, done = kv_util.attention_ref(self.q, self.cache, self.table, self.lens, self.offsets, self.scale, max_q,
                                                 torch.full(self.q.shape, fill), only)
        g = got.double()
        if only is not None:  # the rows looked at
            g, ref, bound, done = g[done], ref[done], bound[done], done[done]
            got = got[:0]
            done = done[:0]
        same_nan = torch.equal(torch.isnan(g), torch.isnan(ref))
        assert same_nan, "NaN in other places"
        room = bound * (1 + HALF[self.dtype]) + HALF[self.dtype] * ref.abs() + 2.0 ** -24
        off = torch.where(torch.isnan(ref), torch.zeros_like(ref), (g - ref).abs() - room)
        assert bool((off <= 0).all()), (float(off.max()), int((off > 0).sum()))
        left = torch.equal(got[~done], torch.full_like(got, fill)[~done])
        assert left, "rows of nobody were written"
        return ref

    def go(self, **kw):
        got = self.run(**kw)
        self.check(got, kw.get("max_q") or 1 << 30)
        return got


HEADS = [(1, 1), (4, 4), (8, 2), (32, 8), (12, 12), (16, 1), (40, 8), (24, 1)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", HEADS)
def test_single_tokens(gpu, dtype, d, hq, hk):
    """Decoding: lengths around 0, a chunk of 16, a tile of 64 and a block."""
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 0, 513]
    Call(gpu, dtype, hq, hk, d, 16 if d == 128 else 32, lens, [1] * len(lens), seed=hq).go()


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_blocks(gpu, bs, d):
    lens = [bs - 1, bs, bs + 1, 3 * bs + 7, 70, 1000]
    Call(gpu, "bf16", 8, 2, d, bs, lens, [1] * 6, seed=bs, width=90).go()
    Call(gpu, "f16", 8, 2, d, bs, lens, [3, 1, 5, 2, 4, 7], seed=bs).go()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (4, 4, 64), (16, 1, 64), (5, 5, 128)])
@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 15, 16, 17, 33])
def test_draft_tokens(gpu, dtype, hq, hk, d, n):
    """A few tokens a request: rows of several tokens and heads share a tile."""
    lens = [n, n + 1, 64, 65 + n, 300, 129]
    counts = [n, max(1, n - 1), 1, n, n, max(1, n // 2)]
    Call(gpu, dtype, hq, hk, d, 16, lens, counts, seed=n).go()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hk,d,bs", [(8, 2, 128, 16), (4, 4, 64, 64), (6, 2, 128, 32), (8, 1, 64, 128)])
def test_prompt_chunks(gpu, dtype, hq, hk, d, bs):
    """Chunks of prompts, with and without a cached beginning, whose rows and keys
    end inside tiles, beside requests that bring one token or none."""
    lens = [100, 257, 500, 128, 333, 64, 90]
    counts = [100, 130, 67, 128, 1, 64, 0]
    Call(gpu, dtype, hq, hk, d, bs, lens, counts, seed=bs).go()


def test_long_chunk(gpu):
    Call(gpu, "bf16", 8, 2, 128, 16, [1500, 900], [700, 513], seed=3).go()


def _some(counts, seed, many=10):
    """Some tokens of every request: the first and last two, and others."""
    r, some, at = np.random.default_rng(seed), set(), 0
    for n in counts:
        pick = [0, 1, n - 2, n - 1] + r.integers(0, n, many).tolist() if n else []
        some |= {at + int(i) for i in pick if 0 <= i < n}
        at += n
    return some


# Enough rows that a part of them is 256 (parts of 128 would take two rounds of 256
# workgroups, these one), tables of more than 32 tiles, and requests that end inside a part.
WIDE = [(32, 8, 16, [4700, 2300], [1024, 1003]), (24, 8, 128, [4200, 1000], [1300, 999]),
        (64, 64, 64, [700], [600]), (40, 8, 32, [3000, 500, 2200], [500, 400, 470])]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hk,bs,lens,counts", WIDE)
def test_long_prompts(gpu, dtype, hq, hk, bs, lens, counts):
    c = Call(gpu, dtype, hq, hk, 128, bs, lens, counts, seed=20 + bs)
    c.check(c.run(), only=_some(counts, bs))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,bs", [(64, 16), (64, 128), (128, 16), (128, 128)])
def test_chunks_over_long_contexts(gpu, dtype, d, bs):
    lens, counts = [4700, 5000, 2049], [300, 260, 257]
    c = Call(gpu, dtype, 8, 2, d, bs, lens, counts, seed=30 + d + bs)
    c.check(c.run(), only=_some(counts, d + bs, 20))


@pytest.mark.parametrize("hq,hk,d,lens,counts", [(32, 8, 128, [1500, 1300], [1000, 900]), (8, 2, 64, [700, 300], [300, 200]),
                                                 (8, 2, 128, [900, 300, 2000], [200, 1, 1]), (8, 2, 128, [90, 3000], [1, 1])])
def test_captured_calls_follow_lengths(gpu, hq, hk, d, lens, counts):
    """A captured call of every kind, replayed with other lengths between eager work:
    each replay is the eager call's result, bit for bit."""
    torch = gpu
    c = Call(torch, "bf16", hq, hk, d, 16, lens, counts, seed=50)
    cache, q, table, offsets = c.handle(), c.q.cuda(), c.table.cuda(), c.offsets.cuda()
    now, o = c.lens.cuda(), torch.zeros(c.q.shape, dtype=c.q.dtype, device="cuda")
    work = pyc_amd.kv_attention_workspace(len(lens), hq, hk, d, c.max_q)
    call = lambda out, ws: pyc_amd.kv_attention(q, cache, table, now, offsets, out, c.scale, c.max_q, workspace=ws)
    call(o, work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(o, work)
    for shorter in (0, 1, 17, 0, 64):
        now.copy_(torch.clamp(c.lens - shorter, min=0).cuda())
        o.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(o, 3.0)
        call(eager, None)
        torch.cuda.synchronize()
        assert torch.equal(o, eager), shorter


# (heads, kv heads, lens, counts): the split kernel's two tilings, parts of 128 and of 256 rows
KINDS = [(4, 2, [70, 200, 130], [1, 1, 1]), (8, 2, [70, 200, 130], [3, 9, 5]), (8, 2, [700, 300], [300, 200]),
         (32, 8, [1500, 1300], [1000, 900])]


@pytest.mark.parametrize("hq,hk,lens,counts", KINDS)
def test_scales_of_any_value(gpu, hq, hk, lens, counts):
    """Scales that are no powers of two, negative, zero, and far from one; the blocks of
    nobody hold NaN."""
    torch = gpu
    c = Call(torch, "bf16", hq, hk, 128, 16, lens, counts, seed=41)
    n = c.blocks
    g = torch.Generator().manual_seed(5)
    for name in ("k_scale", "v_scale"):
        c.cache[name] *= 0.5 + torch.rand((n, hk), generator=g)
    at = c.table.flatten()
    at = at[at >= 0].long()
    c.cache["v_scale"][at[1::7]] = 0.0
    c.cache["v_scale"][at[2::7]] *= -1.0
    c.cache["v_scale"][at[3::7]] *= 2.0 ** -90
    c.cache["k_scale"][at[4::7]] *= -1.0
    c.cache["k_scale"][at[5::7]] = 0.0
    c.cache["v_scale"][at[6::14]] *= 2.0 ** 70
    nobody = sorted(set(range(n)) - set(at.tolist()))
    for i in nobody:
        c.cache["k"][i], c.cache["v"][i] = 0x7F, 0xFF
        c.cache["k_scale"][i], c.cache["v_scale"][i] = float("nan"), float("-inf")
    c.check(c.run(), only=_some(counts, 3))


@pytest.mark.parametrize("hq,hk,lens,counts", KINDS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_queries_of_any_value(gpu, dtype, hq, hk, lens, counts):
    """Rows of q with one large element, of zeros, of tiny ones, with NaN and infinities."""
    torch = gpu
    c = Call(torch, dtype, hq, hk, 128, 16, lens, counts, seed=42, gain=0.25)
    n = c.q.shape[0]
    row = lambda i: i * (n - 1) // 6
    c.q[row(0), :, 17] = 300.0
    c.q[row(1), 0] = 0.0
    c.q[row(2), 1] *= 2.0 ** -13
    if n > 6:
        c.q[row(3), hq - 1, 5] = float("nan")
        c.q[row(4), 0, 99] = float("inf")
        c.q[row(5), 1, 3] = float("-inf")
    ref = c.check(c.run(), only={row(i) for i in range(7)} | _some(counts, 4))
    assert n <= 6 or int(torch.isnan(ref).sum()) >= 128


@pytest.mark.parametrize("hq,hk,lens,counts", KINDS[1:])
def test_nan_values_in_any_tile(gpu, hq, hk, lens, counts):
    """NaN codes among the values all over the keys: only the rows that see them, only
    their channels."""
    torch = gpu
    c = Call(torch, "bf16", hq, hk, 128, 16, lens, counts, seed=43)
    for b in range(len(lens)):
        for i, key in enumerate(range(lens[b] - counts[b] + 1, lens[b], 67)):
            c.cache["v"][c.table[b, key // 16], i % hk, (37 * i) % 128, key % 16] = 0x7F if i & 1 else 0xFF
    ref = c.check(c.run(), only=_some(counts, 5, 20))
    nan = torch.isnan(ref)
    assert bool(nan.any()) and not bool(nan.all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_axis(gpu, dtype):
    """Few rows over long contexts: the work is split along the keys."""
    for hint in (0, 20001):
        Call(gpu, dtype, 8, 2, 128, 64, [20001, 3, 9000], [1, 1, 2], seed=5, width=400).go(max_len=hint)


@pytest.mark.parametrize("hint", [0, 1, 100, 5000, 1 << 30])
def test_hint_is_only_a_hint(gpu, hint):
    Call(gpu, "bf16", 8, 2, 128, 16, [5000, 17, 800], [1, 1, 1], seed=6).go(max_len=hint)


def test_many_requests(gpu):
    r = np.random.default_rng(0)
    lens = r.integers(0, 150, 700).tolist()
    Call(gpu, "bf16", 2, 1, 64, 16, lens, [1] * 700, seed=7).go()


@pytest.mark.parametrize("gain", [0.01, 8.0, 40.0])
def test_flat_and_peaked(gpu, gain):
    """Scores from almost equal to a single key taking all."""
    for dtype in ("bf16", "f16"):
        Call(gpu, dtype, 8, 2, 128, 16, [777, 90], [1, 40], seed=8, gain=gain).go()


def test_rows_without_keys(gpu):
    """More tokens than keys: the first rows see nothing and are zero; a request
    without keys, rows between and behind requests."""
    torch = gpu
    c = Call(torch, "bf16", 4, 2, 64, 16, [3, 0, 40, 0], [5, 2, 1, 70], seed=9)
    c.go()
    c = Call(torch, "bf16", 4, 2, 64, 16, [30, 0, 40], [5, 2, 1], seed=9)
    c.q = torch.cat([c.q, c.q])  # rows behind the last request
    c.go()


def test_rows_past_max_q(gpu):
    """max_q smaller than a request's tokens: its first rows as ever, the others left."""
    c = Call(gpu, "bf16", 8, 2, 128, 16, [100, 60], [9, 3], seed=10)
    c.go(max_q=4)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [6, 1, 20], [40, 90, 3]])
def test_garbage_in_masked_places(gpu, dtype, counts):
    """NaN codes behind a request's last token, NaN and infinite scales and NaN
    codes in blocks that are nobody's: no trace of them."""
    torch = gpu
    lens = [70, 100, 45]
    c = Call(torch, dtype, 8, 2, 64, 32, lens, counts, seed=11, blocks=20)
    c.go()
    used = set()
    for b, n in enumerate(lens):
        ids = c.table[b, :kv_util.ceil_div(n, 32)].tolist()
        used |= set(ids)
        c.cache["k"][ids[-1], :, n % 32 or 32:, :] = 0x7F
        c.cache["v"][ids[-1], :, :, n % 32 or 32:] = 0xFF
    for i in set(range(20)) - used:
        c.cache["k"][i], c.cache["v"][i] = 0x7F, 0x7F
        c.cache["k_scale"][i], c.cache["v_scale"][i] = float("nan"), float("inf")
    c.go()


@pytest.mark.parametrize("counts", [[3, 5], [40, 70]])
def test_nan_that_some_rows_see(gpu, counts):
    """A NaN code of a value among the step's own tokens: NaN in that channel for
    the rows that see the token, nothing for the rows before it; a NaN key makes
    its rows NaN."""
    torch = gpu
    lens = [80, 130]
    c = Call(torch, "bf16", 4, 2, 64, 16, lens, counts, seed=12)
    at = lens[0] - counts[0] + 1  # the second token of the first request
    c.cache["v"][c.table[0, at // 16], 1, 5, at % 16] = 0x7F
    ref = c.check(c.run())
    assert bool(torch.isnan(ref[1:counts[0], 2:, 5]).all()) and not bool(torch.isnan(ref[0]).any())
    at = lens[1] - counts[1] + 2
    c.cache["k"][c.table[1, at // 16], 0, at % 16, 7] = 0x7F
    ref = c.check(c.run())
    first = counts[0]
    assert bool(torch.isnan(ref[first + 2:, :2]).all()) and not bool(torch.isnan(ref[first:first + 2]).any())


def test_nan_query(gpu):
    """A NaN in one row of q stays in that row and head."""
    torch = gpu
    c = Call(torch, "bf16", 8, 2, 64, 16, [50, 60], [1, 9], seed=13)
    c.q[4, 3, 9] = float("nan")
    ref = c.check(c.run())
    assert int(torch.isnan(ref).sum()) == 64


def test_blocks_outside_the_cache(gpu):
    """Ids outside the cache: their keys count as absent; with none left, zero."""
    torch = gpu
    c = Call(torch, "bf16", 8, 2, 64, 16, [80, 40, 16], [1, 2, 1], seed=14)
    c.table[0, 1], c.table[0, 4], c.table[1, 0], c.table[2, 0] = -1, c.blocks, 1 << 30, -(1 << 31)
    c.go()


def test_lengths_outside_the_table(gpu):
    """A length past the table's row is the row's, a negative one nothing; offsets
    past the rows of q end with them."""
    torch = gpu
    c = Call(torch, "bf16", 4, 1, 64, 16, [48, 20, 33], [1, 1, 1], seed=15)
    c.table[0] = torch.tensor([0, 1, 2], dtype=torch.int32)
    c.lens[0], c.lens[1] = 5000, -3
    c.go()
    o = torch.full(c.q.shape, 7.0, dtype=c.q.dtype, device="cuda")
    pyc_amd.kv_attention(c.q.cuda(), c.handle(), c.table.cuda(), c.lens.cuda(),
                         torch.tensor([-5, 2, 1000, 900], dtype=torch.int32).cuda(), o, c.scale, 4)
    torch.cuda.synchronize()


def test_strided_rows_and_blocks(gpu):
    """q as a part of a fused projection, o as a part of a wider row, blocks that
    lie apart, a table that is part of a wider one."""
    torch = gpu
    c = Call(torch, "bf16", 4, 2, 64, 16, [70, 33], [2, 1], seed=16)
    whole = c.run()
    wide = torch.randn((3, 8, 64), device="cuda").to(torch.bfloat16)
    wide[:, :4] = c.q.cuda()
    out = torch.full((3, 6, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    n = 2 * 16 * 64
    room = torch.full((c.blocks, 2 * n + 32), 0x7F, dtype=torch.uint8, device="cuda")
    k, v = room[:, :n].unflatten(1, (2, 16, 64)), room[:, n + 16:2 * n + 16].unflatten(1, (2, 64, 16))
    k.copy_(c.cache["k"])
    v.copy_(c.cache["v"])
    h = pyc_amd.KvCache(k, v, c.cache["k_scale"].cuda(), c.cache["v_scale"].cuda())
    t = torch.full((2, 12), -1, dtype=torch.int32, device="cuda")
    t[:, :5] = c.table.cuda()
    pyc_amd.kv_attention(wide[:, :4], h, t[:, :5], c.lens.cuda(), c.offsets.cuda(), out[:, 2:], c.scale, 2)
    torch.cuda.synchronize()
    assert torch.equal(out[:, 2:].cpu(), whole) and bool((out[:, :2] == 7.0).all())


def test_far_blocks(gpu):
    """Blocks past 2^32 bytes from the cache's beginning."""
    torch = gpu
    c = Call(torch, "bf16", 4, 1, 64, 16, [90], [1], seed=17, blocks=6)
    far = [torch.empty(6 << 30, dtype=torch.uint8, device="cuda").as_strided((6, 1) + s, (1 << 30, 1024) + t)
           for s, t in (((16, 64), (64, 1)), ((64, 16), (16, 1)))]
    far[0].copy_(c.cache["k"])
    far[1].copy_(c.cache["v"])
    h = pyc_amd.KvCache(far[0], far[1], c.cache["k_scale"].cuda(), c.cache["v_scale"].cuda())
    o = torch.empty(c.q.shape, dtype=c.q.dtype, device="cuda")
    pyc_amd.kv_attention(c.q.cuda(), h, c.table.cuda(), c.lens.cuda(), c.offsets.cuda(), o, c.scale, 1)
    torch.cuda.synchronize()
    c.check(o.cpu())


def test_workspace_kept_and_made(gpu):
    """A kept workspace over calls of different shapes, and one made for the call:
    the same results, bit for bit, each time."""
    torch = gpu
    ws = pyc_amd.kv_attention_workspace(8, 32, 8, 128, 64)
    for lens, counts, hq, hk, d in (([3000, 10], [1, 1], 32, 8, 128), ([200] * 8, [5] * 8, 8, 8, 64),
                                    ([4000], [64], 16, 4, 128), ([3000, 10], [1, 1], 32, 8, 128)):
        c = Call(torch, "bf16", hq, hk, d, 16, lens, counts, seed=18)
        a = c.run(workspace=ws)
        assert torch.equal(a, c.run()) and torch.equal(a, c.run(workspace=ws))
        c.check(a)


def test_workspace_of_the_largest_step(gpu):
    """One workspace, made for 2048 tokens a request, for steps of fewer: what a call
    of the same shape with a workspace of its own gives, bit for bit, each time."""
    torch = gpu
    ws = pyc_amd.kv_attention_workspace(32, 32, 8, 128, 2048)
    for n in (4, 12, 16, 17, 300, 9, 1):
        lens = [n + 61 * i % 700 for i in range(32)]
        counts = [n if i % 5 == 0 or n < 20 else 1 + i % 16 for i in range(32)]
        c = Call(torch, "bf16", 32, 8, 128, 16, lens, counts, seed=60 + n)
        a = c.run(workspace=ws)
        assert torch.equal(a, c.run()) and torch.equal(a, c.run(workspace=ws)), n
        c.check(a, only=set(list(_some(counts, n, 0))[::7]))


def test_short_workspace_is_refused(gpu):
    torch = gpu
    c = Call(torch, "bf16", 8, 2, 64, 16, [80], [1], seed=19)
    with pytest.raises(pyc_amd.PycError):
        c.run(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"))


def test_other_stream(gpu):
    """On a stream of its own, as torch's current one and as an argument."""
    torch = gpu
    c = Call(torch, "bf16", 8, 2, 128, 16, [900, 40], [1, 3], seed=20)
    ref = c.run()
    s = torch.cuda.Stream()
    args = (c.q.cuda(), c.handle(), c.table.cuda(), c.lens.cuda(), c.offsets.cuda())
    o = torch.empty((2,) + tuple(c.q.shape), dtype=c.q.dtype, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pyc_amd.kv_attention(*args, o[0], c.scale, 3)
    pyc_amd.kv_attention(*args, o[1], c.scale, 3, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(o[0].cpu(), ref) and torch.equal(o[1].cpu(), ref)


def test_resources_match_the_code_object(gpu):
    """What the registry says of the cache's kernels against the loaded code object."""
    for sym in ("hip_kv_plan", "hip_kv_append_bf16", "hip_kv_append_f16", "hip_kv_attention_bf16", "hip_kv_attention_f16"):
        r = pyc_amd.kernel_resources(sym)
        assert r.device == 1 and r.lds_bytes == r.attr_lds_bytes and r.attr_max_threads >= r.threads, sym
        assert r.waves_per_simd == r.attr_blocks_per_cu * (r.threads // 64) / 4, (sym, r.waves_per_simd, r.attr_blocks_per_cu)
        assert r.attr_scratch_bytes == 0, sym


def _us(torch, f, n=12):
    """The shortest of n calls, with the GPU waited for."""
    best = float("inf")
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, 1000.0 * a.elapsed_time(b))
    return best


class Timed:
    """A batch's call on the device, with codes of any value below NaN. q may have more rows than the requests."""

    def __init__(self, torch, lens, counts, max_q=None, rows=None, hq=32, hk=8, d=128, bs=16):
        need = sum(kv_util.ceil_div(n, bs) for n in lens) + 1
        g = torch.Generator(device="cuda").manual_seed(7)
        k = torch.randint(0, 0x78, (need, hk, bs, d), dtype=torch.uint8, device="cuda", generator=g)
        v = torch.randint(0, 0x78, (need, hk, d, bs), dtype=torch.uint8, device="cuda", generator=g)
        s = torch.full((need, hk), 2.0 ** -9, device="cuda")
        self.cache = pyc_amd.KvCache(k, v, s, s.clone())
        self.table = torch.from_numpy(_tables(lens, bs, need, 7)).to(torch.int32).cuda()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.lens, self.offsets = i32(lens), i32([0] + np.cumsum(counts).tolist())
        self.q = torch.randn((rows or sum(counts), hq, d), generator=g, device="cuda").to(torch.bfloat16)
        self.o, self.max_q, self.scale = torch.empty_like(self.q), max_q or max(counts), d ** -0.5
        self.work = pyc_amd.kv_attention_workspace(len(lens), hq, hk, d, self.max_q)

    def __call__(self):
        pyc_amd.kv_attention(self.q, self.cache, self.table, self.lens, self.offsets, self.o, self.scale, self.max_q,
                             workspace=self.work)


def test_a_token_beside_chunks_is_split(gpu):
    """One token over a long context beside prompt chunks costs about what it does
    alone: its keys are not walked by one workgroup. (Of one workgroup for each kv
    head, 100000 keys took 2900 us, the chunks 320 and the token alone 40.)"""
    chunks, token = [(3800, 2048)] * 3, [(100000, 1)]
    times = []
    for part in (chunks, token, chunks + token):
        call = Timed(gpu, [n for n, _ in part], [m for _, m in part])
        call()
        times.append(_us(gpu, call))
    assert times[2] < 2.0 * (times[0] + times[1]) + 100.0, times


def test_decoding_in_a_step_captured_for_prompts(gpu):
    """A step whose q has room for a prompt of every request, replayed where each
    brings one token: near a call made for single tokens, with the same results up
    to the order of sums, which bf16's rounding hides but for one step of it."""
    torch = gpu
    lens, counts = [40000 + 977 * i for i in range(6)], [1] * 6
    plain, room = Timed(torch, lens, counts), Timed(torch, lens, counts, max_q=512, rows=6 * 512)
    room.q[:6] = plain.q
    plain()
    room()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        room()
    room.o.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    a, b = room.o[:6].double(), plain.o.double()
    assert bool((room.o[6:] == 7.0).all())
    assert bool(((a - b).abs() <= 2.0 ** -6 * b.abs() + 2.0 ** -6 * b.abs().max()).all())
    assert _us(torch, graph.replay) < 2.0 * _us(torch, plain) + 100.0


def test_chunks_among_many_requests(gpu):
    """More requests than a wave has lanes, chunks among their first, the 64th, the
    65th and the last ones, single tokens and requests without any between."""
    r = np.random.default_rng(3)
    lens, counts = r.integers(1, 90, 140).tolist(), [1] * 140
    for i, n in ((0, 150), (63, 90), (64, 131), (129, 70), (139, 33)):
        counts[i], lens[i] = n, n + 45 * (i % 3)
    for i in (1, 65, 70, 138):
        counts[i] = 0
    for dtype, d in (("bf16", 128), ("f16", 64)):
        c = Call(gpu, dtype, 8, 2, d, 16, lens, counts, seed=70 + d)
        c.check(c.run(), only=_some(counts, d, 2))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (8, 2, 128), (32, 8, 128)])
def test_many_chunks(gpu, dtype, hq, hk, d):
    """More chunks than a wave has lanes, in parts of 128 and (32 heads) 256 rows."""
    r = np.random.default_rng(4)
    counts = r.integers(90, 110, 70).tolist()
    lens = [n + int(x) for n, x in zip(counts, r.integers(0, 200, 70))]
    c = Call(gpu, dtype, hq, hk, d, 16, lens, counts, seed=80 + d)
    some = _some(counts, d, 0)
    c.check(c.run(), only=set(sorted(some)[::1 if hq == 8 else 7]))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_draft_tokens_over_long_contexts(gpu, dtype, d):
    """Requests of 17 to 64 rows whose keys several workgroups share."""
    lens, counts = [6100, 3000, 70, 4097], [16, 5, 9, 13]
    c = Call(gpu, dtype, 8, 2, d, 32, lens, counts, seed=90 + d)
    c.check(c.run(), only=_some(counts, d, 3))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hk,lens,counts", KINDS)
def test_rows_of_nobody_stay(gpu, dtype, hq, hk, lens, counts):
    """Rows of q before the first request, behind the last and past max_q, in every
    kind of batch: left as they were, to the bit; the others are as ever."""
    torch = gpu
    c = Call(torch, dtype, hq, hk, 128, 16, lens, counts, seed=44)
    before = 5
    c.q = torch.cat([c.q[:1].expand(before, -1, -1), c.q, c.q[:1].expand(70, -1, -1)])
    c.offsets += before
    most = max(counts) - (1 if max(counts) > 1 else 0)
    got = c.run(max_q=most, fill=7.0)
    mine = torch.zeros(c.q.shape[0], dtype=torch.bool)
    for b, n in enumerate(counts):
        mine[int(c.offsets[b]):int(c.offsets[b]) + min(n, most)] = True
    assert bool((got[~mine] == 7.0).all())
    some = {before + t for t in _some(counts, 6, 3)}
    c.check(got, most, only={t for t in some if bool(mine[t])})


def test_offsets_outside_the_rows(gpu):
    """Offsets below 0 and past the rows of q, or falling, mean the nearest that there are."""
    torch = gpu
    c = Call(torch, "bf16", 4, 1, 64, 16, [48, 20, 33], [1, 1, 1], seed=15)
    c.max_q = 4
    c.offsets = torch.tensor([-5, 2, 1000, 900], dtype=torch.int32)
    got = c.run()
    c.offsets = torch.tensor([0, 2, 3, 3], dtype=torch.int32)
    c.check(got, 4)
    long = Call(torch, "bf16", 8, 2, 128, 16, [300, 200], [100, 90], seed=16)
    want = long.run()
    long.offsets = torch.tensor([-7, 100, 1 << 30], dtype=torch.int32)
    assert torch.equal(long.run(), want)
