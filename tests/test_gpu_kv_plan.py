"""GPU: block tables, slot maps, positions and offsets of a serving step
(pyc_hip_kv_plan_dispatch) against kv_util.plan_ref: whole numbers, equal."""
import numpy as np
import pytest

import pyc_amd
from tests import kv_util

pytestmark = pytest.mark.gpu


def _run(torch, cached, fresh, table, free, count, bs, tokens, alias=False, row_gap=0):
    dev = lambda a: torch.from_numpy(np.array(a, np.int32)).cuda()  # noqa: E731
    B, width = table.shape
    wide = torch.full((B, width + row_gap), -7, dtype=torch.int32, device="cuda")
    t = wide[:, :width]
    t.copy_(dev(table))
    c, f, fl, n = dev(cached), dev(fresh), dev(free), dev([count])
    lens = c if alias else torch.full((B,), -9, dtype=torch.int32, device="cuda")
    after = n if alias else torch.full((1,), -9, dtype=torch.int32, device="cuda")
    q = torch.full((B + 1,), -9, dtype=torch.int32, device="cuda")
    slots = torch.full((tokens,), -9, dtype=torch.int32, device="cuda")
    pos = torch.full((tokens,), -9, dtype=torch.int32, device="cuda")
    pyc_amd.kv_plan(c, f, t, fl, n, bs, lens, q, slots, pos, after)
    torch.cuda.synchronize()
    assert bool((wide[:, width:] == -7).all())
    got = {"table": t, "free": fl, "lens": lens, "q_offsets": q, "slots": slots, "positions": pos, "free_after": after}
    return {k: v.cpu().numpy() for k, v in got.items()}


def _check(torch, cached, fresh, table, free, count, bs, tokens, **kw):
    ref = kv_util.plan_ref(cached, fresh, table, free, count, bs, tokens)
    got = _run(torch, cached, fresh, table, free, count, bs, tokens, **kw)
    for k in ref:
        assert np.array_equal(got[k], ref[k]), (k, got[k], ref[k])


def _random(r, B, bs, width, most, over, spare):
    cached = r.integers(0, width * bs // 2 + 1, B)
    cached[r.random(B) < 0.2] = 0
    fresh = np.where(r.random(B) < 0.5, 1, r.integers(0, most + 1, B))
    fresh = np.where(r.random(B) < over, -1, fresh)
    have = [kv_util.ceil_div(int(c), bs) for c in cached]
    need = sum(kv_util.ceil_div(int(c + max(f, 0)), bs) - h for c, f, h in zip(cached, fresh, have))
    ids = r.permutation(sum(have) + need + spare + 1).astype(np.int32)
    table = r.integers(-5, 1 << 20, (B, width)).astype(np.int32)
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = ids[at:at + h]
        at += h
    free = np.full(len(ids) + 3, -3, np.int32)
    free[:len(ids) - at] = ids[at:]
    return cached.astype(np.int32), fresh.astype(np.int32), table, free, len(ids) - at, int(np.maximum(fresh, 0).sum())


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 255, 1023, 1024, 1025, 2500])
def test_sizes(gpu, B, alias):
    """Any number of requests (one workgroup takes 1024 at a time), with spare
    token room behind the last one."""
    r = np.random.default_rng(B)
    for bs in (16, 128):
        c, f, t, free, n, tokens = _random(r, B, bs, 12, 40, 0.1, 5)
        _check(gpu, c, f, t, free, n, bs, tokens + 7, alias=alias, row_gap=3 if bs == 16 else 0)


@pytest.mark.parametrize("tokens", [4095, 4096, 4097, 20000])
def test_many_tokens(gpu, tokens):
    """On both sides of where the slots get a launch of their own."""
    r = np.random.default_rng(tokens)
    c, f, t, free, n, asked = _random(r, 300, 32, 40, 200, 0.05, 9)
    _check(gpu, c, f, t, free, n, 32, tokens)


def test_long_prompts_and_releases(gpu):
    """Requests that take and give back many blocks each."""
    r = np.random.default_rng(4)
    c, f, t, free, n, tokens = _random(r, 37, 16, 700, 5000, 0.4, 3)
    _check(gpu, c, f, t, free, n, 16, tokens)


@pytest.mark.parametrize("left", [0, 1, 7, 30])
def test_too_few_blocks(gpu, left):
    """The stack holds fewer blocks than are asked for: requests in order until
    it would run out, and those that need none."""
    r = np.random.default_rng(left)
    c, f, t, free, n, tokens = _random(r, 90, 16, 20, 30, 0.03, 0)
    _check(gpu, c, f, t, free, min(n, left), 16, tokens)


@pytest.mark.parametrize("tokens", [0, 1, 5, 100])
def test_too_few_token_places(gpu, tokens):
    r = np.random.default_rng(tokens)
    c, f, t, free, n, _ = _random(r, 70, 16, 20, 30, 0.1, 4)
    _check(gpu, c, f, t, free, n, 16, tokens)


def test_edges(gpu):
    """Full rows, one token past them, nothing brought, lengths that end on a
    block, everybody over, an empty stack, and counts outside their bounds."""
    table = np.arange(24, dtype=np.int32).reshape(6, 4)
    free = np.arange(100, 130, dtype=np.int32)
    _check(gpu, [64, 63, 64, 0, 16, 15], [1, 1, 0, 64, 16, 1], table, free, 10, 16, 200)
    _check(gpu, [64, 63, 64, 0, 16, 15], [-1] * 6, table, free, 10, 16, 8)
    _check(gpu, [0] * 6, [0] * 6, table, free, 0, 16, 3)
    _check(gpu, [0] * 6, [65, 1, 1, 1, 1, 1], table, free, 3, 16, 30)
    _check(gpu, [-4, 1000, 5, 5, 5, 5], [3, -1, 1, 1, 1, 1], table, free, 99, 16, 30)
    _check(gpu, [64] * 6, [-1] * 6, table, free, 20, 16, 1)  # the stack has no room for all of them
    _check(gpu, [5] * 6, [2147483647, 1, 1, 1, 1, 1], table, free, 4, 16, 30)
    _check(gpu, [0], [1], np.zeros((1, 1), np.int32), np.array([9], np.int32), 1, 64, 1)


def test_called_again(gpu):
    """With outputs of their own the same call gives the same plan again."""
    torch = gpu
    r = np.random.default_rng(8)
    c, f, t, free, n, tokens = _random(r, 200, 16, 30, 60, 0.2, 5)
    ref = kv_util.plan_ref(c, f, t, free, n, 16, tokens)
    dev = lambda a: torch.from_numpy(np.array(a, np.int32)).cuda()  # noqa: E731
    C, F, T, FL, N = dev(c), dev(f), dev(t), dev(free), dev([n])
    out = [torch.empty(k, dtype=torch.int32, device="cuda") for k in (200, 201, tokens, tokens, 1)]
    for _ in range(3):
        pyc_amd.kv_plan(C, F, T, FL, N, 16, *out)
    torch.cuda.synchronize()
    for name, x in zip(("lens", "q_offsets", "slots", "positions", "free_after"), out):
        assert np.array_equal(x.cpu().numpy(), ref[name]), name
    assert np.array_equal(T.cpu().numpy(), ref["table"]) and np.array_equal(FL.cpu().numpy(), ref["free"])
