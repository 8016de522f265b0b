"""GPU: every kernel of the products by expert at sizes that the rule gives to it (a CPU test
of the same list says which), against moe_util.product_ref in 64 bits: ragged, empty and
short experts, tiles in turns, depths that are no whole steps, the gate, bias, gather, row
strides, operands past 4 GiB."""
import math

import pytest

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, GATE, RELU

RAGGED = [300, 0, 1, 65, 129, 257, 272]
MANY = [0, 300, 1, 64, 128, 20, 150] * 10 + [300, 2]
# (kernel, argument, rows of each expert, N, depths)
SIXTEEN = [(2, 0, [700, 324], 8192, [64, 72]), (2, 0, RAGGED, 16416, [64, 200]), (2, 0, MANY, 2512, [40]),
           (1, 2, [300, 20, 10, 270], 4104, [64, 136, 1000]), (1, 1, [30, 0, 64, 200, 3], 1000, [64, 328, 8]),
           (0, 0, [30, 0, 64, 200, 3], 1000, [63, 129, 20])]
# (kernel, argument, rows of each expert, N, depths by group); a single expert: the dense product too
FOUR = [(4, 0, [300, 65, 10, 325], 8200, {32: [96], 64: [448], 128: [128, 640]}), (4, 0, [700], 8192, {32: [416], 64: [64], 128: [384]}),
        (4, 1, [200], 1264, {32: [32, 544], 64: [192], 128: [1152]}), (4, 1, [90, 0, 107, 3], 1040, {32: [480], 64: [320], 128: [256]}),
        (4, 2, [200], 2000, {32: [160], 64: [576], 128: [384]}), (4, 2, [90, 0, 107, 3], 2000, {32: [96], 64: [128], 128: [512]}),
        (4, 4, [200], 3600, {32: [352], 64: [64], 128: [256]}), (4, 4, [90, 0, 107, 3], 3600, {32: [96], 64: [192], 128: [256]}),
        # streamed: x through LDS in one turn and in several, beside the weights; scales in turns
        (3, 0, [3], 2056, {32: [7200], 64: [256], 128: [2048]}), (3, 0, [32], 96, {32: [11008], 64: [4160], 128: [3584]}),
        (3, 0, [1, 0, 7, 2, 0, 3, 5, 2], 1040, {32: [4128], 64: [2112], 128: [6016]}),
        (3, 0, [16, 0, 27, 13, 0, 30, 25, 2], 1040, {32: [9376], 64: [2112], 128: [256]})]


def _epilogues(n, group=0):
    return [0, RELU, GATE] if n % 16 == 0 else [0, GATE]


@pytest.mark.parametrize("kind,arg,counts,n,depths", SIXTEEN)
def test_form_of_sixteen_bits(kind, arg, counts, n, depths):
    for k in depths:
        for epi in _epilogues(n):
            assert moe_util.form(False, len(counts), sum(counts), n, k, epi) == (kind, arg)


@pytest.mark.parametrize("kind,arg,counts,n,depths", FOUR)
def test_form_of_four_bits(kind, arg, counts, n, depths):
    for ks in depths.values():
        for k in ks:
            assert moe_util.form(True, len(counts), sum(counts), n, k, dense=len(counts) == 1) == (kind, arg)
            assert moe_util.form(True, len(counts), sum(counts), n, k, GATE) == (kind, arg)


def test_forms_that_need_the_general_kernel():
    for w4 in (False, True):
        assert moe_util.form(w4, 2, 64, 64, 64, x_rows=0)[0] == 0
        assert moe_util.form(w4, 2, 64, 64, 64, x_rows=1 << 20, x_stride=1 << 12)[0] == 0  # past 4 GiB
    assert moe_util.form(False, 2, 64, 64, 64, at=0x10002)[0] == 0
    assert moe_util.form(False, 2, 64, 64, 64, x_stride=68)[0] == 0


def _i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cuda(t):
    return None if t is None else t.cuda()


def _offsets(counts, before):
    return [before + o for o in moe_util.counts_to_offsets(counts)]


def _run(torch, x, offsets, y, call, ref_args, **kw):
    """call(x, offsets, y, rows=, fan=, bias=, epilogue=) against the reference; rows outside every expert stay."""
    rows, bias = kw.get("rows"), kw.get("bias")
    ref, bound = moe_util.product_ref(x, ref_args[0], offsets, y, rows, kw.get("fan", 1), bias, kw.get("epi", 0), spread=ref_args[1])
    d = y.cuda()
    call(x.cuda(), _i32(torch, offsets), d, rows=None if rows is None else _i32(torch, rows), fan=kw.get("fan", 1),
         bias=_cuda(bias), epilogue=kw.get("epi", 0))
    moe_util.check(d, ref, bound)
    ends = moe_util.held(offsets, y.shape[0])
    assert (d[:ends[0]] == 7).all() and (d[ends[-1]:] == 7).all()


def _variants(torch, counts, n, k, dtype, g):
    """The plain call; gated, through an index with repeats and places outside x, with a bias; ReLU; the rows of
    the experts in the middle of y."""
    p = sum(counts)
    bias = torch.randn((len(counts), n), generator=g)
    rows = torch.randint(-2, 2 * p, (p,), generator=g).tolist()  # of p rows behind fan 2; a few are none
    rows[0], rows[-1] = 1 << 30, 2 * p - 1
    yield dict()
    yield dict(epi=GATE, rows=rows, fan=2, bias=bias)
    if n % 16 == 0:
        yield dict(epi=RELU, bias=bias)
    else:
        yield dict(epi=GATE)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind,arg,counts,n,depths", SIXTEEN)
def test_sixteen_bits(gpu, kind, arg, counts, n, depths, dtype):
    g = gpu.Generator().manual_seed(n)
    for k in depths:
        w = (gpu.randn((len(counts), n, k), generator=g) / math.sqrt(k)).to(DT[dtype])
        x = gpu.randn((sum(counts), k), generator=g).to(DT[dtype])
        d = w.cuda()
        for kw in _variants(gpu, counts, n, k, dtype, g):
            y = gpu.full((sum(counts), n // 2 if kw.get("epi") == GATE else n), 7.0, dtype=x.dtype)
            _run(gpu, x, _offsets(counts, 0), y, lambda x, o, y, **a: pyc_amd.grouped_gemm(x, d, o, y, **a), (w.double(), None), **kw)
        # shifted against y: rows before and behind the experts', the last expert cut short
        y = gpu.full((sum(counts), n), 7.0, dtype=x.dtype)
        off = _offsets(counts, 5)
        off[-1] = sum(counts) - 3
        _run(gpu, x, off, y, lambda x, o, y, **a: pyc_amd.grouped_gemm(x, d, o, y, **a), (w.double(), None))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind,arg,counts,n,depths", FOUR)
def test_four_bits(gpu, kind, arg, counts, n, depths, group, dtype):
    g = gpu.Generator().manual_seed(n)
    for k in depths[group]:
        for zeros in (False, True):
            w = moe_util.random_w4(len(counts), n, k, group, dtype, n + k, zeros)
            x = gpu.randn((sum(counts), k), generator=g).to(DT[dtype])
            c, s, z = [_cuda(v) for v in w]
            ref = moe_util.Weights4(*w), moe_util.Weights4(*w, spread=64 if dtype == "bf16" else 272)

            def by_expert(x, o, y, **a):
                pyc_amd.w4a16_grouped_gemm(x, c, s, o, y, zeros=z, **a)

            def dense(x, o, y, rows, fan, bias, epilogue):
                pyc_amd.w4a16_gemm(x, c[0], s[0], y, zeros=None if z is None else z[0], bias=None if bias is None else bias[0],
                                   epilogue=epilogue)

            for kw in _variants(gpu, counts, n, k, dtype, g):
                y = gpu.full((sum(counts), n // 2 if kw.get("epi") == GATE else n), 7.0, dtype=x.dtype)
                _run(gpu, x, _offsets(counts, 0), y, by_expert, ref, **kw)
                if len(counts) == 1 and "rows" not in kw:
                    _run(gpu, x, _offsets(counts, 0), y, dense, ref, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(1024, 8192, 64), (600, 4104, 136), (90, 200, 264)])
def test_wide_rows_of_y(gpu, rows, n, k):
    """y as columns 8 .. of wider rows, on and off 16 bytes: nothing beside them is written."""
    g = gpu.Generator().manual_seed(n)
    counts = [rows // 2 + 7, 0, rows - rows // 2 - 7]
    x = gpu.randn((rows, k), generator=g).bfloat16()
    w = (gpu.randn((3, n, k), generator=g) / math.sqrt(k)).bfloat16()
    offsets = moe_util.counts_to_offsets(counts)
    ref, bound = moe_util.product_ref(x, w.double(), offsets, gpu.zeros((rows, n), dtype=x.dtype))
    for off, wide in ((8, n + 24), (8, n + 27), (3, n + 24)):
        y = gpu.full((rows, wide), 5.0, dtype=x.dtype, device="cuda")
        pyc_amd.grouped_gemm(x.cuda(), w.cuda(), _i32(gpu, offsets), y[:, off:off + n])
        moe_util.check(y[:, off:off + n], ref, bound)
        assert (y[:, :off] == 5).all() and (y[:, off + n:] == 5).all()


@pytest.mark.gpu
def test_no_rows_of_x(gpu):
    """Without rows of x every row is zeros: only the bias goes out. Weights of few bytes."""
    for k, n in ((4096, 1), (128, 3)):
        bias = gpu.arange(2 * n, dtype=gpu.float32).view(2, n) + 1
        codes, scale, _ = moe_util.random_w4(2, n, k, 32, "bf16", 1, False)
        x, o = gpu.empty((0, k), dtype=gpu.bfloat16, device="cuda"), _i32(gpu, [0, 2, 5])
        y = gpu.full((5, n), 7.0, dtype=gpu.bfloat16, device="cuda")
        pyc_amd.w4a16_grouped_gemm(x, codes.cuda(), scale.cuda(), o, y, rows=_i32(gpu, [0] * 5), bias=bias.cuda(), epilogue=0)
        want = bias.bfloat16()[[0, 0, 1, 1, 1]].cuda()
        assert gpu.equal(y, want)
        y.fill_(7.0)
        w = gpu.ones((2, n, k), dtype=gpu.bfloat16, device="cuda")
        pyc_amd.grouped_gemm(x, w, o, y, rows=_i32(gpu, [0] * 5), bias=bias.cuda())
        assert gpu.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_past_4_gib(gpu, bits):
    """x, the experts' weights and y each over 4 GiB, few rows of them used."""
    torch, g = gpu, gpu.Generator().manual_seed(5)
    k, n, far = 2048, 96, 1_100_000
    xs = torch.randn((6, k), generator=g).bfloat16()
    x = torch.empty((far, k), dtype=torch.bfloat16, device="cuda")
    at = [0, 5, 1_048_575, 1_048_576, 1_048_577, far - 1]
    for i, r in enumerate(at):
        x[r] = xs[i].cuda()
    rows, offsets = _i32(torch, at), [0, 2, 6]
    if bits == 16:
        w = (torch.randn((2, n, k), generator=g) / math.sqrt(k)).bfloat16()
        ref, spread, weights = w.double(), None, [w]
    else:
        weights = moe_util.random_w4(2, n, k, 64, "bf16", 2, True)
        ref, spread = moe_util.Weights4(*weights), moe_util.Weights4(*weights, spread=64)
    want, bound = moe_util.product_ref(xs, ref, offsets, torch.zeros((6, n), dtype=torch.bfloat16), spread=spread)
    # experts' weights 4.5 GB apart, rows of y 0.8 GB
    step, per = 4_500_000_000 // weights[0].element_size() // 16 * 16, weights[0][0].numel()
    wide = torch.empty(step + per, dtype=weights[0].dtype, device="cuda")
    far_w = wide.as_strided(weights[0].shape, (step, weights[0].shape[2], 1))
    far_w.copy_(weights[0].cuda())
    y = torch.empty(5 * 400_000_000 + n, dtype=torch.bfloat16, device="cuda").as_strided((6, n), (400_000_000, 1))

    def run(x, rows, w, y):
        if bits == 16:
            pyc_amd.grouped_gemm(x, w, _i32(torch, offsets), y, rows=rows)
        else:
            pyc_amd.w4a16_grouped_gemm(x, w, weights[1].cuda(), _i32(torch, offsets), y, zeros=weights[2].cuda(), rows=rows)

    near = torch.zeros((6, n), dtype=torch.bfloat16, device="cuda")
    for args in ((x, rows, weights[0].cuda(), near), (xs.cuda(), None, far_w, near), (xs.cuda(), None, weights[0].cuda(), y),
                 (x, rows, far_w, y)):
        args[3].fill_(0)
        run(*args)
        moe_util.check(args[3].contiguous(), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("w4", [False, True])
def test_replayed_with_other_routing(gpu, w4):
    """A captured product of many rows follows the offsets and rows that stand there when it is replayed."""
    torch, g = gpu, gpu.Generator().manual_seed(9)
    p, n, k = 1024, 8192, 128
    x = torch.randn((p, k), generator=g).bfloat16()
    if w4:
        w = moe_util.random_w4(4, n, k, 64, "bf16", 3, False)
        ref, spread = moe_util.Weights4(*w), moe_util.Weights4(*w, spread=64)
        c, s = w[0].cuda(), w[1].cuda()
    else:
        w = (torch.randn((4, n, k), generator=g) / math.sqrt(k)).bfloat16()
        ref, spread, c = w.double(), None, w.cuda()
    d, o, r = x.cuda(), _i32(torch, [0, 256, 512, 768, p]), _i32(torch, list(range(p)))
    y = torch.empty((p, n), dtype=x.dtype, device="cuda")

    def run():
        if w4:
            pyc_amd.w4a16_grouped_gemm(d, c, s, o, y, rows=r)
        else:
            pyc_amd.grouped_gemm(d, c, o, y, rows=r)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for offsets in ([0, 0, 1000, 1001, p], [0, p, p, p, p], [3, 130, 400, 400, 900]):
        rows = torch.randint(-1, p, (p,), generator=g)
        o.copy_(_i32(torch, offsets))
        r.copy_(rows.int())
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want, bound = moe_util.product_ref(x, ref, offsets, torch.full((p, n), 7.0, dtype=x.dtype), rows.tolist(), spread=spread)
        moe_util.check(y, want, bound)
        assert (y[:offsets[0]] == 7).all() and (y[offsets[-1]:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group,k", [(32, 96), (64, 192), (128, 384)])
@pytest.mark.parametrize("rows,n", [(3, 2056), (200, 1264), (200, 2000), (200, 3600), (700, 8192)])
def test_four_bits_beside_values_that_are_not_finite(gpu, rows, n, group, k):
    """Infinite and NaN scales of every other row of W, of an expert without rows, and NaN in rows of x of no expert
    change no bit of the other columns: streamed, in tiles of 16, 32, 64 and 128 rows."""
    g = gpu.Generator().manual_seed(n)
    codes, scale, zeros = moe_util.random_w4(2, n, k, group, "bf16", 3, True)
    x = gpu.randn((rows + 4, k), generator=g).bfloat16()
    bad, xbad = scale.clone(), x.clone()
    bad[0, 1::4], bad[0, 3::4], bad[1] = math.inf, math.nan, math.inf
    xbad[rows:] = math.nan
    c, z, o = codes.cuda(), zeros.cuda(), _i32(gpu, [0, rows, rows])
    y = [gpu.full((rows + 4, n), 7.0, dtype=x.dtype, device="cuda") for _ in range(2)]
    pyc_amd.w4a16_grouped_gemm(x.cuda(), c, scale.cuda(), o, y[0], zeros=z)
    pyc_amd.w4a16_grouped_gemm(xbad.cuda(), c, bad.cuda(), o, y[1], zeros=z)
    assert gpu.isfinite(y[0]).all() and gpu.equal(y[0][:, 0::2], y[1][:, 0::2])
    assert not gpu.isfinite(y[1][:rows, 1::2]).any() and (y[1][rows:] == 7).all()
