"""Products of int8 operands against the definition in 64 bits.

Tolerances count roundings.  The sum of products is a whole number, exact in 32 bits, and is rounded to fp32 once; two scales
multiply it: three relative errors of 2^-24.  The bias joins with one rounding of the result, the cast adds half a step
of the output type (fp16 results below its normal range: half of 2^-24).
"""
import ctypes

import pytest
import torch

import flag_gems
from flaggems_b200 import _cabi

pytestmark = pytest.mark.gpu
I8 = torch.int8
F32 = 2.0 ** -24


def _ints(g, *shape, lo=-128, hi=128):
    return torch.randint(lo, hi, shape, generator=g, dtype=I8, device="cuda")


def _operands(m, n, k, seed=0, lo=-128):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a, b = _ints(g, m, k, lo=lo), _ints(g, n, k, lo=lo)
    a_s = torch.rand(m, 1, device="cuda", generator=g) * 0.02 + 1e-3
    b_s = torch.rand(n, device="cuda", generator=g) * 0.002 + 1e-4
    return a, b, a_s, b_s, g


def _definition(a, b, a_s, b_s):
    return (a.double() @ b.double().t()) * a_s.double().reshape(-1, 1) * b_s.double().reshape(1, -1)


def _check(got, pre, bias=None, rounded_before_bias=False):
    """``pre``: the scaled product in 64 bits; ``bias`` joins before the cast, or after it in the output's type."""
    half = torch.finfo(got.dtype).eps / 2
    want = pre if bias is None else pre + bias.double()
    bound = pre.abs() * 3 * F32 + want.abs() * (half + F32 + half * 4 * F32)
    if rounded_before_bias:
        bound = bound + pre.abs() * half * (1 + half)
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (2 if rounded_before_bias else 1)
    err = (got.double() - want).abs()
    assert bool((err <= bound * 1.001).all()), (float(err.max()), float((err / bound.clamp_min(1e-300)).max()))


# few tokens (8, 16 or 32 in registers, up to 128 in TMEM; groups of 16 to 256 weight rows, one or several per CTA; K with and
# without whole blocks of 128), single and paired tiles, ragged edges in every dimension
SHAPES = [(1, 1, 16), (1, 256, 128), (1, 6144, 4096), (1, 2112, 7168), (1, 28672, 1024), (2, 33, 48), (3, 100003, 272), (7, 130, 2064),
          (8, 40000, 528), (9, 37889, 256), (16, 28672, 4096), (17, 75777, 384), (20, 24576, 1040), (24, 15000, 784), (31, 4096, 4096),
          (32, 300, 16), (32, 28672, 2048), (33, 208, 496), (50, 4096, 4096), (64, 9472, 208), (64, 9473, 208), (64, 24576, 1040),
          (65, 60000, 400), (83, 7744, 3888), (97, 37889, 128), (100, 2112, 7168), (127, 20000, 656), (128, 4096, 14336), (128, 76000, 256), (129, 144, 144), (130, 4097, 528), (257, 9500, 256),
          (1024, 6144, 4096), (1037, 6145, 4096), (4099, 8191, 512), (8192, 8192, 1024)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_per_token_per_channel(m, n, k):
    a, b, a_s, b_s, _ = _operands(m, n, k)
    _check(flag_gems.w8a8_int8_matmul(a, b, a_s, b_s), _definition(a, b, a_s, b_s))


@pytest.mark.parametrize("m", [65, 129, 300, 513, 777, 1037, 1300, 3000])
@pytest.mark.parametrize("n", [515, 2112, 4100, 6144, 7168, 11008])
def test_tiles_of_every_width(m, n):
    """Row counts and widths between which the tile's width and kind change; 8 blocks of K and a short one."""
    a, b, a_s, b_s, g = _operands(m, n, 1040, seed=n)
    c = torch.randn(n, device="cuda", generator=g).half()
    _check(flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, c, torch.float16), _definition(a, b, a_s, b_s), c)


@pytest.mark.parametrize("m", [1, 20, 100, 200])
@pytest.mark.parametrize("n", [4096, 30000])
def test_operands_that_the_kernel_before_writes(m, n):
    """The product may be launched while its operands are still being written, into memory that held others before."""
    g = torch.Generator(device="cuda").manual_seed(m)
    w, x = torch.randn(n, 2048, device="cuda", generator=g).bfloat16(), torch.randn(m, 2048, device="cuda", generator=g).bfloat16()
    kept = []
    for i in range(8):
        a, a_s = flag_gems.per_token_quant_int8(x)
        b, b_s = flag_gems.per_token_quant_int8(w)
        c = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s)
        kept.append((a.clone(), b.clone(), a_s.clone(), b_s.clone(), c))
        del a, b, a_s, b_s
        x, w = x.roll(1, 1), w.roll(3, 0) * 1.25
    for a, b, a_s, b_s, c in kept:
        _check(c, _definition(a, b, a_s, b_s))


@pytest.mark.parametrize("m", [1, 5, 12, 31, 60, 120])
def test_few_tokens_twice_at_once(m):
    """The same call on two streams, and one after another without a wait between."""
    ops = [_operands(m, 20000 + 16 * i, 2048, seed=i) for i in range(4)]
    want = [_definition(*o[:4]) for o in ops]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for r in range(3):
        for i, o in enumerate(ops):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, flag_gems.w8a8_int8_matmul(*o[:4])))
    torch.cuda.synchronize()
    for i, c in got:
        _check(c, want[i])
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("m", [1, 5, 20, 40, 128, 300])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float16, torch.float32])
def test_types_and_bias(m, out, bias):
    a, b, a_s, b_s, g = _operands(m, 515, 208, seed=m)
    c = None if bias is None else torch.randn(515, device="cuda", generator=g).to(bias)
    got = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, c, out)
    assert got.dtype == out
    _check(got, _definition(a, b, a_s, b_s), c)


@pytest.mark.parametrize("m,n,k", [(100, 1000, 8192), (128, 4096, 14336), (127, 999, 8208), (129, 1000, 8192), (200, 1001, 8208), (256, 2112, 7168),
                                   (257, 2112, 7184), (300, 1002, 16384), (384, 1000, 8192), (500, 130, 7168), (1000, 64, 7168), (70, 16, 65536)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias", [None, torch.float32])
def test_long_rows_and_narrow_weights(m, n, k, out, bias):
    """Few tiles, so that K is split over a cluster."""
    a, b, a_s, b_s, g = _operands(m, n, k, seed=m)
    c = None if bias is None else torch.randn(n, device="cuda", generator=g).to(bias)
    kept = [flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, c, out) for _ in range(3)]
    _check(kept[0], _definition(a, b, a_s, b_s), c)
    assert torch.equal(kept[0], kept[1]) and torch.equal(kept[0], kept[2])
    one = torch.tensor([0.01], device="cuda")
    _check(flag_gems.w8a8_int8_matmul(a, b, one, one, c, out), _definition(a, b, one.expand(m), one.expand(n)), c)
    assert _cabi.device_status() == 0


# rows below 65: fewer than 128 of them in shared memory, and CTAs of the cluster whose share of the rows is small or empty
@pytest.mark.parametrize("m,n,k", [(33, 16, 65536), (33, 100, 32768), (40, 1000, 16384), (64, 130, 32768), (64, 4096, 16384), (57, 33, 131056),
                                   (20, 6000, 32768), (31, 5001, 32784)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias", [None, torch.float32])
def test_few_rows_with_split_k(m, n, k, out, bias):
    a, b, a_s, b_s, g = _operands(m, n, k, seed=m)
    c = None if bias is None else torch.randn(n, device="cuda", generator=g).to(bias)
    got = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, c, out)
    _check(got, _definition(a, b, a_s, b_s), c)
    assert torch.equal(got, flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, c, out))
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("m,n,k", [(128, 1000, 8192), (300, 576, 7168)])
def test_split_products_in_streams_and_graphs(m, n, k):
    """Operands that the kernel before writes, two streams at once, and two captured graphs replayed with other operands."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = torch.randn(m, k, device="cuda", generator=g).bfloat16(), torch.randn(n, k, device="cuda", generator=g).bfloat16()

    def layer():
        a, a_s = flag_gems.per_token_quant_int8(x)
        b, b_s = flag_gems.per_token_quant_int8(w)
        return a, b, a_s, b_s, flag_gems.w8a8_int8_matmul(a, b, a_s, b_s)

    def check(got):
        _check(got[4], _definition(*got[:4]))

    check(layer())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            got.append(layer())
    torch.cuda.synchronize()
    for r in got:
        check(r)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer()
        graphs.append((graph, out))
    for _ in range(3):
        x.copy_(x.roll(1, 1) * 1.5)
        w.copy_(w.roll(5, 0))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            check(out)
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("m", [1, 3, 200])
def test_scale_shapes(m):
    a, b, a_s, b_s, _ = _operands(m, 96, 64)
    one = torch.tensor(0.01, device="cuda")
    for sa in (a_s, a_s[:, 0], one, one.view(1), one.view(1, 1)):
        for sb in (b_s, b_s[:, None], one, one.view(1), one.view(1, 1)):
            _check(flag_gems.w8a8_int8_matmul(a, b, sa, sb), _definition(a, b, sa.reshape(-1), sb.reshape(-1)))


def test_more_than_two_dimensions():
    a, b, a_s, b_s, _ = _operands(30, 72, 48)
    want = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s)
    for sa in (a_s.view(5, 6, 1), a_s.view(5, 6)):
        got = flag_gems.w8a8_int8_matmul(a.view(5, 6, 48), b, sa, b_s)
        assert got.shape == (5, 6, 72) and torch.equal(got.view(30, 72), want)
    got = flag_gems.w8a8_int8_matmul(a[0], b, a_s[0], b_s)
    assert got.shape == (72,) and torch.equal(got, want[0])
    part = flag_gems.w8a8_int8_matmul(a.view(5, 6, 48).transpose(0, 1), b, a_s.view(5, 6, 1).transpose(0, 1), b_s)
    assert torch.equal(part.transpose(0, 1).reshape(30, 72), want)


def test_strides_and_alignment():
    a, b, a_s, b_s, g = _operands(37, 80, 64)
    want = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s)
    wide_a, wide_b = _ints(g, 37, 160), _ints(g, 80, 160)
    for off in (0, 16, 1, 7):  # aligned rows of a wider matrix are read where they are, others from a copy
        wide_a[:, off:off + 64] = a
        wide_b[:, off:off + 64] = b
        assert torch.equal(flag_gems.w8a8_int8_matmul(wide_a[:, off:off + 64], wide_b[:, off:off + 64], a_s, b_s), want)
    assert torch.equal(flag_gems.w8a8_int8_matmul(a.t().contiguous().t(), b.t().contiguous().t(), a_s, b_s), want)
    row = a[:1]
    got = flag_gems.w8a8_int8_matmul(row.expand(37, 64), b, a_s, b_s)  # one row for all, stride 0
    assert torch.equal(got, flag_gems.w8a8_int8_matmul(row.repeat(37, 1), b, a_s, b_s))
    every_other = torch.empty(160, device="cuda")[::2]
    every_other.copy_(b_s)
    assert torch.equal(flag_gems.w8a8_int8_matmul(a, b, a_s, every_other), want)


@pytest.mark.parametrize("m", [1, 16, 100, 129, 300])
def test_sums_at_the_edge_of_32_bits(m):
    """K as large as it may be with every product 2^14: the largest sum is 2^31 - 2^18."""
    k = 131056
    a = torch.full((m, k), -128, dtype=I8, device="cuda")
    b = torch.full((257, k), -128, dtype=I8, device="cuda")
    b[1::2] = 127
    one = torch.ones(1, device="cuda")
    got = flag_gems.w8a8_int8_matmul(a, b, one, one, None, torch.float32)
    want = (torch.where(torch.arange(257, device="cuda") % 2 == 0, 128 * 128 * k, -128 * 127 * k)).expand(m, 257)
    assert torch.equal(got, want.double().float())


@pytest.mark.parametrize("m,n,k", [(1, 3000017, 128), (12, 9000000, 16), (128, 17000000, 16), (40000, 55000, 64)])
def test_many_groups_and_outputs_past_32_bits(m, n, k):
    """Thousands of groups of weight rows per CTA; up to 2.2e9 outputs (4.4 GB)."""
    a, b, a_s, b_s, g = _operands(m, n, k)
    got = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s)
    assert got.shape == (m, n)
    at = torch.cat([torch.arange(700, device="cuda"), torch.randint(0, n, (4000,), device="cuda", generator=g),
                    torch.arange(n - 700, n, device="cuda")])
    rows = torch.tensor(sorted({0, m // 3, m - 1}), device="cuda")
    _check(got[rows][:, at], _definition(a[rows], b[at], a_s[rows], b_s[at]))
    assert _cabi.device_status() == 0


def test_nothing_to_compute():
    one = torch.ones(1, device="cuda")
    a, b = torch.zeros(0, 64, dtype=I8, device="cuda"), torch.zeros(32, 64, dtype=I8, device="cuda")
    assert flag_gems.w8a8_int8_matmul(a, b, one, one).shape == (0, 32)
    assert flag_gems.w8a8_int8_matmul(b, a, one, one).shape == (32, 0)


def test_special_scales():
    a, b, a_s, b_s, _ = _operands(40, 64, 64)
    a_s[3], a_s[5], b_s[7] = float("inf"), float("nan"), 0.0
    got = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s)
    want = _definition(a, b, a_s, b_s)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    keep = [i for i in range(40) if i not in (3, 5)]
    _check(got[keep], want[keep])


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (33, 208, 496), (90, 9008, 512), (700, 4096, 256)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
def test_cutlass_scaled_mm(m, n, k, bias, out):
    a, b, a_s, b_s, g = _operands(m, n, k)
    c = torch.full((m, n), float("nan"), dtype=out, device="cuda")
    t = torch.randn(n, device="cuda", generator=g).to(out) if bias else None
    flag_gems.cutlass_scaled_mm(c, a, b.t(), a_s, b_s, t)
    _check(c, _definition(a, b, a_s, b_s), t, rounded_before_bias=bias)


@pytest.mark.parametrize("m,n", [(33, 700), (64, 31), (97, 9471), (128, 33), (131, 65), (300, 2845), (1037, 2050), (2500, 6145)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off", [0, 1, 2, 8])
def test_results_between_others(m, n, out, off):
    """Rows that begin at any value, in a wider matrix whose other values stay as they are."""
    a, b, a_s, b_s, _ = _operands(m, n, 272 if m != 131 else 8208, seed=n)
    wide = torch.full((m, (n + off + 31) // 16 * 16), 7.0, dtype=out, device="cuda")
    flag_gems.cutlass_scaled_mm(wide[:, off:off + n], a, b.t(), a_s, b_s)
    _check(wide[:, off:off + n], _definition(a, b, a_s, b_s))
    assert bool((wide[:, :off] == 7).all()) and bool((wide[:, off + n:] == 7).all())
    assert _cabi.device_status() == 0


def test_cutlass_scaled_mm_refusals():
    a, b, a_s, b_s, _ = _operands(16, 128, 256)
    c = torch.empty(16, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(AssertionError, match="Unsupported dtype"):
        flag_gems.cutlass_scaled_mm(c, a, b.to(torch.float8_e4m3fn).t(), a_s, b_s)
    with pytest.raises(AssertionError, match="int8 operands take"):
        flag_gems.cutlass_scaled_mm(c, a, b.t(), torch.ones(16, 2, device="cuda"), torch.ones(2, 1, device="cuda"))
    with pytest.raises(NotImplementedError, match="implemented for float8"):
        flag_gems.scaled_mm(a, b.t(), a_s, b_s.view(1, -1), None, None, torch.bfloat16)  # aten's op stays an FP8 one


# ---- grouped ----------------------------------------------------------------------------------
def _grouped(sizes, n, k, seed=0, tail=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = sum(sizes) + tail
    a, b = _ints(g, m, k), _ints(g, len(sizes), n, k)
    a_s = torch.rand(m, 1, device="cuda", generator=g) * 0.02 + 1e-3
    b_s = torch.rand(len(sizes), n, device="cuda", generator=g) * 0.002 + 1e-4
    offs = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
    return a, b, a_s, b_s, offs, g


def _grouped_definition(a, b, a_s, b_s, offs):
    out = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device="cuda")
    begin = 0
    for e, end in enumerate(offs.tolist()):
        out[begin:end] = _definition(a[begin:end], b[e], a_s[begin:end], b_s[e])
        begin = end
    return out


SIZES = [[1], [0, 1, 0], [5, 0, 31, 1], [0, 0, 129], [128, 256, 127], [1] * 70, [3, 0, 2, 1, 0, 0, 4] * 20, [800, 900, 1000],
         [0, 1300], [2000, 1, 0, 700]]


@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{sum(s)}" for s in SIZES])
@pytest.mark.parametrize("n,k", [(64, 128), (513, 272), (4096, 64)])
def test_grouped(sizes, n, k):
    a, b, a_s, b_s, offs, _ = _grouped(sizes, n, k)
    _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs), _grouped_definition(a, b, a_s, b_s, offs))


FEW = [[1], [16], [0, 1, 0], [8, 8], [0, 15, 0, 0], [3, 0, 2, 1, 0, 0, 4], [1] * 16, [0] * 300 + [2] + [0] * 10 + [7], [0] * 1022 + [5, 1],
       [2] + [0] * 1023, [0, 9, 0, 7], [0, 0, 0]]


@pytest.mark.parametrize("sizes", FEW, ids=[f"{len(s)}x{sum(s)}" for s in FEW])
@pytest.mark.parametrize("n,k", [(16, 16), (515, 272), (4096, 128), (3000, 1040)])
@pytest.mark.parametrize("tail", [0, 2])
def test_grouped_few_rows(sizes, n, k, tail):
    if len(sizes) > 500 and n * k > 200000:
        n, k = 264, 384
    a, b, a_s, b_s, offs, g = _grouped(sizes, n, k, tail=tail)
    if a.shape[0] == 0:
        return
    junk = [torch.full((a.shape[0], n), float("nan"), device="cuda") for _ in range(4)]  # memory that is reused
    del junk
    want = _grouped_definition(a, b, a_s, b_s, offs)
    for out in (torch.bfloat16, torch.float32):
        _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs, output_dtype=out), want)
    group = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(sizes, device="cuda"))
    for bias in (torch.randn(n, device="cuda", generator=g), torch.randn(len(sizes), n, device="cuda", generator=g)):
        got = flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs, bias, torch.float16)
        real = a.shape[0] - tail
        _check(got[:real], want[:real], bias.expand(len(sizes), n)[group])
        assert not got[real:].any()
    assert _cabi.device_status() == 0


def test_grouped_few_rows_of_ends_out_of_range():
    a, b, a_s, b_s, offs, _ = _grouped([2, 0, 3, 1], 515, 272, tail=3)
    want = _grouped_definition(a, b, a_s, b_s, offs)
    low, high = torch.iinfo(torch.int32).min, torch.iinfo(torch.int32).max
    ends = torch.tensor([2, low, 5, 6], dtype=torch.int32, device="cuda")  # groups 0 and 2 share the first two rows
    got = flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, ends, output_dtype=torch.float32)
    _check(got[2:], want[2:])
    ends = torch.tensor([2, 2, 5, high], dtype=torch.int32, device="cuda")  # the last group takes what is left
    want[5:] = _definition(a[5:], b[3], a_s[5:], b_s[3])
    _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, ends, output_dtype=torch.float32), want)
    assert _cabi.device_status() == 0


def test_grouped_ends_out_of_range():
    """As above for more rows, whose tables of tiles a kernel of their own makes."""
    a, b, a_s, b_s, offs, _ = _grouped([20, 0, 30, 10], 515, 272, tail=3)
    want = _grouped_definition(a, b, a_s, b_s, offs)
    low, high = torch.iinfo(torch.int32).min, torch.iinfo(torch.int32).max
    ends = torch.tensor([20, low, 50, 60], dtype=torch.int32, device="cuda")  # groups 0 and 2 share the first 20 rows
    got = flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, ends, output_dtype=torch.float32)
    _check(got[20:], want[20:])
    ends = torch.tensor([20, 20, 50, high], dtype=torch.int32, device="cuda")  # the last group takes what is left
    want[50:] = _definition(a[50:], b[3], a_s[50:], b_s[3])
    _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, ends, output_dtype=torch.float32), want)
    assert _cabi.device_status() == 0


def test_grouped_ends_that_the_kernel_before_writes():
    a, b, a_s, b_s, offs, g = _grouped([4] * 4, 4096, 1024)
    kept = []
    for i in range(12):
        ids = torch.randint(0, 4, (16, 1), device="cuda", generator=g)
        rows, row_s, plan = flag_gems.moe_permute(a, ids, 4, scale=a_s)
        kept.append((rows, row_s, plan.offs, flag_gems.w8a8_int8_grouped_mm(rows, b, row_s, b_s, plan.offs)))
    for rows, row_s, ends, c in kept:
        _check(c, _grouped_definition(rows, b, row_s, b_s, ends))


@pytest.mark.parametrize("sizes", [[700, 0, 130, 400], [100, 250, 97, 3, 300], [1300, 700, 900], [2100, 1500]], ids=str)
@pytest.mark.parametrize("n", [2112, 4096, 6200])
def test_grouped_tiles_of_every_width(sizes, n):
    a, b, a_s, b_s, offs, g = _grouped(sizes, n, 2064, seed=n, tail=5)
    bias = torch.randn(len(sizes), n, device="cuda", generator=g)
    want = _grouped_definition(a, b, a_s, b_s, offs)
    _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs), want)
    group = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(sizes, device="cuda"))
    got = flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs, bias, torch.float16)
    _check(got[:-5], want[:-5], bias[group])
    assert not got[-5:].any()


class _KernelNode(ctypes.Structure):
    """CUDA_KERNEL_NODE_PARAMS of the driver API."""
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3), ("shared", ctypes.c_uint),
                ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def _grids(call):
    """CTAs of the kernels that ``call`` launches, from a captured graph that never runs."""
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    cu, raw, n = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert cu.cuGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    grids = []
    for node in nodes:
        kind, params = ctypes.c_int(), _KernelNode()
        assert cu.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:
            assert cu.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(params)) == 0
            grids.append(params.grid[0] * params.grid[1] * params.grid[2])
    return grids


# rows of the groups, and the tiles of CTA pairs that their products take: 128, 128 and 192 columns
@pytest.mark.parametrize("sizes,n,k,tiles", [([207, 207], 4096, 7168, 64), ([503], 4096, 7168, 64), ([540], 4096, 14336, 66)])
def test_grouped_pairs_have_a_cta_pair_for_every_tile(sizes, n, k, tiles):
    a, b, a_s, b_s, offs, _ = _grouped(sizes, n, k)
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert max(_grids(lambda: flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs))) >= 2 * min(tiles, pairs)
    _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs), _grouped_definition(a, b, a_s, b_s, offs))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", [[700, 0, 130, 33], [1300, 1], [20] * 8], ids=str)
@pytest.mark.parametrize("n", [31, 2050, 2845])
def test_grouped_rows_of_any_alignment(out, sizes, n):
    a, b, a_s, b_s, offs, _ = _grouped(sizes, n, 272, seed=n, tail=3)
    _check(flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs, output_dtype=out), _grouped_definition(a, b, a_s, b_s, offs))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tail", [1, 200])
@pytest.mark.parametrize("n", [64, 65])
def test_grouped_rows_behind_the_last_group_are_zeros(out, tail, n):
    a, b, a_s, b_s, offs, _ = _grouped([7, 0, 30], n, 64, tail=tail)
    junk = [torch.full((37 + tail, n), float("nan"), dtype=out, device="cuda") for _ in range(4)]  # memory that is reused
    del junk
    got = flag_gems.w8a8_int8_grouped_mm(a, b, a_s[:, 0], b_s, offs, output_dtype=out)
    _check(got, _grouped_definition(a, b, a_s, b_s, offs))
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert not flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, none, output_dtype=out).any()


@pytest.mark.parametrize("per_group", [False, True])
def test_grouped_bias_strides_and_copies(per_group):
    a, b, a_s, b_s, offs, g = _grouped([9, 0, 140], 96, 64)
    bias = torch.randn((3, 96) if per_group else (96,), device="cuda", generator=g)
    got = flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs, bias, torch.float32)
    group = torch.tensor([0] * 9 + [2] * 140, device="cuda")
    _check(got, _grouped_definition(a, b, a_s, b_s, offs), bias[group] if per_group else bias.expand(149, 96))
    want = flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs)
    wide = _ints(g, 149, 131)
    wide[:, 3:67] = a
    assert torch.equal(flag_gems.w8a8_int8_grouped_mm(wide[:, 3:67], b, a_s, b_s, offs), want)
    assert torch.equal(flag_gems.w8a8_int8_grouped_mm(a, b.transpose(1, 2).contiguous().transpose(1, 2), a_s, b_s, offs), want)


def test_grouped_nothing_to_compute():
    a, b, a_s, b_s, offs, _ = _grouped([0, 0], 32, 64)
    assert flag_gems.w8a8_int8_grouped_mm(a, b, a_s, b_s, offs).shape == (0, 32)
    a, b, a_s, b_s, offs, _ = _grouped([4], 32, 64)
    got = flag_gems.w8a8_int8_grouped_mm(a, b[:0], a_s, b_s[:0], offs[:0])
    assert got.shape == (4, 32) and not got.any()


# ---- quantisation -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 8), (3, 264), (2, 5, 4096), (64, 7168)])
def test_per_token_quant_int8(dtype, shape):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[..., 0, :] = 0
    q, s = flag_gems.per_token_quant_int8(x.cuda())
    assert q.dtype == I8 and q.shape == x.shape and s.shape == x.shape[:-1] + (1,)
    want_s = x.float().abs().amax(-1, keepdim=True).clamp_min(1e-10) / 127.0
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu(), (x.float() / want_s).round().clamp(-128, 127).to(I8))
    q2, s2 = flag_gems.moe_kernel_quantize_input(x.cuda(), None, I8, True)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_per_token_quant_int8_of_a_transposed_matrix():
    x = torch.randn(64, 40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    for y, z in zip(flag_gems.per_token_quant_int8(x.t()), flag_gems.per_token_quant_int8(x.t().contiguous())):
        assert torch.equal(y, z)
    assert flag_gems.per_token_quant_int8(x[:0])[0].shape == (0, 40)


# ---- how they are called ------------------------------------------------------------------------
class _Off:
    def __getattr__(self, name):
        return lambda *args: None


def test_native_and_python_host_paths_agree(monkeypatch):
    a, b, a_s, b_s, g = _operands(33, 96, 64)
    ga, gb, ga_s, gb_s, offs, _ = _grouped([9, 0, 140], 96, 64)
    bias = torch.randn(96, device="cuda", generator=g)
    x = torch.randn(5, 64, device="cuda", generator=g)
    c = torch.empty(33, 96, dtype=torch.float16, device="cuda")

    def calls():
        flag_gems.cutlass_scaled_mm(c, a, b.t(), a_s, b_s, bias.half())
        return [c.clone(), flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, bias), flag_gems.w8a8_int8_matmul(a[:1], b, a_s[:1], b_s[:1]),
                flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, gb_s, offs, None, torch.float16), *flag_gems.per_token_quant_int8(x)]

    native = calls()
    monkeypatch.setattr(_cabi, "host", _Off())
    for u, v in zip(native, calls()):
        assert u.dtype == v.dtype and torch.equal(u, v)


def test_gradients_that_would_be_lost_are_refused():
    a, b, a_s, b_s, g = _operands(4, 96, 64)
    ga, gb, ga_s, gb_s, offs, _ = _grouped([1, 0, 3], 96, 64)
    bias, x = torch.randn(96, device="cuda", generator=g), torch.randn(4, 64, device="cuda", generator=g)
    calls = [(lambda t: flag_gems.w8a8_int8_matmul(a, b, t, b_s), a_s), (lambda t: flag_gems.w8a8_int8_matmul(a, b, a_s, t), b_s),
             (lambda t: flag_gems.w8a8_int8_matmul(a, b, a_s, b_s, t), bias),
             (lambda t: flag_gems.w8a8_int8_grouped_mm(ga, gb, t, gb_s, offs), ga_s),
             (lambda t: flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, t, offs), gb_s),
             (lambda t: flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, gb_s, offs, t), bias),
             (lambda t: flag_gems.per_token_quant_int8(t)[0], x)]
    for call, t in calls:
        want, leaf = call(t), t.clone().requires_grad_()
        with pytest.raises(NotImplementedError, match="has no gradient"):
            call(leaf)
        with torch.no_grad():
            assert torch.equal(call(leaf), want)
        assert torch.equal(call(leaf.detach()), want)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="has no gradient"):
                call(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
    q, s = flag_gems.moe_kernel_quantize_input(x.clone().requires_grad_(), None, I8, True)  # as its FP8 form: no gradient
    assert torch.equal(q, flag_gems.per_token_quant_int8(x)[0]) and not s.requires_grad


def test_another_stream_and_graph_capture():
    a, b, a_s, b_s, _ = _operands(16, 4096, 4096)
    ga, gb, ga_s, gb_s, offs, _ = _grouped([9, 0, 140], 96, 64)
    want, gwant = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s), flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, gb_s, offs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, ggot = flag_gems.w8a8_int8_matmul(a, b, a_s, b_s), flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, gb_s, offs)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(ggot, gwant)
    graphs = []
    for _ in range(2):  # two graphs of the same call, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, s = flag_gems.per_token_quant_int8(a_s.expand(16, 4096).contiguous())
            out = (flag_gems.w8a8_int8_matmul(a, b, a_s, b_s), flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, gb_s, offs), q)
        graphs.append((graph, out))
    offs.copy_(torch.tensor([0, 100, 149], device="cuda"))
    a.copy_(a.roll(1, 0))
    for graph, _ in graphs:
        graph.replay()
    for _, out in graphs:
        assert torch.equal(out[0], flag_gems.w8a8_int8_matmul(a, b, a_s, b_s))
        assert torch.equal(out[1], flag_gems.w8a8_int8_grouped_mm(ga, gb, ga_s, gb_s, offs))
    assert _cabi.device_status() == 0
