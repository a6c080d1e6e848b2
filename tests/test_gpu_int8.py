"""8-bit rows (csrc/rows_int8.cu) and their products (csrc/linear_int8.cu) against the same in 64 bits."""

import pytest
import torch

from conftest import device
from plain_int8 import check_product, check_rows, gated, normed, product
from test_gpu_kernels import K

pytestmark = [pytest.mark.gpu, pytest.mark.needs_cuda]

TYPES = [torch.bfloat16, torch.float16, torch.float32]
EDGE = 7  # what a guard element holds


def gen(seed):
    return torch.Generator(device=device()).manual_seed(seed)


def rows_of(g, rows, cols, dtype, spread=1.0):
    x = torch.randn(rows, cols, generator=g, device=device())
    return (x * torch.exp(spread * torch.randn(rows, 1, generator=g, device=device()))).to(dtype)


def room(rows, cols, pad=0):
    """8-bit rows inside a larger buffer of guard elements, and a check that nothing around them was written."""
    wide = torch.full((rows + 2, cols + pad), EDGE, dtype=torch.int8, device=device())
    out = wide[1:rows + 1, :cols]

    def untouched():
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[1:rows + 1, :cols] = False
        assert (wide[keep] == EDGE).all()

    return out, untouched


# columns: one; less than a thread's piece; ragged; every number of pieces in registers; rows that are read twice
SIZES = [(1, 1, 0), (3, 7, 0), (5, 64, 16), (2, 100, 28), (33, 1000, 0), (7, 2043, 5), (4, 4096, 0), (9, 8200, 8), (3, 12288, 0),
         (2, 20000, 16), (2, 33000, 8), (3, 40001, 0), (700, 128, 0),
         # many rows, some of which blocks that stay take (32-bit ones; every form: test_gpu_int8_row_forms.py)
         (700, 1024, 0), (2500, 1032, 16), (301, 4096, 0), (640, 12288, 0), (900, 8200, 8), (300, 25600, 0), (299, 16384, 0), (310, 2047, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", SIZES)
def test_rows(rows, cols, pad, dtype):
    x = rows_of(gen(rows * cols), rows, cols + pad, dtype)[:, :cols]
    q, untouched = room(rows, cols, pad)
    scales = torch.full((rows,), 9.0, device=device())
    K().quantize_rows_int8(x, q, scales)
    check_rows(q, scales, x.double(), 0.0, 2.0 ** -24 * 1.01)
    untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("rows,cols,pad", SIZES)
def test_gated_activation(rows, cols, pad, act, dtype):
    x = rows_of(gen(rows + cols), rows, 2 * cols, dtype)
    q, untouched = room(rows, cols, pad)
    scales = torch.full((rows,), 9.0, device=device())
    K().act_mul_int8(x, q, scales, act)
    y, z = gated(x, act)
    # e^-z: 2 steps, and the exponent's own roundings (four); 1 + e^-z, the fast quotient (2 steps), the product with up
    rel = 2.0 ** -22 * (z.abs() + 3)
    # (where the denominator passes 2^126 the quotient is 0; such elements are below 2^-110 of the others here)
    check_rows(q, scales, y, rel, float(rel.max()))
    untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_residual", [True, False])
@pytest.mark.parametrize("rows,cols,pad", SIZES)
def test_norm(rows, cols, pad, with_residual, dtype):
    g = gen(2 * rows + cols)
    x, weight = rows_of(g, rows, cols, dtype), 1 + 0.3 * torch.randn(cols, generator=g, device=device())
    residual = rows_of(g, rows, cols, dtype) if with_residual else None
    y = normed(x, residual, weight, 1e-6)
    want = (x.float() + residual.float()).to(dtype) if with_residual else None
    q, untouched = room(rows, cols, pad)
    scales = torch.full((rows,), 9.0, device=device())
    K().add_rmsnorm_int8(x, residual, weight, 1e-6, q, scales)
    # an element: the sum x + residual and the weight's product.  A scale: besides, half of the sum of squares' error, whose longest
    # chain of additions is cols / 1,024 of a thread and ten of the block; the mean, eps, the root (2 steps), two products
    check_rows(q, scales, y, 2.0 ** -23, 2.0 ** -24 * ((cols / 1024 + 40) / 2 + 10))
    if with_residual:
        assert torch.equal(residual, want)
    untouched()


def placed(x, offset):
    """x [rows, cols] contiguous in memory that begins `offset` elements behind a border of 16 bytes, and a check of what lies around."""
    n, wide = x.numel(), torch.full((x.numel() + 64,), 7.0, dtype=x.dtype, device=device())
    held = wide[16 + offset:16 + offset + n].view(x.shape)
    held.copy_(x)

    def untouched():
        assert (wide[:16 + offset] == 7.0).all() and (wide[16 + offset + n:] == 7.0).all()

    return held, untouched


# rows of any length in memory at any place, their 8 bits on borders of 16 bytes: a group and less; warps' edges; several groups of a thread
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (9, 3), (9, 7), (17, 9), (9, 15), (17, 33), (9, 255), (17, 257), (9, 259), (33, 1003), (17, 2041), (9, 4095),
                                       (9, 8191), (5, 9001), (3, 16387), (3, 32767), (2, 32769), (900, 263), (800, 2043), (700, 4101), (140, 1003), (2000, 531), (70, 2041), (9, 5000),
                                       (5, 4096), (3, 8200)])
def test_rows_of_any_length(rows, cols, dtype):
    g = gen(rows * 7 + cols)
    x, res = rows_of(g, rows, cols, dtype), rows_of(g, rows, cols, dtype)
    gu, weight = rows_of(g, rows, 2 * cols, dtype), 1 + 0.3 * torch.randn(cols, generator=g, device=device())
    y, total, (z, size) = normed(x, res, weight, 1e-6), (x.float() + res.float()).to(dtype), gated(gu, 0)
    wide = -(-cols // 16) * 16 - cols
    rel = 2.0 ** -22 * (size.abs() + 3)
    for offset, other in ((0, 0), (1, 3), (5, 5), (6, 2), (3, 0), (0, 7)):
        q, untouched = room(rows, cols, wide)
        scales = torch.full((rows,), 9.0, device=device())
        a, around = placed(x, offset)
        K().quantize_rows_int8(a, q, scales)
        check_rows(q, scales, x.double(), 0.0, 2.0 ** -24 * 1.01)
        b, around_b = placed(res, other)
        K().add_rmsnorm_int8(a, b, weight, 1e-6, q, scales)
        check_rows(q, scales, y, 2.0 ** -23, 2.0 ** -24 * ((cols / 1024 + 40) / 2 + 10))
        assert torch.equal(b, total) and torch.equal(a, x)
        c, around_c = placed(gu, offset)
        K().act_mul_int8(c, q, scales)
        check_rows(q, scales, z, rel, float(rel.max()))
        for check in (untouched, around, around_b, around_c):
            check()


def test_a_residual_that_is_the_input():
    for cols in (4096, 2043):
        x = rows_of(gen(cols), 9, cols, torch.bfloat16)
        once, weight, scales = x.clone(), torch.ones(cols, device=device()), torch.empty(9, device=device())
        q = K().int8_rows(9, cols)
        K().add_rmsnorm_int8(x, x, weight, 1e-6, q, scales)
        check_rows(q, scales, normed(once, once, weight, 1e-6), 2.0 ** -23, 2.0 ** -24 * 40)
        assert torch.equal(x, (once.float() * 2).to(torch.bfloat16))


def test_ties_go_to_even():
    """A row whose largest element is 127 has the scale 1: what lies between two whole numbers goes to the even one."""
    x = torch.zeros(2, 256, device=device())
    x[0, 0], x[0, 1:] = 127.0, torch.arange(255, device=device()) * 0.5 - 63.5
    x[1] = -x[0]
    q, scales = torch.empty(2, 256, dtype=torch.int8, device=device()), torch.empty(2, device=device())
    K().quantize_rows_int8(x, q, scales)
    assert torch.equal(scales, torch.ones(2, device=device())) and torch.equal(q.float(), torch.round(x))


@pytest.mark.parametrize("cols", [5, 512, 40000])
def test_rows_without_a_scale(cols):
    """Zeros have the scale 0; the smallest and largest numbers have theirs; infinities and NaN give their own row NaN and zeros."""
    x = torch.randn(8, cols, device=device())
    x[1] = 0.0
    x[2, 3], x[3, cols - 1], x[4, 0] = float("inf"), float("nan"), float("-inf")
    x[5] *= 1e-41
    x[6] *= 3e37
    q, scales = torch.full((8, cols), 3, dtype=torch.int8, device=device()), torch.full((8,), 9.0, device=device())
    K().quantize_rows_int8(x, q, scales)
    assert scales[1] == 0 and (q[1:5] == 0).all() and scales[2:5].isnan().all()
    fine = [0, 6, 7]
    check_rows(q[fine], scales[fine], x[fine].double(), 0.0, 2.0 ** -24 * 1.01)
    # (numbers below 2^-126 keep few bits of a scale, and all of the elements')
    held = x[5].double() / (x[5].double().abs().max() / 127)
    assert ((q[5].double() - held).abs() <= 0.5 + 127 * 2.0 ** -23).all()
    gu, y = torch.cat([torch.full_like(x, 20.0), x], 1), x.double() * 20 * torch.sigmoid(torch.tensor(20.0, dtype=torch.float64))
    K().act_mul_int8(gu, q, scales)
    assert scales[1] == 0 and (q[1:5] == 0).all() and scales[2:5].isnan().all()
    check_rows(q[[0, 7]], scales[[0, 7]], y[[0, 7]], 2.0 ** -22 * 23, 2.0 ** -22 * 23)
    weight, res = torch.ones(cols, device=device()), x.clone()
    K().add_rmsnorm_int8(torch.zeros_like(x), res, weight, 1e-6, q, scales)
    assert scales[1] == 0 and (q[1:5] == 0).all() and scales[2:5].isnan().all()
    keep = [0, 1, 5, 7]
    check_rows(q[keep], scales[keep], normed(x[keep], None, weight, 1e-6), 2.0 ** -23, 2.0 ** -19)
    assert torch.equal(res.nan_to_num(1.5, 2.5, 3.5), x.nan_to_num(1.5, 2.5, 3.5))


# ---------------------------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------------------------
def operands(seed, M, N, k, pad=(0, 0), full=False):
    g = gen(seed)

    def rows(n, extra):
        lo = -128 if full else -127
        return torch.randint(lo, 128, (n, k + extra), generator=g, device=device(), dtype=torch.int8)[:, :k]

    scale = lambda n: torch.exp(torch.randn(n, generator=g, device=device())) * 1e-3
    return rows(M, pad[0]), scale(M), rows(N, pad[1]), scale(N)


def run(x, xs, w, ws, dtype, bias=None):
    out = torch.full((x.shape[0] + 1, w.shape[0]), 9.0, dtype=dtype, device=device())
    assert K().linear_int8(x, xs, w, ws, out[:-1], bias) is not None
    K().raise_on_status()
    assert (out[-1] == 9.0).all()
    return out[:-1]


# every width of the token tile and its edges; channels and k that end inside a tile; k of one instruction, one stage, past the ring;
# products whose tiles are shared by 1 to 8 blocks
PRODUCTS = [(1, 1, 16), (1, 6144, 4096), (2, 128, 128), (7, 130, 144), (8, 24576, 1024), (16, 1000, 4096), (17, 257, 400),
            (32, 4096, 2048), (33, 384, 1040), (64, 4096, 12288), (65, 500, 272), (127, 129, 2064), (128, 6144, 1024), (129, 1030, 656),
            (200, 2048, 2048), (256, 640, 512), (257, 1000, 784), (511, 4096, 256), (1000, 2500, 528), (2048, 4096, 4096),
            (16, 7156, 5232), (13, 2000, 8208), (16, 6144, 2064), (20, 300, 2064), (30, 2000, 8208), (31, 6100, 2064), (31, 6683, 7072), (32, 12300, 1040),
            (61, 5000, 2064), (40, 520, 2064), (64, 10000, 528), (100, 24500, 272), (97, 4666, 4320), (125, 6100, 2064), (300, 4090, 2064),
            (333, 12200, 1040), (120, 2393, 5856), (513, 6200, 1040), (2047, 4095, 272), (700, 20001, 400),
            (6, 4239, 5808), (73, 19627, 4096), (257, 24500, 2576), (19, 600, 2384), (769, 6100, 528), (193, 24000, 1040), (385, 9000, 1040), (4, 837, 2512), (19, 1279, 5904), (75, 5209, 7872), (91, 2059, 4640), (1, 6144, 4112)]


def test_the_products_take_every_form():
    """(1,000 x blocks that share a tile + its tokens; negative: pairs of blocks.  148 SMs, which the choice goes by.)"""
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        forms = {K().lib.ullm_linear_int8_form(*p) for p in PRODUCTS}
        assert forms >= {1016, 2016, 4016, 8016, 1032, 2032, 4032, 8032, 1064, 2064, 4064, 1128, 2128, 4128, -128, -192, -256}, forms


@pytest.mark.parametrize("M,N,k", PRODUCTS)
def test_product(M, N, k):
    x, xs, w, ws = operands(M + N + k, M, N, k)
    ref, size = product(x, xs, w, ws)
    for dtype in TYPES:
        check_product(run(x, xs, w, ws, dtype), ref, size)


@pytest.mark.parametrize("M,N,k", [(5, 260, 400), (64, 1001, 2048), (300, 513, 640)])
@pytest.mark.parametrize("dtype", TYPES)
def test_bias(M, N, k, dtype):
    x, xs, w, ws = operands(3, M, N, k)
    bias = torch.randn(N, generator=gen(4), device=device()).to(dtype)
    ref, size = product(x, xs, w, ws, bias)
    check_product(run(x, xs, w, ws, dtype, bias), ref, size)


# k that ends inside a piece of 16 bytes, with rows on borders of 16 (the tensor cores) and anywhere else (the plain kernel)
@pytest.mark.parametrize("M,N,k,pad", [(4, 300, 100, (12, 12)), (70, 257, 1100, (4, 20)), (300, 130, 77, (3, 19)), (1, 1, 1, (15, 15)),
                                       (4, 300, 100, (0, 0)), (70, 257, 1100, (0, 4)), (33, 65, 77, (0, 0)), (1, 40, 1, (0, 0)),
                                       (65, 100, 64, (1, 0)), (3, 5, 63, (0, 1))])
def test_rows_anywhere(M, N, k, pad):
    x, xs, w, ws = operands(M * N, M, N, k, pad)
    ref, size = product(x, xs, w, ws)
    check_product(run(x, xs, w, ws, torch.float32), ref, size)
    check_product(run(x[:, 1:], xs, w[:, 1:], ws, torch.bfloat16), *product(x[:, 1:], xs, w[:, 1:], ws)) if k > 1 else None


# more tokens than a grid has rows of tiles: pairs that go round (rows on borders of 16 bytes), the plain kernel's blocks that go round
@pytest.mark.parametrize("M,N,k", [(65535 * 128 + 300, 3, 16), (65535 * 32 + 100, 5, 3)])
def test_many_tokens(M, N, k):
    x, w = (torch.randint(-128, 128, (n, k), dtype=torch.int8, generator=gen(n % 997), device=device()) for n in (M, N))
    xs, ws = torch.ones(M, device=device()), torch.ones(N, device=device())
    out = torch.full((M, N), 0.5, device=device())
    K().linear_int8(x, xs, w, ws, out)
    sums = sum(x[:, i:i + 1].int() * w[:, i].int() for i in range(k))  # (whole numbers below 2^24)
    assert torch.equal(out, sums.float())


@pytest.mark.parametrize("pad", [0, 1])
def test_largest_sums(pad):
    """k of 131,071 with -128 everywhere: 2^14 k is below 2^31 by 16,384."""
    k = 131071
    x, w = (torch.full((n, k + pad), -128, dtype=torch.int8, device=device())[:, :k] for n in (3, 140))
    w[5] = 127
    one = lambda n: torch.ones(n, device=device())
    ref, size = product(x, one(3), w, one(140))
    assert ref.max() == 2 ** 14 * k and ref.min() == -128 * 127 * k
    check_product(run(x, one(3), w, one(140), torch.float32), ref, size)


@pytest.mark.parametrize("M", [6, 300])
def test_scales_that_are_not_finite_stay_with_their_row(M):
    x, xs, w, ws = operands(9, M, 200, 256)
    want = run(x, xs, w, ws, torch.bfloat16)
    xs[3], ws[7] = float("nan"), 0.0
    got = run(x, xs, w, ws, torch.bfloat16)
    assert got[3].isnan().all()
    got[3], want[3], want[:, 7] = 0.0, 0.0, 0.0
    assert torch.equal(got, want)


def test_rows_from_the_kernels_through_a_feed_forward():
    """Norm, product, gated activation, product, each stage against 64 bits of what the stage before left; eagerly, then captured and
    replayed with other inputs on another stream."""
    kk, T, H, I = K(), 24, 512, 1280
    g = gen(1)
    weights = [(torch.randn(n, k, generator=g, device=device()) * 0.05).to(torch.bfloat16) for n, k in ((2 * I, H), (H, I))]
    held = []
    for w in weights:
        q, s = kk.int8_rows(*w.shape), torch.empty(w.shape[0], device=device())
        kk.quantize_rows_int8(w, q, s)
        check_rows(q, s, w.double(), 0.0, 2.0 ** -24 * 1.01)
        held.append((q, s))
    norm = 1 + 0.2 * torch.randn(H, generator=g, device=device())
    x, res = rows_of(g, T, H, torch.bfloat16), rows_of(g, T, H, torch.bfloat16)
    hq, hs = kk.int8_rows(T, H), torch.empty(T, device=device())
    aq, as_ = kk.int8_rows(T, I), torch.empty(T, device=device())
    gu, out = (torch.empty(T, n, dtype=torch.bfloat16, device=device()) for n in (2 * I, H))

    def layer():
        kk.add_rmsnorm_int8(x, res, norm, 1e-6, hq, hs)
        kk.linear_int8(hq, hs, *held[0], gu)
        kk.act_mul_int8(gu, aq, as_)
        kk.linear_int8(aq, as_, *held[1], out)

    def check(before):
        check_rows(hq, hs, normed(x, before, norm, 1e-6), 2.0 ** -23, 2.0 ** -19)
        check_product(gu, *product(hq, hs, *held[0]))
        y, z = gated(gu, 0)
        check_rows(aq, as_, y, 2.0 ** -22 * (z.abs() + 3), float(2.0 ** -22 * (z.abs().max() + 3)))
        check_product(out, *product(aq, as_, *held[1]))

    before = res.clone()
    layer()
    check(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    stream = torch.cuda.Stream()
    for seed in (5, 6):
        g2 = gen(seed)
        x.copy_(rows_of(g2, T, H, torch.bfloat16))
        res.copy_(rows_of(g2, T, H, torch.bfloat16))
        before = res.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        check(before)
    kk.raise_on_status()


@pytest.mark.parametrize("M", [4, 300])
def test_a_weight_made_right_in_front_of_its_product(M):
    """The product may start beside the kernel that makes its weight; it sees that weight all the same."""
    kk, N, k = K(), 2048, 2048
    x, xs, _, _ = operands(1, M, 8, k)
    q, s = kk.int8_rows(N, k), torch.empty(N, device=device())
    outs, ws = [], [torch.randn(N, k, generator=gen(i), device=device()).to(torch.bfloat16) for i in range(6)]
    torch.cuda.synchronize()
    for w in ws:
        out = torch.empty(M, N, device=device())
        kk.quantize_rows_int8(w, q, s)
        kk.linear_int8(x, xs, q, s, out)
        outs.append(out)
    for w, out in zip(ws, outs):
        kk.quantize_rows_int8(w, q, s)
        torch.cuda.synchronize()
        check_product(out, *product(x, xs, q, s))


def test_two_streams_at_once():
    kk = K()
    sets = [operands(20 + i, 40, 3000, 2048) for i in range(2)]
    outs = [torch.empty(40, 3000, device=device()) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for ops, out, st in zip(sets, outs, streams):
            with torch.cuda.stream(st):
                kk.linear_int8(*ops, out)
    torch.cuda.synchronize()
    for ops, out in zip(sets, outs):
        check_product(out, *product(*ops))


def test_graphs_side_by_side():
    """Two recorded graphs of the same products, replayed on two streams at once: nothing is shared between them."""
    kk = K()
    sets = [operands(30 + i, 24, 2000, 8192) for i in range(2)]
    outs = [torch.empty(24, 2000, device=device()) for _ in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for ops, out in zip(sets, outs):
        kk.linear_int8(*ops, out)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(5):
                kk.linear_int8(*ops, out)
    for out in outs:
        out.fill_(9.0)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for ops, out in zip(sets, outs):
        check_product(out, *product(*ops))


def test_more_than_31_bits_of_elements():
    """A weight of 2.3 G elements made and used, a result of 2.4 G: rows past the 31st bit are where they belong."""
    kk, N, k = K(), 70001, 32768
    w = torch.zeros(N, k, dtype=torch.bfloat16, device=device())
    last = rows_of(gen(1), 300, k, torch.bfloat16)
    w[-300:], w[:300] = last, last.flip(0)
    q, s = kk.int8_rows(N, k), torch.empty(N, device=device())
    kk.quantize_rows_int8(w, q, s)
    del w
    check_rows(q[-300:], s[-300:], last.double(), 0.0, 2.0 ** -24 * 1.01)
    assert torch.equal(q[:300], q[-300:].flip(0)) and not s[300:-300].any() and not q[40000].any()
    for M in (3, 300):
        x, xs, _, _ = operands(2, M, 1, k)
        out = run(x, xs, q, s, torch.bfloat16)
        check_product(out[:, -300:], *product(x, xs, q[-300:], s[-300:]))
        assert torch.equal(out[:, :300], out[:, -300:].flip(1)) and not out[:, 300:-300].any()
    del q, out
    M, N, k = 40000, 60001, 48
    x, xs, w, ws = operands(3, M, N, k)
    out = run(x, xs, w, ws, torch.bfloat16)
    for rows in (slice(0, 64), slice(35000, 35064), slice(M - 64, M)):
        check_product(out[rows], *product(x[rows], xs[rows], w, ws))


def test_refusals_on_the_gpu():
    """The same refusals as on the CPU (test_int8_refusals.py), through the checks that run here; nothing is launched or written."""
    from ullm_b200.csrc.ops import KernelError

    kk = K()
    x, w = torch.zeros(3, 32, dtype=torch.int8, device=device()), torch.zeros(5, 32, dtype=torch.int8, device=device())
    xs, ws, out = torch.zeros(3, device=device()), torch.zeros(5, device=device()), torch.full((3, 5), 9.0, device=device())
    v, gu = torch.zeros(3, 32, device=device()), torch.zeros(3, 64, device=device())
    before = kk.launches
    for call in (lambda: kk.linear_int8(v, xs, w, ws, out), lambda: kk.linear_int8(x[:, :16], xs, w, ws, out),
                 lambda: kk.linear_int8(x, xs[:2], w, ws, out), lambda: kk.linear_int8(x, xs, w, ws.double(), out),
                 lambda: kk.linear_int8(x, xs, w, ws, out.t()), lambda: kk.linear_int8(x, xs, w, ws, out.double()),
                 lambda: kk.linear_int8(x, xs, w, ws, out, ws[:4]), lambda: kk.linear_int8(x, xs, w, ws, out, ws.half()),
                 lambda: kk.linear_int8(x[:1].expand(3, 32), xs, w, ws, out), lambda: kk.linear_int8(x, xs, w.cpu(), ws, out),
                 lambda: kk.linear_int8(x[0], xs, w, ws, out), lambda: kk.linear_int8(x[:, :0], xs, w[:, :0], ws, out),
                 lambda: kk.quantize_rows_int8(v.double(), x, xs), lambda: kk.quantize_rows_int8(v, x[:, :31], xs),
                 lambda: kk.quantize_rows_int8(v, x, xs.cpu()), lambda: kk.quantize_rows_int8(v.t(), x, xs),
                 lambda: kk.quantize_rows_int8(v[:, :0], x[:, :0], xs),
                 lambda: kk.act_mul_int8(gu[:, :63], x, xs), lambda: kk.act_mul_int8(gu, x, xs, 2), lambda: kk.act_mul_int8(v, x, xs),
                 lambda: kk.add_rmsnorm_int8(v, v[:2], torch.ones(32, device=device()), 1e-6, x, xs),
                 lambda: kk.add_rmsnorm_int8(v, None, torch.ones(31, device=device()), 1e-6, x, xs),
                 lambda: kk.add_rmsnorm_int8(gu[:, :32], None, torch.ones(32, device=device()), 1e-6, x, xs)):
        with pytest.raises(KernelError):
            call()
    assert (out == 9.0).all() and kk.launches - before <= 8  # (a launcher's own refusal is counted)
    # no rows: nothing to do
    assert kk.linear_int8(x[:0], xs[:0], w, ws, out[:0]) is not None and kk.quantize_rows_int8(v[:0], x[:0], xs[:0]) is not None
    # eps as a whole number, and no weight on a norm's statistics
    kk.add_rmsnorm_int8(v + 1, None, torch.ones(32, device=device()), 0, x, xs)
    assert (x == 127).all() and torch.allclose(xs, torch.full_like(xs, 1 / 127))
