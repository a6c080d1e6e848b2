"""8-bit rows whose whole numbers are known without a rounding: elements halfway between two of them, and the nearest numbers on both
sides."""

import pytest
import torch

from conftest import device
from plain_int8 import check_rows, gated, normed
from test_gpu_kernels import K

pytestmark = [pytest.mark.gpu, pytest.mark.needs_cuda]

TYPES = [torch.bfloat16, torch.float16, torch.float32]
INTS = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32}
BITS = {torch.bfloat16: 7, torch.float16: 10, torch.float32: 23}


def whole(x):
    """(The whole numbers nearest to 127 x / max|x| of each row, ties to even; how far each element is from a middle between two, of its
    value.)  127 x, n max (n < 128) and their difference take fewer than 53 bits where they matter (24 + 7, and 8 for the distance of an
    element that is not held as 0), so that 64 bits decide exactly."""
    a, most = 127 * x.double().abs(), x.double().abs().amax(1, keepdim=True)
    n = torch.floor(a / most)
    n = n - (a < n * most).double()
    n = n + (a >= (n + 1) * most).double()
    rest = 2 * (a - n * most)
    up = (rest > most) | ((rest == most) & (n % 2 == 1))
    return torch.sign(x.double()) * (n + up), (rest - most).abs() / (2 * a)


def check(q, x):
    """16-bit rows: every whole number is the nearest one.  32-bit rows: the quotient 127 / max is rounded, by a step (2^-23) at most; what is
    not a tie and as near to a middle as that may be on its other side."""
    want, apart = whole(x)
    wrong = q.double() != want
    if x.dtype == torch.float32:
        assert not (wrong & ((apart == 0) | (apart > 2.0 ** -23))).any() and ((q.double() - want).abs() <= 1).all()
    else:
        assert not wrong.any(), f"{int(wrong.sum())} of {q.numel()}"


def border_rows(dtype, rows, cols, exponent, seed=1):
    """Rows whose largest elements go through the type's significands (all of them in 16 bits where the rows suffice), 2^exponent large;
    the others are the numbers of the type next to the middles between whole numbers, and their neighbours on both sides."""
    g = torch.Generator(device=device()).manual_seed(seed)
    count = 1 << BITS[dtype]
    sig = (torch.arange(rows, device=device()) * (1 if rows >= count or count <= 1024 else count // rows)) % count
    if dtype == torch.float32:  # (any low bits)
        sig = (sig + torch.randint(0, count, (rows,), generator=g, device=device())) % count
    most = ((1 + sig.double() / count) * 2.0 ** exponent)[:, None]
    odd = 2 * torch.randint(0, 127, (rows, cols), generator=g, device=device()).double() + 1
    odd = torch.where(torch.rand(rows, cols, generator=g, device=device()) < 0.25, 127.0, odd)  # (the middle that every type holds)
    x = (most * odd / 254).to(dtype)
    step = torch.randint(-1, 2, (rows, cols), generator=g, device=device())
    x = (x.view(INTS[dtype]) + step.to(INTS[dtype])).view(dtype)  # (positive numbers' bits follow one another)
    x = torch.where(x.double() > most, most.to(dtype), x)
    x = torch.where(torch.rand(rows, cols, generator=g, device=device()) < 0.5, x, -x)
    x[:, cols // 2] = most[:, 0].to(dtype)
    # rows whose largest is a multiple of 127 have ties at every odd number
    x[::5] = torch.where(x[::5].abs() == most[::5].to(dtype), x[::5].sign() * 127 * 2.0 ** (exponent - 6),
                         x[::5].sign() * (odd[::5] * 2.0 ** (exponent - 7)).to(dtype))
    return x.contiguous()


# rows in registers, with one to eight elements a thread; pieces shifted into place; element by element; read twice; blocks that stay
SIZES = [(128, 512), (1024, 1024), (256, 4096), (300, 1003), (64, 65), (40, 16384), (16, 40000), (700, 4101), (1200, 8192), (700, 16384), (4096, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_whole_numbers_are_the_nearest_and_ties_go_to_even(rows, cols, dtype):
    x = border_rows(dtype, rows, cols, 3)
    q, scales = K().int8_rows(rows, cols), torch.empty(rows, device=device())
    K().quantize_rows_int8(x, q, scales)
    check(q, x)


@pytest.mark.parametrize("dtype,exponent", [(torch.float16, 14), (torch.float16, -12), (torch.bfloat16, 127), (torch.bfloat16, 101), (torch.bfloat16, -89),
                                            (torch.bfloat16, -91), (torch.bfloat16, -115), (torch.float32, 127), (torch.float32, 99),
                                            (torch.float32, -90), (torch.float32, -102)])
def test_so_do_the_largest_and_smallest_rows(dtype, exponent):
    x = border_rows(dtype, 256, 640, exponent)
    x = torch.where(x.isfinite(), x, x.sign())
    q, scales = torch.empty(256, 640, dtype=torch.int8, device=device()), torch.empty(256, device=device())
    K().quantize_rows_int8(x, q, scales)
    check(q, x)


def test_a_half_of_the_largest_is_64():
    """Every significand of 16-bit rows: 63.5 goes to 64."""
    for dtype in (torch.bfloat16, torch.float16):
        count = 1 << BITS[dtype]
        x = torch.zeros(count, 64, dtype=dtype, device=device())
        x[:, 0] = 1 + torch.arange(count, device=device()) / count
        x[:, 1:] = -x[:, :1] / 2
        q, scales = torch.empty(count, 64, dtype=torch.int8, device=device()), torch.empty(count, device=device())
        K().quantize_rows_int8(x, q, scales)
        assert (q[:, 0] == 127).all() and (q[:, 1:] == -64).all()


# rows in registers (one, two and four groups a thread), of any length, element by element, read twice, and blocks that stay
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("rows,cols", [(4, 5), (9, 1024), (9, 9000), (9, 20000), (4, 40000), (700, 4101), (9, 1003), (600, 16384)])
def test_gates_far_below_zero(rows, cols, act, dtype):
    """Gates whose activation is below 2^-126: rows of these alone, beside ups that make more of it (2^80; float16 has none such), and beside
    ordinary ones."""
    g = torch.Generator(device=device()).manual_seed(cols)
    x = torch.randn(rows, 2 * cols, generator=g, device=device())
    lowest = torch.rand(rows, cols, generator=g, device=device())
    x[:, :cols] = -85 - 60 * lowest if act == 0 else -9.7 - 1.5 * lowest
    x[:, cols:] *= 1.0 if dtype == torch.float16 else 2.0 ** 80
    x[1] = torch.randn(2 * cols, generator=g, device=device())
    x[1, 0], x[1, cols] = -100.0, 1.0  # (nothing that counts)
    x[2, cols - 1] = 30.0 if act == 0 else 9.5  # (and the rest of the row is nothing beside it)
    x[3] = 0.0
    x = x.to(dtype)
    q, scales = K().int8_rows(rows, cols), torch.empty(rows, device=device())
    K().act_mul_int8(x, q, scales, act)
    y, z = gated(x, act)
    rel = 2.0 ** -22 * (z.abs() + 3)
    fine = y.abs().amax(1) > 2.0 ** -125  # (32-bit numbers below 2^-126 have fewer bits)
    fine[3] = True
    check_rows(q[fine], scales[fine], y[fine], rel[fine], float(rel.max()))
    assert scales[3] == 0 and not q[3].any() and fine[:3].sum() >= (2 if dtype == torch.float16 else 3)


# rows in registers (one, two and four groups a thread), of any length, element by element, read twice
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_residual", [True, False])
@pytest.mark.parametrize("cols", [5, 1024, 4096, 9000, 16384, 20000, 33000, 40000, 4101, 1003])
def test_norms_whose_squares_pass_32_bits(cols, with_residual, dtype):
    """Rows of every size with an eps that counts and with none, and rows that hold one element of that size."""
    g = torch.Generator(device=device()).manual_seed(cols)
    sizes = torch.tensor([-110, -80, -64, -63, -50, -40, -38, -10, 0, 40, 45, 50, 55, 60, 63, 64, 65, 80, 100, 110, 122], device=device())
    sizes = sizes.repeat_interleave(2).double()[:, None]
    x = torch.randn(len(sizes), cols, generator=g, device=device(), dtype=torch.float64)
    one = torch.where(torch.arange(cols, device=device()) == cols - 2, 2.0 ** sizes[1::2], 1.0)
    x[::2] *= 2.0 ** sizes[::2]
    x[1::2] *= one
    x = x.to(dtype)
    residual = (x.roll(1, 1) * 0.5) if with_residual else None
    weight = 1 + 0.3 * torch.randn(cols, generator=g, device=device())
    for eps in (1e-6, 0.0, 2.0 ** -60):
        res = residual.clone() if with_residual else None
        q, scales = K().int8_rows(len(x), cols), torch.empty(len(x), device=device())
        K().add_rmsnorm_int8(x, res, weight, eps, q, scales)
        # as for rows of ordinary size (an element: the sum and the weight's product; a scale: besides, half of the sum of squares' error),
        # and squares that are below 2^-126 beside an eps above 2^-73: below 2^-40 of it
        check_rows(q, scales, normed(x, residual, weight, eps), 2.0 ** -23, 2.0 ** -24 * ((cols / 1024 + 40) / 2 + 10))
        if with_residual:
            assert torch.equal(res, (x.float() + residual.float()).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [1 << 23, 5000001])
def test_a_norm_of_millions_of_columns(cols, dtype):
    """A thread's sum of thousands of squares: elements of one size, whose additions would all be rounded the same way, and others."""
    x = torch.full((2, cols), 1.0078125, device=device()).to(dtype)
    x[1] = torch.randn(cols, generator=torch.Generator(device=device()).manual_seed(1), device=device()).abs().to(dtype)
    weight = torch.ones(cols, device=device())
    q, scales = K().int8_rows(2, cols), torch.empty(2, device=device())
    for size in (1.0, 2.0 ** 70):
        K().add_rmsnorm_int8(x * size, None, weight, 1e-6, q, scales)
        # half of the sum's error: eight of a thread's neighbouring elements, ten additions of the block, the sum rounded; the rest of a norm
        check_rows(q, scales, normed(x * size, None, weight, 1e-6), 2.0 ** -23, 2.0 ** -24 * ((8 + 11) / 2 + 10))
