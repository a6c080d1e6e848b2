"""Every form of the kernels of 8-bit rows (csrc/rows_int8.cu, `rq_choose`), for each type and kind of rows, against the same in 64 bits."""

import pytest
import torch

from conftest import device
from plain_int8 import check_rows, gated, normed
from test_gpu_int8 import gen, placed, room, rows_of
from test_gpu_kernels import K

pytestmark = [pytest.mark.gpu, pytest.mark.needs_cuda]

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
PLAIN, GATED, NORMED = 0, 1, 2
PLAIN_REL = 2.0 ** -24 * 1.01

# (rows, columns, columns between rows of the output) that blocks which stay take: fewer rows than the blocks of a full chip would have, and
# numbers of rows that leave some blocks a row less; one and two blocks an SM, every number of groups a thread
STAYING = {2: [(592, 16384, 16384), (1300, 25600, 25600), (700, 20008, 20016), (2049, 16392, 16392), (593, 32768, 32776)],
           4: [(592, 8192, 8192), (1301, 12800, 12800), (700, 9004, 9008), (2049, 8196, 8196), (593, 16384, 16388)]}


def form(kind, dtype, rows, cols, place=2):
    return K().lib.ullm_rows_int8_form(kind, TYPES[dtype], rows, cols, place)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [PLAIN, GATED])
@pytest.mark.parametrize("case", range(5))
def test_blocks_that_stay(case, kind, dtype):
    rows, cols, wide = STAYING[4 if dtype == torch.float32 else 2][case]
    stays = form(kind, dtype, rows, cols) == -1
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        # (the last one's gated rows are too long for two slots of shared memory)
        assert stays or (kind == GATED and case == 4)
    q, untouched = room(rows, cols, wide - cols)
    scales = torch.full((rows,), 9.0, device=device())
    g = gen(rows + cols)
    if kind == PLAIN:
        x = rows_of(g, rows, wide, dtype)[:, :cols]
        K().quantize_rows_int8(x, q, scales)
        check_rows(q, scales, x.double(), 0.0, PLAIN_REL)
    else:
        x = rows_of(g, rows, 2 * cols, dtype)
        for act in (0, 1):
            scales.fill_(9.0)
            K().act_mul_int8(x, q, scales, act)
            for part in range(0, rows, 300):  # (64-bit rows of all would be some GB)
                y, z = gated(x[part:part + 300], act)
                rel = 2.0 ** -22 * (z.abs() + 3)
                check_rows(q[part:part + 300], scales[part:part + 300], y, rel, float(rel.max()))
    untouched()
    K().raise_on_status()


# (rows, columns, place: 2 in pieces of 16 bytes, 1 of any length, 0 with 8-bit rows anywhere)
SHAPES = [(3, 64, 2), (5, 2560, 2), (4, 8192, 2), (3, 12288, 2), (2, 16384, 2), (2, 24576, 2), (2, 33024, 2), (2, 50000, 2), (900, 263, 1), (5, 33, 1),
          (600, 531, 1), (300, 903, 1), (9, 4095, 1), (3, 8191, 1), (3, 9001, 1), (3, 16387, 1), (2, 32767, 1), (2, 5001, 1), (2, 40001, 1),
          (1200, 1003, 1), (3, 5001, 0), (300, 6000, 0), (3, 1001, 0), (3, 9000, 0)]


def test_the_shapes_take_every_form():
    for dtype in TYPES:
        v = 4 if dtype == torch.float32 else 8
        for kind in (PLAIN, GATED, NORMED):
            forms = {form(kind, dtype, *s) for s in SHAPES}
            want = {100 * v + per for per in (0, 1, 2, 4)} | {1000 + 100 * v + per for per in (1, 2, 4)} | {100, 101, 102, 104, 108}
            assert forms == want, (dtype, kind, forms ^ want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,place", SHAPES)
def test_rows_of_every_form(rows, cols, place, dtype):
    g = gen(rows * 11 + cols)
    q, untouched = room(rows, cols, -cols % 16 + (0 if place else 1))
    scales = torch.full((rows,), 9.0, device=device())
    x, gu, res = (rows_of(g, rows, n, dtype) for n in (cols, 2 * cols, cols))
    weight = 1 + 0.3 * torch.randn(cols, generator=g, device=device())
    K().quantize_rows_int8(x, q, scales)
    check_rows(q, scales, x.double(), 0.0, PLAIN_REL)
    K().act_mul_int8(gu, q, scales)
    y, z = gated(gu, 0)
    rel = 2.0 ** -22 * (z.abs() + 3)
    check_rows(q, scales, y, rel, float(rel.max()))
    want, y = (x.float() + res.float()).to(dtype), normed(x, res, weight, 1e-6)
    K().add_rmsnorm_int8(x, res, weight, 1e-6, q, scales)
    check_rows(q, scales, y, 2.0 ** -23, 2.0 ** -24 * ((cols / 1024 + 40) / 2 + 10))
    assert torch.equal(res, want)
    untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,offset", [(9, 4096, 0), (2, 16384, 0), (2, 33024, 0), (2, 40001, 0), (9, 1003, 3), (9, 4091, 0), (5, 9001, 1),
                                              (3, 16387, 5), (300, 2043, 2)])
def test_a_residual_that_is_the_input_in_every_form(rows, cols, offset, dtype):
    """x and residual one tensor: in registers, read twice, element by element, and in pieces whose stores take a neighbour's elements along."""
    once, weight = rows_of(gen(cols), rows, cols, dtype), torch.ones(cols, device=device())
    x, around = placed(once, offset)
    q, untouched = room(rows, cols, -cols % 16)
    scales = torch.empty(rows, device=device())
    K().add_rmsnorm_int8(x, x, weight, 1e-6, q, scales)
    check_rows(q, scales, normed(once, once, weight, 1e-6), 2.0 ** -23, 2.0 ** -24 * ((cols / 1024 + 40) / 2 + 10))
    assert torch.equal(x, (once.float() * 2).to(dtype))
    around()
    untouched()
