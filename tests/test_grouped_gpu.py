"""Products whose matrix is chosen by the row (grouped_matmul, its weight gradient, lora_matmul) against 64-bit sums.

Bounds: a sum of K products in fp32 is within K * 2^-23 of its terms' magnitudes (the tensor core may truncate where a
rounding would take half of that), the one rounding at the store within half a step of the stored type, and the value
between the adapters' two products within half a step squared (it is kept to 2^-22 of itself, fp16's half step squared).
"""

import inspect
import warnings

import pytest
import torch

from gpu_util import assert_device_healthy

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def healthy():
    yield
    assert_device_healthy()


def normal(seed, *shape, kind=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(kind)


def bounds_of(lengths, first=0, dtype=torch.int32):
    at = [first]
    for length in lengths:
        at.append(at[-1] + length)
    return torch.tensor(at, dtype=dtype, device="cuda")


def assert_within(actual, exact, sums):
    """sums: how far the sum may be off before it is rounded to the stored type."""
    step = torch.finfo(actual.dtype).eps / 2
    tiny = torch.finfo(actual.dtype).smallest_normal * step
    error = (actual.double() - exact).abs()
    bound = sums + step * (exact.abs() + sums) + tiny
    worst = (error / bound).max().item() if error.numel() else 0.0
    assert worst <= 1.0, worst


def spans(offsets):
    at = offsets.tolist()
    return list(zip(at[:-1], at[1:]))


def check_grouped(lhs, rhs, offsets, output, before):
    exact, sums = before.double(), torch.zeros_like(before, dtype=torch.float64)
    held = torch.zeros(lhs.shape[0], dtype=torch.bool, device="cuda")
    for e, (a, b) in enumerate(spans(offsets)):
        x, w = lhs[a:b].double(), rhs[e].double()
        exact[a:b] = x @ w
        sums[a:b] = x.abs() @ w.abs() * (lhs.shape[1] * 2.0 ** -23)
        held[a:b] = True
    assert torch.equal(output[~held], before[~held])
    assert_within(output[held], exact[held], sums[held])


def run_grouped(lhs, rhs, offsets):
    from ninetoothed_b200.torch_ops import ops

    output = torch.full((lhs.shape[0], rhs.shape[2]), 7.0, dtype=lhs.dtype, device="cuda")
    before = output.clone()
    ops.grouped_matmul(lhs, rhs, offsets, output)
    check_grouped(lhs, rhs, offsets, output, before)
    return output


# one row, single rows and empty runs, lengths around the 32-row boxes and the 128- and 256-row tiles, long runs
LENGTHS = [[1], [0, 1, 0], [0, 0], [3, 0, 1, 32, 33], [127, 128, 129, 0, 1], [255, 256, 257], [1] * 70, [700, 0, 1100]]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("k, n", [(8, 8), (64, 264), (200, 1000), (520, 136)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_grouped_matmul(lengths, k, n, transposed):
    kind = KINDS[len(lengths) % 2]
    rows, groups = sum(lengths), len(lengths)
    lhs = normal(1, rows + 5, k, kind=kind)
    rhs = normal(2, groups, n, k, kind=kind).transpose(1, 2) if transposed else normal(2, groups, k, n, kind=kind)
    run_grouped(lhs, rhs, bounds_of(lengths, first=2))


@pytest.mark.parametrize("rows, groups, k, n", [(2048, 4, 256, 2056), (6000, 40, 136, 528), (4096, 2048, 72, 64),
                                                (300, 1, 4104, 64)])
def test_grouped_matmul_larger(rows, groups, k, n):
    g = torch.Generator().manual_seed(rows)
    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=g).sort().values.tolist()
    offsets = torch.tensor([0, *cuts, rows], dtype=torch.int64, device="cuda")
    run_grouped(normal(3, rows, k), normal(4, groups, k, n), offsets)


def test_whole_numbers_are_exact():
    """Small whole numbers: every product and sum is exact, so every element must be the same bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    lhs = torch.randint(-3, 4, (900, 136), generator=g, device="cuda").half()
    rhs = torch.randint(-3, 4, (5, 136, 328), generator=g, device="cuda").half()
    lengths = [100, 0, 511, 1, 288]
    output = run_grouped(lhs, rhs, bounds_of(lengths))
    expected = torch.cat([lhs[a:b].double() @ rhs[e].double() for e, (a, b) in enumerate(spans(bounds_of(lengths)))])
    assert torch.equal(output.double(), expected)


def test_grouped_matmul_views_and_strided_bounds():
    lhs = normal(6, 400, 300)[:, 8:208]                       # rows of 200 in rows of 300 (pitch not a multiple of 8)
    wide = normal(6, 400, 304)[:, 8:208]
    rhs = normal(7, 3, 200, 400)[:, :, 16:152]
    offsets = torch.stack([bounds_of([150, 50, 200]), bounds_of([1, 2, 3])], 1)[:, 0]
    assert offsets.stride(0) == 2
    from ninetoothed_b200 import _capi

    run_grouped(wide, rhs, offsets)
    before = _capi.plain_launches()
    with pytest.warns(_capi.SlowPathWarning):
        run_grouped(lhs, rhs, offsets)
    assert _capi.plain_launches() == before + 1
    # outputs: columns of a wider tensor, odd offset, and a transposed tensor
    for output in (torch.full((400, 171), 7.0, dtype=torch.bfloat16, device="cuda")[:, 3:139],
                   torch.full((136, 400), 7.0, dtype=torch.bfloat16, device="cuda").t()):
        first = output.clone()
        _capi.grouped_matmul(wide, rhs, offsets, output)
        check_grouped(wide, rhs, offsets, output, first)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("lengths", [[3, 0, 5, 1], [150, 260, 0, 90], [900, 700, 45, 300]], ids=str)
def test_matrices_between_each_others_rows(lengths, transposed):
    """Matrices held with their index in the middle, which is how some checkpoints have them: on the tensor cores, as others."""
    from ninetoothed_b200 import _capi

    k, n, rank, rows = 264, 520, 24, sum(lengths)

    def middle(t):  # the same matrices in memory as [rows, count, columns], either way round
        if transposed:
            return middle_of(t.transpose(1, 2)).transpose(1, 2)
        return middle_of(t)

    def middle_of(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    before = _capi.plain_launches()
    lhs, grad, offsets = normal(110, rows, k), normal(111, rows, n), bounds_of(lengths)
    run_grouped(lhs, middle(normal(112, 4, k, n)), offsets)
    check_rhs_grad(lhs, grad, offsets, rhs_grad=middle_of(torch.full((4, k, n), float("nan"), dtype=torch.bfloat16, device="cuda")))
    lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, [1, 0, 2, 3], k, n, rank, 4, torch.bfloat16)
    run_lora(lhs, rhs, middle(down), middle(up), scales, offsets, which)
    assert _capi.plain_launches() == before


def test_the_slow_path_warning_names_the_operators_call():
    from ninetoothed_b200 import _capi
    from ninetoothed_b200.torch_ops import ops

    lhs, rhs, offsets = normal(8, 40, 7), normal(9, 2, 7, 9), bounds_of([10, 30])
    output = torch.empty(40, 9, dtype=torch.bfloat16, device="cuda")
    with pytest.warns(_capi.SlowPathWarning) as caught:
        ops.grouped_matmul(lhs, rhs, offsets, output)
    assert (caught[0].filename, caught[0].lineno) == (__file__, inspect.currentframe().f_lineno - 1)


@pytest.mark.parametrize("k, n", [(0, 8), (7, 9), (33, 70)])
def test_grouped_matmul_on_sizes_no_tensor_map_addresses(k, n):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        run_grouped(normal(8, 40, k), normal(9, 4, k, n), bounds_of([5, 0, 30, 1], first=1))


def test_neighbouring_rows_do_not_leak():
    """Infinities and NaN in rows of no run and in another run's rows and matrix stay where they are."""
    lengths = [37, 90, 61]
    offsets = bounds_of(lengths, first=4)
    lhs, rhs = normal(10, 200, 72), normal(11, 3, 72, 80)
    clean = run_grouped(lhs, rhs, offsets)
    lhs[:4] = float("nan")
    lhs[41:131] = float("inf")
    lhs[192:] = float("nan")
    rhs[1] = float("nan")
    from ninetoothed_b200.torch_ops import ops

    output = torch.full_like(clean, 7.0)
    ops.grouped_matmul(lhs, rhs, offsets, output)
    for a, b in ((0, 41), (131, 200)):
        assert torch.equal(output[a:b], clean[a:b])
    assert output[41:131].isnan().all()


@pytest.mark.parametrize("values, meaning", [([-5, 10, 300], [0, 10, 100]), ([0, 60, 30, 80], [0, 60, 60, 80]),
                                             ([90, 20, 95], [90, 90, 95]), ([2 ** 40, 0], [100, 100]),
                                             ([-2 ** 40, 2 ** 40], [0, 100])])
def test_bounds_out_of_order_or_range_stay_inside_the_tensors(values, meaning):
    from ninetoothed_b200.torch_ops import ops

    lhs, rhs = normal(12, 100, 64), normal(13, len(values) - 1, 64, 64)
    offsets = torch.tensor(values, dtype=torch.int64, device="cuda")
    output = torch.full((100, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    before = output.clone()
    ops.grouped_matmul(lhs, rhs, offsets, output)
    check_grouped(lhs, rhs, torch.tensor(meaning), output, before)
    grad = normal(14, 100, 72)
    check_rhs_grad(lhs, grad, offsets, torch.tensor(meaning))


def check_rhs_grad(lhs, grad, offsets, meaning=None, rhs_grad=None):
    from ninetoothed_b200.torch_ops import ops

    groups = offsets.shape[0] - 1
    if rhs_grad is None:
        rhs_grad = torch.full((groups, lhs.shape[1], grad.shape[1]), float("nan"), dtype=lhs.dtype, device="cuda")
    ops.grouped_matmul_rhs_grad(lhs, grad, offsets, rhs_grad)
    for e, (a, b) in enumerate(spans(offsets if meaning is None else meaning)):
        x, y = lhs[a:b].double(), grad[a:b].double()
        assert_within(rhs_grad[e], x.t() @ y, x.abs().t() @ y.abs() * (max(1, b - a) * 2.0 ** -23))
        if a == b:
            assert torch.equal(rhs_grad[e], torch.zeros_like(rhs_grad[e]))
    return rhs_grad


@pytest.mark.parametrize("m, n", [(8, 8), (264, 72), (136, 520), (1000, 384)])
@pytest.mark.parametrize("lengths", LENGTHS + [[16, 17, 63, 64, 65, 79, 80, 81]], ids=str)
def test_rhs_grad(lengths, m, n):
    kind = KINDS[len(lengths) % 2]
    rows = sum(lengths) + 5
    # rows of no run hold NaN: none may enter a sum
    lhs, grad = normal(15, rows, m, kind=kind), normal(16, rows, n, kind=kind)
    for t in (lhs, grad):
        t[:2] = float("nan")
        t[2 + sum(lengths):] = float("nan")
    check_rhs_grad(lhs, grad, bounds_of(lengths, first=2))


def test_rhs_grad_larger_views_and_unaddressable():
    rows, groups = 6000, 40
    g = torch.Generator().manual_seed(1)
    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=g).sort().values.tolist()
    offsets = torch.tensor([0, *cuts, rows], dtype=torch.int64, device="cuda")
    check_rhs_grad(normal(17, rows, 400)[:, 8:336], normal(18, rows, 600)[:, :528], offsets)
    # a gradient in the layout of a transposed view
    out = torch.empty(groups, 528, 328, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    check_rhs_grad(normal(17, rows, 400)[:, 8:336], normal(18, rows, 600)[:, :528], offsets, rhs_grad=out)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        check_rhs_grad(normal(19, 60, 13), normal(20, 60, 21), bounds_of([20, 0, 39], first=1))
        check_rhs_grad(normal(19, 0, 16), normal(20, 0, 24), bounds_of([0, 0]))


def test_rhs_grad_keeps_a_neighbours_infinities_out():
    lengths = [37, 90, 61]
    offsets = bounds_of(lengths)
    lhs, grad = normal(21, 188, 72), normal(22, 188, 80)
    clean = check_rhs_grad(lhs, grad, offsets)
    lhs[37:127] = float("inf")
    grad[37:127] = float("nan")
    from ninetoothed_b200.torch_ops import ops

    out = torch.empty_like(clean)
    ops.grouped_matmul_rhs_grad(lhs, grad, offsets, out)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert out[1].isnan().all()


def check_lora(lhs, rhs, down, up, scales, offsets, adapters, output, before):
    exact, sums = before.double(), torch.zeros_like(before, dtype=torch.float64)
    held = torch.zeros(lhs.shape[0], dtype=torch.bool, device="cuda")
    unit = 2.0 ** -23
    part = (torch.finfo(lhs.dtype).eps / 2) ** 2
    least = torch.finfo(lhs.dtype).smallest_normal * torch.finfo(lhs.dtype).eps
    k, rank = lhs.shape[1], down.shape[2]
    for (a, b), adapter in zip(spans(offsets), adapters.tolist()):
        x = lhs[a:b].double()
        held[a:b] = True
        exact[a:b] = x @ rhs.double()
        sums[a:b] = x.abs() @ rhs.double().abs() * ((k + rank) * unit)
        if 0 <= adapter < down.shape[0]:
            d, u, s = down[adapter].double(), up[adapter].double(), scales[adapter].double()
            low = s * (x @ d)
            low_size = s.abs() * (x.abs() @ d.abs())
            exact[a:b] += low @ u
            off = low_size * ((k + 1) * unit) + low.abs() * part + least
            sums[a:b] += (off + low.abs() * ((k + rank) * unit)) @ u.abs()
    assert torch.equal(output[~held], before[~held])
    assert_within(output[held], exact[held], sums[held])


def run_lora(lhs, rhs, down, up, scales, offsets, adapters, workspace=None):
    from ninetoothed_b200 import _capi
    from ninetoothed_b200.torch_ops import ops

    output = torch.full((lhs.shape[0], rhs.shape[1]), 7.0, dtype=lhs.dtype, device="cuda")
    before = output.clone()
    if workspace is None:
        ops.lora_matmul(lhs, rhs, down, up, scales, offsets, adapters, output)
    else:
        _capi.lora_matmul(lhs, rhs, down, up, scales, offsets, adapters, output, workspace=workspace)
    check_lora(lhs, rhs, down, up, scales, offsets, adapters, output, before)
    return output


def lora_inputs(lengths, adapters, k, n, rank, count, kind, padding=3, first=0):
    rows = sum(lengths) + padding + first
    return (normal(31, rows, k, kind=kind), normal(32, k, n, kind=kind, scale=k ** -0.5),
            normal(33, count, k, rank, kind=kind, scale=k ** -0.5), normal(34, count, rank, n, kind=kind, scale=rank ** -0.5),
            torch.linspace(0.5, 2.0, count, device="cuda"), bounds_of(lengths, first=first),
            torch.tensor(adapters, dtype=torch.int32, device="cuda"))


# (lengths, adapters): none, repeated, out of range on both sides, empty requests, requests that cross tile edges
REQUESTS = [([1], [0]), ([1], [-1]), ([0, 1, 0], [1, 2, 0]), ([1] * 70, [i % 5 - 1 for i in range(70)]),
            ([100, 60, 200, 1], [2, 2, 7, 0]), ([300, 0, 340], [1, 3, 1]), ([31, 33, 64, 127, 1], [3, 2, 1, 0, 4])]


@pytest.mark.parametrize("k, n, rank", [(64, 64, 16), (136, 200, 8), (520, 1032, 40), (256, 2048, 136)])
@pytest.mark.parametrize("lengths, adapters", REQUESTS, ids=str)
def test_lora_matmul(lengths, adapters, k, n, rank):
    run_lora(*lora_inputs(lengths, adapters, k, n, rank, 4, KINDS[len(lengths) % 2], first=len(lengths) % 3))


@pytest.mark.parametrize("turned", [(True, False, False), (False, True, False), (False, False, True), (True, True, True)])
def test_lora_matmul_transposed_views(turned):
    """Every matrix either way round; all three turned is the gradient towards lhs."""
    for lengths, adapters in (([40] * 5, [0, 1, -1, 3, 1]), ([600, 424], [2, 0])):
        lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, adapters, 264, 520, 24, 4, torch.bfloat16)
        rhs = rhs.t().contiguous().t() if turned[0] else rhs
        down = down.transpose(1, 2).contiguous().transpose(1, 2) if turned[1] else down
        up = up.transpose(1, 2).contiguous().transpose(1, 2) if turned[2] else up
        run_lora(lhs, rhs, down, up, scales, offsets, which)


@pytest.mark.parametrize("turned", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("k, n, rank", [(2056, 136, 24), (4104, 130, 20), (72, 264, 128), (264, 8, 8), (4104, 136, 128)])
def test_lora_matmul_few_rows(k, n, rank, turned):
    """Single rows under adapters, whose matrices lie either way round, in wider tensors, ragged in every size."""
    lengths, adapters = [1] * 30 + [0, 5, 3], [i % 6 - 1 for i in range(33)]
    lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, adapters, k, n, rank, 4, torch.bfloat16, first=1)

    def wider(t):  # the same values, rows eight-element aligned inside a wider tensor
        box = torch.full((*t.shape[:-1], t.shape[-1] // 8 * 8 + 24), float("nan"), dtype=t.dtype, device="cuda")
        box[..., 8:8 + t.shape[-1]] = t
        return box[..., 8:8 + t.shape[-1]]

    down = wider(down.transpose(1, 2)).transpose(1, 2) if turned[0] else wider(down)
    up = wider(up.transpose(1, 2)).transpose(1, 2) if turned[1] else wider(up)
    from ninetoothed_b200 import _capi

    before = _capi.plain_launches()
    run_lora(wider(lhs), wider(rhs), down, up, scales, offsets, which)
    assert _capi.plain_launches() == before


def test_lora_matmul_many_requests_and_wide_indices():
    lengths = [i % 3 for i in range(2048)]
    args = lora_inputs(lengths, [(i * 7) % 40 - 2 for i in range(2048)], 128, 136, 16, 36, torch.float16)
    run_lora(*args[:5], args[5].long(), args[6].long())
    # of a rank that goes a tile at a time whatever the requests, and more rows in as many requests
    args = lora_inputs(lengths, [(i * 7) % 40 - 2 for i in range(2048)], 128, 136, 136, 36, torch.bfloat16)
    run_lora(*args[:5], args[5].long(), args[6].long())
    lengths = [i % 5 for i in range(2048)]
    run_lora(*lora_inputs(lengths, [(i * 7) % 40 - 2 for i in range(2048)], 520, 136, 16, 36, torch.bfloat16))


# Grids that take every worker through five or more tiles, so that accumulators, stages and their barriers come round:
# wide tiles (long runs) and narrow ones (short runs), both layouts of the matrices.
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("lengths, k, n", [([2048, 2500, 1536, 2100], 136, 4096), ([70, 0, 128, 101] * 100, 72, 520),
                                           ([33, 64, 50] * 300, 64, 264)], ids=["wide", "middle", "narrow"])
def test_grouped_matmul_many_tiles_a_worker(lengths, k, n, transposed):
    lhs = normal(60, sum(lengths), k)
    rhs = normal(61, len(lengths), n, k).transpose(1, 2) if transposed else normal(61, len(lengths), k, n)
    run_grouped(lhs, rhs, bounds_of(lengths))


@pytest.mark.parametrize("lengths, k", [([2048, 2500, 1536, 2100], 136), ([1500] * 8, 1032)], ids=["short", "long"])
@pytest.mark.parametrize("n", [4104, 520, 264])
def test_grouped_matmul_columns_end_in_a_pairs_first_half(lengths, k, n):
    """The other half of the pair, which has no column of the last tile, keeps step with the ring of stages."""
    run_grouped(normal(64, sum(lengths), k), normal(65, len(lengths), k, n), bounds_of(lengths))


# One run with most of the rows among many short ones, which averages do not show.
@pytest.mark.parametrize("lengths", [[4000] + [40] * 60, [7] * 100 + [3000, 0] + [1] * 40], ids=["ahead", "among"])
def test_skewed_runs(lengths):
    rows, groups = sum(lengths), len(lengths)
    lhs, grad, offsets = normal(66, rows, 264), normal(67, rows, 520), bounds_of(lengths)
    run_grouped(lhs, normal(68, groups, 264, 520), offsets)
    check_rhs_grad(lhs, grad, offsets)
    for kind in KINDS:
        run_lora(*lora_inputs(lengths, [i % 9 - 1 for i in range(groups)], 264, 520, 24, 8, kind))


# (256 x 256 tiles on pairs; 128 x 128 ones take less than half a wave by their rule)
@pytest.mark.parametrize("lengths", [[64, 100, 1, 0, 129, 31, 512, 7], [128] * 8], ids=str)
def test_rhs_grad_many_tiles_a_worker(lengths):
    check_rhs_grad(normal(62, sum(lengths), 2048), normal(63, sum(lengths), 2056), bounds_of(lengths))


@pytest.mark.parametrize("turned", [(False, False, False), (True, True, True)], ids=["as they lie", "transposed"])
@pytest.mark.parametrize("lengths, k, n, rank", [([1500, 0, 300, 4000, 77, 2001], 136, 4096, 40), ([9, 31, 16, 70] * 40, 72, 2056, 16),
                                                 ([5, 100, 17, 33] * 20, 128, 72, 8)], ids=["wide", "ragged", "few columns"])
def test_lora_matmul_many_tiles_a_worker(lengths, k, n, rank, turned):
    which = [(i * 5) % 9 - 1 for i in range(len(lengths))]
    args = list(lora_inputs(lengths, which, k, n, rank, 8, KINDS[len(lengths) % 2]))
    for i, turn in zip((1, 2, 3), turned):
        if turn:
            args[i] = args[i].transpose(-1, -2).contiguous().transpose(-1, -2)
    run_lora(*args)


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_lora_matmul_many_ranks_a_tile(kind):
    """Tiles of one stage of the projection and twenty of an adapter's ranks, which most of the lanes that bring rows have no
    part in: none may be left behind."""
    lengths, which = [3000, 2500, 70, 1100], [1, 0, -1, 2]
    run_lora(*lora_inputs(lengths, which, 72, 2056, 640, 3, kind))


def test_lora_matmul_on_sizes_no_tensor_map_addresses_and_without_adapters():
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        run_lora(*lora_inputs([20, 3, 9], [1, -1, 0], 33, 70, 5, 2, torch.bfloat16, first=1))
        run_lora(*lora_inputs([20, 3, 9], [1, -1, 0], 64, 70, 12, 2, torch.float16))
    args = lora_inputs([20, 3, 9], [1, -1, 0], 64, 72, 16, 2, torch.bfloat16)
    run_lora(args[0], args[1], args[2][:0], args[3][:0], args[4][:0], *args[5:])           # no adapters at all
    run_lora(args[0], args[1], args[2][..., :0], args[3][:, :0], *args[4:])                 # adapters of rank 0
    args = lora_inputs([300, 100], [1, -1], 64, 72, 16, 2, torch.bfloat16)
    run_lora(args[0], args[1], args[2][:0], args[3][:0], args[4][:0], *args[5:])


@pytest.mark.parametrize("rows", [64, 65])
@pytest.mark.parametrize("k, n", [(64, 72), (264, 9608)])
def test_lora_matmul_an_empty_pool_of_a_large_rank(k, n, rows):
    """No adapters at all, but shapes that give them a rank beyond what the few-row kernel holds a row's values of."""
    args = lora_inputs([rows - 24, 24], [1, 0], k, n, 256, 2, torch.bfloat16, padding=0)
    run_lora(args[0], args[1], args[2][:0], args[3][:0], args[4][:0], *args[5:])


def test_a_broken_adapter_stays_with_its_requests():
    lhs, rhs, down, up, scales, offsets, which = lora_inputs([5, 20, 1, 40, 3], [0, 1, 2, 1, 0], 128, 136, 16, 3, torch.bfloat16)
    clean = run_lora(lhs, rhs, down, up, scales, offsets, which)
    from ninetoothed_b200.torch_ops import ops

    for broken in (down, up):
        kept = broken[1].clone()
        broken[1] = float("nan")
        output = torch.full_like(clean, 7.0)
        ops.lora_matmul(lhs, rhs, down, up, scales, offsets, which, output)
        sick = torch.zeros(lhs.shape[0], dtype=torch.bool, device="cuda")
        sick[5:25] = sick[26:66] = True
        assert torch.equal(output[~sick], clean[~sick])
        assert output[sick].isnan().all()
        broken[1] = kept


@pytest.mark.parametrize("rank", [24, 40])
@pytest.mark.parametrize("lengths", [[3, 5], [200, 70]], ids=str)
def test_an_infinite_row_stays_infinite(lengths, rank):
    """Positive matrices: a row that holds an infinity is infinite in every column, none of it NaN, and no other row is."""
    lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, [1, 0], 136, 264, rank, 2, torch.float16)
    lhs, rhs, down, up = lhs.abs(), rhs.abs(), down.abs(), up.abs()
    lhs[1, 17] = float("inf")
    from ninetoothed_b200.torch_ops import ops

    output = torch.zeros(lhs.shape[0], 264, dtype=torch.float16, device="cuda")
    ops.lora_matmul(lhs, rhs, down, up, scales, offsets, which, output)
    assert (output[1] == float("inf")).all()
    output[1] = 0
    assert output.isfinite().all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("whole", [False, True], ids=["any", "whole numbers"])
@pytest.mark.parametrize("lengths, k, n", [([3, 5], 1288, 264), ([3, 5], 136, 264), ([200, 300], 136, 264), ([1500, 900], 136, 2056)],
                         ids=str)
def test_infinities_in_up(lengths, k, n, whole, kind):
    """A value between the products times an infinity is an infinity of its sign (NaN for zero), also where the value is a short
    number, and no other column changes."""
    lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, [1, 0], k, n, 40, 2, kind)
    if whole:
        lhs, down = (t.float().sign().mul(t.abs() > 0.03).to(kind) for t in (lhs, down))
        scales = torch.ones_like(scales)
    from ninetoothed_b200.torch_ops import ops

    clean, output = (torch.zeros(lhs.shape[0], n, dtype=kind, device="cuda") for _ in range(2))
    ops.lora_matmul(lhs, rhs, down, up, scales, offsets, which, clean)
    for adapter, rank, column, value in ((0, 0, 7, "inf"), (0, 39, 8, "-inf"), (1, 17, n - 1, "inf"), (1, 31, 100, "-inf")):
        up[adapter, rank, column] = float(value)
    ops.lora_matmul(lhs, rhs, down, up, scales, offsets, which, output)
    for (a, b), adapter in zip(spans(offsets), which.tolist()):
        x = lhs[a:b].double()
        exact = x @ rhs.double() + scales[adapter].double() * (x @ down[adapter].double()) @ up[adapter].double()
        sick = up[adapter].isinf().any(0)
        torch.testing.assert_close(output[a:b, sick].double(), exact[:, sick], rtol=0, atol=0, equal_nan=True)
        assert torch.equal(output[a:b, ~sick], clean[a:b, ~sick])


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("power", [18, -18])
@pytest.mark.parametrize("lengths, k", [([3, 5], 1288), ([3, 5], 136), ([200, 300], 136), ([1500, 900], 136)], ids=str)
def test_the_value_between_the_products_keeps_its_range(lengths, k, power, kind):
    """scales (lhs . down) far above fp16's largest number, or among its smallest, and up the other way: exact to 2^-22 of that
    value, however many rows the call has."""
    lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, [1, 0], k, 520, 40, 2, kind)
    scales = scales * 2.0 ** power
    up = (up.float() * 2.0 ** (-power // 2)).to(kind)
    from ninetoothed_b200.torch_ops import ops

    output = torch.zeros(lhs.shape[0], 520, dtype=kind, device="cuda")
    ops.lora_matmul(lhs, torch.zeros_like(rhs), down, up, scales, offsets, which, output)
    rank, unit = 40, 2.0 ** -23
    for (a, b), adapter in zip(spans(offsets), which.tolist()):
        x, d, u, s = lhs[a:b].double(), down[adapter].double(), up[adapter].double(), scales[adapter].double()
        low, low_size = s * (x @ d), s * (x.abs() @ d.abs())
        off = low_size * ((k + 1) * unit) + low.abs() * (2.0 ** -22 + (k + rank) * unit)
        assert_within(output[a:b], low @ u, off @ u.abs())


def test_lora_matmul_workspace_of_the_caller():
    from ninetoothed_b200 import _capi

    args = lora_inputs([30, 40], [1, 0], 128, 136, 40, 2, torch.bfloat16)
    size = _capi.lora_matmul_workspace_size(args[0], args[2])
    workspace = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")  # 0xFFFF is a NaN in both types
    assert torch.equal(run_lora(*args, workspace=workspace), run_lora(*args))
    with pytest.raises(ValueError, match="workspace holds"):
        run_lora(*args, workspace=workspace[:-1])
    with pytest.raises(_capi.KernelLaunchError, match="256-byte aligned"):
        run_lora(*args, workspace=torch.empty(size + 16, dtype=torch.uint8, device="cuda")[16:])


def test_gradients_of_an_adapter_layer():
    """Towards the input: the same operator on transposed views.  Towards the adapters, whose rows are one run each:
    grouped_matmul and its weight gradient.  Against differences of the loss sum(output * cotangent), in 64 bits."""
    from ninetoothed_b200.torch_ops import ops

    lengths, k, n, rank = [70, 50, 30], 128, 192, 16
    lhs, rhs, down, up, scales, offsets, which = lora_inputs(lengths, [0, 1, 2], k, n, rank, 3, torch.float16, padding=0)
    ones = torch.ones_like(scales)
    cotangent = normal(41, 150, n, kind=torch.float16)
    lhs_grad = torch.empty_like(lhs)
    ops.lora_matmul(cotangent, rhs.t(), up.transpose(1, 2), down.transpose(1, 2), ones, offsets, which, lhs_grad)
    low, low_grad = (torch.empty(150, rank, dtype=torch.float16, device="cuda") for _ in range(2))
    down_grad, up_grad = torch.empty_like(down), torch.empty_like(up)
    ops.grouped_matmul(lhs, down, offsets, low)
    ops.grouped_matmul(cotangent, up.transpose(1, 2), offsets, low_grad)
    ops.grouped_matmul_rhs_grad(lhs, low_grad, offsets, down_grad)
    ops.grouped_matmul_rhs_grad(low, cotangent, offsets, up_grad)

    leaves = [t.double().requires_grad_() for t in (lhs, down, up)]
    where = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(lengths, device="cuda"))

    def loss(x, d, u):
        y = x @ rhs.double() + ((x[:, None] @ d[where]) @ u[where])[:, 0]
        return (y * cotangent.double()).sum()

    loss(*leaves).backward()
    step = torch.finfo(torch.float16).eps / 2
    for name, got, leaf, terms in (("lhs", lhs_grad, leaves[0], 1), ("down", down_grad, leaves[1], 2), ("up", up_grad, leaves[2], 2)):
        # one rounding for each of the chained 16-bit results, each of which enters every sum: in the 2-norm no more than
        # the same share of it (sums of independent roundings grow slower than the sums they are part of)
        off = (got.double() - leaf.grad).norm() / leaf.grad.norm()
        assert off <= terms * step, (name, off)
        g = torch.Generator(device="cuda").manual_seed(50)
        direction = torch.randn(leaf.shape, generator=g, device="cuda", dtype=torch.float64)
        moved = [[t + s * direction if t is leaf else t for t in leaves] for s in (1e-4, -1e-4)]
        difference = (loss(*moved[0]) - loss(*moved[1])) / 2e-4
        # the loss is at most bilinear in one leaf: the difference is exact to 64-bit rounding
        along = (got.double() * direction).sum()
        assert (along - difference).abs() <= terms * step * got.double().norm() * direction.norm(), name


def test_an_expert_layer_forward_and_backward():
    """Two grouped products with a ReLU between them and all gradients, captured into a graph and replayed on other
    bounds and inputs: equal, bit for bit, to the eager calls."""
    from ninetoothed_b200 import _capi
    from ninetoothed_b200.torch_ops import ops

    rows, k, hidden, groups = 500, 136, 264, 6
    w1, w2 = normal(61, groups, k, hidden, scale=k ** -0.5), normal(62, groups, hidden, k, scale=hidden ** -0.5)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        cuts = torch.randint(0, rows + 1, (groups,), generator=g).sort().values.tolist()
        return {"x": normal(seed, rows, k), "dy": normal(seed + 1, rows, k),
                "offsets": torch.tensor([0, *cuts], dtype=torch.int32, device="cuda")}

    def outputs():
        return {"a": torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda"),
                "y": torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"),
                "da": torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda"),
                "dx": torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"),
                "dw1": torch.empty_like(w1), "dw2": torch.empty_like(w2)}

    def step(i, o):
        ops.grouped_matmul(i["x"], w1, i["offsets"], o["a"])
        active = torch.relu(o["a"])
        ops.grouped_matmul(active, w2, i["offsets"], o["y"])
        ops.grouped_matmul(i["dy"], w2.transpose(1, 2), i["offsets"], o["da"])
        ops.grouped_matmul_rhs_grad(active, i["dy"], i["offsets"], o["dw2"])
        masked = o["da"] * (o["a"] > 0)
        ops.grouped_matmul(masked, w1.transpose(1, 2), i["offsets"], o["dx"])
        ops.grouped_matmul_rhs_grad(i["x"], masked, i["offsets"], o["dw1"])

    _capi.device_status()
    static_in, static_out = inputs(70), outputs()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        step(static_in, static_out)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (80, 90):
        fresh, eager = inputs(seed), outputs()
        for name, tensor in fresh.items():
            static_in[name].copy_(tensor)
        for tensor in static_out.values():
            tensor.zero_()
        graph.replay()
        step(fresh, eager)
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(static_out[name], eager[name]), name
    held = int(fresh["offsets"][-1])
    where = torch.bucketize(torch.arange(held, device="cuda"), fresh["offsets"][1:].long(), right=True)
    x, dy = fresh["x"][:held].double(), fresh["dy"][:held].double()
    hidden_exact = (x[:, None] @ w1.double()[where])[:, 0]
    y = (torch.relu(hidden_exact)[:, None] @ w2.double()[where])[:, 0]
    # one rounding of the hidden values (2^-8 at most of each) and one of the output
    assert (eager["y"][:held].double() - y).norm() <= 2 * 2.0 ** -8 * y.norm()


@pytest.mark.parametrize("lengths", [[1, 0, 3, 2], [130, 0, 260, 31], [900, 700, 45]], ids=str)
def test_calls_in_a_row_share_a_workspace(lengths):
    """A call on the output of the one before, with and without adapters in between, all through one workspace, captured and
    replayed on other bounds: what the same calls give with the device idle between them, bit for bit."""
    from ninetoothed_b200 import _capi

    x, w, down, up, scales, offsets, which = lora_inputs(lengths, [i % 3 - (i == 1) for i in range(len(lengths))], 264, 264, 40, 3,
                                                         torch.bfloat16)
    bare = torch.full_like(which, -1)
    size = _capi.lora_matmul_workspace_size(x, down)

    def chain(workspace, outputs, idle):
        at = x
        for i, output in enumerate(outputs):
            _capi.lora_matmul(at, w, down, up, scales, offsets, bare if i == 2 else which, output, workspace=workspace)
            at = output
            if idle:
                torch.cuda.synchronize()

    def outputs():
        return [torch.zeros_like(x) for _ in range(6)]

    captured, workspace = outputs(), torch.zeros(size, dtype=torch.uint8, device="cuda")
    chain(workspace, captured, idle=True)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        chain(workspace, captured, idle=False)
    torch.cuda.current_stream().wait_stream(stream)
    for shift in (0, 1, 2):
        offsets.copy_(bounds_of(lengths, first=shift))
        expected = outputs()
        chain(torch.zeros(size, dtype=torch.uint8, device="cuda"), expected, idle=True)
        workspace.fill_(255)  # (NaN, were it read before it is written)
        for output in captured:
            output.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, (got, want) in enumerate(zip(captured, expected)):
            assert torch.equal(got, want), i


def test_calls_repeat_themselves():
    """Every call of the same inputs gives the same bits, also where every worker has many ragged tiles."""
    from ninetoothed_b200.torch_ops import ops

    lengths = [(i * 37) % 150 for i in range(64)]
    rows, offsets = sum(lengths), bounds_of(lengths)
    lhs, rhs, grad = normal(101, rows, 520), normal(102, 64, 520, 1032), normal(103, rows, 1032)
    down, up = normal(104, 4, 520, 40), normal(105, 4, 40, 1032)
    scales, which = torch.ones(4, device="cuda"), torch.arange(64, device="cuda") % 5 - 1
    product, rhs_grad, beside = torch.zeros_like(grad), torch.empty_like(rhs), torch.zeros_like(grad)
    first = None
    for _ in range(30):
        for t in (product, rhs_grad, beside):
            t.fill_(float("nan"))
        ops.grouped_matmul(lhs, rhs, offsets, product)
        ops.grouped_matmul_rhs_grad(lhs, grad, offsets, rhs_grad)
        ops.lora_matmul(lhs, rhs[0], down, up, scales, offsets, which, beside)
        if first is None:
            first = [t.clone() for t in (product, rhs_grad, beside)]
        for got, want in zip((product, rhs_grad, beside), first):
            assert torch.equal(got, want)


def test_two_streams_at_once():
    """Calls in flight on two streams, the adapters' workspaces among them, give what each gives alone."""
    args = [lora_inputs([400, 300, 1], [i, 1 - i, i], 520, 1032, 40, 2, torch.bfloat16) for i in range(2)]
    from ninetoothed_b200.torch_ops import ops

    alone = [run_lora(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    outputs = [torch.full_like(o, 7.0) for o in alone]
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, a, o in zip(streams, args, outputs):
            with torch.cuda.stream(stream):
                ops.lora_matmul(*a, o)
    torch.cuda.synchronize()
    for got, expected in zip(outputs, alone):
        assert torch.equal(got, expected)


def test_different_products_on_two_streams_at_once():
    """Products of CTA pairs and of single CTAs in flight together give what each gives alone."""
    from ninetoothed_b200.torch_ops import ops

    lhs, rhs, grad = normal(81, 2000, 264), normal(82, 4, 264, 1032), normal(83, 2000, 1032)
    offsets, few = bounds_of([700, 300, 990, 5]), bounds_of([1, 0, 2, 3])
    calls = [lambda o: ops.grouped_matmul(lhs, rhs, offsets, o[0]), lambda o: ops.grouped_matmul_rhs_grad(lhs, grad, offsets, o[1]),
             lambda o: ops.grouped_matmul(lhs, rhs, few, o[2]), lambda o: ops.grouped_matmul_rhs_grad(lhs, grad, few, o[3])]

    def outputs():
        return [torch.zeros(2000, 1032, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(rhs),
                torch.zeros(2000, 1032, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(rhs)]

    alone, together = outputs(), outputs()
    for call in calls:
        call(alone)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for call in (calls[:2], calls[2:])[i]:
                    call(together)
    torch.cuda.synchronize()
    for got, expected in zip(together, alone):
        assert torch.equal(got, expected)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second device")
def test_tensors_on_another_device_than_the_current_one():
    from ninetoothed_b200.torch_ops import ops

    lhs, rhs, down, up, scales, offsets, which = lora_inputs([100, 60, 7], [1, -1, 0], 136, 264, 24, 2, torch.bfloat16)
    args = lhs, rhs, down, up, scales, offsets, which
    expected = [torch.zeros(lhs.shape[0], n, dtype=lhs.dtype, device="cuda") for n in (24, 264)]
    ops.grouped_matmul(lhs, down, offsets[:3], expected[0])
    ops.lora_matmul(*args, expected[1])
    far = [t.to("cuda:1") for t in args]
    outputs = [torch.zeros_like(t, device="cuda:1") for t in expected]
    ops.grouped_matmul(far[0], far[2], far[5][:3], outputs[0])
    ops.lora_matmul(*far, outputs[1])
    for got, want in zip(outputs, expected):
        assert torch.equal(got.cpu(), want.cpu())


def test_far_rows_pass_32_bit_offsets():
    """More than 2^31 elements in lhs and output: the last run lies behind them."""
    rows, k = 600000, 4096
    lhs = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    lhs[-300:] = normal(91, 300, k)
    rhs = normal(92, 2, k, k, scale=k ** -0.5)
    offsets = torch.tensor([rows - 300, rows - 100, rows], device="cuda")
    output = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    from ninetoothed_b200.torch_ops import ops

    ops.grouped_matmul(lhs, rhs, offsets, output)
    assert not output[:-300].any()
    check_grouped(lhs[-300:], rhs, torch.tensor([0, 200, 300]), output[-300:], torch.zeros_like(output[-300:]))
    grad = torch.empty(2, k, 64, dtype=torch.bfloat16, device="cuda")
    ops.grouped_matmul_rhs_grad(lhs, output[:, :64], offsets, grad)
    for e, (a, b) in enumerate(((-300, -100), (-100, None))):
        x, y = lhs[a:b].double(), output[a:b, :64].double()
        assert_within(grad[e], x.t() @ y, x.abs().t() @ y.abs() * (200 * 2.0 ** -23))


def test_the_operators_raise_what_the_bindings_raise():
    """Refusals come through the custom operators as the bindings' own exceptions, and nothing is written."""
    from ninetoothed_b200 import _capi
    from ninetoothed_b200.torch_ops import ops

    lhs, rhs, offsets = normal(95, 40, 64), normal(96, 2, 64, 72), bounds_of([10, 30])
    output = torch.full((40, 72), 7.0, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError, match="must have the same dtype"):
        ops.grouped_matmul(lhs, rhs.half(), offsets, output)
    with pytest.raises(ValueError, match="must have 3 dimensions"):
        ops.grouped_matmul(lhs, rhs[0], offsets, output)
    with pytest.raises(TypeError, match="int32 or torch.int64"):
        ops.grouped_matmul(lhs, rhs, offsets.short(), output)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.grouped_matmul(lhs, rhs, offsets.cpu(), output)
    with pytest.raises(_capi.KernelLaunchError, match="shapes do not agree"):
        ops.grouped_matmul(lhs, rhs, offsets, output[:, :64])
    with pytest.raises(_capi.KernelLaunchError, match="must hold 3 bounds"):
        ops.grouped_matmul_rhs_grad(lhs, output, offsets[:2], torch.empty_like(rhs))
    down, up, scales = normal(97, 3, 64, 8), normal(98, 3, 8, 72), torch.ones(3, device="cuda")
    adapters = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="scales must be torch.float32"):
        ops.lora_matmul(lhs, rhs[0], down, up, scales.half(), offsets, adapters, output)
    with pytest.raises(_capi.KernelLaunchError, match="shapes do not agree"):
        ops.lora_matmul(lhs, rhs[0], down, up[:, :, :64], scales, offsets, adapters, output)
    assert (output == 7.0).all()
