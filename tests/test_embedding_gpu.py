"""features.embedding on the GPU.  A looked-up row is a rounding of scale T[id]; a
gradient row is a rounding of the fp32 sum of its n rows, which is off by at most
(n + 4) 2^-24 times the sum of their magnitudes."""

import pytest
import torch

from dsl_splat_b200 import _native, features
from test_features_gpu import DTYPES, check, draws

pytestmark = pytest.mark.gpu


def reference(ids, entries, dy, scale):
    flat, rows = ids.reshape(-1).long(), dy.reshape(-1, dy.shape[-1]).double()
    sums = torch.zeros(entries, dy.shape[-1], dtype=torch.float64, device=dy.device)
    sizes = torch.zeros_like(sums)
    sums.index_add_(0, flat, rows)
    sizes.index_add_(0, flat, rows.abs())
    number = torch.bincount(flat, minlength=entries)[:, None]
    return scale * sums, abs(scale) * sizes * (number + 4) * 2.0 ** -24


def run(ids, table, scale, seed=0):
    leaf = table.detach().requires_grad_()
    y = features.embedding(ids, leaf, scale=scale)
    want = table.float()[ids.long()] * torch.tensor(scale, dtype=torch.float32, device="cuda")
    assert torch.equal(y.detach(), want.to(table.dtype))
    dy = draws(seed + 100)(*y.shape, dtype=table.dtype)
    grad, = torch.autograd.grad(y, leaf, dy)
    check(grad, *reference(ids, len(table), dy, scale), "dtable")
    assert torch.equal(torch.autograd.grad(features.embedding(ids, leaf, scale=scale), leaf, dy)[0],
                       grad)
    return grad


def ids_of(count, entries, seed, dtype=torch.int64, power=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(count, generator=g).double() ** power * entries).to(dtype).cuda()


SIZES = [(1, 1, 1), (1, 5, 3), (8, 300, 32), (40, 7, 17), (2048, 64, 8), (2049, 64, 8),
         (5000, 3, 35), (5000, 9000, 16), (3000, 8192, 24), (3000, 8193, 24), (70000, 1000, 64),
         (20000, 200000, 5), (10000, 2, 300), (9000, 40, 1000), (100003, 513, 1),
         (60000, 70000, 2), (33000, 100, 513)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count, entries, channels", SIZES)
def test_sizes(count, entries, channels, dtype):
    table = draws(1)(entries, channels, dtype=dtype)
    run(ids_of(count, entries, 2), table, 0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_skewed_and_single_entries(dtype, ids_dtype):
    table = draws(3)(700, 40, dtype=dtype)
    run(ids_of(50000, 700, 4, ids_dtype, power=8.0), table, 1.0)
    for entry in (0, 699):  # every row the same entry
        grad = run(torch.full((40001,), entry, dtype=ids_dtype, device="cuda"), table, 1.0)
        others = torch.ones(700, dtype=torch.bool)
        others[entry] = False
        assert not grad[others].any()
    run(torch.arange(700, device="cuda").to(ids_dtype).repeat_interleave(61), table, 2.0)


def test_more_than_a_pass_of_bits():
    table = draws(5)((1 << 26) + 5, 1, dtype=torch.bfloat16)
    ids = ids_of(30000, len(table), 6)
    ids[::3] = len(table) - 1
    run(ids, table, 1.0)


def test_a_million_rows():
    table = draws(7)(8192, 64, dtype=torch.bfloat16)
    run(ids_of(1000000, 8192, 8, power=2.0), table, 0.125)


def test_rows_in_order():
    """Whole numbers: sums to the bit, wherever runs cross groups and blocks."""
    g = torch.Generator().manual_seed(9)
    for count, entries, channels in ((200000, 3, 8), (200000, 190, 33), (100000, 50000, 4)):
        ids = torch.randint(0, entries, (count,), generator=g).cuda()
        dy = torch.randint(-8, 9, (count, channels), generator=g).float().cuda()
        table = torch.zeros(entries, channels, device="cuda", requires_grad=True)
        grad, = torch.autograd.grad(features.embedding(ids, table), table, dy)
        want = torch.zeros(entries, channels, dtype=torch.float64, device="cuda")
        want.index_add_(0, ids, dy.double())
        assert torch.equal(grad.double(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [5, 33, 1000, 1024, 1025])
@pytest.mark.parametrize("entries", [1, 2, 300])
def test_few_rows(entries, count, dtype):
    """Up to those that each entry looks for itself: of like and of unlike ids, whole and
    partial pieces of 32 channels."""
    for channels in (3, 32, 70, 512):
        table = draws(20)(entries, channels, dtype=dtype)
        run(ids_of(count, entries, 21), table, 0.5)
        run(torch.full((count,), entries - 1, device="cuda"), table, 1.0)


def test_few_rows_in_order():
    """Sums of whole numbers, whose order has to be the rows' where they are not exact."""
    dy = torch.ones(1024, 40, device="cuda")
    dy[0], dy[-1] = 2.0 ** 24, -(2.0 ** 24)  # a one is lost on the way wherever it comes
    table = torch.zeros(2, 40, device="cuda", requires_grad=True)
    ids = torch.ones(1024, dtype=torch.int64, device="cuda")
    grad, = torch.autograd.grad(features.embedding(ids, table), table, dy)
    assert not grad.any()


def test_shapes_and_strides():
    table = draws(10)(50, 24, dtype=torch.float16)
    ids = ids_of(120, 50, 11).reshape(5, 4, 6)
    for part in (ids, ids[:, 1:3], ids.transpose(0, 2), ids[2, 1, 3]):
        run(part, table, 1.0)
        run(part, table[:, 3:20], 0.5)
    wide = draws(12)(120, 48, dtype=torch.float16).reshape(5, 4, 6, 48)[..., ::2]
    leaf = table.requires_grad_()
    grad, = torch.autograd.grad(features.embedding(ids, leaf), leaf, wide)
    check(grad, *reference(ids, 50, wide.contiguous(), 1.0), "dtable")
    # broadcast upstream
    grad, = torch.autograd.grad(features.embedding(ids, leaf).float().sum(), leaf)
    check(grad, *reference(ids, 50, torch.ones_like(wide), 1.0), "dtable")


def test_no_rows():
    table = torch.ones(4, 3, device="cuda", requires_grad=True)
    y = features.embedding(torch.empty(0, 2, dtype=torch.int64, device="cuda"), table)
    assert y.shape == (0, 2, 3)
    grad, = torch.autograd.grad(y, table, torch.empty_like(y))
    assert grad.shape == (4, 3) and not grad.any()


@pytest.mark.parametrize("count", [10, 50000])
def test_ids_outside_the_table(count):
    """They give zeros and no gradient, and are reported."""
    device = torch.device("cuda", torch.cuda.current_device())
    table = draws(13)(100, 16, dtype=torch.float32)
    ids = ids_of(count, 100, 14)
    bad = ids.clone()
    bad[1::4] = torch.tensor([-1, 100, 1 << 40, -(1 << 40)], device="cuda").repeat(
        count)[:len(bad[1::4])]
    assert _native.device_error(device) == 0
    leaf = table.requires_grad_()
    y = features.embedding(bad, leaf)
    assert _native.device_error(device) == -6 and _native.device_error(device) == 0
    keep = torch.ones(count, dtype=torch.bool, device="cuda")
    keep[1::4] = False
    assert not y[~keep].any() and torch.equal(y[keep], table[ids[keep]])
    dy = draws(15)(count, 16, dtype=torch.float32)
    grad, = torch.autograd.grad(y, leaf, dy)
    check(grad, *reference(ids[keep], 100, dy[keep], 1.0), "dtable")
    grad, = torch.autograd.grad(features.embedding(torch.full_like(ids, -1), leaf), leaf, dy)
    assert not grad.any() and _native.device_error(device) == -6


def test_captured_on_another_stream():
    table = draws(16)(300, 32, dtype=torch.float32)
    ids, dy = ids_of(9000, 300, 17), draws(18)(9000, 32, dtype=torch.float32)
    want = run(ids, table, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = table.detach().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = features.embedding(ids, leaf)
            grad, = torch.autograd.grad(y, leaf, dy)
        graph.replay()
        torch.cuda.synchronize()
        other = ids.flip(0).contiguous()
        first = grad.clone()
        ids.copy_(other)
        graph.replay()
    torch.cuda.synchronize()
    check(first, *reference(other.flip(0), 300, dy, 1.0), "dtable")
    check(grad, *reference(other, 300, dy, 1.0), "dtable")
    assert want.shape == grad.shape


@pytest.mark.parametrize("count", [700, 9000])
def test_replays_give_what_calls_give(count):
    """A captured step replayed with other ids and upstreams gives those of calls, to the bit."""
    table = draws(22)(300, 32, dtype=torch.float32)
    side = torch.cuda.Stream()

    def call(ids, dy):
        leaf = table.detach().requires_grad_()
        y = features.embedding(ids, leaf, scale=0.5)
        return y.detach().clone(), torch.autograd.grad(y, leaf, dy)[0]

    inputs = [(ids_of(count, 300, 23 + i, power=1.0 + i), draws(26 + i)(count, 32,
                                                                       dtype=torch.float32))
              for i in range(3)]
    want = [call(*pair) for pair in inputs]
    ids, dy = (torch.zeros_like(t) for t in inputs[0])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            leaf = table.detach().requires_grad_()
            y = features.embedding(ids, leaf, scale=0.5)
            grad, = torch.autograd.grad(y, leaf, dy)
        for (new_ids, new_dy), (value, gradient) in zip(inputs, want):
            ids.copy_(new_ids)
            dy.copy_(new_dy)
            graph.replay()
            assert torch.equal(y.detach(), value) and torch.equal(grad, gradient)
