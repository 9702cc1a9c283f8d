"""``rotary.rotate`` on the GPU against its plain form in 64 bits, its gradients and captured calls."""

import pickle

import numpy as np
import pytest
import torch

from reelcache_amd import restore_kernels as rk
from reelcache_amd import rotary
from reelcache_amd.errors import StateError

import operator_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _normal(shape, dtype, device, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def _place(x, layout, angles):
    """angles [B, T, pairs] broadcast against ``x`` in its layout."""
    return angles.unsqueeze(-2) if layout == "BTHD" else (angles[0].unsqueeze(-2) if layout == "THD" else angles.unsqueeze(1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", rotary.PAIRINGS)
@pytest.mark.parametrize("shape", [
    # batch, grid, heads, kv heads, head_dim, rotated channels, layout
    (2, (2, 3, 5), 5, 2, 64, 64, "BTHD"), (1, (1, 1, 1), 32, 8, 128, 128, "BTHD"), (3, (1, 7, 3), 4, 4, 80, 40, "BHTD"),
    (1, (2, 9, 13), 3, 1, 128, 96, "THD"), (2, (1, 5, 5), 2, 2, 22, 14, "BTHD"), (1, (3, 4, 4), 9, 9, 96, 96, "BHTD"),
])
@pytest.mark.parametrize("tokens", [False, True])
def test_rotation_matches_its_plain_form(device, dtype, pairing, shape, tokens):
    batch, grid, heads, kv_heads, dim, rotated, layout = shape
    n = int(np.prod(grid))
    cos, sin, sections = oracle.tables(40, rotated // 2)
    table = rk.RopeTable(cos, sin, sections)

    def make(h, seed):
        size = {"BTHD": (batch, n, h, dim), "BHTD": (batch, h, n, dim), "THD": (n, h, dim)}[layout]
        return _normal(size, dtype, device, seed)

    q, k = make(heads, 1), make(kv_heads, 2)
    if tokens:
        rows = torch.randint(0, 40, (batch, n, 3), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
        positions, grid = rotary.TokenRows(table, rows.to(device)), None
    else:
        rows = oracle.grid_rows((5, 1, 2), grid)[None].expand(batch, -1, -1)
        positions = rk.RopePositions(table, (5, 1, 2))
    angles = oracle.token_angles(cos, sin, sections, rows)
    out = rotary.rotate((q, k), positions, grid=grid, layout=layout, pairing=pairing)
    back = rotary.rotate((q, k), positions, grid=grid, layout=layout, pairing=pairing, inverse=True)
    for x, y, z in zip((q, k), out, back):
        c, s = (_place(x, layout, a) for a in angles)
        assert y.shape == x.shape and y.dtype == x.dtype
        assert oracle.worst(y, *oracle.rotate(x, c, s, pairing)) <= 0
        assert oracle.worst(z, *oracle.rotate(x, c, -s, pairing)) <= 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_heads_and_tokens(device, dtype):
    """A call large enough for four heads to a thread, with a head count that four does not divide."""
    cos, sin, sections = oracle.tables(64, 64)
    table = rk.RopeTable(cos, sin, sections)
    grid, heads = (2, 25, 47), 23
    q = _normal((2350, heads, 128), dtype, device, 5)
    out = rotary.rotate(q, rk.RopePositions(table, (7, 0, 3)), grid=grid, layout="THD")
    c, s = oracle.token_angles(cos, sin, sections, oracle.grid_rows((7, 0, 3), grid))
    assert oracle.worst(out, *oracle.rotate(q, c[:, None], s[:, None])) <= 0


def test_dense_tables_strides_and_outputs(device):
    cos, sin, _ = oracle.tables(50, 32)
    table = rk.RopeTable(cos, sin)
    x = _normal((2, 3, 20, 2, 64), torch.bfloat16, device, 1)[:, 1, ::2].transpose(1, 2)  # [2, 2, 10, 64] BHTD, strided
    c, s = cos[4:14], sin[4:14]
    expected = oracle.rotate(x, c, s)
    assert oracle.worst(rotary.rotate(x, rk.RopePositions(table, 4), layout="BHTD"), *expected) <= 0
    rows = torch.arange(4, 14, dtype=torch.int32, device=device)
    assert oracle.worst(rotary.rotate(x, rotary.TokenRows(table, rows), layout="BHTD"), *expected) <= 0
    per = torch.stack([rows, rows.flip(0)])[:, :, None].expand(2, 10, 4)[..., 2]
    turned = rotary.rotate(x, rotary.TokenRows(table, per), layout="BHTD")
    assert oracle.worst(turned[0], *(v[0] for v in expected)) <= 0
    assert oracle.worst(turned[1], *oracle.rotate(x[1], c.flip(0), s.flip(0))) <= 0
    # Unaligned rows (offset by one element), channels that are not next to each other, and a broadcast input.
    odd = torch.empty(2 * 2 * 10 * 64 + 1, dtype=torch.bfloat16, device=device)[1:].view(2, 2, 10, 64).copy_(x)
    assert oracle.worst(rotary.rotate(odd, rk.RopePositions(table, 4), layout="BHTD"), *expected) <= 0
    spread = torch.zeros((2, 2, 10, 64, 2), dtype=torch.bfloat16, device=device)[..., 1].copy_(x)
    assert oracle.worst(rotary.rotate(spread, rk.RopePositions(table, 4), layout="BHTD"), *expected) <= 0
    shared = x[:1].expand(2, -1, -1, -1)
    assert torch.equal(rotary.rotate(shared, rk.RopePositions(table, 4), layout="BHTD")[1],
                       rotary.rotate(x[:1], rk.RopePositions(table, 4), layout="BHTD")[0])
    # In place, into a strided output, and into an output with spread channels.
    result = rotary.rotate(x, rk.RopePositions(table, 4), layout="BHTD")
    target = torch.zeros((2, 10, 3, 64), dtype=torch.bfloat16, device=device)
    assert rotary.rotate(x, rk.RopePositions(table, 4), layout="BHTD", out=target[:, :, :2].transpose(1, 2)) is not None
    assert torch.equal(target[:, :, :2].transpose(1, 2), result) and not target[:, :, 2].any()
    rotary.rotate(x, rk.RopePositions(table, 4), layout="BHTD", out=spread)
    assert torch.equal(spread, result)
    y = x.clone()
    assert rotary.rotate(y, rk.RopePositions(table, 4), layout="BHTD", out=y) is y
    assert torch.equal(y, result)


def test_rows_outside_the_table_turn_to_nan(device):
    cos, sin, sections = oracle.tables(10, 32)
    table = rk.RopeTable(cos, sin, sections, (10, 8, 10))
    rows = torch.tensor([[0, 0, 0], [-1, 0, 0], [0, 8, 0], [0, 0, 1 << 30], [9, 7, 9]], dtype=torch.int32, device=device)
    x = _normal((1, 5, 2, 80), torch.float32, device, 1)
    out = rotary.rotate(x, rotary.TokenRows(table, rows))[0].cpu()
    axis = torch.tensor([0] * sections[0] + [1] * sections[1] + [2] * sections[2]).repeat_interleave(2)
    for token, bad in ((0, None), (1, 0), (2, 1), (3, 2), (4, None)):
        expected = (axis == bad) if bad is not None else torch.zeros(64, dtype=torch.bool)
        assert torch.equal(out[token, 0, :64].isnan(), expected)
        assert torch.equal(out[token, :, 64:], x[0, token, :, 64:].cpu())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", rotary.PAIRINGS)
def test_gradients(device, dtype, pairing):
    """Gradients of queries, keys shared by several uses and a broadcast input, against the transpose."""
    cos, sin, sections = oracle.tables(16, 24)
    table = rk.RopeTable(cos, sin, sections)
    rows = torch.randint(0, 16, (2, 7, 3), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    positions = rotary.TokenRows(table, rows.to(device))
    q, k = (_normal((2, 7, h, 56), dtype, device, h).requires_grad_(True) for h in (4, 2))
    dq, dk = (_normal((2, 7, h, 56), dtype, device, 10 + h) for h in (4, 2))
    out = rotary.rotate((q, k), positions, pairing=pairing)
    grads = torch.autograd.grad(out, (q, k), (dq, dk), retain_graph=True)
    c, s = (a.unsqueeze(-2) for a in oracle.token_angles(cos, sin, sections, rows))
    for g, d in zip(grads, (dq, dk)):
        assert oracle.worst(g, *oracle.rotate(d, c, -s, pairing)) <= 0
    only, = torch.autograd.grad(out[1], (k,), dk)  # the queries' output is unused
    assert torch.equal(only, grads[1])
    leaf = _normal((1, 7, 1, 56), dtype, device, 9).requires_grad_(True)
    total = rotary.rotate(leaf.expand(2, 7, 3, 56), positions, pairing=pairing)
    upstream = _normal((2, 7, 3, 56), dtype, device, 11)
    shared, = torch.autograd.grad(total, (leaf,), upstream)
    each, bound = oracle.rotate(upstream, c, -s, pairing)
    # Six gradients are summed in the type, one rounding of at most the sum of their sizes each.
    sums = bound.sum(dim=(0, 2)) + 6 * oracle.U[dtype] * each.abs().sum(dim=(0, 2))
    assert oracle.worst(shared[0, :, 0], each.sum(dim=(0, 2)), sums) <= 0
    scalar, = torch.autograd.grad(rotary.rotate(q, positions, pairing=pairing).sum(), (q,))  # an expanded gradient
    assert oracle.worst(scalar, *oracle.rotate(torch.ones_like(dq), c, -s, pairing)) <= 0


def test_gradient_against_differences(device):
    cos, sin, sections = oracle.tables(16, 16)
    table = rk.RopeTable(cos, sin, sections)
    positions = rk.RopePositions(table, (3, 1, 2))
    x = _normal((1, 12, 2, 40), torch.float32, device, 1).requires_grad_(True)
    d = _normal((1, 12, 2, 40), torch.float32, device, 2)
    grad, = torch.autograd.grad(rotary.rotate(x, positions, grid=(2, 3, 2)), (x,), d)
    start = x.detach()
    for seed in range(4):
        step = _normal(x.shape, torch.float32, device, 20 + seed)
        with torch.no_grad():
            ends = [rotary.rotate(start + sign * step, positions, grid=(2, 3, 2)).double() for sign in (1, -1)]
        slope = float(((ends[0] - ends[1]) / 2 * d.double()).sum())
        terms = (d.double().abs() * (start.double().abs() + step.double().abs())).sum()
        # x + step, two products, a sum and the table round once each at both ends: 2 * 8 half steps of the
        # terms (each coordinate feeds two outputs); the gradient as many.
        assert abs(float((grad.double() * step.double()).sum()) - slope) <= float(terms) * 64 * oracle.F32
    twice, = torch.autograd.grad(rotary.rotate(x, positions, grid=(2, 3, 2)), (x,), d.clone().requires_grad_(True),
                                 create_graph=True)
    assert twice.requires_grad  # linear: the gradient is differentiable in the upstream gradient


def test_captured_forward_and_backward(device):
    cos, sin, sections = oracle.tables(16, 32)
    table = rk.RopeTable(cos, sin, sections)
    rows = torch.zeros((2, 9, 3), dtype=torch.int32, device=device)
    positions = rotary.TokenRows(table, rows)
    q = _normal((2, 9, 4, 64), torch.bfloat16, device, 1)
    d = _normal((2, 9, 4, 64), torch.bfloat16, device, 2)
    leaf = q.clone().requires_grad_(True)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):  # the table's upload and the first run, outside the capture
        torch.autograd.grad(rotary.rotate(leaf, positions), (leaf,), d)
    torch.cuda.synchronize(device)
    rk.reserve_capture_staging(1 << 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = rotary.rotate(leaf, positions)
        grad, = torch.autograd.grad(out, (leaf,), d)
    for replay in range(3):
        with torch.no_grad():
            leaf.copy_(_normal(q.shape, torch.bfloat16, device, 30 + replay))
        rows.copy_(torch.randint(0, 16, rows.shape, generator=torch.Generator().manual_seed(replay), dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(device)
        with torch.no_grad():
            assert torch.equal(out, rotary.rotate(leaf.detach(), positions))
            assert torch.equal(grad, rotary.rotate(d, positions, inverse=True))


def test_other_stream(device):
    cos, sin, sections = oracle.tables(16, 32)
    x = _normal((1, 9, 4, 64), torch.bfloat16, device, 1)
    expected = rotary.rotate(x, rk.RopePositions(rk.RopeTable(cos, sin, sections), (1, 2, 3)), grid=(1, 3, 3))
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        out = rotary.rotate(x, rk.RopePositions(rk.RopeTable(cos, sin, sections), (1, 2, 3)), grid=(1, 3, 3))
    stream.synchronize()
    assert torch.equal(out, expected)


def test_outputs_that_autograd_saved(device):
    """A result written into a tensor that a backward pass needs is noticed by that pass."""
    cos, sin, sections = oracle.tables(16, 8)
    at = rk.RopePositions(rk.RopeTable(cos.to(device), sin.to(device), sections), 0)
    x, saved = torch.randn(1, 6, 1, 16, device=device), torch.randn(1, 6, 1, 16, device=device)
    weight = torch.randn(1, 6, 1, 16, device=device, requires_grad=True)
    product = (weight * saved).sum()
    with torch.no_grad():
        rotary.rotate(x, at, grid=(1, 2, 3), out=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():
        rotary.rotate(x, at, grid=(1, 2, 3), out=torch.empty_like(x))


def test_rotation_has_the_restores_bits(device):
    """Dense rows restored with RoPE and the same rows rotated: the same bits."""
    cos, sin, sections = oracle.tables(32, 64)
    table = rk.RopeTable(cos, sin, sections)
    grid, positions = (2, 5, 7), rk.RopePositions(table, (3, 1, 0))
    x = _normal((70, 3, 128), torch.bfloat16, device, 1)
    cache = torch.zeros((1, 70, 3, 128), dtype=torch.bfloat16, device=device)
    job = rk.ReconstructionJob(rk.DenseSource(x.reshape(70, 384)), rk.NativeView(cache), grid, rope=positions)
    rk.reconstruct([job]).release()
    assert torch.equal(cache[0], rotary.rotate(x, positions, grid=grid, layout="THD"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", rotary.PAIRINGS)
def test_rows_that_overlap(device, dtype, pairing):
    """Windows of one step over a line of values, forward and as a gradient."""
    cos, sin, sections = oracle.tables(40, 32)
    table = rk.RopeTable(cos, sin, sections)
    line = _normal((200,), dtype, device, 1)
    x = line.as_strided((9, 2, 64), (1, 70, 1))
    c, s = (a[:, None] for a in oracle.token_angles(cos, sin, sections, oracle.grid_rows((2, 0, 1), (1, 3, 3))))
    positions = rk.RopePositions(table, (2, 0, 1))
    for _ in range(2):
        out = rotary.rotate(x, positions, grid=(1, 3, 3), layout="THD", pairing=pairing)
        assert oracle.worst(out, *oracle.rotate(x, c, s, pairing)) <= 0
    leaf = _normal((9, 2, 64), dtype, device, 2).requires_grad_(True)
    grad, = torch.autograd.grad(rotary.rotate(leaf, positions, grid=(1, 3, 3), layout="THD", pairing=pairing), (leaf,), x)
    assert oracle.worst(grad, *oracle.rotate(x, c, -s, pairing)) <= 0


def test_inference_tables_dropped_before_the_backward_pass_are_refused(device):
    """Tables of inference tensors count no updates: their owner drops the copies, and a gradient by others is refused."""
    cos, sin, sections = oracle.tables(16, 8)
    with torch.inference_mode():
        table = rk.RopeTable(cos.clone(), sin.clone(), sections)
    at = rk.RopePositions(table, 0)
    x = _normal((1, 6, 1, 16), torch.float32, device, 1).requires_grad_(True)
    rotary.rotate(x, at, grid=(1, 2, 3)).sum().backward()
    out = rotary.rotate(x, at, grid=(1, 2, 3))
    with torch.inference_mode():
        table.cos.mul_(0.5)
    table.invalidate()
    with pytest.raises(StateError, match="table was changed"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", rotary.PAIRINGS)
def test_rows_that_start_at_any_element(device, dtype, pairing):
    """Inputs and outputs one element off, and head sizes of 4n + 2 channels."""
    for dim, rotated in ((64, 64), (66, 64), (70, 62)):
        cos, sin, _ = oracle.tables(50, rotated // 2)
        positions = rk.RopePositions(rk.RopeTable(cos, sin), 4)
        size = 2 * 10 * 3 * dim
        x = torch.empty(size + 1, dtype=dtype, device=device)[1:].view(2, 10, 3, dim).copy_(_normal((2, 10, 3, dim), dtype, device, 7))
        expected = oracle.rotate(x, cos[4:14, None], sin[4:14, None], pairing)
        assert oracle.worst(rotary.rotate(x, positions, pairing=pairing), *expected) <= 0
        out = torch.empty(size + 3, dtype=dtype, device=device)[3:].view(2, 10, 3, dim)
        rotary.rotate(x, positions, pairing=pairing, out=out)
        assert oracle.worst(out, *expected) <= 0


def test_positions_are_pickled_after_use(device):
    cos, sin, sections = oracle.tables(16, 8)
    positions = rk.RopePositions(rk.RopeTable(cos, sin, sections), (1, 0, 2))
    x = _normal((1, 6, 1, 16), torch.float32, device, 1)
    expected = rotary.rotate(x, positions, grid=(1, 2, 3))
    torch.cuda.synchronize(device)
    positions.table.invalidate()  # device copies and their events stay here
    again = pickle.loads(pickle.dumps(positions))
    assert torch.equal(rotary.rotate(x, again, grid=(1, 2, 3)), expected)


def test_captured_calls_keep_the_tables_angles(device):
    """A table updated, dropped and made again after a capture: replays turn by the angles of the capture."""
    cos, sin, sections = oracle.tables(16, 32)
    table = rk.RopeTable(cos.to(device), sin.to(device), sections)
    positions = rk.RopePositions(table, (3, 1, 2))
    x = _normal((1, 6, 2, 64), torch.bfloat16, device, 1)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        expected = rotary.rotate(x, positions, grid=(1, 2, 3))
    torch.cuda.synchronize(device)
    rk.reserve_capture_staging(1 << 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = rotary.rotate(x, positions, grid=(1, 2, 3))
    for replay in range(3):
        table.cos.mul_(0.5)
        assert not torch.equal(rotary.rotate(x, positions, grid=(1, 2, 3)), expected)
        if replay == 1:
            table.invalidate()
        torch.cuda.synchronize(device)
        junk = [torch.full((size,), 7.0, device=device) for size in (16 * 32 * 4, 1 << 10, 1 << 14) for _ in range(20)]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize(device)
        assert torch.equal(out, expected)
        del junk
