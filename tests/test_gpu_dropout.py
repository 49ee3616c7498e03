"""fastgl.dropout against the generator restated on 64-bit whole numbers: the same elements kept, the kept ones' values to the last
bit (one product in fp32, rounded once), forward and backward."""
import numpy as np
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu

TAG = 0x44524F50


def words(first, n, seed, stream):
    """Word i % 4 of the generator at counter i // 4, for i in first .. first + n - 1 (both multiples of four)."""
    low = np.uint64(0xFFFFFFFF)
    q = np.arange(first // 4, (first + n) // 4, dtype=np.uint64)
    c = [q & low, q >> np.uint64(32), np.full_like(q, stream), np.full_like(q, TAG)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)  # (below 2^64: no bits are lost)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)


def kept(n, p, seed, stream):
    return torch.from_numpy(words(0, (n + 3) // 4 * 4, seed, stream)[:n] >= round(p * 2.0 ** 32))


def expected(x, p, seed, stream, relu):
    x = x.cpu()
    keep = kept(x.numel(), p, seed, stream).view(x.shape)
    v = x.float().clamp(min=0) if relu else x.float()
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32)
    return torch.where(keep, v * scale, torch.zeros(())).to(x.dtype), keep


def test_restated_generator_is_the_oracles(cuda, oracle):
    w = words(0, 40, 0x123456789ABCDEF0, 7)
    for q in range(10):
        assert w[4 * q:4 * q + 4].tolist() == list(oracle.philox4x32_10((q, 0, 7, TAG), (0x9ABCDEF0, 0x12345678)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("rows,cols,stride", [(1, 1, 1), (1, 3, 3), (5, 7, 7), (33, 47, 50), (1000, 47, 47), (100, 64, 100), (4099, 1, 3), (17, 4096, 4099), (3, 4097, 4100),
                                              (5, 20001, 20004), (2, 4095, 5000), (1025, 16, 17)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_values_and_gradients(cuda, dtype, relu, rows, cols, stride, p):
    gen = torch.Generator(device=cuda).manual_seed(rows + cols)
    x = torch.randn((rows, stride), generator=gen, device=cuda).to(dtype)[:, :cols].requires_grad_()
    d = torch.randn((rows, cols), generator=gen, device=cuda).to(dtype)
    seed, stream = 2 ** 63 + 12345, 2 ** 32 - 2
    y = fastgl.dropout(x, p, seed=seed, stream=stream, relu=relu)
    want, keep = expected(x.detach(), p, seed, stream, relu)
    assert y.is_contiguous() and torch.equal(y.detach().cpu(), want)
    g, = torch.autograd.grad(y, x, d)
    mask = keep & (x.detach().cpu() > 0) if relu else keep
    scale = torch.tensor(1.0 / (1.0 - p), dtype=torch.float32)
    assert torch.equal(g.cpu(), torch.where(mask, d.cpu().float() * scale, torch.zeros(())).to(dtype))
    assert torch.equal(fastgl.dropout(x.detach(), p, seed=seed, stream=stream, relu=relu), y)  # nobody records


@pytest.mark.parametrize("p", [0.0, 1e-9, 0.999, 1.0])
@pytest.mark.parametrize("relu", [False, True])
def test_ends_of_the_range_and_odd_values(cuda, p, relu):
    x = torch.randn(997, device=cuda)
    x[::5] = float("nan")
    x[1::5] = float("inf")
    x[2::10] = -float("inf")
    x = x.requires_grad_()
    y = fastgl.dropout(x, p, seed=1, relu=relu)
    want, keep = expected(x.detach(), p, 1, 0, relu)
    assert torch.equal(torch.nan_to_num(y.detach().cpu(), 1e30), torch.nan_to_num(want, 1e30)) and torch.equal(y.isnan().cpu(), want.isnan())
    assert (y.detach().cpu()[~keep] == 0).all()
    g, = torch.autograd.grad(y, x, torch.full_like(x, float("inf")))
    assert torch.equal(g.cpu() != 0, keep & ~(x.detach().cpu() <= 0) if relu else keep)


def test_any_shape_empty_ones_and_gradients_from_views(cuda):
    x = torch.randn((3, 5, 7), device=cuda, requires_grad=True)
    y = fastgl.dropout(x, 0.4, seed=5)
    assert y.shape == x.shape and torch.equal(y.detach().cpu(), expected(x.detach(), 0.4, 5, 0, False)[0])
    g, = torch.autograd.grad(y.sum(), x)  # (an expanded gradient)
    assert torch.equal(g.cpu(), expected(torch.ones((3, 5, 7)), 0.4, 5, 0, False)[0])
    m = torch.randn((6, 8), device=cuda, requires_grad=True)
    g, = torch.autograd.grad(fastgl.dropout(m, 0.4, seed=5, relu=True).t(), m, torch.ones((8, 6), device=cuda))
    assert ((g != 0) <= (m > 0)).all()
    for shape in ((0,), (0, 5), (5, 0)):
        assert fastgl.dropout(torch.zeros(shape, device=cuda)).shape == shape
    with pytest.raises(RuntimeError, match="contiguous"):
        fastgl.dropout(torch.zeros((4, 6), device=cuda).t())
    with pytest.raises(RuntimeError, match="contiguous"):
        fastgl.dropout(torch.zeros((1, 6), device=cuda).expand(4, 6))
    with pytest.raises(RuntimeError, match="dtype"):
        fastgl.dropout(torch.zeros(4, device=cuda, dtype=torch.float16))
    for bad in (dict(p=1.5), dict(p=float("nan")), dict(seed=-1), dict(stream=1 << 32), dict(stream_offset=torch.zeros(1, dtype=torch.int32)),
                dict(stream_offset=torch.zeros(2, dtype=torch.int32, device=cuda)), dict(stream_offset=torch.zeros(1, device=cuda))):
        with pytest.raises(RuntimeError):
            fastgl.dropout(torch.zeros(4, device=cuda), **bad)


@pytest.mark.parametrize("relu", [False, True])
def test_gradients_of_gradients(cuda, relu):
    x = torch.randn((40, 6), device=cuda, requires_grad=True)
    d = torch.randn((40, 6), device=cuda, requires_grad=True)
    y = fastgl.dropout(x, 0.3, seed=8, relu=relu)
    g, = torch.autograd.grad(y, x, d, create_graph=True)
    first, = torch.autograd.grad(fastgl.dropout(x, 0.3, seed=8, relu=relu), x, d.detach())
    assert torch.allclose(g.detach(), first, rtol=2.0 ** -23)
    gg, = torch.autograd.grad((g * g).sum(), d)
    share = torch.where(first != 0, 1 / 0.7, 0.0)
    assert torch.allclose(gg, 2 * first * share, rtol=1e-6)


def test_offsets_beyond_32_bits(cuda):
    n = 2 ** 32 + 4096 + 5
    x = torch.ones(n, device=cuda, dtype=torch.bfloat16)
    y = fastgl.dropout(x, 0.5, seed=77, stream=3)
    for first, count in ((2 ** 31 - 64, 128), (2 ** 32 - 64, 128), (2 ** 32 + 4096, 8)):
        want = np.where(words(first, count, 77, 3) >= 2 ** 31, 2.0, 0.0)[:min(count, n - first)]
        assert np.array_equal(y[first:first + count].float().cpu().numpy(), want)
    del x, y
    base = torch.ones((70, 2 ** 26), device=cuda, dtype=torch.bfloat16)  # rows that start beyond 2^32
    y = fastgl.dropout(base[:, :1001], 0.5, seed=77, stream=3)
    assert torch.equal(y.cpu(), expected(torch.ones((70, 1001), dtype=torch.bfloat16), 0.5, 77, 3, False)[0])


def test_share_of_kept_elements(cuda):
    # n draws of a chance q: the count is off by more than six standard deviations once in 5e8
    n = 1 << 22
    for p in (0.03, 0.5, 0.9):
        k = int((fastgl.dropout(torch.ones(n, device=cuda), p, seed=9) != 0).sum())
        assert abs(k - n * (1 - p)) < 6 * (n * p * (1 - p)) ** 0.5


def test_captured_calls_draw_new_masks(cuda):
    offset = torch.zeros(1, dtype=torch.int32, device=cuda)
    base = torch.randn((300, 40), device=cuda)
    d = torch.randn((300, 40), device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fastgl.dropout(base, 0.5, seed=4, stream=10, stream_offset=offset)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = base.detach().requires_grad_()
        y = fastgl.dropout(x, 0.5, seed=4, stream=10, relu=False, stream_offset=offset)
        g, = torch.autograd.grad(y, x, d)
    for k in range(4):
        offset.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), fastgl.dropout(base, 0.5, seed=4, stream=10 + k)) and torch.equal(g, fastgl.dropout(d, 0.5, seed=4, stream=10 + k))
    # an offset that changed between the passes is an error, not another mask
    x = base.detach().requires_grad_()
    y = fastgl.dropout(x, 0.5, stream_offset=offset)
    offset.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_on_another_stream(cuda):
    x = torch.randn((2000, 100), device=cuda)
    want = fastgl.dropout(x, 0.5, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fastgl.dropout(x, 0.5, seed=2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_layer(cuda):
    x = torch.randn((50, 30), device=cuda)
    layer = fastgl.Dropout(0.5, seed=6)
    a, b = layer(x), layer(x)
    assert layer.calls == 2 and torch.equal(a, fastgl.dropout(x, 0.5, 6, 0)) and torch.equal(b, fastgl.dropout(x, 0.5, 6, 1)) and not torch.equal(a, b)
    layer.calls = 0
    assert torch.equal(layer(x), a)
    assert layer.eval()(x) is x
    relu = fastgl.Dropout(0.5, seed=6, relu=True).eval()
    assert torch.equal(relu(x), x.clamp(min=0))
