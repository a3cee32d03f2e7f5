"""Layer norm against the formula in 64 bits.  Tolerances: the result's own rounding (half a step of its type) plus
32-bit arithmetic; the sums' errors are counted against the sum of the terms' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

from medicalimageanalysis_amd import norm  # noqa: E402

DEV = torch.device("cuda:0")
U32 = 2.0 ** -24


def formula(x, w, b, gy, eps):
    """y, gx, gw, gb in float64 with the sizes their errors are counted against"""
    x, gy = x.double(), gy.double()
    w = torch.ones(x.shape[-1], device=x.device, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    var = (d * d).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = d * rstd
    h = gy * w
    m1, m2 = h.mean(-1, keepdim=True), (h * xh).mean(-1, keepdim=True)
    gx = rstd * (h - m1 - xh * m2)
    rows = tuple(range(x.dim() - 1))
    total = lambda t: t.sum(rows) if rows else t  # noqa: E731  (a sum over no dimensions would be over all)
    # a 32-bit mean is off by a few units of the mean magnitude; x - mean, rstd and what follows inherit it
    off = x.abs().mean(-1, keepdim=True) * rstd + 1 + xh.abs()
    size_y = off * w.abs() + b.abs()
    size_gx = rstd * (h.abs() + h.abs().mean(-1, keepdim=True) + (xh.abs() + off) * (h * xh).abs().mean(-1, keepdim=True)
                      + xh.abs() * (h.abs() * off).mean(-1, keepdim=True))
    return ((xh * w + b, size_y), (gx, size_gx),
            (total(gy * xh), total(gy.abs() * (xh.abs() + off))), (total(gy), total(gy.abs())))


def near(got, want, size, n_sum):
    """half a step of the type for the rounding, 32-bit sums of n_sum terms: blocked sums grow with their depth, which
    stays under 64 + n_sum / 512 here"""
    unit = 0.0 if got.dtype == torch.float64 else torch.finfo(got.dtype).eps / 2
    u = 2.0 ** -53 if got.dtype == torch.float64 else U32
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps  # half a step among the subnormals of fp16
    bound = unit * want.abs() + (64 + n_sum / 512) * u * size + tiny
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / bound).max()))


def check(x, w, b, gy, eps=1e-5):
    x = x.detach().requires_grad_()
    w = None if w is None else w.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    y = norm.layer_norm(x, w, b, eps)
    leaves = {k: t for k, t in (("x", x), ("w", w), ("b", b)) if t is not None}
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(norm.layer_norm(x, w, b, eps), y)
        (wy, sy), (wx, sx), (ww, sw), (wb, sb) = formula(x, w, b, gy, eps)
        n = x.numel() // x.shape[-1]
        near(y, wy, sy, x.shape[-1])
        near(grads["x"], wx, sx, x.shape[-1])
        if w is not None:
            assert grads["w"].dtype == w.dtype
            near(grads["w"], ww, sw, n)
        if b is not None:
            near(grads["b"], wb, sb, n)


def data(n, width, dtype, wdtype=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    wdtype = wdtype or dtype
    return ((r(n, width) * torch.exp(r(width)) + r(n, 1)).to(dtype), (1 + 0.3 * r(width)).to(wdtype),
            r(width).to(wdtype), r(n, width).to(dtype))


TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 7, 64, 128, 129, 255, 400, 784, 1001, 1024, 2047, 4096, 4100, 8191, 16384, 40001])
def test_widths(width, dtype):
    n = 37 if width < 9000 else 5
    check(*data(n, width, dtype, seed=width))


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 513, 1025, 20000])
@pytest.mark.parametrize("width,dtype", [(96, torch.float32), (300, torch.bfloat16), (5000, torch.float16)])
def test_row_counts(n, width, dtype):
    check(*data(n, width, dtype, seed=n))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp32_weights_with_16_bit_rows(dtype):
    check(*data(65, 513, dtype, torch.float32))


def test_absent_weight_and_bias():
    x, w, b, gy = data(33, 200, torch.float32)
    check(x, None, None, gy)
    check(x, w, None, gy)
    check(x, None, b, gy)


def test_strides_views_and_leading_dimensions():
    x, w, b, gy = data(48, 100, torch.bfloat16)
    wide = torch.full((48, 131), 7.0, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:103] = x
    check(wide[:, 3:103], w, b, gy)                       # rows with a stride, at an odd address
    check(x.t().contiguous().t(), w, b, gy)               # the last dimension is not dense
    check(x.view(4, 12, 100), w, b, gy.view(4, 12, 100))
    check(x.view(4, 12, 100).transpose(0, 1), w, b, gy.view(12, 4, 100))
    check(x[:1].expand(48, 100), w, b, gy)                # one row, 48 times
    check(x, w, b, gy[:1].expand(48, 100))                # a gradient that does not differ by row
    check(x[0], w, b, gy[0])
    assert (wide[:, :3] == 7).all() and (wide[:, 103:] == 7).all()


@pytest.mark.parametrize("width", [12, 9000, 40000])
def test_no_rows(width):
    x = torch.empty(0, width, device=DEV, requires_grad=True)
    w, b = torch.ones(width, device=DEV, requires_grad=True), torch.zeros(width, device=DEV, requires_grad=True)
    y = norm.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty(0, width, device=DEV))
    assert y.shape == gx.shape == (0, width) and not gw.any() and not gb.any()


@pytest.mark.parametrize("n,width", [(5, 40), (2000, 300), (700, 5000), (6, 40000)])
def test_each_gradient_alone(n, width):
    x, w, b, gy = data(n, width, torch.float32, seed=n)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    full = torch.autograd.grad(norm.layer_norm(*leaves), leaves, gy)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(norm.layer_norm(*some), some[i], gy)
        assert torch.equal(got, full[i])


def test_differentiable_once():
    x, w, b, gy = data(4, 30, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    plain = torch.autograd.grad(norm.layer_norm(*leaves), leaves, gy)
    graph = torch.autograd.grad(norm.layer_norm(*leaves), leaves, gy, create_graph=True)
    for p, q in zip(plain, graph):
        assert torch.equal(p, q)
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        torch.autograd.grad(graph[0].sum(), leaves)


def test_constant_rows_and_large_means():
    """variance 0: y is the bias; a mean of 1000 times the spread keeps the digits that x has"""
    x, w, b, gy = data(9, 260, torch.float32)
    x[3] = 5.0
    check(x + 1000, w, b, gy)


def test_non_finite_rows_stay_theirs():
    x, w, b, gy = data(6, 130, torch.float32)
    want = norm.layer_norm(x, w, b)
    x[1, 5], x[3, 0] = float("nan"), float("inf")
    got = norm.layer_norm(x, w, b)
    keep = [0, 2, 4, 5]
    assert torch.equal(got[keep], want[keep]) and got[1].isnan().all() and got[3].isnan().all()


def test_same_bits_on_every_run_and_on_another_stream():
    x, w, b, gy = data(3000, 257, torch.bfloat16)

    def once():
        l = [t.detach().requires_grad_() for t in (x, w, b)]
        return torch.autograd.grad(norm.layer_norm(*l), l, gy)

    first = once()
    s = torch.cuda.Stream(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream(DEV).wait_stream(s)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_gradient_against_differences():
    x, w, b, gy = (t[:4] if t.dim() == 2 else t for t in data(4, 11, torch.float64))
    args = [t.detach().requires_grad_() for t in (x, w, b)]
    assert torch.autograd.gradcheck(lambda *a: norm.layer_norm(*a), args)


def test_offsets_beyond_32_bits():
    """rows whose elements lie beyond 2^31 elements and 2^32 bytes of the base"""
    width = 1024
    n = (1 << 21) + 3  # 2^31 elements and three rows
    x = torch.zeros(n, width, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(4)
    tail = torch.randn(8, width, device=DEV, generator=g).to(torch.bfloat16)
    x[-8:] = tail
    y = norm.layer_norm(x)
    assert torch.equal(y[-8:], norm.layer_norm(tail)) and not y[:4].any()


@pytest.mark.parametrize("n,width", [(40, 128), (2000, 300), (6, 40000)])
def test_saved_tensors_moved_to_the_host_and_back(n, width):
    """save_on_cpu returns the rows of a wider tensor as a dense one, with another row stride"""
    x, w, b, gy = data(n, width, torch.float32, seed=n)
    wide = torch.full((n, 2 * width), 3.0, device=DEV)
    wide[:, :width] = x
    leaves = [t.detach().requires_grad_() for t in (wide[:, :width], w, b)]
    want = torch.autograd.grad(norm.layer_norm(*leaves), leaves, gy)
    with torch.autograd.graph.save_on_cpu():
        y = norm.layer_norm(*leaves)
    for p, q in zip(torch.autograd.grad(y, leaves, gy), want):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,width", [(1, 40001), (16, 300000), (40, 33000), (300, 40000)])
def test_long_rows_and_their_parts(n, width, dtype):
    check(*data(n, width, dtype, seed=n))
