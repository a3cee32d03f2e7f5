"""Layer norm, 8-bit blocks and the block product together, as the VAEs' hidden layers call them."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

from medicalimageanalysis_amd import blocks8, norm  # noqa: E402
from medicalimageanalysis_amd.graph import GraphedTrainStep  # noqa: E402
from medicalimageanalysis_amd.model.hyperspherical_vae import HypersphericalVAE  # noqa: E402
from medicalimageanalysis_amd.model.spherical_vae import SphericalVAE  # noqa: E402
from medicalimageanalysis_amd.model.torus_vae import ToroidalVAE  # noqa: E402
from test_gpu_blocks8 import by_blocks, softplus  # noqa: E402

DEV = torch.device("cuda:0")
CONFIG = dict(extrinsic_dim=200, latent_dim=3, sftbeta=2.0, encoder_width=160, encoder_depth=2, decoder_width=130,
              decoder_depth=2, dropout_p=0.1, device="cuda", gamma=1.0, beta=0.01, longest_radius=2.0,
              shortest_radius=1.0, hidden="blocks8", layer_norm=True)


class _Quantised(torch.autograd.Function):
    """values rounded to 8-bit blocks, the gradient passed on as it is"""

    @staticmethod
    def forward(ctx, a, tall):
        return by_blocks(a, tall)

    @staticmethod
    def backward(ctx, g):
        return g, None


class _QuantisedGradient(torch.autograd.Function):
    """y = a w^T with the input's gradient from the 8-bit blocks of y's, the weight's from y's as it is"""

    @staticmethod
    def forward(ctx, a, w):
        ctx.save_for_backward(a, w)
        return a @ w.t()

    @staticmethod
    def backward(ctx, g):
        a, w = ctx.saved_tensors
        return by_blocks(g) @ w, g.t() @ a


class _SoftplusFromBlocks(torch.autograd.Function):
    """blocks of softplus(h); the slope is that at the kept value"""

    @staticmethod
    def forward(ctx, h, beta):
        a = by_blocks(softplus(h, beta))
        ctx.save_for_backward(a)
        ctx.beta = beta
        return a

    @staticmethod
    def backward(ctx, g):
        return g * -torch.expm1(-ctx.beta * ctx.saved_tensors[0]), None


def decode64(model, z):
    """the decoder in 64 bits, with the roundings to 8 bits where the layers have them"""
    def layer(l, h):
        a = _SoftplusFromBlocks.apply(h, model.sftbeta)
        return _QuantisedGradient.apply(a, _Quantised.apply(l.weight, 128)) + l.bias

    def normed(i, h):
        n = model.decoder_norms[i]
        d = h - h.mean(-1, keepdim=True)
        return d / torch.sqrt((d * d).mean(-1, keepdim=True) + n.eps) * n.weight + n.bias

    h = normed(0, model.decoder_function(z))
    for i, l in enumerate(model.decoder_linear_layers):
        h = normed(i + 1, layer(l, h))
    return layer(model.function_x_mu, h)


def test_decoder_and_its_gradients_against_64_bits():
    """Off by 32-bit roundings, except where one of those changes which 8-bit value is nearest: such an element moves by
    up to 2^-3 of itself.  Of n = 64 x 130 elements of a layer one or two may (a 32-bit difference of 1e-6 against steps
    of 1/16: 1.6e-5 n = 0.13 expected per layer), each a change of 2^-3 / sqrt(n) = 1.4e-3 of the norm: 5e-3 for a few."""
    torch.manual_seed(1)
    model = HypersphericalVAE(CONFIG)
    with torch.no_grad():
        for n in model.decoder_norms:
            n.weight.uniform_(0.5, 1.5)
            n.bias.normal_()
    wide = copy.deepcopy(model).double()
    z = torch.nn.functional.normalize(torch.randn(64, 3, device=DEV), dim=-1)
    gy = torch.randn(64, 200, device=DEV)
    z32, z64 = z.clone().requires_grad_(), z.double().requires_grad_()
    y, y64 = model.decode(z32), decode64(wide, z64)
    assert (y.double() - y64).norm() <= 5e-3 * y64.norm()
    y.backward(gy)
    y64.backward(gy.double())
    pairs = [("z", z32.grad, z64.grad)] + [(k, p.grad, q.grad) for (k, p), (_, q) in
                                           zip(model.named_parameters(), wide.named_parameters()) if q.grad is not None]
    assert len(pairs) == 1 + 2 * 4 + 2 * 3
    for name, got, want in pairs:
        assert (got.double() - want).norm() <= 5e-3 * want.norm(), name


@pytest.mark.parametrize("model", [HypersphericalVAE, SphericalVAE, ToroidalVAE])
@pytest.mark.parametrize("change", [{}, {"layer_norm": False}, {"hidden": None}])
def test_models_run_and_every_parameter_has_a_gradient(model, change):
    torch.manual_seed(2)
    m = model(dict(CONFIG, **change))
    x = torch.rand(24, 200, device=DEV)
    z, x_hat, params = m(x)
    loss = sum(m._elbo(x, x_hat, params[i:i + 2]) for i in range(0, len(params), 2))  # (the torus has two angles)
    loss.backward()
    assert torch.isfinite(loss) and torch.isfinite(x_hat).all()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    assert torch.isfinite(m.encode(x)[0]).all()


def _loss(model, z, target):
    return ((model.decode(z) - target) ** 2).mean()


def test_captured_train_step_equals_the_eager_one():
    """Two models take the same steps, one eagerly and one as a replayed graph, with eager work between the replays."""
    torch.manual_seed(3)
    eager = HypersphericalVAE(CONFIG)
    captured = copy.deepcopy(eager)
    start = copy.deepcopy(eager.state_dict())
    z = torch.randn(96, 3, device=DEV)
    target = torch.rand(96, 200, device=DEV)

    def adam(m):
        return torch.optim.Adam([p for k, p in m.named_parameters() if "decoder" in k or "x_mu" in k], lr=1e-3,
                                capturable=True, fused=True)

    opt = adam(captured)
    step = GraphedTrainStep(captured, opt, _loss, [z, target])
    with torch.no_grad():  # back to the start: the warm-up steps moved it
        for k, v in captured.state_dict().items():
            v.copy_(start[k])
    for state in opt.state.values():
        for v in state.values():
            v.zero_()
    reference = adam(eager)
    for i in range(4):
        zi, ti = z + 0.1 * i, target * (1 + i)
        got = float(step(zi, ti))
        torch.cuda.synchronize()
        reference.zero_grad(set_to_none=True)
        want = _loss(eager, zi, ti)
        want.backward()
        reference.step()
        blocks8.quantize(torch.randn(50, 50, device=DEV))  # eager work of the same kernels between two replays
        assert got == pytest.approx(float(want.detach()), rel=1e-6), i
    for (k, p), (_, q) in zip(eager.named_parameters(), captured.named_parameters()):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6), k


def test_two_captured_graphs_on_two_streams_do_not_share_scratch():
    """products that are split over their block columns and weight gradients split over the batch use scratch memory"""
    def work(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(600, 4096, device=DEV, generator=g)
        w = torch.randn(40, 4096, device=DEV, generator=g)
        gy = torch.randn(600, 40, device=DEV, generator=g)
        lw, lb = torch.ones(4096, device=DEV), torch.zeros(4096, device=DEV)

        def run():
            h = norm.layer_norm(x, lw, lb)
            q = blocks8.quantize(h, "softplus")
            return (blocks8.matmul(q, blocks8.quantize_weight(w).rows),) + blocks8.weight_grad(gy, q)
        return run

    runs = [work(1), work(2)]
    want = [[t.clone() for t in r()] for r in runs]
    graphs, results = [], []
    for r in runs:
        s = torch.cuda.Stream(DEV)
        s.wait_stream(torch.cuda.current_stream(DEV))
        with torch.cuda.stream(s):
            r()
        torch.cuda.current_stream(DEV).wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(r())
        graphs.append(g)
    streams = [torch.cuda.Stream(DEV) for _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, w in zip(results, want):
            for p, q in zip(got, w):
                assert torch.equal(p, q)


def test_captured_gradients_with_a_frozen_weight_and_a_bias_of_another_type():
    """x's and the bias's gradients (column sums split over the rows) replayed on a stream of their own, beside eager calls"""
    g = torch.Generator(device=DEV).manual_seed(5)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    x, gy, w8 = r(3000, 300).bfloat16(), r(3000, 200).bfloat16(), blocks8.quantize_weight(r(200, 300))
    w = r(200, 300).bfloat16()

    def once():
        xs, b = x.detach().requires_grad_(), torch.zeros(200, device=DEV, requires_grad=True)
        ws = w.detach().requires_grad_()
        first = torch.autograd.grad(blocks8.linear(xs, w8, b, "softplus"), (xs, b), gy)
        return first + torch.autograd.grad(blocks8.linear(xs, ws, b, "softplus"), (ws, b), gy)

    want = [t.clone() for t in once()]
    s = torch.cuda.Stream(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream(DEV).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    keep = x.clone()
    for i in range(4):
        x.copy_(keep * (1 + i % 2))
        with torch.cuda.stream(s):
            s.wait_stream(torch.cuda.default_stream(DEV))
            graph.replay()
        eager = once()
        torch.cuda.synchronize()
        for p, q, first in zip(got, eager, want):
            assert torch.equal(p, q) and (i % 2 == 1 or torch.equal(p, first))
