"""The operators of a decoder block together: a block against its definition, captured in a graph and replayed; the example."""
import os
import sys

import pytest
import torch

import mx_ref as ref

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _block(mlxq, x, res, w, active):
    """Norm of a sum to 8 bits, a router's product, routing, the experts and their sum, and the gradients of a training step."""
    n, h = mlxq.rms_norm(x, w["norm"], residual=res, mx=True)
    z = mlxq.mx_matmul(n, w["router"], out_dtype=F32)
    r = mlxq.route_experts(z, 2, "sigmoid", bias=w["bias"], groups=2, active=active)
    each = mlxq.mx_experts(n, w["up"], r, out_dtype=BF16)
    y = mlxq.mx_experts(mlxq.mx_quantize(each, "e2m1"), w["down"], r, combine=True)
    dz = mlxq.route_experts_backward(r.weights, z, r.ids, "sigmoid")
    dx, dw = mlxq.rms_norm_backward(y, h, w["norm"], dsum=res)
    return n.codes, n.scales, h, z, *r, each, y, dz, dx, dw


def _operands(mlxq, seed, T, K=96, F=64, E=8):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    w = {"norm": (1 + 0.1 * rnd(K)).to(BF16).cuda(), "router": mlxq.mx_quantize(rnd(E, K).cuda()), "bias": (0.1 * rnd(E)).cuda(),
         "up": mlxq.mx_quantize((rnd(E, F, K) / 8).cuda()), "down": mlxq.mx_quantize((rnd(E, K, F) / 8).cuda())}
    return rnd(T, K).to(BF16).cuda(), rnd(T, K).to(BF16).cuda(), w, (torch.rand(T, generator=g) > 0.2).cuda()


@pytest.mark.parametrize("T", [1, 19, 150])
def test_block(mlxq, T):
    """Each stage against its definition, on what the stage before it gave."""
    x, res, w, active = _operands(mlxq, T, T)
    codes, scales, h, z, ids, weights, starts, rows, each, y, dz, dx, dw = _block(mlxq, x, res, w, active)
    hc = (x.float() + res.float()).to(BF16).cpu()
    assert torch.equal(h.cpu(), hc)
    code, scale = ref.quantized(ref.rms_norm(hc, w["norm"].cpu(), float(torch.tensor(1e-6))), "e4m3")
    assert torch.equal(ref.unpacked(codes), code) and torch.equal(scales.cpu().long(), scale)
    nv, rv = ref.values((codes, scales)), ref.values(w["router"])
    assert ((z.cpu().double() - nv @ rv.t()).abs() <= ref.product_bound(nv, rv, F32, "e4m3")).all()
    want_ids, want_w = ref.route(z.cpu(), 2, "sigmoid", bias=w["bias"].cpu(), groups=2, active=active.cpu())
    assert torch.equal(ids.cpu(), want_ids) and ((weights.cpu().double() - want_w).abs() <= 2.0 ** -23 * want_w).all()
    want_starts, want_rows = ref.plan(want_ids, 8)
    assert torch.equal(starts.cpu(), want_starts) and torch.equal(rows.cpu(), want_rows)
    want, _, uv = ref.experts((codes, scales), w["up"], want_ids, None)
    for t in range(T):
        for j in range(2):
            e = int(want_ids[t, j])
            tol = ref.product_bound(nv[t:t + 1], uv[e], BF16, "e4m3")[0] if e >= 0 else 0.0
            assert ((each[t, j].cpu().double() - want[t, j]).abs() <= tol).all()
    q = mlxq.mx_quantize(each, "e2m1")
    want, xv, dv = ref.experts((q.codes.cpu(), q.scales.cpu()), w["down"], want_ids, None)
    exact = (want * weights.cpu().double()[..., None]).sum(1)
    tol = torch.zeros_like(want)
    for t in range(T):
        for j in range(2):
            if int(want_ids[t, j]) >= 0:
                tol[t, j] = ref.product_bound(xv[t, j:j + 1], dv[want_ids[t, j]], BF16, "e2m1")[0]
    mag = ((want.abs() + tol) * weights.cpu().double()[..., None]).sum(1)
    assert ((y.cpu().double() - exact).abs() <= (tol * weights.cpu().double()[..., None]).sum(1) + (3 * 2.0 ** -23 + 2.0 ** -8) * mag).all()
    want_z, mag = ref.route_gradient(weights.cpu(), z.cpu(), ids.cpu(), "sigmoid", True, 1.0)
    assert ((dz.cpu().double() - want_z).abs() <= 65 * 2.0 ** -24 * mag + 2.0 ** -149).all()
    want_x, want_dw, mag, mag_w = ref.rms_norm_gradient(y.cpu(), hc, w["norm"].cpu(), res.cpu(), 1e-6)
    assert ((dx.cpu().double() - want_x).abs() <= 300 * 2.0 ** -24 * mag * (1 + 2.0 ** -8) + 2.0 ** -8 * want_x.abs()).all()
    assert ((dw.cpu().double() - want_dw).abs() <= (192 + T) * 2.0 ** -24 * mag_w * (1 + 2.0 ** -8) + 2.0 ** -8 * want_dw.abs()).all()


@pytest.mark.parametrize("T", [3, 1300])
def test_block_in_a_graph(mlxq, T):
    """Captured once, replayed with other inputs between eager calls and synchronizations: every replay is the eager result."""
    x, res, w, active = _operands(mlxq, 1, T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(mlxq, x, res, w, active)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _block(mlxq, x, res, w, active)
        for turn in range(4):
            a, b, _, act = _operands(mlxq, 10 + turn, T)
            x.copy_(a)
            res.copy_(b)
            active.copy_(act)
            eager = [t.clone() for t in _block(mlxq, a, b, w, act)]
            for t in out:
                (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).zero_()
            graph.replay()
            torch.cuda.synchronize()
            for i, (p, q) in enumerate(zip(out, eager)):
                assert torch.equal(p.view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p,
                                   q.view(torch.uint8) if q.dtype == torch.float8_e4m3fn else q), i


def test_two_graphs_and_eager_calls_share_nothing(mlxq):
    """Two captured blocks on two streams at once, with eager calls on a third."""
    cases = [_operands(mlxq, 20 + i, 900) for i in range(2)]
    graphs, outs, eager = [], [], []
    streams = [torch.cuda.Stream() for _ in cases]
    for s, c in zip(streams, cases):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            eager.append([t.clone() for t in _block(mlxq, c[0], c[1], c[2], c[3])])
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(_block(mlxq, c[0], c[1], c[2], c[3]))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        _block(mlxq, *cases[0])
    torch.cuda.synchronize()
    for out, want in zip(outs, eager):
        assert all(torch.equal(p.view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p,
                               q.view(torch.uint8) if q.dtype == torch.float8_e4m3fn else q) for p, q in zip(out, want))


def test_example_serves(mlxq):
    import mx_decode
    assert mx_decode.serve(layers=2, hidden=256, experts=4, steps=5, prompts=(19, 1, 3), say=lambda _: None)


def test_example_gradients(mlxq):
    """The loss's gradients against autograd's in 64 bits through the same choice and the same (held) experts' outputs.  f32: the
    norm's and the router's roundings, the product with the router (256 terms) and a mean over 64 x 32 errors, all against the
    gradient's largest element: sums of up to 64 * 256 terms that mostly cancel; 2^-24 * 2^9 of it."""
    import mx_decode
    g = torch.Generator("cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    experts = mlxq.mx_quantize(rnd(6, 32, 256) / 16)
    x, target, norm, router = rnd(64, 256), rnd(64, 32), 1 + 0.1 * rnd(256), rnd(6, 256) / 16
    norm.requires_grad_(True), router.requires_grad_(True)
    mx_decode.moe_loss(x, norm, router, experts, 2, target).backward()
    with torch.no_grad():
        n = mlxq.rms_norm(x, norm)
        r = mlxq.route_experts(n @ router.t(), 2)
        y = mlxq.mx_experts(mlxq.mx_quantize(n, "e4m3"), experts, r, out_dtype=F32).double()
    norm64, router64 = norm.detach().double().requires_grad_(True), router.detach().double().requires_grad_(True)
    n64 = x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt() * norm64
    s = torch.softmax(n64 @ router64.t(), -1).gather(1, r.ids.long())
    (((s / s.sum(-1, keepdim=True))[..., None] * y).sum(1) - target.double()).square().mean().backward()
    for got, want in ((norm.grad, norm64.grad), (router.grad, router64.grad)):
        assert (got.double() - want).abs().max() <= 2.0 ** -15 * want.abs().max()


def test_example_trains(mlxq):
    import mx_decode
    losses = mx_decode.train(tokens=64, steps=3, say=lambda _: None)
    assert len(losses) == 3 and all(v == v and v < float("inf") for v in losses)
