"""Norms of queries and keys with rotation on the GPU: values, gradients, layouts, refusals, against the definition in 64 bits."""
import pytest
import torch

from state_space_models_neuron_b200 import ops

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(autouse=True)
def _status():
    yield
    from state_space_models_neuron_b200.ops import cuda_ops
    torch.cuda.synchronize()
    cuda_ops.check_status()


def tables(positions, rotary):
    inverse = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inverse
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def inputs(B, L, Hq, Hk, D, wide, seed, values=False):
    """queries and keys as views of one projection (with `values`, of one that holds the values too), gradients, weights"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, L, Hq + Hk * (2 if values else 1), D, device="cuda", generator=g)
    x = (x * torch.empty(D, device="cuda").log_normal_(0, 0.5, generator=g)).bfloat16()
    dq, dk = (torch.randn(B, L, h, D, device="cuda", generator=g).bfloat16() for h in (Hq, Hk))
    w = [(1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(torch.float32 if wide else torch.bfloat16) for _ in range(2)]
    return x[:, :, :Hq], x[:, :, Hq:Hq + Hk], dq, dk, *w


def turned(x, cos, sin, at, sign=1.0):
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos[at].double()[:, :, None], sign * sin[at].double()[:, :, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def check(q, k, dq, dk, qw, kw, cos, sin, positions, grads=True):
    B, L = q.shape[:2]
    at = torch.arange(L, device="cuda").expand(B, L) if positions is None else positions.long()
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (q, k, qw, kw)]
    out = ops.qk_norm_rotary(*leaves, EPS, cos, sin, positions)
    wanted = [t for t in leaves if t is not None]
    got = dict(zip(map(id, wanted), torch.autograd.grad(out, wanted, (dq, dk)))) if grads else {}
    for x, w, dy, y, lx, lw in ((q, qw, dq, out[0], leaves[0], leaves[2]), (k, kw, dk, out[1], leaves[1], leaves[3])):
        x, dy, D = x.double(), dy.double(), x.shape[-1]
        r = 1.0 if w is None else (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n = x * r * (1.0 if w is None else w.double())
        ref = turned(n, cos, sin, at)
        # The fp32 steps: a sum of D squares (rounded at most 24 times, halved by the root), the reciprocal root (2^-22), three
        # products, rotation of a pair: below 2^-19 of the row's largest magnitudes.  Then half a step of bf16.
        far = (y.double() - ref).abs()
        assert (far <= 2 ** -8 * ref.abs() + 2 ** -18 * n.abs().amax(-1, keepdim=True)).all()
        if not grads:
            continue
        g = turned(dy, cos, sin, at, -1.0)
        if w is None:
            dx, size = g, g.abs().amax(-1, keepdim=True)
        else:
            h = g * w.double()
            dx = r * h - x * r ** 3 * (h * x).mean(-1, keepdim=True)
            size = (r * h).abs().amax(-1, keepdim=True) + (x.abs().amax(-1, keepdim=True) * r ** 3 * (h * x).abs().mean(-1, keepdim=True))
            terms = g * x * r
            # fp32 sums of at most 400 steps on the way of one term, terms with 2^-19 of their own, and the rounding of the result
            bound = 2 ** -15 * terms.abs().sum((0, 1, 2)) + (2 ** -8 if lw.dtype == torch.bfloat16 else 2 ** -24) * terms.sum((0, 1, 2)).abs()
            assert ((got[id(lw)].double() - terms.sum((0, 1, 2))).abs() <= bound).all()
        assert got[id(lx)].shape == lx.shape
        assert ((got[id(lx)].double() - dx).abs() <= 2 ** -8 * dx.abs() + 2 ** -17 * size).all()
    return out


@pytest.mark.parametrize("B,L,Hq,Hk,D", [(1, 1, 1, 1, 64), (2, 7, 5, 1, 64), (3, 33, 9, 3, 128), (1, 257, 32, 8, 128), (2, 130, 4, 2, 256),
                                         (1, 1, 16, 16, 256), (5, 1, 32, 8, 128), (1, 1025, 3, 1, 128)])
@pytest.mark.parametrize("rotary", [0, 16, 48, None])
@pytest.mark.parametrize("wide", [False, True])
def test_values_and_gradients(B, L, Hq, Hk, D, rotary, wide):
    rotary = D if rotary is None else rotary
    q, k, dq, dk, qw, kw = inputs(B, L, Hq, Hk, D, wide, B * L + Hq)
    cos, sin = tables(L + 3, rotary) if rotary else (None, None)
    check(q, k, dq, dk, qw, kw, cos, sin, None)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, True), (False, False)])
def test_positions_and_missing_norms(dtype, norms):
    q, k, dq, dk, qw, kw = inputs(2, 65, 6, 2, 128, False, 7, values=True)
    cos, sin = tables(9000, 64)
    positions = torch.randint(0, 9000, (2, 65), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    check(q, k, dq, dk, qw if norms[0] else None, kw if norms[1] else None, cos, sin, positions)
    check(q, k, dq, dk, qw if norms[0] else None, kw if norms[1] else None, cos, sin, positions.t().contiguous().t())


def test_layouts():
    """transposed, broadcast, unaligned and gradients that are broadcast"""
    q, k, dq, dk, qw, kw = inputs(2, 24, 4, 2, 64, False, 9)
    cos, sin = tables(24, 64)
    check(q.transpose(1, 2).contiguous().transpose(1, 2), k, dq, dk, qw, kw, cos, sin, None)
    check(q, k, dq.transpose(1, 2).contiguous().transpose(1, 2), dk[:, :1].expand(-1, 24, -1, -1), qw, kw, cos, sin, None)
    wide = torch.zeros(2, 24, 4, 65, device="cuda", dtype=torch.bfloat16)
    wide[..., 1:] = q
    check(wide[..., 1:], k, dq, dk, qw, kw, cos, sin, None)
    check(q, k, dq, dk, torch.cat([qw[:1], qw])[1:], kw, cos, sin, None)
    check(q[:, :1].expand(-1, 24, -1, -1), k, dq, dk, qw, kw, cos, sin, None)
    check(q, k, dq, dk, qw, kw, torch.cat([cos.flatten()[:1], cos.flatten()])[1:].view_as(cos), sin, None)


def test_the_same_weight_twice_and_parts_of_the_gradients():
    q, k, dq, dk, qw, kw = inputs(1, 40, 4, 2, 128, True, 11)
    cos, sin = tables(40, 128)
    w = qw.clone().requires_grad_()
    out = ops.qk_norm_rotary(q, k, w, w, EPS, cos, sin)
    (both,) = torch.autograd.grad(out, (w,), (dq, dk))
    parts = []
    for i, g in enumerate((dq, dk)):
        w2 = qw.clone().requires_grad_()
        parts.append(torch.autograd.grad(ops.qk_norm_rotary(q, k, w2, w2, EPS, cos, sin)[i], (w2,), (g,))[0])
    # one addition of two sums, rounded once
    assert ((both - (parts[0] + parts[1])).abs() <= 2 ** -23 * (parts[0].abs() + parts[1].abs())).all()


def test_gradients_go_to_the_optimizer_buffer():
    q, k, dq, dk, qw, kw = inputs(2, 20, 4, 2, 128, False, 13)
    ref = [t.clone().requires_grad_() for t in (qw, kw)]
    torch.autograd.backward(ops.qk_norm_rotary(q, k, ref[0].float(), ref[1].float(), EPS), (dq, dk))
    w = [t.clone().requires_grad_() for t in (qw, kw)]
    for t in w:
        t.main_grad = torch.full((128,), 3.0, device="cuda")
        t.grad_stale = True
    torch.autograd.backward(ops.qk_norm_rotary(q, k, *w, EPS), (dq, dk))
    first = [t.main_grad.clone() for t in w]
    torch.autograd.backward(ops.qk_norm_rotary(q, k, *w, EPS), (dq, dk))
    for t, f, r in zip(w, first, ref):
        assert t.grad is None and not t.grad_stale
        assert ((f - r.grad.float()).abs() <= 2 ** -8 * f.abs() + 1e-30).all()
        assert torch.equal(t.main_grad, f + f)


def test_one_weight_of_both_goes_to_the_optimizer_buffer():
    q, k, dq, dk, qw, _ = inputs(2, 700, 4, 2, 128, True, 23)
    w = qw.clone().requires_grad_()
    torch.autograd.backward(ops.qk_norm_rotary(q, k, w, w, EPS), (dq, dk))
    for stale in (True, False):
        t = qw.clone().requires_grad_()
        t.main_grad = torch.full((128,), 3.0, device="cuda")
        t.grad_stale = stale
        torch.autograd.backward(ops.qk_norm_rotary(q, k, t, t, EPS), (dq, dk))
        want = w.grad + (0.0 if stale else 3.0)
        assert t.grad is None and not t.grad_stale
        # one fp32 addition more, in another order
        assert ((t.main_grad - want).abs() <= 2 ** -22 * (want.abs() + 3.0 + w.grad.abs().max())).all()


def test_runs_give_the_same_bits():
    q, k, dq, dk, qw, kw = inputs(2, 1500, 8, 2, 128, True, 15)
    cos, sin = tables(1500, 128)
    runs = []
    for _ in range(3):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, qw, kw)]
        out = ops.qk_norm_rotary(*leaves, EPS, cos, sin)
        runs.append([*out, *torch.autograd.grad(out, leaves, (dq, dk))])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_positions_outside_the_tables_are_reported():
    from state_space_models_neuron_b200.ops import cuda_ops
    q, k, dq, dk, qw, kw = inputs(1, 12, 4, 2, 64, False, 17)
    cos, sin = tables(10, 64)
    positions = torch.arange(12, device="cuda")[None] - 1                 # -1 and 10 have no row
    leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    out = ops.qk_norm_rotary(*leaves, EPS, cos, sin, positions)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status 3"):
        cuda_ops.check_status()
    inside = check(q[:, 1:11], k[:, 1:11], dq[:, 1:11], dk[:, 1:11], qw, kw, cos, sin, positions[:, 1:11])
    for y, ref, dx in zip(out, inside, grads):
        assert not y[:, [0, 11]].any() and torch.equal(y[:, 1:11], ref) and not dx[:, [0, 11]].any()


def test_refusals():
    q, k, dq, dk, qw, kw = inputs(1, 4, 4, 2, 64, False, 19)
    cos, sin = tables(4, 24)
    for error, call in ((TypeError, lambda: ops.qk_norm_rotary(q.float(), k, qw, kw, EPS)),
                        (TypeError, lambda: ops.qk_norm_rotary(q, k.half(), qw, kw, EPS)),
                        (TypeError, lambda: ops.qk_norm_rotary(q, k, qw.half(), kw, EPS)),
                        (ValueError, lambda: ops.qk_norm_rotary(q[..., :32], k[..., :32], None, None, EPS)),
                        (ValueError, lambda: ops.qk_norm_rotary(q, k, qw, kw, EPS, cos, sin)),
                        (ValueError, lambda: ops.qk_norm_rotary(q, k, qw.cpu(), kw, EPS)),
                        (ValueError, lambda: ops.qk_norm_rotary(q, k.cpu(), qw, kw, EPS))):
        with pytest.raises(error):
            call()


def test_captured_and_replayed():
    q, k, dq, dk, qw, kw = inputs(2, 50, 4, 2, 128, False, 21)
    cos, sin = tables(50, 128)
    static = [q.clone(), k.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        ops.qk_norm_rotary(*static, qw, kw, EPS, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = ops.qk_norm_rotary(*static, qw, kw, EPS, cos, sin)
    for scale in (1.0, -2.0):
        static[0].copy_(q * scale)
        static[1].copy_(k * scale)
        graph.replay()
        with torch.no_grad():
            ref = ops.qk_norm_rotary(q * scale, k * scale, qw, kw, EPS, cos, sin)
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
