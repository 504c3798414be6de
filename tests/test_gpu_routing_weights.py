"""The routing weights of chosen experts and their gradient, against the formula in 64 bits."""
import pytest
import torch

import moe_rd

pytestmark = pytest.mark.gpu

CASES = [
    # T, E, K, score_fn, bias_mode, renorm, scale, norm_min
    (1, 256, 8, "softmax", "none", True, 1.0, 1e-20),
    (1, 1, 1, "softmax", "none", True, 1.0, 1e-20),
    (67, 256, 8, "sigmoid", "select_and_weight", True, 2.5, 1e-20),
    (300, 60, 6, "softmax", "select_and_weight", True, 1.0, 1e-20),
    (300, 160, 4, "sigmoid", "select", True, 2.5, 1e-20),
    (129, 33, 33 - 1, "softmax", "logit", False, 0.5, 1e-20),
    (129, 64, 2, "sigmoid", "logit", False, 1.0, 1e-20),
    (500, 128, 8, "softmax", "none", True, 1.0, 0.3),      # sums on both sides of norm_min
    (500, 128, 8, "sigmoid", "none", True, 1.0, 6.0),
    (5000, 128, 8, "softmax", "none", True, 1.0, 1e-20),
]


def inputs(T, E, K, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + T + E)
    logits = (torch.randn(T, E, generator=g) * spread).clamp(-10, 10)
    ids = torch.topk(logits + torch.randn(T, E, generator=g), K, dim=1).indices.to(torch.int32)
    return logits, ids, torch.rand(E, generator=g) * 0.2, torch.randn(T, K, generator=g)


class Sigmoid64(torch.autograd.Function):
    """torch.sigmoid whose slope is s(z) s(-z): from z = 37 on, 1 - s(z) is zero in 64 bits while the slope is not."""
    @staticmethod
    def forward(ctx, z):
        ctx.save_for_backward(z)
        return torch.sigmoid(z)

    @staticmethod
    def backward(ctx, grad):
        z, = ctx.saved_tensors
        return grad * torch.sigmoid(z) * torch.sigmoid(-z)


def weights64(logits, ids, bias, score_fn, bias_mode, renorm, scale, norm_min):
    z = logits if bias_mode != "logit" else logits + bias.double()
    s = torch.softmax(z, 1) if score_fn == "softmax" else Sigmoid64.apply(z)
    if bias_mode == "select_and_weight":
        s = s + bias.double()
    valid = (ids >= 0) & (ids < logits.shape[1])
    u = s.gather(1, ids.long().clamp(0, logits.shape[1] - 1)) * valid
    return scale * u / u.sum(1, keepdim=True).clamp(min=norm_min) if renorm else scale * u


def bounds(logits, ids, bias, grad, score_fn, bias_mode, renorm, scale, norm_min):
    """What 32 bits allow, in units of 2^-24.  An exponential's argument is off by up to 20 units (|z - max| <= 20, rounded),
    expf by 4, so a score by 24, its sum by 24 + 35 (at most 32 + 3 additions) and the quotient by 85 in all; u, S (6 more)
    and u / S then by 85 + 91 + 2 < 180 relative.  A gradient element is a sum of products of at most
    s_k, h_k with h_k = (c g_k - c G / S) / S: s_k 85, G 85 + 85 + 8, S twice 91, each operation 1: < 560 of the sum of
    the magnitudes of its terms, which no element of the row exceeds by more than what the row's terms sum up to."""
    z = logits.double() if bias_mode != "logit" else logits.double() + bias.double()
    s = torch.softmax(z, 1) if score_fn == "softmax" else torch.sigmoid(z)
    u = s + bias.double() if bias_mode == "select_and_weight" else s
    pick = ids.long().clamp(0, logits.shape[1] - 1)
    valid = (ids >= 0) & (ids < logits.shape[1])
    sk, uk = s.gather(1, pick) * valid, u.gather(1, pick) * valid
    S = uk.sum(1, keepdim=True)
    g = (scale * grad.double()).abs() * valid
    if renorm:
        m = S.clamp(min=norm_min)
        h = (g + (g * uk).sum(1, keepdim=True) / m) / m
    else:
        h = g
    return 180 * 2.0 ** -24, 560 * 2.0 ** -24 * 2 * (sk * h).sum(1, keepdim=True)


@pytest.mark.parametrize("T,E,K,score_fn,bias_mode,renorm,scale,norm_min", CASES)
def test_weights_and_gradient(T, E, K, score_fn, bias_mode, renorm, scale, norm_min):
    logits, ids, bias, grad = inputs(T, E, K)
    if T > 100:
        ids[::7, 0] = -1
        ids[::11, -1] = E
        ids[5] = -1
        ids[13] = ids[13, :1]  # one expert in every slot
    kw = dict(score_fn=score_fn, bias_mode=bias_mode, renorm=renorm, routed_scale=scale, norm_min=norm_min)
    z = logits.double().requires_grad_()
    want = weights64(z, ids, bias, score_fn, bias_mode, renorm, scale, norm_min)
    want_g = torch.autograd.grad(want, z, grad.double())[0]
    rel, abs_g = bounds(logits, ids, bias, grad, score_fn, bias_mode, renorm, scale, norm_min)
    if renorm:  # a sum that rounding may put on either side of norm_min has no defined gradient
        u = want.detach().sum(1) / scale
        clear = torch.ones(T, dtype=torch.bool) if norm_min < 0.1 else (u - 1).abs() < 1e-9
        clear |= u < 1 - 1e-4
        assert clear.float().mean() > 0.9
    else:
        clear = torch.ones(T, dtype=torch.bool)
    lc, ic, bc = logits.cuda(), ids.cuda(), bias.cuda()
    got = moe_rd.routing_weights(lc, ic, bc, **kw)
    assert ((got.cpu().double() - want.detach()).abs() <= rel * want.detach().abs()).all()
    leaf = lc.clone().requires_grad_()
    out = moe_rd.routing_weights(leaf, ic, bc, **kw)
    assert torch.equal(out.detach(), got)
    out.backward(grad.cuda())
    plain = moe_rd.routing_weights_backward(grad.cuda(), lc, ic, bc, **kw)
    assert torch.equal(plain, leaf.grad)
    err = (plain.cpu().double() - want_g).abs()
    assert (err[clear] <= (abs_g + 1e-37)[clear]).all()
    if T > 100:
        assert (plain[5] == 0).all()
    # against a difference along a random direction: (f(z + hd) - f(z - hd)) / 2h is off by h^2 |f'''| / 6
    if norm_min < 0.1:
        d = torch.randn(T, E, generator=torch.Generator().manual_seed(4)).double()
        h = 1e-5
        f = lambda zz: (weights64(zz, ids, bias, score_fn, bias_mode, renorm, scale, norm_min) * grad.double()).sum()  # noqa: E731
        diff = (f(logits.double() + h * d) - f(logits.double() - h * d)) / (2 * h)
        along = (plain.cpu().double() * d).sum()
        slack = (abs_g * d.abs().sum(1, keepdim=True)).sum() + 1e-8 * d.abs().sum()
        assert (along - diff).abs() <= slack


def test_masked_and_extreme_logits():
    inf = float("inf")
    logits = torch.randn(6, 40)
    logits[0, 3:] = -inf          # masked experts that were not chosen
    logits[1] = torch.finfo(torch.float32).min
    logits[2] = -inf              # a token without anything: no valid id
    logits[3] = float("nan")      # likewise
    logits[4] = 80.0
    logits[4, 7] = -80.0
    logits[5] = torch.linspace(-200, 200, 40)
    ids = torch.tensor([[0, 1, 2], [4, 5, 6], [-1, -1, -1], [-1, 40, -7], [7, 1, 2], [0, 39, 20]], dtype=torch.int32)
    grad = torch.randn(6, 3)
    for score_fn in ("softmax", "sigmoid"):
        for renorm in (True, False):
            z = logits.double().requires_grad_()
            want = weights64(z, ids, None, score_fn, "none", renorm, 1.0, 1e-20)
            want_g = torch.autograd.grad(want, z, grad.double())[0]
            got = moe_rd.routing_weights(logits.cuda(), ids.cuda(), score_fn=score_fn, renorm=renorm).cpu()
            got_g = moe_rd.routing_weights_backward(grad.cuda(), logits.cuda(), ids.cuda(), score_fn=score_fn, renorm=renorm).cpu()
            assert (got[2:4] == 0).all() and (got_g[2:4] == 0).all()
            for t in (0, 4, 5) + ((1,) if score_fn == "softmax" else ()):
                # arguments up to 400 away from the maximum: 400 + 4 units in a score, see bounds() above
                assert ((got[t].double() - want[t].detach()).abs() <= 1e-4 * want[t].detach().abs() + 1e-37).all()
                # The expected gradient has an error of its own, which is all there is of it where the true one is 0 (one sure
                # expert, renormalised): grad / total and sum(grad u) / total^2 are at most max|grad| / total each and are
                # subtracted, as are g and sum(g p) in the softmax, of at most twice that; up to ten roundings of 2^-53 a term.
                total = weights64(logits.double(), ids, None, score_fn, "none", False, 1.0, 1e-20)[t].sum().clamp(max=1.0)
                own = 64 * 2.0 ** -53 * grad[t].abs().max() / total
                assert ((got_g[t].double() - want_g[t]).abs() <= 2e-4 * want_g[t].abs().max() + own + 1e-37).all()


def test_a_logit_that_is_no_number_reaches_all_of_its_token():
    logits = torch.randn(4, 12)
    logits[1, 5] = float("nan")
    ids = torch.tensor([[0, 1], [5, 2], [3, 4], [5, 6]], dtype=torch.int32)
    for score_fn in ("softmax", "sigmoid"):
        w = moe_rd.routing_weights(logits.cuda(), ids.cuda(), score_fn=score_fn).cpu()
        g = moe_rd.routing_weights_backward(torch.ones(4, 2).cuda(), logits.cuda(), ids.cuda(), score_fn=score_fn).cpu()
        assert torch.isnan(w[1]).all() and torch.isnan(g[1, ids[1].long()]).all()
        assert torch.isfinite(w[[0, 2, 3]]).all() and torch.isfinite(g[[0, 2, 3]]).all()


def test_sizes_of_nothing_and_graph():
    e = moe_rd.routing_weights(torch.zeros(0, 8).cuda(), torch.zeros(0, 2, dtype=torch.int32).cuda())
    assert e.shape == (0, 2)
    logits, ids, bias, grad = (t.cuda() for t in inputs(90, 64, 4))
    step = lambda: (moe_rd.routing_weights(logits, ids), moe_rd.routing_weights_backward(grad, logits, ids))  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    logits.normal_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip([t.clone() for t in res], step()))


@pytest.mark.parametrize("T,E,K,score_fn,bias_mode,renorm,scale,norm_min", [
    (33, 4, 2, "softmax", "none", True, 1.0, 1e-20),
    (1, 16, 4, "softmax", "logit", False, 2.5, 1e-20),
    (300, 13, 3, "softmax", "select_and_weight", True, 1.0, 1e-20),
    (300, 16, 4, "sigmoid", "select", True, 1.0, 1e-20),
    (20000, 4, 1, "softmax", "none", False, 1.0, 1e-20),
    (300, 17, 4, "softmax", "none", True, 1.0, 1e-20),
    (16384, 64, 4, "softmax", "none", True, 1.0, 1e-20),
    (16385, 64, 4, "softmax", "none", True, 1.0, 1e-20),
    (16387, 61, 3, "softmax", "logit", False, 0.5, 1e-20),
    (20001, 60, 4, "softmax", "select_and_weight", True, 2.5, 0.3),
    (20001, 64, 4, "sigmoid", "select_and_weight", True, 1.0, 1e-20),
    (16385, 65, 4, "softmax", "none", True, 1.0, 1e-20),
])
def test_weights_and_gradient_of_few_slots(T, E, K, score_fn, bias_mode, renorm, scale, norm_min):
    test_weights_and_gradient(T, E, K, score_fn, bias_mode, renorm, scale, norm_min)
