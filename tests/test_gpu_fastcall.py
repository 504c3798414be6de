"""The ordinary call goes straight to the library (csrc/fastcall.cpp) and every other one through Python: both give the
same results, and what only Python may decide is left to it."""
import threading

import pytest
import torch

import moe_rd
from moe_rd import _cabi

pytestmark = pytest.mark.gpu


class Recorder:
    """Hands the calls on to the compiled module and notes which were taken."""

    def __init__(self, module):
        self.module, self.taken = module, []

    def __getattr__(self, name):
        def call(*args):
            done = getattr(self.module, name)(*args)
            self.taken.append(done is not False)
            return done
        return call


@pytest.fixture
def recorder(monkeypatch):
    _cabi.lib()
    assert not isinstance(_cabi.fast, _cabi._NotLoaded), "moe_rd/_fastcall.so is not built"
    r = Recorder(_cabi.fast)
    monkeypatch.setattr(_cabi, "fast", r)
    return r


def inputs(T=37, K=4, E=16, H=256, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(T * 1000 + K * 10 + E)
    cuda = lambda t: t.cuda()
    x = torch.randn(T, H, generator=g).to(dtype)
    ids = torch.randint(-1, E, (T, K), generator=g, dtype=torch.int32)
    w, logits, bias = torch.rand(T, K, generator=g), torch.randn(T, E, generator=g), torch.rand(E, generator=g)
    grad, grad_w = torch.randn(T, H, generator=g).to(dtype), torch.randn(T, K, generator=g)
    return [cuda(t) for t in (x, ids, w, logits, bias, grad, grad_w)]


def w4(E=16, N=72, K=256, group=64, dtype=torch.bfloat16, zeros=True):
    g = torch.Generator().manual_seed(E * N)
    q = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(E, N, K // group, generator=g) * 0.01).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return moe_rd.pack_w4(q.cuda(), s.cuda(), None if z is None else z.cuda())


def calls(dtype=torch.bfloat16, T=37):
    """Every entry point as a function of ``out``."""
    x, ids, w, logits, bias, grad, grad_w = inputs(T=T, dtype=dtype)
    s = moe_rd.sort_tokens(x, ids, 16)
    out = {
        "sort": lambda out=None: moe_rd.sort_tokens(x, ids, 16, out=out),
        "sort capacity": lambda out=None: moe_rd.sort_tokens(x, ids, 16, capacity=3, out=out),
        "unsort": lambda out=None: moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, x, offsets=s.offsets, out=out),
        "unsort plain": lambda out=None: moe_rd.unsort_tokens(s.rows, s.inverse_perm, out=out),
        "unsort backward": lambda out=None: moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, w, offsets=s.offsets, out=out),
        "unsort backward rows": lambda out=None: moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, out=out),
        "unsort backward weights": lambda out=None: moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, w, need_rows=False, out=out),
        "weights": lambda out=None: moe_rd.routing_weights(logits, ids, out=out),
        "weights sigmoid": lambda out=None: moe_rd.routing_weights(logits, ids, bias, score_fn="sigmoid", bias_mode="select_and_weight", renorm=False,
                                                                   routed_scale=2, out=out),
        "weights logit": lambda out=None: moe_rd.routing_weights(logits, ids, bias, bias_mode="logit", out=out),
        "weights select": lambda out=None: moe_rd.routing_weights(logits, ids, bias, bias_mode="select", out=out),
        "weights backward": lambda out=None: moe_rd.routing_weights_backward(grad_w, logits, ids, bias, bias_mode="logit", routed_scale=2.5, out=out),
    }
    if dtype is not torch.float32:
        p, dense = w4(dtype=dtype), w4(E=1, zeros=False, dtype=dtype)
        out["w4"] = lambda out=None: moe_rd.expert_matvec_w4(s.rows, p, s.offsets, out=out)
        out["w4 one matrix"] = lambda out=None: moe_rd.expert_matvec_w4(x, dense, out=out)
    return out


def tensors(r):
    return [r] if isinstance(r, torch.Tensor) else list(r)


def same(a, b):
    a, b = tensors(a), tensors(b)
    assert len(a) == len(b)
    for u, v in zip(a, b):
        assert (u is None) == (v is None)
        if u is not None:
            assert u.shape == v.shape and u.dtype == v.dtype and u.is_contiguous()
            assert torch.equal(u, v)


@pytest.mark.parametrize("T", [0, 1, 37])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_both_ways_give_the_same(recorder, monkeypatch, dtype, T):
    for name, f in calls(dtype, T).items():
        recorder.taken.clear()
        fast = f()
        again = f(fast)
        assert recorder.taken == [True, True], name
        assert again is fast
        with monkeypatch.context() as m:
            m.setattr(_cabi, "fast", _cabi._NotLoaded())
            slow = f()
        assert type(fast) is type(slow)
        same(fast, slow)


def test_buffers_that_are_reused_are_written_for_autograd(recorder):
    for name, f in calls().items():
        out = f()
        before = [None if t is None else t._version for t in tensors(out)]
        f(out)
        for t, v in zip(tensors(out), before):
            assert t is None or t._version > v, name
    with torch.inference_mode():
        for f in calls().values():
            f(f())


@pytest.mark.parametrize("fast", [True, False])
def test_what_python_decides(recorder, monkeypatch, fast):
    """The same answers with the compiled module and without it."""
    if not fast:
        monkeypatch.setattr(_cabi, "fast", _cabi._NotLoaded())
    x, ids, w, logits, bias, grad, grad_w = inputs()
    s = moe_rd.sort_tokens(x, ids, 16)
    # strides and addresses
    wide = torch.empty(37, 512, dtype=x.dtype, device="cuda")
    wide[:, 8:264] = x
    same(moe_rd.sort_tokens(wide[:, 8:264], ids, 16), s)
    buffer = torch.empty(37 * 256 + 1, dtype=x.dtype, device="cuda")
    odd = buffer[1:].view(37, 256).copy_(x)
    same(moe_rd.sort_tokens(odd, ids.t().contiguous().t(), 16), s)
    same(moe_rd.sort_tokens(x.view(1, 37, 256), ids, 16), s)
    same(moe_rd.sort_tokens(torch.nn.Parameter(x, requires_grad=False), ids, 16), s)
    back = moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, x)
    same(moe_rd.unsort_tokens(s.rows[None], s.inverse_perm, w.t().contiguous().t(), x.view(37, 1, 256)), back)
    # refusals
    with pytest.raises(ValueError, match="share memory"):
        moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, x, out=x)
    with pytest.raises(ValueError, match="share memory"):
        moe_rd.routing_weights(logits[:, :4].contiguous(), ids, out=ids.view(torch.float32))
    with pytest.raises(ValueError, match="out must be"):
        moe_rd.routing_weights(logits, ids, out=torch.empty(37, 5, device="cuda"))
    with pytest.raises(ValueError, match="16-byte aligned"):
        moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, out=odd)
    with pytest.raises(TypeError, match="int32"):
        moe_rd.sort_tokens(x, ids.long(), 16)
    with pytest.raises(TypeError, match="int32"):
        moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, offsets=s.offsets.long())
    with pytest.raises(ValueError, match="score_fn"):
        moe_rd.routing_weights(logits, ids, score_fn="tanh")
    with pytest.raises(ValueError, match="bias_mode"):
        moe_rd.routing_weights(logits, ids, bias, bias_mode="weight")
    with pytest.raises(ValueError, match="tokens"):
        moe_rd.sort_tokens(x[:36], ids, 16)
    with pytest.raises(moe_rd.MoeRdError):
        moe_rd.sort_tokens(x, ids, 257)
    with pytest.raises(moe_rd.MoeRdError):
        moe_rd.sort_tokens(x, ids.repeat(1, 9), 16)
    with pytest.raises(ValueError, match="no gradient is asked for"):
        moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, w, need_rows=False, need_weights=False)
    with pytest.raises(ValueError, match="gradients that are asked for"):
        moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, w, out=moe_rd.UnsortGradients(torch.empty_like(s.rows), None))
    p = w4()
    with pytest.raises(ValueError, match="offsets are needed"):
        moe_rd.expert_matvec_w4(s.rows, p)
    with pytest.raises(ValueError, match="as pack_w4 returns"):
        moe_rd.expert_matvec_w4(s.rows, p._replace(packed=p.packed[:, :-1].contiguous()), s.offsets)
    with pytest.raises(TypeError, match="one type"):
        moe_rd.expert_matvec_w4(s.rows.half(), p, s.offsets)
    with pytest.raises(RuntimeError, match="no gradient"):
        moe_rd.expert_matvec_w4(s.rows.clone().requires_grad_(), p, s.offsets)
    # gradients
    leaf, lw, ll = x.clone().requires_grad_(), w.clone().requires_grad_(), logits.clone().requires_grad_()
    rows = moe_rd.sort_tokens(leaf, ids, 16)
    out = moe_rd.unsort_tokens(rows.rows, rows.inverse_perm, lw, offsets=rows.offsets)
    weights = moe_rd.routing_weights(ll, ids)
    assert out.requires_grad and weights.requires_grad
    torch.autograd.backward([out, weights], [grad, grad_w])
    g = moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, w, offsets=s.offsets)
    same(leaf.grad, moe_rd.unsort_tokens(g.rows, s.inverse_perm))
    same(lw.grad, g.weights)
    same(ll.grad, moe_rd.routing_weights_backward(grad_w, logits, ids))
    with torch.no_grad():
        assert not moe_rd.sort_tokens(leaf, ids, 16).rows.requires_grad
    # a graph that saved a buffer which is overwritten afterwards says so
    saved = moe_rd.unsort_tokens(rows.rows.detach(), rows.inverse_perm, lw)
    moe_rd.sort_tokens(x, ids, 16, out=moe_rd.SortedTokens(*(t.detach() for t in rows)))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward(grad)


def test_on_another_stream_and_captured(recorder):
    fs = calls()
    want = {name: f() for name, f in fs.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = {name: f() for name, f in fs.items()}
    torch.cuda.current_stream().wait_stream(side)
    for name in fs:
        same(got[name], want[name])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = {name: f() for name, f in fs.items()}
    assert all(recorder.taken)
    for r in made.values():
        for t in tensors(r):
            if t is not None:
                t.zero_()
    graph.replay()
    for name in fs:
        same(made[name], want[name])


def test_from_several_threads(recorder):
    fs = calls()
    want = {name: f() for name, f in fs.items()}
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = {name: f() for name, f in fs.items()}
                torch.cuda.current_stream().synchronize()
                for name in fs:
                    same(got[name], want[name])
        except BaseException as e:  # noqa: BLE001 - shown by the assertion below
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("fast", [True, False])
def test_tangents_of_forward_mode_are_refused(recorder, monkeypatch, fast):
    """They would be dropped; a Function of the caller's that carries them on itself may call."""
    import torch.autograd.forward_ad as fwad
    if not fast:
        monkeypatch.setattr(_cabi, "fast", _cabi._NotLoaded())
    x, ids, w, logits, bias, grad, grad_w = inputs(dtype=torch.float32)
    s = moe_rd.sort_tokens(x, ids, 16)
    half, p = x.bfloat16(), w4(E=1)
    scales = p.scales

    class Sorted(torch.autograd.Function):
        @staticmethod
        def forward(x, ids):
            return moe_rd.sort_tokens(x, ids, 16).rows

        @staticmethod
        def setup_context(ctx, inputs, output):
            ctx.ids = inputs[1]

        @staticmethod
        def jvp(ctx, tangent, _):
            return moe_rd.sort_tokens(tangent, ctx.ids, 16).rows

    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))
        for call in (lambda: moe_rd.sort_tokens(dual(x), ids, 16), lambda: moe_rd.sort_tokens(dual(x), ids, 16, out=s),
                     lambda: moe_rd.unsort_tokens(dual(s.rows), s.inverse_perm, w), lambda: moe_rd.unsort_tokens(s.rows, s.inverse_perm, dual(w)),
                     lambda: moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, dual(x)), lambda: moe_rd.unsort_tokens_backward(dual(grad), s.rows, s.inverse_perm, w),
                     lambda: moe_rd.unsort_tokens_backward(grad, s.rows, s.inverse_perm, dual(w)), lambda: moe_rd.routing_weights(dual(logits), ids),
                     lambda: moe_rd.routing_weights(dual(logits.clone().requires_grad_()), ids),
                     lambda: moe_rd.routing_weights(logits, ids, dual(bias), bias_mode="logit"), lambda: moe_rd.routing_weights_backward(dual(grad_w), logits, ids),
                     lambda: moe_rd.routing_weights_backward(grad_w, dual(logits), ids), lambda: moe_rd.expert_matvec_w4(dual(half), p),
                     lambda: moe_rd.expert_matvec_w4(half, p._replace(scales=dual(scales)))):
            recorder.taken.clear()
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            assert not any(recorder.taken)
        same(moe_rd.sort_tokens(x, ids, 16), s)                       # a level that is open changes nothing for others
        primal, tangent = fwad.unpack_dual(Sorted.apply(dual(x), ids))
        assert torch.equal(primal, s.rows) and torch.equal(tangent, moe_rd.sort_tokens(torch.ones_like(x), ids, 16).rows)


@pytest.mark.parametrize("fast", [True, False])
def test_a_sign_that_is_still_to_change(recorder, monkeypatch, fast):
    """The imaginary part of a conjugate is a view whose numbers in memory have the other sign."""
    if not fast:
        monkeypatch.setattr(_cabi, "fast", _cabi._NotLoaded())
    g = torch.Generator().manual_seed(0)
    of = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.complex64).cuda().conj().imag
    rows, w, logits, ids = of(1, 64), of(1, 1), of(1, 1), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    assert all(t.is_neg() for t in (rows, w, logits)) and w.is_contiguous()
    plain = lambda t: t.resolve_neg().contiguous()
    inv = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    same(moe_rd.sort_tokens(rows, ids, 1), moe_rd.sort_tokens(plain(rows), ids, 1))
    got = moe_rd.unsort_tokens(rows, inv, w, rows)
    same(got, moe_rd.unsort_tokens(plain(rows), inv, plain(w), plain(rows)))
    assert (got.double() - (1 + plain(w).double()) * plain(rows).double()).abs().max() <= 2.0 ** -22 * ((1 + w.abs()) * rows.abs().max()).item()
    same(moe_rd.unsort_tokens_backward(rows, rows, inv, w), moe_rd.unsort_tokens_backward(plain(rows), plain(rows), inv, plain(w)))
    config = dict(score_fn="sigmoid", renorm=False)
    same(moe_rd.routing_weights(logits, ids, w, bias_mode="logit", **config), moe_rd.routing_weights(plain(logits), ids, plain(w), bias_mode="logit", **config))
    same(moe_rd.routing_weights_backward(w, logits, ids, **config), moe_rd.routing_weights_backward(plain(w), plain(logits), ids, **config))
    with pytest.raises(ValueError, match="out must be"):
        moe_rd.routing_weights(plain(logits), ids, out=of(1, 1))
