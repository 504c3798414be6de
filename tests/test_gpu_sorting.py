"""Sorting tokens by expert and back, with weights, and the gradients, against plain statements in 64 bits."""
import numpy as np
import pytest
import torch

import moe_rd

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25, "fp32": 2.0 ** -150}   # half of the smallest number of the type


def places(ids, E, capacity):
    """A walk over the pairs: row of every pair, offsets, counts, token of every row."""
    T, K = ids.shape
    lists = [[] for _ in range(E)]
    counts = np.zeros(E, np.int32)
    for t in range(T):
        for k in range(K):
            e = int(ids[t, k])
            if 0 <= e < E:
                counts[e] += 1
                if capacity == 0 or len(lists[e]) < capacity:
                    lists[e].append((t, k))
    inv = np.full((T, K), -1, np.int32)
    offsets = np.zeros(E + 1, np.int32)
    token = []
    for e in range(E):
        for t, k in lists[e]:
            inv[t, k] = len(token)
            token.append(t)
        offsets[e + 1] = len(token)
    return inv, offsets, counts, np.array(token, np.int64)


def ids_of(T, K, E, kind, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + K)
    ids = torch.randint(0, E, (T, K), generator=g, dtype=torch.int32)
    if kind == "padded":
        ids[torch.rand(T, generator=g) < 0.4] = -1
    elif kind == "one expert":
        ids[:] = E - 1
    elif kind == "none":
        ids[:] = -1
    elif kind == "stray":
        ids[torch.rand(T, K, generator=g) < 0.2] = E
        ids[torch.rand(T, K, generator=g) < 0.1] = -2 ** 31
        ids[torch.rand(T, K, generator=g) < 0.1] = 2 ** 31 - 1
    return ids


SORT_CASES = [
    # T, K, E, H, dtype, capacity, ids
    (1, 8, 256, 7168, "bf16", 0, "random"),
    (1, 1, 1, 8, "bf16", 0, "random"),
    (3, 2, 5, 4, "fp32", 0, "padded"),
    (7, 3, 60, 264, "fp16", 1, "random"),
    (2048, 8, 256, 1024, "bf16", 0, "random"),    # 16384 pairs: the last size of the one-kernel form
    (2049, 8, 256, 1024, "bf16", 0, "random"),    # the first of the batch form
    (16384, 1, 3, 8, "bf16", 0, "padded"),        # many tokens a block
    (1025, 1, 7, 20, "fp32", 100, "padded"),
    (33, 32, 4, 72, "fp16", 0, "random"),         # more ids than experts: the same expert several times per token
    (64, 32, 256, 40, "bf16", 3, "stray"),
    (2047, 2, 8, 136, "bf16", 300, "one expert"),
    (2049, 2, 8, 516, "fp32", 0, "stray"),
    (2049, 9, 8, 132, "fp32", 0, "stray"),        # one token into a second group of counting tiles
    (4100, 5, 16, 264, "fp16", 900, "one expert"),
    (700, 32, 33, 72, "bf16", 0, "padded"),
    (8200, 2, 16, 64, "bf16", 0, "none"),
    (40, 4, 16, 64, "bf16", 0, "none"),
    (600, 4, 16, 64, "fp16", 2, "none"),
    (5000, 6, 160, 520, "fp16", 200, "padded"),
]


@pytest.mark.parametrize("T,K,E,H,dtype,capacity,kind", SORT_CASES)
def test_sort_is_exact(T, K, E, H, dtype, capacity, kind):
    ids = ids_of(T, K, E, kind)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(DT[dtype])
    x.view(-1)[::97] = float("nan")
    x.view(-1)[1::89] = float("inf")
    inv, offsets, counts, token = places(ids.numpy(), E, capacity)
    for run in range(2):  # a second call into the buffers of the first, which hold other things by then
        out = None
        if run:
            for t in got:
                t.view(torch.uint8).fill_(0x55)
            out = got
        got = moe_rd.sort_tokens(x.cuda(), ids.cuda(), E, capacity=capacity, out=out)
        np.testing.assert_array_equal(got.inverse_perm.cpu().numpy(), inv)
        np.testing.assert_array_equal(got.offsets.cpu().numpy(), offsets)
        np.testing.assert_array_equal(got.counts.cpu().numpy(), counts)
        R = min(T * K, E * capacity) if capacity else T * K
        assert got.rows.shape == (R, H) and got.row_token.shape == (R,)
        want_token = np.full(R, -1, np.int32)
        want_token[:len(token)] = token
        np.testing.assert_array_equal(got.row_token.cpu().numpy(), want_token)
        want = torch.zeros(R, H, dtype=x.dtype)
        want[:len(token)] = x[torch.from_numpy(token)]
        assert torch.equal(got.rows.cpu().view(torch.uint8), want.view(torch.uint8))  # bit copies, NaN included


def test_sort_of_no_tokens_and_of_views():
    e = torch.zeros((0, 2), dtype=torch.int32).cuda()
    got = moe_rd.sort_tokens(torch.zeros(0, 64, dtype=torch.bfloat16).cuda(), e, 4)
    assert got.rows.shape == (0, 64) and got.offsets.tolist() == [0] * 5 and got.counts.tolist() == [0] * 4
    base = torch.randn(50, 2 * 128 + 1).cuda()
    ids = ids_of(20, 4, 6, "padded").cuda()
    for x in (base[:20, 1:129], base[:40:2, ::2][:, :128], base[:20, :128].reshape(4, 5, 128), base.t()[:20, :48]):
        H = x.shape[-1]
        wide = torch.cat([ids, ids], 1)[:, ::2]  # a strided view of ids
        a = moe_rd.sort_tokens(x, wide, 6)
        b = moe_rd.sort_tokens(x.reshape(20, H).clone(), wide.clone(), 6)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_sort_agrees_with_route_dispatch():
    """The ids, capacity and rows of a routed batch, sorted again: the same places."""
    from moe_rd import workloads
    t, kw = workloads.make("c3", T=3000, H=512)
    r = moe_rd.route_dispatch(t["x"].cuda(), t["w"].cuda(), t["bias"].cuda(), return_row_meta=True, **kw)
    s = moe_rd.sort_tokens(t["x"].cuda(), r.expert_ids, 128, capacity=kw["capacity"])
    live = int(r.offsets[-1])
    assert torch.equal(s.offsets, r.offsets) and torch.equal(s.inverse_perm, r.inverse_perm) and torch.equal(s.counts, r.counts)
    assert torch.equal(s.rows[:live], r.permuted[:live]) and torch.equal(s.row_token[:live], r.row_token[:live])


def random_places(T, K, R, seed, missing=0.2):
    """Every row of 0..n-1 once, in a random order; pairs without a row in between."""
    g = torch.Generator().manual_seed(seed)
    has = torch.rand(T * K, generator=g) >= missing
    n = min(int(has.sum()), R)
    at = torch.nonzero(has)[:, 0][:n]
    inv = torch.full((T * K,), -1, dtype=torch.int32)
    inv[at] = torch.randperm(n, generator=g).to(torch.int32)
    return inv.reshape(T, K), n


UNSORT_CASES = [
    # T, K, H, dtype, weighted, shared
    (1, 8, 7168, "bf16", True, True),
    (1, 1, 8, "bf16", False, False),
    (5, 3, 4, "fp32", True, False),
    (70, 2, 264, "fp16", True, True),
    (33, 8, 1040, "bf16", False, True),
    (300, 20, 264, "bf16", True, False),
    (129, 10, 132, "fp32", False, False),
    (2000, 4, 520, "fp16", True, False),
    (777, 6, 2056, "bf16", True, False),
    (64, 32, 40, "fp16", True, True),
]


def unsort_inputs(T, K, H, dtype, seed=1, missing=0.2):
    R = T * K
    g = torch.Generator().manual_seed(seed + T)
    inv, n = random_places(T, K, R, seed, missing)
    y = torch.randn(R, H, generator=g).to(DT[dtype])
    w = torch.randn(T, K, generator=g)
    sh = torch.randn(T, H, generator=g).to(DT[dtype])
    return y, inv, w, sh, n


def unsort64(y, inv, w, sh):
    """The formula in 64 bits, and the sum of the terms' magnitudes."""
    T, K = inv.shape
    rows = y.double()[inv.clamp(min=0).long()] * (inv >= 0)[..., None]
    terms = rows if w is None else rows * (w.double() * (inv >= 0))[..., None]
    out, mag = terms.sum(1), terms.abs().sum(1)
    if sh is not None:
        out, mag = out + sh.double(), mag + sh.double().abs()
    return out, mag


@pytest.mark.parametrize("T,K,H,dtype,weighted,shared", UNSORT_CASES)
def test_unsort(T, K, H, dtype, weighted, shared):
    y, inv, w, sh, _ = unsort_inputs(T, K, H, dtype)
    w, sh = w if weighted else None, sh if shared else None
    want, mag = unsort64(y, inv, w, sh)
    if weighted:
        w = torch.where(inv < 0, torch.full_like(w, float("nan")), w)   # a pair without a row has no say
    got = moe_rd.unsort_tokens(y.cuda(), inv.cuda(), None if w is None else w.cuda(), None if sh is None else sh.cuda())
    # K fused multiply-adds in 32 bits, each within 2^-24 of a partial sum that the magnitudes bound, then one rounding
    low = K * 2.0 ** -24 * mag * (1 + K * 2.0 ** -24)
    bound = low + HALF_STEP[dtype] * (want.abs() + low) + TINY[dtype]
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_unsort_ignores_rows_out_of_range():
    y = torch.randn(10, 64).cuda()
    inv = torch.tensor([[0, 10], [2 ** 31 - 1, -2 ** 31], [9, -1]], dtype=torch.int32).cuda()
    w = torch.ones(3, 2).cuda()
    got = moe_rd.unsort_tokens(y, inv, w)
    assert torch.equal(got, torch.stack([y[0], torch.zeros_like(y[0]), y[9]]))
    none = moe_rd.unsort_tokens(y[:0], inv, w, y[:3])
    assert torch.equal(none, y[:3])
    # fp32 rows and weights of 1: equal to no weights at all
    assert torch.equal(moe_rd.unsort_tokens(y, inv), got)


def test_unsort_equals_combine():
    y, inv, w, sh, _ = unsort_inputs(400, 8, 512, "bf16")
    a = moe_rd.unsort_tokens(y.cuda(), inv.cuda(), w.cuda(), sh.cuda())
    assert torch.equal(a, moe_rd.combine(y.cuda(), inv.cuda(), w.cuda(), sh.cuda()))


@pytest.mark.parametrize("T,K,H,dtype,weighted,shared", UNSORT_CASES)
@pytest.mark.parametrize("with_offsets", [True, False])
def test_unsort_gradients(T, K, H, dtype, weighted, shared, with_offsets):
    y, inv, w, _, n = unsort_inputs(T, K, H, dtype, seed=3)
    g = torch.randn(T, H, generator=torch.Generator().manual_seed(9)).to(DT[dtype])
    offsets = torch.tensor([0, n], dtype=torch.int32).cuda() if with_offsets else None
    want_y = torch.zeros(T * K, H, dtype=torch.float64)
    has = inv >= 0
    each = (w.double()[..., None] if weighted else 1.0) * g.double()[:, None, :].expand(T, K, H)
    want_y[inv[has].long()] = each[has]
    rows = y.double()[inv.clamp(min=0).long()] * has[..., None]
    want_w = (rows * g.double()[:, None, :]).sum(2)
    mag_w = (rows * g.double()[:, None, :]).abs().sum(2)
    wc = w.cuda() if weighted else None
    got = moe_rd.unsort_tokens_backward(g.cuda(), y.cuda(), inv.cuda(), wc, offsets=offsets, need_weights=True)
    # one product in 32 bits, then one rounding (no rounding at all without weights)
    bound = want_y.abs() * (HALF_STEP[dtype] + 2.0 ** -24 * (1 + HALF_STEP[dtype])) + TINY[dtype]
    assert ((got.rows.cpu().double() - want_y).abs() <= bound).all()
    # a lane adds at most ceil(H / 32) products, 5 + 7 additions join lanes and warps
    assert ((got.weights.cpu().double() - want_w).abs() <= (H / 32 + 9 + 12) * 2.0 ** -24 * mag_w).all()
    assert (got.weights.cpu()[~has] == 0).all()
    # the same bits again, into the buffers of the first call; and each gradient alone
    first = [t.clone() for t in got]
    for t in got:
        t.fill_(float("nan"))
    again = moe_rd.unsort_tokens_backward(g.cuda(), y.cuda(), inv.cuda(), wc, offsets=offsets, need_weights=True, out=got)
    assert again is got and all(torch.equal(p, q) for p, q in zip(first, again))
    assert torch.equal(moe_rd.unsort_tokens_backward(g.cuda(), y.cuda(), inv.cuda(), wc, offsets=offsets, need_weights=False).rows, first[0])
    assert torch.equal(moe_rd.unsort_tokens_backward(g.cuda(), y.cuda(), inv.cuda(), wc, need_rows=False, need_weights=True).weights,
                       first[1])


def test_gradients_of_padded_and_empty_batches():
    z = torch.zeros(0, 2, dtype=torch.int32).cuda()
    got = moe_rd.unsort_tokens_backward(torch.zeros(0, 64).cuda(), torch.randn(5, 64).cuda(), z, need_weights=True)
    assert torch.equal(got.rows, torch.zeros(5, 64).cuda()) and got.weights.shape == (0, 2)
    inv = torch.full((9, 3), -1, dtype=torch.int32).cuda()
    nan = torch.full((9, 64), float("nan")).cuda()
    got = moe_rd.unsort_tokens_backward(nan, torch.randn(27, 64).cuda(), inv, torch.ones(9, 3).cuda(),
                                        offsets=torch.zeros(2, dtype=torch.int32).cuda())
    assert torch.equal(got.rows, torch.zeros(27, 64).cuda()) and torch.equal(got.weights, torch.zeros(9, 3).cuda())


@pytest.mark.parametrize("T,K,E,H,capacity", [(37, 3, 5, 20, 0), (300, 4, 8, 64, 90)])
def test_autograd_against_differences(T, K, E, H, capacity):
    """Sort, a factor per row, and back: the gradients are those of the formula, and agree with differences of it
    along a random direction.  The formula is linear in each argument, so a central difference has no error of its own."""
    g = torch.Generator().manual_seed(T)
    ids = ids_of(T, K, E, "padded", 5)
    inv, _, _, token = places(ids.numpy(), E, capacity)
    R = min(T * K, E * capacity) if capacity else T * K
    x = torch.randn(T, H, generator=g)
    w = torch.rand(T, K, generator=g)
    sh = torch.randn(T, H, generator=g)
    f = torch.randn(R, H, generator=g)
    go = torch.randn(T, H, generator=g)
    invt = torch.from_numpy(inv)

    def loss64(x, w, sh):
        rows = torch.zeros(R, H, dtype=torch.float64)
        rows[:len(token)] = x[torch.from_numpy(token)]
        return (unsort64(rows * f.double(), invt, w, sh)[0] * go.double()).sum()

    leaves = [t.cuda().requires_grad_() for t in (x, w, sh)]
    s = moe_rd.sort_tokens(leaves[0], ids.cuda(), E, capacity=capacity)
    assert s.rows.requires_grad and not s.offsets.requires_grad
    out = moe_rd.unsort_tokens(s.rows * f.cuda(), s.inverse_perm, leaves[1], leaves[2], offsets=s.offsets)
    out.backward(go.cuda())
    ref = [t.double().requires_grad_() for t in (x, w, sh)]
    loss64(*ref).backward()
    for got, want in zip(leaves, ref):
        # at most H + K + 4 roundings of 2^-24 on sums whose terms are below 30 in magnitude here
        err = (got.grad.cpu().double() - want.grad).abs().max()
        assert err <= (H + K + 4) * 2.0 ** -24 * 30 * K
    for i, base in enumerate((x, w, sh)):
        d = torch.randn(base.shape, generator=g).double()
        args = [t.double() for t in (x, w, sh)]
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + d, args[i] - d
        diff = (loss64(*up) - loss64(*down)) / 2
        along = (leaves[i].grad.cpu().double() * d).sum()
        assert (along - diff).abs() <= (H + K + 4) * 2.0 ** -24 * 30 * K * d.abs().sum()


def test_a_training_layer_end_to_end():
    """route_dispatch's ids, routing_weights, sort_tokens, expert products and unsort_tokens: the gradients of the tokens,
    the gate, the experts and the shared branch against the same layer in 64 bits."""
    T, H, E, K, N = 200, 128, 8, 3, 128
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).float()
    wg = torch.randn(H, E, generator=g) * 0.1
    we = torch.randn(E, H, N, generator=g) * 0.1
    go = torch.randn(T, N, generator=g)
    capacity = 90

    leaves = [t.cuda().requires_grad_() for t in (x, wg, we)]
    logits = leaves[0] @ leaves[1]
    r = moe_rd.route_dispatch(x.cuda().to(torch.bfloat16), None, top_k=K, given_logits=logits.detach(), capacity=capacity,
                              scatter_impl="none")
    w = moe_rd.routing_weights(logits, r.expert_ids)
    torch.testing.assert_close(w.detach(), r.combine_weights, rtol=2e-6, atol=0)   # the same function, other roundings
    s = moe_rd.sort_tokens(leaves[0], r.expert_ids, E, capacity=capacity)
    assert torch.equal(s.inverse_perm, r.inverse_perm)
    o = s.offsets.tolist()
    y = torch.cat([s.rows[o[e]:o[e + 1]] @ leaves[2][e] for e in range(E)] + [s.rows[o[E]:] @ leaves[2][0]])
    out = moe_rd.unsort_tokens(y, s.inverse_perm, w, leaves[0], offsets=s.offsets)
    out.backward(go.cuda())

    ids, inv = r.expert_ids.cpu().long(), r.inverse_perm.cpu()
    ref = [t.double().requires_grad_() for t in (x, wg, we)]
    z = torch.softmax(ref[0] @ ref[1], 1).gather(1, ids)
    wr = z / z.sum(1, keepdim=True) * (inv >= 0)
    yr = torch.einsum("th,tkhn->tkn", ref[0], ref[2][ids])
    want = (wr[..., None] * yr).sum(1) + ref[0]
    want.backward(go.double())
    assert (out.detach().cpu().double() - want.detach()).abs().max() <= 1e-4 * want.detach().abs().max()
    for got, exact in zip(leaves, ref):
        # sums of at most T * K * H products in 32 bits; their roundings add up like a random walk: 2^-24 * sqrt(76800) < 2e-5
        assert (got.grad.cpu().double() - exact.grad).norm() <= 2e-5 * exact.grad.norm()


def test_graph_replay_and_streams():
    """The plain functions recorded into a graph and replayed on new inputs; and run on another stream."""
    T, K, E, H = 700, 4, 16, 256
    x, y, ids = torch.randn(T, H).cuda(), torch.randn(T * K, H).cuda(), ids_of(T, K, E, "padded").cuda()
    w, g = torch.rand(T, K).cuda(), torch.randn(T, H).cuda()

    def step():
        s = moe_rd.sort_tokens(x, ids, E)
        few = moe_rd.sort_tokens(x[:9], ids[:9], E)
        out = moe_rd.unsort_tokens(y, s.inverse_perm, w)
        grads = moe_rd.unsort_tokens_backward(g, y, s.inverse_perm, w, offsets=s.offsets)
        dx = moe_rd.unsort_tokens(grads.rows, s.inverse_perm)
        return (*s, *few, out, *grads, dx)

    step()
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for _ in range(2):  # two graphs that share one memory pool, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            res = step()
        graphs.append((graph, res))
    x.normal_()
    y.normal_()
    ids.copy_(ids_of(T, K, E, "stray", 3))
    for graph, res in graphs:
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in res]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, step()))


def test_autograd_is_refused_while_capturing():
    x = torch.randn(8, 64, device="cuda", requires_grad=True)
    y = torch.randn(16, 64, device="cuda", requires_grad=True)
    ids = ids_of(8, 2, 4, "random").cuda()
    inv = moe_rd.sort_tokens(x.detach(), ids, 4).inverse_perm
    torch.cuda.synchronize()
    for fn in (lambda: moe_rd.sort_tokens(x, ids, 4), lambda: moe_rd.unsort_tokens(y, inv)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="not recorded into a CUDA graph"):
            with torch.cuda.graph(graph):
                fn()
    assert torch.equal(moe_rd.sort_tokens(x, ids, 4).inverse_perm, inv)


def test_a_buffer_that_backward_needs_cannot_be_reused_unseen():
    x = torch.randn(50, 64, device="cuda", requires_grad=True)
    ids = ids_of(50, 2, 8, "random").cuda()
    s = moe_rd.sort_tokens(x, ids, 8)
    out = moe_rd.unsort_tokens(s.rows, s.inverse_perm, offsets=s.offsets)
    moe_rd.sort_tokens(x.detach(), ids.flip(0), 8, out=moe_rd.SortedTokens(torch.empty_like(s.rows), *s[1:]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    y = torch.randn(100, 64, device="cuda", requires_grad=True)
    w = torch.rand(50, 2, device="cuda", requires_grad=True)
    out = moe_rd.unsort_tokens(y, s.inverse_perm, w)
    moe_rd.routing_weights(torch.randn(50, 8, device="cuda"), ids, out=w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_out_is_checked():
    x = torch.randn(20, 64, device="cuda")
    ids = ids_of(20, 2, 8, "random").cuda()
    s = moe_rd.sort_tokens(x, ids, 8)
    for bad in (s._replace(rows=s.rows[:39]), s._replace(rows=s.rows.half()), s._replace(rows=s.rows.cpu()), s._replace(offsets=ids.view(-1)[:9]),
                s._replace(counts=s.counts.long()), s._replace(rows=torch.empty(64, 40, device="cuda").t()),
                s._replace(rows=torch.empty(40 * 64 + 1, device="cuda")[1:].view(40, 64))):
        with pytest.raises(ValueError, match="out must"):
            moe_rd.sort_tokens(x, ids, 8, out=bad)
    for bad in (x[:19], x.double(), s.rows[:20], torch.empty(20, 64, device="cuda", requires_grad=True)):
        with pytest.raises(ValueError, match="out must"):
            moe_rd.unsort_tokens(s.rows, s.inverse_perm, out=bad)
    leaf = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="out cannot"):
        moe_rd.sort_tokens(leaf, ids, 8, out=s)
    with pytest.raises(ValueError, match="one device"):
        moe_rd.sort_tokens(x, ids.cpu(), 8)
    with pytest.raises(moe_rd.MoeRdError):
        moe_rd.sort_tokens(x, ids, 257)


def test_rows_past_32_bits():
    """More than 2^31 elements, more than 2^32 bytes of rows: the far end of every buffer is reached."""
    T, K, E, H = 38000, 8, 256, 7168
    assert T * K * H > 2 ** 31
    x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, E, (T, K), device="cuda", dtype=torch.int32)
    ids[::5] = -1
    s = moe_rd.sort_tokens(x, ids, E)
    live = int(s.offsets[-1])
    assert (s.inverse_perm[::5] == -1).all() and int((s.inverse_perm >= 0).sum()) == live
    probe = torch.cat([torch.arange(0, 300), torch.arange(live - 300, live)]).cuda()
    assert torch.equal(s.rows[probe], x[s.row_token[probe].long()])
    assert (s.rows[live:][-200:] == 0).all() and (s.row_token[live:] == -1).all()
    w = torch.rand(T, K, device="cuda")
    back = moe_rd.unsort_tokens(s.rows, s.inverse_perm, w)
    some = torch.tensor([0, 1, 5, T // 2, T - 2, T - 1]).cuda()
    want = x[some].double() * (w[some].double().sum(1) * (ids[some, 0] >= 0))[:, None]
    low = K * 2.0 ** -24 * (1 + K * 2.0 ** -24) * want.abs()    # K additions of one sign in 32 bits, then one rounding
    assert ((back[some].double() - want).abs() <= low + 2.0 ** -8 * (want.abs() + low)).all()
    g = moe_rd.unsort_tokens_backward(x, s.rows, s.inverse_perm, w, offsets=s.offsets)
    at = s.row_token[probe].long()
    k = (s.inverse_perm[at] == probe[:, None].int()).int().argmax(1)
    want = x[at].double() * w[at, k].double()[:, None]
    assert ((g.rows[probe].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -23) * want.abs() + 1e-38).all()
    assert (g.rows[live:][-200:] == 0).all()
    norm = (x[at].double() ** 2).sum(1)
    assert ((g.weights[at, k].double() - norm).abs() <= (H / 32 + 21) * 2.0 ** -24 * norm).all()


def test_batches_of_any_shape_through_autograd():
    """x and the shared branch as [batch, length, H], strided; gradients arrive in their shapes."""
    base = torch.randn(3, 10, 2, 64, device="cuda", requires_grad=True)
    x = base[:, :, 1]
    ids = ids_of(30, 2, 4, "padded").cuda()
    s = moe_rd.sort_tokens(x, ids, 4)
    out = moe_rd.unsort_tokens(s.rows * 2, s.inverse_perm, None, x, offsets=s.offsets)
    out.sum().backward()
    n = (ids >= 0).sum(1).float().view(3, 10, 1)
    want = torch.zeros_like(base)
    want[:, :, 1] = (1 + 2 * n).expand(3, 10, 64)
    assert torch.equal(base.grad, want)


def test_two_threads_on_two_streams():
    import threading
    T, K, E, H = 3000, 4, 64, 256
    data = [(torch.randn(T, H, device="cuda"), ids_of(T, K, E, "padded", i).cuda()) for i in range(2)]
    want = [moe_rd.sort_tokens(x, ids, E) for x, ids in data]
    want_back = [moe_rd.unsort_tokens(w.rows, w.inverse_perm) for w in want]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                s = moe_rd.sort_tokens(*data[i], E)
                b = moe_rd.unsort_tokens(s.rows, s.inverse_perm)
                few = moe_rd.sort_tokens(data[i][0][:100], data[i][1][:100], E)
            torch.cuda.current_stream().synchronize()
            if not (all(torch.equal(p, q) for p, q in zip(s, want[i])) and torch.equal(b, want_back[i]) and few.rows.shape == (400, H)):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("T,R", [(0, 0), (0, 5), (3, 0)])
@pytest.mark.parametrize("rows,weights", [(True, True), (True, False), (False, True)])
def test_gradient_of_an_empty_batch_or_of_no_rows(T, R, rows, weights):
    grad, y = torch.ones(T, 64, device="cuda"), torch.ones(R, 64, device="cuda")
    inv, w = torch.full((T, 2), -1, dtype=torch.int32, device="cuda"), torch.ones(T, 2, device="cuda")
    g = moe_rd.unsort_tokens_backward(grad, y, inv, w, need_rows=rows, need_weights=weights)
    assert (g.rows is not None) == rows and (g.weights is not None) == weights
    assert not rows or torch.equal(g.rows, torch.zeros_like(y))
    assert not weights or torch.equal(g.weights, torch.zeros_like(w))
    leaf, lw = y.clone().requires_grad_(), w.clone().requires_grad_()
    moe_rd.unsort_tokens(leaf, inv, lw).sum().backward()
    assert torch.equal(leaf.grad, torch.zeros_like(y)) and torch.equal(lw.grad, torch.zeros_like(w))


def test_results_of_the_sort_are_read_where_they_are():
    """Its parts may start at any multiple of four bytes; passing them on makes no copies."""
    x, ids = torch.randn(5, 64, device="cuda"), torch.arange(10, dtype=torch.int32, device="cuda").view(5, 2) % 4
    s, w = moe_rd.sort_tokens(x, ids, 4), torch.rand(11, device="cuda")[1:].view(5, 2)
    logits = torch.randn(21, device="cuda")[1:].view(5, 4)
    out = moe_rd.unsort_tokens(s.rows, s.inverse_perm, w)
    g = moe_rd.unsort_tokens_backward(x, s.rows, s.inverse_perm, w, offsets=s.offsets)
    r, rg = moe_rd.routing_weights(logits, ids), moe_rd.routing_weights_backward(w, logits, ids)
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    moe_rd.unsort_tokens(s.rows, s.inverse_perm, w, out=out)
    moe_rd.unsort_tokens_backward(x, s.rows, s.inverse_perm, w, offsets=s.offsets, out=g)
    moe_rd.routing_weights(logits, ids, out=r)
    moe_rd.routing_weights_backward(w, logits, ids, out=rg)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    want = sum(w[:, k, None].double() * x.double() for k in range(2))  # every pair's row is its token's
    assert (out.double() - want).abs().max() <= 4 * 2.0 ** -24 * (2 * w.max() * x.abs().max()).item()
    assert torch.equal(r, moe_rd.routing_weights(logits.clone(), ids)) and torch.equal(rg, moe_rd.routing_weights_backward(w, logits.clone(), ids))


@pytest.mark.parametrize("T,K,E,H,dtype,capacity,kind", [
    (1024, 1, 8, 16, "bf16", 0, "random"),        # the last pairs of the smallest blocks
    (1025, 1, 8, 16, "bf16", 7, "stray"),
    (512, 8, 256, 264, "fp16", 0, "padded"),      # of the middle ones
    (4097, 1, 256, 12, "fp32", 0, "stray"),
    (1024, 32, 256, 24, "bf16", 0, "random"),     # the last pairs of the one-kernel form, for few tokens
    (4096, 8, 3, 40, "bf16", 5000, "one expert"),
    (1025, 32, 256, 24, "bf16", 60, "stray"),     # the first of the batch form
    (4097, 8, 16, 72, "fp16", 0, "none"),
    (4097, 4, 16, 72, "fp16", 0, "padded"),
    (6145, 3, 8, 132, "fp32", 0, "stray"),        # one token into a further group of counting tiles
    (16385, 1, 2, 16, "bf16", 9000, "random"),
    (2048, 8, 64, 4096, "bf16", 0, "random"),     # the last bytes of the one-kernel form
    (2049, 8, 64, 4096, "bf16", 0, "random"),
])
def test_sort_is_exact_at_the_borders_of_its_forms(T, K, E, H, dtype, capacity, kind):
    test_sort_is_exact(T, K, E, H, dtype, capacity, kind)


@pytest.mark.parametrize("T,K,E,H,dtype,rows", [
    (1, 2, 4, 8, "bf16", 5),
    (1, 8, 256, 7168, "bf16", 8),
    (37, 4, 16, 264, "fp16", 148),
    (300, 3, 7, 20, "fp32", 2000),          # more rows than pairs
    (4096, 8, 64, 40, "bf16", 32768),
    (20000, 2, 8, 136, "fp16", 50001),
    (30001, 3, 8, 8, "bf16", 32768 * 64 + 1),   # more blocks that look for rows without a pair
    (3, 2, 4, 8, "bf16", 32768 * 256),          # the last number of rows that they take
    (30001, 3, 8, 8, "fp16", 32768 * 256 + 1),  # the first that they do not
])
@pytest.mark.parametrize("with_offsets", [True, False])
def test_gradient_of_rows_that_lost_their_pair(T, K, E, H, dtype, rows, with_offsets):
    """Pairs taken out of inverse_perm after the sort leave rows below offsets[-1] that nobody has: their gradient is zero."""
    g = torch.Generator().manual_seed(T + K)
    s = moe_rd.sort_tokens(torch.randn(T, H, generator=g).to(DT[dtype]).cuda(), ids_of(T, K, E, "padded").cuda(), E)
    inv = s.inverse_perm.clone()
    inv[torch.rand(T, K, generator=g).cuda() < 0.4] = -1
    inv[:, 0] = torch.where(inv[:, 0] % 5 == 0, 2 ** 31 - 1, inv[:, 0])   # an index outside the rows is a pair without one
    y = torch.zeros(rows, H, dtype=DT[dtype], device="cuda")
    grad = torch.randn(T, H, generator=g).to(DT[dtype]).cuda()
    has = (inv >= 0) & (inv < rows)
    offsets = s.offsets if with_offsets else None
    if with_offsets and T > 100:            # a row from offsets[-1] on is nobody's, whatever a pair says
        offsets = offsets - 13
        has &= inv < offsets[-1]
    want = torch.zeros_like(y)
    want[inv[has].long()] = grad[:, None, :].expand(T, K, H)[has]      # weights of 1: not rounded
    out = moe_rd.UnsortGradients(torch.full_like(y, float("nan")), None)
    got = moe_rd.unsort_tokens_backward(grad, y, inv, offsets=offsets, out=out)
    assert got is out and torch.equal(got.rows, want)
    ones = torch.ones(T, K, device="cuda")
    both = moe_rd.unsort_tokens_backward(grad, y, inv, ones, offsets=offsets,
                                         out=moe_rd.UnsortGradients(torch.full_like(y, float("nan")), torch.full_like(ones, float("nan"))))
    assert torch.equal(both.rows, want) and torch.equal(both.weights, torch.zeros_like(ones))
    leaf = y.requires_grad_()
    moe_rd.unsort_tokens(leaf, inv, ones, offsets=offsets).backward(grad)
    assert torch.equal(leaf.grad, want)


def test_gradient_of_rows_without_a_pair_replayed_for_other_places():
    """A recorded gradient clears the rows of the places that it finds, not of those that it was recorded with."""
    for T, K, H, more in ((50, 2, 64, 0), (20000, 2, 16, 0), (5000, 2, 4, 32768 * 64), (7, 2, 4, 32768 * 256)):
        grad, y = torch.randn(T, H, device="cuda"), torch.zeros(T * K + more, H, device="cuda")
        inv = torch.arange(T * K, dtype=torch.int32, device="cuda").view(T, K)
        offsets = torch.tensor([0, T * K], dtype=torch.int32, device="cuda")
        out = moe_rd.unsort_tokens_backward(grad, y, inv, offsets=offsets)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            moe_rd.unsort_tokens_backward(grad, y, inv, offsets=offsets, out=out)
        for shift in (0, 1, 7):
            inv.copy_(torch.arange(T * K, dtype=torch.int32, device="cuda").view(T, K).roll(shift) - shift)
            graph.replay()
            want = torch.zeros_like(y)
            has = inv >= 0
            want[inv[has].long()] = grad[:, None, :].expand(T, K, H)[has]
            assert torch.equal(out.rows, want)


@pytest.mark.parametrize("leaf", [True, False])
def test_what_the_sort_returns_may_be_changed_part_by_part(leaf):
    """Counts and tokens of rows are the caller's to change in place; the places, which the graph has saved, are not."""
    for part in ("row_token", "counts", "inverse_perm"):
        x = torch.randn(50, 64, device="cuda", requires_grad=leaf)
        ids = ids_of(50, 2, 8, "padded").cuda()
        s = moe_rd.sort_tokens(x, ids, 8)
        y = s.rows if leaf else s.rows.requires_grad_()
        places = [t.clone() for t in (s.inverse_perm, s.offsets)]
        out = moe_rd.unsort_tokens(y, s.inverse_perm, offsets=s.offsets)
        getattr(s, part).add_(1)
        if part == "inverse_perm":
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()
            continue
        out.sum().backward()
        assert torch.equal(s.inverse_perm, places[0]) and torch.equal(s.offsets, places[1])
        n = (ids >= 0).sum(1, keepdim=True).float()
        want = n.expand(50, 64) if leaf else (torch.arange(100, device="cuda") < s.offsets[-1])[:, None].float().expand(100, 64)
        assert torch.equal(x.grad if leaf else y.grad, want)
