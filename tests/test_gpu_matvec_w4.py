"""Products of few rows with 4-bit expert weights against the formula in 64 bits."""
import pytest
import torch

import moe_rd

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
TINY = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25}


def make(E, N, K, group, dtype, zeros, seed=0):
    g = torch.Generator().manual_seed(seed + N + K)
    q = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=torch.uint8)
    s = ((torch.rand(E, N, K // group, generator=g) + 0.1) / 64).to(DT[dtype])
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    w = torch.stack([q & 15, q >> 4], -1).reshape(E, N, K // group, group).double()
    w = ((w - (8.0 if z is None else z[..., None].double())) * s[..., None].double()).reshape(E, N, K)
    return q, s, z, w


def check(x, w, offsets, got, dtype, K):
    want = torch.zeros(got.shape, dtype=torch.float64)
    mag = torch.zeros_like(want)
    for e in range(w.shape[0]):
        lo, hi = offsets[e], offsets[e + 1]
        want[lo:hi] = x[lo:hi].double() @ w[e].t()
        mag[lo:hi] = x[lo:hi].double().abs() @ w[e].t().abs()
    # a matrix instruction adds 16 exact products to its sum, each addend within a unit of 2^-24 of the largest: 17; eight to
    # a group's part; then one product and one addition per 32 inputs of the row, and 16 warps
    low = (8 * 17 + 2 * (K / 32) + 16) * 2.0 ** -24 * mag
    bound = low + HALF_STEP[dtype] * (want.abs() + low) + TINY[dtype]
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # the roundings to the result's type alone may be half a step everywhere; they average 0.58 of that
    assert err.norm() <= HALF_STEP[dtype] * want.norm() + TINY[dtype] * err.numel()


CASES = [
    # E, N, K, group, dtype, zeros, rows of every expert
    (1, 16, 32, 32, "bf16", False, [1]),
    (1, 1, 32, 32, "fp16", True, [3]),
    (1, 4101, 4128, 32, "fp16", True, [3]),
    (1, 100, 1056, 96, "bf16", True, [8]),          # groups of 96, inputs that end inside a tile
    (1, 33, 640, 640, "fp16", False, [9]),          # one group per row; nine rows: a second pass
    (4, 50, 256, 64, "bf16", True, [0, 7, 0, 1]),
    (8, 272, 1024, 128, "fp16", False, [1, 0, 16, 2, 0, 0, 25, 3]),
    (256, 48, 384, 128, "bf16", False, [0] * 100 + [1] * 3 + [0] * 152 + [2]),
    (3, 64, 7168, 128, "bf16", False, [1, 1, 1]),
    (2, 16, 128, 32, "bf16", False, [0, 0]),
    # more than eight rows per expert on average: units of sixteen rows
    (1, 70, 4128, 32, "bf16", True, [16]),
    (1, 33, 384, 64, "fp16", False, [9]),
    (1, 200, 1056, 96, "fp16", True, [17]),
    (3, 64, 2048, 128, "bf16", False, [33, 0, 8]),
    (2, 4096, 256, 256, "bf16", True, [1, 40]),
]


@pytest.mark.parametrize("E,N,K,group,dtype,zeros,rows", CASES)
@pytest.mark.parametrize("behind", [0, 5])
def test_expert_products(E, N, K, group, dtype, zeros, rows, behind):
    q, s, z, w = make(E, N, K, group, dtype, zeros)
    offsets = [0]
    for n in rows:
        offsets.append(offsets[-1] + n)
    R = offsets[-1] + behind
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(R)).to(DT[dtype])
    x[offsets[-1]:] = float("nan")      # rows of no expert
    packed = moe_rd.pack_w4(q.cuda(), s.cuda(), None if z is None else z.cuda())
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    got = moe_rd.expert_matvec_w4(x.cuda(), packed, off)
    check(x, w, offsets, got, dtype, K)
    assert (got[offsets[-1]:] == 0).all()
    buf = torch.full_like(got, float("nan"))
    assert moe_rd.expert_matvec_w4(x.cuda(), packed, off, out=buf) is buf and torch.equal(buf, got)
    if E == 1 and behind == 0:
        assert torch.equal(moe_rd.expert_matvec_w4(x.cuda(), packed), got)


@pytest.mark.parametrize("E,N,K", [(1, 1, 32), (3, 45, 160), (2, 64, 1024), (5, 33, 416)])
def test_weights_laid_out_on_the_gpu_and_on_the_cpu_are_the_same(E, N, K):
    q, s, z, _ = make(E, N, K, 32, "bf16", True)
    for a, b in zip(moe_rd.pack_w4(q, s, z), moe_rd.pack_w4(q.cuda(), s.cuda(), z.cuda())):
        assert torch.equal(a, b.cpu()) if isinstance(a, torch.Tensor) else a == b
    wide = torch.zeros(E, N, K // 2 + 3, dtype=torch.uint8).cuda()
    wide[..., 3:] = q.cuda()
    assert torch.equal(moe_rd.pack_w4(wide[..., 3:], s.cuda(), z.cuda()).packed.cpu(), moe_rd.pack_w4(q, s, z).packed)


def test_every_value_and_zero_point_is_exact():
    """One input at a time: the product is the weight itself, for all 16 values and 16 zero points."""
    q = (torch.arange(16).repeat(16, 2) | (torch.arange(16).repeat(16, 2) << 4)).to(torch.uint8)[:, :16]   # K = 32: every value twice
    z = torch.arange(16, dtype=torch.uint8).reshape(16, 1)
    for dtype in (torch.bfloat16, torch.float16):
        packed = moe_rd.pack_w4(q.cuda(), torch.full((16, 1), 0.25, dtype=dtype).cuda(), z.cuda())
        got = moe_rd.expert_matvec_w4(torch.eye(32, dtype=dtype).cuda(), packed)
        value = torch.stack([q & 15, q >> 4], -1).reshape(16, 32).float()
        assert torch.equal(got.float().cpu(), ((value - z.float()) * 0.25).t())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_nan_and_inf_reach_only_their_rows_and_outputs(dtype):
    """An infinity in a row gives what the formula gives: an infinity of the weight's sign, or no number where the weight is
    zero; rows next to it, and values near the end of the range, are as exact as ever."""
    q, s, z, w = make(1, 40, 1152, 64, dtype, True)
    s[0, 7, 1] = float("nan")
    w[0, 7] = float("nan")
    x = torch.randn(7, 1152).to(DT[dtype])
    x[2, 9] = float("inf")
    x[3, 200] = float("nan")
    x[5, 1100] = -float("inf")
    x[6] = torch.finfo(DT[dtype]).max / 4096      # sums near the end of the range
    got = moe_rd.expert_matvec_w4(x.cuda(), moe_rd.pack_w4(q.cuda(), s.cuda(), z.cuda())).cpu()
    keep = torch.arange(40) != 7
    assert torch.isnan(got[:, 7]).all() and torch.isnan(got[3]).all()
    for r, k, sign in ((2, 9, 1.0), (5, 1100, -1.0)):
        inf = torch.full((40,), float("inf"), dtype=torch.float64) * sign * w[0, :, k]
        assert torch.equal(torch.nan_to_num(got[r, keep].double(), nan=7.0), torch.nan_to_num(inf[keep], nan=7.0))
    rows = [0, 1, 4, 6]
    check(x[rows], w[:, keep], [0, 4], got[rows][:, keep], dtype, 1152)


@pytest.mark.parametrize("K,group", [(160, 32), (192, 64), (288, 96)])
def test_an_infinite_scale_next_to_padded_inputs(K, group):
    """The last group's scale is infinite and the last tile has inputs that do not exist."""
    q, s, z, w = make(1, 9, K, group, "fp16", False)
    s[0, 4, -1] = float("inf")
    keep = torch.arange(9) != 4
    x = torch.zeros(2, K, dtype=torch.float16)
    x[:, -1] = 1.0
    got = moe_rd.expert_matvec_w4(x.cuda(), moe_rd.pack_w4(q.cuda(), s.cuda())).cpu()
    assert not torch.isfinite(got[:, 4]).any()      # infinite weights times inputs of zero and one
    check(x, w[:, keep], [0, 2], got[:, keep], "fp16", K)
    # infinite weights of one sign times inputs of one sign: an infinity, and the inputs that do not exist do not spoil it
    q[0, 4] = 0xFF
    got = moe_rd.expert_matvec_w4(torch.ones_like(x).cuda(), moe_rd.pack_w4(q.cuda(), s.cuda())).cpu()
    assert (got[:, 4] == float("inf")).all() and torch.isfinite(got[:, keep]).all()


def test_offsets_that_make_no_sense_give_zeros():
    q, s, _, _ = make(4, 40, 128, 32, "bf16", False)
    p = moe_rd.pack_w4(q.cuda(), s.cuda())
    x = torch.randn(10, 128).to(torch.bfloat16).cuda()
    for off in ([0, 5, 3, 8, 10], [0, 2, 4, 6, 11], [-1, 2, 4, 6, 10], [0, 2 ** 31 - 1, 4, 6, 10], [0, 1, 2, 2, -2 ** 31]):
        got = moe_rd.expert_matvec_w4(x, p, torch.tensor(off, dtype=torch.int32).cuda())
        assert (got == 0).all()
    got = moe_rd.expert_matvec_w4(x, p, torch.tensor([3, 4, 4, 6, 7], dtype=torch.int32).cuda())
    assert (got[:3] == 0).all() and (got[7:] == 0).all() and (got[3:7] != 0).any(1).all()


def test_the_decode_step_of_a_layer():
    """route_dispatch, the two 4-bit products of a gated expert layer, and combine, for one token and for several."""
    E, H, I, K = 16, 256, 128, 4
    up_q, up_s, _, up = make(E, 2 * I, H, 64, "bf16", False, 1)
    dn_q, dn_s, _, dn = make(E, H, I, 32, "bf16", False, 2)
    up_p, dn_p = moe_rd.pack_w4(up_q.cuda(), up_s.cuda()), moe_rd.pack_w4(dn_q.cuda(), dn_s.cuda())
    gate = (torch.randn(H, E, generator=torch.Generator().manual_seed(3)) * 0.1).to(torch.bfloat16)
    for T in (1, 13):
        x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
        r = moe_rd.route_dispatch(x.cuda(), gate.cuda(), top_k=K)
        a = moe_rd.expert_matvec_w4(r.permuted, up_p, r.offsets).float()
        hidden = (torch.nn.functional.silu(a[:, :I]) * a[:, I:]).to(torch.bfloat16)
        out = moe_rd.combine(moe_rd.expert_matvec_w4(hidden, dn_p, r.offsets), r.inverse_perm, r.combine_weights)
        ids, cw = r.expert_ids.cpu().long(), r.combine_weights.cpu().double()
        want = torch.zeros(T, H, dtype=torch.float64)
        mag = torch.zeros_like(want)
        for t in range(T):
            for k in range(K):
                u = up[ids[t, k]] @ x[t].double()
                h = torch.nn.functional.silu(u[:I]) * u[I:]
                want[t] += cw[t, k] * (dn[ids[t, k]] @ h)
                mag[t] += cw[t, k] * (dn[ids[t, k]].abs() @ (h.abs() + u[I:].abs() + u[:I].abs()))
        # roundings to bf16 on the way: the first product (twice, and silu's slope is below 1.1), the hidden value, the
        # second product and the result, each half a step of 2^-8
        assert ((out.cpu().double() - want).abs() <= 5 * 2.0 ** -8 * 1.1 * mag).all()


def test_graph_and_other_stream():
    q, s, z, w = make(8, 100, 512, 128, "bf16", False)
    packed = moe_rd.pack_w4(q.cuda(), s.cuda())
    x = torch.randn(6, 512).to(torch.bfloat16).cuda()
    off = torch.tensor([0, 1, 1, 3, 3, 3, 6, 6, 6], dtype=torch.int32).cuda()
    moe_rd.expert_matvec_w4(x, packed, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = moe_rd.expert_matvec_w4(x, packed, off)
    x.normal_()
    off.copy_(torch.tensor([0, 0, 2, 2, 2, 4, 4, 5, 6], dtype=torch.int32))
    graph.replay()
    assert torch.equal(res.clone(), moe_rd.expert_matvec_w4(x, packed, off))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = moe_rd.expert_matvec_w4(x[:, :], packed, off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, res)
    # rows that are a view: strided, and starting off a 16-byte boundary
    wide = torch.randn(6, 520).to(torch.bfloat16).cuda()
    assert torch.equal(moe_rd.expert_matvec_w4(wide[:, 3:515], packed, off), moe_rd.expert_matvec_w4(wide[:, 3:515].clone(), packed, off))


def test_weights_past_32_bits():
    """More than 2^32 bytes of weights: the last expert's last outputs."""
    E, N, K, group = 130, 8192, 8192, 128
    q = torch.randint(0, 256, (E, N, K // 2), device="cuda", dtype=torch.uint8)
    s = (torch.rand(E, N, K // group, device="cuda") / 64).to(torch.bfloat16)
    packed = moe_rd.pack_w4(q, s)
    assert packed.packed.numel() > 2 ** 32
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = 1
    off[-1] = 3
    x = torch.randn(3, K, device="cuda").to(torch.bfloat16)
    got = moe_rd.expert_matvec_w4(x, packed, off)
    for rows, e in (([0], 0), ([1, 2], E - 1)):
        w = torch.stack([q[e] & 15, q[e] >> 4], -1).reshape(N, K // group, group).double() - 8.0
        w = (w * s[e].double()[..., None]).reshape(N, K)
        want = x[rows].double() @ w.t()
        err = (got[rows].double() - want).abs()
        low = (8 * 17 + 2 * (K / 32) + 16) * 2.0 ** -24 * (x[rows].double().abs() @ w.abs().t())
        assert (err <= low + 2.0 ** -8 * (want.abs() + low)).all()
