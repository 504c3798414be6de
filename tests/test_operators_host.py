"""What the sorting, routing-weight and 4-bit operators refuse, on the CPU: argument checks before any CUDA call, at the
Python functions and at the C entries; and the layout that pack_w4 makes."""
import ctypes

import pytest
import torch

import moe_rd
from moe_rd import _cabi

I32 = torch.int32


def x(*shape, dtype=torch.bfloat16, **kw):
    return torch.zeros(*shape, dtype=dtype, **kw)


def test_sort_refusals():
    ids = x(4, 2, dtype=I32)
    for bad, why in (((x(4, 64, dtype=torch.float64), ids, 8), TypeError), ((x(4, 63), ids, 8), ValueError),
                     ((x(5, 64), ids, 8), ValueError), ((x(4, 64), ids.long(), 8), TypeError),
                     ((x(4, 64), ids[0], 8), ValueError), ((x(4, 64), ids, 0), ValueError), ((x(64), ids, 8), ValueError)):
        with pytest.raises(why):
            moe_rd.sort_tokens(*bad)
    with pytest.raises(ValueError):
        moe_rd.sort_tokens(x(4, 64), ids, 8, capacity=-1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moe_rd.sort_tokens(x(4, 64), ids, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moe_rd.sort_tokens(x(4, 64, requires_grad=True), ids, 8)


def test_unsort_refusals():
    inv, w, y = x(4, 2, dtype=I32), x(4, 2, dtype=torch.float32), x(8, 64)
    for bad, why in (((x(8, 64, dtype=torch.float64), inv), TypeError), ((y, inv.long()), TypeError),
                     ((y, inv, w.double()), TypeError), ((y, inv, w[:3]), ValueError), ((y, inv, w, x(4, 32)), ValueError),
                     ((y, inv, w, x(3, 64)), ValueError), ((y, inv, w, x(4, 64, dtype=torch.float16)), TypeError),
                     ((x(8, 60), inv), ValueError)):
        with pytest.raises(why):
            moe_rd.unsort_tokens(*bad)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moe_rd.unsort_tokens(y, inv, w)
    g = x(4, 64)
    with pytest.raises(ValueError):
        moe_rd.unsort_tokens_backward(g, y, inv, w, need_rows=False, need_weights=False)
    with pytest.raises(ValueError):
        moe_rd.unsort_tokens_backward(g[:3], y, inv, w)
    with pytest.raises(TypeError):
        moe_rd.unsort_tokens_backward(g.half(), y, inv, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moe_rd.unsort_tokens_backward(g, y, inv, w)


def test_routing_weight_refusals():
    lg, ids = x(4, 8, dtype=torch.float32), x(4, 2, dtype=I32)
    for args, kw, why in (((lg.double(), ids), {}, TypeError), ((lg, ids.long()), {}, TypeError), ((lg[:3], ids), {}, ValueError),
                          ((lg, ids, lg[0, :7]), {}, ValueError), ((lg, ids), dict(score_fn="relu"), ValueError),
                          ((lg, ids), dict(bias_mode="x"), ValueError),
                          ((lg, ids, lg[0].clone().requires_grad_()), {}, ValueError), ((lg, ids), {}, RuntimeError)):
        with pytest.raises(why):
            moe_rd.routing_weights(*args, **kw)
    with pytest.raises(ValueError):
        moe_rd.routing_weights_backward(lg, lg, ids)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moe_rd.routing_weights_backward(x(4, 2, dtype=torch.float32), lg, ids)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pack_w4_layout_and_refusals(dtype):
    E, N, K, group = 2, 45, 160, 32
    g = torch.Generator().manual_seed(1)
    q = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=torch.uint8)
    s = torch.rand(E, N, K // group, generator=g).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8)
    p = moe_rd.pack_w4(q, s, z)
    assert (p.N, p.K, p.group) == (N, K, group) and p.packed.shape == (E, 2, 2, 2048) and p.scales.shape == (E, 2, 5, 8, 4)
    value = torch.stack([q & 15, q >> 4], -1).reshape(E, N, K)
    for e, n, k in [(0, 0, 0), (0, 0, 1), (1, 44, 159), (0, 7, 31), (1, 8, 32), (0, 15, 127), (1, 16, 128), (0, 29, 77), (0, 43, 6)]:
        b, c, part, r = n // 32, k // 128, (n % 32) // 8, n % 8
        m, j, kk = (k % 128) // 32, (k % 32) // 8, k % 8
        at = part * 512 + (4 * r + j) * 16 + 4 * m
        word = int.from_bytes(bytes(p.packed[e, b, c, at:at + 4].tolist()), "little")
        assert (word >> (4 * (kk // 2) + 16 * (kk % 2))) & 15 == int(value[e, n, k])
        assert p.scales[e, b, k // group, r, part] == s[e, n, k // group]
        word = int.from_bytes(bytes(p.zeros[e, b, k // group, r].tolist()), "little")
        assert (word >> (4 * part)) & 15 == int(z[e, n, k // group])
    assert (p.scales[:, 1, :, 5:, 1] == 0).all() and (p.scales[:, 1, :, :, 2:] == 0).all()     # outputs past N
    assert int(p.packed[:, 1, :, 1024:].sum()) == 0
    one = moe_rd.pack_w4(q[0], s[0], z[0])
    assert all(torch.equal(a, b[:1]) for a, b in zip(one[:3], p[:3]))
    for args, why in (((q.int(), s), TypeError), ((q, s.float()), TypeError), ((q, s[:, :20]), ValueError), ((q, s[..., :3]), ValueError),
                      ((q, s, z[..., :4]), ValueError), ((q, s, z.int()), ValueError), ((q, s, z | 16), ValueError),
                      ((q[..., :8], s[..., :1]), ValueError)):
        with pytest.raises(why):
            moe_rd.pack_w4(*args)
    rows = x(3, K, dtype=dtype)
    off = torch.tensor([0, 1, 3], dtype=I32)
    for args, why in (((rows, q), TypeError), ((rows.float(), p, off), TypeError), ((rows.to(torch.float16 if dtype == torch.bfloat16 else torch.bfloat16), p, off), TypeError),
                      ((rows[:, :128], p, off), ValueError), ((rows, p), ValueError), ((rows, p, off[:2]), ValueError),
                      ((rows, p, off.long()), TypeError), ((rows.requires_grad_(), p, off), RuntimeError),
                      ((rows.detach(), p._replace(packed=p.packed[:, :1]), off), ValueError), ((rows.detach(), p, off), RuntimeError)):
        with pytest.raises(why):
            moe_rd.expert_matvec_w4(*args)


def test_c_entries_validate_before_any_cuda_call():
    L = _cabi.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255
    n = ctypes.c_size_t(7)

    def ws(T, H=64, E=256, K=8, dtype=0, to=ctypes.byref(n)):
        return L.moe_rd_sort_workspace_bytes(T, H, E, K, dtype, to)
    # one kernel, without a workspace, up to 32768 pairs of 4096 tokens; then tiles of 64 tokens and groups of 32 tiles
    assert ws(1) == 0 and n.value == 0 and ws(4096) == 0 and n.value == 0
    assert ws(4097) == 0 and n.value == 256 * 4 * 65 + 256 * 4 * 3
    assert ws(2048, H=7168) == 0 and n.value == 256 * 4 * 32 + 256 * 4 and ws(2 ** 31 - 1, K=1, E=1) == 0
    assert ws(1, E=257) == ws(1, K=33) == ws(2 ** 31, K=1) == ws(1, H=12) == -2 and ws(1, dtype=3) == -6 and ws(1, to=None) == -1
    assert ws(2 ** 30, K=1) == -10      # 2^24 tiles x 256 experts are not counted in 32 bits

    def sort(T=4, H=64, E=8, K=2, dtype=0, cap=0, R=8, ptrs=(p,) * 7, ws=0, bytes_=0):
        return L.moe_rd_sort_tokens(T, H, E, K, dtype, cap, R, *ptrs, ws, bytes_, None)
    assert sort(H=60) == sort(H=0) == sort(E=0) == sort(K=0) == sort(T=-1) == sort(R=7) == sort(cap=-1) == -2
    assert sort(H=62, dtype=2) == -2 and sort(dtype=3) == -6
    assert sort(cap=1, R=7) == -2           # 8 experts of one row each
    for i in (0, 1, 2, 3, 4, 5):
        assert sort(ptrs=tuple(0 if j == i else p for j in range(7))) == -1
    assert sort(ptrs=(p + 8,) + (p,) * 6) == -4
    assert sort(T=9000, R=18000) == sort(T=9000, R=18000, ws=p, bytes_=16) == sort(T=9000, R=18000, ws=p + 16, bytes_=1 << 20) == -5

    def unsort(T=4, H=64, K=2, dtype=0, R=8, ptrs=(p, p, p, p, p)):
        return L.moe_rd_unsort_tokens(T, H, K, dtype, ptrs[0], R, *ptrs[1:], None)
    assert unsort(H=63) == unsort(K=33) == unsort(R=-1) == unsort(T=-1) == -2 and unsort(dtype=-1) == -6
    assert unsort(ptrs=(0, p, p, p, p)) == unsort(ptrs=(p, 0, p, p, p)) == unsort(ptrs=(p, p, p, p, 0)) == -1
    assert unsort(ptrs=(p, p, p, p + 4, p)) == -4 and unsort(T=0, ptrs=(0,) * 5) == 0

    def back(T=4, H=64, K=2, dtype=0, R=8, g=p, y=p, inv=p, w=p, n=p, gy=p, gw=p):
        return L.moe_rd_unsort_tokens_backward(T, H, K, dtype, g, y, R, inv, w, n, gy, gw, None)
    assert back(H=63) == back(K=0) == -2 and back(dtype=9) == -6
    assert back(g=0) == back(y=0) == back(inv=0) == back(gy=0, gw=0) == -1 and back(gy=p + 2) == -4
    assert back(T=0, R=0, g=0, y=0, inv=0) == 0

    def rw(T=4, E=8, K=2, fn=0, ptrs=(p,) * 5):
        return L.moe_rd_routing_weights(T, E, K, fn, 1, 1.0, 0.0, *ptrs, None)
    assert rw(E=257) == rw(K=33) == rw(T=-1) == rw(E=0) == -2 and rw(fn=2) == -6
    assert rw(ptrs=(0, p, p, p, p)) == rw(ptrs=(p, 0, p, p, p)) == rw(ptrs=(p, p, p, p, 0)) == -1 and rw(T=0, ptrs=(0,) * 5) == 0
    assert L.moe_rd_routing_weights_backward(4, 8, 2, 0, 1, 1.0, 0.0, p, p, None, None, None, p, None) == -1

    def mv(R=4, N=16, K=64, E=2, group=32, dtype=0, ptrs=(p, p, p, None, p, p)):
        return L.moe_rd_expert_matvec_w4(R, N, K, E, group, dtype, *ptrs, None)
    assert mv(N=0) == mv(K=48) == mv(group=48) == mv(group=16) == mv(E=257) == mv(R=-1) == mv(K=0) == -2
    assert mv(ptrs=(p, p, p, None, None, p)) == -2       # two experts need offsets
    assert mv(dtype=2) == -8 and mv(dtype=5) == -6 and mv(R=0, ptrs=(0,) * 6, E=1) == 0
    assert mv(ptrs=(0, p, p, None, p, p)) == mv(ptrs=(p, p, p, None, p, 0)) == -1
    assert mv(ptrs=(p + 2, p, p, None, p, p)) == mv(ptrs=(p, p + 8, p, None, p, p)) == mv(ptrs=(p, p, p, None, p, p + 1)) == -4

    def pack(E=1, N=8, K=64, q=p, w=p):
        return L.moe_rd_pack_w4(E, N, K, q, w, None)
    assert pack(E=0) == pack(E=257) == pack(N=0) == pack(K=48) == pack(K=0) == -2
    assert pack(q=0) == pack(w=0) == -1 and pack(q=p + 4) == pack(w=p + 8) == -4


def test_capturing_is_refused_where_a_gradient_is_wanted(monkeypatch):
    from moe_rd import sorting
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="not recorded into a CUDA graph"):
        sorting._not_while_capturing("sort_tokens", "unsort_tokens")


def test_the_compiled_calls_leave_everything_else_to_python():
    from moe_rd import _cabi
    _cabi.lib()
    assert not isinstance(_cabi.fast, _cabi._NotLoaded), "moe_rd/_fastcall.so is not built"
    x, ids, w = torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1)
    f = _cabi.fast
    for args in ((), (x,), (x, ids, 4, 0, None), (None,) * 5, (x, ids, "4", 0, None), (1, 2, 3, 4, 5)):
        assert f.sort_tokens(*args) is False
    for args in ((), (x, ids, w, None, None, None), (None,) * 6):
        assert f.unsort_tokens(*args) is False
    for args in ((), (x, x, ids, w, None, True, True, None), (None,) * 8):
        assert f.unsort_tokens_backward(*args) is False
    for args in ((), (None, w, ids, None, 0, 0, True, 1.0, 1e-20, None), (None,) * 10):
        assert f.routing_weights(*args) is False
    for args in ((), (x, (1, 2, 3, 4, 5, 6), None, None), (x, (None,) * 6, None, None), (None,) * 4):
        assert f.expert_matvec_w4(*args) is False


def test_tangents_of_forward_mode_are_refused():
    import torch.autograd.forward_ad as fwad
    rows, ids, w = x(4, 64), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2)
    y, logits, bias = x(8, 64), torch.zeros(4, 8), torch.zeros(8)
    p = moe_rd.pack_w4(torch.zeros(40, 32, dtype=torch.uint8), torch.ones(40, 2).bfloat16())
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))
        calls = (lambda: moe_rd.sort_tokens(dual(rows), ids, 8), lambda: moe_rd.unsort_tokens(dual(y), ids), lambda: moe_rd.unsort_tokens(y, ids, dual(w)),
                 lambda: moe_rd.unsort_tokens(y, ids, w, dual(rows)), lambda: moe_rd.unsort_tokens_backward(dual(rows), y, ids, w),
                 lambda: moe_rd.unsort_tokens_backward(rows, dual(y), ids, w), lambda: moe_rd.unsort_tokens_backward(rows, y, ids, dual(w)),
                 lambda: moe_rd.routing_weights(dual(logits), ids), lambda: moe_rd.routing_weights(logits, ids, dual(bias)),
                 lambda: moe_rd.routing_weights_backward(dual(w), logits, ids), lambda: moe_rd.routing_weights_backward(w, dual(logits), ids),
                 lambda: moe_rd.expert_matvec_w4(dual(rows), p))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_a_module_of_another_torch_is_not_loaded_and_is_built_anew(monkeypatch, tmp_path):
    import shutil
    import subprocess
    from moe_rd import _build
    L = _cabi.lib()
    assert _cabi._load_fast(L) is _cabi.fast                         # compiled for this one
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    with pytest.warns(UserWarning, match="rebuild"):
        assert isinstance(_cabi._load_fast(L), _cabi._NotLoaded)
    there = tmp_path / "_fastcall.so"
    shutil.copy2(_build.FASTCALL, there)
    monkeypatch.setattr(_build, "FASTCALL", there)
    built = []

    def run(cmd, **kw):
        built.append(cmd)
        raise InterruptedError
    monkeypatch.setattr(subprocess, "run", run)
    with pytest.raises(InterruptedError):
        _build.build_fastcall()
    assert any("1.0.0+other" in a for a in built[0])
    monkeypatch.undo()
    assert _build.build_fastcall() == _build.FASTCALL


@pytest.mark.parametrize("why", ["compiler", "headers"])
def test_the_library_is_built_where_the_module_cannot_be(monkeypatch, tmp_path, why):
    import subprocess
    from moe_rd import _build
    monkeypatch.setattr(_build, "FASTCALL", tmp_path / "_fastcall.so")
    (tmp_path / "_fastcall.so").write_bytes(b"of other sources")
    run = subprocess.run

    def without(cmd, **kw):
        if "nvcc" in cmd[0]:
            return run(cmd, **kw)
        if why == "compiler":
            raise FileNotFoundError("g++")
        return subprocess.CompletedProcess(cmd, 1, "", "torch/csrc/autograd/python_variable.h: No such file")
    monkeypatch.setattr(subprocess, "run", without)
    with pytest.warns(UserWarning, match="_fastcall.so is not built"):
        assert _build.build() == _build.LIB and _build.LIB.exists()
    assert list(tmp_path.iterdir()) == []
    assert isinstance(_cabi._load_fast(_cabi.lib()), _cabi._NotLoaded)
