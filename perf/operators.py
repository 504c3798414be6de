"""Cases of the operators around the routing: sorting tokens by expert and back with weights (and both gradients),
the routing weights with their gradient, and products with 4-bit expert weights.

A case names one direction of one operator ("op"), its sizes and its types.  ``own`` chooses between the plain form,
written with elementary torch operations in 32 bits and rounded once, and the calls of this package."""
import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


@functools.cache
def _moe_rd():
    import sys
    from pathlib import Path
    package = str(Path.cwd() / "ernie-evolve-results_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import moe_rd
    return moe_rd


def listed():
    return [
        # one decoded token on its way to 8 of 256 experts: pure latency
        dict(name="sort one token", op="sort", T=1, H=7168, E=256, K=8, dtype="bf16", padded=0.0, factor=0.0),
        # the batch of the 256-expert configuration
        dict(name="sort batch", op="sort", T=8192, H=7168, E=256, K=8, dtype="bf16", padded=0.0, factor=0.0),
        # a padded batch in 32 bits with capacity drops: a ragged token count, rows left without a token
        dict(name="sort padded capacity", op="sort", T=4099, H=1004, E=8, K=2, dtype="fp32", padded=0.2, factor=1.0),
        # the gradient of the sort at the 128-expert configuration's size, half precision
        dict(name="sort gradient", op="sort_grad", T=32768, H=2048, E=128, K=8, dtype="fp16", padded=0.0, factor=1.25),
        # a handful of decoded tokens on their way back, with a shared expert
        dict(name="unsort few tokens", op="unsort", T=5, H=7168, E=256, K=8, dtype="bf16", padded=0.0, factor=0.0, shared=True),
        # the 8-expert configuration on its way back, half precision
        dict(name="unsort batch", op="unsort", T=16384, H=4096, E=8, K=2, dtype="fp16", padded=0.0, factor=0.0, shared=False),
        # the gradients of rows and weights for the 256-expert configuration
        dict(name="unsort gradient batch", op="unsort_grad", T=8192, H=7168, E=256, K=8, dtype="bf16", padded=0.0, factor=0.0),
        # the router's gradient: softmax scores, the 128-expert configuration
        dict(name="weights gradient softmax", op="weights_grad", T=32768, E=128, K=8, score_fn="softmax", bias=False),
        # the routing weights of a decode batch: sigmoid scores, a correction bias in the weights
        dict(name="weights sigmoid", op="weights", T=67, E=256, K=8, score_fn="sigmoid", bias=True),
        # one decoded token through the 4-bit weights of its 8 experts
        dict(name="w4 experts one token", op="w4", T=1, N=2048, K=7168, E=256, top=8, group=128, dtype="bf16", zeros=False),
        # a decode batch: most experts have one row, some have several
        dict(name="w4 experts 16 tokens", op="w4", T=16, N=2048, K=7168, E=256, top=8, group=128, dtype="bf16", zeros=False),
        # one dense matrix (a shared expert) for three rows: an odd number of outputs, small groups with zero points
        dict(name="w4 dense zero points", op="w4", T=3, N=4101, K=4128, E=1, top=1, group=32, dtype="fp16", zeros=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "sort", "sort_grad", "unsort", "unsort_grad", "weights", "weights_grad", "w4", "w4"])
    if op == "w4":
        E = rng.choice([1, 1, 8, 64, 128, 256])
        T, group, top = _log(rng, 1, 16), rng.choice([32, 64, 128]), min(E, rng.choice([1, 2, 4, 8]))
        K = group * max(1, _log(rng, 256, 7168) // group)
        most = 8192 if E == 1 else min(2048, 16 * 8 * 2048 * 7168 // (T * top * K))
        return dict(op=op, T=T, N=_log(rng, 64, most), K=K, E=E, top=top, group=group, dtype=rng.choice(["bf16", "fp16"]),
                    zeros=rng.random() < 0.5)
    E = rng.choice([4, 8, 16, 60, 64, 128, 160, 256])
    K = min(E, rng.choice([1, 2, 3, 4, 6, 8, 10]))
    if op.startswith("weights"):
        return dict(op=op, T=_log(rng, 1, 32768), E=E, K=K, score_fn=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    H = 8 * _log(rng, 8, 896)
    most = max(1, min(32768, 8192 * 8 * 7168 * 2 // (K * H * SIZE[dtype])))
    case = dict(op=op, T=_log(rng, 1, most), H=H, E=E, K=K, dtype=dtype, padded=rng.choice([0.0, 0.0, 0.3]),
                factor=rng.choice([0.0, 0.0, 1.0, 1.25]))
    if op == "unsort":
        case["shared"] = rng.random() < 0.5
    return case


def _capacity(case):
    f = case["factor"]
    return int(math.ceil(f * case["T"] * case["K"] / case["E"])) if f else 0


def _rows(case):
    cap = _capacity(case)
    pairs = case["T"] * case["K"]
    return min(pairs, case["E"] * cap) if cap else pairs


def _routing(T, E, K, gen):
    """Router logits whose experts are unevenly popular, and every token's K experts."""
    popular = 2.0 / (1.0 + torch.randperm(E, generator=gen, device="cuda").float())
    logits = torch.randn(T, E, generator=gen, device="cuda") + popular
    return logits, torch.topk(logits, K, dim=1).indices.to(torch.int32)


def _places(ids, E, capacity):
    """Expert of every pair (E where it has none), counts before drops, offsets, and every pair's row (-1: none), in
    the stable (token, slot) order."""
    flat = ids.reshape(-1).long()
    expert = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    order = torch.argsort(expert, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).index_add_(0, expert, torch.ones_like(expert))
    first = torch.cumsum(counts, 0) - counts
    rank = torch.empty_like(expert).index_copy_(0, order, torch.arange(expert.numel(), device=ids.device) - first[expert[order]])
    kept = counts[:E].clamp(max=capacity) if capacity else counts[:E]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=ids.device), torch.cumsum(kept, 0)])
    has_row = expert < E
    if capacity:
        has_row = has_row & (rank < capacity)
    row = torch.where(has_row, offsets[expert.clamp(max=E - 1)] + rank, torch.full_like(rank, -1))
    return counts[:E].to(torch.int32), offsets.to(torch.int32), row.reshape(ids.shape).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "w4":
        E, N, K, T = case["E"], case["N"], case["K"], case["T"]
        dtype = DTYPES[case["dtype"]]
        state["q"] = torch.randint(0, 256, (E, N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
        state["scales"] = ((0.5 + torch.rand(E, N, K // case["group"], generator=gen, device="cuda")) / (4.6 * math.sqrt(K))).to(dtype)
        state["zeros"] = (torch.randint(0, 16, state["scales"].shape, generator=gen, device="cuda", dtype=torch.uint8)
                          if case["zeros"] else None)
        if E > 1:
            ids = _routing(T, E, case["top"], gen)[1]
            state["offsets"] = _places(ids, E, 0)[1]
        else:
            state["offsets"] = None
        state["x"] = torch.randn(T * case["top"], K, generator=gen, device="cuda").to(dtype)
        if own:  # the weights' layout is made once, when a program loads them
            state["weights"] = _moe_rd().pack_w4(state["q"], state["scales"], state["zeros"])
        return state
    T, E, K = case["T"], case["E"], case["K"]
    logits, ids = _routing(T, E, K, gen)
    if case["op"].startswith("weights"):
        state["logits"], state["ids"] = logits, ids
        state["bias"] = 0.1 * torch.randn(E, generator=gen, device="cuda") if case["bias"] else None
        state["grad"] = torch.randn(T, K, generator=gen, device="cuda")
        return state
    if case["padded"]:
        ids[torch.rand(T, generator=gen, device="cuda") < case["padded"]] = -1
    dtype, H, R = DTYPES[case["dtype"]], case["H"], _rows(case)
    state["capacity"] = _capacity(case)
    if case["op"] == "sort":
        state["ids"] = ids
        state["x"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype)
        return state
    _, state["offsets"], state["inverse_perm"] = _places(ids, E, state["capacity"])
    state["rows"] = torch.randn(R, H, generator=gen, device="cuda").to(dtype)
    chosen = torch.gather(logits, 1, ids.clamp(min=0).long())
    state["weights"] = torch.softmax(chosen, 1)
    if case["op"] == "unsort":
        state["shared"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype) if case["shared"] else None
    if case["op"] == "unsort_grad":
        state["grad"] = torch.randn(T, H, generator=gen, device="cuda").to(dtype)
    return state


def _score_args(state):
    return dict(bias=state["bias"], bias_mode="select_and_weight", score_fn=state["score_fn"], renorm=True,
                routed_scale=2.5 if state["score_fn"] == "sigmoid" else 1.0, norm_min=1e-20)


def run(state):
    if own:
        return _run_own(state)
    return globals()["_plain_" + state["op"]](state)


def _run_own(s):
    m, op = _moe_rd(), s["op"]
    out = s.get("out")  # a loop keeps the buffers of its first pass
    if op == "sort":
        s["out"] = r = m.sort_tokens(s["x"], s["ids"], s["E"], capacity=s["capacity"], out=out)
        return r.rows, r.offsets, r.inverse_perm, r.row_token, r.counts
    if op == "sort_grad":
        s["out"] = m.unsort_tokens(s["rows"], s["inverse_perm"], out=out)
    elif op == "unsort":
        s["out"] = m.unsort_tokens(s["rows"], s["inverse_perm"], s["weights"], s["shared"], out=out)
    elif op == "unsort_grad":
        s["out"] = m.unsort_tokens_backward(s["grad"], s["rows"], s["inverse_perm"], s["weights"], offsets=s["offsets"], out=out)
    elif op == "weights":
        s["out"] = m.routing_weights(s["logits"], s["ids"], **_score_args(s), out=out)
    elif op == "weights_grad":
        s["out"] = m.routing_weights_backward(s["grad"], s["logits"], s["ids"], **_score_args(s), out=out)
    else:
        s["out"] = m.expert_matvec_w4(s["x"], s["weights"], s["offsets"], out=out)
    return s["out"]


def _plain_sort(s):
    x, ids = s["x"], s["ids"]
    T, K = ids.shape
    R = _rows(s)
    counts, offsets, inverse_perm = _places(ids, s["E"], s["capacity"])
    row = torch.where(inverse_perm < 0, torch.full_like(inverse_perm, R), inverse_perm).reshape(-1).long()
    token = torch.arange(T * K, device=x.device) // K
    row_token = torch.full((R + 1,), -1, dtype=torch.int32, device=x.device)
    row_token[row] = token.to(torch.int32)
    row_token = row_token[:R]
    rows = torch.where((row_token < 0)[:, None], torch.zeros((), dtype=x.dtype, device=x.device), x[row_token.clamp(min=0).long()])
    return rows, offsets, inverse_perm, row_token, counts


def _gathered(rows, inverse_perm):
    """The row of every pair in 32 bits; zeros where it has none."""
    found = rows[inverse_perm.clamp(min=0).long()].float() if rows.shape[0] else rows.new_zeros((*inverse_perm.shape, rows.shape[1])).float()
    return torch.where((inverse_perm < 0)[..., None], torch.zeros((), device=rows.device), found)


def _plain_sort_grad(s):
    return _gathered(s["rows"], s["inverse_perm"]).sum(1).to(s["rows"].dtype)


def _plain_unsort(s):
    total = (s["weights"][..., None] * _gathered(s["rows"], s["inverse_perm"])).sum(1)
    if s["shared"] is not None:
        total = total + s["shared"].float()
    return total.to(s["rows"].dtype)


def _plain_unsort_grad(s):
    rows, inverse_perm, grad = s["rows"], s["inverse_perm"], s["grad"].float()
    R = rows.shape[0]
    grad_weights = (_gathered(rows, inverse_perm) * grad[:, None, :]).sum(2)
    each = (s["weights"][..., None] * grad[:, None, :]).to(rows.dtype).reshape(-1, rows.shape[1])
    grad_rows = torch.zeros((R + 1, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    grad_rows[torch.where(inverse_perm < 0, torch.full_like(inverse_perm, R), inverse_perm).reshape(-1).long()] = each
    return grad_rows[:R], grad_weights


def _plain_scores(s):
    """Scores of all experts, what the weights are made of (score plus bias) at the chosen ones, and its clamped sum."""
    a = _score_args(s)
    z = s["logits"]
    if a["score_fn"] == "softmax":
        e = torch.exp(z - z.max(1, keepdim=True).values)
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-z))
    key = score if a["bias"] is None else score + a["bias"]
    u = torch.gather(key, 1, s["ids"].long())
    return a, score, u, u.sum(1, keepdim=True)


def _plain_weights(s):
    a, _, u, total = _plain_scores(s)
    return a["routed_scale"] * (u / total.clamp(min=a["norm_min"]))


def _plain_weights_grad(s):
    a, score, u, total = _plain_scores(s)
    g = a["routed_scale"] * s["grad"]
    below = total.clamp(min=a["norm_min"])
    grad_u = (g - torch.where(total >= a["norm_min"], (g * u).sum(1, keepdim=True) / below, torch.zeros_like(total))) / below
    grad_score = torch.zeros_like(score).scatter_add_(1, s["ids"].long(), grad_u)
    if a["score_fn"] == "softmax":
        return score * (grad_score - (score * grad_score).sum(1, keepdim=True))
    return score * (1.0 / (1.0 + torch.exp(s["logits"]))) * grad_score


def _plain_w4(s):
    x, q = s["x"], s["q"]
    R, E, (N, half) = x.shape[0], s["E"], q.shape[1:]
    if s["offsets"] is None:
        expert = torch.zeros(R, dtype=torch.int64, device=x.device)
    else:
        expert = torch.searchsorted(s["offsets"][1:].contiguous(), torch.arange(R, dtype=torch.int32, device=x.device), right=True)
    if E == 1:
        q, scales, zeros = q[0], s["scales"][0], None if s["zeros"] is None else s["zeros"][0]
    else:
        q, scales, zeros = q[expert], s["scales"][expert], None if s["zeros"] is None else s["zeros"][expert]
    w = torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1, s["group"]).float()
    w = (w - (8.0 if zeros is None else zeros.float()[..., None])) * scales.float()[..., None]
    w = w.reshape(*q.shape[:-1], 2 * half)
    y = x.float() @ w.t() if E == 1 else torch.bmm(w, x.float()[..., None])[..., 0]
    return y.to(x.dtype)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sort":
        lists = [[] for _ in range(case["E"])]  # a walk over the pairs on the host
        for t, chosen in enumerate(s["ids"].tolist()):
            for e in chosen:
                if 0 <= e < case["E"] and not (s["capacity"] and len(lists[e]) >= s["capacity"]):
                    lists[e].append(t)
        token = [t for of in lists for t in of]
        rows = torch.zeros((_rows(s), case["H"]), dtype=torch.float64, device="cuda")
        rows[: len(token)] = s["x"].double()[torch.tensor(token, dtype=torch.int64, device="cuda")]
        return rows, None, None, None, None
    if op in ("sort_grad", "unsort"):
        total = s["shared"].double() if op == "unsort" and s["shared"] is not None else torch.zeros(
            (case["T"], case["H"]), dtype=torch.float64, device="cuda")
        total = total.clone()
        for k in range(case["K"]):
            at = s["inverse_perm"][:, k].long()
            has = at >= 0
            part = s["rows"][at[has]].double()
            total[has] += part if op == "sort_grad" else s["weights"][has, k, None].double() * part
        return total
    if op == "unsort_grad":
        grad = s["grad"].double()
        grad_rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
        grad_weights = torch.zeros((case["T"], case["K"]), dtype=torch.float64, device="cuda")
        for k in range(case["K"]):
            at = s["inverse_perm"][:, k].long()
            has = at >= 0
            grad_rows[at[has]] = s["weights"][has, k, None].double() * grad[has]
            grad_weights[has, k] = (s["rows"][at[has]].double() * grad[has]).sum(1)
        return grad_rows, grad_weights
    if op in ("weights", "weights_grad"):
        a = _score_args(s)
        z = s["logits"].double().requires_grad_()
        score = torch.softmax(z, 1) if a["score_fn"] == "softmax" else torch.sigmoid(z)
        if a["bias"] is not None:
            score = score + a["bias"].double()
        u = score.gather(1, s["ids"].long())
        w = a["routed_scale"] * u / u.sum(1, keepdim=True).clamp(min=a["norm_min"])
        if op == "weights":
            return w.detach()
        return torch.autograd.grad(w, z, s["grad"].double())[0]
    x = s["x"].double()
    y = torch.zeros((x.shape[0], case["N"]), dtype=torch.float64, device="cuda")
    bounds = [0, x.shape[0]] if s["offsets"] is None else s["offsets"].tolist()
    for e in range(case["E"]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi > lo:
            w = torch.empty((case["N"], case["K"]), dtype=torch.float64, device="cuda")
            w[:, 0::2] = (s["q"][e] % 16).double()
            w[:, 1::2] = (s["q"][e] // 16).double()
            zero = torch.full_like(s["scales"][e], 8).double() if s["zeros"] is None else s["zeros"][e].double()
            w -= zero.repeat_interleave(case["group"], 1)
            w *= s["scales"][e].double().repeat_interleave(case["group"], 1)
            y[lo:hi] = x[lo:hi] @ w.t()
    return y


def work(case):
    op = case["op"]
    if op == "w4":
        E, N, K, R = case["E"], case["N"], case["K"], case["T"] * case["top"]
        used = E * (1.0 - (1.0 - case["top"] / E) ** case["T"]) if E > 1 else 1  # experts that get a row, on average
        groups = K // case["group"]
        return {"bytes": used * N * (K / 2 + groups * (2 + (1 if case["zeros"] else 0))) + R * (K + N) * 2 + 4 * (E + 1),
                "flops": 2.0 * R * N * K}
    T, E, K = case["T"], case["E"], case["K"]
    if op == "weights":
        # a sigmoid score needs the chosen logits alone
        return {"bytes": 4.0 * (T * (E if case["score_fn"] == "softmax" else K) + 2 * T * K), "flops": 5.0 * T * K}
    if op == "weights_grad":
        read = T * (E if case["score_fn"] == "softmax" else K)
        return {"bytes": 4.0 * (read + T * E + 2 * T * K), "flops": 8.0 * T * E}
    size, H, R = SIZE[case["dtype"]], case["H"], _rows(case)
    live = (1.0 - case["padded"]) * min(R, T * K)
    if op == "sort":
        return {"bytes": float((T + R) * H * size + 4 * (2 * T * K + R + 2 * E + 1)), "flops": 0.0}
    if op == "sort_grad":
        return {"bytes": float((live + T) * H * size + 4 * T * K), "flops": live * H}
    if op == "unsort":
        return {"bytes": float((live + T * (2 if case["shared"] else 1)) * H * size + 8 * T * K), "flops": 2.0 * live * H}
    return {"bytes": float((live + R + T) * H * size + 12 * T * K), "flops": 3.0 * live * H}
