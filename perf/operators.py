"""Workloads of the operators whose weights are chosen row by row.

Three operators of `include/cute_b200.h`, each beside its plain form:

* ``lora``: a projection shared by all rows plus a low-rank adapter chosen row
  by row, ``y_i = W x_i + s_a B_a (A_a x_i)`` with ``a = ids[i]`` (an id outside
  the table means no adapter);
* ``lora_train``: the same with its gradients with respect to the input and the
  adapters (the shared weight is frozen);
* ``moe``: a whole mixture-of-experts layer for a few tokens: router, softmax,
  top-k, gated experts, weighted sum.

``listed()`` names fixed cases, ``draw()`` draws further ones from the same
ranges.  The plain forms work in 32 bits whatever the type of the inputs and
round once at the end.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One token of one request: a square projection of a mid-sized model.  Latency and the weight's bytes.
        {"name": "lora_token_1", "op": "lora", "m": 1, "n": 4096, "k": 4096, "rank": 16, "adapters": 8,
         "rows": "mixed", "dtype": "bf16", "out": "bf16"},
        # A decode step of 48 requests, nearly each with an adapter of its own.
        {"name": "lora_tokens_48", "op": "lora", "m": 48, "n": 8192, "k": 4096, "rank": 16, "adapters": 64,
         "rows": "mixed", "dtype": "bf16", "out": "bf16"},
        # A step that mixes decoding rows and short prompts, odd sizes, f16, a result kept in f32.
        {"name": "lora_mixed_777", "op": "lora", "m": 777, "n": 2050, "k": 1032, "rank": 40, "adapters": 12,
         "rows": "mixed", "dtype": "f16", "out": "f32"},
        # Packed prompts of many requests, lengths from one token to some thousand.
        {"name": "lora_prompts_8192", "op": "lora", "m": 8192, "n": 4096, "k": 4096, "rank": 64, "adapters": 8,
         "rows": "packed", "dtype": "bf16", "out": "bf16"},
        # A training step of a few adapters on packed sequences.
        {"name": "lora_train_4096", "op": "lora_train", "m": 4096, "n": 4096, "k": 4096, "rank": 16, "adapters": 4,
         "rows": "packed", "dtype": "bf16", "out": "bf16"},
        # One long batch for one adapter of a high rank into a wider projection.
        {"name": "lora_train_8192", "op": "lora_train", "m": 8192, "n": 8192, "k": 2048, "rank": 128, "adapters": 1,
         "rows": "packed", "dtype": "bf16", "out": "bf16"},
        # A small ragged batch with odd sizes in f16, rows of several adapters interleaved.
        {"name": "lora_train_odd", "op": "lora_train", "m": 333, "n": 520, "k": 1000, "rank": 8, "adapters": 5,
         "rows": "mixed", "dtype": "f16", "out": "f16"},
        # One token through few large experts: two of eight.
        {"name": "moe_token_1", "op": "moe", "tokens": 1, "experts": 8, "top": 2, "d": 4096, "f": 14336, "renorm": True,
         "dtype": "bf16"},
        # A small decode batch through many small experts.
        {"name": "moe_tokens_8", "op": "moe", "tokens": 8, "experts": 64, "top": 6, "d": 2048, "f": 1408, "renorm": False,
         "dtype": "bf16"},
        # The largest batch: nearly every expert is chosen by somebody.
        {"name": "moe_tokens_64", "op": "moe", "tokens": 64, "experts": 128, "top": 8, "d": 2048, "f": 768, "renorm": True,
         "dtype": "bf16"},
        # Odd sizes in f16.
        {"name": "moe_odd", "op": "moe", "tokens": 5, "experts": 10, "top": 3, "d": 520, "f": 328, "renorm": True,
         "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mul8(rng, lo, hi):
    return max(lo, _log(rng, lo, hi) // 8 * 8)


def draw(rng):
    op = rng.choice(["lora", "lora", "lora_train", "moe"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "moe":
        experts = _log(rng, 4, 128)
        d, f = _mul8(rng, 256, 4096), _mul8(rng, 128, 8192)
        while experts * d * f > 4.0e8:  # no more than the largest listed case holds
            f = max(128, f // 16 * 8)
            experts = max(4, experts // 2) if f == 128 else experts
        return {"op": op, "tokens": _log(rng, 1, 64), "experts": experts, "top": rng.randint(1, min(8, experts)), "d": d, "f": f,
                "renorm": rng.random() < 0.5, "dtype": dtype}
    # Half of the calls are decoding steps of up to 128 rows, half are prompts.
    m = _log(rng, 1, 128) if op == "lora" and rng.random() < 0.5 else _log(rng, 64, 8192)
    n = _log(rng, 256, 8192) if op == "lora" else _mul8(rng, 256, 8192)
    k = _mul8(rng, 256, 8192)
    while float(m) * n * k > 1.3e11:
        k = max(256, k // 16 * 8)
        n = n if k > 256 else max(256, n // 16 * 8)
    return {"op": op, "m": m, "n": n, "k": k, "rank": 8 * rng.randint(1, 16), "adapters": _log(rng, 1, 64 if m <= 128 else 16),
            "rows": rng.choice(["mixed", "packed"]), "dtype": dtype, "out": rng.choice([dtype, "f32"])}


def _normal(shape, std, dtype, gen):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).mul_(std).to(dtype)


def _ids(case, gen):
    """Adapter of every row: `mixed` rows choose freely (one in ten has none), `packed` rows belong to sequences of
    very different lengths, laid one behind the other."""
    m, adapters = case["m"], case["adapters"]
    ids = torch.randint(0, adapters, (m,), device="cuda", generator=gen, dtype=torch.int32)
    if case["rows"] == "mixed":
        none = torch.rand(m, device="cuda", generator=gen) < 0.1
        return torch.where(none, torch.full_like(ids, -1), ids)
    sequences = 2 * adapters + 1
    cuts = (torch.rand(sequences - 1, device="cuda", generator=gen).square() * (m + 1)).to(torch.int64).sort().values
    return ids[torch.searchsorted(cuts, torch.arange(m, device="cuda"), right=True).clamp(max=m - 1)].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t = TYPES[case["dtype"]]
    if case["op"] == "moe":
        e, d, f = case["experts"], case["d"], case["f"]
        return {"case": case,
                "x": _normal((case["tokens"], d), 1.0, t, gen),
                "router": _normal((e, d), 1.5 / math.sqrt(d), t, gen),
                "gate": _normal((e, f, d), 1.0 / math.sqrt(d), t, gen),
                "up": _normal((e, f, d), 1.0 / math.sqrt(d), t, gen),
                "down": _normal((e, d, f), 1.0 / math.sqrt(f), t, gen)}
    m, n, k, r, a = case["m"], case["n"], case["k"], case["rank"], case["adapters"]
    w = _normal((n, k), 1.0 / math.sqrt(k), t, gen)
    state = {"case": case,
             "x": _normal((m, k), 1.0, t, gen),
             "w": w,
             "a": _normal((a, r, k), 1.0 / math.sqrt(k), t, gen),
             "b": _normal((a, n, r), 0.5 / math.sqrt(r), t, gen),
             "ids": _ids(case, gen),
             "scale": torch.rand(a, device="cuda", generator=gen) + 0.5}
    if case["op"] == "lora_train":
        # The frozen weight is laid out once for the way back, as a training program keeps it.
        state["wt"] = w.t().contiguous()
        state["dy"] = _normal((m, n), 0.5, t, gen)
    return state


def _choice(ids, scale):
    """(rows, adapters): the scale of the row's adapter where the row has that adapter, else 0."""
    hot = ids.long()[:, None] == torch.arange(scale.numel(), device=ids.device)
    return hot * scale


def _plain_lora(s):
    x, choice = s["x"].float(), _choice(s["ids"], s["scale"])
    adapters, r, k = s["a"].shape
    t = (x @ s["a"].float().reshape(adapters * r, k).t()).reshape(-1, adapters, r) * choice[:, :, None]
    b = s["b"].float().permute(1, 0, 2).reshape(-1, adapters * r)
    return x @ s["w"].float().t() + t.reshape(-1, adapters * r) @ b.t(), t


def _plain_lora_train(s):
    out = TYPES[s["case"]["out"]]
    y, t = _plain_lora(s)
    adapters, r, k = s["a"].shape
    n = s["w"].shape[0]
    x, dy, choice = s["x"].float(), s["dy"].float(), _choice(s["ids"], s["scale"])
    b = s["b"].float().permute(1, 0, 2).reshape(n, adapters * r)
    u = (dy @ b).reshape(-1, adapters, r) * choice[:, :, None]
    u = u.reshape(-1, adapters * r)
    dx = dy @ s["w"].float() + u @ s["a"].float().reshape(adapters * r, k)
    da = (u.t() @ x).reshape(adapters, r, k)
    db = (dy.t() @ t.reshape(-1, adapters * r)).reshape(n, adapters, r).permute(1, 0, 2).contiguous()
    return {"y": y.to(out), "dx": dx.to(out), "da": da, "db": db}


def _plain_moe(s):
    case, x = s["case"], s["x"].float()
    # 64 bits: which expert comes in is decided between neighbouring probabilities.
    p = torch.softmax(s["x"].double() @ s["router"].double().t(), dim=-1)
    w, chosen = torch.sort(p, dim=-1, descending=True, stable=True)
    w, chosen = w[:, :case["top"]], chosen[:, :case["top"]]
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = w.float()
    if case["tokens"] * case["top"] < case["experts"]:
        g = (s["gate"][chosen].float() @ x[:, None, :, None]).squeeze(-1)
        u = (s["up"][chosen].float() @ x[:, None, :, None]).squeeze(-1)
        h = g * torch.sigmoid(g) * u
        y = ((s["down"][chosen].float() @ h[..., None]).squeeze(-1) * w[..., None]).sum(1)
    else:
        e, f, d = s["gate"].shape
        all_w = torch.zeros(x.shape[0], e, device=x.device).scatter_(1, chosen, w)
        g = (x @ s["gate"].float().reshape(e * f, d).t()).reshape(-1, e, f)
        u = (x @ s["up"].float().reshape(e * f, d).t()).reshape(-1, e, f)
        h = g * torch.sigmoid(g) * u * all_w[..., None]
        y = (h.transpose(0, 1) @ s["down"].float().transpose(1, 2)).sum(0)
    return y.to(s["x"].dtype)


def _own_desc(lib, case):
    kinds = {"f16": lib.F16, "bf16": lib.BF16, "f32": lib.F32}
    return lib.lora_desc(case["m"], case["n"], case["k"], case["rank"], case["adapters"], kinds[case["dtype"]], kinds[case["out"]])


def _own_lora(s):
    from cute_rs_b200 import _lib as lib
    case, x = s["case"], s["x"]
    stream = torch.cuda.current_stream().cuda_stream
    desc = _own_desc(lib, case)
    y = torch.empty(case["m"], case["n"], device="cuda", dtype=TYPES[case["out"]])
    work = torch.empty(lib.lora_workspace(desc), device="cuda", dtype=torch.uint8)
    lib.lora_tn(desc, x.data_ptr(), s["w"].data_ptr(), s["a"].data_ptr(), s["b"].data_ptr(), s["ids"].data_ptr(),
                s["scale"].data_ptr(), y.data_ptr(), work.data_ptr(), stream)
    if case["op"] == "lora":
        return y
    dx = torch.empty(case["m"], case["k"], device="cuda", dtype=TYPES[case["out"]])
    da = torch.empty(s["a"].shape, device="cuda", dtype=torch.float32)
    db = torch.empty(s["b"].shape, device="cuda", dtype=torch.float32)
    back = torch.empty(lib.lora_backward_workspace(desc), device="cuda", dtype=torch.uint8)
    lib.lora_tn_backward(desc, x.data_ptr(), s["wt"].data_ptr(), s["a"].data_ptr(), s["b"].data_ptr(), s["ids"].data_ptr(),
                         s["scale"].data_ptr(), s["dy"].data_ptr(), work.data_ptr(), dx.data_ptr(), da.data_ptr(),
                         db.data_ptr(), back.data_ptr(), stream)
    return {"y": y, "dx": dx, "da": da, "db": db}


def _own_moe(s):
    from cute_rs_b200 import _lib as lib
    case, x = s["case"], s["x"]
    desc = lib.moe_desc(case["tokens"], case["experts"], case["top"], case["d"], case["f"],
                        lib.F16 if case["dtype"] == "f16" else lib.BF16, case["renorm"])
    y = torch.empty_like(x)
    work = torch.empty(lib.moe_workspace(desc), device="cuda", dtype=torch.uint8)
    lib.moe_tn(desc, x.data_ptr(), s["router"].data_ptr(), s["gate"].data_ptr(), s["up"].data_ptr(), s["down"].data_ptr(),
               y.data_ptr(), work.data_ptr(), torch.cuda.current_stream().cuda_stream)
    return y


def run(state):
    op = state["case"]["op"]
    if op == "moe":
        return _own_moe(state) if own else _plain_moe(state)
    if own:
        return _own_lora(state)
    if op == "lora":
        return _plain_lora(state)[0].to(TYPES[state["case"]["out"]])
    return _plain_lora_train(state)


def work(case):
    if case["op"] == "moe":
        t, e, top, d, f = case["tokens"], case["experts"], case["top"], case["d"], case["f"]
        active = e * (1.0 - (1.0 - top / e) ** t)  # experts chosen by at least one token, on average
        return {"bytes": 2 * (2 * t * d + e * d + 3 * active * d * f), "flops": 2 * t * e * d + 6 * t * top * d * f}
    m, n, k, r = case["m"], case["n"], case["k"], case["rank"]
    used = min(case["adapters"], m)
    out = 4 if case["out"] == "f32" else 2
    product, low = 2 * m * n * k, 2 * m * r * (n + k)
    weights = 2 * (n * k + used * r * (n + k))
    w = {"bytes": weights + 2 * m * k + out * m * n + 4 * m, "flops": product + low}
    if case["op"] == "lora_train":
        w["bytes"] += weights + 2 * m * (n + k) + out * m * k + 4 * case["adapters"] * r * (n + k)
        w["flops"] += product + 2 * low
    return w


def exact(case, seed):
    def lora(s):
        x, w, scale = s["x"].double(), s["w"].double(), s["scale"].double()
        y = x @ w.t()
        train = s["case"]["op"] == "lora_train"
        if train:
            dy = s["dy"].double()
            dx = dy @ w
            da = torch.zeros(s["a"].shape, device="cuda", dtype=torch.float64)
            db = torch.zeros(s["b"].shape, device="cuda", dtype=torch.float64)
        for i in range(s["case"]["adapters"]):
            rows = torch.nonzero(s["ids"] == i).flatten()
            if rows.numel() == 0:
                continue
            a, b, xi = s["a"][i].double(), s["b"][i].double(), x[rows]
            t = scale[i] * (xi @ a.t())
            y[rows] += t @ b.t()
            if train:
                u = scale[i] * (dy[rows] @ b)
                dx[rows] += u @ a
                da[i] = u.t() @ xi
                db[i] = dy[rows].t() @ t
        return {"y": y, "dx": dx, "da": da, "db": db} if train else y

    def moe(s):
        case, x = s["case"], s["x"].double()
        logits = x @ s["router"].double().t()
        y = torch.zeros_like(x)
        for t, row in enumerate(logits.tolist()):
            order = sorted(range(len(row)), key=lambda e: (-row[e], e))[:case["top"]]
            top = max(row)
            weight = [math.exp(row[e] - top) for e in order]
            total = sum(weight) if case["renorm"] else sum(math.exp(v - top) for v in row)
            for e, p in zip(order, weight):
                g, u = s["gate"][e].double() @ x[t], s["up"][e].double() @ x[t]
                y[t] += (p / total) * (s["down"][e].double() @ (g / (1.0 + torch.exp(-g)) * u))
        return y

    state = prepare(case, seed)
    return moe(state) if case["op"] == "moe" else lora(state)
