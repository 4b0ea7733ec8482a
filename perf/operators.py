"""What the expert products and the adapter projection are measured on.

Three operators, each with its plain form (elementary torch operations in 32 bits) and
its call into the framework:

* ``grouped``  -- y[p] = W[e(p)] x[p] for rows in expert order (``grouped_matmul``);
* ``backward`` -- dx[p] = W[e(p)]^T dy[p] and dW[e] = sum_p dy[p] x[p]^T
  (``grouped_matmul_grad_input`` and ``grouped_matmul_grad_weight``);
* ``lora``     -- y[t] = W x[t] + s_a B_a (A_a x[t]), a = the adapter of row t or none
  (``lora_matmul``).

``own`` selects which of the two ``run`` computes.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _grouped(name, dtype, tokens, experts, k, n, kdim, zipf=False, op="grouped"):
    return dict(name=name, op=op, dtype=dtype, tokens=tokens, experts=experts, top=k, n=n,
                k=kdim, zipf=zipf)


def _lora(name, dtype, rows, n, k, rank, adapters, prompts, plain_rows):
    return dict(name=name, op="lora", dtype=dtype, rows=rows, n=n, k=k, rank=rank,
                adapters=adapters, prompts=prompts, plain_rows=plain_rows)


def listed():
    return [
        # One generated token through the up projection of a fine-grained layer: 8 rows,
        # 8 experts of 64; the latency of a call and of streaming 25 MB of weights.
        _grouped("fc1_one_token", "bf16", 1, 64, 8, 768, 2048),
        # A small decode batch (37 sequences) through the down projection: a few rows for
        # nearly every expert.
        _grouped("fc2_decode_batch", "fp16", 37, 64, 8, 2048, 768),
        # A prompt through the down projection of a layer with eight wide experts.
        _grouped("fc2_prompt_wide", "fp16", 4096, 8, 2, 4096, 14336),
        # A prefill batch through a fine-grained layer, experts loaded by a power law.
        _grouped("fc1_prompt_fine", "bf16", 16384, 64, 8, 768, 2048, zipf=True),
        # One optimiser micro-step's backward of a small fp32 layer.
        _grouped("grad_small_fp32", "fp32", 256, 8, 2, 1024, 512, op="backward"),
        # A short, odd fine-tuning batch over 16 experts: weights and their gradients are
        # nearly all of the traffic.
        _grouped("grad_short_batch", "bf16", 333, 16, 2, 6400, 4096, op="backward"),
        # The backward of a pre-training batch over fine-grained experts with skewed load.
        _grouped("grad_fine", "bf16", 16384, 64, 8, 768, 2048, zipf=True, op="backward"),
        # The backward of a training batch over eight wide experts.
        _grouped("grad_wide", "fp16", 4096, 8, 2, 14336, 4096, op="backward"),
        # One request's next token with its adapter.
        _lora("lora_one_token", "bf16", 1, 4096, 4096, 16, 8, 0, 0),
        # 64 requests decoding together, 32 adapters, some requests on the base model.
        _lora("lora_decode_batch", "bf16", 64, 4096, 4096, 16, 32, 0, 7),
        # Prompts and generated tokens in one batch, an odd row count, small ranks.
        _lora("lora_mixed_batch", "fp16", 333, 4096, 2048, 8, 16, 3, 5),
        # Eleven prompts of different adapters prefilled at once, rank 64.
        _lora("lora_prompts", "bf16", 4001, 4096, 4096, 64, 16, 11, 0),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["grouped", "backward", "lora"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    step = 1 if dtype == "fp32" else 8
    while True:
        n, k = _log(rng, 64, 14336, step), _log(rng, 64, 14336, step)
        if op == "lora":
            rows = _log(rng, 1, 8192)
            prompts = rng.randint(0, 12) if rows >= 64 else 0
            case = dict(op=op, dtype=dtype, rows=rows, n=n, k=k,
                        rank=8 * _log(rng, 1, 16), adapters=_log(rng, 1, 128),
                        prompts=prompts, plain_rows=rng.randint(0, max(0, rows // 8)))
        else:
            experts = rng.choice([1, 3, 8, 16, 60, 64, 128])
            case = dict(op=op, dtype=dtype, tokens=_log(rng, 1, 16384), experts=experts,
                        top=rng.randint(1, min(8, experts)), n=n, k=k,
                        zipf=rng.random() < 0.5)
        w = work(case)
        if w["bytes"] <= 2.5e9 and w["flops"] <= (4e10 if dtype == "fp32" else 1.5e12):
            return case


# --------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, scale, dtype, g):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(dtype)


def _weights(e, n, k, dtype, g):
    w = torch.empty((e, n, k), device="cuda", dtype=dtype)
    for i in range(e):
        w[i] = _randn((n, k), 0.02, dtype, g)
    return w


def _group_sizes(case, g):
    """Rows of each expert when `tokens` rows choose their `top` experts by random logits
    (with a power-law bias where the case says so)."""
    t, e = case["tokens"], case["experts"]
    logits = torch.randn((t, e), device="cuda", generator=g)
    if case["zipf"]:
        bias = torch.arange(1, e + 1, device="cuda", dtype=torch.float32).pow(-1.1).log()
        span = (bias.max() - bias.min()).clamp_min(1e-6)
        logits += 3.0 * (bias - bias.min()) / span
    idx = logits.topk(case["top"], dim=1).indices.reshape(-1)
    return torch.bincount(idx, minlength=e)


def _adapter_of_rows(case, g):
    """Adapter of each row: `prompts` runs of adjacent rows, then single rows, the last
    `plain_rows` of them (or of all rows) on the base model."""
    rows, n_ad, prompts = case["rows"], case["adapters"], case["prompts"]
    order = torch.randperm(n_ad, generator=torch.Generator().manual_seed(
        int(torch.randint(0, 2 ** 31, (1,), device="cuda", generator=g))))
    ids = torch.empty(rows, dtype=torch.int32)
    at = 0
    if prompts:
        tail = min(rows // 4, 61) if case["plain_rows"] else 0
        cuts = sorted(torch.randint(1, max(2, rows - tail), (prompts - 1,),
                                    generator=torch.Generator().manual_seed(prompts)).tolist())
        for j, (a, b) in enumerate(zip([0] + cuts, cuts + [rows - tail])):
            ids[a:b] = int(order[j % n_ad])
        at = rows - tail
    for r in range(at, rows):
        ids[r] = int(order[r % n_ad])
    if case["plain_rows"]:
        ids[rows - case["plain_rows"]:] = -1
    return ids.to("cuda")


def _inputs(case, seed):
    g = _gen(seed)
    dt = _DTYPES[case["dtype"]]
    n, k = case["n"], case["k"]
    if case["op"] == "lora":
        rows, r, n_ad = case["rows"], case["rank"], case["adapters"]
        ids = _adapter_of_rows(case, g)
        pick = torch.randint(0, 3, (n_ad,), device="cuda", generator=g)
        return dict(x=_randn((rows, k), 1.0, dt, g), weight=_weights(1, n, k, dt, g)[0],
                    lora_a=_randn((n_ad, r, k), 1.0 / math.sqrt(k), dt, g),
                    lora_b=_randn((n_ad, n, r), 0.05, dt, g), ids=ids,
                    scales=torch.tensor([0.5, 1.0, 2.0], device="cuda")[pick])
    sizes = _group_sizes(case, g)
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = sizes.cumsum(0)
    rows = case["tokens"] * case["top"]
    d = dict(x=_randn((rows, k), 1.0, dt, g), offsets=offsets, sizes=sizes.tolist(),
             weights=_weights(case["experts"], n, k, dt, g))
    if case["op"] == "backward":
        d["dy"] = _randn((rows, n), 0.1, dt, g)
    return d


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"] = case["op"]
    if own:
        from __graft_entry__ import load_package
        state["pkg"] = load_package()
    return state


# ------------------------------------------------------------------------- one pass

def run(state):
    op = state["op"]
    if own:
        pkg = state["pkg"]
        if op == "grouped":
            return pkg.grouped_matmul(state["x"], state["weights"], state["offsets"])
        if op == "backward":
            return {
                "dx": pkg.grouped_matmul_grad_input(state["dy"], state["weights"],
                                                    state["offsets"]),
                "dw": pkg.grouped_matmul_grad_weight(state["x"], state["dy"],
                                                     state["offsets"]),
            }
        return pkg.lora_matmul(state["x"], state["weight"], state["lora_a"],
                               state["lora_b"], state["ids"], state["scales"])
    if op == "lora":
        return _plain_lora(state, torch.float32).to(state["x"].dtype)
    return _plain_grouped(state)


def _spans(sizes):
    at = 0
    for e, c in enumerate(sizes):
        yield e, at, at + c
        at += c


def _plain_grouped(state):
    x, w, dt = state["x"], state["weights"], state["x"].dtype
    if state["op"] == "grouped":
        y = torch.empty((x.shape[0], w.shape[1]), device=x.device, dtype=dt)
        for e, a, b in _spans(state["sizes"]):
            if b > a:
                y[a:b] = (x[a:b].float() @ w[e].float().t()).to(dt)
        return y
    dy = state["dy"]
    dx, dw = torch.empty_like(x), torch.zeros_like(w)
    for e, a, b in _spans(state["sizes"]):
        if b > a:
            d = dy[a:b].float()
            dx[a:b] = (d @ w[e].float()).to(dt)
            dw[e] = (d.t() @ x[a:b].float()).to(dt)
    return {"dx": dx, "dw": dw}


def _plain_lora(state, dt):
    x, a, b = state["x"].to(dt), state["lora_a"].to(dt), state["lora_b"].to(dt)
    n_ad, r, k = a.shape
    ids = state["ids"]
    mine = ids[:, None] == torch.arange(n_ad, device=x.device)[None]
    t = (x @ a.reshape(n_ad * r, k).t()).reshape(-1, n_ad, r) * state["scales"].to(dt)[None, :, None]
    t = torch.where(mine[:, :, None], t, torch.zeros_like(t)).reshape(-1, n_ad * r)
    return x @ state["weight"].to(dt).t() + t @ b.transpose(1, 2).reshape(n_ad * r, -1)


# ------------------------------------------------------------------------ definition

def exact(case, seed):
    """The definition in 64 bits, expert by expert and adapter by adapter."""
    d = _inputs(case, seed)
    x = d["x"].double()
    if case["op"] == "lora":
        y = x @ d["weight"].double().t()
        ids = d["ids"].cpu()
        for a in sorted(set(ids.tolist()) - {-1}):
            rows = (ids == a).nonzero().reshape(-1).to(x.device)
            t = x[rows] @ d["lora_a"][a].double().t()
            y[rows] += float(d["scales"][a]) * (t @ d["lora_b"][a].double().t())
        return y
    w = d["weights"]
    bounds = d["offsets"].tolist()
    if case["op"] == "grouped":
        y = torch.empty((x.shape[0], w.shape[1]), device=x.device, dtype=torch.float64)
        for e in range(w.shape[0]):
            s = slice(bounds[e], bounds[e + 1])
            y[s] = x[s] @ w[e].double().t()
        return y
    dx = torch.empty_like(x)
    dw = torch.zeros(w.shape, device=x.device, dtype=torch.float64)
    for e in range(w.shape[0]):
        s = slice(bounds[e], bounds[e + 1])
        dy = d["dy"][s].double()
        dx[s] = dy @ w[e].double()
        dw[e] = dy.t() @ x[s]
    return {"dx": dx, "dw": dw}


def work(case):
    b, n, k = _BYTES[case["dtype"]], case["n"], case["k"]
    if case["op"] == "lora":
        rows, r = case["rows"], case["rank"]
        with_ad = rows - case["plain_rows"]
        runs = with_ad if not case["prompts"] else min(with_ad, case["prompts"] + 61)
        used = min(case["adapters"], max(runs, 1)) if with_ad else 0
        return {"bytes": b * (rows * (k + n) + n * k + used * r * (n + k)) + 4 * rows,
                "flops": 2 * rows * n * k + 2 * with_ad * r * (n + k)}
    rows, e = case["tokens"] * case["top"], case["experts"]
    # Experts that get at least one row when every token picks `top` of them at random.
    used = e * (1.0 - (1.0 - case["top"] / e) ** case["tokens"]) if case["top"] < e else e
    one = 2 * rows * n * k
    if case["op"] == "grouped":
        return {"bytes": int(b * (rows * (n + k) + used * n * k)) + 4 * (e + 1), "flops": one}
    # dx reads dy and the used weights; dW reads x (dy is counted once) and is written for
    # every expert, the unused ones too.
    return {"bytes": int(b * (rows * (n + 2 * k) + used * n * k + e * n * k)) + 4 * (e + 1),
            "flops": 2 * one}
