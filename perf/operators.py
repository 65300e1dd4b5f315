"""The two projection operators beside ``ops.gemm``, as they are measured.

* ``gated_linear``: h = act(x Wg^T) * (x Wu^T), the first half of a gated feed-forward block
  (the dense counterpart of the expert layer's first grouped GEMM), forward alone (serving) or
  forward and backward (training);
* ``lora_linear``: y = x W^T + s[a] (x A[a]^T) B[a]^T with an adapter a per row (-1: none), a
  shared projection with the low-rank adapters of many requests.

``run`` computes them in elementary torch operations in 32 bits or, where ``own`` is true,
through the package's entry points.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ("silu", "gelu", "gelu_tanh")


def listed():
    gated, lora = [], []
    # One token through the shared expert beside the expert layer (hidden 7168, intermediate 2048).
    gated.append({"name": "gated_one_token", "op": "gated", "train": False, "T": 1, "H": 7168, "I": 2048,
                  "dtype": "bf16", "act": "silu"})
    # A decode batch of an odd size through a wide block.
    gated.append({"name": "gated_decode_37", "op": "gated", "train": False, "T": 37, "H": 4096, "I": 8200,
                  "dtype": "fp16", "act": "gelu_tanh"})
    # A prompt: the expert layer's 4096 tokens per GPU.
    gated.append({"name": "gated_prompt", "op": "gated", "train": False, "T": 4096, "H": 7168, "I": 2048,
                  "dtype": "bf16", "act": "silu"})
    # A training step of the same block.
    gated.append({"name": "gated_train", "op": "gated", "train": True, "T": 4096, "H": 7168, "I": 2048,
                  "dtype": "bf16", "act": "silu"})
    # A small training step with ragged sizes (a fine-tune on short texts).
    gated.append({"name": "gated_train_ragged", "op": "gated", "train": True, "T": 1001, "H": 2056, "I": 5461,
                  "dtype": "fp16", "act": "gelu"})
    # The largest: a long packed batch through a wide block.
    gated.append({"name": "gated_train_large", "op": "gated", "train": True, "T": 8192, "H": 8192, "I": 8192,
                  "dtype": "bf16", "act": "gelu_tanh"})
    # One token of one request.
    lora.append({"name": "lora_one_token", "op": "lora", "T": 1, "K": 4096, "N": 4096, "L": 8, "r": 16,
                 "requests": 1, "dtype": "bf16"})
    # A decode batch in which every request brings its own adapter.
    lora.append({"name": "lora_decode_64", "op": "lora", "T": 64, "K": 7168, "N": 4096, "L": 64, "r": 16,
                 "requests": 64, "dtype": "bf16"})
    # Prompts and single tokens in one batch, odd sizes.
    lora.append({"name": "lora_mixed", "op": "lora", "T": 777, "K": 4104, "N": 4099, "L": 32, "r": 64,
                 "requests": 21, "dtype": "fp16"})
    # Short requests of many adapters interleaved in a long batch.
    lora.append({"name": "lora_many", "op": "lora", "T": 4096, "K": 7168, "N": 4096, "L": 48, "r": 16,
                 "requests": 256, "dtype": "bf16"})
    # Long prompts with wide adapters.
    lora.append({"name": "lora_prompt", "op": "lora", "T": 8192, "K": 8192, "N": 8192, "L": 16, "r": 64,
                 "requests": 11, "dtype": "bf16"})
    return gated + lora


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(step, v // step * step)


def draw(rng):
    dtype = rng.choice(sorted(DTYPES))
    if rng.random() < 0.55:
        case = {"op": "gated", "train": rng.random() < 0.5, "T": _log_int(rng, 1, 8192), "H": _log_int(rng, 64, 8192, 8),
                "I": _log_int(rng, 33, 16384), "dtype": dtype, "act": rng.choice(ACTS)}
        most = 8192 * 8192 * 8192
        while case["T"] * case["H"] * case["I"] > most:
            case["I"] = max(33, case["I"] // 2)
        return case
    T = _log_int(rng, 1, 8192)
    return {"op": "lora", "T": T, "K": _log_int(rng, 64, 8192, 8), "N": _log_int(rng, 33, 8192), "L": _log_int(rng, 1, 128),
            "r": rng.choice([8, 16, 24, 32, 64, 128]), "requests": _log_int(rng, 1, min(T, 256)), "dtype": dtype}


def _used(case):
    """Requests with an adapter (each eighth request has none), and the distinct adapters among them."""
    n = case["requests"]
    active = n - n // 8
    return active, min(active, case["L"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    if case["op"] == "gated":
        T, H, I = case["T"], case["H"], case["I"]
        st = {"case": case, "x": normal(T, H), "w_gate": normal(I, H, std=H ** -0.5), "w_up": normal(I, H, std=H ** -0.5)}
        if case["train"]:
            st["dh"] = normal(T, I, std=0.05)
            for k in ("x", "w_gate", "w_up"):
                st[k].requires_grad_(True)
        return st
    T, K, N, L, r, n = (case[k] for k in ("T", "K", "N", "L", "r", "requests"))
    st = {"case": case, "x": normal(T, K), "w": normal(N, K, std=K ** -0.5), "lora_a": normal(L, r, K, std=K ** -0.5),
          "lora_b": normal(L, N, r, std=0.5 * r ** -0.5),
          "scale": torch.rand(L, generator=g, device="cuda") * 1.5 + 0.5}
    # requests of random lengths, one after another; request i's adapter from a shuffled cycle
    cuts = torch.randperm(T - 1, generator=g, device="cuda")[: n - 1].sort().values + 1 if n > 1 else None
    row_request = torch.zeros(T, dtype=torch.int64, device="cuda")
    if cuts is not None:
        row_request[cuts] = 1
        row_request = row_request.cumsum(0)
    perm = torch.randperm(L, generator=g, device="cuda")
    req = torch.arange(n, device="cuda")
    active, _ = _used(case)
    rank = torch.randperm(n, generator=g, device="cuda")
    by_request = torch.where(rank < active, perm[rank % L], torch.full_like(req, -1))
    st["adapter"] = by_request[row_request].to(torch.int32)
    return st


def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _plain_gated(st):
    case = st["case"]
    x, wg, wu = (st[k].detach().float() for k in ("x", "w_gate", "w_up"))
    dt = st["x"].dtype
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(g, case["act"])
    h = (a * u).to(dt)
    if not case["train"]:
        return h
    dh = st["dh"].float()
    dg, du = dh * u * da, dh * a
    return h, (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)


def _plain_lora(st):
    case = st["case"]
    x, idx = st["x"].float(), st["adapter"].long()
    L, r, N = case["L"], case["r"], case["N"]
    v = (x @ st["lora_a"].float().view(L * r, -1).t()).view(-1, L, r)
    mine = (idx[:, None] == torch.arange(L, device=idx.device)) * st["scale"]
    delta = (v * mine[:, :, None]).view(-1, L * r) @ st["lora_b"].float().permute(0, 2, 1).reshape(L * r, N)
    return (x @ st["w"].float().t() + delta).to(st["x"].dtype)


def _own_gated(st):
    from opengda_b200.ops.ffn import gated_linear

    h = gated_linear(st["x"], st["w_gate"], st["w_up"], act=st["case"]["act"])
    if not st["case"]["train"]:
        return h
    return (h.detach(), *torch.autograd.grad(h, (st["x"], st["w_gate"], st["w_up"]), st["dh"]))


def _own_lora(st):
    from opengda_b200.ops.lora import lora_linear

    return lora_linear(st["x"], st["w"], st["lora_a"], st["lora_b"], st["adapter"], scale=st["scale"])


def run(state):
    if state["case"]["op"] == "gated":
        if own:
            return _own_gated(state)
        return _plain_gated(state)
    if own:
        return _own_lora(state)
    return _plain_lora(state)


def work(case):
    T = case["T"]
    if case["op"] == "gated":
        H, I = case["H"], case["I"]
        if not case["train"]:
            return {"bytes": 2 * (T * H + 2 * I * H + T * I), "flops": 4 * T * H * I}
        # in: x, dh, both weights; out: h, dx and both weights' gradients
        return {"bytes": 2 * (T * H + T * I + 2 * I * H) * 2, "flops": 12 * T * H * I}
    K, N, r = case["K"], case["N"], case["r"]
    active, distinct = _used(case)
    rows = T * active // case["requests"]
    return {"bytes": 2 * (T * K + N * K + T * N + distinct * r * (K + N)) + 4 * T + 4 * distinct,
            "flops": 2 * T * N * K + 2 * rows * r * (K + N)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gated":
        x, wg, wu = (st[k].detach().double() for k in ("x", "w_gate", "w_up"))
        gate, up = torch.matmul(x, wg.T), torch.matmul(x, wu.T)
        if case["act"] == "silu":
            sig = torch.reciprocal(1 + torch.exp(-gate))
            act, slope = gate * sig, sig + gate * sig * (1 - sig)
        elif case["act"] == "gelu":
            phi = 0.5 * torch.special.erfc(-gate / math.sqrt(2))
            act, slope = gate * phi, phi + gate * torch.exp(-gate * gate / 2) / math.sqrt(2 * math.pi)
        else:
            inner = math.sqrt(2 / math.pi) * gate * (1 + 0.044715 * gate * gate)
            half = 1 / (1 + torch.exp(-2 * inner))  # (1 + tanh(inner)) / 2
            act = gate * half
            slope = half + gate * 2 * half * (1 - half) * math.sqrt(2 / math.pi) * (1 + 0.134145 * gate * gate)
        if not case["train"]:
            return act * up
        dh = st["dh"].double()
        dgate, dup = dh * up * slope, dh * act
        return (act * up, torch.matmul(dgate, wg) + torch.matmul(dup, wu), torch.matmul(dgate.T, x),
                torch.matmul(dup.T, x))
    x = st["x"].double()
    y = torch.matmul(x, st["w"].double().T)
    for a in range(case["L"]):
        rows = (st["adapter"] == a).nonzero().flatten()
        if rows.numel():
            low = torch.matmul(x[rows], st["lora_a"][a].double().T) * st["scale"][a].double()
            y[rows] += torch.matmul(low, st["lora_b"][a].double().T)
    return y
