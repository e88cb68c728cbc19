"""Cases of the output-head operators: the loss of a large vocabulary with its
gradient, and the head held in 4 bits (its products, the display statistics
over them, and the quantiser that lays the weight out).

``own`` false computes each operator in elementary torch operations in 32
bits; ``own`` true makes the calls a user makes of ``cid_engine``.

Operators (``case["op"]``):

* ``cross_entropy``: labels [rows], -100 where a position carries no loss;
  hidden [rows, H] and weight [V, H] bf16 or fp16; per-position loss and
  log-sum-exp, and the gradients of hidden and weight for a per-position
  weight of the loss (1 / mask ratio in masked diffusion);
* ``quantized_logits``: hidden [rows, H] times a [V, H] weight of 4-bit codes
  with a scale for each group of ``group`` columns;
* ``quantized_statistics``: confidence, argmax and current-token confidence
  over those products (float32 logits);
* ``quantize``: the codes and scales of a [V, H] weight, returned as the
  values they stand for.

Packed codes: int32 [V, H / 8], eight codes q + 8 (q in [-8, 7]) a word; the
code of column 8 j + k sits at bit ``_SHIFTS[k]`` of word j.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)
_IGNORE = -100


def _engine():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cid-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import cid_engine

    return cid_engine


def listed():
    return [
        # the smoke test's head: a call of a few microseconds of work, where launches count
        {"name": "loss 64x4096 h64", "op": "cross_entropy", "rows": 64, "vocab": 4096, "hidden": 64, "kept": 0.5, "dtype": "bf16"},
        # configuration 1's display [4, 256] over 32000 tokens, half its positions masked
        {"name": "loss 1024x32000 h2048", "op": "cross_entropy", "rows": 1024, "vocab": 32000, "hidden": 2048, "kept": 0.5, "dtype": "bf16"},
        # a few supervised positions at the full vocabulary: weight and its gradient stream past
        {"name": "loss 24x128256 h4096", "op": "cross_entropy", "rows": 24, "vocab": 128256, "hidden": 4096, "kept": 1.0, "dtype": "bf16"},
        # odd sizes in fp16: configuration 3's vocabulary, ragged rows and width, few positions kept
        {"name": "loss 999x50257 h1000 fp16", "op": "cross_entropy", "rows": 999, "vocab": 50257, "hidden": 1000, "kept": 0.3, "dtype": "fp16"},
        # a training step's micro-batch at the benchmark's head, seven positions of ten masked
        {"name": "loss 4096x128256 h4096", "op": "cross_entropy", "rows": 4096, "vocab": 128256, "hidden": 4096, "kept": 0.7, "dtype": "bf16"},
        # one position against a small head: the smallest product
        {"name": "logits4 1x32000 h2048", "op": "quantized_logits", "rows": 1, "vocab": 32000, "hidden": 2048, "group": 128, "dtype": "bf16"},
        # odd rows and vocabulary, small groups, fp16
        {"name": "logits4 7x50257 h1600 g32 fp16", "op": "quantized_logits", "rows": 7, "vocab": 50257, "hidden": 1600, "group": 32, "dtype": "fp16"},
        # the benchmark's head for a block of sixteen display positions
        {"name": "logits4 16x128256 h4096", "op": "quantized_logits", "rows": 16, "vocab": 128256, "hidden": 4096, "group": 128, "dtype": "bf16"},
        # four positions of a small head, straight to statistics
        {"name": "stats4 4x32000 h1024 g64", "op": "quantized_statistics", "rows": 4, "vocab": 32000, "hidden": 1024, "group": 64, "dtype": "bf16"},
        # the benchmark's 64-row decode step from 4-bit weights
        {"name": "stats4 64x128256 h4096", "op": "quantized_statistics", "rows": 64, "vocab": 128256, "hidden": 4096, "group": 128, "dtype": "bf16"},
        # laying out a small head
        {"name": "quantize 5000x512 g64 fp16", "op": "quantize", "vocab": 5000, "hidden": 512, "group": 64, "dtype": "fp16"},
        # laying out the benchmark's head
        {"name": "quantize 128256x4096", "op": "quantize", "vocab": 128256, "hidden": 4096, "group": 128, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("cross_entropy", "cross_entropy", "quantized_logits", "quantized_statistics", "quantize"))
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16")), "vocab": _log_int(rng, 1000, 152064)}
    if op == "cross_entropy":
        case["hidden"] = 8 * _log_int(rng, 8, 512)
        case["kept"] = round(rng.uniform(0.15, 1.0), 2)
        most = 4096 * 128256 * 4096 / (case["vocab"] * case["hidden"]) * min(1.0, 0.7 / case["kept"])
        case["rows"] = _log_int(rng, 1, min(8192, int(most)))
        return case
    case["group"] = rng.choice((32, 64, 128, 128))
    case["hidden"] = case["group"] * _log_int(rng, max(1, 256 // case["group"]), 4096 // case["group"])
    if op != "quantize":
        case["rows"] = _log_int(rng, 1, 128)
    return case


def _kept(case):
    return max(1, int(round(case["rows"] * case["kept"])))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    V, H = case["vocab"], case["hidden"]
    # logits of a standard deviation of about 2, as the benchmark's display logits
    weight = torch.empty(V, H, dtype=dt, device=dev).normal_(0.0, 2.0 / math.sqrt(H), generator=g)
    state = {"op": case["op"], "weight": weight}
    if case["op"] == "quantize":
        state["group"] = case["group"]
        return state
    N = case["rows"]
    ids = torch.randint(0, V, (N,), generator=g, device=dev)
    hidden = torch.randn(N, H, generator=g, device=dev)
    # positions that point at their token by 0 to 12 in the logits, as positions of a trained model do
    lift = torch.rand(N, 1, generator=g, device=dev) * 12.0
    own_row = weight[ids].float()
    hidden = (hidden + lift * own_row / own_row.square().sum(1, keepdim=True).clamp_min(1e-3)).to(dt)
    state["hidden"] = hidden
    if case["op"] == "cross_entropy":
        keep = torch.zeros(N, dtype=torch.bool, device=dev)
        keep[torch.randperm(N, generator=g, device=dev)[: _kept(case)]] = True
        state["labels"] = torch.where(keep, ids, torch.full_like(ids, _IGNORE))
        # 1 / mask ratio of each position's row, over the number of positions; fp16 training scales its loss
        state["scale"] = (1.0 / (0.1 + 0.9 * torch.rand(N, generator=g, device=dev))) / N
        if dt == torch.float16:
            state["scale"] *= 1024.0
        return state
    codes, scales = _codes(weight, case["group"])
    word = torch.zeros(V, H // 8, dtype=torch.int32, device=dev)
    c = (codes + 8).to(torch.int32).view(V, H // 8, 8)
    for k, s in enumerate(_SHIFTS):
        word |= c[:, :, k] << s
    del state["weight"]
    # half of the current tokens are other tokens than the one pointed at
    other = torch.randint(0, V, (N,), generator=g, device=dev)
    state.update(packed=word, scales=scales, ids=torch.where(lift.view(-1) > 6.0, ids, other))
    return state


def _codes(weight, group):
    """Codes in [-8, 7] (as float32, [V, H]) and scales ([V, H / group]) of a weight."""
    V, H = weight.shape
    w = weight.float().view(V, H // group, group)
    scales = (w.abs().amax(-1) / 7.0).to(weight.dtype)
    s = scales.float().unsqueeze(-1)
    q = torch.where(s > 0, (w / s).round(), torch.zeros_like(w)).clamp(-8, 7)
    return q.view(V, H), scales


def _values(packed, scales):
    """The float32 weight that packed codes and scales stand for."""
    shifts = torch.tensor(_SHIFTS, dtype=torch.int32, device=packed.device)
    q = ((packed.unsqueeze(-1) >> shifts) & 15) - 8
    V, G = scales.shape
    return (q.view(V, G, -1).float() * scales.float().unsqueeze(-1)).view(V, -1)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    E = _engine()
    op = state["op"]
    if op == "cross_entropy":
        h = state["hidden"].detach().requires_grad_()
        w = state["weight"].detach().requires_grad_()
        loss, lse = E.lm_head_cross_entropy(state["labels"], h, w, ignore_index=_IGNORE)
        dh, dw = torch.autograd.grad(loss, (h, w), grad_outputs=state["scale"])
        return {"loss": loss.detach(), "lse": lse.detach(), "grad_hidden": dh, "grad_weight": dw}
    if op == "quantized_logits":
        return {"logits": E.lm_head_quantized_logits(state["hidden"], state["packed"], state["scales"])}
    if op == "quantized_statistics":
        c, p, u = E.lm_head_quantized_display_statistics(state["ids"], state["hidden"], state["packed"], state["scales"], round_bf16=False)
        return {"confidence": c, "predicted": p, "current": u}
    packed, scales = E.lm_head_quantize(state["weight"], group_size=state["group"])
    return {"scales": scales, "values": E.lm_head_dequantize(packed, scales)}


def _run_plain(state):
    op = state["op"]
    if op == "cross_entropy":
        dt = state["hidden"].dtype
        labels = state["labels"]
        keep = labels != _IGNORE
        h = torch.where(keep.unsqueeze(1), state["hidden"].float(), 0.0)
        w = state["weight"].float()
        at = torch.where(keep, labels, 0).unsqueeze(1)
        logits = h @ w.T
        top = logits.amax(1, keepdim=True)
        e = (logits - top).exp()
        total = e.sum(1, keepdim=True)
        lse = (top + total.log()).squeeze(1)
        loss = torch.where(keep, lse - logits.gather(1, at).squeeze(1), 0.0)
        lse = torch.where(keep, lse, 0.0)
        d = e / total
        d.scatter_add_(1, at, -torch.ones_like(at, dtype=d.dtype))
        d *= torch.where(keep, state["scale"], 0.0).unsqueeze(1)
        return {"loss": loss, "lse": lse, "grad_hidden": (d @ w).to(dt), "grad_weight": (d.T @ h).to(dt)}
    if op == "quantize":
        q, scales = _codes(state["weight"], state["group"])
        V, G = scales.shape
        values = (q.view(V, G, -1) * scales.float().unsqueeze(-1)).view(V, -1)
        return {"scales": scales, "values": values.to(scales.dtype)}
    logits = state["hidden"].float() @ _values(state["packed"], state["scales"]).T
    if op == "quantized_logits":
        return {"logits": logits.to(state["hidden"].dtype)}
    top, first = logits.amax(1), logits.argmax(1)
    total = (logits - top.unsqueeze(1)).exp().sum(1)
    current = logits.gather(1, state["ids"].unsqueeze(1)).squeeze(1)
    return {"confidence": 1.0 / total, "predicted": first, "current": (current - top).exp() / total}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        w = s["weight"].double()
        V, H = w.shape
        w = w.reshape(V, H // case["group"], case["group"])
        step = (w.abs().max(-1, keepdim=True).values / 7.0).to(s["weight"].dtype).double()
        q = torch.round(w / torch.where(step == 0, torch.ones_like(step), step)).clamp_(-8, 7)
        return {"scales": step[..., 0], "values": (q * step).reshape(V, H)}
    h = s["hidden"].double()
    if case["op"] == "cross_entropy":
        w = s["weight"].double()
        rows = (s["labels"] >= 0).nonzero().view(-1)
        lab = s["labels"][rows]
        z = h[rows] @ w.T
        norm = torch.logsumexp(z, 1)
        N = case["rows"]
        loss, lse = torch.zeros(N, dtype=torch.float64, device=h.device), torch.zeros(N, dtype=torch.float64, device=h.device)
        lse[rows] = norm
        loss[rows] = norm - z[torch.arange(len(rows), device=h.device), lab]
        p = torch.exp(z - norm.unsqueeze(1))
        del z
        p[torch.arange(len(rows), device=h.device), lab] -= 1.0
        p *= s["scale"][rows].double().unsqueeze(1)
        gh = torch.zeros_like(h)
        gh[rows] = p @ w
        return {"loss": loss, "lse": lse, "grad_hidden": gh, "grad_weight": p.T @ h[rows]}
    # column by column of a word: the same codes, taken out one position at a time
    V, words = s["packed"].shape
    G = s["scales"].shape[1]
    q = torch.empty(V, words, 8, dtype=torch.float64, device=h.device)
    for k in range(8):
        q[:, :, k] = (torch.bitwise_right_shift(s["packed"].long() & 0xFFFFFFFF, _SHIFTS[k]) % 16) - 8
    w = q.view(V, G, -1) * s["scales"].double().view(V, G, 1)
    z = h @ w.view(V, -1).T
    if case["op"] == "quantized_logits":
        return {"logits": z}
    prob = torch.softmax(z, 1)
    return {"confidence": prob.max(1).values, "predicted": None, "current": prob[torch.arange(len(h), device=h.device), s["ids"]]}


def work(case):
    V, H = case["vocab"], case["hidden"]
    if case["op"] == "quantize":
        # read the weight; write codes and scales; read those; write the values
        packed = V * H // 2 + V * (H // case["group"]) * 2
        return {"bytes": 4 * V * H + 2 * packed, "flops": 4 * V * H}
    N = case["rows"]
    if case["op"] == "cross_entropy":
        n = _kept(case)
        # logits once, their gradient against weight and hidden: three products over the kept rows
        return {"bytes": 4 * V * H + 2 * n * H + 2 * N * H + N * (8 + 4 + 8), "flops": 6 * n * V * H}
    packed = V * H // 2 + V * (H // case["group"]) * 2
    out = 2 * N * V if case["op"] == "quantized_logits" else N * (8 + 16)
    return {"bytes": packed + 2 * N * H + out, "flops": 2 * N * V * H}
