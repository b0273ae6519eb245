"""The 4-bit-weight and expert-routing operators of quadmul_b200 as cases that can be timed and compared.

Every case is one call (or, for the gradients, one backward pass) that a serving or training program makes:

  gemm_w4          y[m, n] = x[m, k] . (codes * group scales)[n, k]^T, 16-bit x, packed signed 4-bit codes
  quantize_w4      w[n, k] -> packed codes and one scale per row and group
  moe_sort         rows of x copied into expert order, with the experts' offsets and every assignment's slot
  moe_sort_grad    its gradient: the slots' rows summed back per token
  moe_gemm_w4      gemm_w4 with one weight matrix per expert over the sorted rows
  moe_combine      y[t] = sum_j weight[t, j] . ys[slot[t, j]]
  moe_combine_grad its gradients with respect to ys and to the weights

With `own` false, run() computes these with elementary torch operations in 32 bits; with `own` true it calls quadmul_b200.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_COST = 4096 * 2 * 11008 * 4096  # the largest listed product: rows x n x k


def listed():
    return [
        # one token through a square projection of a decoder layer: the smallest call, latency counts
        {"name": "gemm_w4_decode_1x4096x4096", "op": "gemm_w4", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "group": 128, "scale": "bf16"},
        # a small odd batch on a ragged layer: k is no multiple of the group, n none of a tile; fp16 with fp32 scales
        {"name": "gemm_w4_ragged_37x1100x2208", "op": "gemm_w4", "m": 37, "n": 1100, "k": 2208, "type": "fp16", "group": 64, "scale": "fp32"},
        # a prompt of 2048 tokens through a fused query-key-value projection
        {"name": "gemm_w4_prefill_2048x12288x4096", "op": "gemm_w4", "m": 2048, "n": 12288, "k": 4096, "type": "bf16", "group": 128, "scale": "bf16"},
        # weights of one projection, as they are quantised when a checkpoint is loaded
        {"name": "quantize_w4_4096x4096", "op": "quantize_w4", "n": 4096, "k": 4096, "type": "bf16", "group": 128, "scale": "bf16"},
        # the gate and up projections of a feed-forward layer, kept in fp32 until they are quantised, in small groups
        {"name": "quantize_w4_22016x4096_fp32", "op": "quantize_w4", "n": 22016, "k": 4096, "type": "fp32", "group": 32, "scale": "fp32"},
        # experts' products of a decode step: 16 sequences, 8 of 32 experts each, about four rows an expert
        {"name": "moe_gemm_w4_decode_128rows", "op": "moe_gemm_w4", "tokens": 16, "top_k": 8, "experts": 32, "n": 4096, "k": 4096, "type": "bf16",
         "group": 128, "scale": "bf16", "drop": 0.0},
        # experts' products of a long prompt: 4096 tokens, 2 of 8 experts each
        {"name": "moe_gemm_w4_prefill_8192rows", "op": "moe_gemm_w4", "tokens": 4096, "top_k": 2, "experts": 8, "n": 11008, "k": 4096, "type": "fp16",
         "group": 128, "scale": "fp16", "drop": 0.0},
        # sorting a decode step's tokens; some sequences of the batch are padding and go nowhere
        {"name": "moe_sort_16x8", "op": "moe_sort", "tokens": 16, "top_k": 8, "experts": 64, "hidden": 4096, "type": "bf16", "ids": "int64", "drop": 0.1},
        # sorting a training batch of 8192 tokens
        {"name": "moe_sort_8192x2", "op": "moe_sort", "tokens": 8192, "top_k": 2, "experts": 8, "hidden": 4096, "type": "bf16", "ids": "int64", "drop": 0.0},
        # its gradient, at an odd count of tokens and many experts, in fp32
        {"name": "moe_sort_grad_3001x6_fp32", "op": "moe_sort_grad", "tokens": 3001, "top_k": 6, "experts": 128, "hidden": 2048, "type": "fp32", "ids": "int32",
         "drop": 0.05},
        # the experts' results of a prompt brought back to token order
        {"name": "moe_combine_4096x8", "op": "moe_combine", "tokens": 4096, "top_k": 8, "experts": 64, "hidden": 4096, "type": "bf16", "weight": "fp32", "drop": 0.0},
        # the gradients of that step in a training batch
        {"name": "moe_combine_grad_4096x4", "op": "moe_combine_grad", "tokens": 4096, "top_k": 4, "experts": 64, "hidden": 4096, "type": "fp16",
         "weight": "fp32", "drop": 0.05},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["gemm_w4", "gemm_w4", "gemm_w4", "quantize_w4", "moe_gemm_w4", "moe_gemm_w4", "moe_sort", "moe_sort_grad", "moe_combine", "moe_combine_grad"])
    kind = rng.choice(["bf16", "fp16"])
    if op in ("gemm_w4", "quantize_w4", "moe_gemm_w4"):
        # most layers have k a multiple of 32; one case in eight has any even k
        k = 2 * _log(rng, 16, 5504) if rng.random() < 0.125 else 32 * _log(rng, 2, 344)
        n = _log(rng, 64, 12288)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        case = {"op": op, "n": n, "k": k, "type": kind, "group": rng.choice([32, 64, 128, 256])}
        case["scale"] = rng.choice([kind, "fp32"])
        if op == "quantize_w4":
            case["type"] = rng.choice(["bf16", "fp16", "fp32"])
            case["scale"] = rng.choice([case["type"], "fp32"])
            return case
        if op == "gemm_w4":
            case["m"] = _log(rng, 1, min(4096, _COST // (n * k)))
            return case
        experts = rng.choice([4, 8, 16, 32])
        case["n"] = n = min(n, (1 << 29) // (experts * k))
        top_k = rng.choice([1, 2, 3, 4])
        return {**case, "experts": experts, "top_k": top_k, "tokens": _log(rng, 1, min(4096, _COST // (n * k * top_k))), "drop": rng.choice([0.0, 0.1])}
    case = {"op": op, "tokens": _log(rng, 1, 8192), "top_k": rng.choice([1, 2, 4, 6, 8]), "experts": rng.choice([4, 8, 60, 128, 256]),
            "hidden": rng.choice([64, 120, 1000, 2048, 4096, 5119]), "type": rng.choice(["bf16", "fp16", "fp32"]), "drop": rng.choice([0.0, 0.0, 0.2])}
    case["tokens"] = max(1, min(case["tokens"], (1 << 28) // (case["top_k"] * case["hidden"] * _BYTES[case["type"]])))
    case["top_k"] = min(case["top_k"], case["experts"])
    if op.startswith("moe_sort"):
        case["ids"] = rng.choice(["int32", "int64"])
    else:
        case["weight"] = rng.choice([case["type"], "fp32"])
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------


def _activations(rows, width, kind, gen):
    """Normal values whose channels differ in size, as the activations of a trained network do."""
    size = torch.exp(0.5 * torch.randn(width, device="cuda", generator=gen))
    return (torch.randn(rows, width, device="cuda", generator=gen) * size).to(_TYPES[kind])


def _weights(lead, n, k, group, scale, gen):
    """Packed codes and scales of normal weights quantised by their groups' largest value."""
    groups = -(-k // group)
    w = torch.zeros(lead * n, groups * group, device="cuda")
    w[:, :k] = 0.02 * torch.randn(lead * n, k, device="cuda", generator=gen)
    w = w.view(lead * n, groups, group)
    scales = (w.abs().amax(-1) / 7).to(_TYPES[scale])
    q = torch.clamp(torch.round(w / scales.float().unsqueeze(-1)), -8, 7).to(torch.int8).view(lead * n, -1)[:, :k]
    packed = (q[:, 0::2] & 0xF) | (q[:, 1::2] << 4)
    return packed.view(lead, n, k // 2).contiguous(), scales.view(lead, n, groups).contiguous()


def _router(case, gen):
    """Expert of every assignment [tokens, top_k] (-1: dropped), as a router's top-k gives them, and its weights."""
    t, e, top = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn(t, e, device="cuda", generator=gen) + 0.5 * torch.randn(e, device="cuda", generator=gen)
    value, ids = torch.topk(logits, top, dim=1)
    weights = torch.softmax(value, dim=1)
    if case["drop"] > 0:
        ids = torch.where(torch.rand(t, 1, device="cuda", generator=gen) < case["drop"], -1, ids)
    return ids, weights


def _order(ids, experts):
    """Offsets [experts + 1] and slots [tokens, top_k] of a stable sort by expert; -1 where an assignment is dropped."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    place = torch.argsort(key, stable=True)
    slots = torch.empty_like(place)
    slots[place] = torch.arange(flat.numel(), device=flat.device)
    slots = torch.where(key < experts, slots, -1)
    counts = (key.unsqueeze(0) == torch.arange(experts, device=flat.device).unsqueeze(1)).sum(1)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.cumsum(counts, 0)
    return offsets.int(), slots.int().view(ids.shape)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, kind = case["op"], case["type"]
    s = {"op": op, "case": case}
    if op == "gemm_w4":
        b, scales = _weights(1, case["n"], case["k"], case["group"], case["scale"], gen)
        s.update(x=_activations(case["m"], case["k"], kind, gen), b=b[0], scales=scales[0], group=case["group"])
    elif op == "quantize_w4":
        s.update(w=(0.02 * torch.randn(case["n"], case["k"], device="cuda", generator=gen)).to(_TYPES[kind]), group=case["group"], scale=_TYPES[case["scale"]])
    elif op == "moe_gemm_w4":
        ids, _ = _router(case, gen)
        offsets, _ = _order(ids, case["experts"])
        rows = case["tokens"] * case["top_k"]
        b, scales = _weights(case["experts"], case["n"], case["k"], case["group"], case["scale"], gen)
        s.update(x=_activations(rows, case["k"], kind, gen), b=b, scales=scales, offsets=offsets, group=case["group"],
                 # the most rows that one expert has: how large a batched product has to be
                 capacity=int((offsets[1:] - offsets[:-1]).max()),
                 # rows behind the last expert's stay as they are
                 out=torch.zeros(rows, case["n"], dtype=_TYPES[kind], device="cuda"))
    else:
        ids, weights = _router(case, gen)
        rows, width = case["tokens"] * case["top_k"], case["hidden"]
        offsets, slots = _order(ids, case["experts"])
        if op == "moe_sort":
            s.update(x=_activations(case["tokens"], width, kind, gen), ids=ids.to(getattr(torch, case["ids"])), experts=case["experts"],
                     out=torch.zeros(rows, width, dtype=_TYPES[kind], device="cuda"))
        elif op == "moe_sort_grad":
            s.update(d=_activations(rows, width, kind, gen), slots=slots)
        elif op == "moe_combine":
            s.update(ys=_activations(rows, width, kind, gen), slots=slots, weights=weights.to(_TYPES[case["weight"]]))
        else:
            s.update(ys=_activations(rows, width, kind, gen), slots=slots, weights=weights.to(_TYPES[case["weight"]]),
                     dy=_activations(case["tokens"], width, kind, gen), out=torch.zeros(rows, width, dtype=_TYPES[kind], device="cuda"))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------


def _unpacked(b):
    """Packed codes [..., k/2] -> signed values [..., k] in fp32; the even element is in the low nibble."""
    b = b.to(torch.int32)
    low, high = (b << 28) >> 28, (b << 24) >> 28
    return torch.stack([low, high], -1).view(*b.shape[:-1], -1).float()


def _dequantised(b, scales, group):
    q = _unpacked(b)
    at = torch.arange(q.shape[-1], device=q.device) // group
    return q * scales.float()[..., at]


def run(state):
    op = state["op"]
    if own:
        import quadmul_b200 as qm

        if op == "gemm_w4":
            return qm.gemm_w4(state["x"], state["b"], state["scales"], state["group"])
        if op == "quantize_w4":
            packed, scales = qm.quantize_w4(state["w"], state["group"], scale_dtype=state["scale"])
            return {"codes": qm.unpack(packed), "scales": scales}
        if op == "moe_gemm_w4":
            return qm.moe_gemm_w4(state["x"], state["b"], state["scales"], state["offsets"], state["group"], out=state["out"])
        if op == "moe_sort":
            xs, offsets, slots = qm.moe_sort(state["x"], state["ids"], state["experts"], out=state["out"])
            return {"xs": xs, "offsets": offsets, "slots": slots}
        if op == "moe_sort_grad":
            return qm.moe_sort_grad(state["d"], state["slots"])
        if op == "moe_combine":
            return qm.moe_combine(state["ys"], state["slots"], state["weights"])
        dys, dweights = qm.moe_combine_grad(state["dy"], state["ys"], state["slots"], state["weights"], out=state["out"])
        return {"dys": dys, "dweights": dweights}

    if op == "gemm_w4":
        return (state["x"].float() @ _dequantised(state["b"], state["scales"], state["group"]).T).to(state["x"].dtype)
    if op == "quantize_w4":
        w, group = state["w"].float(), state["group"]
        n, k = w.shape
        groups = -(-k // group)
        padded = torch.zeros(n, groups * group, device=w.device)
        padded[:, :k] = w
        padded = padded.view(n, groups, group)
        scales = (padded.abs().amax(-1) / 7).to(state["scale"])
        # quotients next to the middle between two codes need 64 bits
        codes = torch.round(padded.double() / scales.double().unsqueeze(-1)).nan_to_num(0.0).clamp(-8, 7)
        return {"codes": codes.to(torch.int8).view(n, -1)[:, :k].contiguous(), "scales": scales}
    if op == "moe_gemm_w4":
        x, offsets, rows = state["x"].float(), state["offsets"].long(), state["x"].shape[0]
        row = torch.arange(rows, device=x.device)
        # expert of every row: how many experts end at or before it; a batch of equal size for every expert
        expert = (row.unsqueeze(1) >= offsets[1:]).sum(1)
        live = (expert < offsets.numel() - 1).unsqueeze(1)
        expert = expert.clamp(max=offsets.numel() - 2)
        place = (row - offsets[expert]).clamp(max=max(0, state["capacity"] - 1))
        batch = torch.zeros(offsets.numel() - 1, max(1, state["capacity"]), x.shape[1], device=x.device)
        batch.index_put_((expert, place), torch.where(live, x, 0.0), accumulate=True)
        y = torch.bmm(batch, _dequantised(state["b"], state["scales"], state["group"]).transpose(1, 2))
        return torch.where(live, y[expert, place].to(state["x"].dtype), state["out"])
    if op == "moe_sort":
        offsets, slots = _order(state["ids"], state["experts"])
        at = slots.reshape(-1).long()
        top = slots.shape[1]
        source = torch.arange(at.numel(), device=at.device) // top
        # one spare row takes the dropped assignments
        xs = torch.cat([state["out"], state["out"][:1]])
        xs[torch.where(at >= 0, at, at.numel())] = state["x"][source]
        return {"xs": xs[:-1], "offsets": offsets, "slots": slots}
    slots = state["slots"].long()
    live = (slots >= 0).unsqueeze(-1)
    if op == "moe_sort_grad":
        return torch.where(live, state["d"][slots.clamp(min=0)].float(), 0.0).sum(1).to(state["d"].dtype)
    rows = torch.where(live, state["ys"][slots.clamp(min=0)].float(), 0.0)
    if op == "moe_combine":
        return (rows * state["weights"].float().unsqueeze(-1)).sum(1).to(state["ys"].dtype)
    dy = state["dy"].float()
    dweights = (rows * dy.unsqueeze(1)).sum(-1).to(state["weights"].dtype)
    dys = torch.cat([state["out"], state["out"][:1]])
    back = (state["weights"].float().unsqueeze(-1) * dy.unsqueeze(1)).to(state["ys"].dtype)
    at = slots.reshape(-1)
    dys[torch.where(at >= 0, at, at.numel())] = back.view(at.numel(), -1)
    return {"dys": dys[:-1], "dweights": dweights}


def work(case):
    """Bytes that one pass has to read and write, and its multiplications and additions."""
    op, size = case["op"], _BYTES[case["type"]]
    if op in ("gemm_w4", "quantize_w4", "moe_gemm_w4"):
        n, k = case["n"], case["k"]
        packed = n * k // 2 + n * -(-k // case["group"]) * _BYTES[case["scale"]]
        if op == "gemm_w4":
            return {"bytes": packed + case["m"] * (k + n) * size, "flops": 2 * case["m"] * n * k}
        if op == "quantize_w4":
            return {"bytes": n * k * size + packed, "flops": 4 * n * k}
        rows = round(case["tokens"] * case["top_k"] * (1 - case["drop"]))
        # experts that at least one token chose
        active = case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** (case["tokens"] * (1 - case["drop"])))
        return {"bytes": int(active * packed) + rows * (k + n) * size, "flops": 2 * rows * n * k}
    width, tokens, top = case["hidden"], case["tokens"], case["top_k"]
    rows = round(tokens * top * (1 - case["drop"]))
    if op == "moe_sort":
        ids = 8 if case["ids"] == "int64" else 4
        return {"bytes": (tokens + rows) * width * size + tokens * top * (ids + 4) + 4 * (case["experts"] + 1), "flops": 0}
    index = tokens * top * 4
    if op == "moe_sort_grad":
        return {"bytes": (tokens + rows) * width * size + index, "flops": rows * width}
    index += tokens * top * _BYTES[case["weight"]]
    if op == "moe_combine":
        return {"bytes": (tokens + rows) * width * size + index, "flops": 2 * rows * width}
    return {"bytes": (tokens + 2 * rows) * width * size + index + tokens * top * _BYTES[case["weight"]], "flops": 3 * rows * width}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def _weights64(b, scales, group):
    """Row by row of the definition: w[.., i] = code(i) * scale[.., i // group]."""
    code = b.to(torch.int64) & 0xFF
    both = torch.empty(*b.shape[:-1], 2 * b.shape[-1], dtype=torch.float64, device=b.device)
    for half, nibble in ((0, code % 16), (1, code // 16)):
        both[..., half::2] = torch.where(nibble > 7, nibble - 16, nibble).double()
    return both * scales.double().repeat_interleave(group, dim=-1)[..., : both.shape[-1]]


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "gemm_w4":
        return torch.matmul(s["x"].double(), _weights64(s["b"], s["scales"], s["group"]).t())
    if op == "quantize_w4":
        w, group = s["w"].double(), s["group"]
        largest = [w[:, at : at + group].abs().max(dim=1).values for at in range(0, w.shape[1], group)]
        return {"codes": None, "scales": torch.stack(largest, 1) / 7}
    if op == "moe_gemm_w4":
        out, ends = s["out"].double(), s["offsets"].tolist()
        for e in range(case["experts"]):
            first, last = ends[e], ends[e + 1]
            if last > first:
                out[first:last] = s["x"][first:last].double() @ _weights64(s["b"][e], s["scales"][e], s["group"]).t()
        return out
    if op == "moe_sort":
        ids, out = s["ids"].reshape(-1), s["out"].double()
        order = torch.cat([torch.nonzero(ids == e).reshape(-1) for e in range(case["experts"])])
        out[: order.numel()] = s["x"].double()[torch.div(order, case["top_k"], rounding_mode="floor")]
        return {"xs": out, "offsets": None, "slots": None}
    slots, tokens = s["slots"].long(), case["tokens"]
    width = case["hidden"]
    if op == "moe_combine_grad":
        dys, dweights = s["out"].double(), torch.zeros(slots.shape, dtype=torch.float64, device="cuda")
        for j in range(case["top_k"]):
            on = torch.nonzero(slots[:, j] >= 0).reshape(-1)
            at = slots[on, j]
            dys[at] = s["dy"][on].double() * s["weights"][on, j].double().unsqueeze(1)
            dweights[on, j] = torch.einsum("th,th->t", s["dy"][on].double(), s["ys"][at].double())
        return {"dys": dys, "dweights": dweights}
    y = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        on = torch.nonzero(slots[:, j] >= 0).reshape(-1)
        part = (s["d"] if op == "moe_sort_grad" else s["ys"])[slots[on, j]].double()
        y[on] += part if op == "moe_sort_grad" else part * s["weights"][on, j].double().unsqueeze(1)
    return y
