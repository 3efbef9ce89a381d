"""The operators around the expert products when a mixture-of-experts layer is trained: what is measured of them, and their plain forms.

Four kinds of work, as one training step of such a layer runs them beside the forward products and those with the weights transposed:

  rows     tokens sorted by expert and back: `dispatch` copies a token's row to its places among the experts' rows, `combine` adds the
           experts' rows of a token up by the gate weights; `dispatch_backward` and `combine_backward` are their gradients, those of
           the gate weights among them;
  glu      SwiGLU between the two products with its input kept in 8 bits (`swiglu_checkpoint`), and its gradient from that
           (`swiglu_backward`), which may give the activation again for the gradient of the down projection's weights;
  gate     the gradient of the picked gate weights brought back to the gate's logits (`topk_backward`);
  weights  the gradient of every expert's weights: a product over the rows of each expert (`matmul` with both operands ragged).

With `own` the package's operators are called, without it the same is computed with elementary torch operations.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ALPHA, LIMIT = 1.702, 7.0


def _rows(name, direction, tokens, hidden, experts, k, acts, gates, dropped=False):
    return {"name": name, "kind": "rows", "direction": direction, "tokens": tokens, "hidden": hidden, "experts": experts, "k": k, "acts": acts,
            "gates": gates, "dropped": dropped}


def _glu(name, direction, rows, inter, acts, again=False):
    return {"name": name, "kind": "glu", "direction": direction, "rows": rows, "inter": inter, "acts": acts, "again": again}


def _gate(name, tokens, experts, k, logits, softmax):
    return {"name": name, "kind": "gate", "tokens": tokens, "experts": experts, "k": k, "logits": logits, "softmax": softmax}


def _weights(name, tokens, k, rows, columns, experts, acts, out):
    return {"name": name, "kind": "weights", "tokens": tokens, "k": k, "rows": rows, "columns": columns, "experts": experts, "acts": acts, "out": out}


def listed():
    return [
        # a last, short batch: a launch and the trip to memory
        _rows("dispatch_64", "dispatch", 64, 2880, 128, 4, "bf16", False),
        # a batch of long texts handed to the experts
        _rows("dispatch_16384", "dispatch", 16384, 2880, 128, 4, "bf16", False),
        # a ragged batch in float16 whose experts had no room for some of the tokens
        _rows("combine_1021_f16", "combine", 1021, 2016, 60, 6, "f16", True, dropped=True),
        # the gradient of the long batch's sum: rows and gate weights
        _rows("combine_backward_16384", "combine_backward", 16384, 2880, 128, 4, "bf16", True),
        # gate weights applied in front of the experts, in float32, no size round
        _rows("dispatch_backward_4099_f32", "dispatch_backward", 4099, 1063, 32, 2, "f32", True),
        # the long batch's activation, kept in 8 bits for the backward pass
        _glu("swiglu_checkpoint_65536", "checkpoint", 65536, 2880, "bf16"),
        # its gradient, with the activation again for the weights' gradient
        _glu("swiglu_backward_65536", "backward", 65536, 2880, "bf16", again=True),
        # a short batch of a smaller model in float16, its last group of 8-bit values not full
        _glu("swiglu_backward_260_f16", "backward", 260, 1005, "f16"),
        # the gate of the long batch
        _gate("topk_backward_16384", 16384, 128, 4, "f32", True),
        # a ragged batch, 16-bit logits, gate weights without a softmax
        _gate("topk_backward_1021_bf16", 1021, 60, 6, "bf16", False),
        # a ragged batch of a smaller model: few rows per expert, the gradients' bytes count
        _weights("weights_333_f16", 333, 4, 2016, 2112, 32, "f16", "f16"),
        # the long batch, up projection: the matrix units count
        _weights("weights_16384", 16384, 4, 2880, 5760, 32, "bf16", "bf16"),
    ]


def _spread(rng, low, high, step=1):
    """A whole multiple of `step` between `low` and `high`, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, round(v / step) * step))


def draw(rng):
    kind = rng.choices(("rows", "glu", "gate", "weights"), (4, 3, 1, 2))[0]
    acts = rng.choice(("bf16", "bf16", "f16", "f32"))
    experts = rng.choice((8, 16, 32, 60, 64, 128))
    k = rng.choice((1, 2, 4, 4, 6, 8))
    if kind == "rows":
        direction = rng.choice(("dispatch", "combine", "combine_backward", "dispatch_backward"))
        hidden = _spread(rng, 64, 5760, rng.choice((1, 8, 32)))
        tokens = _spread(rng, 1, max(1, min(65536, 16384 * 4 * 2880 * 2 // (k * hidden * BYTES[acts]))))
        gates = rng.random() < (0.8 if direction.startswith("combine") else 0.3)
        return {"kind": kind, "direction": direction, "tokens": tokens, "hidden": hidden, "experts": experts, "k": k, "acts": acts, "gates": gates,
                "dropped": rng.random() < 0.25}
    if kind == "glu":
        inter = _spread(rng, 16, 5760, rng.choice((1, 16, 16)))
        direction = rng.choice(("checkpoint", "backward"))
        return {"kind": kind, "direction": direction, "rows": _spread(rng, 1, min(131072, 65536 * 2880 * 2 // (inter * BYTES[acts]))), "inter": inter,
                "acts": acts, "again": direction == "backward" and rng.random() < 0.5}
    if kind == "gate":
        experts = rng.choice((8, 32, 60, 64, 128, 256, 512))
        return {"kind": kind, "tokens": _spread(rng, 1, 16384 * 128 // experts), "experts": experts, "k": k, "logits": rng.choice(("f32", "bf16", "f16")),
                "softmax": rng.random() < 0.75}
    step = rng.choice((1, 8, 32))
    rows, columns = _spread(rng, 64, 5760, step), _spread(rng, 64, 5760, step)
    experts = rng.choice([e for e in (8, 16, 32, 60, 64, 128) if e * rows * columns <= 32 * 2880 * 5760] or [8])
    tokens = _spread(rng, 1, max(1, min(16384, int(16384 * 4 * 2880 * 5760 / (k * rows * columns)))))
    acts = rng.choice(("bf16", "bf16", "f16"))
    return {"kind": kind, "tokens": tokens, "k": k, "rows": rows, "columns": columns, "experts": experts, "acts": acts, "out": rng.choice((acts, acts, "f32"))}


# ---------------------------------------------------------------------------------------------------------------------


def _picked(T, E, k, randn):
    """[T, k] experts of T tokens: some experts are liked better than others."""
    return torch.topk(randn(T, E) + 0.5 * randn(E), k, dim=1).indices


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["kind"] == "rows":
        T, H, E, k = (case[n] for n in ("tokens", "hidden", "experts", "k"))
        acts = TYPES[case["acts"]]
        expert = _picked(T, E, k, randn).flatten()
        if case["dropped"]:                                   # picks that found no room: behind all others, without a row
            expert = torch.where(torch.rand(T * k, generator=g, device="cuda") < 0.06, E, expert)
        place = torch.empty(T * k, dtype=torch.int32, device="cuda")
        place[torch.sort(expert, stable=True).indices] = torch.arange(T * k, dtype=torch.int32, device="cuda")
        s["places"] = torch.where(expert < E, place, -1).view(T, k)
        s["gates"] = torch.softmax(randn(T, k), 1) if case["gates"] else None
        by_token, by_row = lambda: randn(T, H).to(acts), lambda: randn(T * k, H).to(acts)  # noqa: E731
        s["given"] = by_token() if case["direction"] in ("dispatch", "combine_backward") else by_row()
        if case["gates"] and case["direction"].endswith("backward"):          # what the forward pass had, for the gate weights' gradient
            s["kept"] = by_row() if case["direction"] == "combine_backward" else by_token()
        if case["dropped"] and case["direction"] in ("dispatch", "combine_backward"):
            s["into"] = torch.zeros(T * k, H, dtype=acts, device="cuda")       # rows that no token goes to stay as they are
    elif case["kind"] == "glu":
        M, N = case["rows"], case["inter"]
        acts = TYPES[case["acts"]]
        a = (randn(M, 2 * N) * torch.exp(0.7 * randn(M, 1))).to(acts)         # (the linear and the gate's limit are met)
        if case["direction"] == "checkpoint":
            s["a"] = a
        else:
            s["values"], s["scales"] = _in_8_bits(a.float())
            s["dout"] = randn(M, N).to(acts)
    elif case["kind"] == "gate":
        T, E, k = case["tokens"], case["experts"], case["k"]
        s["logits"] = (2.0 * randn(T, E)).to(TYPES[case["logits"]])
        s["indx"] = torch.topk(s["logits"].float(), k, dim=1).indices.to(torch.int16)
        s["dvals"] = randn(T, k).to(TYPES[case["logits"]])
    else:
        T, k, M, N, E = (case[n] for n in ("tokens", "k", "rows", "columns", "experts"))
        sizes = torch.bincount(_picked(T, E, k, randn).flatten(), minlength=E)
        s["sizes"], s["most"] = sizes.to(torch.int32), int(sizes.max())
        s["x"], s["d"] = randn(T * k, M).to(TYPES[case["acts"]]), randn(T * k, N).to(TYPES[case["acts"]])
        if own:
            from triton_amd.tensor import make_ragged_tensor_metadata
            s["ragged"] = make_ragged_tensor_metadata(s["sizes"], T * k)       # (the forward pass has them from the routing)
    return s


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        if kind == "rows":
            from triton_amd import dispatch as D
            if case["direction"] == "dispatch":
                return D.dispatch(s["given"], s["places"], gates=s["gates"], out=s.get("into"))
            if case["direction"] == "combine":
                return D.combine(s["given"], s["places"], gates=s["gates"])
            if case["direction"] == "combine_backward":
                return D.combine_backward(s["given"], s["places"], rows=s.get("kept"), gates=s["gates"], out=s.get("into"))
            return D.dispatch_backward(s["given"], s["places"], x=s.get("kept"), gates=s["gates"])
        if kind == "glu":
            from triton_amd.swiglu import PrecisionConfig, swiglu_backward, swiglu_checkpoint
            if case["direction"] == "checkpoint":
                return swiglu_checkpoint(s["a"], ALPHA, PrecisionConfig(limit=LIMIT))
            return swiglu_backward(s["dout"], s["values"], s["scales"], ALPHA, PrecisionConfig(limit=LIMIT), return_out=case["again"])
        if kind == "gate":
            from triton_amd.topk import topk_backward
            return topk_backward(s["logits"], s["indx"], s["dvals"], apply_softmax=case["softmax"])
        from triton_amd.matmul import PrecisionConfig as Precision
        from triton_amd.matmul import matmul
        return matmul(s["x"].t(), s["d"], None, s["ragged"], s["ragged"], precision_config=Precision(out_dtype=TYPES[case["out"]]))
    return {"rows": _plain_rows, "glu": _plain_glu, "gate": _plain_gate, "weights": _plain_weights}[kind](s)


def _plain_rows(s):
    case, places, given = s["case"], s["places"].long(), s["given"].float()
    n, there = places.numel(), places >= 0
    gates = 1.0 if s["gates"] is None else s["gates"][..., None]
    if case["direction"] in ("dispatch", "combine_backward"):
        rows = torch.zeros(n + 1, given.shape[1], device="cuda")
        rows[torch.where(there, places, n)] = given[:, None] * gates
        rows = rows[:n].to(s["given"].dtype)
        if case["direction"] == "dispatch":
            return rows
        if s["gates"] is None:
            return rows, None
        dots = (s["kept"].float()[places.clamp(min=0)] * given[:, None]).sum(-1)
        return rows, torch.where(there, dots, 0.0)
    rows = torch.where(there[..., None], given[places.clamp(min=0)], 0.0)
    total = (rows * gates).sum(1).to(s["given"].dtype)
    if case["direction"] == "combine":
        return total
    return total, None if s["gates"] is None else (rows * s["kept"].float()[:, None]).sum(-1)


def _power(e):
    """2^e in float32 for whole e of [-126, 127], and 0 for -127: by the bits, which exp2 and pow may miss by one."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _in_8_bits(a):
    """float32 [M, L] -> e4m3 values [M, L] and e8m0 scales [M, ceil(L / 32)]: the smallest powers of two that bring a group to 448 at most."""
    M, L = a.shape
    groups = torch.nn.functional.pad(a, (0, -L % 32)).view(M, -1, 32)
    most = groups.abs().amax(-1)
    part, exponent = torch.frexp(most)                        # most = part * 2^exponent, part in [1/2, 1): 448 is 0.875 * 2^9
    exponent = torch.where(most > 0, exponent - 9 + (part > 0.875), -127).clamp(min=-127)
    q = groups * _power(-exponent)[..., None]
    return q.flatten(1)[:, :L].to(torch.float8_e4m3fn), (exponent + 127).to(torch.uint8)


def _from_8_bits(values, scales):
    return values.float() * _power(scales.int() - 127).repeat_interleave(32, 1)[:, :values.shape[1]]


def _plain_glu(s):
    case = s["case"]
    a = s["a"].float() if case["direction"] == "checkpoint" else _from_8_bits(s["values"], s["scales"])
    gate, linear = a[:, 0::2].clamp(max=LIMIT), a[:, 1::2].clamp(-LIMIT, LIMIT)
    sigmoid = 1.0 / (1.0 + torch.exp(-ALPHA * gate))
    out = gate * sigmoid * (linear + 1.0)
    if case["direction"] == "checkpoint":
        return out.to(s["a"].dtype), *_in_8_bits(a)
    d, dtype = s["dout"].float(), s["dout"].dtype
    dgate = d * (linear + 1.0) * sigmoid * (1.0 + ALPHA * gate * (1.0 - sigmoid)) * (a[:, 0::2] <= LIMIT)
    dlinear = d * gate * sigmoid * (a[:, 1::2].abs() <= LIMIT)
    return torch.stack([dgate, dlinear], -1).flatten(1).to(dtype), out.to(dtype) if case["again"] else None


def _plain_gate(s):
    indx, d = s["indx"].long(), s["dvals"].float()
    if s["case"]["softmax"]:
        z = torch.gather(s["logits"].float(), 1, indx)
        p = torch.exp(z - z.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        d = p * (d - (p * d).sum(1, keepdim=True))
    return torch.zeros(s["logits"].shape, device="cuda").scatter_(1, indx, d).to(s["logits"].dtype)


def _plain_weights(s):
    at = torch.cumsum(s["sizes"], 0)[:, None] - s["sizes"][:, None]
    line = torch.arange(s["most"], device="cuda")[None, :]
    there = line < s["sizes"][:, None]                        # every expert's rows, filled up with zeros to those of the largest
    row = torch.where(there, at + line, 0)
    x = torch.where(there[..., None], s["x"].float()[row], 0.0)
    return torch.bmm(x.transpose(1, 2), s["d"].float()[row]).to(TYPES[s["case"]["out"]])


def work(case):
    if case["kind"] == "rows":
        T, H, k, size = case["tokens"], case["hidden"], case["k"], BYTES[case["acts"]]
        n = T * k * (0.94 if case["dropped"] else 1.0)
        both = case["gates"] and case["direction"].endswith("backward")
        moved = (T + n) * H + both * (n if case["direction"] == "combine_backward" else T) * H
        return {"bytes": moved * size + T * k * (4 + 4 * case["gates"] + 4 * both), "flops": (2.0 * both + 2.0) * n * H}
    if case["kind"] == "glu":
        M, N, size = case["rows"], case["inter"], BYTES[case["acts"]]
        eight = M * (2 * N + -(-2 * N // 32))
        if case["direction"] == "checkpoint":
            return {"bytes": 3 * M * N * size + eight, "flops": 14.0 * M * N}
        return {"bytes": (3 + case["again"]) * M * N * size + eight, "flops": 22.0 * M * N}
    if case["kind"] == "gate":
        T, E, k, size = case["tokens"], case["experts"], case["k"], BYTES[case["logits"]]
        return {"bytes": T * E * size + T * k * (2 + size + size * case["softmax"]), "flops": 8.0 * T * k}
    T, k, M, N, E = (case[n] for n in ("tokens", "k", "rows", "columns", "experts"))
    return {"bytes": T * k * (M + N) * BYTES[case["acts"]] + E * M * N * BYTES[case["out"]], "flops": 2.0 * T * k * M * N}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_rows(s):
    case = s["case"]
    T, k, H = case["tokens"], case["k"], case["hidden"]
    given = s["given"].double()
    kept = s["kept"].double() if "kept" in s else None
    by_row = case["direction"] in ("dispatch", "combine_backward")
    out = torch.zeros(T * k if by_row else T, H, dtype=torch.float64, device="cuda")
    dgates = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    for j in range(k):                                        # one pick of every token after the other
        token = torch.nonzero(s["places"][:, j] >= 0)[:, 0]
        row = s["places"][token, j].long()
        weight = 1.0 if s["gates"] is None else s["gates"][token, j].double()[:, None]
        if by_row:
            out.index_copy_(0, row, given.index_select(0, token) * weight)
        else:
            out.index_add_(0, token, given.index_select(0, row) * weight)
        if kept is not None:
            a, b = (kept.index_select(0, row), given.index_select(0, token)) if by_row else (given.index_select(0, row), kept.index_select(0, token))
            dgates[token, j] = a.mul_(b).sum(1)
    if case["direction"].endswith("backward"):
        return out, dgates if s["gates"] is not None else None
    return out


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_8_bits(a):
    """What the 8-bit values are from the definition: a group's scale by a search over the powers of two, every value to the nearest of its
    binade's eight steps (ties to even), and to multiples of 2^-9 below 2^-6."""
    M, L = a.shape
    G = -(-L // 32)
    values, scales = torch.empty_like(a), torch.empty(M, G, dtype=torch.uint8, device="cuda")
    powers = _power64(torch.arange(-127, 128, device="cuda"))
    for g in range(G):
        part = a[:, 32 * g:32 * g + 32]
        at = torch.searchsorted(448.0 * powers, part.abs().max(1).values, side="left")     # the first whose 448 is not below
        at = torch.where(part.abs().max(1).values == 0, 0, at)
        q = part / powers[at][:, None]
        step = _power64(torch.frexp(q.abs().clamp(min=2.0 ** -6))[1] - 4)
        values[:, 32 * g:32 * g + 32], scales[:, g] = torch.round(q / step) * step, at.to(torch.uint8)
    return values, scales


def _exact_glu(s):
    case = s["case"]
    if case["direction"] == "checkpoint":
        a = s["a"].double()
    else:
        a = s["values"].double()
        for g in range(s["scales"].shape[1]):
            a[:, 32 * g:32 * g + 32] *= _power64(s["scales"][:, g].long() - 127)[:, None]
    up, linear = torch.clamp(a[:, 0::2], max=LIMIT), torch.clamp(a[:, 1::2], min=-LIMIT, max=LIMIT)
    s1 = torch.sigmoid(ALPHA * up)
    out = up * s1 * (1 + linear)
    if case["direction"] == "checkpoint":
        return out, *_exact_8_bits(a)
    d = s["dout"].double()
    da = torch.empty_like(a)
    da[:, 0::2] = torch.where(a[:, 0::2] > LIMIT, 0.0, d * (1 + linear) * (s1 + ALPHA * up * s1 * (1 - s1)))
    da[:, 1::2] = torch.where((a[:, 1::2] > LIMIT) | (a[:, 1::2] < -LIMIT), 0.0, d * up * s1)
    return da, out if case["again"] else None


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rows":
        return _exact_rows(s)
    if case["kind"] == "glu":
        return _exact_glu(s)
    if case["kind"] == "gate":
        T, E, k = case["tokens"], case["experts"], case["k"]
        dx, d = torch.zeros(T, E, dtype=torch.float64, device="cuda"), s["dvals"].double()
        token = torch.arange(T, device="cuda")
        if case["softmax"]:
            p = torch.softmax(torch.stack([s["logits"].double()[token, s["indx"][:, j].long()] for j in range(k)], 1), 1)
            along = torch.diag_embed(p) - p[:, :, None] * p[:, None, :]       # the derivatives of every gate weight by every picked logit
            d = (along * d[:, None, :]).sum(2)
        for j in range(k):
            dx[token, s["indx"][:, j].long()] = d[:, j]
        return dx
    T, k, M, N, E = (case[n] for n in ("tokens", "k", "rows", "columns", "experts"))
    out = torch.zeros(E, M, N, dtype=torch.float64, device="cuda")
    end = 0
    for e, size in enumerate(s["sizes"].tolist()):
        start, end = end, end + size
        if size:
            out[e] = s["x"][start:end].double().t().contiguous().matmul(s["d"][start:end].double())
    return out
