"""The operators of one decoding step behind the attention: what is measured of them, and their plain forms.

Three kinds of work, in the order in which a serving program runs them for a handful of tokens:

  moe      a whole mixture-of-experts layer: top-k of the gate's logits, up projection with SwiGLU and down projection of the
           picked experts (MXFP4 weights), sum of the experts' rows by their gate weights;
  matvec   a few rows times a matrix of 4-bit weights with a scale (and possibly a zero point) per group: projections around
           the attention, the output head;
  sample   one token per row from the head's logits, with temperature, top-k, top-p and min-p, by given random numbers.

With `own` the package's operators are called, without it the same is computed with elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

SIXTEEN_BIT = {"bf16": torch.bfloat16, "f16": torch.float16}
TYPES = {"f32": torch.float32, **SIXTEEN_BIT}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ALPHA, LIMIT = 1.702, 7.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _moe(name, tokens, hidden, inter, experts, k, acts, layout="blocks", logits="f32"):
    return {"name": name, "kind": "moe", "tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts, "k": k, "acts": acts,
            "layout": layout, "logits": logits}


def _matvec(name, rows, inner, columns, group, acts, zeros, bias, out):
    return {"name": name, "kind": "matvec", "rows": rows, "inner": inner, "columns": columns, "group": group, "acts": acts, "zeros": zeros,
            "bias": bias, "out": out}


def _sample(name, rows, vocabulary, logits, temperature, top_k, top_p, min_p, masked=False, mixed=False):
    return {"name": name, "kind": "sample", "rows": rows, "vocabulary": vocabulary, "logits": logits, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "masked": masked, "mixed": mixed}


def listed():
    return [
        # decoding for one user: four experts of 128 are read
        _moe("moe_1", 1, 2880, 2880, 128, 4, "bf16"),
        # a few users of a smaller model in float16, weights as the quantiser leaves them, no size round, logits of 16 bits
        _moe("moe_5_f16_strided", 5, 2016, 1056, 32, 4, "f16", "strided", "f16"),
        # a small batch: about 50 experts with one or two rows each
        _moe("moe_16", 16, 2880, 2880, 128, 4, "bf16"),
        # the largest batch that counts as a few tokens: nearly every expert is read
        _moe("moe_64", 64, 2880, 2880, 128, 4, "bf16"),
        # one user's projection in front of the attention, fine groups
        _matvec("matvec_1_projection", 1, 2880, 5120, 32, "bf16", False, True, "bf16"),
        # a batch's projection in float16 with zero points, sizes that are not round
        _matvec("matvec_7_f16_zeros", 7, 4160, 5003, 64, "f16", True, False, "f16"),
        # one user's output head: the widest matrix of a model, logits in float32
        _matvec("matvec_1_head", 1, 4096, 131072, 128, "bf16", False, False, "f32"),
        # several prompts' last tokens and drafts together through a square projection
        _matvec("matvec_48", 48, 8192, 8192, 128, "bf16", True, False, "bf16"),
        # one user: a few hundred candidates, most of the mass
        _sample("sample_1", 1, 131072, "f32", 0.8, 50, 0.9, 0.0),
        # a batch, by mass alone
        _sample("sample_64_top_p", 64, 131072, "f32", 1.0, 0, 0.95, 0.0),
        # a few rows of 16-bit logits, a grammar masks a part of them, an odd vocabulary
        _sample("sample_7_bf16_masked", 7, 50001, "bf16", 0.7, 0, 1.0, 0.05, masked=True),
        # a large batch whose requests each come with settings of their own
        _sample("sample_256_mixed", 256, 100003, "f32", 1.0, 0, 1.0, 0.0, mixed=True),
    ]


def _spread(rng, low, high, step=1):
    """A whole multiple of `step` between `low` and `high`, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, round(v / step) * step))


def draw(rng):
    kind = rng.choice(("moe", "matvec", "sample"))
    if kind == "moe":
        hidden, inter = _spread(rng, 512, 5760, 32), _spread(rng, 256, 2880, 32)
        most = 1.7e9 / (3 * hidden * inter * 0.53)      # experts that fit: bytes of the widest listed layer
        experts = rng.choice([e for e in (8, 16, 32, 60, 64, 128) if e <= most] or [8])
        k = rng.choice((1, 2, 4, 4, 6, 8))
        tokens = _spread(rng, 1, max(1, min(64, int(256 * 2880 * 2880 / (k * hidden * inter)))))
        return {"kind": kind, "tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts, "k": k, "acts": rng.choice(("bf16", "bf16", "f16")),
                "layout": rng.choice(("blocks", "blocks", "strided")), "logits": rng.choice(("f32", "bf16", "f16"))}
    if kind == "matvec":
        group = rng.choice((32, 64, 128))
        rows, inner = _spread(rng, 1, 64), _spread(rng, 256, 16384, group)
        columns = _spread(rng, 64, max(64, min(131072, int(4096 * 131072 / inner))))
        acts = rng.choice(("bf16", "bf16", "f16"))
        return {"kind": kind, "rows": rows, "inner": inner, "columns": columns, "group": group, "acts": acts, "zeros": rng.choice((True, False)),
                "bias": rng.choice((True, False)), "out": rng.choice((acts, acts, "f32"))}
    rows = _spread(rng, 1, 256)
    return {"kind": kind, "rows": rows, "vocabulary": _spread(rng, 1000, min(262144, int(256 * 100003 / rows))),
            "logits": rng.choice(("f32", "f32", "bf16", "f16")), "temperature": rng.choice((0.0, 0.3, 0.7, 1.0, 1.3)),
            "top_k": rng.choice((0, 0, 1, 20, 50, 1000)), "top_p": rng.choice((1.0, 0.99, 0.9, 0.5)), "min_p": rng.choice((0.0, 0.0, 0.02, 0.1)),
            "masked": rng.choice((False, False, True)), "mixed": rng.choice((False, False, True))}


# ---------------------------------------------------------------------------------------------------------------------


def _codes(E, N, K, g):
    """Packed e2m1 codes [E, N, K/2] of normally distributed weights and their e8m0 scales [E, N, K/32] (standard deviation about 0.02):
    a value of the grid comes as often as rounding x * 2.6, x ~ N(0, 1), gives it."""
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda", dtype=torch.float64)
    q = (torch.arange(256, device="cuda", dtype=torch.float64) + 0.5) / 256
    x = 2.6 * math.sqrt(2.0) * torch.erfinv(2.0 * q - 1.0)
    code = torch.bucketize(x.abs(), edges) + 8 * (x < 0)                            # 256 equally likely nibbles
    pairs = (code[None, :] + 16 * code[:, None]).reshape(-1).to(torch.uint8)         # 65536 equally likely bytes
    values = torch.empty((E, N, K // 2), dtype=torch.uint8, device="cuda")
    for e in range(E):
        values[e] = pairs[torch.randint(0, 65536, (N, K // 2), generator=g, device="cuda", dtype=torch.int32)]
    return values, torch.randint(119, 122, (E, N, K // 32), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["kind"] == "moe":
        T, H, I, E = case["tokens"], case["hidden"], case["inter"], case["experts"]
        s["x"] = randn(T, H).to(SIXTEEN_BIT[case["acts"]])
        s["logits"] = randn(T, E).to(TYPES[case["logits"]])
        s["v1"], s["s1"] = _codes(E, 2 * I, H, g)
        s["v2"], s["s2"] = _codes(E, H, I, g)
        s["b1"], s["b2"] = 0.1 * randn(E, 2 * I), 0.1 * randn(E, H)
        if own:
            s["layer"] = _moe_weights(s)
    elif case["kind"] == "matvec":
        M, K, N, G = case["rows"], case["inner"], case["columns"], case["group"]
        acts = SIXTEEN_BIT[case["acts"]]
        s["x"] = randn(M, K).to(acts)
        s["codes"] = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
        s["scales"] = (0.004 * (1.0 + 0.2 * randn(N, K // G)).clamp_(0.2, 2.0)).to(acts)
        s["zeros"] = torch.randint(5, 12, (N, K // G), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8) if case["zeros"] else None
        s["bias"] = 0.1 * randn(N) if case["bias"] else None
        if own:
            from triton_amd.matvec import pack_int4
            zeros = s["zeros"].t() if case["zeros"] else None
            s["weights"] = pack_int4(s["codes"].t(), s["scales"].t(), zeros=zeros, group_size=G)     # once, when a model is loaded
    else:
        R, V = case["rows"], case["vocabulary"]
        logits = 2.5 * randn(R, V)
        likely = torch.randint(0, V, (R, 24), generator=g, device="cuda")           # what a text goes on with
        logits.scatter_add_(1, likely, 5.0 + 2.0 * randn(R, 24))
        if case["masked"]:
            logits.masked_fill_(torch.rand((R, V), generator=g, device="cuda") < 0.3, -math.inf)
        s["logits"] = logits.to(TYPES[case["logits"]])
        s["u"] = torch.rand(R, generator=g, device="cuda")
        pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (R,), generator=g, device="cuda")]  # noqa: E731
        s["settings"] = ([pick(0.0, 0.5, 0.8, 1.0, 1.3), pick(0, 0, 20, 50, 400).to(torch.int32), pick(1.0, 0.98, 0.9, 0.6), pick(0.0, 0.0, 0.02, 0.1)]
                         if case["mixed"] else [case["temperature"], case["top_k"], case["top_p"], case["min_p"]])
    return s


def _moe_weights(s):
    """The layer's weights as a serving program keeps them: laid out once, with the options that go with them."""
    from triton_amd.matmul import FnSpecs, FusedActivation, PrecisionConfig
    from triton_amd.swiglu import swiglu_fn
    from triton_amd.tensor import FP4, convert_layout, wrap_torch_tensor
    from triton_amd.tensor_details.layout import CDNA4MXScaleLayout, CDNA4MXValueLayout
    layer = {"activation": FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), (ALPHA, LIMIT))}
    for n in ("1", "2"):
        w, scale = s["v" + n].transpose(-1, -2), s["s" + n].transpose(-1, -2)
        if s["case"]["layout"] == "blocks":
            w = convert_layout(wrap_torch_tensor(w, dtype=FP4), CDNA4MXValueLayout())
            scale = convert_layout(wrap_torch_tensor(scale), CDNA4MXScaleLayout())
        layer["w" + n], layer["pc" + n] = w, PrecisionConfig(b_mx_scale=scale, b_microblock_size=32)
    return layer


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "moe":
            from triton_amd.moe_layer import moe_layer
            w = s["layer"]
            return moe_layer(s["x"], s["logits"], s["case"]["k"], w["w1"], s["b1"], w["w2"], s["b2"], precision_config1=w["pc1"],
                             precision_config2=w["pc2"], fused_activation=w["activation"])
        if kind == "matvec":
            from triton_amd.matvec import matvec
            return matvec(s["x"], s["weights"], s["bias"], out_dtype=TYPES[s["case"]["out"]])
        from triton_amd.sampling import sample
        temperature, top_k, top_p, min_p = s["settings"]
        return sample(s["logits"], s["u"], temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    return {"moe": _plain_moe, "matvec": _plain_matvec, "sample": _plain_sample}[kind](s)


def _dequantise(values, scales):
    """[N, K/2] packed codes and [N, K/32] scale bytes -> float32 [N, K]"""
    grid = torch.tensor(E2M1, device="cuda")
    w = torch.stack([grid[(values & 15).int()], grid[(values >> 4).int()]], -1)
    return (w.reshape(*scales.shape, 32) * torch.exp2(scales.float() - 127.0)[..., None]).flatten(-2)


def _plain_moe(s):
    x, k = s["x"].float(), s["case"]["k"]
    logits, picked = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    picked, gates = picked[:, :k], torch.exp(logits[:, :k] - logits[:, :1])
    gates = gates / gates.sum(1, keepdim=True)
    y = torch.zeros(x.shape[0], s["b2"].shape[1], device="cuda")
    for e in picked.unique().tolist():                       # every picked expert with the tokens that picked it
        t, j = torch.nonzero(picked == e, as_tuple=True)
        h = x[t] @ _dequantise(s["v1"][e], s["s1"][e]).t() + s["b1"][e]
        gate, linear = h[:, 0::2].clamp(max=LIMIT), h[:, 1::2].clamp(-LIMIT, LIMIT)
        h = gate / (1.0 + torch.exp(-ALPHA * gate)) * (linear + 1.0)
        y[t] += gates[t, j, None] * (h @ _dequantise(s["v2"][e], s["s2"][e]).t() + s["b2"][e])
    return y.to(s["x"].dtype)


def _plain_matvec(s):
    codes, scales, group = s["codes"], s["scales"].float(), s["case"]["group"]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().reshape(*scales.shape, group)
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    y = s["x"].float() @ ((q - zeros) * scales[..., None]).flatten(-2).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[s["case"]["out"]])


def _plain_sample(s):
    z = s["logits"].double()
    column = lambda v: v[:, None] if isinstance(v, torch.Tensor) else torch.full((z.shape[0], 1), v, device="cuda")  # noqa: E731
    temperature, top_k, top_p, min_p = (column(v) for v in s["settings"])
    z, order = torch.sort(z, dim=1, descending=True, stable=True)      # the order that everything goes by: ties by their index
    place = torch.arange(z.shape[1], device="cuda")[None, :]
    greedy = temperature <= 0
    w = torch.exp((z - z[:, :1]) / torch.where(greedy, 1.0, temperature.double()))
    keep = (place < top_k) | (top_k <= 0)
    mass = torch.where(keep, w, 0.0)
    before = torch.cumsum(mass, 1) - mass
    keep &= ((before < top_p.double() * mass.sum(1, keepdim=True)) | (top_p >= 1)) & (w >= min_p.double())
    keep = torch.where(greedy, place < 1, keep | (place < 1))
    total = torch.cumsum(torch.where(keep, w, 0.0), 1)
    at = (total <= s["u"].double()[:, None] * total[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(at, keep.sum(1, keepdim=True) - 1)
    return torch.gather(order, 1, at)[:, 0].int()


def work(case):
    if case["kind"] == "moe":
        T, H, I, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "k"))
        read = E * (1.0 - (1.0 - k / E) ** T)                # experts that tokens pick, each on its own, in the mean
        weights = 3 * H * I * (0.5 + 1 / 32) + 4 * (2 * I + H)
        return {"bytes": read * weights + T * (2 * H * 2 + E * BYTES[case["logits"]]), "flops": 2.0 * T * k * 3 * H * I}
    if case["kind"] == "matvec":
        M, K, N, G = (case[n] for n in ("rows", "inner", "columns", "group"))
        return {"bytes": N * K / 2 + N * (K // G) * (2.5 if case["zeros"] else 2) + M * K * 2 + M * N * BYTES[case["out"]] + 4 * N * case["bias"],
                "flops": 2.0 * M * K * N}
    R, V = case["rows"], case["vocabulary"]
    return {"bytes": R * V * BYTES[case["logits"]] + R * (8 + 16 * case["mixed"]), "flops": 3.0 * R * V}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits


def _e2m1_value(code):
    sign, exponent, mantissa = 1 - 2 * (code >> 3).double(), (code >> 1 & 3).double(), (code & 1).double()
    return sign * torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2.0 ** (exponent - 1))


def _weights64(values, scales):
    v = values.long()
    w = torch.empty((v.shape[0], 2 * v.shape[1]), dtype=torch.float64, device=v.device)
    w[:, 0::2], w[:, 1::2] = _e2m1_value(v & 15), _e2m1_value(v >> 4)
    return w * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "moe":
        T, k = case["tokens"], case["k"]
        logits = s["logits"].double().cpu().numpy()
        x = s["x"].double()
        y = torch.zeros((T, case["hidden"]), dtype=torch.float64, device="cuda")
        rows = {}                                             # expert -> (token, its gate weight)
        for t in range(T):
            best = sorted(range(case["experts"]), key=lambda e: (-logits[t, e], e))[:k]
            e = np.exp(logits[t, best] - logits[t, best].max())
            for expert, gate in zip(best, e / e.sum()):
                rows.setdefault(expert, []).append((t, float(gate)))
        for expert, those in rows.items():
            w1, w2 = _weights64(s["v1"][expert], s["s1"][expert]), _weights64(s["v2"][expert], s["s2"][expert])
            for t, gate in those:
                a = w1.mv(x[t]) + s["b1"][expert].double()
                up, linear = torch.clamp(a[0::2], max=LIMIT), torch.clamp(a[1::2], min=-LIMIT, max=LIMIT)
                y[t] += gate * (w2.mv(up * torch.sigmoid(ALPHA * up) * (1 + linear)) + s["b2"][expert].double())
        return y
    if case["kind"] == "matvec":
        y = torch.empty((case["rows"], case["columns"]), dtype=torch.float64, device="cuda")
        x, G = s["x"].double(), case["group"]
        for n in range(0, case["columns"], 4096):             # (a part of the columns at a time: 64 bits take sixteen times the room)
            c = s["codes"][n:n + 4096].long()
            q = torch.empty((c.shape[0], 2 * c.shape[1]), dtype=torch.float64, device="cuda")
            q[:, 0::2], q[:, 1::2] = (c % 16).double(), (c // 16).double()
            q -= 8 if s["zeros"] is None else s["zeros"][n:n + 4096].double().repeat_interleave(G, 1)
            q *= s["scales"][n:n + 4096].double().repeat_interleave(G, 1)
            y[:, n:n + 4096] = x.matmul(q.t())
        return y if s["bias"] is None else y + s["bias"].double()
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    settings = [v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(case["rows"], np.float32(v), np.float64) for v in s["settings"]]
    tokens = []
    for z, r, temperature, top_k, top_p, min_p in zip(logits, u, *settings):
        order = np.argsort(-z, kind="stable")
        if temperature <= 0:
            tokens.append(int(order[0]))
            continue
        w = np.exp((z[order] - z[order[0]]) / temperature)
        n = len(w) if top_k <= 0 else min(int(top_k), len(w))
        if top_p < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w[:n]), top_p * w[:n].sum(), side="left")))
        n = max(1, min(n, int((w >= min_p).sum())))
        c = np.cumsum(w[:n])
        tokens.append(int(order[min(n - 1, int(np.searchsorted(c, r * c[-1], side="right")))]))
    return torch.tensor(tokens, dtype=torch.int32)
