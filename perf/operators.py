"""Products of a network's layers as cases to time: 8-bit products with a scale for each row and each column, and the gated unit
act(Y t(Wg) + bg) * (Y t(Wu) + bu) in 8 bits and in the operands' own type, with its gradients.

A case is one call of a layer on the device: the rows Y (tokens, or rows of a table), weights that stay in HBM between the calls (one row of
weights per output column; of a gated unit the gate's nOut rows first, then the other projection's), an output that the caller holds. `own`
chooses between the plain form in elementary torch operations and the library's entry points. Eight bits: a row of Y is x / s rounded to the
nearest whole number, ties to even, s = (largest magnitude of the row) / 127 in fp32; a column of weights likewise.
"""
import math

import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST_FLOPS = 1.1e12


def listed():
    return [
        # One token through a projection: weights once through the chip, and a launch.
        {"name": "q8_token", "op": "q8", "type": "bf16", "rows": 1, "inp": 4096, "out": 4096, "bias": False},
        # A few sequences' tokens together, odd sizes, with a bias.
        {"name": "q8_tokens_odd", "op": "q8", "type": "f16", "rows": 37, "inp": 5001, "out": 7681, "bias": True},
        # Rows of a decompressed table (fp64, as the library's matrices are) through a first layer.
        {"name": "q8_table", "op": "q8", "type": "f64", "rows": 100_003, "inp": 100, "out": 512, "bias": True},
        # A long prompt: rows quantised once for two weight matrices of unlike widths.
        {"name": "q8_shared", "op": "q8_shared", "type": "bf16", "rows": 8192, "inp": 8192, "out": 7168, "out2": 1024, "bias": False},
        # The gated unit of one token.
        {"name": "q8_gate_token", "op": "q8_gate", "type": "bf16", "rows": 1, "inp": 4096, "out": 12288, "bias": False, "act": "silu"},
        # ... of a long prompt.
        {"name": "q8_gate", "op": "q8_gate", "type": "bf16", "rows": 4096, "inp": 4096, "out": 12288, "bias": False, "act": "silu"},
        # The gated unit in 16 bits: four tokens of four sequences.
        {"name": "gate_token", "op": "gate", "type": "bf16", "rows": 4, "inp": 4096, "out": 12288, "bias": False, "act": "silu"},
        # ... a training batch.
        {"name": "gate", "op": "gate", "type": "bf16", "rows": 4096, "inp": 4096, "out": 12288, "bias": False, "act": "silu"},
        # In fp32 with biases, odd sizes.
        {"name": "gate_f32_odd", "op": "gate", "type": "f32", "rows": 1021, "inp": 1001, "out": 1531, "bias": True, "act": "gelu"},
        # A gated linear unit as the first layer over a table, in fp64.
        {"name": "gate_table", "op": "gate", "type": "f64", "rows": 400_009, "inp": 100, "out": 64, "bias": True, "act": "sigmoid"},
        # The training batch's gradients.
        {"name": "gate_backward", "op": "gate_backward", "type": "bf16", "rows": 4096, "inp": 4096, "out": 8192, "bias": False, "act": "silu"},
        # The table's gradients: sums over many rows into few weights.
        {"name": "gate_backward_table", "op": "gate_backward", "type": "f64", "rows": 100_003, "inp": 100, "out": 64, "bias": True, "act": "sigmoid"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["q8", "q8", "q8_shared", "q8_gate", "q8_gate", "gate", "gate", "gate_backward", "gate_backward"])
    c = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32", "f64"])}
    c["bias"] = rng.random() < 0.5
    if rng.random() < 0.2:  # rows of a table
        c.update(rows=_log(rng, 10_000, 100_000), inp=rng.randint(8, 200), out=_log(rng, 16, 512))
    else:
        c.update(rows=_log(rng, 1, 8192), inp=_log(rng, 64, 8192), out=_log(rng, 64, 12288))
        if rng.random() < 0.5:  # layers are mostly of whole multiples
            c.update(inp=-(-c["inp"] // 64) * 64, out=-(-c["out"] // 64) * 64)
    if op == "q8_shared":
        c["out2"] = _log(rng, 64, 2048)
    if "gate" in op:
        c["act"] = rng.choice(["silu", "gelu", "gelu_tanh", "sigmoid", "relu", "none"])
    # fp32 and fp64 are a sixteenth and a thirtieth of the 16-bit rate: smaller work
    most = MOST_FLOPS / (1 if c["type"] in ("bf16", "f16") or ("q8" in op and c["type"] == "f32") else 16)
    while work(c)["flops"] > most:
        c["rows"] = max(1, c["rows"] // 2)
        if c["rows"] == 1:
            break
    return c


# ---- inputs, made on the GPU

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _inputs(case, seed):
    """Rows Y with a few wide columns among them (what makes a scale for each row necessary), weights of variance 1 / nIn, biases, an
    incoming gradient."""
    g, t = _gen(seed), TYPES[case["type"]]
    m, k, n = case["rows"], case["inp"], case["out"]
    wide = 1 + 15 * (torch.rand(k, device="cuda", generator=g) < 0.01).float()

    def normal(rows, cols, by=1.0):
        x = torch.empty(rows, cols, dtype=t, device="cuda")
        for r in range(0, rows, 8192):
            x[r:r + 8192] = torch.randn(min(8192, rows - r), cols, device="cuda", generator=g).mul_(by).to(t)
        return x

    d = {"Y": normal(m, k)}
    for r in range(0, m, 8192):
        d["Y"][r:r + 8192] *= wide.to(t)
    if m >= 64:  # the rows behind a batch's last token
        d["Y"][m - m // 64:] = 0
    widths = [n, case["out2"]] if case["op"] == "q8_shared" else [2 * n if "gate" in case["op"] else n]
    d["W"] = [normal(w, k, k ** -0.5) for w in widths]
    d["b"] = [normal(1, w, 0.1).reshape(w) if case["bias"] else None for w in widths]
    if case["op"] == "gate_backward":
        d["G"] = normal(m, n)
    if "q8" in case["op"]:  # 8-bit weights and their scales are what a program loads
        q = [_quantise(w) for w in d.pop("W")]
        d["Wq"], d["Ws"] = [x for x, _ in q], [s for _, s in q]
    return d


def _quantise(x):
    """(whole numbers as int8, fp32 scales) of each row; the quotients in 64 bits, since next to a half fp32 rounds to the other side."""
    q, s = torch.empty(x.shape, dtype=torch.int8, device=x.device), torch.empty(x.shape[0], device=x.device)
    step = max(1, (1 << 26) // x.shape[1])
    for r in range(0, x.shape[0], step):
        y = x[r:r + step].double()
        s[r:r + step] = (y.abs().amax(1).float() / 127)
        by = s[r:r + step].double()[:, None]
        q[r:r + step] = torch.where(by > 0, torch.round(y / by.clamp(min=1e-300)), torch.zeros_like(y)).clamp_(-127, 127).to(torch.int8)
    return q, s


def prepare(case, seed):
    """Operands, weights on the device, outputs; with `own` the weights' handles, laid out once, and the workspace."""
    t, m, k, n = TYPES[case["type"]], case["rows"], case["inp"], case["out"]
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from systemds_amd import capi
        torch.cuda.init()
        capi.init(torch.cuda.current_device())
        s["capi"], s["stream"] = capi, torch.cuda.current_stream().cuda_stream
        s["type"] = capi.TYPES[case["type"]]
        s["act"] = capi.ACTIVATIONS[case["act"]] if "act" in case else 0
        if "q8" in case["op"]:
            s["h"] = []
            for q, scale in zip(s["Wq"], s["Ws"]):
                h = capi.ClaQ8(k, q.shape[0])
                h.set_stream(s["stream"])
                h.set_values_dev(q.data_ptr(), k, scale.data_ptr(), by_column=True)
                s["h"].append(h)
            s["out"] = [torch.empty(m, n if "gate" in case["op"] else q.shape[0], dtype=t, device="cuda") for q in s["Wq"]]
            ws = s["h"][0].workspace(m)
            if case["op"] == "q8_shared":
                s["ldq"] = -(-k // 16) * 16
                s["q"], s["qs"] = torch.empty(m, s["ldq"], dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
        else:
            back = case["op"] == "gate_backward"
            ws = capi.gate_workspace(s["type"], m, k, n, back)
            if back:
                s["out"] = [torch.empty(m, k, dtype=t, device="cuda"), torch.empty(2 * n, k, dtype=t, device="cuda")]
                s["out"] += [torch.empty(2 * n, dtype=t, device="cuda")] if case["bias"] else []
            else:
                s["out"] = [torch.empty(m, n, dtype=t, device="cuda")]
        s["ws_bytes"], s["ws"] = ws, torch.empty(max(ws, 1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return s


# ---- the plain form: 32 bits, 64 for fp64 operands and for the quotients of the quantisation

def _act(x, kind):
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if kind == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    return x


def _act_slope(x, kind):
    if kind == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 - s)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    if kind == "relu":
        return (x > 0).to(x.dtype)
    return torch.ones_like(x)


def _plain(state):
    case = state["case"]
    t = TYPES[case["type"]]
    wide = torch.float64 if t == torch.float64 else torch.float32
    n = case["out"]
    if "q8" in case["op"]:
        q, s = _quantise(state["Y"])
        q, s = q.to(wide), s.to(wide)[:, None]
        outs = []
        for wq, ws, b in zip(state["Wq"], state["Ws"], state["b"]):
            o = (q @ wq.to(wide).t()) * (s * ws.to(wide))
            if b is not None:
                o = o + b.to(wide)
            if case["op"] == "q8_gate":
                o = _act(o[:, :n], case["act"]) * o[:, n:]
            outs.append(o.to(t))
        return outs
    y, w, b = state["Y"].to(wide), state["W"][0].to(wide), state["b"][0]
    o = y @ w.t()
    if b is not None:
        o = o + b.to(wide)
    g, u = o[:, :n], o[:, n:]
    if case["op"] == "gate":
        return [(_act(g, case["act"]) * u).to(t)]
    d = state["G"].to(wide)
    p = torch.cat([d * u * _act_slope(g, case["act"]), d * _act(g, case["act"])], 1)
    outs = [(p @ w).to(t), (p.t() @ y).to(t)]
    return outs + [p.sum(0).to(t)] if b is not None else outs


def run(state):
    if not own:
        return _plain(state)
    case, Y = state["case"], state["Y"]
    m, k, n = case["rows"], case["inp"], case["out"]
    b = [None if x is None else x.data_ptr() for x in state["b"]]
    ws, ws_bytes, t, out = state["ws"].data_ptr(), state["ws_bytes"], state["type"], state["out"]
    if case["op"] == "q8":
        state["h"][0].lmm_dev_async(Y.data_ptr(), t, m, k, b[0], out[0].data_ptr(), n, ws, ws_bytes)
    elif case["op"] == "q8_gate":
        state["h"][0].gate_dev_async(state["act"], Y.data_ptr(), t, m, k, b[0], out[0].data_ptr(), n, ws, ws_bytes)
    elif case["op"] == "q8_shared":
        q, qs, ldq = state["q"].data_ptr(), state["qs"].data_ptr(), state["ldq"]
        state["capi"].quantize_rows_dev_async(Y.data_ptr(), t, m, k, k, q, ldq, qs, state["stream"])
        for h, bias, o in zip(state["h"], b, out):
            h.lmm_quantized_dev_async(q, ldq, qs, m, bias, o.data_ptr(), t, h.n_cols)
    elif case["op"] == "gate":
        state["capi"].gate_dev_async(state["act"], t, Y.data_ptr(), m, k, k, state["W"][0].data_ptr(), k, b[0], n, out[0].data_ptr(), n, ws, ws_bytes,
                                     state["stream"])
    else:
        state["capi"].gate_backward_dev_async(state["act"], t, Y.data_ptr(), m, k, k, state["W"][0].data_ptr(), k, b[0], n, state["G"].data_ptr(), n,
                                              out[0].data_ptr(), k, out[1].data_ptr(), k, out[2].data_ptr() if len(out) > 2 else None, ws, ws_bytes,
                                              state["stream"])
    return out


def work(case):
    """Operands and outputs once; 8-bit weights at a byte and a scale for each column. Multiply-adds of the projections; backward: the
    projections again, then the gradients of Y and of the weights."""
    e = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    m, k, n = case["rows"], case["inp"], case["out"]
    cols = n + case["out2"] if case["op"] == "q8_shared" else 2 * n if "gate" in case["op"] else n
    bias = e * cols if case["bias"] else 0
    flops = 2 * m * k * cols
    if "q8" in case["op"]:
        return {"bytes": e * m * k + cols * (k + 4) + bias + e * m * (n if case["op"] == "q8_gate" else cols), "flops": flops}
    if case["op"] == "gate":
        return {"bytes": e * (m * k + cols * k + m * n) + bias, "flops": flops}
    return {"bytes": e * (2 * m * k + 2 * cols * k + m * n) + 2 * bias, "flops": 3 * flops}


# ---- the definition in 64 bits, a block of rows at a time

def _phi(x):
    return 0.5 * torch.special.erfc(-x / math.sqrt(2.0))


def _value_and_slope(x, kind):
    """An activation and its derivative in 64 bits."""
    one = torch.ones_like(x)
    if kind in ("sigmoid", "silu"):
        s = torch.sigmoid(x)
        ds = torch.sigmoid(x) * torch.sigmoid(-x)
        return (s, ds) if kind == "sigmoid" else (x * s, s + x * ds)
    if kind == "gelu":
        return x * _phi(x), _phi(x) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":  # (1 + tanh(a)) / 2 is the sigmoid of 2 a
        a2 = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        s = torch.sigmoid(a2)
        return x * s, s + x * s * torch.sigmoid(-a2) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * x ** 2)
    if kind == "relu":
        return x.clamp(min=0), torch.heaviside(x, torch.zeros_like(x))
    return x, one


def exact(case, seed):
    d = _inputs(case, seed)
    m, n, kind = case["rows"], case["out"], case.get("act")
    eight = "q8" in case["op"]
    weights = [w.double() * s.double().unsqueeze(1) for w, s in zip(d["Wq"], d["Ws"])] if eight else [d["W"][0].double()]
    got = [[] for _ in weights]
    sums = [torch.zeros_like(weights[0]), torch.zeros(weights[0].shape[0], dtype=torch.float64, device="cuda")]
    for r in range(0, m, 8192):
        y = d["Y"][r:r + 8192].double()
        if eight:
            scale = (y.abs().max(dim=1, keepdim=True).values.float() / 127.0).double()
            y = torch.where(scale > 0, torch.round(y / torch.where(scale > 0, scale, torch.ones_like(scale))), torch.zeros_like(y)) * scale
        for i, w in enumerate(weights):
            z = torch.nn.functional.linear(y, w, None if d["b"][i] is None else d["b"][i].double())
            if "gate" not in case["op"]:
                got[i].append(z)
                continue
            gate, up = z.split(n, dim=1)
            value, slope = _value_and_slope(gate, kind)
            if case["op"] != "gate_backward":
                got[i].append(value * up)
                continue
            back = d["G"][r:r + 8192].double()
            pre = torch.cat((back * up * slope, back * value), dim=1)
            got[i].append(pre.mm(w))
            sums[0].addmm_(pre.t(), y)
            sums[1] += pre.sum(dim=0)
    outs = [torch.cat(x) for x in got]
    if case["op"] == "gate_backward":
        outs.append(sums[0])
        if case["bias"]:
            outs.append(sums[1])
    return outs
