"""What is measured of the recurrent block's operators.

Four operators around the scan: the RMS norm with the residual's addition and an
8-bit output (``rms_norm``, ``rms_norm_grad``), the 8-bit quantiser
(``quantize8``), the product of 8-bit matrices with a scale for each block of
128 (``matmul8``), and the gated linear recurrence (``gated_scan``,
``gated_scan_grad``).  ``run`` is one call as a layer makes it; with ``own``
false it computes the same values from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

GROUP = 128          # columns (or rows and columns) that share a scale
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a batch of 16: the norm before the projections, to 8 bits
        {"name": "norm_step", "op": "norm", "rows": 16, "cols": 4096, "x": "bf16", "res": "bf16", "out": "e4m3"},
        # a prefill of 8192 tokens of a 64 x 64-channel layer
        {"name": "norm_prefill", "op": "norm", "rows": 8192, "cols": 4096, "x": "bf16", "res": "bf16", "out": "e4m3"},
        # a layer kept in 32 bits with a width that is no multiple of anything
        {"name": "norm_ragged", "op": "norm", "rows": 1537, "cols": 2501, "x": "f32", "res": "f32", "out": "f32"},
        # its gradient over a training batch
        {"name": "norm_grad", "op": "norm_grad", "rows": 16384, "cols": 4096, "x": "bf16", "res": "bf16"},
        # an activation or its gradient for the weight's gradient: groups along the tokens
        {"name": "quant_turned", "op": "quant", "rows": 8192, "cols": 4096, "x": "bf16", "blocks": False, "turn": True},
        # a master weight of odd size to 8 bits
        {"name": "quant_weight", "op": "quant", "rows": 4100, "cols": 1111, "x": "f32", "blocks": True, "turn": False},
        # a decode step's projection: the weights are all that is read
        {"name": "product_step", "op": "product", "m": 16, "n": 8192, "k": 4096, "blocks": True, "out": "bf16"},
        # a prefill's projection to values and gates
        {"name": "product_prefill", "op": "product", "m": 8192, "n": 8192, "k": 4096, "blocks": True, "out": "bf16"},
        # a weight's gradient over 5000 tokens, scales along the tokens on both sides
        {"name": "product_wgrad", "op": "product", "m": 4000, "n": 2500, "k": 5000, "blocks": False, "out": "f32"},
        # one token of each of 64 sequences, states updated
        {"name": "scan_step", "op": "scan", "seqs": 64, "toks": 1, "chans": 4096, "x": "bf16", "ragged": False, "train": False},
        # a long document
        {"name": "scan_long", "op": "scan", "seqs": 1, "toks": 131072, "chans": 1024, "x": "bf16", "ragged": False, "train": False},
        # a padded training batch, forward and backward
        {"name": "scan_train", "op": "scan", "seqs": 4, "toks": 8192, "chans": 2048, "x": "bf16", "ragged": True, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "quant", "product", "product", "scan", "scan"])
    if op in ("norm", "norm_grad"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.5:
            cols = max(64, cols // 128 * 128)
        rows = _log(rng, 1, max(1, min(16384, (1 << 26) // cols)))
        x = rng.choice(["bf16", "bf16", "f32"])
        res = "f32" if x == "f32" else rng.choice(["bf16", "f32", "none"])
        case = {"op": op, "rows": rows, "cols": cols, "x": x, "res": res}
        if op == "norm":
            case["out"] = rng.choice(["e4m3", "e4m3", x])
        return case
    if op == "quant":
        cols = _log(rng, 64, 16384)
        return {"op": op, "rows": _log(rng, 1, max(1, min(16384, (1 << 25) // cols))), "cols": cols,
                "x": rng.choice(["bf16", "f32"]), "blocks": rng.random() < 0.5, "turn": rng.random() < 0.5}
    if op == "product":
        m = _log(rng, 1, 8192)
        n, k = _log(rng, 128, 8192), _log(rng, 128, 8192)
        while m * n * k > 1 << 38:
            k = max(128, k // 2)
        if rng.random() < 0.5:
            n, k = max(128, n // 128 * 128), max(128, k // 128 * 128)
        blocks = rng.random() < 0.7
        return {"op": op, "m": m, "n": n, "k": k, "blocks": blocks, "out": "bf16" if blocks else "f32"}
    chans = _log(rng, 64, 8192)
    if rng.random() < 0.5:
        chans = max(64, chans // 64 * 64)
    seqs = _log(rng, 1, 64)
    train = rng.random() < 0.5
    most = (1 << 25) // (chans * seqs) if train else (1 << 26) // (chans * seqs)
    return {"op": op, "seqs": seqs, "toks": _log(rng, 1, max(1, min(65536, most))), "chans": chans,
            "x": rng.choice(["bf16", "bf16", "f32"]), "ragged": rng.random() < 0.4, "train": train}


def _groups(n):
    return -(-n // GROUP)


def work(case):
    op = case["op"]
    size = {"bf16": 2, "f32": 4, "e4m3": 1, "none": 0}
    if op == "norm":
        cells = case["rows"] * case["cols"]
        x, r, o = size[case["x"]], size[case["res"]], size[case["out"]]
        scales = 4 * case["rows"] * _groups(case["cols"]) if case["out"] == "e4m3" else 0
        return {"bytes": cells * (x + 2 * r + o) + 4 * case["cols"] + scales, "flops": 6 * cells}
    if op == "norm_grad":
        cells = case["rows"] * case["cols"]
        x, r = size[case["x"]], size[case["res"]] or size[case["x"]]
        # dout and dx in x's type, the stored sum and its gradient in the residual's
        return {"bytes": cells * (2 * x + 2 * r) + 8 * case["cols"] + 4 * case["rows"], "flops": 10 * cells}
    if op == "quant":
        cells = case["rows"] * case["cols"]
        if case["blocks"]:
            scales = _groups(case["rows"]) * _groups(case["cols"])
        elif case["turn"]:
            scales = _groups(case["rows"]) * case["cols"]
        else:
            scales = case["rows"] * _groups(case["cols"])
        return {"bytes": cells * (size[case["x"]] + 1) + 4 * scales, "flops": 3 * cells}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = _groups(k) * (m + (_groups(n) if case["blocks"] else n))
        return {"bytes": m * k + n * k + 4 * scales + m * n * size[case["out"]], "flops": 2 * m * n * k}
    cells = case["seqs"] * case["toks"] * case["chans"]
    state = 4 * case["seqs"] * case["chans"]
    b = size[case["x"]]
    if case["train"]:
        # forward: v, g read, y written; backward: v, g, dy read, dv, dg written; h0, h1, dh1, dh0
        return {"bytes": 8 * b * cells + 4 * state, "flops": 30 * cells}
    return {"bytes": 3 * b * cells + 2 * state, "flops": 10 * cells}


# --------------------------------------------------------------------------- inputs

def _randn(gen, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).add_(mean)


def _activations(gen, rows, cols):
    """Normal values, with a column in 64 ten times as large: what a residual stream looks like."""
    x = _randn(gen, rows, cols)
    x[:, torch.randperm(cols, generator=gen, device="cuda")[: max(1, cols // 64)]] *= 10.0
    return x


def _in_8_bits(x, blocks):
    """(q, scale) of x, q's rows padded to whole 16 bytes as the framework's quantiser lays them out."""
    rows, cols = x.shape
    q, scale = _quant(x, blocks)
    held = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn)
    held.view(torch.uint8)[:, :cols] = q.view(torch.uint8)
    return held[:, :cols], scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    s = {"case": dict(case)}
    if op == "norm":
        s["x"] = _activations(gen, case["rows"], case["cols"]).to(TYPES[case["x"]])
        if case["res"] != "none":
            s["res"] = _activations(gen, case["rows"], case["cols"]).to(TYPES[case["res"]])
        s["w"] = _randn(gen, case["cols"], mean=1.0, std=0.1)
    elif op == "norm_grad":
        x = _activations(gen, case["rows"], case["cols"])
        s["sum"] = x.to(TYPES[case["res"] if case["res"] != "none" else case["x"]])
        # what the forward pass kept for each row
        s["rstd"] = torch.rsqrt(s["sum"].float().square().mean(1) + EPS)
        s["dout"] = _randn(gen, case["rows"], case["cols"], std=0.01).to(TYPES[case["x"]])
        if case["res"] != "none":
            s["dsum"] = _randn(gen, case["rows"], case["cols"], std=0.01).to(s["sum"].dtype)
        s["w"] = _randn(gen, case["cols"], mean=1.0, std=0.1)
    elif op == "quant":
        s["x"] = _activations(gen, case["rows"], case["cols"]).to(TYPES[case["x"]])
    elif op == "product":
        s["a"], s["sa"] = _in_8_bits(_activations(gen, case["m"], case["k"]), False)
        s["b"], s["sb"] = _in_8_bits(_randn(gen, case["n"], case["k"], std=case["k"] ** -0.5), case["blocks"])
    else:
        shape = (case["seqs"], case["toks"])
        c, t = case["chans"], TYPES[case["x"]]
        # values and gates lie side by side in the projection's output; gates mostly keep
        vg = torch.empty(*shape, 2 * c, dtype=t, device="cuda")
        vg[..., :c] = _randn(gen, *shape, c)
        vg[..., c:] = _randn(gen, *shape, c, mean=3.0, std=2.0)
        s["v"], s["g"] = vg[..., :c], vg[..., c:]
        s["h0"] = _randn(gen, case["seqs"], c)
        s["lengths"] = None
        if case["ragged"]:
            n = torch.randint(0, case["toks"] + 1, (case["seqs"],), generator=gen, device="cuda", dtype=torch.int32)
            n[0] = case["toks"]
            s["lengths"] = n
        if case["train"]:
            s["dy"] = _randn(gen, *shape, c).to(t)
            s["dh1"] = _randn(gen, case["seqs"], c)
    return s


# --------------------------------------------------------------------------- plain forms

def _in_groups(x, dim):
    """x with dimension `dim` filled up with zeros to whole groups and cut into (groups, 128)."""
    short = -x.shape[dim] % GROUP
    if short:
        shape = list(x.shape)
        shape[dim] = short
        x = torch.cat([x, x.new_zeros(shape)], dim)
    return x.unflatten(dim, (-1, GROUP))


def _quant(x, blocks):
    rows, cols = x.shape
    if blocks:
        t = _in_groups(_in_groups(x.float(), 1), 0)              # (R, 128, C, 128)
        scale = t.abs().amax((1, 3)).clamp_min(AMAX_FLOOR) / E4M3_MAX
        t = (t / scale[:, None, :, None]).flatten(0, 1).flatten(1, 2)
    else:
        t = _in_groups(x.float(), 1)                             # (rows, C, 128)
        scale = t.abs().amax(2).clamp_min(AMAX_FLOOR) / E4M3_MAX
        t = (t / scale[:, :, None]).flatten(1, 2)
    return t[:rows, :cols].clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _spread(scale, rows, cols, blocks):
    """A scale for each value."""
    scale = scale.repeat_interleave(GROUP, 1)[:, :cols]
    return scale.repeat_interleave(GROUP, 0)[:rows] if blocks else scale


def _gates(s):
    """f and 1 - f of each token; a token past its sequence's length keeps the state."""
    g = s["g"].float()
    f, z = torch.sigmoid(g), torch.sigmoid(-g)
    v = s["v"].float()
    live = None
    if s["lengths"] is not None:
        live = torch.arange(g.shape[1], device=g.device)[None, :, None] < s["lengths"][:, None, None]
        f, z, v = f.where(live, torch.ones_like(f)), z.where(live, torch.zeros_like(z)), v.where(live, torch.zeros_like(v))
    return f, z, v, live


def _recur(a, b, first):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = first, by doubling steps."""
    a, b = a.clone(), b.clone()
    b[:, 0] += a[:, 0] * first
    step = 1
    while step < a.shape[1]:
        more = a[:, step:] * b[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        b[:, step:] += more
        step *= 2
    return b


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        t = s["x"].float()
        if "res" in s:
            t = t + s["res"].float()
        n = t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS) * s["w"]
        got = {"sum": t.to(s["res"].dtype)} if "res" in s else {}
        if case["out"] == "e4m3":
            got["out"], got["scale"] = _quant(n, False)
        else:
            got["out"] = n.to(TYPES[case["out"]])
        return got
    if op == "norm_grad":
        t, r = s["sum"].float(), s["rstd"][:, None]
        d = s["dout"].float()
        dw = (d * t * r).sum(0)
        d = d * s["w"]
        d = r * (d - t * r.square() * (d * t).mean(1, keepdim=True))
        if "dsum" in s:
            d = d + s["dsum"].float()
        return {"dx": d.to(s["dout"].dtype), "dweight": dw}
    if op == "quant":
        q, scale = _quant(s["x"].T if case["turn"] else s["x"], case["blocks"])
        return {"q": q, "scale": scale}
    if op == "product":
        a = s["a"].float() * _spread(s["sa"], case["m"], case["k"], False)
        b = s["b"].float() * _spread(s["sb"], case["n"], case["k"], case["blocks"])
        return {"out": (a @ b.T).to(TYPES[case["out"]])}
    f, z, v, live = _gates(s)
    h = _recur(f, z * v, s["h0"])
    y = (h if live is None else h.where(live, torch.zeros_like(h))).to(s["v"].dtype)
    got = {"y": y, "h1": h[:, -1]}
    if case["train"]:
        dy = s["dy"].float()
        if live is not None:
            dy = dy.where(live, torch.zeros_like(dy))
        # lam_t = dy_t + f_{t+1} lam_{t+1}: the same recurrence from the end
        back = torch.cat([torch.ones_like(f[:, :1]), f.flip(1)[:, :-1]], 1)
        lam = _recur(back, dy.flip(1), s["dh1"]).flip(1)
        before = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
        dg = lam * (before - v) * f * z
        got["dv"], got["dg"] = (lam * z).to(s["v"].dtype), dg.to(s["g"].dtype)
        got["dh0"] = lam[:, 0] * f[:, 0]
    return got


def run(state):
    if not own:
        return _plain(state)
    import helix_b200 as hx
    s, case = state, state["case"]
    op = case["op"]
    if op == "norm":
        r = hx.rms_norm(s["x"], s["w"], s.get("res"), eps=EPS, out_dtype=TYPES[case["out"]])
        got = {"out": r.out}
        if "res" in s:
            got["sum"] = r.sum
        if r.scale is not None:
            got["scale"] = r.scale
        return got
    if op == "norm_grad":
        dx, dw = hx.rms_norm_grad(s["dout"], s["sum"], s["rstd"], s["w"], s.get("dsum"))
        return {"dx": dx, "dweight": dw}
    if op == "quant":
        q, scale = hx.quantize8(s["x"], blocks=case["blocks"], transpose=case["turn"])
        return {"q": q, "scale": scale}
    if op == "product":
        return {"out": hx.matmul8(s["a"], s["sa"], s["b"], s["sb"], out_dtype=TYPES[case["out"]])}
    if not case["train"]:
        y, h1 = hx.gated_scan(s["v"], s["g"], s["h0"], lengths=s["lengths"])
        return {"y": y, "h1": h1}
    y, h1, states = hx.gated_scan(s["v"], s["g"], s["h0"], lengths=s["lengths"], keep_states=True)
    dv, dg, dh0 = hx.gated_scan_grad(s["dy"], s["v"], s["g"], states, s["dh1"], lengths=s["lengths"])
    return {"y": y, "h1": h1, "dv": dv, "dg": dg, "dh0": dh0}


# --------------------------------------------------------------------------- definitions in 64 bits

def _group_peaks(x, blocks):
    """Largest magnitude of each group, one slice of 128 columns at a time."""
    cols = [x[:, c:c + GROUP].abs().amax(1) for c in range(0, x.shape[1], GROUP)]
    peaks = torch.stack(cols, 1)
    if blocks:
        peaks = torch.stack([peaks[r:r + GROUP].amax(0) for r in range(0, x.shape[0], GROUP)], 0)
    return peaks


def _as_quantised(x, blocks):
    """The scale, and the value that is rounded to 8 bits."""
    scale = torch.clamp(_group_peaks(x, blocks), min=AMAX_FLOOR) / E4M3_MAX
    at = torch.arange(x.shape[1], device=x.device) // GROUP
    rows = torch.arange(x.shape[0], device=x.device)
    return x / scale[rows // GROUP if blocks else rows][:, at], scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        t = s["x"].double() + (s["res"].double() if "res" in s else 0.0)
        n = t / torch.sqrt((t * t).sum(1, keepdim=True) / case["cols"] + EPS) * s["w"].double()
        got = {"sum": t} if "res" in s else {}
        if case["out"] == "e4m3":
            got["out"], got["scale"] = _as_quantised(n, False)
        else:
            got["out"] = n
        return got
    if op == "norm_grad":
        t, r, d, w = s["sum"].double(), s["rstd"].double(), s["dout"].double(), s["w"].double()
        unit = t * r[:, None]
        along = torch.einsum("rc,rc,c->r", d, unit, w) / case["cols"]
        dx = r[:, None] * (d * w - unit * along[:, None])
        if "dsum" in s:
            dx = dx + s["dsum"].double()
        return {"dx": dx, "dweight": torch.einsum("rc,rc->c", d, unit)}
    if op == "quant":
        x = s["x"].double()
        q, scale = _as_quantised(x.T.contiguous() if case["turn"] else x, case["blocks"])
        return {"q": q, "scale": scale}
    if op == "product":
        m, n = case["m"], case["n"]
        out = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        for j, c in enumerate(range(0, case["k"], GROUP)):
            right = s["sb"][:, j].double()
            if case["blocks"]:
                right = right[torch.arange(n, device="cuda") // GROUP]
            part = s["a"][:, c:c + GROUP].double() @ s["b"][:, c:c + GROUP].double().T
            out += part * s["sa"][:, j].double()[:, None] * right[None, :]
        return {"out": out}
    seqs, toks, c = case["seqs"], case["toks"], case["chans"]
    g, v = s["g"].double(), s["v"].double()
    f = 1.0 / (1.0 + torch.exp(-g))
    live = torch.ones(seqs, toks, 1, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        live = (torch.arange(toks, device="cuda")[None, :] < s["lengths"][:, None])[:, :, None]
    h = s["h0"].double()
    hs = torch.empty(seqs, toks + 1, c, dtype=torch.float64, device="cuda")
    hs[:, 0] = h
    for t in range(toks):
        h = torch.where(live[:, t], h + (1.0 - f[:, t]) * (v[:, t] - h), h)
        hs[:, t + 1] = h
    got = {"y": hs[:, 1:] * live, "h1": h}
    if case["train"]:
        dy = s["dy"].double() * live
        lam = s["dh1"].double()
        dv, dg = torch.empty_like(v), torch.empty_like(v)
        for t in range(toks - 1, -1, -1):
            lam = lam + dy[:, t]
            dv[:, t] = lam * (1.0 - f[:, t])
            dg[:, t] = lam * (hs[:, t] - v[:, t]) * f[:, t] * (1.0 - f[:, t])
            lam = torch.where(live[:, t], lam * f[:, t], lam)
        got["dv"], got["dg"], got["dh0"] = dv * live, dg * live, lam
    return got
