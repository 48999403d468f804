"""The operators around FP8 experts: tokens sorted by expert and back (with their gradients), quantisation to 8 bits
with one scale per 128 values, and the matrix product of such operands, for one matrix and for one per expert.

Formulas. A plan `topk_row` [N, k] names the row that slot s of token t takes among rows sorted by expert (-1: none);
`counts` / `offsets` give each expert's rows. d(.) is the gradient of what follows.

  sort      rows[topk_row[t, s]] = x[t]                     dx[t] = sum_s drows[topk_row[t, s]]
  back      y[t] = sum_s w[t, s] rows[topk_row[t, s]]       drows[topk_row[t, s]] = w[t, s] dy[t]
                                                            dw[t, s] = <dy[t], rows[topk_row[t, s]]>
  quant     per row and 128 values: scale = max|v| / 448 (in 32 bits), code = e4m3(v / scale); v a row of x, or of the
            gated activation act(gate) * up of h = [gate | up]
  product   c[m, n] = sum_k a[m, k] sa[m, k/128] w[n, k] sw[n/128, k/128]; `transpose`: the same weights contracted
            over n, c[m, k] = sum_n a[m, n] sa[m, n/128] w[n, k] sw[n/128, k/128] (the gradient of the input)
  experts   product, where every expert's rows meet the expert's own matrix
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0


def listed():
    return [
        # one token of a decode step comes back from its two experts: latency of one small call
        dict(name="back 1 token", kind="back", tokens=1, hidden=4096, experts=8, top_k=2, dtype="bf16", weights="bf16", grad=False, dropped=0.0, skew=0.0),
        # a serving batch whose per-token row comes back from 8 of 128 experts, with the gradient of a training step
        dict(name="back grad 8191 tokens", kind="back", tokens=8191, hidden=2048, experts=128, top_k=8, dtype="bf16", weights="fp32", grad=True, dropped=0.0, skew=1.1),
        # a small serving batch sorted by expert
        dict(name="sort 64 tokens", kind="sort", tokens=64, hidden=2048, experts=128, top_k=8, dtype="bf16", grad=False, dropped=0.0, skew=1.1),
        # a training batch of a ragged length, fp16, some slots dropped for capacity, forward and gradient
        dict(name="sort grad 4095 tokens", kind="sort", tokens=4095, hidden=2880, experts=128, top_k=4, dtype="fp16", grad=True, dropped=0.03, skew=0.0),
        # a decode batch quantised on its way into the experts' rows
        dict(name="quant sorted 16 tokens", kind="quant", tokens=16, hidden=7168, experts=256, top_k=8, dtype="bf16", dropped=0.0, skew=0.0),
        # the activation between the two products of a prefill batch, width not a multiple of 128, with its gradient
        dict(name="glu grad 4096 tokens", kind="glu", tokens=4096, inter=2880, experts=128, top_k=4, dtype="bf16", act="swiglu_clamp", grad=True, skew=0.0),
        # one token through one projection (a shared expert's gate and up): the weights' bytes and latency
        dict(name="product 1 token", kind="product", rows=1, n=4096, k=7168, transpose=False, out="bf16"),
        # the same projection for a prefill batch: arithmetic
        dict(name="product 4096 tokens", kind="product", rows=4096, n=4096, k=7168, transpose=False, out="bf16"),
        # the gradient of a projection's input, sizes not multiples of 128
        dict(name="product grad 1000 tokens", kind="product", rows=1000, n=5760, k=2880, transpose=True, out="bf16"),
        # a decode batch of 16 tokens over 128 small experts
        dict(name="experts 16 tokens", kind="experts", tokens=16, experts=128, top_k=8, n=1536, k=2048, transpose=False, out="bf16", skew=1.1),
        # a prefill batch through 8 large experts' gate and up
        dict(name="experts 4096 tokens", kind="experts", tokens=4096, experts=8, top_k=2, n=28672, k=4096, transpose=False, out="bf16", skew=0.0),
        # the rows one GPU of eight receives, gradient through the down projection of its 32 experts
        dict(name="experts grad 16384 rows", kind="experts", tokens=16384, experts=32, top_k=1, n=7168, k=2048, transpose=True, out="bf16", skew=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["sort", "back", "quant", "glu", "product", "experts"])
    experts = rng.choice([8, 16, 32, 60, 64, 128, 256])
    top_k = rng.randint(1, min(8, experts))
    skew = rng.choice([0.0, 0.5, 1.1])
    if kind in ("sort", "back", "quant"):
        hidden = 8 * rng.randint(32, 896) + rng.choice([0, 0, 0, rng.randint(1, 7)])
        tokens = min(_log_int(rng, 1, 8192), max(1, 8192 * 8 * 2048 // (top_k * hidden)))
        case = dict(kind=kind, tokens=tokens, hidden=hidden, experts=experts, top_k=top_k, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    dropped=rng.choice([0.0, 0.0, 0.1]), skew=skew)
        if kind != "quant":
            case["grad"] = rng.random() < 0.5
        if kind == "back":
            case["weights"] = rng.choice(["bf16", "fp32"])
        return case
    if kind == "glu":
        inter = 8 * rng.randint(16, 448)
        tokens = min(_log_int(rng, 1, 8192), max(1, 4096 * 4 * 2880 // (top_k * inter)))
        return dict(kind=kind, tokens=tokens, inter=inter, experts=experts, top_k=top_k, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    act=rng.choice(["silu", "swiglu_clamp", "gelu_tanh"]), grad=rng.random() < 0.5, skew=skew)
    if kind == "product":
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), n=rng.randint(128, 7168), k=rng.randint(128, 7168), transpose=rng.random() < 0.35,
                    out=rng.choice(["bf16", "fp16", "fp32"]))
    n, k = 8 * rng.randint(16, 512), 16 * rng.randint(8, 256)
    experts = max(1, min(experts, 600_000_000 // (n * k)))
    return dict(kind=kind, tokens=_log_int(rng, 1, 4096), experts=experts, top_k=min(top_k, experts), n=n, k=k, transpose=rng.random() < 0.35,
                out=rng.choice(["bf16", "fp16", "fp32"]), skew=skew)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _up(v, to):
    return -(-v // to) * to


def _blocks(v):
    return -(-v // BLOCK)


def _plan(case, gen):
    """Random routes, and where they put every slot: each expert's rows start at a multiple of 128."""
    n, e, k = case["tokens"], case["experts"], case["top_k"]
    dev = "cuda"
    rank = torch.randperm(e, generator=gen, device=dev).float() + 1
    gumbel = -torch.log(-torch.log(torch.rand(n, e, generator=gen, device=dev).clamp(1e-9, 1 - 1e-7)))
    idx = (gumbel - case["skew"] * rank.log()).topk(k, dim=1).indices
    keep = torch.rand(n, k, generator=gen, device=dev) >= case.get("dropped", 0.0)
    flat = torch.where(keep, idx, e).reshape(-1)
    counts = torch.bincount(flat, minlength=e + 1)[:e]
    starts = torch.zeros(e + 1, dtype=torch.int64, device=dev)
    starts[1:] = ((counts + 127) // 128 * 128).cumsum(0)
    order = flat.argsort(stable=True)
    before = torch.zeros(e + 1, dtype=torch.int64, device=dev)
    before[1:] = counts.cumsum(0)
    row = torch.empty_like(flat)
    row[order] = torch.arange(n * k, device=dev) - before[flat[order]] + starts[flat[order]]
    row = torch.where(flat < e, row, -1)
    return dict(topk_row=row.reshape(n, k).to(torch.int32), counts=counts.to(torch.int32), offsets=starts.to(torch.int32),
                num_rows=_up(n * k + min(e, n * k) * 127, 128), most=int(counts.max()), used=n * k)


def _normal(gen, *shape):
    """Activations: normal values, a few channels an order of magnitude larger."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    return x * torch.where(torch.rand(shape[-1], generator=gen, device="cuda") < 0.01, 12.0, 1.0)


def _codes(rows, cols):
    """Room for 8-bit codes [rows, cols] whose rows start at multiples of 16 bytes, and for their scales, 128-block major."""
    q = torch.zeros(rows, _up(cols, 16), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :cols]
    s = torch.zeros(_blocks(cols), _up(rows, 4), device="cuda")[:, :rows].t()
    return q, s


def _quantised_rows(x):
    rows, cols = x.shape
    q, s = _codes(rows, cols)
    pad = torch.nn.functional.pad(x, (0, _blocks(cols) * BLOCK - cols)).view(rows, -1, BLOCK)
    scale = pad.abs().amax(-1) / E4M3_MAX
    s.copy_(scale)
    q.view(torch.uint8).copy_((pad / scale.clamp_min(1e-30)[..., None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :cols].view(torch.uint8))
    return q, s


def _weights(gen, experts, n, k):
    """Matrices of a checkpoint with one scale per 128 x 128 block."""
    ld = _up(k, 16)
    q = torch.zeros(experts, n, ld, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :, :k]
    s = torch.empty(experts, _blocks(n), _blocks(k), device="cuda")
    for e in range(experts):
        w = torch.randn(n, k, generator=gen, device="cuda") * 0.02
        w = torch.nn.functional.pad(w, (0, _blocks(k) * BLOCK - k, 0, _blocks(n) * BLOCK - n)).view(_blocks(n), BLOCK, _blocks(k), BLOCK)
        s[e] = w.abs().amax((1, 3)) / E4M3_MAX
        c = (w / s[e][:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(_blocks(n) * BLOCK, -1)
        q[e].view(torch.uint8).copy_(c[:n, :k])
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind == "product":
        into, out = (case["n"], case["k"]) if case["transpose"] else (case["k"], case["n"])
        st["a"], st["sa"] = _quantised_rows(_normal(gen, case["rows"], into))
        w, sw = _weights(gen, 1, case["n"], case["k"])
        st["w"], st["sw"] = w[0], sw[0]
        return st
    st.update(_plan(case, gen))
    n, k, r = case["tokens"], case["top_k"], st["num_rows"]
    if kind == "experts":
        into, out = (case["n"], case["k"]) if case["transpose"] else (case["k"], case["n"])
        st["a"], st["sa"] = _quantised_rows(_normal(gen, r, into))
        st["w"], st["sw"] = _weights(gen, case["experts"], case["n"], case["k"])
        st["out"] = torch.zeros(r, out, dtype=DTYPES[case["out"]], device="cuda")
        return st
    dt = DTYPES[case["dtype"]]
    if kind == "glu":
        i = case["inter"]
        st["h"] = (_normal(gen, r, 2 * i) * 2).to(dt)
        st["q"], st["s"] = _codes(r, i)
        if case["grad"]:
            st["da"], st["dh"] = _normal(gen, r, i).to(dt), torch.zeros(r, 2 * i, dtype=dt, device="cuda")
        return st
    h = case["hidden"]
    if kind == "quant":
        st["x"] = _normal(gen, n, h).to(dt)
        st["q"], st["s"] = _codes(r, h)
    elif kind == "sort":
        st["x"], st["rows"] = _normal(gen, n, h).to(dt), torch.zeros(r, h, dtype=dt, device="cuda")
        if case["grad"]:
            st["drows"] = _normal(gen, r, h).to(dt)
    else:
        st["rows"] = _normal(gen, r, h).to(dt)
        st["w"] = torch.softmax(torch.randn(n, k, generator=gen, device="cuda"), 1).to(DTYPES[case["weights"]])
        if case["grad"]:
            st["dy"], st["drows"] = _normal(gen, n, h).to(dt), torch.zeros(r, h, dtype=dt, device="cuda")
    return st


# ---- plain forms --------------------------------------------------------------------------------------------------
def _gathered(rows, topk_row):
    return torch.where((topk_row >= 0)[..., None], rows[topk_row.clamp_min(0).long()], 0)


def _scattered(into, topk_row, values):
    """into[topk_row[t, s]] = values[t, s]; what no slot names stays. Each slot of no row goes to a row of its own behind."""
    r, (n, k) = into.shape[0], topk_row.shape
    at = torch.where(topk_row >= 0, topk_row.long(), r + torch.arange(n * k, device=topk_row.device).view(n, k))
    more = torch.cat([into, into.new_zeros(n * k, into.shape[1])])
    more[at.view(-1)] = values.reshape(n * k, -1)
    into.copy_(more[:r])
    return into


def _e4m3(v):
    """Values of 64 bits to the nearest of the format, ties to even, at most 448."""
    v = v.clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).to(torch.float8_e4m3fn)


def _quantise(v):
    """Codes and scales of 32-bit rows; the quotients in 64 bits, for the values next to a border of two codes."""
    rows, cols = v.shape
    pad = torch.nn.functional.pad(v, (0, _blocks(cols) * BLOCK - cols)).view(rows, -1, BLOCK)
    scale = (pad.abs().amax(-1).double() / E4M3_MAX).float()
    quotient = torch.where(scale[..., None] > 0, pad.double() / scale.double()[..., None], 0)
    return _e4m3(quotient).view(rows, -1)[:, :cols], scale


def _act(name, g, u):
    if name == "silu":
        return g / (1 + torch.exp(-g)) * u
    if name == "swiglu_clamp":
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        return g / (1 + torch.exp(-1.702 * g)) * (u + 1)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u


def _act_grad(name, g, u, da):
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return da * u * s * (1 + g * (1 - s)), da * g * s
    if name == "swiglu_clamp":
        inside_g, inside_u = g <= 7.0, u.abs() <= 7.0
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        s = 1 / (1 + torch.exp(-1.702 * g))
        return torch.where(inside_g, da * (u + 1) * s * (1 + 1.702 * g * (1 - s)), 0), torch.where(inside_u, da * g * s, 0)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    d = 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    return da * u * d, da * 0.5 * g * (1 + t)


def _live(st):
    """Which rows hold a slot, and each row's expert and place among the expert's."""
    r = torch.arange(st["num_rows"], device="cuda")
    e = (torch.searchsorted(st["offsets"][1:].long(), r, right=True)).clamp_max(st["counts"].numel() - 1)
    place = r - st["offsets"][e]
    return e, place, place < st["counts"][e]


def _plain_rows(q, s):
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _plain_matrix(q, s):
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :q.shape[-2], :].repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "sort":
        k = st["topk_row"].shape[1]
        rows = _scattered(st["rows"], st["topk_row"], st["x"][:, None].expand(-1, k, -1))
        if not case["grad"]:
            return rows
        return rows, _gathered(st["drows"].float(), st["topk_row"]).sum(1).to(rows.dtype)
    if kind == "back":
        taken, w = _gathered(st["rows"].float(), st["topk_row"]), st["w"].float()
        y = (taken * w[..., None]).sum(1).to(st["rows"].dtype)
        if not case["grad"]:
            return y
        dy = st["dy"].float()
        drows = _scattered(st["drows"], st["topk_row"], (dy[:, None] * w[..., None]).to(y.dtype))
        return y, drows, (taken * dy[:, None]).sum(-1)
    if kind == "quant":
        q, s = _quantise(st["x"].float())
        k = st["topk_row"].shape[1]
        codes = _scattered(st["q"].view(torch.uint8), st["topk_row"], q.view(torch.uint8)[:, None].expand(-1, k, -1))
        return codes.view(torch.float8_e4m3fn), _scattered(st["s"], st["topk_row"], s[:, None].expand(-1, k, -1))
    if kind == "glu":
        live = _live(st)[2][:, None]
        g, u = st["h"].float().chunk(2, 1)
        q, s = _quantise(_act(case["act"], g, u))
        st["q"].view(torch.uint8).copy_(torch.where(live, q.view(torch.uint8), st["q"].view(torch.uint8)))
        st["s"].copy_(torch.where(live, s, st["s"]))
        if not case["grad"]:
            return st["q"], st["s"]
        dh = torch.cat(_act_grad(case["act"], g, u, st["da"].float()), 1).to(st["dh"].dtype)
        st["dh"].copy_(torch.where(live, dh, st["dh"]))
        return st["q"], st["s"], st["dh"]
    a, w = _plain_rows(st["a"], st["sa"]), _plain_matrix(st["w"], st["sw"])
    w = w if case["transpose"] else w.transpose(-1, -2)
    if kind == "product":
        return (a @ w).to(DTYPES[case["out"]])
    e, place, live = _live(st)
    at = (st["offsets"][:-1, None] + torch.arange(max(1, st["most"]), device="cuda")).clamp_max(st["num_rows"] - 1)
    c = torch.bmm(a[at], w)[e, place.clamp_max(max(1, st["most"]) - 1)]
    st["out"].copy_(torch.where(live[:, None], c.to(st["out"].dtype), st["out"]))
    return st["out"]


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _own(st):
    from xcaliber_b200 import fp8, ops

    case, kind = st["case"], st["case"]["kind"]
    if kind == "sort":
        rows = ops.permute(st["x"], st["topk_row"], out=st["rows"])
        return (rows, ops.permute_backward(st["drows"], st["topk_row"])) if case["grad"] else rows
    if kind == "back":
        y = ops.unpermute(st["rows"], st["topk_row"], st["w"])
        if not case["grad"]:
            return y
        return (y, *ops.unpermute_backward(st["dy"], st["rows"], st["topk_row"], st["w"], out=st["drows"]))
    if kind == "quant":
        return fp8.quant(st["x"], topk_row=st["topk_row"], out=(st["q"], st["s"]))
    if kind == "glu":
        q, s = fp8.glu_quant(st["h"], case["act"], counts=st["counts"], offsets=st["offsets"], out=(st["q"], st["s"]))
        if not case["grad"]:
            return q, s
        return q, s, fp8.glu_backward(st["da"], st["h"], case["act"], counts=st["counts"], offsets=st["offsets"], out=st["dh"])
    if kind == "product":
        return fp8.matmul(st["a"], st["sa"], st["w"], st["sw"], transpose=case["transpose"], out_dtype=DTYPES[case["out"]])
    return fp8.grouped_matmul(st["a"], st["sa"], st["w"], st["sw"], st["counts"], st["offsets"], transpose=case["transpose"],
                              rows_in_use=st["used"], out=st["out"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def _live_experts(case):
    """How many experts a batch reaches when every one is as likely."""
    return case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** case["tokens"])


def work(case):
    kind = case["kind"]
    if kind in ("product", "experts"):
        rows = case["rows"] if kind == "product" else case["tokens"] * case["top_k"]
        into, out = (case["n"], case["k"]) if case["transpose"] else (case["k"], case["n"])
        matrices = 1 if kind == "product" else _live_experts(case)
        weights = case["n"] * case["k"] + 4 * _blocks(case["n"]) * _blocks(case["k"])
        return {"bytes": matrices * weights + rows * (into + 4 * _blocks(into) + out * SIZE[case["out"]]), "flops": 2 * rows * case["n"] * case["k"]}
    slots = case["tokens"] * case["top_k"] * (1 - case.get("dropped", 0.0))
    es = SIZE[case["dtype"]]
    if kind == "glu":
        i = case["inter"]
        grad = 3 * i * es if case["grad"] else 0
        return {"bytes": slots * (2 * i * es + i + 4 * _blocks(i) + grad), "flops": slots * i * (30 if case["grad"] else 12)}
    h, n = case["hidden"], case["tokens"]
    plan = 4 * case["tokens"] * case["top_k"]
    if kind == "quant":
        return {"bytes": plan + n * h * es + slots * (h + 4 * _blocks(h)), "flops": 3 * n * h}
    both = (n + slots) * h * es
    if kind == "sort":
        return {"bytes": plan + both * (2 if case["grad"] else 1), "flops": slots * h if case["grad"] else 0}
    plan += case["tokens"] * case["top_k"] * SIZE[case["weights"]]
    return {"bytes": plan + both * (2 if case["grad"] else 1) + (4 * slots if case["grad"] else 0), "flops": slots * h * (5 if case["grad"] else 2)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _exact_codes(v, scale):
    """Each quotient's nearest value of the format, from the list of all of them; of two as near the one with the even code."""
    codes = torch.arange(127, device="cuda", dtype=torch.uint8)
    values = codes.view(torch.float8_e4m3fn).double()
    quotient = torch.where(scale > 0, v / torch.where(scale > 0, scale, 1), 0)
    size = quotient.abs().clamp_max(E4M3_MAX)
    hi = torch.searchsorted(values, size).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    up, down = values[hi] - size, size - values[lo]
    near = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.where(quotient < 0, -values[near], values[near])


def _exact_quant(v):
    """Codes and scales of 64-bit rows, block by block; the scale is held in 32 bits."""
    codes, scales = [], []
    for at in range(0, v.shape[1], BLOCK):
        part = v[:, at:at + BLOCK]
        scale = (part.abs().max(1).values / E4M3_MAX).float()
        codes.append(_exact_codes(part, scale.double()[:, None]))
        scales.append(scale)
    return torch.cat(codes, 1), torch.stack(scales, 1)


def _exact_placed(st, values, rows):
    """[num_rows, ...] in 64 bits, zero where no slot goes."""
    out = torch.zeros(st["num_rows"], values.shape[-1], dtype=torch.float64, device="cuda")
    t, s = torch.nonzero(st["topk_row"] >= 0, as_tuple=True)
    out[st["topk_row"][t, s].long()] = rows(t, s)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("product", "experts"):
        if case.get("rows", case.get("tokens", 0) * case.get("top_k", 1)) * case["n"] * case["k"] > 4e12:
            return None
        step = torch.arange(max(case["n"], case["k"]), device="cuda") // BLOCK
        a = st["a"].to(torch.float64) * st["sa"].double()[:, step[:st["a"].shape[1]]]
        w, sw = (st["w"][None], st["sw"][None]) if kind == "product" else (st["w"], st["sw"])
        out = torch.zeros(a.shape[0], case["k"] if case["transpose"] else case["n"], dtype=torch.float64, device="cuda")
        for e in range(w.shape[0]):
            lo, hi = (0, a.shape[0]) if kind == "product" else (int(st["offsets"][e]), int(st["offsets"][e] + st["counts"][e]))
            if hi > lo:
                m = w[e].to(torch.float64) * sw[e].double()[step[:case["n"]]][:, step[:case["k"]]]
                out[lo:hi] = torch.einsum("rn,nk->rk" if case["transpose"] else "rk,nk->rn", a[lo:hi], m)
        return out
    if kind == "glu":
        g, u = (t.requires_grad_(case["grad"]) for t in st["h"].double().tensor_split(2, dim=1))
        if case["act"] == "silu":
            v = torch.nn.functional.silu(g) * u
        elif case["act"] == "gelu_tanh":
            v = torch.nn.functional.gelu(g, approximate="tanh") * u
        else:
            gc, uc = torch.minimum(g, torch.full_like(g, 7.0)), torch.clamp(u, -7.0, 7.0)
            v = gc * torch.sigmoid(1.702 * gc) * (uc + 1)
        live = torch.zeros(st["num_rows"], 1, dtype=torch.float64, device="cuda")
        for lo, c in zip(st["offsets"].tolist(), st["counts"].tolist()):
            live[lo:lo + c] = 1
        q, s = _exact_quant(v.detach())
        if not case["grad"]:
            return q * live, s.double() * live
        # at the clamps' borders the gradient is the inside's, as autograd's clamp has it; minimum() halves it there
        dg, du = torch.autograd.grad(v, (g, u), st["da"].double())
        if case["act"] == "swiglu_clamp":
            at = g.detach() == 7.0
            dg = torch.where(at, 2 * dg, dg)
        return q * live, s.double() * live, torch.cat([dg, du], 1) * live
    if kind == "quant":
        q, s = _exact_quant(st["x"].double())
        return _exact_placed(st, q, lambda t, _: q[t]), _exact_placed(st, s.double(), lambda t, _: s.double()[t])
    t, s = torch.nonzero(st["topk_row"] >= 0, as_tuple=True)
    r = st["topk_row"][t, s].long()
    if kind == "sort":
        x = st["x"].double()
        rows = _exact_placed(st, x, lambda t, _: x[t])
        if not case["grad"]:
            return rows
        return rows, torch.zeros_like(x).index_add_(0, t, st["drows"][r].double())
    w, rows = st["w"].double(), st["rows"]
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    y.index_add_(0, t, rows[r].double() * w[t, s][:, None])
    if not case["grad"]:
        return y
    dy = st["dy"].double()
    dw = torch.zeros_like(w)
    dw[t, s] = torch.einsum("ij,ij->i", dy[t], rows[r].double())
    return y, _exact_placed(st, dy, lambda t, s: dy[t] * w[t, s][:, None]), dw
