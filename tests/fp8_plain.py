"""The operators around FP8 experts in 64 bits, for the tests: straight from the formulas, plain torch on any device."""
import math

import torch

BLOCK = 128


def blocks(n):
    return -(-n // BLOCK)


def e4m3_values(dev="cpu"):
    """The 127 magnitudes of the format, in order; index = code."""
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64).to(dev)


def e4m3_round(v):
    """Nearest value, ties to the even code, at most 448."""
    values = e4m3_values(v.device)
    a = v.abs().clamp_max(448.0)
    hi = torch.searchsorted(values, a).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    up, down = values[hi] - a, a - values[lo]
    near = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(values[near], v)


def quant(x):
    """(codes as float64, scale float64 holding fp32 values) of finite rows x."""
    x = x.double()
    rows, cols = x.shape
    pad = torch.nn.functional.pad(x, (0, blocks(cols) * BLOCK - cols)).view(rows, -1, BLOCK)
    scale = (pad.abs().amax(-1) / 448.0).float().double()
    q = torch.where(scale[..., None] > 0, pad / torch.where(scale > 0, scale, 1.0)[..., None], 0.0)
    return e4m3_round(q).view(rows, -1)[:, :cols], scale


def rows64(codes, scale):
    return codes.double() * scale.double().repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def weight64(codes, scale):
    s = scale.double().repeat_interleave(BLOCK, -2)[..., :codes.shape[-2], :].repeat_interleave(BLOCK, -1)
    return codes.double() * s[..., :codes.shape[-1]]


def act(name, g, u, alpha=1.702, limit=7.0):
    if name == "silu":
        return g * torch.sigmoid(g) * u
    if name == "swiglu_clamp":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g * torch.sigmoid(alpha * g) * (u + 1)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u


def unpermute(rows, topk_row, w=None):
    """(sum, sum of magnitudes) in 64 bits."""
    ok = (topk_row >= 0) & (topk_row < rows.shape[0])
    taken = rows.double()[topk_row.clamp(0, rows.shape[0] - 1).long()] * ok[..., None]
    if w is not None:
        taken = taken * w.double()[..., None]
    return taken.sum(1), taken.abs().sum(1)


def plan(n, e, k, seed=0, dropped=0.0, num_rows=None):
    """A random plan as route_pack makes it: (topk_row, counts, offsets, num_rows), on the CPU."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(n)]) if n else torch.zeros(0, k, dtype=torch.int64)
    idx = torch.where(torch.rand(n, k, generator=g) < dropped, -1, idx)
    row = torch.full((n, k), -1, dtype=torch.int32)
    counts, offsets = torch.zeros(e, dtype=torch.int32), torch.zeros(e + 1, dtype=torch.int32)
    for x in range(e):
        t, s = torch.nonzero(idx == x, as_tuple=True)
        counts[x] = len(t)
        row[t, s] = offsets[x] + torch.arange(len(t), dtype=torch.int32)
        offsets[x + 1] = offsets[x] + (len(t) + 127) // 128 * 128
    return row, counts, offsets, num_rows or max(128, int(offsets[-1]))
