"""8-bit experts: block-scaled FP8 (e4m3) operands, their products, and the gated activation between them.

The format is that of block-scaled FP8 checkpoints: weights carry one fp32 scale per 128 x 128 block, activations one per
row and 128 columns; a value is code * scale. Activation scales are kept block-major (a tensor [rows, blocks] with
strides (1, ld)), the order in which the product reads them; codes' rows start at multiples of 16 bytes. `quant`,
`glu_quant` and `quant_weight` return both in that layout.

The functions have no gradient of their own, whatever their inputs require: gradients come from `Fp8MoE.forward_routed`, or by
hand from `glu_backward` and the products with transpose=True.

All compute is in libxmoe_b200.so (through the registered ops of torch_ops.py); a missing library or a failed call raises.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib, ops, torch_ops
from ._lib import check

BLOCK = 128
_ACT = ops._ACT


def _up(v: int, to: int) -> int:
    return -(-v // to) * to


def empty_rows(rows: int, cols: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """Uninitialised (codes [rows, cols], scale [rows, ceil(cols / 128)]) in the layout described above."""
    codes = torch.empty(rows, _up(cols, 16), dtype=torch.float8_e4m3fn, device=device)[:, :cols]
    scale = torch.empty(_up(cols, BLOCK) // BLOCK, _up(rows, 4), dtype=torch.float32, device=device)[:, :rows].t()
    return codes, scale


def _zero_rows(rows: int, cols: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    codes, scale = empty_rows(rows, cols, device)
    codes.view(torch.uint8).zero_()
    scale.zero_()
    return codes, scale


def quant(x: torch.Tensor, topk_row: torch.Tensor | None = None, num_rows: int | None = None,
          out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantises rows x [M, K] (bf16 / fp16 / fp32, contiguous rows of any stride): (codes e4m3 [M, K], scale fp32
    [M, ceil(K / 128)]), scale = max|x| / 448 per 128 columns, codes to nearest, ties to even. A block of zeros has scale
    0; a block with an infinity or a NaN has NaN codes.

    With topk_row (int32 [M, k], as ops.permute takes it) every token is quantised once and its codes and scales go to the
    rows topk_row names: `quant(permute(x))` without the intermediate rows. `out` then keeps the rows that no slot names;
    without it they are zero."""
    if out is None:
        if topk_row is None:
            out = empty_rows(x.shape[0], x.shape[1], x.device)
        elif num_rows is None:
            raise RuntimeError("quant into sorted rows needs num_rows or out")
        else:
            out = _zero_rows(num_rows, x.shape[1], x.device)
    else:
        ops._refuse_grad("quant", *out)
    torch_ops.op("fp8_quant")(x, topk_row, out[0], out[1])
    return out


def quant_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantises weights [N, K] or [E, N, K] (bf16 / fp16 / fp32): (codes, scale fp32 [.., ceil(N / 128), ceil(K / 128)])."""
    w3 = (w if w.dim() == 3 else w[None]).contiguous()
    e, n, k = w3.shape
    codes = torch.zeros(e, n, _up(k, 16), dtype=torch.uint8, device=w.device).view(torch.float8_e4m3fn)[:, :, :k]
    scale = torch.empty(e, _up(n, BLOCK) // BLOCK, _up(k, BLOCK) // BLOCK, dtype=torch.float32, device=w.device)
    torch_ops.op("fp8_quant_weight")(w3, codes, scale)
    return (codes, scale) if w.dim() == 3 else (codes[0], scale[0])


def dequant(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values of quantised rows (scale [M, blocks]) or weights (scale [.., blocks, blocks]); plain torch, for checks."""
    s = scale.repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]
    if scale.shape[-2] != codes.shape[-2]:
        s = s.repeat_interleave(BLOCK, -2)[..., :codes.shape[-2], :]
    return codes.float() * s


def glu_quant(h: torch.Tensor, activation: str = "silu", alpha: float = 1.702, limit: float = 7.0,
              counts: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
              out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gated activation of h = gate | up [R, 2I], quantised: (codes [R, I], scale). activation "silu": silu(g) * u;
    "swiglu_clamp": min(g, limit) * sigmoid(alpha * min(g, limit)) * (clamp(u, -limit, limit) + 1); "gelu_tanh". With
    counts / offsets (ops.Routes) only the experts' live rows are read and written (`out` keeps the others, without it
    they are zero)."""
    i = h.shape[1] // 2
    if out is None:
        out = empty_rows(h.shape[0], i, h.device) if counts is None else _zero_rows(h.shape[0], i, h.device)
    else:
        ops._refuse_grad("glu_quant", *out)
    torch_ops.op("glu_fp8_quant")(h, _ACT[activation], alpha, limit, counts, offsets, out[0], out[1])
    return out


def glu_backward(da: torch.Tensor, h: torch.Tensor, activation: str = "silu", alpha: float = 1.702, limit: float = 7.0,
                 counts: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of h from the gradient da [R, I] of the activation (taken as not quantised)."""
    if out is None:
        out = torch.empty_like(h) if counts is None else torch.zeros_like(h)
    else:
        ops._refuse_grad("glu_backward", out)
    torch_ops.op("glu_backward")(da, h, _ACT[activation], alpha, limit, counts, offsets, out)
    return out


def matmul(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, transpose: bool = False,
           out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [M, K] times w [N, K] transposed -> [M, N]; with transpose=True x [M, N] times w -> [M, K] (the gradient of the
    input through the same stored weight). Every 128-block's product is taken from the tensor core and added in fp32 with
    its two scales. Scales of another layout than quant's are laid out anew on every call."""
    if out is None:
        return torch_ops.op("fp8_matmul_new")(x, x_scale, w, w_scale, transpose, out_dtype)
    ops._refuse_grad("matmul", out)
    torch_ops.op("fp8_matmul")(x, x_scale, w, w_scale, transpose, out)
    return out


def grouped_matmul(rows: torch.Tensor, row_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                   counts: torch.Tensor, offsets: torch.Tensor, transpose: bool = False, rows_in_use: int = 0,
                   out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """matmul, where rows [offsets[e], offsets[e] + counts[e]) meet matrix e of w [E, N, K]. Segments start at multiples
    of 16 (ops.route_pack: of 128). rows_in_use: an upper bound of the sum of counts, it picks the kernel's tile. Pass it
    for small batches: 0 stands for all rows, the padding between segments too, and a decode batch then runs in tiles many
    times its size. `out` keeps the rows outside the segments; without it they are zero."""
    if out is None:
        out = torch.zeros(rows.shape[0], w.shape[-1 if transpose else -2], dtype=out_dtype, device=rows.device)
    else:
        ops._refuse_grad("grouped_matmul", out)
    torch_ops.op("fp8_grouped_matmul")(rows, row_scale, w, w_scale, counts, offsets, transpose, rows_in_use, out)
    return out


def status(device=None) -> int:
    """First error the products have met on the device since the last call (0 = ok). Synchronises the current stream."""
    out = C.c_uint32(0)
    with torch.cuda.device(device):
        rc = _lib.lib().xmoe_fp8_status(C.byref(out), torch.cuda.current_stream().cuda_stream)
    if rc not in (0, 5):
        check(rc, "xmoe_fp8_status")
    return out.value


# ---------------------------------------------------------------------------------------
# an expert layer of them
# ---------------------------------------------------------------------------------------
class _Experts(torch.autograd.Function):
    """rows -> experts' outputs, sorted rows in and out. The gradient goes to x only: the weights are frozen codes. It
    takes the quantisers as the identity (straight through) and quantises the gradients it multiplies the same way."""

    @staticmethod
    def forward(ctx, x, topk_row, layer, r):
        codes, scale = quant(x, topk_row, out=layer._rows(r, layer.shape.hidden))
        h = layer._product(codes, scale, "w13", r, False)
        codes, scale = glu_quant(h, *layer._act, r.counts, r.offsets, out=layer._rows(r, layer.shape.inter))
        rows = layer._product(codes, scale, "w2", r, False)
        ctx.layer, ctx.r = layer, r
        ctx.save_for_backward(topk_row, h)
        return rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        layer, r = ctx.layer, ctx.r
        topk_row, h = ctx.saved_tensors
        codes, scale = quant(drows.contiguous())
        da = layer._product(codes, scale, "w2", r, True)
        dh = glu_backward(da, h, *layer._act, r.counts, r.offsets, out=torch.empty_like(h))
        codes, scale = quant(dh)
        return ops.permute_backward(layer._product(codes, scale, "w13", r, True), topk_row), None, None, None


class Fp8MoE:
    """One MoE layer on block-scaled FP8 experts: routed experts first, shared ones behind, w13 codes [E_tot, 2I, H] (gate
    rows, then up rows) and w2 codes [E_tot, H, I] with their 128 x 128 scales. `forward(x, router_logits)` as FusedMoE's:
    router -> permutation -> quantise into sorted rows -> product -> gated activation + quantise -> product -> weighted sum
    back. Routing weights are applied at the sum.

    `forward_routed` takes the routing, and is differentiable in x and topk_w over the frozen experts."""

    def __init__(self, shape, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
                 router_bias: torch.Tensor | None = None):
        e, h, i = shape.e_tot, shape.hidden, shape.inter
        if tuple(w13.shape) != (e, 2 * i, h) or tuple(w2.shape) != (e, h, i):
            raise RuntimeError("w13 must be [E_tot, 2I, H] and w2 [E_tot, H, I]")
        if shape.act_topk_keep:
            raise RuntimeError("the FP8 layer has no activation top-k")
        if router_bias is not None and router_bias.shape != (shape.num_experts,):
            raise RuntimeError("router_bias must be [num_experts]")
        self.shape = shape
        self.w13, self.w13_scale, self.w2, self.w2_scale = w13, w13_scale, w2, w2_scale
        self.router_bias = None if router_bias is None else router_bias.to(w13.device).float().contiguous()
        self.lut = ops.sigmoid_lut(w13.device) if self.router_bias is not None or shape.n_group > 1 else None
        self.expert_scale = None
        self._act = (shape.activation, shape.swiglu_alpha, shape.swiglu_limit)

    @classmethod
    def from_weights(cls, shape, w13: torch.Tensor, w2: torch.Tensor, router_bias=None) -> "Fp8MoE":
        """From bf16 / fp16 / fp32 weights, quantised here."""
        return cls(shape, *quant_weight(w13), *quant_weight(w2), router_bias)

    def _rows(self, r, cols):
        # rows that no slot names are read into tiles but never stored: they need no values
        return empty_rows(r.num_rows, cols, self.w13.device)

    def _product(self, codes, scale, name, r, transpose):
        w = getattr(self, name)
        out = torch.empty(r.num_rows, w.shape[2 if transpose else 1], dtype=torch.bfloat16, device=w.device)
        return grouped_matmul(codes, scale, w, getattr(self, name + "_scale"), r.counts, r.offsets, transpose,
                              r.rows_in_use, out=out)

    def _check_x(self, x):
        if x.dim() != 2 or x.shape[1] != self.shape.hidden or x.dtype != torch.bfloat16 or not x.is_contiguous():
            raise RuntimeError("x must be a contiguous bf16 tensor [N, hidden]")
        if not x.is_cuda or x.device != self.w13.device:
            raise RuntimeError("x must be a CUDA tensor on the device of the weights")

    def _check_logits(self, x, router_logits):
        if (router_logits.shape != (x.shape[0], self.shape.num_experts) or router_logits.dtype != torch.bfloat16
                or router_logits.device != x.device):
            raise RuntimeError("router_logits must be a bf16 tensor [N, num_experts] on x's device")

    def forward(self, x: torch.Tensor, router_logits: torch.Tensor) -> torch.Tensor:
        self._check_x(x)
        self._check_logits(x, router_logits)
        if x.shape[0] == 0:  # nothing to route
            idx, w = (torch.empty(0, self.shape.top_k, dtype=t, device=x.device) for t in (torch.int32, torch.bfloat16))
            return self.forward_routed(x, idx, w)
        with torch.cuda.device(x.device):
            idx, w = ops.router_topk(router_logits.contiguous(), self.shape, self)
        return self.forward_routed(x, idx, w)

    def forward_routed(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor) -> torch.Tensor:
        """x bf16 [N, H]; topk_idx int32 [N, top_k] (-1: no expert, as is any other id outside the routed experts), topk_w
        bf16 or fp32 [N, top_k]."""
        self._check_x(x)
        if topk_idx.shape != (x.shape[0], self.shape.top_k):
            raise RuntimeError("topk_idx must be [N, top_k]")
        shared = self.shape.num_shared_experts
        r = ops.route_pack(topk_idx, topk_w.detach().to(torch.bfloat16), self.shape.num_experts, shared)
        w = topk_w
        if shared:
            w = torch.cat([topk_w, topk_w.new_ones(x.shape[0], shared)], dim=1)
        rows = _Experts.apply(x, r.topk_row, self, r)
        return ops.unpermute(rows, r.topk_row, w)
