"""Integer linear layers for Hugging Face Qwen3 models, mined with cuPOW on MI355X: the public
surface of the reference's miner/ampere/uwc_ampere/model.py (hadamard, rotate, quant_rows,
MinedLinear, convert_qwen3) over this package's HIP kernels.

The integer math of a layer (model.py:1-17): weights quantized once per output row and activations
per token, both symmetric to [-64, 64] after an optional block-diagonal orthonormal Walsh-Hadamard
rotation of the k axis; the output is bf16((f32(q_x q_W^T) * s_x) * s_w) (+ bias), computed with
the exact int8 GEMM, so every mode below except "bf16" produces the same bits.

  "bf16"   the original weights in bf16 (baseline);
  "int"    the integer math through the plain exact GEMM, any number of rows;
  "plain"  the integer math through the mining GEMM kernel with no transcript (a provider that
           does not mine), for mineable shapes;
  "mined"  MinedWeight.forward: commitment, noise, hashed GEMM and exact denoise, for mineable
           shapes.
A shape that cannot be mined runs the "int" math in every integer mode.

For serving without the integer math's exactness, convert_4bit puts linears with 4-bit weights (uwc_amd.w4) in their place,
a feed-forward block's gate, up, activation and product in one kernel.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops, w4

QMAX = 64
MODES = ("bf16", "int", "plain", "mined")


def hadamard(n: int, device, dtype=torch.float32) -> torch.Tensor:
    """The orthonormal Sylvester-Hadamard matrix of order n (a power of two): entry (i, j) is
    (-1)^popcount(i & j) / sqrt(n) (model.py:30-35)."""
    if n < 1 or n & (n - 1):
        raise AssertionError(f"hadamard: n={n} is not a power of two")
    idx = torch.arange(n)
    both = idx[:, None] & idx[None, :]
    parity = torch.zeros_like(both)
    while bool(both.any()):
        parity ^= both & 1
        both = both >> 1
    return ((1 - 2 * parity).to(torch.float32) / math.sqrt(n)).to(device=device, dtype=dtype)


def rotate(x: torch.Tensor, H: torch.Tensor | None) -> torch.Tensor:
    """x with every block of H.shape[0] consecutive entries of its last axis multiplied by H
    (model.py:38-43); the identity without H."""
    if H is None:
        return x
    blocks = x.to(H.dtype).unflatten(-1, (-1, H.shape[0]))
    return torch.matmul(blocks, H).flatten(-2)


def quant_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric per-row quantization (model.py:46-51): s = max(max|x_row|, 1e-8) / 64,
    q = round-half-even(x / s) clamped to [-64, 64]; returns (int8 q, fp32 s per row)."""
    xf = x.to(torch.float32)
    scale = torch.clamp(xf.abs().amax(-1), min=1e-8) / QMAX
    q = torch.clamp(torch.round(xf / scale.unsqueeze(-1)), -QMAX, QMAX)
    return q.to(torch.int8), scale


def mineable_shape(n: int, k: int, r: int, tile_n: int) -> bool:
    """Shapes the mining path takes (model.py:93-97): k at least max(1024, 16 r) and at most 4 r^2
    (Pearl's rank rule), k a multiple of r and of the 64-wide k step, n a multiple of the GEMM
    tile's N."""
    return max(1024, 16 * r) <= k <= 4 * r * r and k % r == 0 and k % 64 == 0 and n % tile_n == 0


class MinedLinear(nn.Module):
    """One nn.Linear, or several that read the same input concatenated along n, as an integer
    linear that can mine (model.py:54-141). `splits` are the fused layers' output widths."""

    def __init__(self, linears: list[nn.Linear], device, mode: str = "mined", hadamard_block: int = 512,
                 r: int = 128, cfg: str | None = None):
        super().__init__()
        if mode not in MODES:
            raise ValueError(f"MinedLinear: unknown mode {mode!r} (one of {MODES})")
        self.mode, self.r = mode, r
        self.cfg = cfg or ops.DEFAULT_CFG
        self.splits = [lin.out_features for lin in linears]
        self.k = linears[0].in_features
        self.n = sum(self.splits)
        self.bias = self._fused_bias(linears, device)
        self.H = hadamard(min(hadamard_block, self.k & -self.k), device) if hadamard_block else None
        self.mw: ops.MinedWeight | None = None
        self.hashed_macs = 0  # padded rows * n * k over mined calls
        self.useful_macs = 0  # rows * n * k over all calls
        if mode == "bf16":
            self.W = torch.cat([lin.weight.detach().to(device, torch.bfloat16) for lin in linears])
        else:
            self.Wq, self.sw = self._quantize_weights(linears, device)
        self._run = {"bf16": self._run_bf16, "int": self._run_int, "plain": self._run_plain,
                     "mined": self._run_mined}[mode]

    @staticmethod
    def _fused_bias(linears, device):
        if all(lin.bias is None for lin in linears):
            return None
        parts = [lin.bias.detach() if lin.bias is not None else lin.weight.new_zeros(lin.out_features)
                 for lin in linears]
        return torch.cat([p.to(device) for p in parts]).to(torch.bfloat16)

    def _quantize_weights(self, linears, device, rows_per_pass: int = 8192):
        """Rotate and quantize the weight rows on the GPU a slab at a time (an lm_head never needs
        a full fp32 copy on the device)."""
        qs, ss = [], []
        for lin in linears:
            W = lin.weight.detach()
            for r0 in range(0, W.shape[0], rows_per_pass):
                slab = W[r0:r0 + rows_per_pass].to(device=device, dtype=torch.float32)
                q, s = quant_rows(rotate(slab, self.H))
                qs.append(q)
                ss.append(s)
        return torch.cat(qs).contiguous(), torch.cat(ss).contiguous()

    @property
    def mineable(self) -> bool:
        return mineable_shape(self.n, self.k, self.r, ops.BN)

    def setup_block(self, job_key_for_k, bound_for_k):
        """Prepare the mined mode for a block template: job_key_for_k(k) -> 32-byte job key,
        bound_for_k(k) -> 8 little-endian target words. No-op for other modes and unmineable
        shapes."""
        if self.mode != "mined" or not self.mineable:
            return
        if self.mw is None:
            self.mw = ops.MinedWeight(Bt=self.Wq, b_scale=self.sw, r=self.r)
        self.mw.setup_block(job_key_for_k(self.k), bound_for_k(self.k))

    # ---- the integer paths: bf16 rows in, bf16 rows out
    def _quantize_acts(self, rows: torch.Tensor, pad_to: int = 1):
        """Rotation and quantization fused in one kernel; rows padded with zeros to a multiple of
        pad_to (zero rows quantize to zero and are cut from the output)."""
        extra = -rows.shape[0] % pad_to
        xb = rows.to(torch.bfloat16)
        if extra:
            xb = F.pad(xb, (0, 0, 0, extra))
        return ops.quant_rows_had(xb.contiguous(), self.H.shape[0] if self.H is not None else 0)

    def _exact_bf16(self, xq: torch.Tensor, sx: torch.Tensor) -> torch.Tensor:
        y = torch.empty((xq.shape[0], self.n), dtype=torch.bfloat16, device=xq.device)
        ops.gemm(xq, self.Wq, a_scale=sx, b_scale=self.sw, out=y, out_mode=ops.OUT_BF16)
        return y

    def _run_bf16(self, rows: torch.Tensor) -> torch.Tensor:
        return F.linear(rows.to(torch.bfloat16), self.W)

    def _run_int(self, rows: torch.Tensor) -> torch.Tensor:
        xq, sx = self._quantize_acts(rows)
        return self._exact_bf16(xq, sx)

    def _run_plain(self, rows: torch.Tensor) -> torch.Tensor:
        if not self.mineable:
            return self._run_int(rows)
        xq, sx = self._quantize_acts(rows, ops.BM)
        y = torch.empty((xq.shape[0], self.n), dtype=torch.bfloat16, device=xq.device)
        ops.gemm(xq, self.Wq, a_scale=sx, b_scale=self.sw, out=y, out_mode=ops.OUT_BF16, cfg=self.cfg)
        return y[:rows.shape[0]]

    def _run_mined(self, rows: torch.Tensor) -> torch.Tensor:
        if not self.mineable:
            return self._run_int(rows)
        if self.mw is None:
            raise RuntimeError("MinedLinear: setup_block() must run before a mined forward")
        xq, sx = self._quantize_acts(rows, ops.BM)
        self.hashed_macs += xq.shape[0] * self.n * self.k
        return self.mw.forward(xq, sx.contiguous(), out_mode=ops.OUT_BF16)[:rows.shape[0]]

    @torch.compiler.disable
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        rows = x.reshape(-1, self.k)
        y = self._run(rows)
        self.useful_macs += rows.shape[0] * self.n * self.k
        if self.bias is not None:
            y = y + self.bias
        return y.reshape(*x.shape[:-1], self.n)


class _SharedOutput:
    """The fused output of one MinedLinear for the input it was last called with, handed out a
    slice at a time to the modules that stand in for the original linears. A slice is served
    from the cache while the input is the same tensor object at the same version (the cache
    holds the input itself, so a later tensor that reuses its address never matches); once
    every part has taken its slice the cache and the input are dropped, so no activation
    outlives its layer. Inference tensors (torch.inference_mode) have no version: nothing is kept of them,
    each part is computed when it is asked for, alone where the linear can."""

    def __init__(self, ml: MinedLinear):
        self.ml = ml
        self._x = None
        self._version = None
        self._parts = None
        self._pending = 0

    def part(self, x: torch.Tensor, index: int) -> torch.Tensor:
        if x.is_inference():
            if hasattr(self.ml, "part"):
                return self.ml.part(x, index)
            return torch.split(self.ml(x), self.ml.splits, dim=-1)[index]
        if self._parts is None or self._x is not x or self._version != x._version:
            self._parts = torch.split(self.ml(x), self.ml.splits, dim=-1)
            self._x, self._version, self._pending = x, x._version, len(self._parts)
        y = self._parts[index]
        self._pending -= 1
        if self._pending == 0:
            self._parts = self._x = self._version = None
        return y


class _Part(nn.Module):
    """Stands in for one of the linears fused into a MinedLinear (q/k/v, gate/up)."""

    def __init__(self, shared: _SharedOutput, index: int):
        super().__init__()
        self.shared, self.index = shared, index
        if index == 0:  # the group's parameters live in the module tree once, under its first part
            self.ml = shared.ml

    @torch.compiler.disable
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.shared.part(x, self.index)


def _fuse(parent: nn.Module, names: list[str], device, mode, hadamard_block, cfg) -> MinedLinear:
    """Replace parent.<name> for every name by one MinedLinear over all of them."""
    ml = MinedLinear([getattr(parent, nm) for nm in names], device, mode, hadamard_block, cfg=cfg)
    if len(names) == 1:
        setattr(parent, names[0], ml)
    else:
        shared = _SharedOutput(ml)
        for i, nm in enumerate(names):
            setattr(parent, nm, _Part(shared, i))
    return ml


def convert_qwen3(model, device, mode="mined", hadamard_block=512, mine_lm_head=True, cfg=None) -> list[MinedLinear]:
    """Replace every linear of a Hugging Face Qwen3 model (a CausalLM or a bare Qwen3Model) by a
    MinedLinear, q/k/v and gate/up fused; returns them per layer (qkv, o, gate_up, down), then
    the lm_head (model.py:175-197)."""
    decoder = getattr(model, "model", model)
    out = []
    for layer in decoder.layers:
        att, mlp = layer.self_attn, layer.mlp
        for parent, group in ((att, ["q_proj", "k_proj", "v_proj"]), (att, ["o_proj"]),
                              (mlp, ["gate_proj", "up_proj"]), (mlp, ["down_proj"])):
            out.append(_fuse(parent, group, device, mode, hadamard_block, cfg))
    if mine_lm_head and hasattr(model, "lm_head"):
        out.append(_fuse(model, ["lm_head"], device, mode, hadamard_block, cfg))
    return out


class FourBitLinear(nn.Module):
    """One nn.Linear, or several that read the same input concatenated along n, with weights of 4 bits (uwc_amd.w4).
    `splits` are the fused layers' output widths. Rows keep their type, bfloat16 or float16."""

    def __init__(self, linears: list[nn.Linear], device):
        super().__init__()
        self.splits = [lin.out_features for lin in linears]
        self.k, self.n = linears[0].in_features, sum(self.splits)
        parts = [w4.quantize(lin.weight.detach().to(device)) for lin in linears]
        self.register_buffer("codes", torch.cat([c for c, _ in parts]))
        self.register_buffer("scales", torch.cat([s for _, s in parts]))
        bias = None
        if any(lin.bias is not None for lin in linears):
            bias = torch.cat([(lin.bias.detach() if lin.bias is not None else lin.weight.new_zeros(lin.out_features)).to(device) for lin in linears])
        self.register_buffer("bias", bias)

    @torch.compiler.disable
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return w4.linear(x, self.codes, self.scales, self.bias)

    def part(self, x: torch.Tensor, index: int) -> torch.Tensor:
        """What the fused layer number `index` gives."""
        at = sum(self.splits[:index])
        rows = slice(at, at + self.splits[index])
        return w4.linear(x, self.codes[rows], self.scales[rows], None if self.bias is None else self.bias[rows])


class FourBitMLP(nn.Module):
    """down(silu(gate(x)) * up(x)) with weights of 4 bits: two kernels."""

    def __init__(self, mlp: nn.Module, device):
        super().__init__()
        self.check(mlp)
        self.gate_up, self.down = FourBitLinear([mlp.gate_proj, mlp.up_proj], device), FourBitLinear([mlp.down_proj], device)

    @staticmethod
    def check(mlp: nn.Module):
        if mlp.gate_proj.bias is not None or mlp.up_proj.bias is not None:
            raise AssertionError("FourBitMLP: gate and up projections must have no bias")
        z = torch.linspace(-4, 4, 33)
        if not torch.allclose(mlp.act_fn(z), F.silu(z), rtol=1e-5, atol=1e-6):
            raise AssertionError("FourBitMLP: the activation must be silu")

    @torch.compiler.disable
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down(w4.gated(x, self.gate_up.codes, self.gate_up.scales))


def _check_4bit(name: str, lin: nn.Linear):
    w = lin.weight.detach()
    if w.dtype not in (torch.bfloat16, torch.float16):
        raise AssertionError(f"convert_4bit: {name} must be bfloat16 or float16, got {w.dtype}")
    if w.dim() != 2 or w.shape[1] == 0 or w.shape[1] % w4.GROUP:
        raise AssertionError(f"convert_4bit: {name} must have a positive multiple of {w4.GROUP} inputs, got weights {tuple(w.shape)}")
    if w.numel() and not torch.isfinite(torch.stack(torch.aminmax(w))).all():
        raise AssertionError(f"convert_4bit: {name} must have finite weights")


def convert_4bit(model, device, lm_head: bool = False) -> list[nn.Module]:
    """Replace the linears of a Hugging Face Qwen3 or Llama model (a CausalLM or the bare model), in bfloat16 or float16, by
    FourBitLinears, q/k/v fused and each feed-forward block a FourBitMLP; returns them per layer (qkv, o, feed-forward), then
    the lm_head where it is asked for. The weights are rounded to 4 bits as they are, without calibration. A model that cannot
    be converted is refused before anything in it is replaced."""
    decoder = getattr(model, "model", model)
    for i, layer in enumerate(decoder.layers):
        FourBitMLP.check(layer.mlp)
        for name in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj"):
            _check_4bit(f"layers.{i}.{name}", layer.get_submodule(name))
    if lm_head and hasattr(model, "lm_head"):
        _check_4bit("lm_head", model.lm_head)
    out = []
    for layer in decoder.layers:
        att = layer.self_attn
        qkv = FourBitLinear([att.q_proj, att.k_proj, att.v_proj], device)
        shared = _SharedOutput(qkv)
        for i, name in enumerate(("q_proj", "k_proj", "v_proj")):
            setattr(att, name, _Part(shared, i))
        att.o_proj = FourBitLinear([att.o_proj], device)
        layer.mlp = FourBitMLP(layer.mlp, device)
        out += [qkv, att.o_proj, layer.mlp]
    if lm_head and hasattr(model, "lm_head"):
        model.lm_head = FourBitLinear([model.lm_head], device)
        out.append(model.lm_head)
    return out
