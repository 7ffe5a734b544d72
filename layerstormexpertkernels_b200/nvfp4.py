"""NVFP4 experts: the weight layout, quantising bf16 weights, and the whole
routed layer on 4-bit experts (lsek_moe_layer_forward_nvfp4).

An NVFP4 tensor is codes (uint8, two E2M1 codes a byte, the even element in
the low nibble), scales (float8_e4m3fn, one for 16 elements of a row) and one
float32 global scale (per expert for weights).  The GEMMs take the scales of
weights in the tiles of `nvfp4_tile_scales`; those of activations stay rows.
The code / scale pair is the reference's (ref_nvfp4_dequant,
tests/test_reference.py:19-53); it documents the expert GEMMs on it
(USAGE.md:25-32) but ships them in a separate library.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _C
from .layer import LayerWorkspace, StageEvents

E2M1_MAX = 6.0
E4M3_MAX = 448.0
MIN_GLOBAL_SCALE = 2.0 ** -100


def nvfp4_tile_scales(scales: torch.Tensor, parts: int = 1) -> torch.Tensor:
    """Weight scales [E, N, K/16] (float8_e4m3fn) -> the tiles that the NVFP4
    GEMMs read, [E, parts * ceil(N / parts / 128), K/64, 512]: in a tile of
    128 rows and four scales, row r lies at byte 16 * (r % 32) + 4 * (r // 32).
    `parts` = 2 for gate/up weights (gate rows and up rows are tiled apart),
    1 otherwise.  Rows past the last are zero.  Done once, when weights are
    loaded; K must be a multiple of 64."""
    if scales.dtype != torch.float8_e4m3fn:
        raise ValueError(f"nvfp4_tile_scales: scales must be float8_e4m3fn, got {scales.dtype}")
    if scales.dim() != 3:
        raise ValueError("nvfp4_tile_scales: scales must be [E, N, K/16]")
    e, n, s = scales.shape
    if parts < 1 or n % parts != 0:
        raise ValueError(f"nvfp4_tile_scales: {n} rows cannot be split in {parts} equal parts")
    if s % 4 != 0:
        raise ValueError(f"nvfp4_tile_scales: K must be a multiple of 64, got {16 * s}")
    rows = n // parts
    tall = -(-rows // 128)
    full = scales.new_zeros((e, parts, tall * 128, s), dtype=torch.uint8)
    full[:, :, :rows] = scales.view(torch.uint8).reshape(e, parts, rows, s)
    full = full.view(e, parts, tall, 4, 32, s // 4, 4).permute(0, 1, 2, 5, 4, 3, 6)
    return full.reshape(e, parts * tall, s // 4, 512).view(torch.float8_e4m3fn)


def weight_global_scales(w: torch.Tensor) -> torch.Tensor:
    """[E] float32 of weights [E, N, K]: see nvfp4_quantize_weights."""
    if not w.numel():
        return w.new_ones(w.shape[0], dtype=torch.float32)
    amax = torch.stack([x.abs().nan_to_num_(0.0, posinf=0.0).amax() for x in w]).float()
    return torch.where(amax > 0, (amax / (E2M1_MAX * E4M3_MAX)).clamp_(min=MIN_GLOBAL_SCALE), 1.0)


def nvfp4_quantize_weights(w: torch.Tensor, parts: int = 1):
    """Expert weights [E, N, K] bf16 or fp16 -> (codes [E, N, K/2], tiled
    scales, global scales [E] float32).  An expert's global scale is its
    largest finite magnitude / (6 * 448), which puts its largest block scale at
    the top of E4M3 (1 for an expert of zeros, and never below 2^-100, the
    least that the quantiser takes).  A block that holds an infinity or a NaN
    gets the scale NaN; the expert's other blocks are as without it."""
    if w.dim() != 3:
        raise ValueError("nvfp4_quantize_weights: weights must be [E, N, K]")
    glob = weight_global_scales(w)
    codes, scales = _C.nvfp4_quantize(w, glob)
    return codes, nvfp4_tile_scales(scales, parts), glob


def moe_layer_forward_nvfp4(hidden: torch.Tensor, logits: torch.Tensor,
                            bias: Optional[torch.Tensor], w_gu: torch.Tensor,
                            w_gu_scales: torch.Tensor,
                            w_gu_global_scale: Optional[torch.Tensor], w_down: torch.Tensor,
                            w_down_scales: torch.Tensor,
                            w_down_global_scale: Optional[torch.Tensor], topk: int, n_group: int,
                            topk_group: int, routed_scaling_factor: float, renormalize: bool,
                            scoring_func: str = "sigmoid", swiglu_limit: float = 0.0,
                            hidden_global_scale: Optional[torch.Tensor] = None,
                            inter_global_scale: Optional[torch.Tensor] = None,
                            return_routing: bool = False):
    """One MoE layer forward on NVFP4 experts (moe_layer_forward's flow).

    hidden [T, H] bf16, logits [T, E] f32, bias [E] f32 or None; w_gu
    [E, 2I, H/2] and w_down [E, H, I/2] uint8 codes with tiled scales
    (nvfp4_tile_scales, parts=2 and 1) and global scales [E].  The tokens are
    quantised with hidden_global_scale, the activated intermediate with
    inter_global_scale (one float32 each, None for 1).  Returns out [T, H]
    bf16, and (topk_weights, topk_indices) when return_routing is set.
    """
    T, H = hidden.shape
    E = logits.shape[1]
    inter = 2 * w_down.shape[2]
    ws = torch.empty(_C.moe_layer_nvfp4_workspace_size(T, H, inter, E, topk), dtype=torch.uint8,
                     device=hidden.device)
    out = torch.empty_like(hidden)
    w = idx = None
    if return_routing:
        w = torch.empty(T, topk, dtype=torch.float32, device=hidden.device)
        idx = torch.empty(T, topk, dtype=torch.int32, device=hidden.device)
    _C.moe_layer_forward_nvfp4_out(out, hidden, logits, bias, w_gu, w_gu_scales, w_gu_global_scale,
                                   w_down, w_down_scales, w_down_global_scale, hidden_global_scale,
                                   inter_global_scale, topk, n_group, topk_group,
                                   routed_scaling_factor, renormalize, scoring_func, swiglu_limit,
                                   ws, w, idx)
    if return_routing:
        return out, w, idx
    return out


class MoELayerNVFP4(LayerWorkspace):
    """A routed-expert layer with resident NVFP4 weights and a reusable
    workspace: MoELayer's interface on 4-bit experts.

    Takes weights in the form of moe_layer_forward_nvfp4, or bf16 weights
    through `from_weights`.  As with MoELayer the workspace grows to the
    largest token count seen, and calls on different streams need a layer
    each (they would share the workspace).
    """

    def __init__(self, w_gu: torch.Tensor, w_gu_scales: torch.Tensor,
                 w_gu_global_scale: Optional[torch.Tensor], w_down: torch.Tensor,
                 w_down_scales: torch.Tensor, w_down_global_scale: Optional[torch.Tensor],
                 bias: Optional[torch.Tensor] = None, *, topk: int = 8, n_group: int = 8,
                 topk_group: int = 4, routed_scaling_factor: float = 2.5,
                 renormalize: bool = True, scoring_func: str = "sigmoid",
                 swiglu_limit: float = 0.0, hidden_global_scale: Optional[torch.Tensor] = None,
                 inter_global_scale: Optional[torch.Tensor] = None, max_tokens: int = 0):
        if w_gu.dim() != 3 or w_down.dim() != 3:
            raise ValueError("w_gu must be [E, 2I, H/2] and w_down [E, H, I/2]")
        self.w_gu, self.w_gu_scales, self.w_gu_global_scale = w_gu, w_gu_scales, w_gu_global_scale
        self.w_down, self.w_down_scales = w_down, w_down_scales
        self.w_down_global_scale = w_down_global_scale
        self.bias = bias
        self.num_experts = w_gu.shape[0]
        self.hidden_dim = 2 * w_gu.shape[2]
        self.inter_dim = 2 * w_down.shape[2]
        self.topk, self.n_group, self.topk_group = topk, n_group, topk_group
        self.routed_scaling_factor = routed_scaling_factor
        self.renormalize = renormalize
        self.scoring_func = scoring_func
        self.swiglu_limit = swiglu_limit
        self.hidden_global_scale = hidden_global_scale
        self.inter_global_scale = inter_global_scale
        self._init_workspace(w_gu.device, max_tokens)

    @classmethod
    def from_weights(cls, w_gu: torch.Tensor, w_down: torch.Tensor,
                     bias: Optional[torch.Tensor] = None, **kwargs) -> "MoELayerNVFP4":
        """Quantises w_gu [E, 2I, H] and w_down [E, H, I] (bf16 or fp16); the
        keyword arguments are the constructor's."""
        return cls(*nvfp4_quantize_weights(w_gu, 2), *nvfp4_quantize_weights(w_down, 1), bias,
                   **kwargs)

    def workspace_bytes(self, num_tokens: int) -> int:
        return _C.moe_layer_nvfp4_workspace_size(num_tokens, self.hidden_dim, self.inter_dim,
                                                 self.num_experts, self.topk)

    def forward(self, hidden: torch.Tensor, logits: torch.Tensor,
                out: Optional[torch.Tensor] = None,
                topk_weights: Optional[torch.Tensor] = None,
                topk_indices: Optional[torch.Tensor] = None,
                stage_events: Optional[StageEvents] = None) -> torch.Tensor:
        """As MoELayer.forward; the row copy stage quantises the tokens."""
        self._ensure_workspace(hidden.shape[0])
        if out is None:
            out = torch.empty_like(hidden)
        handles = [] if stage_events is None else stage_events.handles
        _C.moe_layer_forward_nvfp4_out(
            out, hidden, logits, self.bias, self.w_gu, self.w_gu_scales, self.w_gu_global_scale,
            self.w_down, self.w_down_scales, self.w_down_global_scale, self.hidden_global_scale,
            self.inter_global_scale, self.topk, self.n_group, self.topk_group,
            self.routed_scaling_factor, self.renormalize, self.scoring_func, self.swiglu_limit,
            self.workspace, topk_weights, topk_indices, handles)
        return out

    __call__ = forward
