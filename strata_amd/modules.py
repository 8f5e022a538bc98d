"""Drop-in modules for the Strata transformer block, backed by ``torch.ops.strata_hip``.

State-dict keys and parameter registration order match the reference's
manifests (tests/regression_data/sweep1_...param_order.txt:3-12, pinned by
tests/test_param_order.py:87-119): per block ``attn.qkv.{weight,bias}``,
``attn.proj.{weight,bias}``, optional ``attn.gate_proj.{weight,bias}``,
``mlp.layers.0.{weight,bias}``, ``mlp.layers.2.{weight,bias}``; the two
LayerNorms are non-affine and carry no parameters.

The modules run bf16 weights and activations on one GPU (fp32 accumulation
inside the kernels).  They never fall back to eager PyTorch math: CPU tensors
or a missing HIP library raise.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib, ops  # noqa: F401  (ops registers torch.ops.strata_hip)

_ACT = {"tanh": _lib.ACT_GELU_TANH, "none": _lib.ACT_GELU_ERF}


def _triple(v) -> list[int]:
    return [v, v, v] if isinstance(v, int) else [int(x) for x in v]


class GemmGeluMlp(nn.Module):
    """``layers = Sequential(fc1, GELU, fc2)`` computed as two fused GEMM launches.

    Drop-in for physicsnemo's ``Mlp`` (layer indices 0/2 per
    screamcast/checkpoint_compat.py:243-249; GELU(tanh) per
    screamcast/strata_wrappers.py:76-100): fc1 + bias + GELU is one launch,
    fc2 + bias (+ the block's residual) another.  Under autograd (tanh GELU)
    fc1's launch also writes gelu'(pre-activation), which the backward multiplies
    by the upstream gradient in the epilogue of its product with fc2's weight.
    """

    def __init__(self, in_features: int, hidden_features: int, out_features: Optional[int] = None,
                 bias: bool = True, approximate: str = "tanh"):
        super().__init__()
        out_features = out_features or in_features
        self.layers = nn.Sequential(
            nn.Linear(in_features, hidden_features, bias=bias),
            nn.GELU(approximate=approximate),
            nn.Linear(hidden_features, out_features, bias=bias),
        )

    @classmethod
    def from_mlp(cls, mlp: nn.Module) -> "GemmGeluMlp":
        """Wrap an existing ``Mlp``-shaped module, sharing its Linear layers."""
        fc1, act, fc2 = mlp.layers
        if not (isinstance(fc1, nn.Linear) and isinstance(act, nn.GELU) and isinstance(fc2, nn.Linear)):
            raise TypeError("expected layers = Sequential(Linear, GELU, Linear)")
        new = cls.__new__(cls)
        nn.Module.__init__(new)
        new.layers = mlp.layers
        return new

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        fc1, act, fc2 = self.layers
        train = torch.is_grad_enabled() and (x.requires_grad or fc1.weight.requires_grad)
        if train and act.approximate == "tanh" and not (fc1.in_features % 8 or fc1.out_features % 8
                                                        or fc2.out_features % 8):
            return ops.mlp_gelu_train(x, fc1.weight, fc1.bias, fc2.weight, fc2.bias, residual)[0]
        if train and act.approximate == "tanh":
            # fc1's launch also writes gelu'(pre-activation) for the backward (no recomputed GEMM)
            h, _ = ops.gemm_gelu_train(x, fc1.weight, fc1.bias)
        else:
            h = ops.gemm_bias_act(x, fc1.weight, fc1.bias, None, _ACT[act.approximate])
        return ops.gemm_bias_act(h, fc2.weight, fc2.bias, residual, _lib.ACT_NONE)


class ExpertMlp(nn.Module):
    """A sparse ``GemmGeluMlp``: every token takes ``top_k`` of ``experts`` MLPs.

    ``router`` (Linear without a bias) gives a token's logits, ``ops.expert_route`` its experts and
    their weights, ``ops.expert_mlp`` their weighted sum and the block's residual: the experts'
    weights are stacked, ``w1 [E, H, C]``, ``b1 [E, H]``, ``w2 [E, N, H]``, ``b2 [E, N]``.  ``score``,
    ``groups``, ``top_groups``, ``renormalize`` and ``scale`` are ``expert_route``'s.  With ``balance``
    a buffer of that name (fp32 ``[E]``, zeros) is added to the scores for the choice alone; the
    training loop moves it against the experts' load (``route`` returns the choice, ``bincount`` of
    its index the load) and it stays fp32 when the module is cast.  bf16 on one GPU, as the MLP it
    stands for; differentiable in x, the residual and every parameter."""

    def __init__(self, in_features: int, hidden_features: int, experts: int, top_k: int = 2,
                 out_features: Optional[int] = None, bias: bool = True, score: str = "softmax", groups: int = 1,
                 top_groups: int = 1, renormalize: bool = True, scale: float = 1.0, balance: bool = False):
        super().__init__()
        out_features = out_features or in_features
        if score not in ops.SCORES:
            raise ValueError(f"score must be one of {sorted(ops.SCORES)}, got {score!r}")
        if experts % groups or not 1 <= top_groups <= groups or not 1 <= top_k <= experts // groups * top_groups:
            raise ValueError(f"top_k {top_k} of {experts} experts in {top_groups} of {groups} groups is not a choice")
        self.top_k, self.score, self.groups, self.top_groups = top_k, score, groups, top_groups
        self.renormalize, self.scale = renormalize, scale
        self.router = nn.Linear(in_features, experts, bias=False)
        self.w1 = nn.Parameter(torch.empty(experts, hidden_features, in_features))
        self.b1 = nn.Parameter(torch.empty(experts, hidden_features)) if bias else None
        self.w2 = nn.Parameter(torch.empty(experts, out_features, hidden_features))
        self.b2 = nn.Parameter(torch.empty(experts, out_features)) if bias else None
        self.register_buffer("balance", torch.zeros(experts) if balance else None)
        with torch.no_grad():  # each expert as the Linear layers of the dense MLP start
            for w, b in ((self.w1, self.b1), (self.w2, self.b2)):
                bound = w.shape[2] ** -0.5
                w.uniform_(-bound, bound)
                if b is not None:
                    b.uniform_(-bound, bound)

    def _apply(self, fn, recurse=True):
        balance = self.balance
        super()._apply(fn, recurse)
        if balance is not None and self.balance.dtype != torch.float32:
            self.balance = balance.to(self.balance.device)
        return self

    def route(self, x: Tensor) -> tuple[Tensor, Tensor]:
        """``(weights, index)`` ``[..., top_k]`` of tokens ``[..., C]``."""
        logits = ops.gemm_bias_act(x, self.router.weight, None, None, _lib.ACT_NONE)
        return ops.expert_route(logits, self.top_k, self.score, self.balance, self.groups, self.top_groups,
                                self.renormalize, self.scale)

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        weights, index = self.route(x)
        return ops.expert_mlp(x, weights, index, self.w1, self.b1, self.w2, self.b2, residual)


class FusedNA3DAttention(nn.Module):
    """qkv GEMM -> (qk RMSNorm +) RoPE + QKV pack -> NA3D -> (gate) -> proj GEMM (+ residual).

    Drop-in for the physicsnemo Strata attention's ``qkv -> split -> RoPE ->
    natten.na3d -> proj`` chain (keys attn.qkv / attn.proj / attn.gate_proj;
    gate applied as ``a * sigmoid(gate_proj(x))`` before proj, fused into the
    gate GEMM's epilogue).  ``qk_norm`` (screamcast/config.py:91-93) RMS-
    normalises q and k per head inside the RoPE pack kernel; with
    ``qk_norm_affine`` the weights live in ``attn.q_norm`` / ``attn.k_norm``
    (nn.RMSNorm, registered after the manifest keys).

    ``depthwise``: the block attends along the depth (z) axis only, every token
    to the whole column of tokens at its (y, x): NA3D with the window (Z, 1, 1)
    of the input's Z, the same qkv / proj / gate parameters (the production
    manifest's blocks all carry the same keys).  This is this build's reading of
    ``do_alt_depthwise_attn`` (screamcast/config.py:101-103, passed at
    screamcast/strata_wrappers.py:329; "depth" is the vertical axis of
    ``input_shape=(depth, height, width)``, :317); the arithmetic lives in
    physicsnemo, absent here, so parity of the convention is unpinned.
    """

    def __init__(self, dim: int, num_heads: int, kernel_size, dilation=1, qkv_bias: bool = True,
                 gated: bool = False, rope_layout: int = _lib.ROPE_HALF, scale: Optional[float] = None,
                 qk_norm: bool = False, qk_norm_affine: bool = False, qk_norm_eps: float = 1e-6,
                 depthwise: bool = False):
        super().__init__()
        if dim % num_heads:
            raise ValueError("dim must be divisible by num_heads")
        self.depthwise = depthwise
        self.dim, self.num_heads = dim, num_heads
        self.head_dim = dim // num_heads
        self.kernel_size = _triple(kernel_size)
        self.dilation = _triple(dilation)
        self.rope_layout = rope_layout
        self.scale = scale
        self.qkv = nn.Linear(dim, 3 * dim, bias=qkv_bias)
        self.proj = nn.Linear(dim, dim)
        if gated:
            self.gate_proj = nn.Linear(dim, dim)
        else:
            self.gate_proj = None
        self.qk_norm, self.qk_norm_eps = qk_norm, qk_norm_eps
        if qk_norm and qk_norm_affine:
            self.q_norm = nn.RMSNorm(self.head_dim, eps=qk_norm_eps)
            self.k_norm = nn.RMSNorm(self.head_dim, eps=qk_norm_eps)
        else:
            self.q_norm = self.k_norm = None

    # Children an attention module of the reference may own, besides parameter-free ones.
    _KNOWN_CHILDREN = ("qkv", "proj", "gate_proj", "q_norm", "k_norm")

    @classmethod
    def from_attention(cls, attn: nn.Module, num_heads: int, kernel_size, dilation=1, qk_norm: bool = False,
                       qk_norm_eps: float = 1e-6, rope_layout: int = _lib.ROPE_HALF,
                       scale: Optional[float] = None, depthwise: bool = False) -> "FusedNA3DAttention":
        """Wrap an existing attention module, sharing its Linear (and RMSNorm) children.

        The children are re-registered in the module's own order, so the state-dict
        keys (``qkv``, ``proj``, ``gate_proj``, ``q_norm``, ``k_norm``) and the
        ``named_parameters()`` order are unchanged.  A child that holds parameters
        under any other name raises ``TypeError`` (its role would be unknown)."""
        qkv, proj = getattr(attn, "qkv", None), getattr(attn, "proj", None)
        if not (isinstance(qkv, nn.Linear) and isinstance(proj, nn.Linear)):
            raise TypeError("expected an attention module with nn.Linear children qkv and proj")
        dim = qkv.in_features
        if qkv.out_features != 3 * dim or proj.in_features != dim or dim % num_heads:
            raise TypeError(f"qkv {tuple(qkv.weight.shape)} / proj {tuple(proj.weight.shape)} do not fit "
                            f"a {num_heads}-head attention")
        for name, child in attn.named_children():
            if name not in cls._KNOWN_CHILDREN and any(True for _ in child.parameters()):
                raise TypeError(f"attention child {name!r} holds parameters this drop-in does not use")
        new = cls.__new__(cls)
        nn.Module.__init__(new)
        new.gate_proj = new.q_norm = new.k_norm = None
        for name, child in attn.named_children():
            setattr(new, name, child)
        gate = getattr(attn, "gate_proj", None)
        if gate is not None and not isinstance(gate, nn.Linear):
            raise TypeError("gate_proj must be an nn.Linear")
        for nname in ("q_norm", "k_norm"):
            norm = getattr(attn, nname, None)
            w = getattr(norm, "weight", None) if norm is not None else None
            setattr(new, nname, norm if isinstance(w, torch.Tensor) else None)
        new.dim, new.num_heads = dim, num_heads
        new.head_dim = dim // num_heads
        new.kernel_size = _triple(kernel_size)
        new.dilation = _triple(dilation)
        new.rope_layout = rope_layout
        new.scale = scale
        new.qk_norm, new.qk_norm_eps = qk_norm, qk_norm_eps
        new.depthwise = depthwise
        return new

    def window(self, z: int) -> tuple[list[int], list[int]]:
        """NA3D kernel and dilation for an input of depth ``z``."""
        if self.depthwise:
            return [z, 1, 1], [1, 1, 1]
        return self.kernel_size, self.dilation

    def attention(self, x: Tensor, rope: Optional[tuple[Tensor, Tensor]] = None) -> Tensor:
        """Attention output before the projection, ``[B, Z, Y, X, C]``."""
        B, Z, Y, X, C = x.shape
        H, D = self.num_heads, self.head_dim
        kernel, dilation = self.window(Z)
        qkv = ops.gemm_bias_act(x, self.qkv.weight, self.qkv.bias, None, _lib.ACT_NONE)
        if rope is None and self.qk_norm:  # normalise in the pack kernel with identity rotations
            ident = torch.ones(B, 1, Y, X, D // 2, device=x.device)
            rope = (ident, torch.zeros_like(ident))
        if rope is not None:
            qw = self.q_norm.weight if self.q_norm is not None else None
            kw = self.k_norm.weight if self.k_norm is not None else None
            # Inference: v is read straight out of qkv (a strided view), the pack writes q and
            # k only.  Training: the pack copies v too, so the backward writes d(qkv) in one
            # pass (its v columns from dv) instead of zero-filling it, scattering dv into the
            # view and adding the two.
            train = torch.is_grad_enabled() and qkv.requires_grad
            if not train and not self.qk_norm and self.rope_layout == _lib.ROPE_HALF:
                # Inference: the queries can be rotated inside the small-window NA3D kernel,
                # q read unrotated straight out of qkv, so the pack writes k only.
                qkv6 = qkv.view(B, Z, Y, X, 3, H, D)
                q, v = qkv6[..., 0, :, :], qkv6[..., 2, :, :]
                kst = [Z * Y * X * H * D, Y * X * H * D, X * H * D, H * D, D]
                if ops.na3d_rope_q_supported(q, kst, v, rope[0], rope[1], kernel, dilation, self.scale):
                    _, k, _ = ops.rope_qkv_pack(qkv, rope[0], rope[1], H, self.rope_layout, pack_v=False,
                                                pack_q=False)
                    a = ops.na3d_fwd_rope_q(q, k, v, rope[0], rope[1], kernel, dilation, self.scale)
                    return self._gate(x, a.view(B, Z, Y, X, C))
            q, k, v = ops.rope_qkv_pack(qkv, rope[0], rope[1], H, self.rope_layout, self.qk_norm, self.qk_norm_eps,
                                        qw, kw, pack_v=train)
            if not train:
                v = qkv.view(B, Z, Y, X, 3, H, D)[..., 2, :, :]
        else:
            qkv6 = qkv.view(B, Z, Y, X, 3, H, D)
            q, k, v = qkv6[..., 0, :, :], qkv6[..., 1, :, :], qkv6[..., 2, :, :]
        a = ops.na3d(q, k, v, kernel, dilation, self.scale)
        return self._gate(x, a.view(B, Z, Y, X, C))

    def _gate(self, x: Tensor, a: Tensor) -> Tensor:
        if self.gate_proj is not None:  # a * sigmoid(x @ Wg^T + bg) in one GEMM
            a = ops.gemm_bias_act(x, self.gate_proj.weight, self.gate_proj.bias, a, _lib.ACT_SIGMOID, _lib.RES_MUL)
        return a

    def forward(self, x: Tensor, rope: Optional[tuple[Tensor, Tensor]] = None,
                residual: Optional[Tensor] = None) -> Tensor:
        a = self.attention(x, rope)
        return ops.gemm_bias_act(a, self.proj.weight, self.proj.bias, residual, _lib.ACT_NONE)


class StrataBlock(nn.Module):
    """Pre-norm Strata transformer block (the configs[3] block).

    ``x = x + proj(na3d(rope(qkv(LN(x)))))``; ``x = x + fc2(GELU(fc1(LN(x))))``
    with non-affine LayerNorms (eps 1e-6).  Stand-in for physicsnemo's
    ``StrataTransformer3DBlock`` (tests/test_dit_3d_pixel.py:109-111) with the
    same parameter names and order.  ``experts``: the MLP is an ``ExpertMlp`` of that
    many experts (``expert_options``: its other arguments), which the reference's
    block does not have.
    """

    def __init__(self, dim: int, num_heads: int, kernel_size, mlp_ratio: float = 4.0, dilation=1,
                 qkv_bias: bool = True, gated: bool = False, eps: float = 1e-6, qk_norm: bool = False,
                 qk_norm_affine: bool = False, qk_norm_eps: float = 1e-6, depthwise: bool = False, experts: int = 0,
                 expert_options: Optional[dict] = None):
        super().__init__()
        self.eps = eps
        self.attn = FusedNA3DAttention(dim, num_heads, kernel_size, dilation, qkv_bias, gated,
                                       qk_norm=qk_norm, qk_norm_affine=qk_norm_affine, qk_norm_eps=qk_norm_eps,
                                       depthwise=depthwise)
        hidden = int(dim * mlp_ratio)
        self.mlp = ExpertMlp(dim, hidden, experts, **(expert_options or {})) if experts else GemmGeluMlp(dim, hidden)

    def forward(self, x: Tensor, rope: Optional[tuple[Tensor, Tensor]] = None) -> Tensor:
        h = ops.layer_norm(x, self.eps)
        x = self.attn(h, rope, residual=x)
        h = ops.layer_norm(x, self.eps)
        return self.mlp(h, residual=x)


class StrataPixelBlock(nn.Module):
    """Pixel-stage block conditioned on the semantic stage's tokens by a spatially
    varying adaLN (``use_bilinear_dw_gelu_project_adaln_pixel``,
    screamcast/strata_wrappers.py:443,471-477,490-495; parameters
    tests/regression_data/pixeldit_...param_order.txt:245-256, in that order:
    ``attn.qkv``, ``attn.proj``, ``mlp.layers.0``, ``mlp.layers.2``,
    ``adaln_bilinear_dw_conv``, ``adaln_bilinear_dw_proj``).  The block itself
    (physicsnemo's ``StrataPixel3DBlock``) is absent here; this build's convention,
    parity unpinned beyond its parts, is DiT's adaLN-Zero with per-token modulations:

        mod = adaln_bilinear_dw_proj(GELU_tanh(dwconv3x3(bilinear_up(cond))))
            -> shift1, scale1, gate1, shift2, scale2, gate2      (each ``dim`` wide)
        x = x + gate1 * proj(attn(LN(x) * (1 + scale1) + shift1))
        x = x + gate2 * mlp(LN(x) * (1 + scale2) + shift2)

    ``cond``: the semantic tokens ``[B, Z, Y / factor, X / factor, cond_dim]``
    (``factor`` = the semantic stage's horizontal patch; its vertical patch is 1, as the
    reference requires for this mode, screamcast/strata_wrappers.py:471-477).  The
    upsampling, depth-wise convolution and GELU run in one HIP kernel, the projection
    on the library's GEMM, the modulated LayerNorms and gated residuals in two more.
    Inference only."""

    def __init__(self, dim: int, num_heads: int, kernel_size, cond_dim: int, factor: int, mlp_ratio: float = 4.0,
                 dilation=1, qkv_bias: bool = True, eps: float = 1e-6, qk_norm: bool = False,
                 qk_norm_affine: bool = False, qk_norm_eps: float = 1e-6):
        super().__init__()
        self.eps, self.factor, self.dim = eps, int(factor), dim
        self.attn = FusedNA3DAttention(dim, num_heads, kernel_size, dilation, qkv_bias, False, qk_norm=qk_norm,
                                       qk_norm_affine=qk_norm_affine, qk_norm_eps=qk_norm_eps)
        self.mlp = GemmGeluMlp(dim, int(dim * mlp_ratio))
        self.adaln_bilinear_dw_conv = nn.Conv3d(cond_dim, cond_dim, (1, 3, 3), padding=(0, 1, 1), groups=cond_dim)
        self.adaln_bilinear_dw_proj = nn.Linear(cond_dim, 6 * dim)

    def modulation(self, cond: Tensor) -> Tensor:
        """The six modulations ``[B, Z, Y, X, 6 * dim]`` from the semantic tokens."""
        conv, proj = self.adaln_bilinear_dw_conv, self.adaln_bilinear_dw_proj
        c = ops.upsample_dw_gelu(cond, conv.weight, conv.bias, self.factor)
        return ops.gemm_bias_act(c, proj.weight, proj.bias, None, _lib.ACT_NONE)

    def forward(self, x: Tensor, cond: Tensor, rope: Optional[tuple[Tensor, Tensor]] = None) -> Tensor:
        if cond.shape[0] != x.shape[0] or cond.shape[1] != x.shape[1] or \
                cond.shape[2] * self.factor != x.shape[2] or cond.shape[3] * self.factor != x.shape[3]:
            raise ValueError(f"cond {tuple(cond.shape)} does not match x {tuple(x.shape)} at factor {self.factor}")
        sh1, sc1, g1, sh2, sc2, g2 = self.modulation(cond).split(self.dim, dim=-1)
        h = ops.layer_norm_modulate(x, sh1, sc1, self.eps)
        x = ops.gated_add(x, g1, self.attn(h, rope))
        h = ops.layer_norm_modulate(x, sh2, sc2, self.eps)
        return ops.gated_add(x, g2, self.mlp(h))


def swap_mlps(model: nn.Module) -> int:
    """Replace every ``Mlp``-shaped child (``layers = Sequential(Linear, GELU, Linear)``)
    by a :class:`GemmGeluMlp` sharing its parameters, in the pattern of the
    reference's ``_use_tanh_gelu`` (screamcast/strata_wrappers.py:76-100).
    Keys and parameter order are unchanged.  Returns the number swapped."""
    n = 0
    for parent in list(model.modules()):
        for name, child in list(parent.named_children()):
            if isinstance(child, GemmGeluMlp):
                continue
            layers = getattr(child, "layers", None)
            if (
                isinstance(layers, nn.Sequential)
                and len(layers) == 3
                and isinstance(layers[0], nn.Linear)
                and isinstance(layers[1], nn.GELU)
                and isinstance(layers[2], nn.Linear)
            ):
                setattr(parent, name, GemmGeluMlp.from_mlp(child))
                n += 1
    return n


def _is_attention(m: nn.Module) -> bool:
    qkv, proj = getattr(m, "qkv", None), getattr(m, "proj", None)
    return (isinstance(qkv, nn.Linear) and isinstance(proj, nn.Linear) and qkv.out_features == 3 * qkv.in_features
            and proj.in_features == qkv.in_features)


def swap_attention(model: nn.Module, num_heads, kernel_size, dilation=1, qk_norm=False, qk_norm_eps: float = 1e-6,
                   rope_layout: int = _lib.ROPE_HALF, scale: Optional[float] = None, depthwise=False) -> int:
    """Replace every attention-shaped child (``nn.Linear`` children ``qkv`` [3C, C] and
    ``proj`` [C, C], optionally ``gate_proj`` and RMSNorms ``q_norm`` / ``k_norm``) by a
    :class:`FusedNA3DAttention` sharing those modules: the qkv GEMM, the (qk-norm +)
    RoPE + pack kernel, NA3D, the gate GEMM and the proj GEMM on the HIP library.

    The pattern is the reference's post-construction ``_use_tanh_gelu`` swap
    (screamcast/strata_wrappers.py:76-100, applied at :342 and :509): modules are
    found by structure, parameters are shared, and state-dict keys and
    ``named_parameters()`` order stay as they were (tests/test_param_order.py:87-119).
    ``num_heads``, ``kernel_size``, ``dilation``, ``qk_norm`` and ``depthwise`` are either
    one value for every swapped module or a sequence with one entry per module, in
    ``model.modules()`` order (a per-block dilation schedule, or
    :func:`alternating_depthwise`, for instance).
    Returns the number of modules swapped; raises ``RuntimeError`` if there were
    none (as ``_use_tanh_gelu`` does)."""
    targets = [(parent, name, child) for parent in list(model.modules())
               for name, child in list(parent.named_children())
               if not isinstance(child, FusedNA3DAttention) and _is_attention(child)]
    if not targets:
        raise RuntimeError("swap_attention found no module with qkv [3C, C] and proj [C, C] Linear children")

    def pick(v, i, is_scalar):
        if is_scalar(v):
            return v
        v = list(v)
        if len(v) != len(targets):
            raise ValueError(f"{len(v)} per-module values for {len(targets)} attention modules")
        return v[i]

    for i, (parent, name, child) in enumerate(targets):
        new = FusedNA3DAttention.from_attention(
            child,
            pick(num_heads, i, lambda v: isinstance(v, int)),
            pick(kernel_size, i, lambda v: isinstance(v, int) or (len(v) == 3 and all(isinstance(t, int) for t in v))),
            pick(dilation, i, lambda v: isinstance(v, int) or (len(v) == 3 and all(isinstance(t, int) for t in v))),
            pick(qk_norm, i, lambda v: isinstance(v, bool)),
            qk_norm_eps, rope_layout, scale,
            pick(depthwise, i, lambda v: isinstance(v, bool)))
        setattr(parent, name, new)
    return len(targets)


def interleaved_dilations(n_layers: int, na_dilation: int, kernel_size, grid, interleaved: bool = True) -> list:
    """Per-block NA3D dilations for ``do_interleaved_dilation`` / ``na_dilations``
    (screamcast/config.py:97-98, passed at screamcast/strata_wrappers.py:326-328).

    The schedule itself lives in physicsnemo's Strata (not available here), so this
    one is this build's reading of the flag names, parity unpinned: without
    interleaving every block is undilated; with it, even blocks are undilated and
    odd blocks dilate every axis by ``na_dilation`` where ``kernel * na_dilation``
    fits the token grid (NATTEN's requirement), else that axis stays undilated.
    Feed the result to ``swap_attention(..., dilation=...)`` or ``StrataBlock``."""
    k = _triple(kernel_size)
    if not interleaved or na_dilation <= 1:
        return [[1, 1, 1] for _ in range(n_layers)]
    odd = [na_dilation if kk * na_dilation <= L else 1 for kk, L in zip(k, grid)]
    return [[1, 1, 1] if i % 2 == 0 else list(odd) for i in range(n_layers)]


def alternating_depthwise(n_layers: int, alternate: bool = True) -> list[bool]:
    """Per-block depth-wise flags for ``do_alt_depthwise_attn`` ("depthwise attention every
    other DiTBlock", screamcast/config.py:101-103).  Which blocks alternate is defined in
    physicsnemo (absent here); this build's convention, parity unpinned: odd-indexed blocks
    are depth-wise, even ones keep the neighbourhood window.  Feed the result to
    ``swap_attention(..., depthwise=...)`` or to ``StrataBlock(depthwise=...)``."""
    return [alternate and i % 2 == 1 for i in range(n_layers)]


def init_xavier_(module: nn.Module, generator: torch.Generator) -> None:
    """Xavier-uniform weights, zero biases (DiT-style init), from one CPU generator."""
    for m in module.modules():
        if isinstance(m, nn.Linear):
            fan_out, fan_in = m.weight.shape
            bound = (6.0 / (fan_in + fan_out)) ** 0.5
            with torch.no_grad():
                w = torch.rand(m.weight.shape, generator=generator, dtype=torch.float32) * (2 * bound) - bound
                m.weight.copy_(w)
                if m.bias is not None:
                    m.bias.zero_()
        elif isinstance(m, ExpertMlp):
            with torch.no_grad():
                for t, b in ((m.w1, m.b1), (m.w2, m.b2)):
                    bound = (6.0 / (t.shape[1] + t.shape[2])) ** 0.5
                    t.copy_(torch.rand(t.shape, generator=generator, dtype=torch.float32) * (2 * bound) - bound)
                    if b is not None:
                        b.zero_()


def block_param_names(gated: bool = False) -> Sequence[str]:
    names = ["attn.qkv.weight", "attn.qkv.bias", "attn.proj.weight", "attn.proj.bias"]
    if gated:
        names += ["attn.gate_proj.weight", "attn.gate_proj.bias"]
    return names + ["mlp.layers.0.weight", "mlp.layers.0.bias", "mlp.layers.2.weight", "mlp.layers.2.bias"]
