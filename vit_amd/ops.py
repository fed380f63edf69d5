"""Torch-tensor wrappers over the per-kernel C-ABI entry points.

Each function mirrors the torch module/function it replaces on the encoder path
(names and argument meaning as in ``transformers`` ``modeling_vit.py``): tensors are CUDA
(ROCm) tensors; results are new tensors. All work is done by libvit_amd.so on the current
torch stream -- there is no eager fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import VIT_BF16, VIT_F32, EPI_BIAS, EPI_GELU, EPI_QUICK_GELU, EPI_RESIDUAL  # noqa: F401

_DT = {torch.float32: VIT_F32, torch.bfloat16: VIT_BF16}
_EPI = {None: EPI_BIAS, "none": EPI_BIAS, "gelu": EPI_GELU, "quick_gelu": EPI_QUICK_GELU}


def dtype_code(t: torch.dtype) -> int:
    try:
        return _DT[t]
    except KeyError:
        raise TypeError(f"vit_amd supports float32 and bfloat16 tensors, got {t}") from None


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dev(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU (vit_amd has no CPU path)")
    return t.contiguous()


def _f32(t, name):
    return None if t is None else _dev(t, name).float()


def _ptr(t):
    return None if t is None else t.data_ptr()


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float) -> torch.Tensor:
    """``nn.LayerNorm(D, eps)`` over the last dim (modeling_vit.py:261-262)."""
    x = _dev(x, "x")
    w, b = _f32(weight, "weight"), _f32(bias, "bias")
    d = x.shape[-1]
    rows = x.numel() // d if d else 0
    y = torch.empty_like(x)
    _lib.check(_lib.load().vit_layernorm_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), rows, d, d, d,
                                             float(eps), dtype_code(x.dtype), _stream()))
    return y


def layer_norm_stats(x: torch.Tensor, eps: float) -> torch.Tensor:
    """Per-row ``(mean * rstd, rstd)`` of nn.LayerNorm's statistics, fp32 ``[..., 2]`` (bf16 input)."""
    x = _bf16(x, "x")
    d = x.shape[-1]
    rows = x.numel() // d
    stats = torch.empty(*x.shape[:-1], 2, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().vit_layernorm_stats(x.data_ptr(), stats.data_ptr(), rows, d, d, float(eps), _lib.VIT_BF16, _stream()))
    return stats


def layer_norm_fold(weight: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, bias: torch.Tensor | None = None):
    """Fold a LayerNorm's affine part into the Linear after it: returns ``(weight * gamma [bf16], colsum, bias')``
    for ``linear_ln_folded`` (include/vit_amd.h, vit_layernorm_fold)."""
    w = _bf16(weight, "weight")
    g, b0 = _f32(gamma, "gamma"), _f32(beta, "beta")
    b = _f32(bias, "bias")
    n, k = w.shape
    wg = torch.empty_like(w)
    c = torch.empty(n, dtype=torch.float32, device=w.device)
    d = torch.empty(n, dtype=torch.float32, device=w.device)
    _lib.check(_lib.load().vit_layernorm_fold(w.data_ptr(), g.data_ptr(), b0.data_ptr(), _ptr(b), wg.data_ptr(), c.data_ptr(),
                                              d.data_ptr(), n, k, _stream()))
    return wg, c, d


def linear_ln_folded(x: torch.Tensor, folded, stats: torch.Tensor, activation: str | None = None) -> torch.Tensor:
    """``act(F.linear(layer_norm(x), weight, bias))`` from the UN-normalised ``x`` [bf16], the output of
    ``layer_norm_fold`` and ``layer_norm_stats(x)`` (modeling_vit.py:274 + :216-218, :281 + :250-251)."""
    x = _bf16(x, "x")
    wg, c, d = folded
    k, n = x.shape[-1], wg.shape[0]
    if wg.shape[1] != k:
        raise ValueError(f"linear_ln_folded: x has {k} features, weight expects {wg.shape[1]}")
    m = x.numel() // k
    out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    _lib.check(_lib.load().vit_gemm_ln_folded(x.data_ptr(), wg.data_ptr(), d.data_ptr(), c.data_ptr(), stats.data_ptr(),
                                              out.data_ptr(), m, n, k, _EPI[activation], _stream()))
    return out


def row_stats_finalize(row_part: torch.Tensor, eps: float, stats: torch.Tensor | None = None) -> torch.Tensor:
    """(mean * rstd, rstd) per row from the ``[dim / 64, rows, 2]`` fp32 row sums a residual GEMM left."""
    ng, m, _ = row_part.shape
    if stats is None:
        stats = torch.empty(m, 2, dtype=torch.float32, device=row_part.device)
    _lib.check(_lib.load().vit_row_stats_finalize(row_part.data_ptr(), stats.data_ptr(), m, ng * 64, float(eps), _stream()))
    return stats


def linear_residual_row_stats(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor,
                              eps: float, out=None, part=None, finalize: bool = True):
    """``F.linear(x, weight, bias) + residual`` [bf16] together with the folded-LayerNorm statistics of the rows it stored
    (what ``layer_norm_stats(out, eps)`` computes, bit for bit): the residual epilogue leaves per-64-column row sums and a
    small launch finalises them (modeling_vit.py:236 + :277 -> :281, :252 + :284 -> :274). Returns (out, stats, row_part)."""
    x = _bf16(x, "x")
    w = _bf16(weight, "weight")
    r = _bf16(residual, "residual")
    b = _f32(bias, "bias")
    k, n = x.shape[-1], w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"linear_residual_row_stats: x has {k} features, weight expects {w.shape[1]}")
    m = x.numel() // k
    if out is None:
        out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    if part is None:
        part = torch.empty(max(n // 64, 1), m, 2, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().vit_gemm_residual_row_stats(x.data_ptr(), w.data_ptr(), _ptr(b), r.data_ptr(), out.data_ptr(),
                                                       part.data_ptr(), m, n, k, _stream()))
    stats = row_stats_finalize(part, eps) if finalize else None
    return out, stats, part


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` followed by an activation or a residual add
    (modeling_vit.py:216-218, 236+277, 250-252+284). weight is [out, in]."""
    x = _dev(x, "x")
    w = _dev(weight, "weight").to(x.dtype)
    b = _f32(bias, "bias")
    k = x.shape[-1]
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"linear: x has {k} features, weight expects {w.shape[1]}")
    m = x.numel() // k if k else 0
    out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    if residual is not None:
        if activation not in (None, "none"):
            raise ValueError("linear: activation and residual are mutually exclusive epilogues")
        residual = _dev(residual, "residual").to(x.dtype)
        if residual.shape != out.shape:
            raise ValueError("linear: residual shape mismatch")
        epi = EPI_RESIDUAL
    else:
        if activation not in _EPI:
            raise ValueError(f"linear: unknown activation {activation!r}")
        epi = _EPI[activation]
    _lib.check(_lib.load().vit_gemm_bias_act(x.data_ptr(), w.data_ptr(), _ptr(b), _ptr(residual), out.data_ptr(), m, n,
                                             k, epi, dtype_code(x.dtype), _stream()))
    return out


def attention(qkv: torch.Tensor, num_heads: int) -> torch.Tensor:
    """Fused softmax(QK^T/sqrt(dh))V on the packed projection output.

    qkv: [B, N, 3*D] (q | k | v along the last dim) -> [B, N, D], equal to
    eager_attention_forward(...)'s attn_output after ``.reshape(B, N, D)``
    (modeling_vit.py:164-189, 235)."""
    qkv = _dev(qkv, "qkv")
    b, n, d3 = qkv.shape
    if d3 % (3 * num_heads):
        raise ValueError("attention: last dim must be 3 * num_heads * head_dim")
    d = d3 // 3
    out = torch.empty(b, n, d, dtype=qkv.dtype, device=qkv.device)
    _lib.check(_lib.load().vit_attention_fwd(qkv.data_ptr(), out.data_ptr(), b, n, num_heads, d // num_heads,
                                             dtype_code(qkv.dtype), _stream()))
    return out


def patch_embed(pixel_values: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, cls_token: torch.Tensor,
                position_embeddings: torch.Tensor, patch_size: int) -> torch.Tensor:
    """ViTEmbeddings.forward (modeling_vit.py:129-161): Conv2d(k=s=P) patch projection as an
    im2col-free GEMM, CLS prepend and position add. weight is the Conv2d weight [D, C, P, P]."""
    px = _dev(pixel_values, "pixel_values")
    b, c, h, w_ = px.shape
    if h != w_ or h % patch_size:
        raise ValueError("patch_embed: square images divisible by the patch size only")
    dt = dtype_code(px.dtype)
    d = weight.shape[0]
    kreal = c * patch_size * patch_size
    kpad = _lib.load().vit_patch_kpad(c, patch_size, dt)
    wmat = _dev(weight, "weight").reshape(d, kreal).to(px.dtype)
    if kpad != kreal:  # zero-pad K to the kernel's 16-byte chunk granularity
        wmat = torch.nn.functional.pad(wmat, (0, kpad - kreal))
    n = (h // patch_size) ** 2 + 1
    cls = _f32(cls_token, "cls_token").reshape(d)
    pos = _f32(position_embeddings, "position_embeddings").reshape(n, d)
    bias = _f32(bias, "bias")
    out = torch.empty(b, n, d, dtype=px.dtype, device=px.device)
    _lib.check(_lib.load().vit_patch_embed_fwd(px.data_ptr(), wmat.data_ptr(), _ptr(bias), cls.data_ptr(),
                                               pos.data_ptr(), out.data_ptr(), b, c, h, patch_size, d, dt, _stream()))
    return out


# --------------------------------------------------------------------------- training-step ops
_EPI_GRAD = {"gelu": _lib.EPI_DGELU, "quick_gelu": _lib.EPI_DQUICK_GELU}


def _bf16(t: torch.Tensor, name: str) -> torch.Tensor:
    t = _dev(t, name)
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the training kernels take bfloat16 activations, got {t.dtype}")
    return t


def linear_train(x, weight, bias, activation: str):
    """fc1 of ViTMLP in a training forward: returns (act(x W^T + b), x W^T + b) -- the
    pre-activation is what the backward multiplies with (modeling_vit.py:250-251)."""
    x, w = _bf16(x, "x"), _bf16(weight, "weight")
    b = _f32(bias, "bias")
    m, k, n = x.numel() // x.shape[-1], x.shape[-1], w.shape[0]
    out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    pre = torch.empty_like(out)
    _lib.check(_lib.load().vit_gemm_ex(x.data_ptr(), w.data_ptr(), _ptr(b), None, out.data_ptr(), pre.data_ptr(), m, n, k,
                                       _EPI[activation], 0, _stream()))
    return out, pre


def linear_dgrad(dy, weight_t, pre_activation=None, activation: str | None = None):
    """dX = dY W as an NT GEMM on the transposed weight ``weight_t`` = W^T ([in, out]); with
    ``pre_activation`` the result is multiplied by act'(pre_activation) in the epilogue."""
    dy, wt = _bf16(dy, "dy"), _bf16(weight_t, "weight_t")
    m, k, n = dy.numel() // dy.shape[-1], dy.shape[-1], wt.shape[0]
    out = torch.empty(*dy.shape[:-1], n, dtype=dy.dtype, device=dy.device)
    epi, aux = _lib.EPI_BIAS, None
    if pre_activation is not None:
        epi, aux = _EPI_GRAD[activation], _bf16(pre_activation, "pre_activation").data_ptr()
    _lib.check(_lib.load().vit_gemm_ex(dy.data_ptr(), wt.data_ptr(), None, aux, out.data_ptr(), None, m, n, k, epi, 0,
                                       _stream()))
    return out


def transpose_pad(x2d, pad_to: int = 128, colsum: bool = False, skip_first_of: int = 0):
    """[R, C] bf16 -> [C, Rpad] (zero padded), optionally with the fp32 column sums of the input."""
    x2d = _bf16(x2d, "x")
    rows_mem, c = x2d.shape
    r = rows_mem if skip_first_of == 0 else rows_mem // (skip_first_of + 1) * skip_first_of
    rpad = (r + pad_to - 1) // pad_to * pad_to
    out = torch.empty(c, rpad, dtype=x2d.dtype, device=x2d.device)
    cs = torch.zeros(c, dtype=torch.float32, device=x2d.device) if colsum else None
    _lib.check(_lib.load().vit_transpose_pad(x2d.data_ptr(), out.data_ptr(), _ptr(cs), r, c, rpad, skip_first_of,
                                             _stream()))
    return (out, cs) if colsum else out


def linear_wgrad(dy_t, x_t):
    """dW [out, in] (fp32) = dY^T X from the transposed, zero-padded operands
    dy_t = dY^T [out, Mpad], x_t = X^T [in, Mpad]."""
    dy_t, x_t = _bf16(dy_t, "dy_t"), _bf16(x_t, "x_t")
    if dy_t.shape[1] != x_t.shape[1]:
        raise ValueError("linear_wgrad: operands disagree on the padded token count")
    m, k, n = dy_t.shape[0], dy_t.shape[1], x_t.shape[0]
    out = torch.empty(m, n, dtype=torch.float32, device=dy_t.device)
    _lib.check(_lib.load().vit_gemm_ex(dy_t.data_ptr(), x_t.data_ptr(), None, None, out.data_ptr(), None, m, n, k,
                                       _lib.EPI_BIAS, 1, _stream()))
    return out


def attention_train(qkv, num_heads: int):
    """attention() that also returns the base-2 log-sum-exp [B, H, N] the backward needs."""
    qkv = _bf16(qkv, "qkv")
    b, n, d3 = qkv.shape
    d = d3 // 3
    out = torch.empty(b, n, d, dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty(b, num_heads, n, dtype=torch.float32, device=qkv.device)
    _lib.check(_lib.load().vit_attention_fwd_train(qkv.data_ptr(), out.data_ptr(), lse.data_ptr(), b, n, num_heads,
                                                   d // num_heads, _stream()))
    return out, lse


def attention_backward(qkv, out, d_out, lse, num_heads: int):
    """Gradient of attention() w.r.t. the packed qkv (eager_attention_forward, modeling_vit.py:164-189)."""
    qkv, out, d_out = _bf16(qkv, "qkv"), _bf16(out, "out"), _bf16(d_out, "d_out")
    b, n, d3 = qkv.shape
    d = d3 // 3
    dqkv = torch.empty_like(qkv)
    delta = torch.empty(b, num_heads, n, dtype=torch.float32, device=qkv.device)
    _lib.check(_lib.load().vit_attention_bwd(qkv.data_ptr(), out.data_ptr(), d_out.data_ptr(), lse.data_ptr(),
                                             delta.data_ptr(), dqkv.data_ptr(), b, n, num_heads, d // num_heads,
                                             _stream()))
    return dqkv


def layer_norm_backward(x, dy, weight, eps: float, d_residual=None):
    """Returns (dx [+ d_residual], dgamma, dbeta) of nn.LayerNorm (modeling_vit.py:261-262)."""
    x, dy = _bf16(x, "x"), _bf16(dy, "dy")
    w = _f32(weight, "weight")
    d = x.shape[-1]
    rows = x.numel() // d
    dx = torch.empty_like(x)
    dg = torch.zeros(d, dtype=torch.float32, device=x.device)
    db = torch.zeros(d, dtype=torch.float32, device=x.device)
    dres = None if d_residual is None else _bf16(d_residual, "d_residual").data_ptr()
    _lib.check(_lib.load().vit_layernorm_bwd(x.data_ptr(), dy.data_ptr(), w.data_ptr(), dres, dx.data_ptr(),
                                             dg.data_ptr(), db.data_ptr(), rows, d, float(eps), _stream()))
    return dx, dg, db


# --------------------------------------------------------------------------- norms of query / key heads with rotation
_NORM = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}


def rope_table(grid, rot_dim: int, theta: float | None = None, device="cuda") -> torch.Tensor:
    """(cos, sin) fp32 ``[grid_h * grid_w, rot_dim / 2, 2]`` for ``qk_norm_rope``: on a ``(grid_h, grid_w)`` grid half of the
    pairs turn with the row and half with the column (``theta`` 100), on a sequence ``(1, n)`` all of them with the place
    (``theta`` 10000). Frequencies ``theta ** (-i / pairs)``; the angles are computed in 64 bits."""
    gh, gw = (int(v) for v in grid)
    if gh < 1 or gw < 1 or rot_dim < 4 or rot_dim % 4:
        raise ValueError(f"rope_table: grid {gh} x {gw}, rot_dim {rot_dim}")
    y = torch.arange(gh, dtype=torch.float64).repeat_interleave(gw)
    x = torch.arange(gw, dtype=torch.float64).repeat(gh)

    def angles(place, pairs, base):
        return place[:, None] * base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)

    if gh == 1:
        a = angles(x, rot_dim // 2, 10000.0 if theta is None else float(theta))
    else:
        base = 100.0 if theta is None else float(theta)
        a = torch.cat([angles(y, rot_dim // 4, base), angles(x, rot_dim // 4, base)], dim=-1)
    return torch.stack([a.cos(), a.sin()], dim=-1).float().to(device)


def _elsewhere(t: torch.Tensor) -> bool:
    """whether ``t`` lives on another device than the current one (the calls below then enter it)"""
    return t.is_cuda and t.get_device() != torch._C._cuda_getDevice()  # (a tensor is there, so the device is set up)


def _raw_stream(t: torch.Tensor) -> int:
    """The current stream of ``t``'s device as a handle: what ``torch.cuda.current_stream().cuda_stream`` gives, without building
    the Stream object (2.6 us of a 5 us call)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _vec(t, name: str, n: int, ref: torch.Tensor, what: str):
    """an fp32 contiguous vector of ``n`` on ``ref``'s device, or None"""
    if t is None:
        return None
    if t.shape != (n,):
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected ({n},)")
    return _single(_near(t, name, ref))


def _single(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.float().contiguous()


def _near(t: torch.Tensor, name: str, ref: torch.Tensor) -> torch.Tensor:
    if t.get_device() != ref.get_device():
        raise ValueError(f"{name} is on {t.device}, qkv on {ref.device}")
    return t


def _packed_heads(qkv: torch.Tensor, num_heads: int, num_kv_heads: int | None, what: str):
    """(batch, tokens, key / value heads, head_dim) of a packed [B, N, (H + 2 Hk) dh] projection output"""
    if qkv.dim() != 3:
        raise ValueError(f"{what}: qkv must be [batch, tokens, (heads + 2 kv_heads) * head_dim], got {tuple(qkv.shape)}")
    hk = num_heads if num_kv_heads is None else num_kv_heads
    if num_heads < 1 or hk < 1 or num_heads % hk:
        raise ValueError(f"{what}: {num_heads} heads, {hk} key / value heads")
    b, n, w = qkv.shape
    if b == 0 or n == 0 or w == 0 or w % (num_heads + 2 * hk):
        raise ValueError(f"{what}: shape {tuple(qkv.shape)} for {num_heads} + 2 * {hk} heads")
    return b, n, hk, w // (num_heads + 2 * hk)


def _qk_norm_args(qkv, num_heads, num_kv_heads, eps, rope, positions, interleaved, norm, what):
    if norm not in _NORM:
        raise ValueError(f"{what}: unknown norm {norm!r}")
    b, n, hk, dh = _packed_heads(qkv, num_heads, num_kv_heads, what)
    rot_dim = rope_len = per_sample = 0
    if rope is not None:
        shape = rope.shape
        if len(shape) != 3 or shape[2] != 2 or shape[0] == 0:
            raise ValueError(f"{what}: rope must be [positions, rot_dim / 2, 2], got {tuple(shape)}")
        rope = _single(_near(rope, "rope", qkv))
        rope_len, rot_dim = shape[0], 2 * shape[1]
    if positions is not None:
        if rope is None:
            raise ValueError(f"{what}: positions without a rope table")
        shape = positions.shape
        per_sample = len(shape) == 2
        if positions.dtype is not torch.int32 or shape != ((b, n) if per_sample else (n,)):
            raise ValueError(f"{what}: positions must be int32 [{n}] or [{b}, {n}], got {positions.dtype} {tuple(shape)}")
        positions = _near(positions, "positions", qkv).contiguous()
    cfg = _lib.vit_qk_norm_config(b, n, num_heads, hk, dh, _NORM[norm], rot_dim, bool(interleaved), rope_len, per_sample,
                                  dtype_code(qkv.dtype), eps)
    return cfg, dh, rope, positions


def _out_like(ref: torch.Tensor, out, what: str) -> torch.Tensor:
    if out is None:
        return torch.empty_like(ref)
    if out.shape != ref.shape or out.dtype != ref.dtype or out.device != ref.device or not out.is_contiguous():
        raise ValueError(f"{what}: out must be a contiguous {ref.dtype} tensor of shape {tuple(ref.shape)} on {ref.device}")
    return out


def qk_norm_rope(qkv: torch.Tensor, num_heads: int, q_weight: torch.Tensor, k_weight: torch.Tensor, q_bias=None, k_bias=None,
                 eps: float = 1e-6, rope: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 interleaved: bool = False, norm: str = "rms", num_kv_heads: int | None = None, out=None) -> torch.Tensor:
    """Norm of every query and key head of a packed projection output (``norm``: "rms", or "layer" with optional biases;
    weights ``[head_dim]`` shared by the heads), then the rotary rotation of the token's position, in one pass: the step
    between ``linear`` and ``attention`` / ``attention_rel_bias``.

    qkv ``[B, N, (H + 2 Hk) * dh]`` fp32 or bf16, q heads | k heads | v heads; the values pass through. ``rope``: (cos, sin) fp32
    ``[P, rot_dim / 2, 2]`` (``rope_table``); pairs are ``(i, i + rot_dim / 2)``, or neighbours with ``interleaved``.
    ``positions``: int32 ``[N]`` or ``[B, N]`` rows of ``rope`` (default: the token's index); one outside ``[0, P)`` leaves its token
    unturned (-1 for CLS). ``out=qkv`` works in place."""
    if _elsewhere(qkv):
        with torch.cuda.device(qkv.device):
            return qk_norm_rope(qkv, num_heads, q_weight, k_weight, q_bias, k_bias, eps, rope, positions, interleaved, norm, num_kv_heads, out)
    if norm != "layer" and (q_bias is not None or k_bias is not None):
        raise ValueError("qk_norm_rope: biases belong to norm='layer'")
    if out is not None and not qkv.is_contiguous():
        raise ValueError("qk_norm_rope: out needs a contiguous qkv")
    what = "qk_norm_rope"
    qkv = _dev(qkv, "qkv")
    cfg, dh, rope, positions = _qk_norm_args(qkv, num_heads, num_kv_heads, eps, rope, positions, interleaved, norm, what)
    # (named: a converted copy lives until the launch is enqueued)
    qw, kw = _vec(q_weight, "q_weight", dh, qkv, what), _vec(k_weight, "k_weight", dh, qkv, what)
    qb, kb = _vec(q_bias, "q_bias", dh, qkv, what), _vec(k_bias, "k_bias", dh, qkv, what)
    out = _out_like(qkv, out, what)
    _lib.check(_lib.load().vit_qk_norm_rope_fwd(cfg, qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), _ptr(qb), _ptr(kb), _ptr(rope),
                                                _ptr(positions), out.data_ptr(), _raw_stream(qkv)))
    return out


def qk_norm_rope_backward(qkv: torch.Tensor, d_out: torch.Tensor, num_heads: int, q_weight: torch.Tensor, k_weight: torch.Tensor,
                          eps: float = 1e-6, rope: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                          interleaved: bool = False, norm: str = "rms", num_kv_heads: int | None = None, out=None):
    """Gradient of ``qk_norm_rope`` from its INPUT ``qkv`` and the gradient of its output (what ``attention_backward`` returns):
    ``(dqkv, dq_weight, dk_weight, dq_bias, dk_bias)``, parameter gradients fp32 (biases: ``None`` unless norm is "layer").
    ``out=d_out`` works in place. Bitwise reproducible."""
    if _elsewhere(qkv):
        with torch.cuda.device(qkv.device):
            return qk_norm_rope_backward(qkv, d_out, num_heads, q_weight, k_weight, eps, rope, positions, interleaved, norm, num_kv_heads, out)
    what = "qk_norm_rope_backward"
    if out is not None and not d_out.is_contiguous():
        raise ValueError(f"{what}: out needs a contiguous d_out")
    qkv, d_out = _dev(qkv, "qkv"), _near(_dev(d_out, "d_out"), "d_out", qkv)
    if d_out.shape != qkv.shape or d_out.dtype != qkv.dtype:
        raise ValueError(f"{what}: d_out {d_out.dtype} {tuple(d_out.shape)} for qkv {qkv.dtype} {tuple(qkv.shape)}")
    cfg, dh, rope, positions = _qk_norm_args(qkv, num_heads, num_kv_heads, eps, rope, positions, interleaved, norm, what)
    qw, kw = _vec(q_weight, "q_weight", dh, qkv, what), _vec(k_weight, "k_weight", dh, qkv, what)
    out = _out_like(d_out, out, what)
    lib = _lib.load()
    sums = torch.empty((4 if norm == "layer" else 2, dh), dtype=torch.float32, device=qkv.device)
    need = lib.vit_qk_norm_rope_bwd_workspace_bytes(cfg)
    ws = torch.empty((need,), dtype=torch.uint8, device=qkv.device)
    grads = [*sums.unbind()] + [None] * (4 - sums.shape[0])
    _lib.check(lib.vit_qk_norm_rope_bwd(cfg, qkv.data_ptr(), d_out.data_ptr(), qw.data_ptr(), kw.data_ptr(), _ptr(rope), _ptr(positions),
                                        out.data_ptr(), *map(_ptr, grads), ws.data_ptr(), need, _raw_stream(qkv)))
    return (out, *grads)


# --------------------------------------------------------------------------- attention with a relative position bias
def _rel_args(qkv, num_heads, table, buckets, lengths, num_kv_heads, scale, what):
    b, n, hk, dh = _packed_heads(qkv, num_heads, num_kv_heads, what)
    if n != buckets.seq:
        raise ValueError(f"{what}: qkv has {n} tokens, the buckets are for {buckets.seq}")
    if table.shape != (buckets.num_buckets, num_heads):
        raise ValueError(f"{what}: table has shape {tuple(table.shape)}, expected ({buckets.num_buckets}, {num_heads})")
    table = _single(_near(table, "table", qkv))
    if buckets.bucket_of is not None:
        _near(buckets.bucket_of, "buckets", qkv)
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.shape != (b,):
            raise ValueError(f"{what}: lengths must be int32 [{b}], got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = _near(lengths, "lengths", qkv).contiguous()
    return b, n, hk, dh, table, lengths, dh ** -0.5 if scale is None else scale


def attention_rel_bias(qkv: torch.Tensor, num_heads: int, table: torch.Tensor, buckets, lengths: torch.Tensor | None = None,
                       num_kv_heads: int | None = None, scale: float | None = None) -> torch.Tensor:
    """``attention`` with a learned relative position bias: softmax(scale Q K^T + table[bucket(i, j), head]) V.

    qkv ``[B, N, (H + 2 Hk) * dh]`` fp32 or bf16 -> ``[B, N, H * dh]``; ``table`` ``[num_buckets, H]`` (entries below -1e30 mask their
    pairs, whose keys and values have to be finite all the same; a query left without a key gives zeros; others up to 1e30 in size,
    also where every key of a query carries one: a finite mask is a number like any other); ``buckets``:
    ``rel_pos.RelPosBuckets``; ``lengths``: int32 ``[B]``, tokens in use (rows behind are never read and give zeros); ``scale`` defaults
    to ``dh ** -0.5``."""
    if _elsewhere(qkv):
        with torch.cuda.device(qkv.device):
            return attention_rel_bias(qkv, num_heads, table, buckets, lengths, num_kv_heads, scale)
    qkv = _dev(qkv, "qkv")
    b, n, hk, dh, table, lengths, scale = _rel_args(qkv, num_heads, table, buckets, lengths, num_kv_heads, scale, "attention_rel_bias")
    out = qkv.new_empty((b, n, num_heads * dh))
    _lib.check(_lib.load().vit_attention_rel_fwd(buckets._c(), qkv.data_ptr(), table.data_ptr(), _ptr(lengths), out.data_ptr(), None,
                                                 b, num_heads, hk, dh, scale, dtype_code(qkv.dtype), _raw_stream(qkv)))
    return out


def attention_rel_bias_train(qkv: torch.Tensor, num_heads: int, table: torch.Tensor, buckets, lengths: torch.Tensor | None = None,
                             num_kv_heads: int | None = None, scale: float | None = None):
    """``attention_rel_bias`` (bf16) that also returns what its backward needs: ``(out, saved)``, ``saved`` the base-2 log-sum-exp of
    every row ``[B, H, N]`` (+inf where a query has no key; the backward makes the statistic of rows beyond +-256 anew)."""
    if _elsewhere(qkv):
        with torch.cuda.device(qkv.device):
            return attention_rel_bias_train(qkv, num_heads, table, buckets, lengths, num_kv_heads, scale)
    qkv = _bf16(qkv, "qkv")
    b, n, hk, dh, table, lengths, scale = _rel_args(qkv, num_heads, table, buckets, lengths, num_kv_heads, scale, "attention_rel_bias_train")
    out = qkv.new_empty((b, n, num_heads * dh))
    lse = torch.empty((b, num_heads, n), dtype=torch.float32, device=qkv.device)
    _lib.check(_lib.load().vit_attention_rel_fwd(buckets._c(), qkv.data_ptr(), table.data_ptr(), _ptr(lengths), out.data_ptr(),
                                                 lse.data_ptr(), b, num_heads, hk, dh, scale, _lib.VIT_BF16, _raw_stream(qkv)))
    return out, lse


def attention_rel_bias_backward(qkv: torch.Tensor, out: torch.Tensor, d_out: torch.Tensor, saved, num_heads: int, table: torch.Tensor,
                                buckets, lengths: torch.Tensor | None = None, num_kv_heads: int | None = None, scale: float | None = None):
    """Gradient of ``attention_rel_bias`` from ``attention_rel_bias_train``'s ``(out, saved)`` and the gradient of ``out``:
    ``(dqkv bf16, d_table fp32 [num_buckets, H])``. The other arguments as in the forward. Bitwise reproducible."""
    if _elsewhere(qkv):
        with torch.cuda.device(qkv.device):
            return attention_rel_bias_backward(qkv, out, d_out, saved, num_heads, table, buckets, lengths, num_kv_heads, scale)
    qkv, out, d_out = _bf16(qkv, "qkv"), _bf16(out, "out"), _bf16(d_out, "d_out")
    b, n, hk, dh, table, lengths, scale = _rel_args(qkv, num_heads, table, buckets, lengths, num_kv_heads, scale, "attention_rel_bias_backward")
    wide = (b, n, num_heads * dh)
    if out.shape != wide or d_out.shape != wide or out.device != qkv.device or d_out.device != qkv.device:
        raise ValueError(f"attention_rel_bias_backward: out and d_out must be {wide} on {qkv.device}, got {tuple(out.shape)} on {out.device}, "
                         f"{tuple(d_out.shape)} on {d_out.device}")
    if saved.shape != (b, num_heads, n) or saved.dtype != torch.float32 or saved.device != qkv.device or not saved.is_contiguous():
        raise ValueError(f"attention_rel_bias_backward: saved is not what attention_rel_bias_train returned for {tuple(qkv.shape)}")
    lib = _lib.load()
    c = buckets._c()
    need = lib.vit_attention_rel_bwd_workspace_bytes(c, b, num_heads, dh)
    ws = torch.empty((need,), dtype=torch.uint8, device=qkv.device)
    dqkv = torch.empty_like(qkv)
    d_table = torch.empty((buckets.num_buckets, num_heads), dtype=torch.float32, device=qkv.device)
    _lib.check(lib.vit_attention_rel_bwd(c, qkv.data_ptr(), table.data_ptr(), _ptr(lengths), out.data_ptr(), d_out.data_ptr(),
                                         saved.data_ptr(), dqkv.data_ptr(), d_table.data_ptr(), ws.data_ptr(), need,
                                         b, num_heads, hk, dh, scale, _raw_stream(qkv)))
    return dqkv, d_table
