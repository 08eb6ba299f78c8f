"""CPU oracle for the IR-SDE score network ``ConditionalUNet`` (TEST INFRASTRUCTURE ONLY, see oracle/__init__.py).

Functional restatement on a flat ``state_dict`` of (U = /root/reference/legacy/third_party/
universal-image-restoration/config/daclip-sde/models/modules/):
  U/DenoisingUNet_arch.py:118-174  forward (input assembly, reflect pad, time/prompt embedding, down/mid/up, crop)
  U/module_util.py:27-48           Residual, SinusoidalPosEmb
  U/module_util.py:77-97           gain-only channel LayerNorm, PreNorm
  U/module_util.py:100-153         Upsample / Downsample / Block / ResBlock
  U/module_util.py:157-185         LinearAttention
  U/attention.py:37-64,152-261     GEGLU feed-forward, CrossAttention, BasicTransformerBlock, SpatialTransformer
Pinned by tests/golden/unet_*.npz, generated by running the reference module itself.
"""
from __future__ import annotations

import math
from typing import Dict, List, Optional

import torch
import torch.nn.functional as F

SD = Dict[str, torch.Tensor]


def sinusoidal_pos_emb(time: torch.Tensor, dim: int) -> torch.Tensor:
    half = dim // 2                                                                   # module_util.py:41-48
    e = math.log(10000) / (half - 1)
    e = torch.exp(torch.arange(half) * -e)
    e = time[:, None] * e[None, :]
    return torch.cat((e.sin(), e.cos()), dim=-1)


# The reference picks eps by dtype (module_util.py:83): 1e-5 for float32, 1e-3 for anything else -- INCLUDING
# float64.  The golden "_f64" vectors therefore carry eps = 1e-3; they pin this restatement's math to ~1e-12.
# GPU parity tests need a high-precision version of the *fp32 function* instead: they set FORCE_EPS = 1e-5.
FORCE_EPS: Optional[float] = None


def chan_layernorm(x: torch.Tensor, g: torch.Tensor) -> torch.Tensor:
    eps = FORCE_EPS if FORCE_EPS is not None else (1e-5 if x.dtype == torch.float32 else 1e-3)   # :83
    var = torch.var(x, dim=1, unbiased=False, keepdim=True)
    mean = torch.mean(x, dim=1, keepdim=True)
    return (x - mean) * (var + eps).rsqrt() * g


def res_block(sd: SD, p: str, x: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
    ss = F.linear(F.silu(t), sd[p + "mlp.1.weight"], sd[p + "mlp.1.bias"])[:, :, None, None]   # :134-136,143-147
    scale, shift = ss.chunk(2, dim=1)
    h = F.conv2d(x, sd[p + "block1.proj.weight"], None, padding=1)
    h = F.silu(h * (scale + 1) + shift)                                               # :121-128
    h = F.silu(F.conv2d(h, sd[p + "block2.proj.weight"], None, padding=1))
    r = F.conv2d(x, sd[p + "res_conv.weight"]) if (p + "res_conv.weight") in sd else x
    return h + r                                                                      # :153


def linear_attention(sd: SD, p: str, x: torch.Tensor, heads: int = 4) -> torch.Tensor:
    b, c, h, w = x.shape                                                              # :170-185
    q, k, v = F.conv2d(x, sd[p + "to_qkv.weight"]).chunk(3, dim=1)
    q, k, v = (t.reshape(b, heads, -1, h * w) for t in (q, k, v))
    dh = q.shape[2]
    q = q.softmax(dim=-2) * dh ** -0.5
    k = k.softmax(dim=-1)
    v = v / (h * w)
    ctx = torch.einsum("bhdn,bhen->bhde", k, v)
    out = torch.einsum("bhde,bhdn->bhen", ctx, q).reshape(b, -1, h, w)
    out = F.conv2d(out, sd[p + "to_out.0.weight"], sd[p + "to_out.0.bias"])
    return chan_layernorm(out, sd[p + "to_out.1.g"])


def _mh_attention(q, k, v, heads: int) -> torch.Tensor:
    b, n, d = q.shape
    dh = d // heads
    sp = lambda t: t.reshape(b, t.shape[1], heads, dh).transpose(1, 2)  # noqa: E731
    a = torch.softmax(sp(q) @ sp(k).transpose(-1, -2) * dh ** -0.5, dim=-1)          # attention.py:176-190
    return (a @ sp(v)).transpose(1, 2).reshape(b, n, d)


def spatial_transformer(sd: SD, p: str, x: torch.Tensor, context: torch.Tensor) -> torch.Tensor:
    b, c, h, w = x.shape                                                              # attention.py:250-261
    heads = c // 32
    y = F.group_norm(x, 32, sd[p + "norm.weight"], sd[p + "norm.bias"], 1e-6)
    y = F.conv2d(y, sd[p + "proj_in.weight"], sd[p + "proj_in.bias"])
    y = y.reshape(b, c, h * w).transpose(1, 2)
    t = p + "transformer_blocks.0."
    ln = lambda z, nm: F.layer_norm(z, (c,), sd[t + nm + ".weight"], sd[t + nm + ".bias"], 1e-5)  # noqa: E731
    z = ln(y, "norm1")
    a = _mh_attention(F.linear(z, sd[t + "attn1.to_q.weight"]), F.linear(z, sd[t + "attn1.to_k.weight"]),
                      F.linear(z, sd[t + "attn1.to_v.weight"]), heads)
    y = F.linear(a, sd[t + "attn1.to_out.0.weight"], sd[t + "attn1.to_out.0.bias"]) + y        # :213
    z = ln(y, "norm2")
    a = _mh_attention(F.linear(z, sd[t + "attn2.to_q.weight"]), F.linear(context, sd[t + "attn2.to_k.weight"]),
                      F.linear(context, sd[t + "attn2.to_v.weight"]), heads)
    y = F.linear(a, sd[t + "attn2.to_out.0.weight"], sd[t + "attn2.to_out.0.bias"]) + y        # :214
    z = ln(y, "norm3")
    u, gate = F.linear(z, sd[t + "ff.net.0.proj.weight"], sd[t + "ff.net.0.proj.bias"]).chunk(2, dim=-1)
    y = F.linear(u * F.gelu(gate), sd[t + "ff.net.2.weight"], sd[t + "ff.net.2.bias"]) + y      # :215
    y = y.transpose(1, 2).reshape(b, c, h, w)
    return F.conv2d(y, sd[p + "proj_out.weight"], sd[p + "proj_out.bias"]) + x


def attn_block(sd: SD, p: str, x: torch.Tensor, image_context: Optional[torch.Tensor]) -> torch.Tensor:
    """Residual(PreNorm(dim, LinearAttention | SpatialTransformer))."""
    y = chan_layernorm(x, sd[p + "fn.norm.g"])
    if (p + "fn.fn.to_qkv.weight") in sd:
        return linear_attention(sd, p + "fn.fn.", y) + x
    return spatial_transformer(sd, p + "fn.fn.", y, image_context) + x


def unet_forward(sd: SD, xt: torch.Tensor, cond: torch.Tensor, time, text_context: Optional[torch.Tensor] = None,
                 image_context: Optional[torch.Tensor] = None, taps: Optional[dict] = None) -> torch.Tensor:
    depth = 0
    while f"downs.{depth}.0.block1.proj.weight" in sd:
        depth += 1
    nf = sd["init_conv.weight"].shape[0]
    if isinstance(time, (int, float)):
        time = torch.tensor([time])                                                   # DenoisingUNet_arch.py:120-121
    x = torch.cat([xt - cond, cond], dim=1)
    H, W = x.shape[2:]
    s = 2 ** depth
    x = F.pad(x, (0, (s - W % s) % s, 0, (s - H % s) % s), "reflect")               # :111-116
    x = F.conv2d(x, sd["init_conv.weight"], None, padding=3)
    x_ = x
    dt = x.dtype
    t = sinusoidal_pos_emb(time, nf).to(dt)
    t = F.linear(F.gelu(F.linear(t, sd["time_mlp.1.weight"], sd["time_mlp.1.bias"])), sd["time_mlp.3.weight"],
                 sd["time_mlp.3.bias"])
    if "prompt" in sd and text_context is not None:                                   # :133-137
        pe = F.linear(F.silu(F.linear(text_context, sd["text_mlp.0.weight"], sd["text_mlp.0.bias"])),
                      sd["text_mlp.2.weight"], sd["text_mlp.2.bias"])
        pe = torch.softmax(pe, dim=1) * sd["prompt"]
        t = t + F.linear(pe, sd["prompt_mlp.weight"], sd["prompt_mlp.bias"])
    ctx = image_context                                                               # :139-140; (B, L, D): L states
    if ctx is not None and ctx.dim() == 2:
        ctx = ctx.unsqueeze(1)
    if taps is not None:
        taps["t"], taps["init"] = t, x
    hs: List[torch.Tensor] = []
    for i in range(depth):
        p = f"downs.{i}."
        x = res_block(sd, p + "0.", x, t)
        hs.append(x)
        x = res_block(sd, p + "1.", x, t)
        x = attn_block(sd, p + "2.", x, ctx)
        hs.append(x)
        if taps is not None:
            taps[f"down{i}"] = x
        if i != depth - 1:
            x = F.conv2d(x, sd[p + "3.weight"], sd[p + "3.bias"], stride=2, padding=1)
        else:
            x = F.conv2d(x, sd[p + "3.weight"], None, padding=1)
    x = res_block(sd, "mid_block1.", x, t)
    x = attn_block(sd, "mid_attn.", x, ctx)
    x = res_block(sd, "mid_block2.", x, t)
    if taps is not None:
        taps["mid"] = x
    for j in range(depth):
        i = depth - 1 - j
        p = f"ups.{j}."
        x = res_block(sd, p + "0.", torch.cat([x, hs.pop()], dim=1), t)
        x = res_block(sd, p + "1.", torch.cat([x, hs.pop()], dim=1), t)
        x = attn_block(sd, p + "2.", x, ctx)
        if taps is not None:
            taps[f"up{j}"] = x
        if i != 0:
            x = F.interpolate(x, scale_factor=2, mode="nearest")
            x = F.conv2d(x, sd[p + "3.1.weight"], sd[p + "3.1.bias"], padding=1)
        else:
            x = F.conv2d(x, sd[p + "3.weight"], None, padding=1)
    x = res_block(sd, "final_res_block.", torch.cat([x, x_], dim=1), t)
    x = F.conv2d(x, sd["final_conv.weight"], sd["final_conv.bias"], padding=1)
    return x[..., :H, :W].contiguous()
