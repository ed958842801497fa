"""The decoder-block operators from their definitions in binary64, with the bound that fp32 arithmetic may be off by."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
U = 2.0 ** -24  # half a step of fp32


def half_step(type):
    return torch.finfo(TYPES[type]).eps / 2


def rounding(x, type):
    """How far rounding x to the type may move it: half a step, and half of the smallest step below the normal range."""
    f = torch.finfo(TYPES[type])
    return half_step(type) * x.abs() + f.tiny * f.eps / 2


def attention(q, k, v, q_start, k_start, k_len, scale, causal, type):
    """(out, lse, tolerance of out, tolerance of lse); rows outside the sequences: NaN."""
    total, heads, dim = q.shape
    group = heads // k.shape[1]
    dev = q.device
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=dev)
    lse = torch.full((total, heads), math.nan, dtype=torch.float64, device=dev)
    tol, tol_lse = out.clone(), lse.clone()
    for i in range(len(k_len)):
        a, b, n = q_start[i], q_start[i + 1], k_len[i]
        if a == b:
            continue
        kk, vv = (z[k_start[i]:k_start[i] + n].double().repeat_interleave(group, 1) for z in (k, v))
        qq = q[a:b].double()
        s = torch.einsum("thd,jhd->htj", qq, kk) * scale
        size = torch.einsum("thd,jhd->htj", qq.abs(), kk.abs()) * abs(scale)
        if causal:
            see = torch.arange(n, device=dev)[None] <= torch.arange(b - a, device=dev)[:, None] + (n - (b - a))
            s = s.masked_fill(~see, -math.inf)
            size = size.masked_fill(~see, 0)
        m = s.amax(2, keepdim=True) if n else torch.full((heads, b - a, 1), -math.inf, dtype=torch.float64, device=dev)
        m0 = torch.where(m == -math.inf, 0.0, m)
        e = torch.exp(s - m0)
        l = e.sum(2, keepdim=True)
        p = e / torch.where(l > 0, l, 1.0)
        o = torch.einsum("htj,jhd->thd", p, vv)
        spread = torch.einsum("htj,jhd->thd", p, vv.abs())
        # a score: dim products added in fp32, the scale, the difference to the maximum in units of log 2, the power's
        # 2 ulp; an fp32 sum of n weights; weights kept in the type (below its normal range: half its smallest step,
        # against a largest weight of at least 1)
        big = size.amax(2) if n else torch.zeros(heads, b - a, dtype=torch.float64, device=dev)
        off = (dim + 4) * U * big + 4 * U * 1.45 * m0[..., 0].abs() + 4 * U
        off = off + n * U
        f = torch.finfo(TYPES[type])
        vmax = vv.abs().amax() if n else 0.0
        out[a:b], lse[a:b] = o, (m0 + l.log())[..., 0].t()
        tol[a:b] = (half_step(type) + 2 * off.t()[..., None]) * spread + rounding(o, type) + n * f.tiny * f.eps / 2 * vmax
        tol_lse[a:b] = off.t() + 4 * U * lse[a:b].nan_to_num(0, 0, 0).abs()
    return out, lse, tol, tol_lse


def _norm(v, gamma, beta, layer, eps, off):
    """(normalised v, its bound) where v is off by `off`.  Sums run over at most 48 additions deep."""
    cols = v.shape[1]
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    d = v - mean
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + eps)
    depth = (cols / 256 + 64) * U
    off_d = off + (off.mean(1, keepdim=True) + depth * v.abs().mean(1, keepdim=True) if layer else 0) + U * (v.abs() + mean.abs())
    off_r = r * r * (d.abs() * off_d).mean(1, keepdim=True) + depth + 4 * U  # relative
    z = d * r
    tol = off_d * r + z.abs() * (off_r + 2 * U)
    g = gamma.double() if gamma is not None else torch.ones(cols, dtype=torch.float64, device=v.device)
    b = beta.double() if beta is not None else torch.zeros(cols, dtype=torch.float64, device=v.device)
    return z * g + b, tol * g.abs() + 2 * U * ((z * g).abs() + b.abs())


def norm(a, x, gate, gate_rows, scale, post, post_gamma, post_beta, pre_gamma, pre_beta, layer, eps, x_type, h_type):
    """(y, h, tolerance of y, tolerance of h)."""
    z = a.double()
    off = torch.zeros_like(z)
    if post:
        z, off = _norm(z, post_gamma, post_beta, layer, eps, off)
    if gate is not None:
        g = gate.double()[torch.arange(a.shape[0], device=a.device) // gate_rows]
        z, off = z * g, off * g.abs() + U * (z * g).abs()
    z, off = z * scale, off * abs(scale) + U * (z * scale).abs()
    y = z if x is None else z + x.double()
    off = off + 2 * U * (y.abs() + z.abs())
    h, off_h = _norm(y, pre_gamma, pre_beta, layer, eps, off)
    return y, h, off + rounding(y, x_type), off_h + rounding(h, h_type)


def rope(x, bias, pos, turns, rot, interleaved, magnitude, heads, kv_heads, dim, type):
    """(all heads [tokens][heads + 2 kv_heads][dim], their tolerance)."""
    x = x.double()
    off = torch.zeros_like(x)
    if bias is not None:
        x = x + bias.double()
        off = U * x.abs()
    x = x.view(x.shape[0], heads + 2 * kv_heads, dim).clone()
    off = off.view_as(x).clone()
    if rot:
        a = pos.double()[:, None] * turns[None]
        a = 2 * math.pi * (a - torch.round(a))
        c, s = (f(a)[:, None, :] * magnitude for f in (torch.cos, torch.sin))
        i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        qk, o = x[:, :heads + kv_heads], off[:, :heads + kv_heads]
        u, w, ou, ow = qk[..., i].clone(), qk[..., j].clone(), o[..., i].clone(), o[..., j].clone()
        qk[..., i], qk[..., j] = u * c - w * s, w * c + u * s
        # cos and sin: half a step of the fraction of a turn (times 2 pi), 2 ulp of the functions, the magnitude's product;
        # then two products and a sum
        e = magnitude * (2 * math.pi * U / 2 + 8 * U) * (u.abs() + w.abs()) + (ou + ow) * magnitude
        o[..., i], o[..., j] = e, e
    return x, off + rounding(x, type)


def quantize(x):
    """(codes, scales): the scale is fp32 by definition, the codes exact."""
    s = (x.double().abs().amax(1) / 127).float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    q = torch.round(x.double() / torch.where(s > 0, s, torch.ones_like(s)).double()[:, None])
    return torch.where(s[:, None] > 0, q, torch.zeros_like(q)), s


def i8gemm(a, sa, b, sb, bias, type):
    """(out, tolerance): exact sums, then four fp32 roundings and the type's."""
    v = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None]
    o = v if bias is None else v + bias.double()
    return o, 3.1 * U * v.abs() + 1.1 * U * o.abs() + rounding(o, type)
