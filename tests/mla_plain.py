"""Plain 64-bit restatements of the 4-bit latent cache and of latent attention,
for the tests of pbmoe_mla_q4_* and pbmoe_mla_prefill, with bounds derived
from the kernels' roundings (half a step: fp16 2^-11, bf16 2^-8 relative)."""

import math

import torch

NOPE, ROPE, LAT, V = 128, 64, 512, 128
F16, BF16, F32 = 2.0**-11, 2.0**-8, 2.0**-24


def quantise(x):
    """f32 rows [n, 512] -> (stored nibbles int64 [n, 512], scales bf16 [n, 8]); f32 arithmetic as the format says."""
    n = x.shape[0]
    g = x.float().reshape(n, 8, 64)
    s = (g.abs().amax(-1) / 7).to(torch.bfloat16)
    sf = s.float().unsqueeze(-1)
    q = torch.where(sf > 0, torch.round(g / sf), torch.zeros_like(g)).clamp(-7, 7)
    return (q + 8).long().reshape(n, LAT), s


def pack(u):
    return (u[:, 0::2] | (u[:, 1::2] << 4)).to(torch.uint8)


def unpack(codes):
    c = codes.long()
    return torch.stack((c & 15, c >> 4), -1).reshape(codes.shape[0], LAT)


def values(codes, scales):
    """f64 latent rows that codes and scales stand for."""
    q = (unpack(codes) - 8).double().reshape(-1, 8, 64)
    return (q * scales.double().unsqueeze(-1)).reshape(-1, LAT)


def rope(x, pos, theta=10000.0):
    """f32 rotation (unfused) of [..., 64] at positions [n], with the cos/sin table rounded from f64."""
    a = pos.double().unsqueeze(-1) * theta ** (-torch.arange(0, ROPE, 2, device=pos.device).double() / ROPE)
    c, s = a.cos().float(), a.sin().float()
    while c.dim() < x.dim():
        c, s = c.unsqueeze(1), s.unsqueeze(1)
    x0, x1 = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.cat((x0 * c - x1 * s, x1 * c + x0 * s), -1)


def normed(lat, w, eps):
    """f32 RMSNorm rows with the mean square in f64."""
    scale = (1 / torch.sqrt(lat.double().square().mean(-1, keepdim=True) + eps)).float()
    return lat.float() * scale * w


def attend(q, lat, kr, wuk, wuv, first=None, scale=0.0):
    """f64 latent attention of q [t, h, 192] over rows lat [n, 512], kr [n, 64]; token i sees rows 0 .. first + i
    (first None: all). Returns (out [t, h, 128], A, F, delta): A = sum_t p_t sum_c |W_UV| |c_t|, F the same with every
    p_t = 1, and delta the largest error of a score when its products are rounded once to fp16."""
    q, lat, kr, wuk, wuv = (x.double() for x in (q, lat, kr, wuk, wuv))
    scale = scale or 1 / math.sqrt(NOPE + ROPE)
    t, h, n = q.shape[0], q.shape[1], lat.shape[0]
    out = torch.empty(t, h, V, dtype=torch.float64, device=q.device)
    mag, flat = torch.empty_like(out), torch.empty_like(out)
    delta = torch.zeros(h, dtype=torch.float64, device=q.device)
    hide = None
    if first is not None:
        hide = torch.arange(n, device=q.device) > first + torch.arange(t, device=q.device).unsqueeze(1)
    for i in range(h):
        ql = q[:, i, :wuk.shape[1]] @ wuk[i]
        qr = q[:, i, wuk.shape[1]:]
        s = (ql @ lat.T + qr @ kr.T) * scale
        err = (ql.abs() @ lat.abs().T * F16 + qr.abs() @ kr.abs().T * F16) * scale
        if hide is not None:
            s = s.masked_fill(hide, -math.inf)
            err = err.masked_fill(hide, 0)
        p = torch.softmax(s, -1)
        delta[i] = err.max()
        out[:, i] = (p @ lat) @ wuv[i].T
        mag[:, i] = (p @ lat.abs()) @ wuv[i].abs().T
        flat[:, i] = lat.abs().sum(0) @ wuv[i].abs().T
    return out, mag, flat, delta


def attend_expanded(q, lat, kr, wuk, wuv, first, scale=0.0):
    """f64 latent attention, one head at a time over K = c W_UK^T, V = c W_UV^T: token i of q [t, h, 192] sees rows
    0 .. first + i. Returns (out, bound): the bound of |kernel - out| when queries, K, key parts, V and p are each
    rounded once to fp16 (2^-11 relative, 2^-25 below its normal range) and sums are f32 (2^-16 of their terms covers
    the longest): scores off by delta, so p by e^(2 delta) - 1."""
    q, lat, kr, wuk, wuv = (x.double() for x in (q, lat, kr, wuk, wuv))
    scale = scale or 1 / math.sqrt(NOPE + ROPE)
    t, h, n = q.shape[0], q.shape[1], lat.shape[0]
    out = torch.empty(t, h, V, dtype=torch.float64, device=q.device)
    bound = torch.empty_like(out)
    hide = torch.arange(n, device=q.device) > first + torch.arange(t, device=q.device).unsqueeze(1)
    for i in range(h):
        k, v = torch.cat((lat @ wuk[i].T, kr), 1), lat @ wuv[i].T
        s = (q[:, i] @ k.T * scale).masked_fill(hide, -math.inf)
        mag = q[:, i].abs() @ k.abs().T
        err = (mag * (2 * F16 + 2.0**-16) + 2.0**-25 * (q[:, i].abs().sum(1, keepdim=True) + k.abs().sum(1))) * scale
        delta = err.masked_fill(hide, 0).amax(1, keepdim=True)
        p = torch.softmax(s, -1)
        out[:, i] = p @ v
        bound[:, i] = (torch.expm1(2 * delta) + 2 * F16 + 2.0**-16) * (p @ v.abs()) + 2.0**-24
    return out, bound


def attend_plain(q, lat, kr, wuk, wuv):
    """f64 latent attention of one token's q [h, 192] over all rows lat [n, 512], kr [n, 64]: out [h, 128]."""
    q, lat, kr, wuk, wuv = (x.double() for x in (q, lat, kr, wuk, wuv))
    ql = torch.einsum("hd,hdc->hc", q[:, :wuk.shape[1]], wuk)
    s = (ql @ lat.T + q[:, wuk.shape[1]:] @ kr.T) / math.sqrt(q.shape[1])
    return torch.einsum("hc,hdc->hd", torch.softmax(s, -1) @ lat, wuv)


def rms(got, want):
    """Norm of the error over the norm of what is wanted."""
    return float((got.double() - want).norm() / want.norm())


def rms_limit(q_scale, bf16_out=False):
    """What random roundings of the 4-bit decode add up to, as a share of an output's norm: a weight's two to fp16 and
    its score's 2^-11 / sqrt(3) of the latent part's deviation (0.37 q_scale for N(0, 1) rows, N(0, 0.02) weights) are
    4e-4 + 1.1e-4 q_scale; a bf16 output adds up to 2^-8 / sqrt(3)."""
    return 1e-3 + F16 * q_scale + (3e-3 if bf16_out else 0.0)
