"""Group norm and grid attention from their definitions, in float64 torch (CPU or GPU).  Test infrastructure only: what the tests hold
rgbd_gan_amd.functional.group_norm / attention against.  Differentiable by autograd; `attention_parts` also returns the matrices whose
sums bound what the kernels' roundings can do (tests derive their tolerances from them)."""
import math

import torch


def group_norm(x, gamma, beta, groups, eps=1e-5, act=None, slope=0.2):
    """x (B, ..., C): statistics of each sample over its pixels and C / groups neighbouring channels."""
    shape, C = x.shape, x.shape[-1]
    v = x.reshape(shape[0], -1, groups, C // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    z = ((v - mean) / torch.sqrt(var + eps)).reshape(shape) * gamma + beta
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "lrelu":
        return torch.where(z > 0, z, slope * z)
    return z


def offsets(rows, cols, q_start, lq, lk, device="cpu"):
    """(lq, lk) places in the flattened (2 rows - 1, 2 cols - 1) bucket map."""
    i = torch.arange(q_start, q_start + lq, device=device)[:, None]
    j = torch.arange(lk, device=device)[None, :]
    return (i // cols - j // cols + rows - 1) * (2 * cols - 1) + (i % cols - j % cols + cols - 1)


def attention_parts(q, k, v, table=None, bucket_map=None, scale=None, cap=0.0, lengths=None, q_start=0):
    """q (B,Lq,H,D), k, v (B,Lk,Hkv,D) float64; bucket_map (2 rows - 1, 2 cols - 1) int64 -> o (B,Lq,H,D), p (B,H,Lq,Lk),
    t = tanh of the scaled scores (or None), place (Lq,Lk) bucket of every pair (or None), kr, vr: k, v per query head."""
    B, Lq, H, D = q.shape
    Lk, rep = k.shape[1], H // k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    qh = q.permute(0, 2, 1, 3)
    kr, vr = (t.permute(0, 2, 1, 3).repeat_interleave(rep, dim=1) for t in (k, v))
    s = scale * torch.matmul(qh, kr.transpose(-1, -2).contiguous())
    t = place = None
    if cap:
        t = torch.tanh(s / cap)
        s = cap * t
    if table is not None:
        rows, cols = (bucket_map.shape[0] + 1) // 2, (bucket_map.shape[1] + 1) // 2
        place = bucket_map.reshape(-1)[offsets(rows, cols, q_start, Lq, Lk, q.device)]
        s = s + table[:, place]
    if lengths is not None:
        keep = torch.arange(Lk, device=q.device) < lengths.reshape(B, 1, 1, 1)
        s = torch.where(keep, s, torch.full_like(s, -math.inf))
    m = s.detach().amax(dim=-1, keepdim=True) if Lk else s.new_zeros(B, H, Lq, 1)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    z = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(z > 0, z, torch.ones_like(z))
    o = torch.matmul(p, vr).permute(0, 2, 1, 3)
    return o, p, t, place, kr, vr


def attention(*args, **kw):
    return attention_parts(*args, **kw)[0]
