"""Plain 64-bit forms of the chunk attention, the key weights and the evictions (CPU), and how far a kernel may be from them."""

import math

import torch

D, GROUP = 128, 32


def unpack64(pack, bits=4):
    """float64 scale * code + minimum of a packed operand (last dimension unpacked)."""
    code, scale, mn = (t.cpu() for t in pack)
    per = 32 // bits
    w = code.to(torch.int64) & 0xFFFFFFFF
    c = torch.stack([(w >> (bits * i)) & (2 ** bits - 1) for i in range(per)], -1).flatten(-2).double()
    return c * scale.double().repeat_interleave(GROUP, -1) + mn.double().repeat_interleave(GROUP, -1)


def scores64(q, k_pack, k_fp, t_sys, mask=None, live=None):
    """(scores [B,Hq,L,keys] in cache order [visual | fp] with -inf where a key takes no part, bound on the error of each)."""
    q, k_fp = q.cpu().double(), k_fp.cpu().double()
    B, L, Hq, _ = q.shape
    Hkv, cap = k_fp.shape[1], k_fp.shape[2]
    live = cap if live is None else live
    k = k_fp
    size = k_fp.abs()                    # |terms| of each key's elements: a packed one is code * scale + minimum
    t_vis = 0
    if k_pack is not None and k_pack[0].numel():
        vis = unpack64(k_pack).transpose(2, 3)
        t_vis = vis.shape[2]
        mn = k_pack[2].cpu().double().abs().repeat_interleave(GROUP, -1).transpose(2, 3)
        k, size = torch.cat([vis, k], 2), torch.cat([vis.abs() + 2 * mn, size], 2)
    rep = Hq // Hkv
    k, size = k.repeat_interleave(rep, 1), size.repeat_interleave(rep, 1)
    qh = q.transpose(1, 2)
    dead = torch.arange(t_vis + cap) >= t_vis + live
    k, size = k.masked_fill(dead[:, None], 0.0), size.masked_fill(dead[:, None], 0.0)
    hidden = torch.zeros(B, 1, L, t_vis + cap, dtype=torch.bool)
    last = live - L + torch.arange(L)
    hidden[..., t_vis:] = torch.arange(cap) > last[:, None]
    add = torch.zeros(B, 1, 1, t_vis + cap, dtype=torch.float64)
    if mask is not None:
        m = mask.cpu().double().reshape(B, -1)
        m = torch.cat([m[:, t_sys:t_sys + t_vis], m[:, :t_sys], m[:, t_sys + t_vis:]], 1)
        gone = torch.isneginf(m)
        k, size = k.masked_fill(gone[:, None, :, None], 0.0), size.masked_fill(gone[:, None, :, None], 0.0)
        hidden = hidden | gone[:, None, None]
        add = m.masked_fill(gone, 0.0)[:, None, None]
    s = qh @ k.transpose(2, 3) / math.sqrt(D)
    # 256 products in fp32: the tensor core cuts a sum off at 2^-22 of its largest term at each of 16 steps, 2^-18 in all; then
    # the mask is added and the scale applied, 2^-23 of the result each
    err = 2.0 ** -18 * (qh.abs() @ size.transpose(2, 3)) / math.sqrt(D) + 2.0 ** -22 * (s + add).abs()
    return (s + add).masked_fill(hidden, -math.inf), err.masked_fill(hidden, 0.0)


def attention64(q, k_pack, v_pack, k_fp, v_fp, t_sys, mask=None, live=None):
    """(out [B,L,Hq,D], lse [B,Hq,L], bound of out, bound of lse)."""
    dt = q.dtype
    s, err = scores64(q, k_pack, k_fp, t_sys, mask, live)
    rep = q.shape[2] // k_fp.shape[1]
    v = v_fp.cpu().double()
    if v_pack is not None and v_pack[0].numel():
        v = torch.cat([unpack64(v_pack), v], 2)
    t_vis = v.shape[2] - v_fp.shape[2]
    seen_by_any = torch.isfinite(s).any(2)                                             # [B,Hq,keys]
    v = v.repeat_interleave(rep, 1).masked_fill(~seen_by_any[..., None], 0.0)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(torch.isneginf(lse), 0.0)[..., None])
    out = (p @ v).transpose(1, 2)
    # Half a step each for the result, the probabilities and the unpacked values; and a probability is off by the error of its score
    # (e^x - 1) and by that of their sum
    u = torch.finfo(dt).eps / 2
    each = torch.expm1(err.clamp(max=50.0))
    total = (p * each).sum(-1, keepdim=True)
    room = ((p * (2 * u + 2 * each + 2 * total + 2.0 ** -16)) @ v.abs()).transpose(1, 2) + u * out.abs() + torch.finfo(dt).tiny
    return out, lse, room * 1.01, 2 * total.squeeze(-1) + 2.0 ** -20 * (1 + lse.abs().nan_to_num(0, 0, 0))


def weights64(q, lse, k_pack, k_fp, t_sys, mask=None, live=None):
    """((w_vis, w_fp) of one call [B,Hkv,..], bounds of both)."""
    s, err = scores64(q, k_pack, k_fp, t_sys, mask, live)
    Hkv, rep = k_fp.shape[1], q.shape[2] // k_fp.shape[1]
    lse = lse.cpu().double()
    p = torch.exp(s - lse.masked_fill(torch.isneginf(lse), 0.0)[..., None])
    p = p.masked_fill(torch.isneginf(lse)[..., None], 0.0)
    n = p.shape[2] * rep
    # exp of an argument that is off by the score's error and by 2^-22 of its size; n terms summed in fp32
    room = p * (2 * err + 2.0 ** -20 * (1 + s.abs().nan_to_num(0, 0, 0)) + n * 2.0 ** -23)
    both = [t.unflatten(1, (Hkv, rep)).sum((2, 3)) for t in (p, room)]
    t_vis = s.shape[-1] - k_fp.shape[2]
    return tuple((t[..., :t_vis], t[..., t_vis:]) for t in both)


def kept_largest(rank, keep):
    """Indices of the keep largest numbers of each row (ties to the lowest index, NaN the largest), ascending; plain Python."""
    rows = rank.double().flatten(0, 1).tolist()
    out = []
    for row in rows:
        order = sorted(range(len(row)), key=lambda i: (0 if math.isnan(row[i]) else 1, 0 if math.isnan(row[i]) else -row[i], i))
        out.append(sorted(order[:keep]))
    return torch.tensor(out).view(*rank.shape[:2], keep)


def within(got, want, room):
    """Whether every number of ``got`` is within ``room`` of ``want`` (equal where that is not finite)."""
    got, bad = got.cpu().double(), ~torch.isfinite(want)
    same = torch.equal(got[bad], want[bad])
    off = ((got - want).abs() - room).masked_fill(bad, -1.0)
    return same and bool(torch.isfinite(got[~bad]).all()) and float(off.max() if off.numel() else 0.0) <= 0.0
