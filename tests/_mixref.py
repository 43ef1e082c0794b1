"""The token mixers by their definitions, in 64 bits (numpy / torch on the CPU)."""
import math

import numpy as np
import torch


def theta(rot, base, scaling="none", factor=1.0, orig_len=0.0, beta_fast=32.0, beta_slow=1.0, freq_factors=None):
    """Angle per position of each pair."""
    out = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "by_parts":
            turns = orig_len * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - beta_slow) / (beta_fast - beta_slow)))
            f *= keep + (1 - keep) / factor
        if freq_factors is not None:
            f /= float(freq_factors[i])
        out.append(f)
    return np.array(out)


def rotate(x, pos, th, interleaved, mscale=1.0):
    """x [n, heads, d] float64 turned to pos [n]."""
    r = 2 * len(th)
    a = np.asarray(pos, dtype=np.float64)[:, None, None] * th
    c, s = np.cos(a) * mscale, np.sin(a) * mscale
    y = np.array(x, dtype=np.float64)
    i0, i1 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


def pair_size(x, rot, interleaved, mscale=1.0):
    """|a| + |b| of the pair that each value belongs to (|x| past rot)."""
    y = np.abs(np.asarray(x, dtype=np.float64))
    i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    t = (y[..., i0] + y[..., i1]) * mscale
    y[..., i0], y[..., i1] = t, t
    return y


def attention(q, k, v, pk, pv, lens, scale, mask=None):
    """q [s, m, hq, d]; k, v [s, cap, hkv, d]; pk, pv [p, hkv, d]; mask [s, m] of ints or None. Returns the output and,
    per value, (sum_j p_j |v_j|, the largest sum_d |q_d k_jd| scale of the row's keys, keys seen): what the
    tolerances are made of. Entries that a row does not see are never touched."""
    s, m, hq, d = q.shape
    hkv = k.shape[2]
    out, size = np.zeros((s, m, hq, d)), np.zeros((s, m, hq, d))
    reach, seen = np.zeros((s, m, hq, 1)), np.zeros((s, m, hq, 1))
    for i in range(s):
        if lens[i] < 0:
            continue
        for r in range(m):
            bits = (1 << (r + 1)) - 1 if mask is None else int(mask[i][r]) & ((1 << 64) - 1)
            new = [lens[i] + j for j in range(m) if bits >> j & 1]
            at = list(range(lens[i])) + new
            for h in range(hq):
                g = h // (hq // hkv)
                kk = np.concatenate([pk[:, g], k[i, at, g]]).astype(np.float64)
                vv = np.concatenate([pv[:, g], v[i, at, g]]).astype(np.float64)
                if not len(kk):
                    continue
                z = kk @ q[i, r, h].astype(np.float64) * scale
                with np.errstate(invalid="ignore"):
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    out[i, r, h] = p @ vv
                    size[i, r, h] = p @ np.abs(vv)
                    reach[i, r, h] = (np.abs(kk) @ np.abs(q[i, r, h].astype(np.float64))).max() * abs(scale)
                seen[i, r, h] = len(kk)
    return out, size, reach, seen


def attention_bound(d, size, reach, seen):
    """How far fp32 arithmetic may be off, entry by entry. A score's sum of d products (each of two or three limb
    products) is off by (2 d + 8) 2^-24 of sum |q k| at most, its argument of exp by one more rounding of its size; p is
    off by twice that in the worst case (its own and the sum's), by exp's 4 units and the limbs' 2^-20; sums over the
    keys add one rounding a key and partial sums their few. All relative to sum_j p_j |v_j|."""
    return size * (2 * ((2 * d + 16) * 2.0 ** -24 * reach) + (seen + 64) * 2.0 ** -24 + 2.0 ** -20)


def delta(q, k, v, g, beta, state, lens=None, l2norm=False, scale=None):
    """Token by token in float64. q, k [s, t, hk, dk], v [s, t, hv, dv]; returns o, the states after each token
    [s, t, hv, dk, dv] and the last state."""
    q, k, v, g, beta = (torch.as_tensor(x).double().cpu() for x in (q, k, v, g, beta))
    s, t, hk, dk = k.shape
    hv, dv = v.shape[2], v.shape[3]
    if l2norm:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q = q * (dk ** -0.5 if scale is None else scale)
    q, k = (x.repeat_interleave(hv // hk, 2) for x in (q, k))
    cur = torch.zeros(s, hv, dk, dv, dtype=torch.float64) if state is None else torch.as_tensor(state).double().cpu()
    o, kept = torch.zeros(s, t, hv, dv, dtype=torch.float64), torch.zeros(s, t, hv, dk, dv, dtype=torch.float64)
    for i in range(t):
        on = torch.ones(s, dtype=torch.bool) if lens is None else torch.as_tensor([i < n for n in lens])
        new = cur * torch.exp(g[:, i])[..., None, None]
        miss = v[:, i] - (new * k[:, i, :, :, None]).sum(-2)
        new = new + k[:, i, :, :, None] * (beta[:, i, :, None] * miss)[:, :, None, :]
        o[:, i] = (new * q[:, i, :, :, None]).sum(-2)
        cur = torch.where(on[:, None, None, None], new, cur)
        kept[:, i] = cur
    return o, kept, cur
