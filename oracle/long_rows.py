"""64-bit restatement of the long-row operators (attention with score modifications, norm + rotation) on the CPU, with the bound on
what rounding may do to every element of every result.

The bounds follow the operators' arithmetic: inputs are exact, products and sums are fp32 (unit roundoff 2^-24), probabilities and
score gradients are rounded to the element type (unit roundoff u) before they enter a second product, results are rounded once.
With A >= the sum of the absolute terms, a sum of n terms in fp32 is off by at most n 2^-24 A.
"""
import math

import torch

F32 = 2.0 ** -24


def unit(dtype):
    """Half a step of the type, relative to the value."""
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half of the smallest step (subnormal numbers)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def attention(q, k, v, scale=None, causal=False, prefix=None, q_doc=None, k_doc=None, kv_len=None, softcap=0.0, slopes=None,
              rel_bias=None, rel_buckets=None, dout=None, dlse=None, dtype=torch.float32):
    """Results and bounds as dictionaries: out, lse and, with ``dout`` (and / or ``dlse``), dq, dk, dv, dbias.  ``dtype`` is the type
    the operator under test computes in."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, Lq, H, dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = dh ** -0.5 if scale is None else scale
    u, up, fl = unit(dtype), 0.0 if dtype == torch.float32 else unit(dtype), floor_of(dtype)
    n32 = (max(Lk, Lq) + dh + 16) * F32
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)
    val = {"out": zeros(B, Lq, H, dh), "lse": torch.full((B, H, Lq), -math.inf, dtype=torch.float64)}
    tol = {"out": zeros(B, Lq, H, dh), "lse": zeros(B, H, Lq)}
    back = dout is not None or dlse is not None
    if back:
        do = dout.detach().cpu().double() if dout is not None else torch.zeros_like(q)
        dl = dlse.detach().cpu().double() if dlse is not None else zeros(B, H, Lq)
        for d in (val, tol):
            d["dq"], d["dk"], d["dv"] = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
            if rel_bias is not None:
                d["dbias"] = zeros(*rel_bias.shape)
    cpu = lambda t: None if t is None else t.detach().cpu()
    prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets = map(cpu, (prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets))
    j = torch.arange(Lk)
    if back and dtype == torch.float16:
        # What bounds the score gradients of the whole call: the largest |dout|, |v| and |dlse| of live rows and keys.  They are scaled by the
        # power of two that takes 2 max|dout| max|v| + max|dlse| into (2^14, 2^15]; the smallest step is then 2^-24.
        lens = torch.full((B, 1), Lk) if kv_len is None else kv_len.long().clamp(0, Lk)[:, None]
        live_q = torch.ones(B, Lq, dtype=torch.bool) if q_doc is None else q_doc >= 0
        live_k = (j[None] < lens) & (True if k_doc is None else k_doc >= 0)
        most = lambda rows, live: float(torch.where(live & torch.isfinite(rows), rows, torch.zeros((), dtype=torch.float64)).max()) if rows.numel() else 0.0
        glob = 2 * most(do.norm(dim=-1), live_q[..., None]) * most(v.norm(dim=-1), live_k[..., None]) + most(dl.abs(), live_q[:, None])
    for b in range(B):
        n = Lk if kv_len is None else max(0, min(int(kv_len[b]), Lk))
        p = n - Lq + torch.arange(Lq)
        see = (j < n)[None].expand(Lq, Lk)
        if causal:
            see = see & ((j[None] <= p[:, None]) | (j < (0 if prefix is None else int(prefix[b])))[None])
        dead_q, dead_k = torch.zeros(Lq, dtype=torch.bool), j >= n
        if q_doc is not None:
            see = see & (q_doc[b][:, None] == k_doc[b][None]) & (q_doc[b] >= 0)[:, None] & (k_doc[b] >= 0)[None]
            dead_q, dead_k = q_doc[b] < 0, dead_k | (k_doc[b] < 0)
        apart = j[None] - p[:, None]
        if rel_bias is not None:
            reach = rel_buckets.numel() // 2
            bucket = rel_buckets.long()[apart.clamp(-reach, reach) + reach].clamp(0, rel_bias.shape[1] - 1)
        for h in range(H):
            g = h // G
            clean = lambda t, dead: torch.where(dead[:, None], torch.zeros((), dtype=torch.float64), t)   # what is hidden may be NaN
            Q, K, V = clean(q[b, :, h], dead_q), clean(k[b, :, g], dead_k), clean(v[b, :, g], dead_k)
            raw = scale * (Q @ K.t())
            e = (dh + 4) * F32 * scale * (Q.abs() @ K.abs().t())             # bound on the error of the score
            x = raw
            if softcap:
                t = torch.tanh(raw / softcap)
                x = softcap * t
                e = e + 8 * F32 * x.abs() + 4 * F32 * softcap * t.abs()
            if slopes is not None:
                x = x - float(slopes[h]) * apart.abs().double()
                e = e + 4 * F32 * float(slopes[h]) * apart.abs().double()
            if rel_bias is not None:
                entry = rel_bias[h].double()             # clamped to +-2^14; at or below -2^100: a mask
                entry = torch.where(entry <= -2.0 ** 100, -math.inf, entry.clamp(-2.0 ** 14, 2.0 ** 14))
                x = x + entry[bucket]
                e = e + 4 * F32 * entry.abs()[bucket].clamp_max(2.0 ** 14)
            x = x.masked_fill(~see, -math.inf)
            lse = torch.logsumexp(x, -1) if Lk else torch.full((Lq,), -math.inf, dtype=torch.float64)
            some = lse > -math.inf
            P = torch.where(some[:, None], torch.exp(x - lse[:, None].masked_fill(~some[:, None], 0.0)), torch.zeros((), dtype=torch.float64))
            fin = torch.where(see & (x > -math.inf), x.abs(), torch.zeros((), dtype=torch.float64))
            # log2 e once more on score, maximum and log-sum, the exponential itself 2^-21
            err = torch.where(P > 0, e + 8 * F32 * fin, torch.zeros((), dtype=torch.float64))
            worst = err.amax(-1, keepdim=True) if Lk else zeros(Lq, 1)
            ep = err + worst + 2.0 ** -20 + 4 * F32 * lse.abs().masked_fill(~some, 0.0)[:, None]
            val["lse"][b, h] = lse
            tol["lse"][b, h] = worst[:, 0] + 2.0 ** -20 + (Lk + 16) * F32 + 4 * F32 * lse.abs().masked_fill(~some, 0.0)
            O = P @ V
            eO = (P * (ep + up + n32)) @ V.abs()
            val["out"][b, :, h] = O
            tol["out"][b, :, h] = eO + u * (O.abs() + eO) + fl
            if not back:
                continue
            D = clean(do[b, :, h], dead_q)
            dl_row = dl[b, h].masked_fill(dead_q, 0.0)
            dP = D @ V.t()
            delta = (D * O).sum(-1, keepdim=True) - dl_row[:, None]
            dU = P * (dP - delta)
            e_dp = (dh + 4) * F32 * (D.abs() @ V.abs().t())
            e_delta = (D.abs() * (tol["out"][b, :, h] + (dh + 4) * F32 * O.abs())).sum(-1, keepdim=True) + 2 * F32 * dl_row.abs()[:, None]
            eU = ep * dU.abs() + P * (e_dp + e_delta) + 4 * F32 * P * (dP.abs() + delta.abs())
            dS, eS = dU, eU
            if softcap:
                slope = 1 - t * t
                dS = dU * slope
                eS = eU * slope + dU.abs() * (2 * t.abs() * e / softcap + 8 * F32)
            e_in = eS + up * (dS.abs() + eS)
            if dtype == torch.float16:
                e_in = e_in + torch.where(P > 0, 2.0 ** -38 * glob, 0.0)
            val["dq"][b, :, h] = scale * (dS @ K)
            w = scale * (e_in + n32 * dS.abs())
            tol["dq"][b, :, h] = w @ K.abs()
            val["dk"][b, :, g] += scale * (dS.t() @ Q)
            tol["dk"][b, :, g] += w.t() @ Q.abs()
            val["dv"][b, :, g] += P.t() @ D
            tol["dv"][b, :, g] += (P * (ep + up + n32)).t() @ D.abs()
            if rel_bias is not None:
                # fp32 all the way: the correction of delta leaves the error of the products
                e_fix = e_dp + (P * (e_dp + (ep + 8 * F32) * (dP - delta).abs())).sum(-1, keepdim=True) + 8 * F32 * (dP.abs() + delta.abs())
                eT = ep * dU.abs() + P * e_fix + (Lk + Lq) * F32 * dU.abs()
                eT = torch.where(P > 0, eT, torch.zeros((), dtype=torch.float64))
                val["dbias"][h] += torch.bincount(bucket.flatten(), dU.flatten(), minlength=rel_bias.shape[1])
                tol["dbias"][h] += torch.bincount(bucket.flatten(), eT.flatten(), minlength=rel_bias.shape[1])
    if back:
        for name in ("dq", "dk", "dv"):
            tol[name] = tol[name] + u * (val[name].abs() + tol[name]) + fl
        if rel_bias is not None:
            tol["dbias"] = tol["dbias"] + F32 * val["dbias"].abs()
    for name in val:
        assert not (torch.isfinite(val[name]) & ~torch.isfinite(tol[name])).any(), f"the bound on {name} would pass anything"
    return val, tol


def norm_rope(x, weight, inv_freq, positions, eps, interleaved, gy=None):
    """One tensor (B,L,H,dh): y, dx, dw and their bounds."""
    dtype, w_dtype = x.dtype, weight.dtype
    x, w, f = x.detach().cpu().double(), weight.detach().cpu().double(), inv_freq.detach().cpu().double()
    B, L, H, dh = x.shape
    pos = torch.arange(L).expand(B, L) if positions is None else positions.cpu()
    ang = (pos.double()[..., None] * f)[:, :, None]
    half = f.numel()
    m = torch.arange(half)
    ia, ib = (2 * m, 2 * m + 1) if interleaved else (m, m + half)
    c, s = ang.cos(), ang.sin()
    u, fl = unit(dtype), floor_of(dtype)
    e_ang = 8 * F32 + 4e-16 * ang.abs()            # cosine and sine: fp32 of an angle reduced in 64 bits
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    hat = x * r
    n = hat * w
    e_n = (dh + 8) * F32 * n.abs()

    def turn(z, e, sign):
        z, e, y, ey = z, e, z.clone(), e.clone()
        a, b = z[..., ia], z[..., ib]
        y[..., ia], y[..., ib] = a * c - sign * b * s, b * c + sign * a * s
        both = (e[..., ia] * c.abs() + e[..., ib] * s.abs(), e[..., ib] * c.abs() + e[..., ia] * s.abs())
        extra = (a.abs() + b.abs()) * (e_ang + 4 * F32)
        ey[..., ia], ey[..., ib] = both[0] + extra, both[1] + extra
        return y, ey
    y, ey = turn(n, e_n, 1)
    if gy is None:
        return {"y": y}, {"y": ey + u * (y.abs() + ey) + fl}
    g, eg = turn(gy.detach().cpu().double(), torch.zeros_like(x), -1)
    dw = (g * hat).sum((0, 1, 2))
    e_dw = (eg * hat.abs() + g.abs() * hat.abs() * ((dh + 8) * F32)).sum((0, 1, 2)) + (B * L * H + 16) * F32 * (g * hat).abs().sum((0, 1, 2))
    t, et = g * w, eg * w.abs()
    dot = (t * hat).mean(-1, keepdim=True)
    e_dot = (et * hat.abs() + (2 * dh + 24) * F32 * (t * hat).abs()).mean(-1, keepdim=True)
    dx = r * (t - hat * dot)
    e_dx = r * (et + hat.abs() * e_dot + (2 * dh + 24) * F32 * (t.abs() + hat.abs() * dot.abs()))
    uw = unit(w_dtype)
    return {"y": y, "dx": dx, "dw": dw}, {"y": ey + u * (y.abs() + ey) + fl, "dx": e_dx + u * (dx.abs() + e_dx) + fl,
                                          "dw": e_dw + uw * (dw.abs() + e_dw) + floor_of(w_dtype)}
