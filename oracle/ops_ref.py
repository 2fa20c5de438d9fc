"""Plain 64-bit statements of the stand-alone operators (``bidiff.ops``): forward and gradients written from the
formulas, and, beside each value, the sum of absolute terms that bounds what rounding may do to it.

``U`` is half a bf16 step relative to the value (2^-8), ``F`` half an fp32 step (2^-24)."""
import math

import torch

U = 2.0 ** -8
F = 2.0 ** -24


# ---------------------------------------------------------------- rotary positions
def rotary(x, table, positions, interleaved, inverse=False):
    """x [..., tokens, heads, D], positions [..., tokens]; table [n, rd / 2, 2]. Positions outside the table: NaN."""
    x, table = x.double(), table.double()
    half = table.shape[1]
    rd = 2 * half
    inside = (positions >= 0) & (positions < table.shape[0])
    cs = table[positions.clamp(0, table.shape[0] - 1)]
    cs = torch.where(inside[..., None, None], cs, torch.full_like(cs, math.nan))[..., None, :, :]
    cos, sin = cs[..., 0], cs[..., 1] * (-1.0 if inverse else 1.0)
    a = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    b = a + (1 if interleaved else half)
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


# ---------------------------------------------------------------- differential attention
def mm(a, b):
    """Batched product of contiguous operands (the library's batched products of transposed views have faulted a GPU)."""
    return torch.matmul(a.contiguous(), b.contiguous())


def _one(q, k, v, lam, seen, dout, scale, tol):
    """One sequence: q [Lq, 2H, D], k [Lk, 2Hkv, D], v [Lk, Hkv, E], lam [Lq, H], seen [Lk] bool. Results as float64;
    with ``tol`` also the error each may have when products take bf16 operands and sum in fp32."""
    Lq, H, Hkv, D, E = q.shape[0], q.shape[1] // 2, v.shape[1], q.shape[2], v.shape[2]
    share = H // Hkv
    qh = q.view(Lq, H, 2, D).permute(1, 2, 0, 3)
    kh = k.view(-1, Hkv, 2, D).permute(1, 2, 0, 3).repeat_interleave(share, 0)
    vh = v.permute(1, 0, 2).repeat_interleave(share, 0)
    kh = torch.where(seen[:, None], kh, torch.zeros_like(kh))
    vh = torch.where(seen[:, None], vh, torch.zeros_like(vh))
    s = mm(qh, kh.transpose(-1, -2)) * scale
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    p = torch.softmax(s, -1) if bool(seen.any()) else torch.zeros_like(s)
    w = lam.t()[..., None]                                                   # [H, Lq, 1]
    pc = p[:, 0] - w * p[:, 1]
    out = mm(pc, vh)
    res = {"out": out.permute(1, 0, 2)}
    if tol:
        # a score's error: D products summed in fp32, the scaling, the exponent's arithmetic (a few steps of values
        # up to |s| log2 e); weights inherit it relatively, twice (numerator and normaliser)
        es = (mm(qh.abs(), kh.abs().transpose(-1, -2)) * scale).amax(-1, keepdim=True) * (D + 8) * F * 2 + 64 * F
        pa = p[:, 0] + w.abs() * p[:, 1]
        ep = es.amax(1)
        res["out_tol"] = (U * 1.01 * (mm(pa, vh.abs()) + out.abs()) + ep * mm(pa, vh.abs())).permute(1, 0, 2)
    if dout is None:
        return res
    do = dout.permute(1, 0, 2)
    dp = mm(do, vh.transpose(-1, -2))
    delta = (p * dp[:, None]).sum(-1, keepdim=True)
    fac = torch.stack([torch.ones_like(w), -w], 1)
    ds = fac * p * (dp[:, None] - delta)
    dq = mm(ds, kh) * scale
    dk = mm(ds.transpose(-1, -2), qh) * scale
    dv = mm(pc.transpose(-1, -2), do)
    group = lambda x: x.view(Hkv, share, *x.shape[1:]).sum(1)  # noqa: E731
    res["dq"] = dq.permute(2, 0, 1, 3).reshape(q.shape)
    res["dk"] = group(dk).permute(2, 0, 1, 3).reshape(k.shape)
    res["dv"] = group(dv).permute(1, 0, 2)
    res["dlam"] = -delta[:, 1, :, 0].t()
    if tol:
        pv = mm(p, vh.abs()[:, None])                                           # [H, 2, Lq, E]
        # delta from the forward's sums (weights rounded to bf16) or from fp32 products; dP: E products in fp32
        edp = mm(do.abs(), vh.abs().transpose(-1, -2)) * (E + 8) * F * 2
        pdp = (p * mm(do.abs(), vh.abs().transpose(-1, -2))[:, None]).sum(-1, keepdim=True)
        edelta = (do.abs()[:, None] * pv).sum(-1, keepdim=True) * (U * 1.01 + (E + 8) * F) + pdp * (es + 16 * F) + (p * edp[:, None]).sum(-1, keepdim=True)
        fa = fac.abs()
        eds = fa * (U * 1.01 * (ds / fac.where(fac != 0, torch.ones_like(fac))).abs() + p * (edelta + edp[:, None] + (dp[:, None] - delta).abs() * (es + 16 * F)))
        long_sum = lambda n: 1.0 + n * F  # noqa: E731
        # (the weight lam may join the bf16 value or the fp32 sum)
        res["dq_tol"] = ((mm(eds, kh.abs()) * scale + U * 1.01 * dq.abs()) * long_sum(k.shape[0]) + mm(ds.abs(), kh.abs()) * scale * k.shape[0] * F).permute(2, 0, 1, 3).reshape(q.shape)
        dka = group((mm(eds.transpose(-1, -2), qh.abs()) + mm(ds.abs().transpose(-1, -2), qh.abs()) * Lq * share * F) * scale)
        res["dk_tol"] = (dka + U * 1.01 * group(dk).abs()).permute(2, 0, 1, 3).reshape(k.shape)
        epc = U * 1.01 * pc.abs() + pa * (ep + 16 * F + Lq * share * F)
        res["dv_tol"] = (group(mm(epc.transpose(-1, -2), do.abs())) + U * 1.01 * group(dv).abs()).permute(1, 0, 2)
        res["dlam_tol"] = edelta[:, 1, :, 0].t()
    return res


def differential_attention(q, k, v, lam, spans, seen, total_q, total_k, dout=None, scale=None, tol=False):
    """Flat rows: q [total_q, 2H, D] ...; spans: (query slice, key slice) of each sequence; seen [total_k] bool.
    Returns a dict of flat results (rows outside every span are zero)."""
    q, k, v, lam = q.double(), k.double(), v.double(), lam.double()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    H, E = q.shape[1] // 2, v.shape[2]
    shapes = {"out": (total_q, H, E), "dq": q.shape, "dk": k.shape, "dv": v.shape, "dlam": (total_q, H)}
    names = ["out"] if dout is None else list(shapes)
    res = {n: torch.zeros(shapes[n], dtype=torch.float64, device=q.device) for n in names}
    if tol:
        res.update({n + "_tol": torch.zeros(shapes[n], dtype=torch.float64, device=q.device) for n in names})
    for rows, keys in spans:
        if rows.stop == rows.start or keys.stop == keys.start:
            continue
        r = _one(q[rows], k[keys], v[keys], lam[rows], seen[keys], None if dout is None else dout[rows].double(), scale, tol)
        for n, x in r.items():
            at = keys if n.split("_")[0] in ("dk", "dv") else rows
            res[n][at] = x
    return res


# ---------------------------------------------------------------- vocabulary head
def linear_cross_entropy(hidden, weight, targets, w, gout=1.0, tol=False):
    """hidden [M, d], weight [V, d], w [M] row weights. Loss, dhidden, dweight (and their tolerances)."""
    h, e, w = hidden.double(), weight.double(), w.double()
    live = w != 0
    count = w.sum()
    res = {"loss": torch.zeros((), dtype=torch.float64, device=h.device), "dh": torch.zeros_like(h), "dw": torch.zeros_like(e)}
    if tol:
        res.update({"loss_tol": torch.zeros_like(res["loss"]), "dh_tol": torch.zeros_like(h), "dw_tol": torch.zeros_like(e)})
    if not bool(live.any()):
        return res
    x, t, wl = h[live], targets[live], w[live]
    z = x @ e.t()
    logp = torch.log_softmax(z, -1)
    res["loss"] = -(logp.gather(1, t[:, None])[:, 0] * wl).sum() / count
    dz = logp.exp()
    p = dz.clone()
    dz[torch.arange(len(t), device=h.device), t] -= 1.0
    dz = dz * wl[:, None]
    c = gout / count
    res["dh"][live] = c * (dz @ e)
    res["dw"] = c * (dz.t() @ x)
    if tol:
        n, V, d = len(t), e.shape[0], e.shape[1]
        # a logit: d products in fp32; the log-sum-exp: its largest logit's error and a few steps of its size
        ez = ((x.abs() @ e.abs().t()).amax(-1) + z.abs().amax(-1)) * (d + 8) * F * 2 + 64 * F
        res["loss_tol"] = ((2 * ez + 64 * F * (1 + torch.logsumexp(z, -1).abs())) * wl).sum() / count + (n + 8) * F * ((-logp.gather(1, t[:, None])[:, 0]) * wl).sum().abs() / count
        edz = U * 1.01 * dz.abs() + (p * wl[:, None]) * (2 * ez[:, None] + 16 * F) + wl[:, None] * 2 * F * 0
        res["dh_tol"][live] = abs(c) * (edz @ e.abs() + (dz.abs() @ e.abs()) * V * F) + U * 1.01 * res["dh"][live].abs()
        res["dw_tol"] = abs(c) * (edz.t() @ x.abs() + (dz.abs().t() @ x.abs()) * n * F) + U * 1.01 * res["dw"].abs()
    return res


# ---------------------------------------------------------------- a block's attention with both
def block_attention(rotary_base):
    """``backbone_ref.attention`` with rotary positions (half layout, base ``rotary_base`` or None) and, where the state
    dict holds ``lambda_weight``, differential maps. Differentiable torch, any dtype."""
    import torch.nn.functional as Fn

    def attention(x, sd, prefix, num_heads, attention_mask, dropout=None, site=0):
        B, L, d = x.shape
        dh = d // num_heads
        q, k, v = (Fn.linear(x, sd[f"{prefix}.{n}_proj.weight"], sd[f"{prefix}.{n}_proj.bias"]).view(B, L, num_heads, dh) for n in "qkv")
        if rotary_base is not None:
            ang = torch.arange(L, dtype=torch.float64)[:, None] * rotary_base ** (-2.0 * torch.arange(dh // 2, dtype=torch.float64) / dh)
            cos, sin = ang.cos().to(x.dtype)[:, None, :], ang.sin().to(x.dtype)[:, None, :]

            def turn(t):
                a, b = t[..., :dh // 2], t[..., dh // 2:]
                return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
            q, k = turn(q), turn(k)
        s = torch.einsum("blhd,bmhd->bhlm", q, k) / math.sqrt(dh)
        if attention_mask is not None:
            s = s.masked_fill(~attention_mask.to(torch.bool)[:, None, None, :], -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        lam = sd.get(f"{prefix}.lambda_weight")
        if lam is not None:
            p = p[:, 0::2] - lam[None, :, None, None] * p[:, 1::2]
            v = v.reshape(B, L, num_heads // 2, 2 * dh)
        out = torch.einsum("bhlm,bmhd->blhd", p, v).reshape(B, L, d)
        return Fn.linear(out, sd[f"{prefix}.out_proj.weight"], sd[f"{prefix}.out_proj.bias"])
    return attention
