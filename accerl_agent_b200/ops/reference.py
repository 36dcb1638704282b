"""fp32 PyTorch implementations of every native op.

They serve two purposes: the oracle that each CUDA kernel test compares against, and the compute
path for CPU tensors (the gloo / CPU smoke configuration). They favour clarity over speed.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    y = (xf * rstd).to(x.dtype) * w
    return y.to(x.dtype), rstd.squeeze(-1)


def rmsnorm_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, rstd: torch.Tensor):
    dyf, xf, wf = dy.float(), x.float(), w.float()
    r = rstd.float().unsqueeze(-1)
    xhat = xf * r
    g = dyf * wf
    dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    dw = (dyf * xhat).sum(0)
    return dx, dw


def rope_cos_sin(pos: torch.Tensor, head_dim: int, theta: float, dtype=torch.float32):
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=pos.device) / head_dim))
    freqs = pos.float().unsqueeze(-1) * inv_freq
    emb = torch.cat([freqs, freqs], dim=-1)
    return emb.cos().to(dtype), emb.sin().to(dtype)


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    return torch.cat([-x[..., half:], x[..., :half]], dim=-1)


def apply_rope(x: torch.Tensor, pos: torch.Tensor, theta: float, inverse: bool = False) -> torch.Tensor:
    """x: [T, H, D]; returns the rotated tensor in x's dtype (fp32 math)."""
    cos, sin = rope_cos_sin(pos, x.shape[-1], theta)
    if x.dtype == torch.bfloat16:
        cos = cos.to(torch.bfloat16).float()
        sin = sin.to(torch.bfloat16).float()
    if inverse:
        sin = -sin
    xf = x.float()
    out = xf * cos.unsqueeze(1) + rotate_half(xf) * sin.unsqueeze(1)
    return out.to(x.dtype)


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    inter = gu.shape[-1] // 2
    g, u = gu[..., :inter], gu[..., inter:]
    return (torch.nn.functional.silu(g.float()).to(gu.dtype) * u).to(gu.dtype)


def swiglu_backward(dh: torch.Tensor, gu: torch.Tensor) -> torch.Tensor:
    inter = gu.shape[-1] // 2
    g, u = gu[..., :inter].float(), gu[..., inter:].float()
    sig = torch.sigmoid(g)
    act = g * sig
    dact = sig * (1 + g * (1 - sig))
    dhf = dh.float()
    return torch.cat([dhf * u * dact, dhf * act], dim=-1).to(gu.dtype)


def quantize_rows(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """Rows of ``x`` [rows, K] in 8 bits into ``q`` int8 [rows, >= K] (zeros behind K) and ``scale`` [rows]:
    a = max |x|, scale = a / 127, q = round(127 x / a) with ties to even (the quotient in 64 bits, where 127 x
    is exact). Rows of zeros: scale 0. Rows with an infinity or NaN: scale NaN, q = 0."""
    xf = x.float()
    a = xf.abs().amax(1, keepdim=True)
    ok = torch.isfinite(a)
    r = torch.round(127.0 * xf.double() / a.double())
    q.zero_()
    q[:, : x.shape[1]] = torch.where(ok & (a > 0), r, torch.zeros_like(r)).to(torch.int8)
    scale.copy_(torch.where(ok, a / 127.0, torch.full_like(a, float("nan"))).squeeze(1))


def linear_int8(qx, sx, qw, sw, bias=None, residual=None) -> torch.Tensor:
    """fp32 ``sx sw (qx qw^T) (+ bias) (+ residual)``; the integer sum in 64-bit floats, where it is exact. Scaled first
    by the token, then by the channel, as the kernels do: the sum times a token's scale, up to 2^96 (larger ones are taken
    2^64 times smaller and the result back), stays in fp32's range, the product of two scales need not."""
    acc = qx.double() @ qw.double().t()
    large = sx > 2.0 ** 96
    y = (acc.float() * torch.where(large, sx * 2.0 ** -64, sx).unsqueeze(1)) * sw.unsqueeze(0)
    y = y * torch.where(large, 2.0 ** 64, 1.0).to(y.dtype).unsqueeze(1)
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y


def attention_varlen(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, scale: float, causal: bool = True
) -> Tuple[torch.Tensor, torch.Tensor]:
    """q: [T, Hq, D], k/v: [T, Hkv, D]. Returns (o [T, Hq, D] in q.dtype, lse [Hq, T] fp32)."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    group = Hq // Hkv
    out = torch.zeros(T, Hq, D, dtype=torch.float32, device=q.device)
    lse = torch.zeros(Hq, T, dtype=torch.float32, device=q.device)
    cu = cu_seqlens.tolist()
    for b in range(len(cu) - 1):
        s, e = cu[b], cu[b + 1]
        if e <= s:
            continue
        qb = q[s:e].float().transpose(0, 1)  # [Hq, L, D]
        kb = k[s:e].float().transpose(0, 1).repeat_interleave(group, 0)
        vb = v[s:e].float().transpose(0, 1).repeat_interleave(group, 0)
        scores = torch.matmul(qb, kb.transpose(1, 2)) * scale
        if causal:
            L = e - s
            mask = torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1)
            scores = scores.masked_fill(mask, float("-inf"))
        lse_b = torch.logsumexp(scores, dim=-1)
        probs = torch.exp(scores - lse_b.unsqueeze(-1))
        out[s:e] = torch.matmul(probs, vb).transpose(0, 1)
        lse[:, s:e] = lse_b
    return out.to(q.dtype), lse


def attention_varlen_qk(q, k, v, cu_q, cu_k, scale: float, causal: bool = True):
    """Queries ``q[cu_q[b]:cu_q[b+1]]`` are the last ones of sequence b whose keys are
    ``k[cu_k[b]:cu_k[b+1]]`` (causal mask aligned to the end)."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    group = Hq // Hkv
    out = torch.zeros(T, Hq, D, dtype=torch.float32, device=q.device)
    lse = torch.zeros(Hq, T, dtype=torch.float32, device=q.device)
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cq) - 1):
        qs, qe, ks, ke = cq[b], cq[b + 1], ck[b], ck[b + 1]
        Lq, Lk = qe - qs, ke - ks
        if Lq <= 0:
            continue
        qb = q[qs:qe].float().transpose(0, 1)
        kb = k[ks:ke].float().transpose(0, 1).repeat_interleave(group, 0)
        vb = v[ks:ke].float().transpose(0, 1).repeat_interleave(group, 0)
        scores = torch.matmul(qb, kb.transpose(1, 2)) * scale
        if causal:
            qpos = torch.arange(Lq, device=q.device).unsqueeze(1) + (Lk - Lq)
            kpos = torch.arange(Lk, device=q.device).unsqueeze(0)
            scores = scores.masked_fill(kpos > qpos, float("-inf"))
        lse_b = torch.logsumexp(scores, dim=-1)
        out[qs:qe] = torch.matmul(torch.exp(scores - lse_b.unsqueeze(-1)), vb).transpose(0, 1)
        lse[:, qs:qe] = lse_b
    return out.to(q.dtype), lse


def logsoftmax_label(logits: torch.Tensor, labels: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    lf = logits.float()
    lse = torch.logsumexp(lf, dim=-1)
    lp = lf.gather(1, labels.view(-1, 1)).squeeze(1) - lse
    probs = torch.softmax(lf, dim=-1)
    entropy = lse - (probs * lf).sum(-1)
    return lp, lse, entropy


def paged_decode(q, k_cache, v_cache, block_table, seq_lens, scale):
    """q: [S, Hq, D]; caches [NB, BS, Hkv, D]. Returns [S, Hq, D] (q dtype)."""
    S, Hq, D = q.shape
    bs = k_cache.shape[1]
    Hkv = k_cache.shape[2]
    group = Hq // Hkv
    out = torch.zeros(S, Hq, D, dtype=torch.float32, device=q.device)
    for s in range(S):
        n = int(seq_lens[s])
        nblk = (n + bs - 1) // bs
        blocks = block_table[s, :nblk].long()
        kk = k_cache[blocks].reshape(-1, Hkv, D)[:n].float().repeat_interleave(group, 1)
        vv = v_cache[blocks].reshape(-1, Hkv, D)[:n].float().repeat_interleave(group, 1)
        sc = torch.einsum("hd,thd->ht", q[s].float(), kk) * scale
        p = torch.softmax(sc, dim=-1)
        out[s] = torch.einsum("ht,thd->hd", p, vv)
    return out.to(q.dtype)


def sample_reference(logits: torch.Tensor, temperature: torch.Tensor, generator: Optional[torch.Generator] = None,
                     top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None):
    """Sampling with torch RNG (CPU path of the engine, and the oracle of the device sampler).

    Row i: argmax if temperature <= 0; otherwise softmax(x / T) restricted to the values >= the
    top_k-th largest (top_k <= 0: no restriction) and then to the nucleus of the renormalised
    distribution: the tokens, in descending probability, whose preceding cumulative mass is below
    top_p. Returns (tokens, log-probability of each token under the untempered softmax)."""
    lf = logits.float()
    logp = torch.log_softmax(lf, dim=-1)
    tokens = torch.empty(lf.shape[0], dtype=torch.long, device=lf.device)
    for i in range(lf.shape[0]):
        t = float(temperature[i])
        if t <= 0:
            tokens[i] = int(torch.argmax(lf[i]))
            continue
        z = lf[i] / t
        k = int(top_k[i]) if top_k is not None else 0
        if 0 < k < z.numel():
            z = z.masked_fill(z < torch.topk(z, k).values[-1], float("-inf"))
        probs = torch.softmax(z, dim=-1)
        p = float(top_p[i]) if top_p is not None else 1.0
        if p < 1.0:
            sorted_p, order = torch.sort(probs, descending=True)
            before = torch.cumsum(sorted_p, 0) - sorted_p
            kept = torch.zeros_like(probs).scatter_(0, order, sorted_p * (before < p))
            probs = kept / kept.sum()
        tokens[i] = int(torch.multinomial(probs, 1, generator=generator))
    return tokens, logp.gather(1, tokens.view(-1, 1)).squeeze(1)


def sample_inverse_cdf(logits, u, temperature, top_k=None, top_p=None, min_p=None):
    """Row by row in 64 bits: sort, cut (top_k, min_p, top_p), first cumulative weight above u times the sum."""
    rows = logits.shape[0]
    tokens = torch.zeros(rows, dtype=torch.long, device=logits.device)
    lps = torch.full((rows,), float("-inf"), dtype=torch.float32, device=logits.device)
    for i in range(rows):
        x = logits[i].double()
        ids = torch.nonzero(x > float("-inf")).squeeze(1)  # NaN and -inf compare false
        if ids.numel() == 0:
            continue
        vals, order = torch.sort(x[ids], descending=True, stable=True)
        ids = ids[order]
        first = vals == vals[0]
        gap = torch.where(first, torch.zeros_like(vals), vals - vals[0])  # inf - inf counts as 0
        t = float(temperature[i])
        w = torch.where(first, torch.ones_like(gap), torch.exp(gap / t)) if t > 0 else first.double()
        w = torch.nan_to_num(w)  # -inf / inf: no weight
        n = w.numel() if t > 0 else 1
        k = int(top_k[i]) if top_k is not None else 0
        if 0 < k < n:
            n = k
        m = float(min_p[i]) if min_p is not None else 0.0
        if m > 0:
            n = min(n, max(1, int((w >= m).sum())))
        cum = torch.cumsum(w[:n], 0)
        p = float(top_p[i]) if top_p is not None else 1.0
        if p < 1.0 and t > 0:
            n = int(torch.nonzero(cum >= max(p, 0.0) * cum[-1])[0]) + 1
            cum = cum[:n]
        r = float(u[i])
        r = min(max(r, 0.0), 1.0 - 2.0 ** -53) if r == r else 0.0
        above = torch.nonzero(cum > r * cum[-1])
        at = int(above[0]) if above.numel() else int(torch.nonzero(w[:n] > 0)[-1])
        tokens[i] = ids[at]
        lps[i] = (gap[at] - torch.exp(gap).sum().log()).float()
    return tokens, lps


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
