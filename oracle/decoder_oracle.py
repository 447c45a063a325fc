"""Plain definitions of the decoder-block operators (rotary positions with several axes, cross attention, the residual
update with its norms), differentiable, in the dtype of their inputs: the tests call them in float64."""
import torch


def rope_axes(x, pos, sections, base=10000.0, interleaved=False, shared_ladder=False):
    """x [B, N, H, D], pos [N, A] or [B, N, A]: each pair of dims as a plane, turned by its axis's angle."""
    bases = base if isinstance(base, (tuple, list)) else (base,) * len(sections)
    if pos.dim() == 2:
        pos = pos[None]
    P = sum(sections)
    out = list(x.unbind(-1))
    p = 0
    for a, n in enumerate(sections):
        for j in range(n):
            e = p / P if shared_ladder else j / n
            ang = (pos[..., a].to(torch.float64) * bases[a] ** -e)[:, :, None].expand(x.shape[:3])
            c, s = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
            i1, i2 = (2 * p, 2 * p + 1) if interleaved else (p, P + p)
            x1, x2 = x[..., i1], x[..., i2]
            out[i1], out[i2] = x1 * c - x2 * s, x2 * c + x1 * s
            p += 1
    return torch.stack(out, -1)


def allowed_keys(B, Nk, kv_len=None, key_mask=None):
    if key_mask is not None:
        return key_mask
    if kv_len is None:
        return torch.ones(B, Nk, dtype=torch.bool)
    return torch.arange(Nk)[None] < kv_len[:, None]


def cross_attn(q, k, v, keep, scale=None):
    """q [B, Nq, Hq, D], k and v [B, Nk, Hk, D], keep [B, Nk] bool.  Rows of masked keys are dropped before anything is
    computed from them; a sample without a key gives zeros."""
    B, Nq, Hq, D = q.shape
    G = Hq // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    outs = []
    for b in range(B):
        idx = keep[b].nonzero().flatten()
        if idx.numel() == 0:
            outs.append(q[b] * 0)
            continue
        kb, vb = (t[b, idx].repeat_interleave(G, 1) for t in (k, v))
        p = torch.softmax(scale * torch.einsum("qhd,khd->hqk", q[b], kb), -1)
        outs.append(torch.einsum("hqk,khd->qhd", p, vb))
    return torch.stack(outs)


def _norm(v, kind, weight, bias, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def norm_gate_residual(x, u, gate=None, branch_scale=None, res_scale=1.0, post=None, post_weight=None, post_bias=None,
                       pre=None, pre_weight=None, pre_bias=None, eps=1e-6):
    p = _norm(u, post, post_weight, post_bias, eps)
    if gate is not None:
        p = p * (gate if gate.dim() == 1 else gate[:, None])
    if branch_scale is not None:
        p = torch.where(branch_scale[:, None, None] == 0, torch.zeros_like(p), p * branch_scale[:, None, None])
    y = res_scale * x + p
    return y, (_norm(y, pre, pre_weight, pre_bias, eps) if pre is not None else None)
