"""Plain float64 restatements of the policy memory's operators (ilrl_amd/memory.py), step by step and row by row, for the
tests.  Every result is a sum of products with non-negative coefficients, so the same function on absolute values gives the
sum of its terms' magnitudes, which the rounding bounds are taken from."""
import torch


def _rep(x, h):
    return x.double().repeat_interleave(h // x.shape[2], 2)


def _marks(b, s, reset, lengths):
    cut = torch.zeros(b, s, dtype=torch.bool) if reset is None else reset.bool().cpu()
    n = torch.full((b,), s) if lengths is None else lengths.long().cpu().clamp(0, s)
    return cut, n


def attention(q, k, v, log_decay, state, reset, lengths, scale):
    """(out, final state) in float64 on the CPU; unseen rows are chosen away, never multiplied by zero."""
    b, s, h, dk = q.shape
    q, k, v = q.double().cpu(), _rep(k.cpu(), h), _rep(v.cpu(), h)
    lam = torch.exp(log_decay.double().cpu())[:, None, None]
    cut, n = _marks(b, s, reset, lengths)
    S = torch.zeros(b, h, v.shape[3], dk, dtype=torch.float64) if state is None else state.double().cpu().clone()
    out = torch.zeros(b, s, h, v.shape[3], dtype=torch.float64)
    for i in range(b):
        for t in range(int(n[i])):
            kept = torch.zeros_like(S[i]) if cut[i, t] else lam * S[i]
            S[i] = kept + v[i, t][:, :, None] * k[i, t][:, None, :]
            out[i, t] = scale * (S[i] * q[i, t][:, None, :]).sum(-1)
    return out, S


def attention_grad(d_out, d_state, q, k, v, log_decay, state, reset, lengths, scale):
    """(dq, dk, dv, d_state_in) in float64 on the CPU."""
    b, s, h, dk = q.shape
    g, dv = k.shape[2], v.shape[3]
    do, q, kk, vv = d_out.double().cpu(), q.double().cpu(), _rep(k.cpu(), h), _rep(v.cpu(), h)
    lam = torch.exp(log_decay.double().cpu())[:, None, None]
    cut, n = _marks(b, s, reset, lengths)
    S = torch.zeros(b, h, dv, dk, dtype=torch.float64) if state is None else state.double().cpu().clone()
    R = torch.zeros(b, h, dv, dk, dtype=torch.float64) if d_state is None else d_state.double().cpu().clone()
    gq, gk, gv = torch.zeros_like(q), torch.zeros_like(kk), torch.zeros_like(vv)
    for i in range(b):
        for t in range(int(n[i])):
            kept = torch.zeros_like(S[i]) if cut[i, t] else lam * S[i]
            S[i] = kept + vv[i, t][:, :, None] * kk[i, t][:, None, :]
            gq[i, t] = scale * (S[i] * do[i, t][:, :, None]).sum(1)
        for t in range(int(n[i]) - 1, -1, -1):
            here = R[i] + scale * do[i, t][:, :, None] * q[i, t][:, None, :]
            gk[i, t] = (here * vv[i, t][:, :, None]).sum(1)
            gv[i, t] = (here * kk[i, t][:, None, :]).sum(2)
            R[i] = torch.zeros_like(here) if cut[i, t] else lam * here
    return gq, gk.view(b, s, g, h // g, dk).sum(3), gv.view(b, s, g, h // g, dv).sum(3), R


def norm(x, weight, bias, eps):
    x = x.double().cpu()
    h = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + eps)
    y = h if weight is None else h * weight.double().cpu()
    return y if bias is None else y + bias.double().cpu()


def norm_grad(dy, x, mean, rstd, weight):
    """(dx, d_weight, d_bias) for given statistics [rows]."""
    x, dy = x.double().cpu(), dy.double().cpu()
    mean, rstd = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    h = (x - mean) * rstd
    g = dy if weight is None else dy * weight.double().cpu()
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx, (dy * h).sum(0), dy.sum(0)
