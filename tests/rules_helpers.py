"""The operators' definitions in 64 bits, written apart from the kernels: key ranges pair by pair, rotary positions, and
attention with a score cap, distance slopes and a range of keys a row, with its gradients."""
import torch


def visible(Nq, Nk, b, causal=False, window=None, offsets=None, prefixes=None, lengths=None, starts=0):
    """(Nq, Nk) booleans of batch entry b, from the definition; the arguments are lists or ints on the host."""
    t = torch.arange(Nq).view(-1, 1) + (starts[b] if isinstance(starts, (list, tuple)) else starts)
    j = torch.arange(Nk).view(1, -1)
    see = (j < (Nk if lengths is None else lengths[b])) & (t == t)
    front = torch.zeros_like(see)
    if offsets is not None:
        off = offsets[b] if isinstance(offsets[0], (list, tuple)) else offsets
        same = torch.zeros_like(see)
        for m in range(len(off) - 1):
            mine = (t >= off[m]) & (t < off[m + 1]) & (j >= off[m]) & (j < off[m + 1])
            same |= mine
            if prefixes is not None:
                pre = prefixes[b] if isinstance(prefixes[0], (list, tuple)) else prefixes
                front |= mine & (j < off[m] + pre[m])
        see = see & same
    elif prefixes is not None:
        front = j < prefixes[b]
    if window is not None:
        see = see & (t - j < window) & (j - t < window)
    if causal:
        see = see & ((j <= t) | front)
    return see


def attention64(q, k, v, see, positions, scale, cap=None, slopes=None, grad=None):
    """(o, lse) or (o, lse, dq, dk, dv) in 64 bits.  see: (B, Nq, Nk) booleans, positions: (B, Nq)."""
    q, k, v = (t.double() for t in (q, k, v))
    B, Nq, H, D = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    see, positions = see.to(q.device), positions.to(q.device)
    o, lse = torch.zeros_like(q), torch.full((B, H, Nq), float("-inf"), dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    distance = (positions.unsqueeze(2) - torch.arange(Nk, device=q.device)).abs().double()
    for b in range(B):
        some = see[b].any(dim=1)
        for h in range(H):
            hk = h * Hkv // H
            s = q[b, :, h] @ k[b, :, hk].T * scale
            bend = torch.ones_like(s)
            if cap is not None:
                t = torch.tanh(s / cap)
                s, bend = cap * t, 1 - t * t
            if slopes is not None:
                s = s - float(slopes[h]) * distance[b]
            s = s.masked_fill(~see[b], float("-inf"))
            p = torch.zeros_like(s)
            p[some] = torch.softmax(s[some], dim=1)
            lse[b, h, some] = torch.logsumexp(s[some], dim=1)
            o[b, :, h] = p @ v[b, :, hk]
            if grad is not None:
                g = grad[b, :, h].double()
                dv[b, :, hk] += p.T @ g
                dp = g @ v[b, :, hk].T
                ds = p * (dp - (p * dp).sum(dim=1, keepdim=True)) * bend * scale
                dq[b, :, h] = ds @ k[b, :, hk]
                dk[b, :, hk] += ds.T @ q[b, :, h]
    return (o, lse) if grad is None else (o, lse, dq, dk, dv)


def rotary64(x, positions, inv_freq, interleaved, factor=1.0, inverse=False):
    """x turned (or turned back) by position, pair by pair, as complex numbers."""
    half = inv_freq.shape[0]
    x = x.double()
    angle = positions.double().unsqueeze(-1) * inv_freq.double() * (-1 if inverse else 1)
    turn = torch.polar(torch.full_like(angle, factor), angle).unsqueeze(2)
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        y = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
        y = torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((y, rest), dim=-1)


def rel(got, want):
    """Relative L2 distance; 0 where both are nothing but zeros."""
    got, want = got.double(), want.double().to(got.device)
    norm = want.norm().item()
    err = (got - want).norm().item()
    return err / norm if norm else err
