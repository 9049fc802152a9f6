"""8-bit integers by their definition, in 64 bits: s = max(max|v| / 127, 2^-126) in float32,
q = the integer nearest to v / s (ties to even); and the order that weights are kept in."""

import torch


def held(v, dim):
    """(integers int64, scales float32 with ``dim`` kept) of v."""
    v = v.double()
    most = v.abs().amax(dim, keepdim=True)
    s = (most / 127.0).float().clamp(min=2.0**-126)
    bad = ~torch.isfinite(v).all(dim, keepdim=True)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    q = torch.where(bad, torch.zeros_like(v), torch.round(v / s.double()))
    return q.nan_to_num(0.0).to(torch.int64), s


def pitch(n):
    return -(-n // 128) * 128


def blocks(q):
    """Integers [E,K,N] in the order of an Int8Weight's codes, one element at a time's worth of
    index arithmetic."""
    E, K, N = q.shape
    out = torch.zeros(E, -(-N // 64), pitch(K) // 64, 4, 4, 16, 16, dtype=torch.int8)
    k, n = torch.arange(K).view(K, 1), torch.arange(N).view(1, N)
    c = n % 64
    i, t = 4 * (c // 16) + c % 4, c // 4 % 4
    for e in range(E):
        out[e][n // 64, k // 64, t, k % 64 // 16, i, k % 16] = q[e].to(torch.int8)
    return out


def plain_rows(codes):
    """Rows [16 A', pitch] of codes [A', pitch / 64, 4, 16, 16]."""
    a, kb = codes.shape[:2]
    return codes.permute(0, 3, 1, 2, 4).reshape(16 * a, 64 * kb)


def product(qx, sx, qw, sw, offsets):
    """Rows by their experts' weights in float64: integers [A,K], scales [A,1], integers [E,K,N],
    scales [E,1,N]; rows past the last offset are zero."""
    out = torch.zeros(qx.shape[0], qw.shape[2], dtype=torch.float64)
    for e in range(qw.shape[0]):
        a, b = offsets[e], offsets[e + 1]
        sums = (qx[a:b].double() @ qw[e].double())  # exact: below 2^53
        out[a:b] = sums * sw[e].double() * sx[a:b].double()
    return out
