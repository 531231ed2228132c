"""The paged KV cache's definitions in plain loops and 64 bits, on the CPU, for
the tests of its kernels."""
import math

import torch

PAGE = 64
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rotate(x, cos, sin, interleaved):
    """x [heads, dim] of one token by one row of angles, in 64 bits, not rounded."""
    y = x.double().clone()
    half = len(cos)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, w = y[:, a].clone(), y[:, b].clone()
        y[:, a] = u * cos[i].double() - w * sin[i].double()
        y[:, b] = w * cos[i].double() + u * sin[i].double()
    return y


def rotate32(x, cos, sin, interleaved):
    """The same in single f32 operations, rounded to bf16: what the operator is defined to give, bit for bit."""
    y = x.float().clone()
    half = len(cos)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    u, w = y[:, a].clone(), y[:, b].clone()
    y[:, a] = u * cos - w * sin
    y[:, b] = w * cos + u * sin
    return y.to(torch.bfloat16)


def quantise32(x, kind):
    """Codes and scale of one head's page x (bf16 values), in single f32 operations."""
    q = torch.tensor(QMAX[kind])
    a = x.float().abs().max().clamp(2.0 ** -40, 2.0 ** 60)
    y = (x.float() * (q * (1.0 / a))).clamp(-float(q), float(q))
    return (y.round().to(torch.int8) if kind == torch.int8 else y.to(kind)), a * (1.0 / q)


def values(codes, scale):
    return (codes.double() if codes.dtype == torch.int8 else codes.float().double()) * scale.double()


def cached(pool, pages, tail, n, h):
    """K and V [n, dim] of a sequence in 64 bits. pool: six CPU tensors (k, v, k_scale, v_scale, k_tail, v_tail)."""
    k, v, ks, vs, kt, vt = pool
    d = k.shape[3]
    kk, vv = torch.zeros(n, d, dtype=torch.float64), torch.zeros(n, d, dtype=torch.float64)
    for p in range(0, n, PAGE):
        m = min(PAGE, n - p)
        if m == PAGE:
            kk[p:p + m] = values(k[pages[p // PAGE], h], ks[pages[p // PAGE], h])
            vv[p:p + m] = values(v[pages[p // PAGE], h], vs[pages[p // PAGE], h]).T
        else:
            kk[p:p + m] = kt[tail, h, :m].double()
            vv[p:p + m] = vt[tail, h, :, :m].double().T
    return kk, vv


def attend(pool, pages, tail, start, q, scale, softcap=0.0, slopes=None, window=0, prefix=0, first=None):
    """q [n, q heads, dim] of one sequence whose rows are at start, start + 1, ... Returns out, lse and a
    bound on the error of a kernel that keeps products and sums in f32, weights in 11 bits and rounds
    the output to bf16 (8 bits): per element of out, per row of lse.

    The bound: a score is off by at most 2^-20 (a few roundings of f32 over up to 256 terms) of the sum
    A of its terms' absolute values, and 16 units more for its exponent; a weight by that and 2^-11;
    weights below 2^-26 of the largest by 2^-37 of it; the output's rounding is 2^-8."""
    n, hq, d = q.shape
    hk = pool[0].shape[1]
    out, lse = torch.zeros(n, hq, d, dtype=torch.float64), torch.full((n, hq), -math.inf, dtype=torch.float64)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    length = start + n
    j = torch.arange(length)
    pos = start + torch.arange(n)
    see = (j[None] <= pos[:, None]) | (j[None] < prefix)
    if first is not None:
        see &= j[None] >= first[:, None]
    if window:
        see &= j[None] > pos[:, None] - window
    for h in range(hk):
        k, v = cached(pool, pages, tail, length, h)
        for g in range(hq // hk):
            head = h * (hq // hk) + g
            x = (q[:, head].double() @ k.T) * scale
            a = (q[:, head].double().abs() @ k.abs().T) * abs(scale)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                a = a + softcap
            if slopes is not None:
                bias = slopes[head].double() * (pos[:, None] - j[None]).abs()
                x, a = x - bias, a + bias.abs()
            for i in range(n):
                s = see[i]
                if not bool(s.any()):
                    continue
                xi, vi = x[i, s], v[s]
                lse[i, head] = torch.logsumexp(xi, 0)
                w = torch.exp(xi - lse[i, head])
                # a key of weight 0 (a score of -inf) must not bring its value in
                out[i, head] = (w[:, None] * vi).sum(0)
                off = 2.0 ** -20 * (float(a[i, s].max()) + 16)
                lse_tol[i, head] = off
                wide = (w[:, None] * vi.abs()).sum(0)
                tol[i, head] = 2.0 ** -8 * out[i, head].abs() + (2.0 ** -11 + 2 * off) * wide + \
                    2.0 ** -36 * float(w.max()) * vi.abs().sum(0)
    return out, lse, tol, lse_tol
