"""What the tests of a text stage's operators share: their definitions in 64 bits, row by row, and how far a kernel may be off."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # of a rounding, relative to the value


def seen_keys(Sq, Sk, causal=False, window=None, prefix=None, q_starts=None, k_starts=None):
    """(seen, away): [Sq,Sk] whether a query sees a key, and the key's position less the query's (0 where they share no document)."""
    seen, away = torch.zeros(Sq, Sk, dtype=torch.bool), torch.zeros(Sq, Sk, dtype=torch.int64)
    q_starts, k_starts = q_starts or [0, Sq], k_starts or [0, Sk]
    for n in range(len(q_starts) - 1):
        rows, keys = range(q_starts[n], q_starts[n + 1]), range(k_starts[n], k_starts[n + 1])
        for i in rows:
            place = i - rows.start + len(keys) - len(rows)
            for j in keys:
                d = (j - keys.start) - place
                away[i, j] = d
                see = not (causal and d > 0) and not (window is not None and abs(d) >= window)
                seen[i, j] = see or (prefix is not None and j - keys.start < prefix[n])
    return seen, away


def attention(q, k, v, scale, seen, away, cap=0.0, slopes=None, distance=None):
    """(o, tolerance) of one batch row: q [Sq,H,D], k, v [Sk,Hkv,D]. What keys that are not seen hold does not count.

    The tolerance counts, relative to a = sum_j p_j |v_j| (the most that a sum of the row's values can be): half a step for each probability
    and for the result; n additions in 32 bits; and a score's error, which is the probability's relative one: 32-bit products of D terms, the
    rounding of the score, its bias and its exponent (units of log2, two more roundings), and of a cap 2^-21 (exp2 and reciprocal of 1 ulp in
    1 - 2 / (1 + e), scaled by the cap twice). In fp16 a probability may also fall below the least number, 2^-25 each, as the row's sum is 1
    at least."""
    Sq, H, D = q.shape
    Sk, Hkv = k.shape[:2]
    u, dtype = HALF_STEP[q.dtype], q.dtype
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    o, tol = torch.zeros(Sq, H, D, dtype=torch.float64), torch.zeros(Sq, H, D, dtype=torch.float64)
    for h in range(H):
        for i in range(Sq):
            js = seen[i].nonzero()[:, 0]
            if len(js) == 0:
                continue
            kk, vv, d = k[js, h // (H // Hkv)], v[js, h // (H // Hkv)], away[i, js]
            s = kk @ q[i, h] * scale
            terms = float(((kk.abs() @ q[i, h].abs()) * scale).max())
            if cap:
                s = cap * torch.tanh(s / cap)
            bias = torch.zeros_like(s)
            if slopes is not None:
                bias = -float(slopes[h]) * d.abs().double()
            if distance is not None:
                r = distance.shape[1] // 2
                bias = distance[h].double().cpu()[d.clamp(-r, r) + r]
            size = float(s.abs().max()) + float(bias.abs().max())
            s = s + bias
            p = torch.exp(s - s.max())
            p = p / p.sum()
            o[i, h] = p @ vv
            a = p @ vv.abs()
            off = 2.0 ** -23 * (D * terms + 6.0 * size + 8.0) + cap * 2.0 ** -21
            tol[i, h] = (u * 1.01 + 2.0 * off + len(js) * 2.0 ** -23) * a + u * 1.01 * o[i, h].abs() + 1e-30
            if dtype == torch.float16:
                tol[i, h] += 2.0 ** -25 * (1.0 + len(js) * vv.abs().amax(dim=0))
    return o, tol


def rotated(x, positions, turns, neox, magnitude):
    """(y, tolerance) of x [T,H,D]: pairs of features as complex numbers. Tolerance: the result's rounding, and cos and sin in 32 bits
    (of a reduced angle rounded to 24 bits: 2 pi 2^-26), the products and the sum."""
    u, tiny = HALF_STEP[x.dtype], 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    y = x.double().cpu().clone()
    half = turns.numel()
    # (whole turns taken off in exact integers of 2^-52 turn, not in the kernel's way)
    angle = torch.tensor([[math.fmod(int(p) * float(t), 1.0) for t in turns] for p in positions], dtype=torch.float64).reshape(-1, 1, half) * 2 * math.pi
    a, b = (y[..., :half].clone(), y[..., half:2 * half].clone()) if neox else (y[..., 0:2 * half:2].clone(), y[..., 1:2 * half:2].clone())
    c, s = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    tol = torch.zeros_like(y)
    parts = (slice(0, half), slice(half, 2 * half)) if neox else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    for part, value in zip(parts, (a * c - b * s, b * c + a * s)):
        y[..., part] = value
        tol[..., part] = u * value.abs() * 1.01 + 2.0 ** -21 * abs(magnitude) * (a.abs() + b.abs()) + tiny
    return y, tol


def within(got, want, tol):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((off / tol.clamp_min(1e-300)).nan_to_num(math.inf).max()))
