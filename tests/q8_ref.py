"""Plain implementations of the 8-bit cache's operators for its tests: the
rotation and attention in 64 bits, the quantiser by its definition."""
import numpy as np
import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # half a unit in the last place


def rope(x, pos, sections, rot, pairing, interleave, ladder, theta, sign=1.0, factors=None):
    """x [T][H][hd] float64, pos [axes][T]; the rotation by its formula."""
    axis, used = [], [0] * len(sections)
    if interleave:
        left, a = list(sections), 0
        while any(left):
            if left[a]:
                axis.append(a)
                left[a] -= 1
            a = (a + 1) % len(sections)
    else:
        for a, n in enumerate(sections):
            axis += [a] * n
    y = x.copy()
    for i, a in enumerate(axis):
        f = theta ** (-used[a] / sections[a]) if ladder else theta ** (-2.0 * i / rot)
        used[a] += 1
        if factors is not None:
            f /= factors[i]
        f = float(np.float32(f))        # frequencies are 32-bit floats
        ang = sign * pos[a].astype(np.float64)[:, None] * f
        p, r = (2 * i, 2 * i + 1) if pairing == "adjacent" else (i, i + rot // 2)
        y[..., p] = x[..., p] * np.cos(ang) - x[..., r] * np.sin(ang)
        y[..., r] = x[..., p] * np.sin(ang) + x[..., r] * np.cos(ang)
    return y


def code(x, fmt):
    """Codes of float32 x in units of its scale."""
    x = torch.nan_to_num(x, nan=0.0, posinf=1e30, neginf=-1e30)
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def values(codes, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def write(codes, scales, x, start, block, fmt):
    """One slot's codes [S][hd] (uint8) and scales, written in place at `start`
    with x [n][hd] float32."""
    n = x.shape[0]
    for b in range(start // block, (start + n - 1) // block + 1 if n else 0):
        lo = b * block
        a, e = max(lo, start), min(lo + block, start + n)
        y = x[a - start:e - start]
        top = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y)).max()
        s = (top * (torch.tensor(1.0) / torch.tensor(QMAX[fmt]))).clamp(2.0 ** -40, 2.0 ** 40)
        if a > lo and scales[b] >= s:
            s = scales[b].clone()
        elif a > lo:
            codes[lo:a] = code(values(codes[lo:a], fmt) * (scales[b] / s), fmt)
        scales[b] = s
        codes[a:e] = code(y * (torch.tensor(1.0) / s), fmt)


def attend(q, k, v, pos, scale, causal, window):
    """q [T][G][hd], k and v [S][hd] float64, pos [T]: out [T][G][hd], lse [T][G],
    and the sums that bound the rounding: sum p |v| and the largest sum |q k|."""
    T, G, hd = q.shape
    S = k.shape[0]
    z = np.einsum("tgd,sd->tgs", q, k) * scale
    j = np.arange(S)[None]
    seen = np.broadcast_to(j >= 0, (T, S))
    if causal:
        seen = j <= pos[:, None]
        if window:
            seen = seen & (j > pos[:, None] - window)
    z = np.where(seen[:, None], z, -np.inf)
    m = z.max(-1, initial=-np.inf, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    p = np.exp(z - m)
    l = p.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (m + np.log(l))[..., 0]
    p = p / np.where(l > 0, l, 1.0)
    size = np.einsum("tgd,sd->tgs", np.abs(q), np.abs(k)).max(initial=0.0) * abs(scale)
    return p @ v, lse, p @ np.abs(v), size
