"""MXFP4 and routing in plain numpy, 64 bits: what the GPU tests compare with."""
import numpy as np

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6])


def quantize(w):
    """float64 [R, K] (numbers of a 16- or 32-bit type) -> (codes uint8 [R, K], bytes uint8 [R, K/32])."""
    b = w.reshape(w.shape[0], -1, 32)
    amax = np.abs(b).max(-1)
    finite = np.isfinite(amax)
    _, ex = np.frexp(np.where(finite & (amax > 0), amax, 1.0))               # amax = f * 2^ex, f in [0.5, 1)
    e = np.where(amax > 0, np.maximum(ex - 1 - 2, -127), -127)
    with np.errstate(invalid="ignore"):
        m = np.abs(b) * np.exp2(-e.astype(np.float64))[..., None]
    code = np.zeros(b.shape, np.uint8)
    near = np.full(b.shape, np.inf)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):                                       # even codes first: a tie stays with them
        d = np.abs(np.minimum(np.where(finite[..., None], m, 0.0), 6.0) - VALUES[c])
        code, near = np.where(d < near, c, code), np.minimum(d, near)
    code = np.where(np.signbit(b), code + 8, code)
    code = np.where(finite[..., None], code, 0).astype(np.uint8)
    return code.reshape(w.shape), np.where(finite, e + 127, 255).astype(np.uint8)


def pack(code):
    """uint8 [.., K] -> uint32 [.., K/8], the first code in the lowest bits."""
    c = code.reshape(code.shape[:-1] + (-1, 8)).astype(np.uint32)
    return np.bitwise_or.reduce(c << np.arange(0, 32, 4, dtype=np.uint32), axis=-1)


def unpack(words):
    w = np.ascontiguousarray(words).view(np.uint32)
    return ((w[..., None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15).astype(np.uint8).reshape(w.shape[:-1] + (-1,))


def values(words, bytes_):
    """float64 [.., K] of a packed pair."""
    v = VALUES[unpack(words)].reshape(bytes_.shape + (32,))
    s = np.where(bytes_ == 255, np.nan, np.exp2(bytes_.astype(np.float64) - 127.0))
    return (v * s[..., None]).reshape(bytes_.shape[:-1] + (-1,))


def route(logits, k, score, bias, groups, kept, top, renorm, scale):
    """(idx, w) of float64 logits, by sorting: descending choice, the lower expert (group) first."""
    z = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    T, E = z.shape
    with np.errstate(invalid="ignore", over="ignore"):
        if score == "softmax":
            mx = z.max(1, keepdims=True)
            p = np.where(z == mx, np.where(mx == -np.inf, 0.0, 1.0), np.exp(z - mx))
            s = p.sum(1, keepdims=True)
            p = p / np.where(s == 0, 1.0, s)
        else:
            p = 1.0 / (1.0 + np.exp(-z))
    # without a bias the scores grow with the logits, also where 64 bits no longer show it
    choice = z if bias is None and (groups == 1 or top == 1) else p if bias is None else p + bias.astype(np.float64)
    choice = np.where(np.isnan(choice), -np.inf, choice)
    idx, w = np.zeros((T, k), np.int32), np.zeros((T, k))
    per = E // groups
    for t in range(T):
        best = [np.sort(choice[t, g * per:(g + 1) * per])[::-1][:top].sum() for g in range(groups)] if groups > 1 else [0.0]
        keep = sorted(range(groups), key=lambda g: (-best[g], g))[:kept] if groups > 1 else [0]
        allowed = [e for g in keep for e in range(g * per, (g + 1) * per)]
        idx[t] = sorted(allowed, key=lambda e: (-choice[t, e], e))[:k]
        s = p[t, idx[t]]
        w[t] = s / (s.sum() + 1e-20) * scale if renorm else s * scale
    return idx, w
