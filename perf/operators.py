"""Routing to experts and microscaled 4-bit (MXFP4) weights: the calls that are timed, and their plain forms.

A packed MXFP4 tensor is a pair (codes, scales): `codes` int32 [.., K/8], eight 4-bit e2m1 numbers per word, the first in
the lowest bits; `scales` uint8 [.., K/32], one power of two 2^(byte - 127) per 32 numbers.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass, plain or (own = True) through the package; returns its outputs
    work(case)          bytes and operations one pass cannot do without
    exact(case, seed)   the outputs from the definitions in 64 bits
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # router of one decoded token, softmax scores over 128 experts: the smallest call, latency only
        {"name": "route_1x128_softmax", "kind": "route", "T": 1, "E": 128, "k": 8, "score": "softmax", "bias": False,
         "groups": 1, "kept": 1, "top": 1, "renorm": True, "scale": 1.0, "dtype": "bf16"},
        # a ragged batch of requests in decode over the 512-expert layer, softmax scores chosen with a balance bias
        {"name": "route_61x512_softmax_bias", "kind": "route", "T": 61, "E": 512, "k": 10, "score": "softmax", "bias": True,
         "groups": 1, "kept": 1, "top": 1, "renorm": True, "scale": 1.0, "dtype": "f32"},
        # a prefill chunk: sigmoid scores, balance bias, the best 4 of 8 groups
        {"name": "route_4096x256_sigmoid_groups", "kind": "route", "T": 4096, "E": 256, "k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "kept": 4, "top": 2, "renorm": True, "scale": 2.5, "dtype": "f32"},
        # the converter and the loader's way back: one float16 matrix to 4 bits and back
        {"name": "quantize_4096x4096_f16", "kind": "quantize", "N": 4096, "K": 4096, "dtype": "f16"},
        # a ragged shard: odd number of rows, a row length that is a multiple of 32 only
        {"name": "quantize_1001x2080_bf16", "kind": "quantize", "N": 1001, "K": 2080, "dtype": "bf16"},
        # one decoded token through one projection
        {"name": "linear_1x4096x4096_bf16", "kind": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # a ragged batch of requests in decode, odd number of outputs, float16
        {"name": "linear_12x5001x2048_f16", "kind": "linear", "M": 12, "N": 5001, "K": 2048, "dtype": "f16"},
        # a prefill chunk through the wide projection, 16-bit activations
        {"name": "linear_2048x11008x4096_bf16", "kind": "linear", "M": 2048, "N": 11008, "K": 4096, "dtype": "bf16"},
        # activations quantised on the way in, both operands in 4 bits: a batch of requests in decode
        {"name": "linear4_16x14336x4096", "kind": "linear4", "M": 16, "N": 14336, "K": 4096, "dtype": "bf16"},
        # the same, a long prefill chunk: the largest contraction
        {"name": "linear4_4096x14336x4096", "kind": "linear4", "M": 4096, "N": 14336, "K": 4096, "dtype": "bf16"},
        # the eight routed experts of one decoded token, one projection
        {"name": "gather_8x768x2048_128experts", "kind": "gather", "T": 1, "k": 8, "E": 128, "N": 768, "K": 2048,
         "dtype": "bf16"},
        # the routed experts of a 2048-token prefill chunk, one projection
        {"name": "gather_16384x768x2048_128", "kind": "gather", "T": 2048, "k": 8, "E": 128, "N": 768, "K": 2048,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "route", "quantize", "linear", "linear", "linear4", "gather"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = max(4, _log(rng, 16, 512) // groups)
        kept = rng.randint(1, groups)
        return {"kind": kind, "T": _log(rng, 1, 4096), "E": per * groups, "k": rng.randint(1, min(16, per * kept)),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.6, "groups": groups, "kept": kept,
                "top": rng.choice([1, 2]), "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]),
                "dtype": rng.choice(["bf16", "f32", "f16"])}
    if kind == "quantize":
        return {"kind": kind, "N": _log(rng, 1, 8192), "K": 32 * _log(rng, 2, 350), "dtype": rng.choice(["f16", "bf16", "f32"])}
    K = 64 * _log(rng, 8, 172)
    N = _log(rng, 256, 14336)
    if rng.random() < 0.5:
        N = max(64, N // 64 * 64)
    most = 4096 * 14336 * 4096 // (N * K)
    if kind == "gather":
        E, N, K = rng.choice([8, 32, 128, 160]), min(N, 1536), min(K, 4096)
        return {"kind": kind, "T": _log(rng, 1, 2048), "k": rng.choice([1, 2, 4, 8]), "E": E, "N": N, "K": K, "dtype": dtype}
    M = max(1, min(most, _log(rng, 1, 4096)))
    if kind == "linear4":
        return {"kind": kind, "M": M, "N": N, "K": K + rng.choice([0, 0, 32]), "dtype": dtype}
    return {"kind": kind, "M": min(M, max(1, most // 2)), "N": N, "K": K + (rng.choice([0, 32]) if M <= 16 else 0),
            "dtype": dtype}


# ---- inputs ------------------------------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _packed(gen, rows, K):
    """Quantised weights of a checkpoint, drawn from N(0, 0.02)."""
    step = max(1, (1 << 27) // K)
    parts = [_quantize(_normal(gen, (min(step, rows - r), K), torch.bfloat16, 0.02)) for r in range(0, rows, step)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": {k: v for k, v in c.items() if k != "name"}}
    if c["kind"] == "route":
        st["logits"] = _normal(gen, (c["T"], c["E"]), DTYPES[c["dtype"]], 1.5)
        st["bias"] = _normal(gen, (c["E"],), torch.float32, 0.05) if c["bias"] else None
    elif c["kind"] == "quantize":
        st["w"] = _normal(gen, (c["N"], c["K"]), DTYPES[c["dtype"]], 0.02)
    elif c["kind"] == "gather":
        wq, s = _packed(gen, c["E"] * c["N"], c["K"])
        st["wq"], st["s"] = wq.reshape(c["E"], c["N"], -1), s.reshape(c["E"], c["N"], -1)
        st["x"] = _normal(gen, (c["T"], c["K"]), DTYPES[c["dtype"]])
        # the k experts of a token are distinct, as a router's are
        st["idx"] = torch.rand((c["T"], c["E"]), generator=gen, device="cuda").argsort(-1)[:, :c["k"]].int().contiguous()
        if own:
            import jangq_b200 as jq
            st["bank"] = jq.MXFP4ExpertBank(st["wq"], st["s"])
    else:
        st["wq"], st["s"] = _packed(gen, c["N"], c["K"])
        st["x"] = _normal(gen, (c["M"], c["K"]), DTYPES[c["dtype"]])
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------

def _quantize(w):
    """Shared exponent floor(log2(max)) - 2 per 32 numbers, numbers to the nearest of 0 .5 1 1.5 2 3 4 6 (ties to the even
    code, 6 and above to 6)."""
    b = w.float().reshape(w.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, torch.full_like(amax, -127, dtype=torch.int32)).clamp(-127, 127)
    m = torch.ldexp(b.abs(), -e[..., None])
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int() + (m >= 3.5).int()
            + (m > 5.0).int() + 8 * torch.signbit(b).int())
    word = code.reshape(w.shape[0], -1, 8)
    at = torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)
    return (word << at).sum(-1, dtype=torch.int32), (e + 127).to(torch.uint8)


def _dequantize(wq, s):
    at = torch.arange(0, 32, 4, device=wq.device, dtype=torch.int32)
    code = (wq[..., None] >> at) & 15
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=wq.device)
    v = table[code.long()].reshape(s.shape + (32,))
    return torch.ldexp(v, s.int()[..., None] - 127).reshape(wq.shape[:-1] + (-1,))


def _route(logits, bias, c):
    # 64 bits: neighbouring scores decide which expert is taken
    z = logits.double()
    if c["score"] == "softmax":
        z = torch.exp(z - z.amax(-1, keepdim=True))
        s = z / z.sum(-1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    choice = s if bias is None else s + bias.double()
    if c["groups"] > 1:
        g = choice.reshape(choice.shape[0], c["groups"], -1)
        best = g.sort(-1, descending=True).values[..., :c["top"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(mask[..., None], g, -math.inf).reshape(choice.shape)
    idx = choice.sort(dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = s.gather(1, idx)
    if c["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return idx.int(), (w * c["scale"]).float()


def _gather(x, wq, s, idx):
    T, k = idx.shape
    y = torch.empty((T * k, wq.shape[1]), device=x.device)
    flat = idx.reshape(-1).long()
    if T * k <= 64:
        w = _dequantize(wq[flat], s[flat])
        rows = x.float().repeat_interleave(k, 0)
        return torch.matmul(w, rows[..., None])[..., 0].to(x.dtype)
    for e in range(wq.shape[0]):
        at = (flat == e).nonzero()[:, 0]
        y[at] = x[at // k].float() @ _dequantize(wq[e], s[e]).t()
    return y.to(x.dtype)


def run(state):
    c = state["case"]
    if own:
        import jangq_b200 as jq
        if c["kind"] == "route":
            return jq.route_topk(state["logits"], c["k"], score=c["score"], bias=state["bias"], groups=c["groups"],
                                 groups_kept=c["kept"], group_top=c["top"], renorm=c["renorm"], scale=c["scale"])
        if c["kind"] == "quantize":
            return jq.mxfp4_dequantize(*jq.mxfp4_quantize(state["w"]), dtype=state["w"].dtype)
        if c["kind"] == "linear":
            return jq.mxfp4_matmul(state["x"], state["wq"], state["s"])
        if c["kind"] == "linear4":
            xq, xs = jq.mxfp4_quantize(state["x"])
            return jq.mxfp4_matmul(xq, state["wq"], state["s"], x_scales=xs, dtype=state["x"].dtype)
        return jq.mxfp4_gather_matmul(state["x"], state["bank"], rhs_indices=state["idx"])
    if c["kind"] == "route":
        return _route(state["logits"], state["bias"], c)
    if c["kind"] == "quantize":
        return _dequantize(*_quantize(state["w"])).to(state["w"].dtype)
    if c["kind"] == "gather":
        return _gather(state["x"], state["wq"], state["s"], state["idx"])
    x = state["x"]
    xf = _dequantize(*_quantize(x)) if c["kind"] == "linear4" else x.float()
    return (xf @ _dequantize(state["wq"], state["s"]).t()).to(x.dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "route":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["T"] * (c["E"] * size + 8 * c["k"]) + (4 * c["E"] if c["bias"] else 0), "flops": 10 * c["T"] * c["E"]}
    if c["kind"] == "quantize":
        n = c["N"] * c["K"]
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": 2 * size * n + 2 * (n * 17 // 32), "flops": 4 * n}
    if c["kind"] == "gather":
        hit = c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** c["T"])         # distinct experts of T independent choices
        pairs = c["T"] * c["k"]
        return {"bytes": int(hit * c["N"] * c["K"] * 17 / 32) + 2 * c["T"] * c["K"] + pairs * (2 * c["N"] + 4),
                "flops": 2 * pairs * c["N"] * c["K"]}
    m, n, k = c["M"], c["N"], c["K"]
    return {"bytes": n * k * 17 // 32 + 2 * m * (n + k), "flops": 2 * m * n * k}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------

def _values64(wq, s):
    """The numbers a packed pair stands for, from the bits of a code: sign, two exponent bits, one mantissa bit."""
    word = wq.long() % (1 << 32)
    code = torch.stack([(word // 16 ** j) % 16 for j in range(8)], -1).reshape(s.shape + (32,))
    sign, ex, man = 1.0 - 2.0 * (code // 8).double(), (code // 2) % 4, (code % 2).double()
    mag = torch.where(ex == 0, 0.5 * man, (1.0 + 0.5 * man) * torch.exp2((ex - 1).double()))
    scale = torch.exp2(s.double() - 127.0)
    return (sign * mag * scale[..., None]).reshape(wq.shape[:-1] + (-1,))


def _rounded64(x):
    """A tensor's nearest MXFP4 numbers, by distance to each of the eight magnitudes (a tie goes to the even code)."""
    b = x.double().reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    ex = torch.floor(torch.log2(amax))
    ex = ex + (torch.exp2(ex + 1) <= amax).double() - (torch.exp2(ex) > amax).double()        # log2 next to a power of two
    unit = torch.exp2((ex - 2.0).clamp(-127.0, 127.0))
    m = (b.abs() / unit).clamp(max=6.0)
    best, near = torch.zeros_like(m), m.clone()
    for code, v in enumerate([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], 1):
        d = (m - v).abs()
        take = (d < near) | ((d == near) & (code % 2 == 0))
        best, near = torch.where(take, torch.full_like(m, v), best), torch.minimum(d, near)
    return torch.where(amax > 0, torch.sign(b) * best * unit, torch.zeros_like(b)).reshape(x.shape)


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["kind"] == "route":
        import numpy as np
        z = st["logits"].double().cpu().numpy()
        if c["score"] == "softmax":
            p = np.exp(z - z.max(1)[:, None])
            p /= p.sum(1)[:, None]
        else:
            p = 1.0 / (1.0 + np.exp(-z))
        choice = p + (st["bias"].double().cpu().numpy() if c["bias"] else 0.0)
        idx, w = np.zeros((c["T"], c["k"]), np.int32), np.zeros((c["T"], c["k"]))
        per = c["E"] // c["groups"]
        for t in range(c["T"]):
            allowed = range(c["E"])
            if c["groups"] > 1:
                best = [np.sort(choice[t, g * per:(g + 1) * per])[::-1][:c["top"]].sum() for g in range(c["groups"])]
                keep = sorted(range(c["groups"]), key=lambda g: (-best[g], g))[:c["kept"]]
                allowed = [e for g in keep for e in range(g * per, (g + 1) * per)]
            pick = sorted(allowed, key=lambda e: (-choice[t, e], e))[:c["k"]]
            idx[t] = pick
            w[t] = p[t, pick] / (p[t, pick].sum() + 1e-20) if c["renorm"] else p[t, pick]
        return torch.from_numpy(idx), torch.from_numpy(w * c["scale"])
    if c["kind"] == "quantize":
        return _rounded64(st["w"])
    x = st["x"]
    if c["kind"] == "gather":
        flat = st["idx"].reshape(-1).long()
        y = torch.empty((flat.numel(), c["N"]), dtype=torch.float64, device=x.device)
        for e in sorted(set(flat.tolist())):
            at = torch.where(flat == e)[0]
            y[at] = torch.matmul(x.double()[torch.div(at, c["k"], rounding_mode="floor")], _values64(st["wq"][e], st["s"][e]).T)
        return y
    return torch.matmul(_rounded64(x) if c["kind"] == "linear4" else x.double(), _values64(st["wq"], st["s"]).T)
