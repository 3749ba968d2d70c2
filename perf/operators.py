"""Cases of the operators around a decoder's output: 4-bit microscaled floating point
(OCP MXFP4: e2m1 codes, one power-of-two scale per 32 values) -- quantisation and
product -- and the draw of tokens from logits with temperature, top-k, top-p and min-p.

`run` computes an operator in elementary torch operations, or, where `own` is true,
through the package's entry points. `exact` states the definitions again in 64 bits.
"""
import importlib.util
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # magnitudes of e2m1


def _pk():
    """The package (its directory's name is no module name, so it is loaded by path)."""
    if "parakeet_b200" not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet.cpp_b200")
        spec = importlib.util.spec_from_file_location("parakeet_b200", os.path.join(at, "__init__.py"),
                                                      submodule_search_locations=[at])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["parakeet_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["parakeet_b200"]


def listed():
    return [
        # one streaming window of encoder frames, made ready for a 4-bit product
        {"name": "quantize window", "op": "quantize", "rows": 14, "k": 1024, "x": "f32", "pad": 0},
        # a ragged batch of frames in half precision: odd row count, a width that ends inside a block, padded rows
        {"name": "quantize ragged", "op": "quantize", "rows": 66043, "k": 1000, "x": "bf16", "pad": 24},
        # the joint's output layer for one live utterance
        {"name": "product one", "op": "linear", "rows": 1, "k": 640, "n": 8198, "x": "f32", "y": "f32", "bias": True, "pad": 0},
        # the same layer for a live batch
        {"name": "product live", "op": "linear", "rows": 64, "k": 640, "n": 8198, "x": "f32", "y": "f32", "bias": True, "pad": 0},
        # a CTC head over the frames of a batch: odd width, odd rows
        {"name": "product ctc head", "op": "linear", "rows": 16391, "k": 1024, "n": 1025, "x": "bf16", "y": "f32", "bias": True, "pad": 0},
        # the encoder projection of a large batch
        {"name": "product frames", "op": "linear", "rows": 66044, "k": 1024, "n": 640, "x": "f32", "y": "f32", "bias": True, "pad": 0},
        # a wide generic layer over a full batch
        {"name": "product wide", "op": "linear", "rows": 8192, "k": 4096, "n": 8192, "x": "bf16", "y": "bf16", "bias": False, "pad": 0},
        # one utterance's next token
        {"name": "sample one", "op": "sample", "rows": 1, "vocab": 8193, "x": "f32", "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "spread": 2.5, "mixed": False, "pad": 0},
        # a live batch, every request with its own settings, some greedy, some masked out altogether
        {"name": "sample live", "op": "sample", "rows": 64, "vocab": 8193, "x": "f32", "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "spread": 2.5, "mixed": True, "pad": 5},
        # alignments drawn for a batch of frames: temperature alone
        {"name": "sample frames", "op": "sample", "rows": 66044, "vocab": 1025, "x": "f32", "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "spread": 2.5, "mixed": False, "pad": 0},
        # a batch over a joint's whole vocabulary, top-p and min-p
        {"name": "sample nucleus", "op": "sample", "rows": 4096, "vocab": 8193, "x": "f32", "temperature": 0.7, "top_k": 0, "top_p": 0.9, "min_p": 0.02, "spread": 2.5, "mixed": False, "pad": 0},
        # few requests over a large generic vocabulary in half precision
        {"name": "sample large vocab", "op": "sample", "rows": 4, "vocab": 131072, "x": "bf16", "temperature": 0.9, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "spread": 2.0, "mixed": False, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "sample"])
    if op == "quantize":
        k = _log_int(rng, 24, 4200)
        return {"op": op, "rows": _log_int(rng, 1, max(1, 64_000_000 // k)), "k": k,
                "x": rng.choice(["f32", "f16", "bf16"]), "pad": rng.choice([0, 0, 1, 8, 17])}
    if op == "linear":
        k, n = _log_int(rng, 33, 4200), _log_int(rng, 17, 8300)
        rows = _log_int(rng, 1, max(1, min(66044, 42_000_000 // max(k, n))))
        if rng.random() < 0.3:
            k = -(-k // 32) * 32
        return {"op": op, "rows": rows, "k": k, "n": n, "x": rng.choice(["f32", "f16", "bf16"]),
                "y": rng.choice(["f32", "f32", "bf16"]), "bias": rng.random() < 0.5, "pad": rng.choice([0, 0, 4, 3])}
    v = _log_int(rng, 40, 131072)
    return {"op": op, "rows": _log_int(rng, 1, max(1, 33_000_000 // v)), "vocab": v, "x": rng.choice(["f32", "f32", "f16", "bf16"]),
            "temperature": round(rng.uniform(0.3, 1.5), 3), "top_k": rng.choice([0, 0, 1, 20, 64, 500]),
            "top_p": rng.choice([1.0, 0.99, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.05]),
            "spread": round(rng.uniform(0.5, 4.0), 2), "mixed": rng.random() < 0.3, "pad": rng.choice([0, 0, 1, 8])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    rows, t = case["rows"], DTYPES[case["x"]]
    if case["op"] == "sample":
        v = case["vocab"]
        l = torch.randn(rows, v + case["pad"], generator=g, device="cuda").mul_(case["spread"])
        # a few likely tokens per row, the last one (a decoder's blank) often
        l.scatter_add_(1, (uniform(rows, 3) * v).long().clamp_(max=v - 1), 3.0 * case["spread"] * uniform(rows, 3))
        l[:, v - 1] += 4.0 * case["spread"] * uniform(rows)
        s["u"] = uniform(rows)
        if case["mixed"]:
            pick = uniform(rows)
            s["temperatures"] = torch.where(pick < 0.1, 0.0, 0.3 + 1.2 * uniform(rows))
            s["top_ks"] = torch.where(uniform(rows) < 0.4, 0.0, 1 + 99 * uniform(rows)).int()
            s["top_ps"] = torch.where(uniform(rows) < 0.4, 1.0, 0.4 + 0.59 * uniform(rows))
            s["min_ps"] = torch.where(uniform(rows) < 0.6, 0.0, 0.1 * uniform(rows))
            # grammar masks: a part of the vocabulary, and now and then all of it
            l.masked_fill_(uniform(rows, v + case["pad"]) < 0.3, float("-inf"))
            l.masked_fill_((uniform(rows) < 0.05)[:, None], float("-inf"))
        s["logits"] = l.to(t)[:, :v]
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(rows, device="cuda")
        return s
    k = case["k"]
    x = normal(rows, k + case["pad"])
    x[:, :: 97] *= 8.0                                  # outlier channels
    x *= torch.exp2(4.0 * uniform(rows, 1) - 2.0)       # loud and quiet frames
    if rows > 8:
        x[5] = 0.0                                      # a padding frame
    s["x_in"] = x.to(t)[:, :k]
    nb = -(-k // 32)
    if case["op"] == "quantize":
        s["codes"] = torch.empty(rows, nb * 16, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, nb, dtype=torch.uint8, device="cuda")
        s["out"] = torch.empty(rows, k, dtype=t, device="cuda")
        return s
    n = case["n"]
    w = normal(n, k) * k ** -0.5
    s["b"] = 0.1 * normal(n) if case["bias"] else None
    s["w"] = rounded(w)                                  # the weights that the 4 bits stand for
    s["y_out"] = torch.empty(rows, n, dtype=DTYPES[case["y"]], device="cuda")
    if own:
        s["layer"] = _pk().Mx4Linear(w.data_ptr(), n, k, bias=s["b"].data_ptr() if case["bias"] else None, on_device=True)
        s["work"] = torch.empty(max(1, s["layer"].workspace(rows)), dtype=torch.uint8, device="cuda")
    return s


def rounded(x):
    """x in the values that its e2m1 codes and block scales stand for, in 32 bits."""
    r, k = x.shape
    nb = -(-k // 32)
    v = torch.nn.functional.pad(x.float(), (0, nb * 32 - k)).view(r, nb, 32)
    a = v.abs().amax(-1, keepdim=True)
    e = torch.clamp(torch.frexp(a).exponent - 3, min=-127)       # floor(log2 a) - 2
    m = torch.ldexp(v.abs(), -e)
    # even codes win ties: up only past the midpoint after an even code, from the midpoint after an odd one
    q = torch.zeros_like(m)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        q = torch.where(m > mid if i % 2 == 0 else m >= mid, GRID[i + 1], q)
    q = torch.copysign(torch.ldexp(q, e), v)
    return torch.where(torch.isfinite(a), q, float("nan")).view(r, nb * 32)[:, :k]


def drawn(l, u, temp, top_k, top_p, min_p):
    """Tokens and log-probabilities of rows of logits, in 64 bits; the settings are columns."""
    rows, v = l.shape
    l = l.double()
    l = torch.where(torch.isnan(l), float("-inf"), l)
    mx, best = l.max(1, keepdim=True)
    none = mx == float("-inf")
    greedy = ~(temp > 0)
    a = torch.where(l == mx, 0.0, (l - mx) / torch.where(greedy, 1.0, temp))
    a = torch.where(torch.isneginf(l) | torch.isnan(a), float("-inf"), a)
    l, order = torch.sort(l, dim=1, descending=True, stable=True)
    w = torch.exp(torch.gather(a, 1, order))
    rank = torch.arange(v, device=l.device)[None]
    w = torch.where((top_k <= 0) | (rank < top_k), w, 0.0)
    upto = torch.cumsum(w, 1)
    keep = ((upto - w < top_p * upto[:, -1:]) | (top_p >= 1) | (rank == 0)) & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    del l, order, upto, keep
    upto = torch.cumsum(w, 1)
    total = upto[:, -1:]
    past = (upto > u * total) & (w > 0)
    tok = torch.where(past.any(1, keepdim=True), past.to(torch.uint8).argmax(1, keepdim=True), best)
    logp = torch.gather(a, 1, tok) - torch.log(total)
    # the lowest index of the largest logit; max() may give another of equal ones
    first = (a == 0).to(torch.uint8).argmax(1, keepdim=True)
    tok = torch.where(none, -1, torch.where(greedy, first, tok))
    logp = torch.where(none, float("-inf"), torch.where(greedy, 0.0, logp))
    return tok[:, 0].int(), logp[:, 0].float()


def run(s):
    op, rows = s["op"], s["rows"]
    if own:
        pk, stream = _pk(), torch.cuda.current_stream().cuda_stream
        if op == "sample":
            if s["mixed"]:
                pk.sample(s["logits"].data_ptr(), rows, s["vocab"], s["u"].data_ptr(), s["tokens"].data_ptr(), dtype=s["x"],
                          row_stride=s["vocab"] + s["pad"], logprobs=s["logprobs"].data_ptr(),
                          temperatures=s["temperatures"].data_ptr(), top_ks=s["top_ks"].data_ptr(),
                          top_ps=s["top_ps"].data_ptr(), min_ps=s["min_ps"].data_ptr(), stream=stream)
            else:
                pk.sample(s["logits"].data_ptr(), rows, s["vocab"], s["u"].data_ptr(), s["tokens"].data_ptr(), dtype=s["x"],
                          row_stride=s["vocab"] + s["pad"], logprobs=s["logprobs"].data_ptr(), temperature=s["temperature"],
                          top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], stream=stream)
            return s["tokens"], s["logprobs"]
        if op == "quantize":
            pk.mx4_quantize(s["x_in"].data_ptr(), rows, s["k"], s["codes"].data_ptr(), s["scales"].data_ptr(), dtype=s["x"],
                            row_stride=s["k"] + s["pad"], stream=stream)
            pk.mx4_dequantize(s["codes"].data_ptr(), s["scales"].data_ptr(), rows, s["k"], s["out"].data_ptr(), dtype=s["x"],
                              stream=stream)
            return s["out"]
        s["layer"].forward(s["x_in"].data_ptr(), rows, s["y_out"].data_ptr(), x_dtype=s["x"], y_dtype=s["y"],
                           x_stride=s["k"] + s["pad"], workspace=s["work"].data_ptr(), workspace_bytes=s["work"].numel(),
                           stream=stream)
        return s["y_out"]
    if op == "sample":
        if s["mixed"]:
            column = [s[n].double()[:, None] for n in ("temperatures", "top_ks", "top_ps", "min_ps")]
        else:   # the settings are 32-bit numbers at the entry point
            column = [torch.tensor(s[n], dtype=torch.float32, device="cuda").double() for n in ("temperature", "top_k", "top_p", "min_p")]
        return drawn(s["logits"], s["u"].double()[:, None], *column)
    q = rounded(s["x_in"])
    if op == "quantize":
        return q.to(DTYPES[s["x"]])
    y = q @ s["w"].t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["y"]])


def work(case):
    rows = case["rows"]
    if case["op"] == "sample":
        v = case["vocab"]
        return {"bytes": rows * (v * SIZE[case["x"]] + 12 + (16 if case["mixed"] else 0)), "flops": 10 * rows * v}
    k, nb = case["k"], -(-case["k"] // 32)
    if case["op"] == "quantize":   # codes and scales are written, and read again to be values
        return {"bytes": rows * (2 * k * SIZE[case["x"]] + 2 * 17 * nb), "flops": 4 * rows * k}
    n = case["n"]
    return {"bytes": rows * (k * SIZE[case["x"]] + n * SIZE[case["y"]]) + n * (17 * nb + (4 if case["bias"] else 0)),
            "flops": 2 * rows * k * n}


def _exact_rounded(x):
    """Nearest representable value by distance to every grid point, in 64 bits."""
    r, k = x.shape
    nb = -(-k // 32)
    v = torch.zeros(r, nb * 32, dtype=torch.float64, device=x.device)
    v[:, :k] = x.double()
    v = v.view(r, nb, 32)
    a = v.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(a > 0, a, 1.0)))
    e = torch.where(torch.exp2(e) > a, e - 1, e)                 # log2 rounded up to a whole number
    e = torch.where(torch.exp2(e + 1) <= a, e + 1, e)
    scale = torch.exp2(torch.where(a > 0, (e - 2).clamp(min=-127), -127.0))
    m = v.abs() / scale
    best, dist = torch.zeros_like(m), m.clone()
    for code in (2, 4, 6, 1, 3, 5, 7):                           # even codes first: they keep a tie
        d = (m - GRID[code]).abs()
        best, dist = torch.where(d < dist, GRID[code], best), torch.minimum(d, dist)
    return (torch.sign(v) * best * scale).view(r, nb * 32)[:, :k]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "quantize":
        return _exact_rounded(s["x_in"])
    if case["op"] == "linear":
        y = _exact_rounded(s["x_in"]) @ s["w"].double().t()
        return y if s["b"] is None else y + s["b"].double()
    logits, u = s["logits"].float().cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
    rows, v = logits.shape
    tok, logp = np.full(rows, -1, np.int32), np.full(rows, -np.inf)
    names = ("temperature", "top_k", "top_p", "min_p")
    if case["mixed"]:
        sets = np.stack([s[n + "s"].cpu().numpy().astype(np.float64) for n in names], 1)
    else:
        sets = np.tile(np.array([np.float32(case[n]) for n in names], np.float64), (rows, 1))
    for r in range(rows):
        l = np.where(np.isnan(logits[r]), -np.inf, logits[r])
        t, k, p, m = sets[r]
        top = l.max()
        if top == -np.inf:
            continue
        if not t > 0:
            tok[r], logp[r] = int(np.argmax(l)), 0.0
            continue
        a = np.full(v, -np.inf)
        fine = l > -np.inf
        a[fine] = (l[fine] - top) / t
        w = np.exp(a)
        if 0 < k < v or p < 1:
            order = np.argsort(-l, kind="stable")
            if 0 < k < v:
                w[order[int(k):]] = 0.0
            if p < 1:
                inc = np.cumsum(w[order])
                n_keep = int(np.searchsorted(inc, p * inc[-1], side="left")) + 1   # the first to reach p, and all before it
                w[order[n_keep:]] = 0.0
        if m > 0:
            w[w < m] = 0.0
        inc = np.cumsum(w)
        tok[r] = int(np.searchsorted(inc, u[r] * inc[-1], side="right"))
        logp[r] = a[tok[r]] - np.log(inc[-1])
    return tok, logp
