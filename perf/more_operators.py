"""Cases of a second set of operators around a decoder's output: floating point of 8 bits with a
power-of-two scale for each block of 128 (e4m3 codes; rows in blocks of 1 x 128, weights of
128 x 128) -- quantisation and product -- and the verification of drafted tokens against the
target's distribution.

`run` computes an operator in elementary torch operations, or, where `own` is true, through the
package's entry points. `exact` states the definitions again in 64 bits.
"""
import importlib.util
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SETTINGS = ("temperature", "top_k", "top_p", "min_p")


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
        # one streaming window of encoder frames, made ready for an 8-bit product
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
        # one utterance's four drafts
        {"name": "verify one", "op": "verify", "sequences": 1, "drafts": 4, "vocab": 8193, "x": "f32", "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "spread": 2.5, "gap": 0.7, "certain": False, "mixed": False, "pad": 0},
        # a live batch, every request with its own settings and count of drafts, some greedy, some masked out altogether
        {"name": "verify live", "op": "verify", "sequences": 64, "drafts": 4, "vocab": 8193, "x": "f32", "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "spread": 2.5, "gap": 0.7, "certain": False, "mixed": True, "pad": 5},
        # a full batch, temperature alone
        {"name": "verify batch", "op": "verify", "sequences": 1024, "drafts": 4, "vocab": 8193, "x": "f32", "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "spread": 2.5, "gap": 0.7, "certain": False, "mixed": False, "pad": 0},
        # long drafts in half precision, top-p and min-p
        {"name": "verify nucleus", "op": "verify", "sequences": 256, "drafts": 8, "vocab": 8193, "x": "bf16", "temperature": 0.7, "top_k": 0, "top_p": 0.9, "min_p": 0.02, "spread": 2.5, "gap": 0.7, "certain": False, "mixed": False, "pad": 0},
        # drafts that were looked up, not drawn, over a large generic vocabulary
        {"name": "verify looked up", "op": "verify", "sequences": 4, "drafts": 8, "vocab": 131072, "x": "bf16", "temperature": 0.9, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "spread": 2.0, "gap": 0.7, "certain": True, "mixed": False, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "verify"])
    if op == "quantize":
        k = _log_int(rng, 24, 4200)
        return {"op": op, "rows": _log_int(rng, 1, max(1, 64_000_000 // k)), "k": k,
                "x": rng.choice(["f32", "f16", "bf16"]), "pad": rng.choice([0, 0, 1, 8, 17])}
    if op == "linear":
        k, n = _log_int(rng, 33, 4200), _log_int(rng, 17, 8300)
        rows = _log_int(rng, 1, max(1, min(66044, 42_000_000 // max(k, n))))
        if rng.random() < 0.3:
            k = -(-k // 128) * 128
        return {"op": op, "rows": rows, "k": k, "n": n, "x": rng.choice(["f32", "f16", "bf16"]),
                "y": rng.choice(["f32", "f32", "bf16"]), "bias": rng.random() < 0.5, "pad": rng.choice([0, 0, 4, 3])}
    v, d, certain = _log_int(rng, 40, 131072), rng.randint(1, 12), rng.random() < 0.3
    return {"op": op, "sequences": _log_int(rng, 1, max(1, 33_000_000 // (v * (2 * d + 1)))), "drafts": d, "vocab": v,
            "x": rng.choice(["f32", "f32", "f16", "bf16"]), "temperature": round(rng.uniform(0.3, 1.5), 3),
            "top_k": rng.choice([0, 0, 1, 20, 64, 500]), "top_p": rng.choice([1.0, 1.0, 0.99, 0.9, 0.5]),
            "min_p": rng.choice([0.0, 0.0, 0.05]), "spread": round(rng.uniform(0.5, 4.0), 2),
            "gap": round(rng.uniform(0.2, 1.5), 2), "certain": certain, "mixed": rng.random() < 0.3,
            "pad": rng.choice([0, 0, 1, 8])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    t = DTYPES[case["x"]]
    if case["op"] == "verify":
        q, d, v = case["sequences"], case["drafts"], case["vocab"]
        l = normal(q * (d + 1), v + case["pad"]).mul_(case["spread"])
        # a few likely tokens per row, the last one (a decoder's blank) often
        l.scatter_add_(1, (uniform(l.shape[0], 3) * v).long().clamp_(max=v - 1), 3.0 * case["spread"] * uniform(l.shape[0], 3))
        l[:, v - 1] += 4.0 * case["spread"] * uniform(l.shape[0])
        # the draft's logits: the target's, seen less well
        m = l.view(q, d + 1, -1)[:, :d].reshape(q * d, -1) + case["gap"] * normal(q * d, v + case["pad"])
        s["uniforms"] = uniform(q, d + 1)
        if case["mixed"]:
            pick = uniform(q)
            s["temperatures"] = torch.where(pick < 0.1, 0.0, 0.3 + 1.2 * uniform(q))
            s["top_ks"] = torch.where(uniform(q) < 0.4, 0.0, 1 + 99 * uniform(q)).int()
            s["top_ps"] = torch.where(uniform(q) < 0.4, 1.0, 0.4 + 0.59 * uniform(q))
            s["min_ps"] = torch.where(uniform(q) < 0.6, 0.0, 0.1 * uniform(q))
            s["counts"] = (uniform(q) * (d + 1.99)).int().clamp_(max=d)
            # grammar masks of a sequence: a part of the vocabulary, and now and then all of it
            mask = (uniform(q, v + case["pad"]) < 0.3) | (uniform(q) < 0.05)[:, None]
            l.view(q, d + 1, -1).masked_fill_(mask[:, None], float("-inf"))
            m.view(q, d, -1).masked_fill_(mask[:, None], float("-inf"))
        s["logits_in"], m = l.to(t)[:, :v], m.to(t)[:, :v]
        s["draft_logits"] = None if case["certain"] else m
        # the drafts: drawn as the draft's model would, or the likeliest by its logits
        tok = []
        at = max(1, 16_000_000 // v)
        for i in range(0, q * d, at):
            w = m[i:i + at].double()
            if case["certain"]:
                tok.append(torch.where(w.amax(1) > float("-inf"), w.argmax(1), -1))
                continue
            w = kept_weights(w, *(c[i:i + at] for c in columns(s, d)))
            upto = w.cumsum(1)
            u = uniform(w.shape[0], 1).double() * upto[:, -1:]
            tok.append(torch.where(upto[:, -1] > 0, ((upto > u) & (w > 0)).to(torch.uint8).argmax(1), -1))
        s["tokens_in"] = torch.cat(tok).int().view(q, d)
        s["tokens"] = torch.empty(q, d + 1, dtype=torch.int32, device="cuda")
        s["accepted"] = torch.empty(q, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(q, d + 1, device="cuda")
        if own:
            s["work"] = torch.empty(max(1, _pk().verify_workspace(q, d, v)), dtype=torch.uint8, device="cuda")
        return s
    rows, k = case["rows"], case["k"]
    x = normal(rows, k + case["pad"])
    x[:, :: 97] *= 8.0                                  # outlier channels
    x *= torch.exp2(4.0 * uniform(rows, 1) - 2.0)       # loud and quiet frames
    if rows > 8:
        x[5] = 0.0                                      # a padding frame
    s["x_in"] = x.to(t)[:, :k]
    nb = -(-k // 128)
    if case["op"] == "quantize":
        s["codes"] = torch.empty(rows, -(-k // 16) * 16, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, nb, dtype=torch.uint8, device="cuda")
        s["out"] = torch.empty(rows, k, dtype=t, device="cuda")
        return s
    n = case["n"]
    w = normal(n, k) * k ** -0.5
    s["b"] = 0.1 * normal(n) if case["bias"] else None
    s["w"] = rounded(w, 128)                             # the weights that the 8 bits stand for
    s["y_out"] = torch.empty(rows, n, dtype=DTYPES[case["y"]], device="cuda")
    if own:
        s["layer"] = _pk().Fp8Linear(w.data_ptr(), n, k, bias=s["b"].data_ptr() if case["bias"] else None, on_device=True)
        s["work"] = torch.empty(max(1, s["layer"].workspace(rows)), dtype=torch.uint8, device="cuda")
    return s


def rounded(x, block_rows):
    """x in the values that its e4m3 codes and block scales stand for, in 32 bits."""
    r, k = x.shape
    nr, nb = -(-r // block_rows), -(-k // 128)
    v = torch.nn.functional.pad(x.float(), (0, nb * 128 - k, 0, nr * block_rows - r)).view(nr, block_rows, nb, 128)
    a = v.abs().amax((1, 3), keepdim=True)
    f = torch.frexp(a)
    # the smallest power of two by which the largest magnitude comes to 448 (0.875 * 2^9) at most
    e = torch.clamp(f.exponent - torch.where(f.mantissa <= 0.875, 9, 8), min=-127)
    m = torch.ldexp(v.abs(), -e)
    step = torch.clamp(torch.frexp(m).exponent - 4, min=-9)      # three bits behind the first, from 2^-6 up
    q = torch.ldexp(torch.round(torch.ldexp(m, -step)), step)    # ties to even
    q = torch.copysign(torch.ldexp(q, e), v)
    return torch.where(torch.isfinite(a), q, float("nan")).reshape(nr * block_rows, nb * 128)[:r, :k]


def columns(s, repeat):
    """The settings as columns, one row for each of a sequence's `repeat` rows."""
    q = s["sequences"]
    if s["mixed"]:
        c = [s[n + "s"].double() for n in SETTINGS]
    else:   # 32-bit numbers at the entry point
        c = [torch.full((q,), float(np.float32(s[n])), dtype=torch.float64, device="cuda") for n in SETTINGS]
    return [x.repeat_interleave(repeat)[:, None] for x in c]


def kept_weights(l, temp, top_k, top_p, min_p):
    """Weights that the settings leave of rows of logits (64 bits): exp((l - max) / T), zero for what is cut."""
    v = l.shape[1]
    l = torch.where(torch.isnan(l), float("-inf"), l)
    mx = l.amax(1, keepdim=True)
    greedy = ~(temp > 0)
    a = torch.where(l == mx, 0.0, (l - mx) / torch.where(greedy, 1.0, temp))
    a = torch.where(torch.isneginf(l) | torch.isnan(a), float("-inf"), a)
    w = torch.exp(a)
    if bool((((top_k > 0) & (top_k < v)) | ~(top_p >= 1) | (min_p > 0)).any()):
        order = torch.sort(l, dim=1, descending=True, stable=True).indices
        ws = torch.gather(w, 1, order)
        rank = torch.arange(v, device=l.device)[None]
        ws = torch.where((top_k <= 0) | (rank < top_k), ws, 0.0)
        upto = torch.cumsum(ws, 1)
        keep = ((upto - ws < top_p * upto[:, -1:]) | (top_p >= 1) | (rank == 0)) & (ws >= min_p)
        w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    # greedy: the first of the largest alone
    first = torch.zeros_like(w).scatter_(1, (l == mx).to(torch.uint8).argmax(1, keepdim=True), 1.0)
    return torch.where(mx == float("-inf"), 0.0, torch.where(greedy, first, w))


def verified(s):
    """Tokens, accepted drafts and log-probabilities, in 64 bits."""
    q, d, v = s["sequences"], s["drafts"], s["vocab"]
    dev = s["logits_in"].device
    at = torch.arange(d + 1, device=dev)[None]
    n = s["counts"].long()[:, None] if s["mixed"] else torch.full((q, 1), d, device=dev)
    w = kept_weights(s["logits_in"].double(), *columns(s, d + 1))
    total = w.sum(1, keepdim=True)
    p = (w / torch.where(total > 0, total, 1.0)).view(q, d + 1, v)
    del w
    tok = s["tokens_in"].long()
    fine = (tok >= 0) & (tok < v)
    tok0 = torch.where(fine, tok, 0)[:, :, None]
    pd = torch.where(fine, torch.gather(p[:, :d], 2, tok0)[:, :, 0], 0.0)
    if s["draft_logits"] is None:
        f = None
        qd = fine.double()
    else:
        w = kept_weights(s["draft_logits"].double(), *columns(s, d))
        total = w.sum(1, keepdim=True)
        f = (w / torch.where(total > 0, total, 1.0)).view(q, d, v)
        del w
        qd = torch.where(fine, torch.gather(f, 2, tok0)[:, :, 0], 0.0)
    u = s["uniforms"].double()
    bad = ~(u[:, :d] * qd < pd) & (at[:, :d] < n)
    first = torch.where(bad.any(1), bad.to(torch.uint8).argmax(1), n[:, 0])[:, None]     # drafts accepted
    rejected = first < n
    here = torch.gather(p, 1, first[:, :, None].expand(-1, -1, v))[:, 0]
    place = first.clamp(max=d - 1)
    if f is None:
        other = torch.zeros_like(here).scatter_(1, torch.gather(tok0[:, :, 0], 1, place),
                                                torch.gather(fine, 1, place).double())
    else:
        other = torch.gather(f, 1, place[:, :, None].expand(-1, -1, v))[:, 0]
    rest = torch.where(rejected, (here - other).clamp(min=0.0), here)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, here)
    upto = rest.cumsum(1)
    past = (upto > u[:, d:] * upto[:, -1:]) & (rest > 0)
    new = torch.where(past.any(1, keepdim=True), past.to(torch.uint8).argmax(1, keepdim=True), -1)
    pnew = torch.where(new >= 0, torch.gather(here, 1, new.clamp(min=0)), 0.0)
    out = torch.where(at < first, torch.nn.functional.pad(tok, (0, 1)), torch.where(at == first, new, -1))
    pp = torch.where(at < first, torch.nn.functional.pad(pd, (0, 1)), torch.where(at == first, pnew, 0.0))
    return out.int(), first[:, 0].int(), torch.log(pp).float()


def run(s):
    op = s["op"]
    if own:
        pk, stream = _pk(), torch.cuda.current_stream().cuda_stream
        if op == "verify":
            kw = dict(temperatures=s["temperatures"].data_ptr(), top_ks=s["top_ks"].data_ptr(), top_ps=s["top_ps"].data_ptr(),
                      min_ps=s["min_ps"].data_ptr(), n_drafts=s["counts"].data_ptr()) if s["mixed"] else \
                 dict(temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
            pk.verify(s["logits_in"].data_ptr(), s["sequences"], s["drafts"], s["vocab"], s["tokens_in"].data_ptr(),
                      s["uniforms"].data_ptr(), s["tokens"].data_ptr(), s["accepted"].data_ptr(),
                      draft_logits=0 if s["draft_logits"] is None else s["draft_logits"].data_ptr(), dtype=s["x"],
                      row_stride=s["vocab"] + s["pad"], draft_stride=s["vocab"] + s["pad"], logprobs=s["logprobs"].data_ptr(),
                      workspace=s["work"].data_ptr(), workspace_bytes=s["work"].numel(), stream=stream, **kw)
            return s["tokens"], s["accepted"], s["logprobs"]
        if op == "quantize":
            pk.fp8_quantize(s["x_in"].data_ptr(), s["rows"], s["k"], s["codes"].data_ptr(), s["scales"].data_ptr(), dtype=s["x"],
                            row_stride=s["k"] + s["pad"], stream=stream)
            pk.fp8_dequantize(s["codes"].data_ptr(), s["scales"].data_ptr(), s["rows"], s["k"], s["out"].data_ptr(), dtype=s["x"],
                              stream=stream)
            return s["out"]
        s["layer"].forward(s["x_in"].data_ptr(), s["rows"], s["y_out"].data_ptr(), x_dtype=s["x"], y_dtype=s["y"],
                           x_stride=s["k"] + s["pad"], workspace=s["work"].data_ptr(), workspace_bytes=s["work"].numel(),
                           stream=stream)
        return s["y_out"]
    if op == "verify":
        return verified(s)
    q = rounded(s["x_in"], 1)
    if op == "quantize":
        return q.to(DTYPES[s["x"]])
    y = q @ s["w"].t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["y"]])


def work(case):
    if case["op"] == "verify":
        q, d, v = case["sequences"], case["drafts"], case["vocab"]
        rows = q * (d + 1 if case["certain"] else 2 * d + 1)
        return {"bytes": rows * v * SIZE[case["x"]] + q * (16 * d + 16 + (20 if case["mixed"] else 0)), "flops": 10 * rows * v}
    rows, k, nb = case["rows"], case["k"], -(-case["k"] // 128)
    if case["op"] == "quantize":   # codes and scales are written, and read again to be values
        return {"bytes": rows * (2 * k * SIZE[case["x"]] + 2 * (k + nb)), "flops": 4 * rows * k}
    n = case["n"]
    return {"bytes": rows * (k * SIZE[case["x"]] + n * SIZE[case["y"]]) + n * (k + (4 if case["bias"] else 0)) + -(-n // 128) * nb,
            "flops": 2 * rows * k * n}


def _exact_rounded(x, block_rows):
    """Nearest representable value, found in the sorted list of all of them, in 64 bits."""
    r, k = x.shape
    nr, nb = -(-r // block_rows), -(-k // 128)
    v = torch.zeros(nr * block_rows, nb * 128, dtype=torch.float64, device=x.device)
    v[:r, :k] = x.double()
    v = v.view(nr, block_rows, nb, 128)
    a = v.abs().amax(3, keepdim=True).amax(1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(a > 0, a, 1.0) / 448.0)))
    scale = torch.where(scale * 448.0 < a, scale * 2, scale)      # log2 rounded past a whole number
    scale = torch.where(scale * 224.0 >= a, scale / 2, scale)
    scale = torch.where(a > 0, scale.clamp(min=2.0 ** -127), 2.0 ** -127)
    grid = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    grid = torch.tensor(grid[:127], dtype=torch.float64, device=x.device)            # code 127 is no number
    m = (v.abs() / scale).contiguous()
    up = torch.searchsorted(grid, m).clamp_(max=126)              # the first not below
    down = (up - 1).clamp(min=0)
    far, near = grid[up] - m, m - grid[down]
    code = torch.where((far < near) | ((far == near) & (up % 2 == 0)), up, down)
    return (torch.sign(v) * grid[code] * scale).reshape(nr * block_rows, nb * 128)[:r, :k]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "quantize":
        return _exact_rounded(s["x_in"], 1)
    if case["op"] == "linear":
        y = _exact_rounded(s["x_in"], 1) @ s["w"].double().t()
        return y if s["b"] is None else y + s["b"].double()
    q, d, v = case["sequences"], case["drafts"], case["vocab"]
    target = s["logits_in"].float().cpu().numpy().astype(np.float64).reshape(q, d + 1, v)
    draft = None if case["certain"] else s["draft_logits"].float().cpu().numpy().astype(np.float64).reshape(q, d, v)
    given, u = s["tokens_in"].cpu().numpy(), s["uniforms"].cpu().numpy().astype(np.float64)
    if case["mixed"]:
        sets = np.stack([s[n + "s"].cpu().numpy().astype(np.float64) for n in SETTINGS], 1)
        count = s["counts"].cpu().numpy()
    else:
        sets = np.tile(np.array([np.float32(case[n]) for n in SETTINGS], np.float64), (q, 1))
        count = np.full(q, d)

    def chances(l, t, k, p, m):
        l = np.where(np.isnan(l), -np.inf, l)
        top = l.max()
        c = np.zeros(v)
        if top == -np.inf:
            return c
        if not t > 0:
            c[int(np.argmax(l))] = 1.0
            return c
        fine = l > -np.inf
        c[fine] = np.exp((l[fine] - top) / t)
        if 0 < k < v or p < 1:
            order = np.argsort(-l, kind="stable")
            if 0 < k < v:
                c[order[int(k):]] = 0.0
            if p < 1:
                inc = np.cumsum(c[order])
                c[order[int(np.searchsorted(inc, p * inc[-1], side="left")) + 1:]] = 0.0   # the first to reach p stays
        if m > 0:
            c[c < m] = 0.0
        return c / c.sum()

    out = np.full((q, d + 1), -1, np.int32)
    logp = np.full((q, d + 1), -np.inf)
    ok = np.zeros(q, np.int32)
    for i in range(q):
        for j in range(int(count[i]) + 1):
            p = chances(target[i, j], *sets[i])
            if j < count[i]:
                t = int(given[i, j])
                f = np.zeros(v)
                if draft is not None:
                    f = chances(draft[i, j], *sets[i])
                elif 0 <= t < v:
                    f[t] = 1.0
                if 0 <= t < v and u[i, j] * f[t] < p[t]:
                    out[i, j], logp[i, j] = t, np.log(p[t])
                    ok[i] += 1
                    continue
                rest = np.maximum(p - f, 0.0)
                rest = rest if rest.sum() > 0 else p
            else:
                rest = p
            if rest.sum() > 0:
                inc = np.cumsum(rest)
                t = int(np.searchsorted(inc, u[i, d] * inc[-1], side="right"))
                out[i, j], logp[i, j] = t, np.log(p[t])
            break
    return out, ok, logp
