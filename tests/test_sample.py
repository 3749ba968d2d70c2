"""Drawing tokens from logits: pk_sample against the definition in f64, the CTC path that
calls it, and the refusals."""
import ctypes as C

import numpy as np
import pytest

DEFAULTS = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)


@pytest.fixture(scope="module")
def built(pk):
    pk.build()
    return pk


def ref_row(l, u, temperature, top_k, top_p, min_p):
    """(token, log-probability) of one row by sorting and summing in f64."""
    return ref_draw(l, u, temperature, top_k, top_p, min_p)[:2]


def ref_draw(l, u, temperature, top_k, top_p, min_p):
    """The same, and how far u times the kept sum lies from the nearest border between two tokens."""
    l = np.asarray(l, np.float64)
    v = len(l)
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    if top == -np.inf:
        return -1, -np.inf, np.inf
    if not temperature > 0:
        return int(np.argmax(l)), 0.0, np.inf
    a = np.full(v, -np.inf)
    fine = (l > -np.inf) & (l < top) & (top < np.inf)   # a maximum of +infinity leaves the others nothing
    with np.errstate(over="ignore"):
        a[fine] = (l[fine] - top) / np.float64(np.float32(temperature))
    a[l == top] = 0.0
    w = np.exp(a)
    w[w <= 2.0 ** -44] = 0.0                            # what 64-bit fixed point drops
    order = np.argsort(-l, kind="stable")
    n = v if top_k <= 0 else min(top_k, v)
    s = w[order]
    s[n:] = 0.0
    if not top_p >= 1:
        before = np.cumsum(s) - s
        keep = before < np.float64(np.float32(top_p)) * s.sum() if top_p > 0 else np.zeros(v, bool)
        keep[0] = True
        s = np.where(keep, s, 0.0)
    if min_p > 0:
        s = np.where(s >= min(np.float64(np.float32(min_p)), 1.0), s, 0.0)
    w = np.zeros(v)
    w[order] = s
    run = np.cumsum(w)
    u = 0.0 if not u > 0 else min(float(np.float32(u)), float(np.float32(1 - 2 ** -24)))
    tok = int(np.searchsorted(run, u * run[-1], side="right"))
    tok = min(tok, int(np.flatnonzero(w)[-1]))
    return tok, a[tok] - np.log(run[-1]), np.abs(run - u * run[-1]).min()


def run(pk, l, u, dtype="f32", pad=0, shift=0, stream=None, rows_apart=False, **kw):
    import torch
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    l = np.asarray(l, np.float32)
    r, v = l.shape
    buf = torch.full((r * (v + pad) + shift + 32,), 1e4, dtype=t, device="cuda")     # larger than any logit
    x = buf[shift:shift + r * (v + pad)].view(r, v + pad)
    x[:, :v] = torch.from_numpy(l).cuda().to(t)
    uu = torch.from_numpy(np.asarray(u, np.float32)).cuda()
    tok = torch.full((r + 8,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((r + 8,), 123.0, device="cuda")
    args, keep = {}, []
    for name, val in kw.items():
        if np.ndim(val):
            d = torch.from_numpy(np.asarray(val, np.int32 if name == "top_k" else np.float32)).cuda()
            keep.append(d)
            args[name + "s"] = d.data_ptr()
        else:
            args[name] = val
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    pk.sample(x.data_ptr(), r, v, uu.data_ptr(), tok.data_ptr(), dtype=dtype, row_stride=v + pad, logprobs=lp.data_ptr(),
              stream=s, **args)
    torch.cuda.synchronize()
    assert (tok[r:] == -7).all() and (lp[r:] == 123.0).all()
    return x[:, :v].float().cpu().numpy(), tok[:r].cpu().numpy(), lp[:r].cpu().numpy()


def check(seen, u, tok, lp, **kw):
    """Tokens equal; log-probabilities: a f64 number rounded once (2^-24 of it) whose sum of weights
    is off by 2^-44 a token at most. Where f32 sums may have settled the token, its sum of weights is off
    by their bound instead, and (l - max) / T by three roundings, 3 2^-24 of it:
    rows of up to 2048 tokens with nothing cut, 512 and more of them: 8 2^-24 for each exponential,
    2.78 log2 V <= 31 for its argument, 19 for the additions, 58 2^-24 < 2^-18 of the sum;
    rows of up to 16384 tokens with top-p: 8, 2.78 log2 V <= 39 and 19, 66 2^-24 < 2^-17 of the sum."""
    kw = {**DEFAULTS, **kw}
    r, v = seen.shape
    f32 = r >= 512 and v <= 2048 and all(np.ndim(x) == 0 for x in kw.values()) and not (
        0 < kw["top_k"] < v or kw["top_p"] < 1 or kw["min_p"] > 0)   # one short row in a warp
    for i in range(r):
        one = {n: (x[i] if np.ndim(x) else x) for n, x in kw.items()}
        t, p = ref_row(seen[i], u[i], **one)
        if tok[i] != t:
            # Rounding each weight to 2^-43 moves a border by half of that for every token before it and
            # u times the sum by as much: v 2^-43 in all, and one more for the product's own rounding.
            # Nearer to a border than that the definition in fixed point names the other token.
            near = ref_draw(seen[i], u[i], **one)[2]
            assert near <= (v + 1) * 2.0 ** -43, (i, tok[i], t, one, u[i], near)
            continue
        if np.isinf(p):
            assert lp[i] == p
        else:
            tol = 2.0 ** -24 * abs(p) + v * 2.0 ** -43 + 2.0 ** -40
            bound = 2.0 ** -18 if f32 else 2.0 ** -17 if one["top_p"] < 1 and v <= 16384 else 0.0
            if bound:
                top = np.nanmax(seen[i]).astype(np.float64)
                a = abs(seen[i][t] - top) / one["temperature"] if one["temperature"] > 0 and np.isfinite(top) else 0.0
                tol += bound + 3 * 2.0 ** -24 * a
            assert abs(lp[i] - p) <= tol, (i, lp[i], p)


# ---- CPU -----------------------------------------------------------------------

def test_reference_known_answers():
    l = np.log([0.5, 0.25, 0.125, 0.125])
    assert [ref_row(l, u, 1.0, 0, 1.0, 0.0)[0] for u in (0.0, 0.49, 0.51, 0.76, 0.9)] == [0, 0, 1, 2, 3]
    assert [ref_row(l, u, 1.0, 2, 1.0, 0.0)[0] for u in (0.66, 0.67)] == [0, 1]
    assert [ref_row(l, u, 1.0, 3, 1.0, 0.0)[0] for u in (0.99,)] == [2]           # the tie keeps the lower index
    assert ref_row(l, 0.99, 1.0, 0, 0.5, 0.0) == (0, 0.0)
    assert ref_row(l, 0.99, 1.0, 0, 0.51, 0.0)[0] == 1
    assert ref_row(l, 0.99, 1.0, 0, 1.0, 0.3)[0] == 1
    assert ref_row([1, 3, 3], 0.9, 0.0, 0, 1.0, 0.0) == (1, 0.0)
    assert ref_row([-np.inf, np.nan], 0.5, 1.0, 0, 1.0, 0.0) == (-1, -np.inf)


def test_refusals(built):
    pk, abi, L = built, built.abi, built.lib()
    assert C.sizeof(abi.pk_sample_args) == 104 and C.sizeof(abi.pk_ctc_draw) == 32
    p = 1 << 20

    def call(device=99, **kw):
        d = dict(logits=p, logits_type=0, vocab=10, rows=3, row_stride=10, uniforms=p, tokens=p)
        d.update(kw)
        return L.pk_sample(device, C.byref(abi.pk_sample_args(**d)), None)

    assert call() == abi.PK_ERR_NO_DEVICE and call(device=-1) == abi.PK_ERR_NO_DEVICE
    for kw in (dict(logits_type=8), dict(vocab=0), dict(vocab=abi.PK_SAMPLE_MAX_VOCAB + 1, row_stride=1 << 20), dict(rows=-1),
               dict(rows=1 << 31), dict(row_stride=9), dict(row_stride=1 << 40), dict(logits=None), dict(uniforms=None),
               dict(tokens=None), dict(logits=p + 2), dict(logits_type=1, logits=p + 1), dict(tokens=p + 2), dict(uniforms=p + 1),
               dict(logprobs=p + 2), dict(temperatures=p + 2), dict(top_ks=p + 1), dict(top_ps=p + 3), dict(min_ps=p + 2)):
        assert call(**kw) == abi.PK_ERR_INVALID, kw
        assert b"pk_sample" in L.pk_last_error()
    assert L.pk_sample(0, None, None) == abi.PK_ERR_INVALID
    for vocab in (0, -1, abi.PK_SAMPLE_MAX_VOCAB + 1, (1 << 32) + 4):       # nothing that 32 bits would cut to a size
        with pytest.raises(ValueError, match="vocab"):
            pk.sample(p, 1, vocab, p, p)
    assert L.pk_ctc_decode(None, None, None, 0, None, None, 0, None, None, None, 0, None, None, None) == abi.PK_ERR_INVALID


# ---- GPU -----------------------------------------------------------------------

SETS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=64, temperature=1.3), dict(top_p=0.9),
        dict(top_p=0.3, temperature=2.0), dict(min_p=0.05), dict(top_k=50, top_p=0.95, min_p=0.02, temperature=0.8),
        dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0), dict(top_k=7, top_p=0.999, min_p=1e-6)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETS, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()) or "plain")
@pytest.mark.parametrize("v", [1, 2, 31, 33, 257, 1025, 8193])
def test_matches_definition(built, v, kw):
    rng = np.random.default_rng(v)
    r = 40
    l = rng.standard_normal((r, v)) * rng.choice([0.0, 0.5, 3.0, 12.0], (r, 1))
    u = rng.random(r).astype(np.float32)
    u[:3] = (0.0, 1.0 - 2.0 ** -24, 0.5)
    seen, tok, lp = run(built, l, u, **kw)
    check(seen, u, tok, lp, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("f32", 3, 1), ("bf16", 0, 0)])
@pytest.mark.parametrize("v", [1, 5, 33, 257, 1024, 1025, 1280])
def test_many_short_rows(built, v, dtype, pad, shift):
    """Rows that f32 sums may settle: random numbers anywhere, and right at the borders between tokens,
    where they must not; flat, peaked and masked rows."""
    rng = np.random.default_rng(v)
    r = 1200
    l = rng.standard_normal((r, v)) * rng.choice([0.0, 0.3, 2.0, 8.0], (r, 1))
    l[rng.random((r, v)) < 0.05] = -np.inf
    l[5], l[6] = -np.inf, np.nan
    l[7, v // 2] = np.inf
    l[8, :] = np.where(np.arange(v) % 2, np.nan, 0.0)
    u = rng.random(r)
    t = {"f32": np.float32, "bf16": np.float32}[dtype]
    for i in range(200, r):                                # the border behind a random token, as near as u's 24 bits go
        x = np.where(np.isnan(l[i]), -np.inf, l[i].astype(t).astype(np.float64))
        w = np.exp(x - x.max()) if np.isfinite(x.max()) else np.ones(v)
        u[i] = (np.cumsum(w) / w.sum())[rng.integers(v)] + rng.choice([0.0, 2.0 ** -24, -2.0 ** -24, 1e-6, -1e-6])
    u = np.clip(u, 0, 1 - 2.0 ** -24).astype(np.float32)
    for kw in (dict(), dict(temperature=0.6), dict(temperature=1e-35), dict(temperature=float("inf"))):
        seen, tok, lp = run(built, l, u, dtype, pad, shift, **kw)
        check(seen, u, tok, lp, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [1281, 2047, 2048])
def test_many_rows_of_two_thousand(built, v):
    """The longest rows that f32 sums may settle, flat ones among them: their sums are off the most."""
    rng = np.random.default_rng(v)
    r = 1184
    l = rng.standard_normal((r, v)) * rng.choice([0.0, 0.3, 2.0, 8.0], (r, 1))
    l[rng.random((r, v)) < 0.05] = -np.inf
    u = rng.random(r)
    w = np.exp(l - l.max(1, keepdims=True))
    u[200:] = (np.cumsum(w, 1) / w.sum(1, keepdims=True))[np.arange(r), rng.integers(v, size=r)][200:]   # at borders
    u = np.clip(u, 0, 1 - 2.0 ** -24).astype(np.float32)
    seen, tok, lp = run(built, l, u, "f32", 1, 1)
    check(seen, u, tok, lp)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(top_k=9), dict(top_p=0.9, temperature=0.8), dict(top_k=200, top_p=0.97, min_p=0.002)],
                         ids=["k", "p", "all"])
@pytest.mark.parametrize("r,v", [(2960, 33), (2960, 1056), (3000, 1057), (593, 257), (593, 5120), (593, 5121), (592, 2049), (297, 2049),
                                 (296, 2049), (592, 2048)])
def test_either_side_of_each_team(built, r, v, kw):
    """Row counts and lengths where one size of team gives way to the next; the same row is the same token
    in the batch and among few."""
    rng = np.random.default_rng(r + v)
    l = rng.standard_normal((r, v)) * rng.choice([0.0, 0.5, 2.5, 9.0], (r, 1))
    l[rng.random((r, v)) < 0.02] = -np.inf
    l[3] = -np.inf
    u = rng.random(r).astype(np.float32)
    seen, tok, lp = run(built, l, u, "f32", 3, 0, **kw)
    some = np.unique(np.concatenate([np.arange(40), rng.integers(r, size=160), [r - 1]]))
    check(seen[some], u[some], tok[some], lp[some], **kw)
    _, few, _ = run(built, l[some[:60]], u[some[:60]], **kw)
    assert np.array_equal(few, tok[some[:60]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 1, 1), ("f32", 4, 0), ("f16", 0, 0), ("f16", 3, 1), ("bf16", 0, 0), ("bf16", 7, 1), ("bf16", 8, 0)])
@pytest.mark.parametrize("v", [5, 1024, 1030, 8193])
def test_types_and_strides(built, v, dtype, pad, shift):
    """Half precision makes many equal logits: ties go by index."""
    rng = np.random.default_rng(v + pad)
    r = 30
    l = rng.standard_normal((r, v)) * 2
    u = rng.random(r).astype(np.float32)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.8), dict(top_k=100, top_p=0.7, min_p=0.01, temperature=0.9)):
        seen, tok, lp = run(built, l, u, dtype, pad, shift, **kw)
        check(seen, u, tok, lp, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [20000, 131072, 262145])
@pytest.mark.parametrize("r", [1, 5])
def test_large_vocabularies(built, v, r):
    rng = np.random.default_rng(v)
    l = rng.standard_normal((r, v)) * 2.5
    u = rng.random(r).astype(np.float32)
    for dtype in ("f32", "bf16"):
        for kw in (dict(), dict(top_k=50), dict(top_p=0.95, temperature=0.8), dict(top_k=3000, top_p=0.9, min_p=0.001)):
            seen, tok, lp = run(built, l, u, dtype, **kw)
            check(seen, u, tok, lp, **kw)


@pytest.mark.gpu
def test_largest_vocabulary(built):
    """2^19 equal logits: the fixed-point sum's largest value; the token is u's place among them."""
    v = built.abi.PK_SAMPLE_MAX_VOCAB
    u = np.array([0.0, 0.25, 0.75, 1 - 2.0 ** -24], np.float32)
    _, tok, lp = run(built, np.zeros((4, v)), u)
    assert tok.tolist() == [int(x * v) for x in u.astype(np.float64)]
    assert np.allclose(lp, -np.log(v), rtol=2.0 ** -23)
    _, tok, _ = run(built, np.zeros((4, v)), u, top_p=0.5)
    assert tok.tolist() == [int(x * (v // 2)) for x in u.astype(np.float64)]
    _, tok, _ = run(built, np.zeros((4, v)), u, top_k=1000)
    assert tok.tolist() == [int(x * 1000) for x in u.astype(np.float64)]


@pytest.mark.gpu
def test_settings_of_each_row(built):
    rng = np.random.default_rng(8)
    r, v = 300, 2000
    l = rng.standard_normal((r, v)) * 3
    l[rng.random((r, v)) < 0.3] = -np.inf
    l[17] = -np.inf
    u = rng.random(r).astype(np.float32)
    kw = dict(temperature=np.where(rng.random(r) < 0.2, 0.0, rng.uniform(0.2, 2, r)).astype(np.float32),
              top_k=rng.choice([0, -3, 1, 2, 50, 1999, 2000, 5000], r).astype(np.int32),
              top_p=rng.choice([0.1, 0.5, 0.9, 1.0, 2.0], r).astype(np.float32),
              min_p=rng.choice([0.0, -1.0, 0.01, 0.5], r).astype(np.float32))
    seen, tok, lp = run(built, l, u, **kw)
    check(seen, u, tok, lp, **kw)
    # a row by itself draws what it draws in the batch
    for i in (0, 17, 123, 299):
        one = {n: x[i:i + 1] for n, x in kw.items()}
        _, t1, p1 = run(built, l[i:i + 1], u[i:i + 1], **one)
        assert t1[0] == tok[i] and (p1[0] == lp[i])


@pytest.mark.gpu
@pytest.mark.parametrize("v", [6, 700, 9000, 40000])
def test_masks_and_special_values(built, v):
    low = float(np.finfo(np.float32).min)
    rng = np.random.default_rng(v)
    base = rng.standard_normal(v)
    rows = []
    rows.append(np.full(v, -np.inf))                                  # nothing left
    rows.append(np.full(v, np.nan))
    rows.append(np.where(np.arange(v) % 2, np.nan, -np.inf))
    rows.append(np.full(v, low))                                      # masked by the lowest number: all equal
    rows.append(np.where(np.arange(v) == v - 2, base, -np.inf))       # one token left
    rows.append(np.where(np.arange(v) % 3, low, base))
    x = base.copy(); x[0] = np.nan; x[3] = np.inf; x[5] = np.inf
    rows.append(x)                                                    # two infinities share it all
    x = base.copy(); x[1] = np.nan
    rows.append(x)
    rows.append(np.zeros(v))
    rows.append(np.where(np.arange(v) % 2, 0.0, -0.0))                # signed zeros are equal
    rows.append(base * 1e30)
    x = np.full(v, low); x[2] = -low
    rows.append(x)                                                    # a difference past f32's range
    l = np.array(rows)
    for u in (0.0, 0.37, 0.99999):
        uu = np.full(len(l), u, np.float32)
        for kw in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(top_k=2, top_p=0.99, min_p=0.1),
                   dict(temperature=1e-30), dict(temperature=float("inf")), dict(temperature=float("nan"))):
            seen, tok, lp = run(built, l, uu, **kw)
            check(seen, uu, tok, lp, **kw)


@pytest.mark.gpu
def test_cut_inside_equal_logits(built):
    """Ties at the border of top-k and top-p keep the lower indices, wherever they lie."""
    rng = np.random.default_rng(4)
    r, v = 64, 3001
    l = rng.integers(-3, 4, (r, v)).astype(np.float64)
    for kw in (dict(top_k=1), dict(top_k=10), dict(top_k=450), dict(top_k=1500), dict(top_p=0.25), dict(top_p=0.7),
               dict(top_k=777, top_p=0.613, temperature=3.0)):
        u = rng.random(r).astype(np.float32)
        u[0], u[1] = 0.0, 1 - 2.0 ** -24
        seen, tok, lp = run(built, l, u, **kw)
        check(seen, u, tok, lp, **kw)


@pytest.mark.gpu
def test_random_numbers_out_of_range(built):
    l = np.random.default_rng(0).standard_normal((5, 50))
    u = np.array([-1.0, np.nan, 1.0, 7.0, np.inf], np.float32)
    seen, tok, lp = run(built, l, u, top_k=10)
    check(seen, u, tok, lp, top_k=10)


@pytest.mark.gpu
def test_drawn_frequencies(built):
    """10^5 evenly spread random numbers: each token is drawn as often as its probability says, to one draw."""
    n = 100_000
    l = np.log(np.array([0.4, 0.05, 0.3, 0.2, 0.05]))
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    _, tok, _ = run(built, np.tile(l, (n, 1)), u)
    got = np.bincount(tok, minlength=5)
    assert np.abs(got - n * np.array([0.4, 0.05, 0.3, 0.2, 0.05])).max() <= 2


@pytest.mark.gpu
def test_no_rows_and_other_stream(built):
    import torch
    pk = built
    pk.sample(0, 0, 10, 0, 0)
    s = torch.cuda.Stream()
    rng = np.random.default_rng(2)
    l, u = rng.standard_normal((20, 500)), rng.random(20).astype(np.float32)
    torch.cuda.synchronize()
    seen, tok, lp = run(pk, l, u, stream=s.cuda_stream, top_p=0.9)
    check(seen, u, tok, lp, top_p=0.9)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [300, 9000, 140000])
def test_captured_and_replayed(built, v):
    import torch
    pk = built
    rng = np.random.default_rng(v)
    r = 6
    l = torch.zeros(r, v, device="cuda")
    u = torch.zeros(r, device="cuda")
    tok = torch.zeros(r, dtype=torch.int32, device="cuda")
    lp = torch.zeros(r, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        pk.sample(l.data_ptr(), r, v, u.data_ptr(), tok.data_ptr(), logprobs=lp.data_ptr(), temperature=0.8, top_k=40, top_p=0.95,
                  stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        a, b = rng.standard_normal((r, v)).astype(np.float32), rng.random(r).astype(np.float32)
        l.copy_(torch.from_numpy(a))
        u.copy_(torch.from_numpy(b))
        g.replay()
        torch.cuda.synchronize()
        check(a, b, tok.cpu().numpy(), lp.cpu().numpy(), temperature=0.8, top_k=40, top_p=0.95)


@pytest.mark.gpu
def test_two_streams_at_once(built):
    """Calls that overlap on two streams, large and small, draw what they draw alone."""
    import torch
    pk = built
    rng = np.random.default_rng(12)
    jobs = []
    for r, v, kw in ((3, 70000, dict(top_p=0.9)), (700, 1025, dict()), (40, 9000, dict(top_k=300, top_p=0.8)), (2000, 300, dict(top_k=5))):
        l = torch.from_numpy(rng.standard_normal((r, v)).astype(np.float32) * 2).cuda()
        u = torch.from_numpy(rng.random(r).astype(np.float32)).cuda()
        alone = torch.empty(r, dtype=torch.int32, device="cuda")
        pk.sample(l.data_ptr(), r, v, u.data_ptr(), alone.data_ptr(), **kw)       # the default stream
        jobs.append((l, u, alone, torch.empty_like(alone), kw))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n in range(6):
        for i, (l, u, alone, out, kw) in enumerate(jobs):
            out.fill_(-9)
        torch.cuda.synchronize()
        for i, (l, u, alone, out, kw) in enumerate(jobs):
            pk.sample(l.data_ptr(), l.shape[0], l.shape[1], u.data_ptr(), out.data_ptr(), stream=streams[(i + n) % 2].cuda_stream, **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(alone, out) for _, _, alone, out, _ in jobs)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [600, 3])
def test_values_too_close_for_a_bin(built, r):
    """More equal and all but equal logits than a list takes, down to the smallest numbers: every level of
    the histogram has to part them."""
    tiny = np.float32(1.401298464e-45)
    rng = np.random.default_rng(1)
    v = 3000
    rows = [np.where(rng.random(v) < 0.5, tiny, 0.0), rng.integers(0, 5, v) * tiny, np.float32(1.0) + rng.integers(0, 3, v) * np.float32(2 ** -23),
            np.where(rng.random(v) < 0.5, 3.4028235e38, 3.4028233e38), -np.abs(rng.standard_normal(v)) * np.float32(1e-38),
            np.where(np.arange(v) % 2, 0.0, -tiny)]
    l = np.array(rows)[np.arange(r) % len(rows)].astype(np.float32)
    u = rng.random(r).astype(np.float32)
    for kw in (dict(top_k=700), dict(top_p=0.37), dict(top_k=1600, top_p=0.9), dict(top_k=1600, top_p=0.9, temperature=1e-30)):
        seen, tok, lp = run(built, l, u, **kw)
        check(seen, u, tok, lp, **kw)


def collapse(path, blank, prev):
    toks, frs = [], []
    for t, x in enumerate(path):
        if x != blank and x != prev:
            toks.append(int(x))
            frs.append(t)
        prev = int(x)
    return toks, frs, prev


@pytest.mark.gpu
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("with_head", [False, True])
@pytest.mark.parametrize("on_device", [False, True])
def test_ctc_decode(built, with_head, drawn, on_device):
    """Frames through the 4-bit head, the draw and the collapse in one call: the same as the
    parts by themselves, utterance by utterance, windows carried."""
    import torch
    pk = built
    rng = np.random.default_rng(11)
    v, k, n_frames = 65, 96, np.array([40, 0, 1, 300, 77], np.int32)
    offs = np.concatenate([[0], np.cumsum(n_frames)[:-1]]).astype(np.int64) + 2
    total = int(n_frames.sum()) + 2
    w = rng.standard_normal((v, k)).astype(np.float32)
    b = rng.standard_normal(v).astype(np.float32)
    b[v - 1] += 6
    head = pk.Mx4Linear(w, bias=b) if with_head else None
    x = rng.standard_normal((total, k if with_head else v)).astype(np.float32) * 0.5
    if not with_head:
        x[:, v - 1] += 2
        x[50] = -np.inf                                   # a frame with nothing to draw
    u = rng.random(total).astype(np.float32)
    kw = dict(temperature=0.9, top_k=30, top_p=0.95, min_p=0.001)
    # the parts
    s = torch.cuda.current_stream().cuda_stream
    dx, du = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    lg = dx
    if with_head:
        lg = torch.empty(total, v, device="cuda")
        ws = torch.empty(head.workspace(total), dtype=torch.uint8, device="cuda")
        head.forward(dx.data_ptr(), total, lg.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=s)
    if drawn:
        tok = torch.empty(total, dtype=torch.int32, device="cuda")
        pk.sample(lg.data_ptr(), total, v, du.data_ptr(), tok.data_ptr(), stream=s, **kw)
        path = tok.cpu().numpy()
        path[path < 0] = v - 1
    else:
        path = lg.cpu().numpy().argmax(1)
    ctc = pk.CtcGreedy(v, v - 1)
    prev0 = np.array([3, 5, int(path[offs[2]]), -1, 2], np.int32)
    torch.cuda.synchronize()
    got, frames, prev = ctc.decode_frames(dx.data_ptr() if on_device else x, offs, n_frames, head=head,
                                          uniforms=(du.data_ptr() if on_device else u) if drawn else None,
                                          uniforms_on_device=on_device, prev=prev0, on_device=on_device, with_frames=True,
                                          **(kw if drawn else {}))
    for i in range(len(n_frames)):
        t, f, p = collapse(path[offs[i]:offs[i] + n_frames[i]], v - 1, prev0[i])
        assert got[i].tolist() == t and frames[i].tolist() == f and prev[i] == p
    if not with_head and not drawn:
        again, _, _ = ctc.decode(x, offs, n_frames, prev=prev0)
        assert all(np.array_equal(a, c) for a, c in zip(got, again))
    ctc.close()


@pytest.mark.gpu
def test_ctc_decode_wide_head(built):
    """A head so wide that its logits, not the frames, bound a product. Small integers throughout: every
    sum is exact, whichever kernel takes it."""
    import torch
    pk = built
    rng = np.random.default_rng(2)
    v, k, total = 40_000, 64, 7_000
    w = rng.integers(-2, 3, (v, k)).astype(np.float32)
    x = rng.integers(-2, 3, (total, k)).astype(np.float32)
    path = (torch.from_numpy(x).cuda() @ torch.from_numpy(w).cuda().T).cpu().numpy().argmax(1)   # the first of equal ones
    ctc = pk.CtcGreedy(v, v - 1)
    got, _, prev = ctc.decode_frames(x, [0], [total], head=pk.Mx4Linear(w))
    t, _, p = collapse(path, v - 1, -1)
    assert got[0].tolist() == t and prev[0] == p
    ctc.close()


@pytest.mark.gpu
def test_ctc_decode_many_frames_and_refusals(built):
    """More frames than one product takes; a head of another width is refused."""
    pk = built
    rng = np.random.default_rng(1)
    v, k, total = 40, 64, 40_000
    head = pk.Mx4Linear(rng.standard_normal((v, k)).astype(np.float32))
    ctc = pk.CtcGreedy(v, 0)
    x = rng.standard_normal((total, k)).astype(np.float32)
    got, _, _ = ctc.decode_frames(x, [0, 15_000], [15_000, 25_000], head=head)
    parts = [ctc.decode_frames(x[a:a + n], [0], [n], head=head)[0][0] for a, n in ((0, 15_000), (15_000, 25_000))]
    assert all(np.array_equal(a, b) for a, b in zip(got, parts))
    with pytest.raises(pk.PkError, match="vocab_size wide"):
        pk.CtcGreedy(v + 1, 0).decode_frames(x, [0], [10], head=head)
    with pytest.raises(ValueError, match="random numbers"):
        ctc.decode_frames(x, [0], [10], head=head, uniforms=np.zeros(9, np.float32))
    out, _, prev = ctc.decode_frames(np.zeros((0, k), np.float32), [], [], head=head)
    assert out == [] and len(prev) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("r,v", [(1, 1000), (40, 1000), (300, 1500), (297, 8193), (600, 4000)])
@pytest.mark.parametrize("quads", [1, 4, 8, 128])
def test_nan_logits_with_top_p(built, r, v, quads, dtype):
    """NaN logits count as -infinity however many threads meet one: a multiple of four of them, each with one
    of the heaviest tokens beside it, must not pass for a sum without them."""
    rng = np.random.default_rng(quads * 100 + v)
    l = rng.standard_normal((r, v)) * 0.3
    for q in range(quads):
        l[:, 4 * q] = np.nan
        l[:, 4 * q + 1] = 4.0 + 0.25 * (q % 7)
    u = rng.random(r).astype(np.float32)
    for kw in (dict(top_p=0.9), dict(top_p=0.5, temperature=0.7), dict(top_p=0.99, min_p=0.001)):
        seen, tok, lp = run(built, l, u, dtype, **kw)
        check(seen, u, tok, lp, **kw)
        assert not np.isnan(seen[np.arange(r), tok]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(min_p=1e-6), dict(top_p=0.9999999)], ids=["plain", "m", "p"])
@pytest.mark.parametrize("v", [64, 450, 900])
def test_halves_of_the_same_weights(built, v, kw):
    """Rows whose second half holds the first one's weights in another order, all of them near the largest: with
    u = 1/2 the running sum over the first half is u times the total exactly, so the token is the second half's
    first, whatever the order in which the weights were added up (v weights of 2^43 stay below 2^53: u times
    their total is not rounded)."""
    rng = np.random.default_rng(v)
    h = v // 2
    for r in (1, 7, 300, 700, 1300, 3100):
        base = (-0.01 * rng.random((r, h))).astype(np.float32)
        base[:, 0] = 0.0
        l = np.concatenate([rng.permuted(base, axis=1), rng.permuted(base, axis=1)], 1)
        _, tok, _ = run(built, l, np.full(r, 0.5, np.float32), **kw)
        assert (tok == h).all(), (r, np.unique(tok))


def test_closed_head_is_refused(built):
    """A closed layer's handle is null, which the C entry point takes for frames that are logits already."""
    pk = built
    ctc = pk.CtcGreedy.__new__(pk.CtcGreedy)               # no device here: nothing is called with these handles
    ctc._h, ctc.vocab_size, ctc.blank_id = None, 1025, 1024
    head = pk.Mx4Linear.__new__(pk.Mx4Linear)
    head.h, head.n, head.k, head.device = C.c_void_p(), 1025, 1024, 0      # as close() leaves it
    with pytest.raises(ValueError, match="closed"):
        ctc.decode_frames(np.zeros((4, 1024), np.float32), [0], [4], head=head)


def test_arrays_too_short_are_refused(built):
    """Offsets, previous tokens or logits for fewer utterances than there are: the C entry points would read past them."""
    pk = built
    ctc = pk.CtcGreedy.__new__(pk.CtcGreedy)
    ctc._h, ctc.vocab_size, ctc.blank_id = None, 5, 0
    x = np.zeros((8, 5), np.float32)
    for call in (ctc.decode, ctc.decode_frames):
        for offs, n, prev in (([0], [4, 4], None), ([0, 4, 8], [4, 4], None), ([0, 4], [4, 4], [1]), ([0, 4], [4, 4], [1, 2, 3])):
            with pytest.raises(ValueError, match="utterances"):
                call(x, offs, n, prev=prev)
        with pytest.raises(ValueError, match="values"):
            call(x, [0, 4], [4, 5])
        with pytest.raises(pk.PkError):                    # lengths agree: on to the handle, which is null here
            call(x, [0, 4], [4, 4], prev=[1, 2])


@pytest.mark.gpu
def test_ctc_reads_only_its_utterances(built):
    """A short window far into a large buffer costs the window: no memory for the frames before it. Utterances far
    apart, out of order, overlapping and empty ones between them are what they are side by side."""
    import torch
    pk = built
    rng = np.random.default_rng(6)
    v, k, far = 33, 32, 1 << 25
    head = pk.Mx4Linear(rng.standard_normal((v, k)).astype(np.float32))
    x = torch.empty(far + 64, k, device="cuda")            # 4 GiB, of which three pieces are used
    parts = {0: 700, 5000: 3, 5003: 40, 12000: 9, far: 64}
    for a, n in parts.items():
        x[a:a + n] = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32)).cuda()
    u = torch.rand(far + 64, device="cuda")
    offs = np.array([12000, far, 0, 7, 5003, 5000, 40, far + 10], np.int64)
    n = np.array([9, 64, 700, 0, 40, 43, 500, 50], np.int32)
    prev = np.array([1, 2, 3, 4, 5, 6, 7, 8], np.int32)
    for kw in (dict(), dict(uniforms=u.data_ptr(), uniforms_on_device=True, temperature=0.8, top_p=0.95)):
        ctc = pk.CtcGreedy(v, 0)
        torch.cuda.synchronize()
        ctc.decode_frames(x.data_ptr(), [3], [5], head=head, on_device=True, **kw)
        free = torch.cuda.mem_get_info()[0]
        ctc.decode_frames(x.data_ptr(), [far], [64], head=head, on_device=True, **kw)
        assert free - torch.cuda.mem_get_info()[0] <= 16 << 20   # 128 MiB for the frames before it
        got, frames, after = ctc.decode_frames(x.data_ptr(), offs, n, head=head, on_device=True, prev=prev, with_frames=True, **kw)
        for i in range(len(n)):
            one = dict(kw, uniforms=u[offs[i]:].data_ptr()) if kw else {}
            t, f, p = ctc.decode_frames(x[offs[i]:].data_ptr(), [0], [n[i]], head=head, on_device=True, prev=prev[i:i + 1],
                                        with_frames=True, **one)
            assert np.array_equal(got[i], t[0]) and np.array_equal(frames[i], f[0]) and after[i] == p[0], i
        ctc.close()
    # the same utterances from host memory, logits and uniforms of a gap worth leaving out
    total = 40_000
    lg = rng.standard_normal((total, v)).astype(np.float32)
    uu = rng.random(total).astype(np.float32)
    ctc = pk.CtcGreedy(v, 0)
    o, m = np.array([39_000, 0, 20_000], np.int64), np.array([1000, 300, 77], np.int32)
    for kw in (dict(), dict(uniforms=uu, top_k=9)):
        got, _, _ = ctc.decode_frames(lg, o, m, **kw)
        for i in range(3):
            one = dict(kw, uniforms=uu[o[i]:o[i] + m[i]]) if kw else {}
            t, _, _ = ctc.decode_frames(lg[o[i]:o[i] + m[i]], [0], [m[i]], **one)
            assert np.array_equal(got[i], t[0])
    greedy, _, _ = ctc.decode(lg, o, m)
    assert all(np.array_equal(a, b) for a, b in zip(greedy, ctc.decode_frames(lg, o, m)[0]))
    with pytest.raises(pk.PkError, match="out of range"):
        ctc.decode_frames(x.data_ptr(), [1 << 62], [4], on_device=True)
    ctc.close()


def strictly(seen, u, tok, lp, **kw):
    """check(), with no way round it: where u times the kept sum lies nearer to a border between two kept tokens
    than the weights' roundings move it (each weight by 2^-44 and 2^-42 of itself, the border and the sum once
    each), the token is one of the two, and it is that token's log-probability. f32 sums are allowed for only where
    pk_sample takes them: rows with nothing cut of up to 2048 logits from 1184 rows on, and top-p without a cut by
    k for up to 16384 logits, except for few long rows (up to 296 of more than 2048) and many short ones (2960
    and more of up to 1056). Their sums are off by 58 and 66 times 2^-24 (see check), the f32 logarithm by two
    steps of itself and one of its argument."""
    kw = {**DEFAULTS, **kw}
    r, v = seen.shape
    near = 0
    for i in range(r):
        o = {n: (x[i] if np.ndim(x) else x) for n, x in kw.items()}
        temp, k, p, m = np.float64(np.float32(o["temperature"])), int(o["top_k"]), np.float64(np.float32(o["top_p"])), np.float64(np.float32(o["min_p"]))
        l = np.where(np.isnan(seen[i]), -np.inf, seen[i].astype(np.float64))
        a = (l - l.max()) / temp
        w = np.exp(a)
        w[w < 2.0 ** -44] = 0.0
        order = np.argsort(-l, kind="stable")
        s = w[order]
        if 0 < k < v:
            s[k:] = 0.0
        slack = 2 * (v * 2.0 ** -44 + s.sum() * 2.0 ** -42)
        if p < 1:
            before = np.cumsum(s) - s
            assert np.abs(before - p * s.sum())[s > 0].min() > slack       # the cut itself is never in doubt
            s = np.where((before < p * s.sum()) | (np.arange(v) == 0), s, 0.0)
        if m > 0:
            assert np.abs(s[s > 0] / m - 1).min() > 1e-12
            s = np.where(s >= m, s, 0.0)
        w = np.zeros(v)
        w[order] = s
        some = np.flatnonzero(w)
        ends = np.cumsum(w[some])
        x = float(np.float32(u[i])) * ends[-1]
        j = min(int(np.searchsorted(ends, x, side="right")), len(some) - 1)
        allowed = {int(some[j])}
        if j > 0 and x - ends[j - 1] <= slack:
            allowed.add(int(some[j - 1]))
        if j + 1 < len(some) and ends[j] - x <= slack:
            allowed.add(int(some[j + 1]))
        near += len(allowed) > 1
        assert int(tok[i]) in allowed, (i, tok[i], allowed, o, u[i])
        want = a[tok[i]] - np.log(ends[-1])
        cut = 0 < k <= int((l > l.max() - 31 * temp).sum())    # fewer than k tokens with any weight are not cut by k
        filters = 0 < k < v or p < 1 or m > 0 or any(np.ndim(x) for n, x in kw.items() if n != "temperature")
        f32 = (v <= 2048 and r >= 1184) if not filters else (
            not cut and p < 1 and v <= 16384 and not (v <= 1056 and r >= 2960) and not (r <= 296 and v > 2048))
        tol = 2.0 ** -24 * abs(want) + v * 2.0 ** -43 + 2.0 ** -40
        if f32:
            tol += 2.0 ** -24 * ((66 if filters else 58) + 1 + 2 * abs(np.log(ends[-1])) + 3 * abs(a[tok[i]]))
        assert abs(lp[i] - want) <= tol, (i, lp[i], want, tol)
    assert near <= r // 100 + 1                            # or the test says little


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.97, min_p=0.003, temperature=1.3),
                                dict(top_k=30, top_p=0.9, min_p=0.01)], ids=["plain", "T", "k", "p", "pm", "kpm"])
@pytest.mark.parametrize("r,v", [(40, 33), (40, 1025), (300, 8193), (600, 2048), (1200, 1025), (3000, 1025), (20, 40001)])
def test_tokens_strictly(built, r, v, kw):
    rng = np.random.default_rng(r + v)
    l = rng.standard_normal((r, v)) * rng.choice([0.3, 2.5], (r, 1))
    l[rng.random((r, v)) < 0.1] = -np.inf
    u = rng.random(r).astype(np.float32)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    seen, tok, lp = run(built, l, u, "f32", 1, 0, **kw)
    strictly(seen, u, tok, lp, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("r,v", [(2, 500_001), (80, 102_001), (40, 204_001)])
def test_rows_past_shared_memory(built, r, v, dtype):
    """Rows whose share of a cluster's block does not fit its shared memory are read anew in each pass."""
    rng = np.random.default_rng(v)
    l = rng.standard_normal((r, v)).astype(np.float32) * 3
    l[:, ::5] = -np.inf
    l[:, 7::1001] = np.nan
    l[-1, [5, v - 1]] = np.inf
    if r > 2:
        l[1], l[2] = -np.inf, 0.0
    u = rng.random(r).astype(np.float32)
    some = np.unique(np.concatenate([np.arange(min(r, 6)), [r - 1]]))
    for kw in (dict(), dict(temperature=0.0), dict(top_k=40), dict(top_k=5000, top_p=0.9), dict(top_p=0.95, temperature=0.8), dict(min_p=0.01)):
        seen, tok, lp = run(built, l, u, dtype, 3, 1, **kw)
        check(seen[some], u[some], tok[some], lp[some], **kw)
