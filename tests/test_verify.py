"""Verification of drafted tokens: pk_verify against its definition in f64, against pk_sample where they meet, as part
of a draft-and-verify step through the 4-bit and 8-bit heads, and its refusals."""
import ctypes as C
import subprocess
import sys

import numpy as np
import pytest

DEFAULTS = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
TYPES = ("f32", "f16", "bf16")


@pytest.fixture(scope="module")
def built(pk):
    pk.build()
    return pk


def chances(l, temperature, top_k, top_p, min_p):
    """The distribution that pk_sample draws a row's token from, by sorting and summing in f64; zeros: none."""
    l = np.asarray(l, np.float64)
    v = len(l)
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    w = np.zeros(v)
    if top == -np.inf:
        return w
    if not temperature > 0:
        w[int(np.argmax(l))] = 1.0
        return w
    fine = (l > -np.inf) & (l < top) & (top < np.inf)   # a maximum of +infinity leaves the others nothing
    with np.errstate(over="ignore", under="ignore"):
        w[fine] = np.exp((l[fine] - top) / np.float64(np.float32(temperature)))
    w[l == top] = 1.0
    order = np.argsort(-l, kind="stable")
    s = w[order]
    if top_k > 0:
        s[top_k:] = 0.0
    if not top_p >= 1:
        before = np.cumsum(s) - s
        keep = before < np.float64(np.float32(top_p)) * s.sum() if top_p > 0 else np.zeros(v, bool)
        keep[0] = True
        s = np.where(keep, s, 0.0)
    if min_p > 0:
        s = np.where(s >= min(np.float64(np.float32(min_p)), 1.0), s, 0.0)
    w = np.zeros(v)
    w[order] = s
    return w / w.sum()


def ref_verify(p_rows, q_rows, drafts, u, **kw):
    """(tokens, log-probabilities, how near a decision came to going the other way) of one sequence; the rows are its
    own: one more of the target than there are drafts."""
    kw = {**DEFAULTS, **kw}
    u = [0.0 if not x > 0 else min(float(np.float32(x)), 1 - 2.0 ** -24) for x in u]
    out, lp, near = [], [], np.inf
    n = len(drafts)
    for j in range(n + 1):
        p = rest = chances(p_rows[j], **kw)
        v = len(p)
        if j < n:
            d = int(drafts[j])
            inside = 0 <= d < v
            q = chances(q_rows[j], **kw) if q_rows is not None else np.zeros(v)
            if q_rows is None and inside:
                q[d] = 1.0
            if inside:
                near = min(near, abs(u[j] * q[d] - p[d]) if p[d] > 0 and q[d] > 0 else np.inf)
                if u[j] * q[d] < p[d]:
                    out.append(d)
                    lp.append(np.log(p[d]))
                    continue
            rest = np.maximum(p - q, 0.0)
            if not rest.sum() > 0:
                rest = p
        if rest.sum() > 0:
            run = np.cumsum(rest)
            t = min(int(np.searchsorted(run, u[-1] * run[-1], side="right")), int(np.flatnonzero(rest)[-1]))
            near = min(near, np.abs(run - u[-1] * run[-1]).min())
            out.append(t)
            lp.append(np.log(p[t]))
        else:
            out.append(-1)
            lp.append(-np.inf)
        break
    return out, lp, near


def to_device(a, dtype, pad, shift):
    """Rows [r][v] in a buffer of larger values, row stride v + pad, `shift` elements in."""
    import torch
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    r, v = a.shape
    buf = torch.full((r * (v + pad) + shift + 32,), 1e4, dtype=t, device="cuda")
    x = buf[shift:shift + r * (v + pad)].view(r, v + pad)
    x[:, :v] = torch.from_numpy(np.asarray(a, np.float32)).cuda().to(t)
    return buf, x


class Call:
    """One call's device memory: run() queues it, answer() waits and reads."""

    def __init__(self, pk, p, q, drafts, u, counts=None, dtype="f32", pad=0, shift=0, **kw):
        import torch
        self.pk = pk
        s, d1, v = p.shape
        self.s, self.d, self.v, self.pad, self.dtype = s, d1 - 1, v, pad, dtype
        self.pbuf, self.p = to_device(p.reshape(-1, v), dtype, pad, shift)
        self.q = None
        if q is not None:
            self.qbuf, self.q = to_device(np.asarray(q).reshape(-1, v), dtype, pad, shift)
        self.drafts = torch.from_numpy(np.asarray(drafts, np.int32).reshape(s, -1).copy()).cuda()
        self.u = torch.from_numpy(np.asarray(u, np.float32).copy()).cuda()
        self.counts = None if counts is None else torch.from_numpy(np.asarray(counts, np.int32)).cuda()
        self.tok = torch.full((s * d1 + 8,), -7, dtype=torch.int32, device="cuda")
        self.acc = torch.full((s + 8,), -7, dtype=torch.int32, device="cuda")
        self.lp = torch.full((s * d1 + 8,), 123.0, device="cuda")
        need = pk.verify_workspace(s, self.d, v)
        self.ws = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        self.args, self.keep = {}, []
        for name, val in kw.items():
            if np.ndim(val):
                t = torch.from_numpy(np.asarray(val, np.int32 if name == "top_k" else np.float32)).cuda()
                self.keep.append(t)
                self.args[name + "s"] = t.data_ptr()
            else:
                self.args[name] = val

    def run(self, stream=None):
        import torch
        s = torch.cuda.current_stream().cuda_stream if stream is None else stream
        self.pk.verify(self.p.data_ptr(), self.s, self.d, self.v, self.drafts.data_ptr(), self.u.data_ptr(), self.tok.data_ptr(),
                       self.acc.data_ptr(), draft_logits=0 if self.q is None else self.q.data_ptr(),
                       n_drafts=0 if self.counts is None else self.counts.data_ptr(), dtype=self.dtype,
                       row_stride=self.v + self.pad, draft_stride=self.v + self.pad, logprobs=self.lp.data_ptr(),
                       workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel() - 64, stream=s, **self.args)
        return self

    def answer(self):
        import torch
        torch.cuda.synchronize()
        n = self.s * (self.d + 1)
        assert (self.tok[n:] == -7).all() and (self.lp[n:] == 123.0).all() and (self.acc[self.s:] == -7).all()
        assert (self.ws[-64:] == 0xA5).all()
        return (self.tok[:n].view(self.s, -1).cpu().numpy(), self.acc[:self.s].cpu().numpy(), self.lp[:n].view(self.s, -1).cpu().numpy())

    def seen(self):
        def rows(x, per):
            return x[:, :self.v].float().cpu().numpy().reshape(self.s, per, self.v)
        return rows(self.p, self.d + 1), None if self.q is None else rows(self.q, self.d)


def check(call, drafts, u, counts=None, excused=0, **kw):
    """Tokens and counts equal. Weights are rounded to 2^-43 of the largest one by one, which moves a distribution's
    sums by v 2^-43 at most, the difference of two by twice that, its product with u by as much again; nearer than
    (v + 4) 2^-41 to a border the definition's other answer is the fixed point's. At most `excused` sequences may be.
    Log-probabilities, in units of 2^-24: (l - l_0) / T by f32's 1 / T and log2(e), three roundings, and rounded once; the
    logarithm of a sum of f32 weights, off by 8 for each exponential, 2.78 for each unit of its argument (log2 V and
    24 at most on average) and the additions (v / 512 and 24), to f32 (one, and 16 for a logarithm below 17); or of a
    sum off by v 2^-43."""
    tok, acc, lp = call.answer()
    p, q = call.seen()
    near_ones = 0
    for i in range(call.s):
        one = {n: (x[i] if np.ndim(x) else x) for n, x in kw.items()}
        n = call.d if counts is None else max(0, min(int(counts[i]), call.d))
        want, wlp, near = ref_verify(p[i, :n + 1], None if q is None else q[i, :n], drafts[i][:n], u[i], **one)
        full = want + [-1] * (call.d + 1 - len(want))
        if tok[i].tolist() != full or acc[i] != len(want) - 1:
            near_ones += 1
            assert near <= (call.v + 4) * 2.0 ** -41, (i, tok[i], full, acc[i], near, one)
            continue
        for j, x in enumerate(wlp):
            if np.isinf(x):
                assert lp[i, j] == x
            else:
                tol = 2.0 ** -24 * (5 * abs(x) + 8 + 2.78 * (np.log2(call.v) + 24) + call.v / 512 + 24 + 17) + call.v * 2.0 ** -43
                assert abs(lp[i, j] - x) <= tol, (i, j, lp[i, j], x)
        assert np.isneginf(lp[i, len(want):]).all()
    assert near_ones <= excused


def make(rng, s, d, v, spread=2.0, gap=0.7, dtype="f32", certain=False, **kw):
    """Rows of a target, rows of a draft that sees it less well, and drafts drawn from the latter."""
    p = rng.standard_normal((s, d + 1, v)) * spread
    p[..., -1] += 3 * spread * rng.random((s, d + 1))
    q = p[:, :d] + gap * rng.standard_normal((s, d, v))
    kw = {**DEFAULTS, **{n: x for n, x in kw.items() if not np.ndim(x)}}
    drafts = np.zeros((s, d), np.int32)
    for i in range(s):
        for j in range(d):
            c = chances(q[i, j].astype(np.float32), **kw)
            drafts[i, j] = int(np.argmax(q[i, j])) if certain else min(int(np.searchsorted(np.cumsum(c), rng.random(), side="right")), v - 1)
    return p, None if certain else q, drafts, rng.random((s, d + 1)).astype(np.float32)


# ---- CPU -----------------------------------------------------------------------

def test_reference_known_answers():
    p = np.log(np.array([[0.5, 0.25, 0.25], [0.2, 0.3, 0.5]]))
    q = np.log(np.array([[0.25, 0.5, 0.25]]))
    assert ref_verify(p, q, [1], [0.49, 0.6])[0] == [1, 2]                # 0.49 < 0.5: accepted, then 0.2 + 0.3 <= 0.6
    assert ref_verify(p, q, [1], [0.51, 0.99])[0] == [0]                  # only token 0 has more in p
    assert ref_verify(p, q, [0], [0.999, 0.1])[0] == [0, 0]               # q below p: always
    assert ref_verify(p, None, [0], [0.51, 0.4])[0] == [1]
    assert ref_verify(p, q, [7], [0.0, 0.4])[0] == [0]
    assert ref_verify(p, p[:1], [-1], [0.0, 0.6])[0] == [1]               # nothing left over: from p
    assert ref_verify(p, q, [0], [0.9, 0.9], temperature=0.0)[0] == [0, 2]
    assert ref_verify(np.full((2, 3), -np.inf), q, [0], [0.0, 0.9])[0] == [-1]


def test_refusals(built):
    pk, L, abi = built, built.lib(), built.abi
    g = 1 << 20                                         # never read

    def call(device=99, **kw):
        d = dict(logits=g, draft_logits=g, logits_type=0, vocab=30000, sequences=3, max_drafts=4, reserved=0, row_stride=30000, draft_stride=30000,
                 drafts=g, n_drafts=g, uniforms=g, tokens=g, accepted=g, logprobs=g, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 temperatures=None, top_ks=None, top_ps=None, min_ps=None, workspace=g, workspace_bytes=1 << 20)
        d.update(kw)
        return L.pk_verify(device, C.byref(abi.pk_verify_args(*d.values())), None)

    assert call() == abi.PK_ERR_NO_DEVICE
    for kw in (dict(logits_type=8), dict(vocab=0), dict(vocab=abi.PK_SAMPLE_MAX_VOCAB + 1), dict(sequences=-1), dict(sequences=1 << 40),
               dict(max_drafts=-1), dict(max_drafts=65536), dict(row_stride=29999), dict(row_stride=1 << 40), dict(draft_stride=29999),
               dict(draft_stride=1 << 40), dict(logits=None), dict(drafts=None), dict(uniforms=None), dict(tokens=None), dict(accepted=None),
               dict(workspace=None), dict(workspace_bytes=pk.verify_workspace(3, 4, 30000) - 1), dict(logits=g + 2), dict(draft_logits=g + 2),
               dict(drafts=g + 1), dict(n_drafts=g + 2), dict(uniforms=g + 2), dict(tokens=g + 2), dict(accepted=g + 2), dict(logprobs=g + 1),
               dict(temperatures=g + 1), dict(top_ks=g + 2), dict(top_ps=g + 1), dict(min_ps=g + 2), dict(workspace=g + 4)):
        assert call(**kw) == abi.PK_ERR_INVALID, kw
        assert b"pk_verify" in L.pk_last_error()
    assert call(draft_logits=None, draft_stride=0, n_drafts=None, logprobs=None) == abi.PK_ERR_NO_DEVICE
    assert call(max_drafts=0, drafts=None) == abi.PK_ERR_NO_DEVICE
    assert call(sequences=0, logits=None, tokens=None, workspace=None, workspace_bytes=0) == abi.PK_ERR_NO_DEVICE
    assert L.pk_verify(0, None, None) == abi.PK_ERR_INVALID
    assert call(vocab=1000, workspace=None, workspace_bytes=0) == abi.PK_ERR_NO_DEVICE
    assert pk.verify_workspace(0, 0, 1) == 0 and pk.verify_workspace(2, 3, 10) == 0 and pk.verify_workspace(2, 3, 30000) > 0
    for bad in ((-1, 1, 10), (1, -1, 10), (1, 65536, 10), (1, 1, 0), (1, 1, 1 << 20), (1 << 28, 1, 10)):
        assert pk.verify_workspace(*bad) == -1
    for kw in (dict(vocab=0), dict(max_drafts=-1)):
        with pytest.raises(ValueError):
            pk.verify(**{**dict(logits=g, sequences=1, max_drafts=1, vocab=5, drafts=g, uniforms=g, tokens=g, accepted=g), **kw})


# ---- GPU -----------------------------------------------------------------------

SETTINGS = [{}, dict(temperature=0.7, top_k=20), dict(top_p=0.9), dict(temperature=1.3, top_k=50, top_p=0.95, min_p=0.01), dict(min_p=0.05),
            dict(temperature=0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS)
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("s,d,v", [(1, 1, 1), (3, 2, 7), (5, 4, 33), (40, 3, 257), (9, 5, 1025), (2, 4, 8193)])
def test_matches_definition(built, s, d, v, certain, kw):
    p, q, drafts, u = make(np.random.default_rng(s * v + d), s, d, v, certain=certain, **kw)
    check(Call(built, p, q, drafts, u, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(top_p=0.9), dict(top_k=64, top_p=0.95)])
@pytest.mark.parametrize("s,d,v", [(450, 3, 300), (700, 2, 1050), (200, 3, 1600), (130, 2, 2100), (70, 2, 6000), (170, 2, 5000)])
def test_either_side_of_each_team(built, s, d, v, kw):
    """As many rows as each of the row kernels takes."""
    p, q, drafts, u = make(np.random.default_rng(s), s, d, v, **kw)
    check(Call(built, p, q, drafts, u, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 1, 1), ("f32", 4, 2), ("f16", 0, 0), ("f16", 3, 5), ("bf16", 0, 0), ("bf16", 1, 7)])
@pytest.mark.parametrize("v", [65, 1030, 8193])
def test_types_and_strides(built, v, dtype, pad, shift):
    for kw in ({}, dict(temperature=0.8, top_p=0.9)):
        p, q, drafts, u = make(np.random.default_rng(v), 6, 3, v, **kw)
        check(Call(built, p, q, drafts, u, dtype=dtype, pad=pad, shift=shift, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("s,d,v", [(1, 2, 20000), (3, 1, 131072), (40, 1, 30001), (1, 1, 524288)])
@pytest.mark.parametrize("kw", [dict(temperature=0.9), dict(temperature=0.6, top_p=0.9), dict(top_k=700)])
def test_large_vocabularies(built, s, d, v, kw):
    p, q, drafts, u = make(np.random.default_rng(v), s, d, v, spread=2.5, gap=0.4, **kw)
    check(Call(built, p, q, drafts, u, dtype="bf16", **kw).run(), drafts, u, excused=1, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("s,d,v", [(64, 4, 500), (30, 6, 8193), (12, 3, 30000)])
def test_settings_and_counts_of_each_sequence(built, s, d, v, certain):
    """Settings, numbers of drafts (out of range among them) and masks by sequence; what lies behind the drafts is
    not read, nor are the drafts behind the first rejection needed."""
    rng = np.random.default_rng(v)
    kw = dict(temperature=np.where(rng.random(s) < 0.15, 0.0, 0.3 + 1.2 * rng.random(s)), top_k=np.where(rng.random(s) < 0.4, 0, rng.integers(1, 100, s)),
              top_p=np.where(rng.random(s) < 0.4, 1.0, 0.4 + 0.6 * rng.random(s)), min_p=np.where(rng.random(s) < 0.6, 0.0, 0.1 * rng.random(s)))
    p, q, drafts, u = make(rng, s, d, v, certain=certain)
    mask = rng.random((s, 1, v)) < 0.3
    mask[rng.random(s) < 0.1] = True
    p = np.where(mask, -np.inf, p)
    q = None if certain else np.where(mask, -np.inf, q)
    counts = rng.integers(-2, d + 3, s)
    drafts[rng.random((s, d)) < 0.1] = -1
    for i in range(s):
        n = max(0, min(int(counts[i]), d))
        p[i, n + 1:] = np.nan
        drafts[i, n:] = 1 << 30
        if not certain:
            q[i, n:] = np.inf
    check(Call(built, p, q, drafts, u, counts=counts, **kw).run(), drafts, u, counts, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS)
@pytest.mark.parametrize("v", [40, 1500, 9000, 30000])
def test_special_values(built, v, kw):
    """Infinities, NaN and rows without any logit, in the target and in the draft; drafts that no one drew."""
    rng = np.random.default_rng(v)
    s, d = 24, 2
    p, q, drafts, u = make(rng, s, d, v, **kw)
    p[0, 0], q[1, 0], p[2, 2] = -np.inf, -np.inf, -np.inf
    p[3, 0, 5] = np.inf
    q[4, 0, 7] = np.inf
    p[5, 0, [3, 9]], q[5, 0, [9, 11]] = np.inf, np.inf
    p[6, 0, 4], q[6, 0, 5] = np.nan, np.nan
    p[7, 0], q[7, 0] = np.nan, np.nan
    p[8], q[8] = np.finfo(np.float32).min, np.finfo(np.float32).min          # a mask of the type's lowest value
    p[9, :, : v - 1], q[9, :, : v - 1] = np.finfo(np.float32).min, np.finfo(np.float32).min
    drafts[10], drafts[11], drafts[12] = -1, v, np.iinfo(np.int32).max
    drafts[13], drafts[14] = np.iinfo(np.int32).min, [v - 1, -1]
    q[15] = p[15, :d]                                                        # equal rows: accepted whatever u
    u[15] = 1 - 2.0 ** -24
    q[16, 0], drafts[16] = p[16, 0], -1                                       # and a draft that neither has
    p[17, 0], q[17, 0] = 1.0, 1.0
    u[18], u[19], u[20], u[21] = np.nan, 2.0, -1.0, 1.0
    p[22, 0, 0], drafts[22, 0] = 1e30, 0
    p[23] *= 1e-30
    check(Call(built, p, q, drafts, u, **kw).run(), drafts, u, **kw)
    check(Call(built, p, None, drafts, u, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(top_k=5), dict(top_p=0.5), dict(top_k=300, top_p=0.7)])
@pytest.mark.parametrize("v", [60, 2000, 9000])
def test_cut_inside_equal_logits(built, v, kw):
    """Cuts among equal logits, which go by index: drafts on either side of them, residues of parted ties."""
    rng = np.random.default_rng(v)
    s, d = 40, 1
    p = np.round(rng.standard_normal((s, d + 1, v)))
    p[::2] = 0.0
    q = np.round(p[:, :d] + 0.6 * rng.standard_normal((s, d, v)))
    drafts = rng.integers(0, v, (s, d))
    drafts[::4, 0] = rng.integers(0, 8, len(drafts[::4]))
    drafts[1::4, 0] = p[1::4, 0].argmax(1)
    u = rng.random((s, d + 1)).astype(np.float32)
    check(Call(built, p, q, drafts, u, **kw).run(), drafts, u, **kw)
    check(Call(built, p, None, drafts, u, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.001)])
@pytest.mark.parametrize("s,v", [(3, 8193), (2000, 1025), (2, 131072), (200, 24000)])
def test_without_drafts_it_is_sample(built, s, v, kw):
    import torch
    rng = np.random.default_rng(s)
    p, _, _, u = make(rng, s, 0, v)
    call = Call(built, p, None, np.zeros((s, 0)), u, **kw).run()
    tok, acc, lp = call.answer()
    t2, l2 = torch.zeros(s, dtype=torch.int32, device="cuda"), torch.zeros(s, device="cuda")
    built.sample(call.p.data_ptr(), s, v, call.u.data_ptr(), t2.data_ptr(), logprobs=l2.data_ptr(), **kw)
    assert (acc == 0).all() and np.array_equal(tok[:, 0], t2.cpu().numpy())
    assert np.abs(lp[:, 0] - l2.cpu().numpy()).max() <= 2.0 ** -16      # each within 2^-17 of its value


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(temperature=0.9, top_k=9)])
def test_tokens_are_distributed_as_the_target(built, kw):
    """Drafts drawn by pk_sample from one row, verified against another, 200,000 times: the first token comes as often
    as the target's row says, and as often is the draft accepted as the two rows overlap, within six deviations."""
    import torch
    pk, n, v = built, 200_000, 12
    g = torch.Generator(device="cuda").manual_seed(5)
    p0, q0 = torch.randn(v, generator=g, device="cuda") * 1.5, torch.randn(v, generator=g, device="cuda") * 1.5
    p, q = p0.expand(n, 2, v).contiguous(), q0.expand(n, 1, v).contiguous()
    u0, u = torch.rand(n, generator=g, device="cuda"), torch.rand(n, 2, generator=g, device="cuda")
    drafts, tok = torch.zeros(n, 1, dtype=torch.int32, device="cuda"), torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    acc, ws = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(pk.verify_workspace(n, 1, v), dtype=torch.uint8, device="cuda")
    pk.sample(q.data_ptr(), n, v, u0.data_ptr(), drafts.data_ptr(), **kw)
    pk.verify(p.data_ptr(), n, 1, v, drafts.data_ptr(), u.data_ptr(), tok.data_ptr(), acc.data_ptr(), draft_logits=q.data_ptr(),
              workspace=ws.data_ptr(), workspace_bytes=ws.numel(), **kw)
    cp, cq = (chances(x.cpu().numpy(), **{**DEFAULTS, **kw}) for x in (p0, q0))
    freq = np.bincount(tok[:, 0].cpu().numpy(), minlength=v) / n
    assert (np.abs(freq - cp) <= 6 * np.sqrt(cp * (1 - cp) / n)).all()
    both = np.minimum(cp, cq).sum()
    assert abs(acc.float().mean().item() - both) <= 6 * np.sqrt(both * (1 - both) / n)
    second = tok[:, 1][acc == 1].cpu().numpy()            # the row behind is drawn from whenever the draft stands
    freq = np.bincount(second, minlength=v) / len(second)
    assert (np.abs(freq - cp) <= 6 * np.sqrt(cp * (1 - cp) / len(second))).all()
    assert (tok[:, 1][acc == 0] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("s,d,v", [(64, 4, 500), (30, 6, 8193), (12, 3, 30000)])
def test_temperatures_and_counts_without_filters(built, s, d, v):
    """Temperatures, numbers of drafts and masks by sequence, with nothing else to cut."""
    rng = np.random.default_rng(v + 1)
    kw = dict(temperature=np.where(rng.random(s) < 0.15, 0.0, 0.3 + 1.2 * rng.random(s)))
    p, q, drafts, u = make(rng, s, d, v)
    mask = rng.random((s, 1, v)) < 0.3
    mask[rng.random(s) < 0.1] = True
    p, q = np.where(mask, -np.inf, p), np.where(mask, -np.inf, q)
    counts = rng.integers(-2, d + 3, s)
    drafts[rng.random((s, d)) < 0.1] = -1
    u[:, :d] *= rng.random((s, 1))                        # many accepted
    for i in range(s):
        n = max(0, min(int(counts[i]), d))
        p[i, n + 1:], q[i, n:], drafts[i, n:] = np.nan, np.inf, 1 << 30
    check(Call(built, p, q, drafts, u, counts=counts, **kw).run(), drafts, u, counts, **kw)
    check(Call(built, p, None, drafts, u, counts=counts, **kw).run(), drafts, u, counts, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [np.inf, 1e30, 300.0, 1e-3, 1e-20, 1e-38, -1.0, np.nan])
@pytest.mark.parametrize("kw", [{}, dict(top_p=0.9), dict(min_p=0.3)])
def test_extreme_temperatures(built, temperature, kw):
    rng = np.random.default_rng(6)
    for s, d, v in ((5, 2, 300), (2, 2, 7000)):
        p, q, drafts, u = make(rng, s, d, v, gap=0.3)
        if temperature > 100:                            # equal weights: any cut falls among them, by the logits' order
            drafts = rng.integers(0, v, (s, d)).astype(np.int32)
        # A lead of g of the largest logit leaves the others exp(-g / T): at T = 0.001 a lead of 0.031 puts them below 2^-44, and
        # where both rows have the same largest logit p - q is below 2^-43 throughout, which the definition lets be lost. Such
        # a sequence lies within check()'s bound of a border and may get p's token instead.
        excused = s if temperature < 0.01 else 0
        check(Call(built, p, q, drafts, u, temperature=temperature, **kw).run(), drafts, u, excused=excused, temperature=temperature, **kw)
        check(Call(built, p, None, drafts, u, temperature=temperature, **kw).run(), drafts, u, temperature=temperature, **kw)


@pytest.mark.gpu
def test_many_drafts(built):
    """More drafts than a block has threads, most of them accepted."""
    rng = np.random.default_rng(2)
    p, q, drafts, u = make(rng, 2, 1300, 9, gap=0.01)
    u[:, :1290] *= 0.9
    check(Call(built, p, q, drafts, u).run(), drafts, u)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(temperature=0.8, top_p=0.9), dict(temperature=0.8)])
@pytest.mark.parametrize("v", [500, 8193, 40000])
def test_captured_and_replayed(built, v, kw):
    """Two graphs with workspaces of their own replayed on two streams, with new inputs each time."""
    import torch
    rng = np.random.default_rng(v)
    first = [make(rng, 4, 3, v, **kw) for _ in range(2)]
    calls = [Call(built, *x, **kw) for x in first]
    graphs, streams = [torch.cuda.CUDAGraph() for _ in calls], [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for c, g in zip(calls, graphs):
        with torch.cuda.graph(g):
            c.run()
    for _ in range(3):
        new = [make(rng, 4, 3, v, **kw) for _ in calls]
        for c, (p, q, drafts, u) in zip(calls, new):
            c.p[:, :v] = torch.from_numpy(p.reshape(-1, v).astype(np.float32)).cuda()
            c.q[:, :v] = torch.from_numpy(q.reshape(-1, v).astype(np.float32)).cuda()
            c.drafts.copy_(torch.from_numpy(drafts))
            c.u.copy_(torch.from_numpy(u))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for c, (_, _, drafts, u) in zip(calls, new):
            check(c, drafts, u, **kw)


@pytest.mark.gpu
def test_no_sequences_and_the_same_answer_again(built):
    """No sequences: nothing happens. Equal calls give equal bits, alone or among other sequences."""
    import torch
    pk = built
    pk.verify(0, 0, 3, 50, 0, 0, 0, 0)
    rng = np.random.default_rng(1)
    p, q, drafts, u = make(rng, 300, 3, 1200)
    a = Call(pk, p, q, drafts, u, top_p=0.9).run().answer()
    b = Call(pk, p, q, drafts, u, top_p=0.9).run().answer()
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    c = Call(pk, p[:5], q[:5], drafts[:5], u[:5], top_p=0.9).run().answer()
    assert np.array_equal(a[0][:5], c[0]) and np.array_equal(a[1][:5], c[1])
    assert torch.cuda.current_device() == 0


@pytest.mark.gpu
def test_first_call_may_be_captured(built):
    code = """
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("parakeet_b200", sys.argv[1] + "/__init__.py", submodule_search_locations=[sys.argv[1]])
pk = importlib.util.module_from_spec(spec); sys.modules["parakeet_b200"] = pk; spec.loader.exec_module(pk)
p, q = torch.randn(5, 4, 9000, device="cuda"), torch.randn(5, 3, 9000, device="cuda")
d = torch.randint(0, 9000, (5, 3), dtype=torch.int32, device="cuda"); u = torch.rand(5, 4, device="cuda")
tok = torch.full((5, 4), -5, dtype=torch.int32, device="cuda"); acc = torch.full((5,), -5, dtype=torch.int32, device="cuda")
ws = torch.empty(pk.verify_workspace(5, 3, 9000), dtype=torch.uint8, device="cuda")
def run(s):
    pk.verify(p.data_ptr(), 5, 3, 9000, d.data_ptr(), u.data_ptr(), tok.data_ptr(), acc.data_ptr(), draft_logits=q.data_ptr(), top_p=0.9,
              workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=s)
g = torch.cuda.CUDAGraph(); torch.cuda.synchronize()
with torch.cuda.graph(g):
    run(torch.cuda.current_stream().cuda_stream)
g.replay(); torch.cuda.synchronize()
a, b = tok.clone(), acc.clone()
run(0); torch.cuda.synchronize()
assert torch.equal(a, tok) and torch.equal(b, acc) and (tok[:, 0] >= 0).all() and (acc >= 0).all()
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code, built.PKG_DIR], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(temperature=1.0), dict(temperature=0.7, top_k=30, top_p=0.9)])
def test_draft_and_verify_through_both_heads(built, kw):
    """As they are used: hidden rows through the 4-bit head draft tokens, the same rows through the 8-bit head are the
    target, and what comes out agrees with the definition on the logits that both computed."""
    import torch
    pk, rng = built, np.random.default_rng(8)
    s, d, k, v = 16, 3, 640, 1025
    w = rng.standard_normal((v, k)).astype(np.float32) * 0.06
    cheap, good = pk.Mx4Linear(w), pk.Fp8Linear(w)
    h = torch.from_numpy(rng.standard_normal((s, d + 1, k)).astype(np.float32)).cuda()
    hd = h[:, :d].contiguous()
    st = torch.cuda.Stream()
    u0, u = torch.rand(s * d, device="cuda"), torch.rand(s, d + 1, device="cuda")
    q, p = torch.zeros(s, d, v, device="cuda"), torch.zeros(s, d + 1, v, device="cuda")
    drafts, tok = torch.zeros(s, d, dtype=torch.int32, device="cuda"), torch.zeros(s, d + 1, dtype=torch.int32, device="cuda")
    acc, lp = torch.zeros(s, dtype=torch.int32, device="cuda"), torch.zeros(s, d + 1, device="cuda")
    w4 = torch.zeros(max(1, cheap.workspace(s * d)), dtype=torch.uint8, device="cuda")
    w8 = torch.zeros(max(1, good.workspace(s * (d + 1))), dtype=torch.uint8, device="cuda")
    wv = torch.zeros(pk.verify_workspace(s, d, v), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    cs = st.cuda_stream
    cheap.forward(hd.data_ptr(), s * d, q.data_ptr(), workspace=w4.data_ptr(), workspace_bytes=w4.numel(), stream=cs)
    pk.sample(q.data_ptr(), s * d, v, u0.data_ptr(), drafts.data_ptr(), stream=cs, **kw)
    good.forward(h.data_ptr(), s * (d + 1), p.data_ptr(), workspace=w8.data_ptr(), workspace_bytes=w8.numel(), stream=cs)
    pk.verify(p.data_ptr(), s, d, v, drafts.data_ptr(), u.data_ptr(), tok.data_ptr(), acc.data_ptr(), draft_logits=q.data_ptr(),
              logprobs=lp.data_ptr(), workspace=wv.data_ptr(), workspace_bytes=wv.numel(), stream=cs, **kw)
    torch.cuda.synchronize()
    full = h.cpu().numpy().reshape(-1, k).astype(np.float64) @ w.T.astype(np.float64)
    # both heads are the layer, rounded: 8 bits move a logit by some 2^-4 sqrt(2 / 3) of its deviation, 4 bits by more
    assert np.abs(p.cpu().numpy().reshape(-1, v) - full).std() < 0.08 * full.std()
    for i in range(s):
        want, wlp, near = ref_verify(p[i].cpu().numpy(), q[i].cpu().numpy(), drafts[i].tolist(), u[i].tolist(), **kw)
        assert tok[i].tolist() == want + [-1] * (d + 1 - len(want)) or near <= (v + 4) * 2.0 ** -41
        assert acc[i] == len(want) - 1 or near <= (v + 4) * 2.0 ** -41
    assert 0 < acc.sum() and (acc < d).any()


# Rows too long for a block's shared memory: one of up to 45056 logits fits, or two of 22528. v is above both.

@pytest.mark.gpu
@pytest.mark.parametrize("certain", [True, False])
@pytest.mark.parametrize("kw", [dict(temperature=0.0), dict(temperature=-1.0, top_p=0.9), dict(temperature=np.nan, top_k=5)])
@pytest.mark.parametrize("v", [45057, 131072])
def test_greedy_long_rows(built, v, kw, certain):
    """T <= 0: the first of the largest alone is kept, so its log-probability is 0 whatever draft was rejected for it, one just
    below the largest, a later one as large or a second +infinity among them."""
    rng = np.random.default_rng(v)
    s, d = 8, 2
    p, q, drafts, u = make(rng, s, d, v, certain=certain, **kw)
    top = p.argmax(2)
    for i, off in enumerate((0.5, 0.01, 20.0)):
        drafts[i, 0] = (top[i, 0] + 7) % v
        p[i, 0, drafts[i, 0]] = p[i, 0, top[i, 0]] - off
    p[3, 0, [11, 40]], drafts[3, 0] = 50.0, 40                   # a later one of the largest
    p[4, 0, [9, 30, v - 1]], drafts[4, 0] = np.inf, v - 1        # a second +infinity
    drafts[5, :], drafts[6, 0], drafts[6, 1] = top[5, :d], top[6, 0], (top[6, 1] + 1) % v
    p[7, 0], drafts[7] = 0.0, [v // 2, 0]                        # all alike
    call = Call(built, p, q, drafts, u, **kw).run()
    check(call, drafts, u, **kw)
    tok, acc, lp = call.answer()
    assert (lp[np.arange(s), acc] == 0).all()
    if certain:
        assert acc.tolist()[:5] == [0] * 5 and acc[5] == 2 and acc[6] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(temperature=0.6), dict(temperature=0.7, top_k=20), dict(top_p=0.9), dict(temperature=1.3, top_k=50, top_p=0.95, min_p=0.01)])
@pytest.mark.parametrize("s,d,v,dtype", [(3, 3, 50001, "f32"), (1, 8, 131072, "bf16"), (80, 1, 45057, "f16"), (200, 1, 45057, "f32"), (2, 1, 524288, "f32")])
def test_long_rows_with_drafts_that_were_looked_up(built, s, d, v, dtype, kw):
    p, q, drafts, u = make(np.random.default_rng(v + s), s, d, v, certain=True, **kw)
    drafts[::3, 0] = (drafts[::3, 0] + 1) % v                    # unlikely ones among them
    check(Call(built, p, q, drafts, u, dtype=dtype, **kw).run(), drafts, u, excused=1, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("certain", [True, False])
@pytest.mark.parametrize("filters", [False, True])
def test_long_rows_with_settings_and_counts_of_each_sequence(built, filters, certain):
    """As for short rows: settings (greedy ones among them), numbers of drafts and masks by sequence, drafts out of range."""
    rng = np.random.default_rng(4)
    s, d, v = 20, 3, 46001
    kw = dict(temperature=np.where(rng.random(s) < 0.3, 0.0, 0.3 + 1.2 * rng.random(s)))
    if filters:
        kw.update(top_k=np.where(rng.random(s) < 0.4, 0, rng.integers(1, 100, s)), top_p=np.where(rng.random(s) < 0.4, 1.0, 0.4 + 0.6 * rng.random(s)),
                  min_p=np.where(rng.random(s) < 0.6, 0.0, 0.1 * rng.random(s)))
    p, q, drafts, u = make(rng, s, d, v, certain=certain)
    mask = rng.random((s, 1, v)) < 0.3
    mask[[4, 9]] = True
    p = np.where(mask, -np.inf, p)
    q = None if certain else np.where(mask, -np.inf, q)
    counts = rng.integers(-2, d + 3, s)
    drafts[rng.random((s, d)) < 0.1] = -1
    for i in range(s):
        n = max(0, min(int(counts[i]), d))
        p[i, n + 1:], drafts[i, n:] = np.nan, 1 << 30
        if not certain:
            q[i, n:] = np.inf
    check(Call(built, p, q, drafts, u, counts=counts, pad=3, shift=1, **kw).run(), drafts, u, counts, excused=1, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS)
def test_long_rows_with_special_values(built, kw):
    """Infinities, NaN, rows without any logit, equal logits and drafts that no one drew."""
    v, s, d = 45601, 18, 2
    rng = np.random.default_rng(v)
    p, q, drafts, u = make(rng, s, d, v, **kw)
    p[0, 0], q[1, 0], p[2, 2] = -np.inf, -np.inf, -np.inf
    p[3, 0, 5], p[5, 0, [3, 9]] = np.inf, np.inf
    q[4, 0, 7], q[5, 0, [9, 11]] = np.inf, np.inf
    p[6, 0, 4], q[6, 0, 5] = np.nan, np.nan
    p[7, 0], q[7, 0] = np.nan, np.nan
    p[8], q[8] = np.finfo(np.float32).min, np.finfo(np.float32).min
    p[9, :, : v - 1], q[9, :, : v - 1] = np.finfo(np.float32).min, np.finfo(np.float32).min
    drafts[10], drafts[11], drafts[12], drafts[13] = -1, v, np.iinfo(np.int32).max, np.iinfo(np.int32).min
    q[14] = p[14, :d]
    u[14], u[15], u[16] = 1 - 2.0 ** -24, np.nan, 2.0
    p[17] = np.round(p[17])                                              # cuts among equal logits
    drafts[3, 0], drafts[5, 0] = 7, 9
    check(Call(built, p, q, drafts, u, **kw).run(), drafts, u, excused=1, **kw)
    check(Call(built, p, None, drafts, u, **kw).run(), drafts, u, excused=1, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("certain", [True, False])
@pytest.mark.parametrize("temperature", [1e-2, 1e-3, 1e-20, 1e-38, 0.0, -1.0, np.nan])
@pytest.mark.parametrize("kw", [{}, dict(top_p=0.9), dict(min_p=0.3)])
def test_drafts_of_low_temperatures(built, temperature, kw, certain):
    """Drafts drawn at the temperature that they are verified with: no answer needs the excuse of a border."""
    rng = np.random.default_rng(9)
    kw = dict(kw, temperature=temperature)
    for s, d, v in ((6, 3, 300), (3, 2, 7000), (2, 2, 46000)):
        p, q, drafts, u = make(rng, s, d, v, gap=0.3, certain=certain, **kw)
        check(Call(built, p, q, drafts, u, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(top_k=11), dict(top_k=700), dict(top_k=11, min_p=1e-25), dict(top_k=60, top_p=0.99999)])
@pytest.mark.parametrize("v", [24, 1030, 1500, 9000, 30000, 46001])
def test_drafts_below_all_weight(built, v, kw):
    """At a low temperature fewer than k tokens weigh as much as 2^-44 of the largest. A draft below them is kept or cut by
    its rank all the same: with equal rows in the target and the draft it is accepted if it is among the first k, and
    rejected if not."""
    rng = np.random.default_rng(v)
    s, d = 12, 2
    kw = dict(kw, temperature=0.05)
    p = rng.standard_normal((s, d + 1, v)) * 2
    p[::3] = np.round(p[::3])                                    # ties, which go by index
    q = p[:, :d].copy()
    ranks = rng.integers(0, v, (s, d))
    k = min(kw["top_k"], v - 1)
    ranks[:4, 0], ranks[4:8, 0], ranks[8, 0] = rng.integers(0, k, 4), rng.integers(k, v, 4), k
    order = np.argsort(-p.astype(np.float32), axis=2, kind="stable")
    drafts = np.array([[order[i, j, ranks[i, j]] for j in range(d)] for i in range(s)], np.int32)
    u = rng.random((s, d + 1)).astype(np.float32)
    call = Call(built, p, q, drafts, u, **kw).run()
    check(call, drafts, u, **kw)
    _, acc, _ = call.answer()
    assert ((acc > 0) <= (ranks[:, 0] < kw["top_k"])).all()
    check(Call(built, p, None, drafts, u, **kw).run(), drafts, u, **kw)
    u[:, :d] = 0.0                                               # 0 q(d) < p(d): accepted wherever the target keeps it
    check(Call(built, p, None, drafts, u, **kw).run(), drafts, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(top_k=1), dict(top_k=1, top_p=0.9, min_p=0.05), dict(top_p=0.5), dict(min_p=0.5), dict(top_k=500, top_p=0.5, min_p=0.05), {}])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("s,v", [(5, 300), (700, 300), (6, 1500), (5, 9000), (40, 7000), (3, 18000), (3, 46001)])
def test_certain_tokens_have_probability_one(built, s, v, certain, kw):
    """Rows of which one token is all that is left, by the filters or by its lead (60, in units of T): its log-probability is
    0, accepted or drawn, and no log-probability is above."""
    rng = np.random.default_rng(v + s)
    d = 2
    p = rng.standard_normal((s, d + 1, v)) * 3 + rng.uniform(-40, 40, (s, d + 1, 1))
    top = rng.integers(0, v, (s, d + 1))
    for i in range(s):
        for j in range(d + 1):
            p[i, j, top[i, j]] = p[i, j].max() + 60 * 0.7
    q = None if certain else p[:, :d] + 0.3 * rng.standard_normal((s, d, v))
    drafts = top[:, :d].astype(np.int32).copy()
    drafts[::3, 1] = (drafts[::3, 1] + 1) % v
    u = rng.random((s, d + 1)).astype(np.float32)
    kw = dict(kw, temperature=0.7)
    call = Call(built, p, q, drafts, u, **kw).run()
    # Nothing cut: a second draft has e^-60 or less in both rows, and may stand. Where it is rejected, p - q is at most
    # 2 v e^-60 < 2^-66 in all, below the 2^-43 that may be lost, and the token may come from p.
    nothing_cut = not certain and len(kw) == 1
    check(call, drafts, u, excused=-(-s // 3) if nothing_cut else 0, **kw)
    tok, acc, lp = call.answer()
    assert (lp[tok == top] == 0).all() and (lp <= 0).all() and (tok[:, 0] == top[:, 0]).all()
    assert nothing_cut or ((lp[tok >= 0] == 0).all() and acc.min() == 1 and acc.max() == 2)
    p, q, drafts, u = make(rng, s, d, v, spread=6.0, gap=0.2, certain=certain, **kw)
    tok, _, lp = Call(built, p, q, drafts, u, **kw).run().answer()
    assert (lp <= 0).all()
