"""MXFP4 rows and layers: quantisation, the values back, the product, and their refusals.

The reference restates the format in numpy: scales from the exponent of the block's
largest magnitude, codes by nearest value with ties to the even code, products in f64.
GGUF MXFP4 blocks are checked against gguf-py's own dequantisation.
"""
import ctypes as C

import numpy as np
import pytest

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
NP = {"f32": np.float32, "f16": np.float16}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative


@pytest.fixture(scope="module")
def built(pk):
    pk.build()
    return pk


def ref_quantize(x):
    """x [rows][K] f64 -> (codes 0..15 [rows][K], scale bytes [rows][nb], values [rows][K])."""
    x = np.asarray(x, np.float64)
    r, k = x.shape
    nb = -(-k // 32)
    v = np.zeros((r, nb * 32))
    v[:, :k] = x
    v = v.reshape(r, nb, 32)
    bad = ~np.isfinite(v).all(-1)
    a = np.abs(np.where(np.isfinite(v), v, 0)).max(-1)
    e = np.frexp(np.where(a > 0, a, 1.0))[1] - 1 - 2
    e = np.where(a > 0, np.maximum(e, -127), -127)
    m = np.abs(np.where(bad[..., None], 0, v)) * np.exp2(-e.astype(np.float64))[..., None]
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])          # an even code keeps a tie
    code = order[np.abs(m[..., None] - GRID[order]).argmin(-1)]
    val = np.copysign(GRID[code], v) * np.exp2(e.astype(np.float64))[..., None]
    code = code + 8 * np.signbit(v)
    code = np.where(bad[..., None], 0, code)
    val = np.where(bad[..., None], np.nan, val)
    byte = np.where(bad, 255, e + 127)
    return (code.reshape(r, -1)[:, :k].astype(np.uint8), byte.astype(np.uint8), val.reshape(r, -1)[:, :k])


def pack(code, nb):
    c = np.zeros((code.shape[0], nb * 32), np.uint8)
    c[:, :code.shape[1]] = code
    return c[:, 0::2] | c[:, 1::2] << 4


def gguf_blocks(code, byte):
    """GGUF MXFP4 bytes of codes [n][k] and scale bytes: value j in the low half of byte j, value 16 + j in the high."""
    n, nb = byte.shape
    c = code.reshape(n, nb, 32)
    return np.concatenate([byte[..., None], c[..., :16] | c[..., 16:] << 4], -1).astype(np.uint8)


# ---- CPU -----------------------------------------------------------------------

def test_reference_known_answers():
    x = np.array([[6.0, -6.0, 5.0, 2.5, 1.75, 0.25, 0.75, -0.25, 7.9, 0.0]])
    code, byte, val = ref_quantize(x)
    assert byte.tolist() == [[127]]
    assert val.tolist() == [[6, -6, 4, 2, 2, 0, 1, 0, 6, 0]]
    assert code.tolist() == [[7, 15, 6, 4, 4, 0, 2, 8, 7, 0]]
    _, byte, val = ref_quantize(np.array([[2.0 ** -140, 0.0], [np.inf, 1.0], [0.0, 0.0]]))
    assert byte[:, 0].tolist() == [0, 255, 0] and val[0, 0] == 0 and np.isnan(val[1]).all()


def test_refusals(built):
    pk, L, abi = built, built.lib(), built.abi
    p = 1 << 20                                         # never read: refused or no device before that
    ok = [0, p, 0, 4, 64, 64, p, p, None]
    for at, bad in ((2, 8), (2, 39), (3, -1), (3, 1 << 31), (4, 0), (4, (1 << 20) + 1), (5, 63), (5, 1 << 40),
                    (1, None), (6, None), (7, None), (1, p + 2), (6, p + 2)):
        a = list(ok)
        a[at] = bad
        assert L.pk_mx4_quantize(*a) == abi.PK_ERR_INVALID, (at, bad)
        assert b"pk_mx4_quantize" in L.pk_last_error()
    assert L.pk_mx4_quantize(99, *ok[1:]) == abi.PK_ERR_NO_DEVICE
    okd = [0, p, p, 4, 64, p, 1, 64, None]
    for at, bad in ((6, 2), (3, -1), (4, 0), (7, 63), (1, None), (2, None), (5, None), (5, p + 1), (1, p + 1)):
        a = list(okd)
        a[at] = bad
        assert L.pk_mx4_dequantize(*a) == abi.PK_ERR_INVALID, (at, bad)
    w = np.zeros((4, 64), np.float32)
    h = C.c_void_p()

    def create(**kw):
        d = dict(data=w.ctypes.data, type=0, ne0=64, ne1=4, nbytes=w.nbytes, device=99, on_device=0, bias=None)
        d.update(kw)
        t = abi.pk_tensor(d["data"], d["type"], 0, d["ne0"], d["ne1"], d["nbytes"])
        return L.pk_mx4_create(d["device"], C.byref(t), d["on_device"], d["bias"], C.byref(h))

    assert create() == abi.PK_ERR_NO_DEVICE
    assert create(data=None) == abi.PK_ERR_INVALID
    assert create(on_device=1, data=p + 1) == abi.PK_ERR_INVALID
    assert create(on_device=1, bias=p + 2) == abi.PK_ERR_INVALID
    for kw in (dict(type=2), dict(ne0=0), dict(ne1=0), dict(ne1=(1 << 20) + 1), dict(nbytes=w.nbytes - 4),
               dict(type=8, ne0=33, nbytes=4 * 34), dict(type=39, ne0=63, nbytes=4 * 2 * 17), dict(type=39, nbytes=4 * 2 * 17 + 1)):
        assert create(**kw) == abi.PK_ERR_MODEL, kw
    t = abi.pk_tensor(w.ctypes.data, 0, 0, 64, 4, w.nbytes)
    assert L.pk_mx4_create(0, C.byref(t), 0, None, None) == abi.PK_ERR_INVALID
    assert L.pk_mx4_create(0, None, 0, None, C.byref(h)) == abi.PK_ERR_INVALID
    assert L.pk_mx4_workspace(None, 5) == -1
    assert L.pk_mx4_linear(None, p, 0, 1, 64, p, 0, 4, p, 1 << 20, None) == abi.PK_ERR_INVALID
    L.pk_mx4_destroy(None)


# ---- GPU -----------------------------------------------------------------------

def cuda(a, dtype="f32", pad=0, shift=0):
    """Device rows of `dtype` holding a [rows][k], row stride k + pad, `shift` elements into its buffer."""
    import torch
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    r, k = a.shape
    buf = torch.full((r * (k + pad) + shift + 64,), 77.0, dtype=t, device="cuda")
    v = buf[shift:shift + r * (k + pad)].view(r, k + pad)
    v[:, :k] = torch.from_numpy(np.asarray(a, np.float32)).cuda().to(t)
    return buf, v


def run_quantize(pk, a, dtype="f32", pad=0, shift=0):
    import torch
    buf, v = cuda(a, dtype, pad, shift)
    r, k = a.shape
    nb = -(-k // 32)
    codes = torch.full((r * nb * 16 + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((r * nb + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    pk.mx4_quantize(v.data_ptr(), r, k, codes.data_ptr(), scales.data_ptr(), dtype=dtype, row_stride=k + pad, stream=s)
    assert (codes[r * nb * 16:] == 0xA5).all() and (scales[r * nb:] == 0xA5).all()
    return v[:, :k].float().cpu().numpy(), codes, scales


def values_like(rng, r, k):
    x = rng.standard_normal((r, k)) * np.exp2(rng.integers(-20, 20, (r, 1)))
    x[:, ::7] *= 2.0 ** -3
    if r > 2:
        x[1] = 0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("f32", 3, 1), ("f32", 4, 0), ("f16", 0, 0), ("f16", 1, 3), ("bf16", 8, 0), ("bf16", 5, 1)])
@pytest.mark.parametrize("r,k", [(1, 1), (1, 32), (3, 33), (5, 255), (2, 256), (7, 257), (65, 640), (4, 1000), (129, 1024)])
def test_quantize_and_back(built, dtype, pad, shift, r, k):
    import torch
    pk = built
    x = values_like(np.random.default_rng(r * 1000 + k), r, k)
    if dtype == "f16":
        x = np.clip(x, -6e4, 6e4)
    seen, codes, scales = run_quantize(pk, x, dtype, pad, shift)
    nb = -(-k // 32)
    code, byte, val = ref_quantize(seen)
    assert np.array_equal(codes[:r * nb * 16].view(r, -1).cpu().numpy(), pack(code, nb))
    assert np.array_equal(scales[:r * nb].view(r, nb).cpu().numpy(), byte)
    s = torch.cuda.current_stream().cuda_stream
    for out, opad, oshift in (("f32", 0, 0), ("f32", 1, 1), ("bf16", 8, 0), ("f16", 3, 0)):
        buf, y = cuda(np.full((r, k), 5.0), out, opad, oshift)
        before = buf.clone()
        pk.mx4_dequantize(codes.data_ptr(), scales.data_ptr(), r, k, y.data_ptr(), dtype=out, row_stride=k + opad, stream=s)
        want = torch.from_numpy(val).to(y.dtype).float().numpy()     # torch rounds f64 once to nearest even
        assert np.array_equal(y[:, :k].float().cpu().numpy(), want)
        y[:, :k] = 5.0
        assert torch.equal(buf, before)                              # nothing else was written


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("f32", 3, 1), ("f16", 1, 3), ("bf16", 0, 0), ("bf16", 2, 1)])
@pytest.mark.parametrize("k", [1, 7, 24, 31, 32, 33, 49, 64, 65, 104, 128, 129, 250, 256])
def test_many_short_rows(built, k, dtype, pad, shift):
    """Several rows a warp and several warps' rounds of them, every phase of a row's start; a NaN and an
    infinity stay with their own row's block."""
    import torch
    pk = built
    r = 3001
    x = values_like(np.random.default_rng(k), r, k)
    if dtype == "f16":
        x = np.clip(x, -6e4, 6e4)
    x[5, k // 2], x[900, 0], x[3000, k - 1] = np.nan, np.inf, -np.inf
    seen, codes, scales = run_quantize(pk, x, dtype, pad, shift)
    nb = -(-k // 32)
    code, byte, val = ref_quantize(seen)
    assert np.array_equal(codes[:r * nb * 16].view(r, -1).cpu().numpy(), pack(code, nb))
    assert np.array_equal(scales[:r * nb].view(r, nb).cpu().numpy(), byte)
    s = torch.cuda.current_stream().cuda_stream
    for out, opad, oshift in (("f32", 0, 0), ("f32", 1, 1), ("f32", 2, 2), ("bf16", 0, 0), ("bf16", 7, 5), ("f16", 3, 7)):
        buf, y = cuda(np.full((r, k), 5.0), out, opad, oshift)
        before = buf.clone()
        pk.mx4_dequantize(codes.data_ptr(), scales.data_ptr(), r, k, y.data_ptr(), dtype=out, row_stride=k + opad, stream=s)
        want = torch.from_numpy(val).to(y.dtype).float().numpy()
        assert np.array_equal(y[:, :k].float().cpu().numpy(), want, equal_nan=True)
        y[:, :k] = 5.0
        assert torch.equal(buf, before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("bf16", 3, 1)])
@pytest.mark.parametrize("k", [1, 24, 32, 33, 64, 65, 128, 129, 256])
def test_product_of_short_rows(built, k, dtype, pad, shift):
    """Rows whose scales do not fill the words that the product reads, next to a row of NaN."""
    pk = built
    rng = np.random.default_rng(k)
    w = rng.standard_normal((70, k)).astype(np.float32)
    x = rng.standard_normal((515, k)).astype(np.float32)
    x[11] = np.nan
    seen, y = product(pk, w, x, x_dtype=dtype, xpad=pad, shift=shift)
    assert np.isnan(y[11]).all()
    keep = np.arange(515) != 11
    check_product(ref_quantize(w)[2], seen[keep], y[keep])


@pytest.mark.gpu
def test_quantize_borders(built):
    """Every tie and neighbour of a tie, at the lowest, a middle and the highest scale; special blocks."""
    pk = built
    mids = (GRID[1:] + GRID[:-1]) / 2
    pts = np.concatenate([GRID, mids, np.nextafter(mids.astype(np.float32), 9).astype(float),
                          np.nextafter(mids.astype(np.float32), 0).astype(float)])
    pts = np.concatenate([pts, -pts])
    rows = []
    for e in (-127, -126, -60, 0, 31, 125):
        x = np.concatenate([[4.0], pts[:31], [-4.0], pts[27:58]]) * 2.0 ** e
        rows.append(x.astype(np.float32).astype(np.float64))
    rows.append(np.zeros(64))
    rows.append(np.full(64, -0.0))
    rows.append(np.full(64, 2.0 ** -149))
    rows.append(np.full(64, np.finfo(np.float32).max))
    for v in (np.inf, -np.inf, np.nan):
        x = np.ones(64)
        x[40] = v                                       # the first block stays a number
        rows.append(x)
    x = np.array(rows)
    seen, codes, scales = run_quantize(pk, x)
    assert np.array_equal(np.nan_to_num(seen, nan=9), np.nan_to_num(x.astype(np.float32), nan=9))
    code, byte, val = ref_quantize(seen)
    got = codes[:x.shape[0] * 32].view(x.shape[0], 32).cpu().numpy()
    assert np.array_equal(got, pack(code, 2))
    assert np.array_equal(scales[:x.shape[0] * 2].view(-1, 2).cpu().numpy(), byte)


@pytest.mark.gpu
def test_values_at_the_ends(built):
    """Every code at every scale byte, in each type: subnormal, infinite and NaN values as rounding the
    exact value gives them; and back to the same bytes from bf16 where the block's largest code says so."""
    import torch
    pk = built
    byte = np.arange(256, dtype=np.uint8)
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 2))                    # 32 values a row
    codes = torch.from_numpy(pack(code, 1)).cuda()
    scales = torch.from_numpy(byte).cuda()
    val = np.where(code & 8, -1.0, 1.0) * GRID[code & 7] * np.exp2(byte.astype(np.float64) - 127)[:, None]
    val[255] = np.nan
    s = torch.cuda.current_stream().cuda_stream
    for name, t in (("f32", torch.float32), ("f16", torch.float16), ("bf16", torch.bfloat16)):
        out = torch.empty(256, 32, dtype=t, device="cuda")
        pk.mx4_dequantize(codes.data_ptr(), scales.data_ptr(), 256, 32, out.data_ptr(), dtype=name, stream=s)
        want = torch.from_numpy(val).to(t).float().numpy()
        assert np.array_equal(out.float().cpu().numpy(), want, equal_nan=True), name
    # bf16 holds every one of them below 2^126 x 4: quantised again they keep codes and bytes (a block's
    # largest code is 6, so its exponent is the byte's; byte 0 and 1 both end at 2^-127)
    keep = byte[2:252]
    x = torch.from_numpy(val[2:252]).to(torch.bfloat16).cuda()
    c2 = torch.empty(250, 16, dtype=torch.uint8, device="cuda")
    s2 = torch.empty(250, dtype=torch.uint8, device="cuda")
    pk.mx4_quantize(x.data_ptr(), 250, 32, c2.data_ptr(), s2.data_ptr(), dtype="bf16", stream=s)
    assert np.array_equal(s2.cpu().numpy(), keep) and np.array_equal(c2.cpu().numpy(), pack(code[2:252], 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_quantize_half_precision_borders(built, dtype):
    """All magnitudes of half precision of six binades under one block maximum of four, at several scales."""
    import torch
    pk = built
    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    step = 2.0 ** -7 if dtype == "bf16" else 2.0 ** -10
    m = np.concatenate([(1 + np.arange(0, 1, step)) * 2.0 ** e for e in range(-4, 3)])
    m = m[m <= 7.99]
    n = -(-len(m) // 31) * 31
    m = np.concatenate([m, np.zeros(n - len(m))]).reshape(-1, 31)
    x = np.concatenate([np.full((len(m), 1), 4.0), m], 1)
    x = np.concatenate([x, -x])
    for e in ((-126, -30, 0, 100) if dtype == "bf16" else (-10, 0, 10)):
        seen, codes, scales = run_quantize(pk, np.ldexp(x, e), dtype)
        code, byte, _ = ref_quantize(seen)
        r = len(x)
        assert np.array_equal(codes[:r * 16].view(r, -1).cpu().numpy(), pack(code, 1))
        assert np.array_equal(scales[:r].view(r, 1).cpu().numpy(), byte)
    assert t is not None


def product(pk, w, x, bias=None, x_dtype="f32", y_dtype="f32", xpad=0, ypad=0, shift=0, layer=None, stream=None):
    import torch
    r, k = x.shape
    n = w.shape[0] if layer is None else layer.n
    layer = pk.Mx4Linear(w, bias=bias) if layer is None else layer
    _, xv = cuda(x, x_dtype, xpad, shift)
    buf, yv = cuda(np.full((r, n), -3.0), y_dtype, ypad, shift)
    before = buf.clone()
    ws = torch.full((layer.workspace(r) + 64,), 0xFF, dtype=torch.uint8, device="cuda")   # NaN scales if read unwritten
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    layer.forward(xv.data_ptr(), r, yv.data_ptr(), x_dtype=x_dtype, y_dtype=y_dtype, x_stride=k + xpad, y_stride=n + ypad,
                  workspace=ws.data_ptr(), workspace_bytes=layer.workspace(r), stream=s)
    y = yv[:, :n].float().cpu().numpy()
    assert (ws[-64:] == 0xFF).all()
    yv[:, :n] = -3.0
    assert torch.equal(buf, before)
    return xv[:, :k].float().cpu().numpy(), y


def check_product(w_val, x_seen, y, bias=None, y_dtype="f32"):
    """Products of two 4-bit values and their powers of two are exact in 32 bits; what rounds is
    one addition per block of 32, each by 2^-24 of the partial sums at most, four times that for
    sums cut rather than rounded in the tensor cores: (nb + 2) 2^-22 sum |q w|, and y's own type."""
    q = ref_quantize(x_seen)[2]
    want = q @ w_val.T + (0 if bias is None else np.asarray(bias, np.float64))
    mass = np.abs(q) @ np.abs(w_val).T + (0 if bias is None else np.abs(bias))
    nb = -(-q.shape[1] // 32)
    tol = (nb + 2) * 2.0 ** -22 * mass + EPS[y_dtype] * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -126
    assert np.array_equal(np.isnan(want), np.isnan(y))
    bad = ~np.isnan(want) & ~(np.abs(y - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], y[bad][:5], want[bad][:5])


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(1, 1), (7, 33), (64, 32), (65, 64), (128, 640), (129, 257), (193, 96), (640, 1024), (1025, 512), (1030, 640), (300, 4099)])
@pytest.mark.parametrize("r", [1, 2, 3, 8, 9, 17, 33, 64, 65, 128, 129, 300])
def test_product(built, n, k, r):
    rng = np.random.default_rng(n * 7 + k * 3 + r)
    w = rng.standard_normal((n, k)) * np.exp2(rng.integers(-3, 3, (n, 1)))
    x = values_like(rng, r, k) * 2.0 ** -5
    b = rng.standard_normal(n).astype(np.float32) if (n + r) % 2 else None
    seen, y = product(built, w.astype(np.float32), x, bias=b)
    check_product(ref_quantize(w.astype(np.float32))[2], seen, y, b)


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype,y_dtype,xpad,ypad,shift", [("f32", "f32", 1, 1, 1), ("f32", "f32", 4, 4, 0), ("f16", "f32", 0, 3, 0),
                                                             ("bf16", "bf16", 0, 0, 0), ("bf16", "bf16", 3, 1, 1), ("f16", "f16", 8, 8, 0), ("f32", "f16", 2, 5, 3)])
@pytest.mark.parametrize("r,n,k", [(5, 130, 200), (1, 1025, 640), (260, 321, 512), (64, 96, 70)])
def test_product_types_and_strides(built, x_dtype, y_dtype, xpad, ypad, shift, r, n, k):
    rng = np.random.default_rng(r + n + k)
    w = rng.standard_normal((n, k)).astype(np.float32)
    seen, y = product(built, w, rng.standard_normal((r, k)), None, x_dtype, y_dtype, xpad, ypad, shift)
    check_product(ref_quantize(w)[2], seen, y, None, y_dtype)


@pytest.mark.gpu
def test_product_large_rows(built):
    """More rows than one wave of tiles, a row count that ends inside a tile."""
    rng = np.random.default_rng(5)
    w = rng.standard_normal((96, 320)).astype(np.float32)
    x = rng.standard_normal((40001, 320)).astype(np.float32)
    seen, y = product(built, w, x)
    check_product(ref_quantize(w)[2], seen, y)


@pytest.mark.gpu
@pytest.mark.parametrize("y_dtype,ypad", [("f32", 0), ("f32", 1), ("bf16", 0), ("f16", 6)])
@pytest.mark.parametrize("r,n,k", [(2600, 1300, 320), (2561, 1152, 1030), (2700, 1147, 96), (2561, 1152, 1600), (2600, 1300, 2055)])
def test_product_many_tiles(built, r, n, k, y_dtype, ypad):
    """Tiles for every SM several times over, both tile widths, ragged at each end; y rows that can and
    cannot be stored 16 bytes at a time."""
    rng = np.random.default_rng(r + n)
    w = rng.standard_normal((n, k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    seen, y = product(built, w, rng.standard_normal((r, k)), b, "f32", y_dtype, 0, ypad)
    check_product(ref_quantize(w)[2], seen, y, b, y_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [3, 40, 200])
def test_product_nonfinite_rows_stay_apart(built, r):
    rng = np.random.default_rng(r)
    w = rng.standard_normal((70, 96)).astype(np.float32)
    x = rng.standard_normal((r, 96))
    x[1, 50] = np.inf
    x[r - 1, 3] = np.nan
    seen, y = product(built, w, x)
    assert np.isnan(y[[1, r - 1]]).all()
    keep = [i for i in range(r) if i not in (1, r - 1)]
    check_product(ref_quantize(w)[2], seen[keep], y[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "q8_0", "mxfp4"])
@pytest.mark.parametrize("r", [1, 33, 150])
def test_layer_from_gguf_blocks(built, kind, r):
    gguf = pytest.importorskip("gguf")
    pk = built
    rng = np.random.default_rng(r)
    n, k = 77, 160
    w = rng.standard_normal((n, k)).astype(np.float32)
    if kind == "mxfp4":
        code, byte, val = ref_quantize(w)
        blocks = gguf_blocks(code, byte)
        deq = gguf.quants.dequantize(blocks.reshape(n, -1), gguf.GGMLQuantizationType.MXFP4)
        assert np.array_equal(deq.astype(np.float64), val)
        t = pk.synth.Tensor(np.ascontiguousarray(blocks.reshape(-1)), 39, k, n)
    elif kind == "q8_0":
        raw = gguf.quants.quantize(w, gguf.GGMLQuantizationType.Q8_0)
        val = ref_quantize(gguf.quants.dequantize(raw, gguf.GGMLQuantizationType.Q8_0))[2]
        t = pk.synth.Tensor(np.ascontiguousarray(raw.reshape(-1)), 8, k, n)
    else:
        t = pk.synth.Tensor(np.ascontiguousarray(w.astype(np.float16)).view(np.uint8).reshape(-1), 1, k, n)
        val = ref_quantize(w.astype(np.float16))[2]
    layer = pk.Mx4Linear(t)
    seen, y = product(pk, w, rng.standard_normal((r, k)), layer=layer)
    check_product(val, seen, y)


@pytest.mark.gpu
def test_layer_on_device_weight(built):
    """A weight written on a stream just before the layer is made, as device memory."""
    import torch
    pk = built
    w = torch.randn(200, 300, device="cuda").to(torch.bfloat16)
    b = torch.randn(200, device="cuda")
    layer = pk.Mx4Linear(w.data_ptr(), 200, 300, bias=b.data_ptr(), dtype="bf16", on_device=True)
    seen, y = product(pk, None, np.random.default_rng(0).standard_normal((9, 300)), layer=layer)
    check_product(ref_quantize(w.float().cpu().numpy())[2], seen, y, b.cpu().numpy())
    import ctypes
    rc = pk.lib().pk_mx4_linear(layer.h, 256, 0, 1, 300, 256, 0, 200, 256, layer.workspace(1) - 1, None)
    assert rc == pk.abi.PK_ERR_INVALID
    rc = pk.lib().pk_mx4_linear(layer.h, 256, 0, 1, 299, 256, 0, 200, 256, layer.workspace(1), None)
    assert rc == pk.abi.PK_ERR_INVALID
    rc = pk.lib().pk_mx4_linear(layer.h, 256, 0, 1, 300, 256, 0, 199, 256, layer.workspace(1), None)
    assert rc == pk.abi.PK_ERR_INVALID
    rc = pk.lib().pk_mx4_linear(layer.h, 256, 0, 1, 300, 256, 0, 200, 128 + 16, layer.workspace(1), None)
    assert rc == pk.abi.PK_ERR_INVALID
    assert pk.lib().pk_mx4_linear(layer.h, None, 0, 0, 300, None, 0, 200, None, 0, None) == pk.abi.PK_OK
    assert isinstance(layer.h, ctypes.c_void_p)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [1, 20, 700])
def test_captured_and_replayed(built, r):
    """Two graphs of one layer, each with its own workspace, replayed on two streams with new inputs."""
    import torch
    pk = built
    rng = np.random.default_rng(r)
    n, k = 333, 640
    w = rng.standard_normal((n, k)).astype(np.float32)
    layer = pk.Mx4Linear(w)
    sides = []
    for _ in range(2):
        x = torch.zeros(r, k, device="cuda")
        y = torch.zeros(r, n, device="cuda")
        ws = torch.zeros(layer.workspace(r), dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            layer.forward(x.data_ptr(), r, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                          stream=torch.cuda.current_stream().cuda_stream)
        sides.append((x, y, ws, g, torch.cuda.Stream()))
    for _ in range(3):
        xs = [rng.standard_normal((r, k)).astype(np.float32) for _ in sides]
        for (x, *_), v in zip(sides, xs):
            x.copy_(torch.from_numpy(v))
        torch.cuda.synchronize()
        for _, _, _, g, st in sides:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (x, y, *_), v in zip(sides, xs):
            check_product(ref_quantize(w)[2], v, y.cpu().numpy())


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_batch(built):
    """A row's result for row counts on either side of every kernel's range stays within the bound,
    and equal calls give equal bits."""
    import torch
    pk = built
    rng = np.random.default_rng(3)
    w = rng.standard_normal((257, 384)).astype(np.float32)
    layer = pk.Mx4Linear(w)
    x = rng.standard_normal((600, 384)).astype(np.float32)
    for r in (1, 4, 16, 32, 48, 64, 96, 128, 256, 600):
        seen, y = product(pk, w, x[:r], layer=layer)
        check_product(ref_quantize(w)[2], seen, y)
        assert np.array_equal(y, product(pk, w, x[:r], layer=layer)[1])
    assert torch.cuda.current_device() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("k,most", [(640, 32), (1024, 32), (1025, 31), (2048, 16), (2049, 0)])
def test_few_rows_need_no_workspace(built, k, most):
    """No workspace up to the row count at which the rows get a launch of their own; never less for more rows."""
    import torch
    pk = built
    rng = np.random.default_rng(k)
    w = rng.standard_normal((130, k)).astype(np.float32)
    layer = pk.Mx4Linear(w)
    need = [layer.workspace(r) for r in range(0, 70)]
    assert all(n == 0 for n in need[:most + 1]) and all(n > 0 for n in need[most + 1:]) and need == sorted(need)
    for r in (most, most + 1):
        if r == 0:
            continue
        x = rng.standard_normal((r, k)).astype(np.float32)
        if r == most:
            xd, y = torch.from_numpy(x).cuda(), torch.zeros(r, 130, device="cuda")
            layer.forward(xd.data_ptr(), r, y.data_ptr())
            torch.cuda.synchronize()
            check_product(ref_quantize(w)[2], x, y.cpu().numpy())
        check_product(ref_quantize(w)[2], *product(pk, w, x, layer=layer))


@pytest.mark.gpu
def test_first_call_may_be_captured(built):
    """A process whose first product and first draw are captured into a graph."""
    import subprocess
    import sys
    code = """
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("parakeet_b200", sys.argv[1] + "/__init__.py", submodule_search_locations=[sys.argv[1]])
pk = importlib.util.module_from_spec(spec); sys.modules["parakeet_b200"] = pk; spec.loader.exec_module(pk)
w = torch.randn(200, 2100, device="cuda")
layer = pk.Mx4Linear(w.data_ptr(), 200, 2100, on_device=True)
x = torch.randn(300, 2100, device="cuda"); y = torch.zeros(300, 200, device="cuda")
u = torch.rand(300, device="cuda"); tok = torch.full((300,), -5, dtype=torch.int32, device="cuda")
ws = torch.empty(layer.workspace(300), dtype=torch.uint8, device="cuda")
g = torch.cuda.CUDAGraph(); torch.cuda.synchronize()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    layer.forward(x.data_ptr(), 300, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=s)
    pk.sample(y.data_ptr(), 300, 200, u.data_ptr(), tok.data_ptr(), top_p=0.9, stream=s)
g.replay(); torch.cuda.synchronize()
a, b = y.clone(), tok.clone()
layer.forward(x.data_ptr(), 300, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel())
pk.sample(y.data_ptr(), 300, 200, u.data_ptr(), tok.data_ptr(), top_p=0.9)
torch.cuda.synchronize()
assert torch.equal(a, y) and torch.equal(b, tok) and (tok >= 0).all()
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code, built.PKG_DIR], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_an_error_stays_with_its_call(built):
    """A layer too large for the device is refused for memory; neither the next call nor torch finds that error again."""
    import torch
    pk, L, abi = built, built.lib(), built.abi
    x = torch.randn(4, 64, device="cuda")
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), torch.zeros(4, 2, dtype=torch.uint8, device="cuda")
    small = pk.Mx4Linear(np.ones((8, 64), np.float32))
    y = torch.zeros(4, 8, device="cuda")
    n = 1 << 20                                            # 512 GiB of codes: never laid out, the weight never read
    for after in range(3):
        t = abi.pk_tensor(codes.data_ptr(), abi.PK_GGML_F32, 0, n, n, n * n * 4)
        h = C.c_void_p()
        assert L.pk_mx4_create(0, C.byref(t), 1, None, C.byref(h)) == abi.PK_ERR_OOM and not h.value
        if after == 0:
            pk.mx4_quantize(x.data_ptr(), 4, 64, codes.data_ptr(), scales.data_ptr())
        elif after == 1:
            small.forward(x.data_ptr(), 4, y.data_ptr())
        torch.cuda.synchronize()
        assert torch.ones(3, device="cuda").sum().item() == 3


def test_option_refusals(built):
    assert built.lib().pk_mx4_set_option(None, built.abi.PK_OPT_TIMEOUT_US, 5) == built.abi.PK_ERR_INVALID
    assert built.lib().pk_mx4_timeouts(None) == -1


def stalled(pk, layer, x, y, ws):
    """Queues a product whose first block's (or pair's second block's) loads never come, its waits bounded to 20 ms."""
    import torch
    layer.set_option(pk.abi.PK_OPT_TIMEOUT_US, 20_000)
    layer.set_option(pk.abi.PK_OPT_TEST_STALL, 1)
    layer.forward(x.data_ptr(), x.shape[0], y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                  stream=torch.cuda.current_stream().cuda_stream)
    layer.set_option(pk.abi.PK_OPT_TIMEOUT_US, 2_000_000)


@pytest.mark.gpu
@pytest.mark.parametrize("r,n,k", [(5, 333, 640), (200, 64, 640), (200, 333, 640), (3000, 640, 512)], ids=["few", "one tile", "unaligned", "TMA"])
def test_a_wait_that_runs_out_is_reported(built, r, n, k):
    """The call after it says so, once; the layer then works as before."""
    import time

    import torch
    pk = built
    rng = np.random.default_rng(r)
    w = rng.standard_normal((n, k)).astype(np.float32)
    x = rng.standard_normal((r, k)).astype(np.float32)
    layer = pk.Mx4Linear(w)
    for option, value in ((pk.abi.PK_OPT_TIMEOUT_US, 0), (pk.abi.PK_OPT_TIMEOUT_US, -1), (pk.abi.PK_OPT_MATH, 1)):
        with pytest.raises(pk.PkError):
            layer.set_option(option, value)
    dx, y = torch.from_numpy(x).cuda(), torch.zeros(r, n, device="cuda")
    ws = torch.zeros(max(1, layer.workspace(r)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(2):
        t0 = time.perf_counter()
        stalled(pk, layer, dx, y, ws)
        torch.cuda.synchronize()
        assert 0.015 < time.perf_counter() - t0 < 1.0
        with pytest.raises(pk.PkError) as e:
            product(pk, w, x, layer=layer)
        assert e.value.status == pk.abi.PK_ERR_TIMEOUT
        check_product(ref_quantize(w)[2], *product(pk, w, x, layer=layer))


@pytest.mark.gpu
@pytest.mark.parametrize("r,n,k", [(2600, 1300, 2048), (2561, 1152, 2055)], ids=["192", "128"])
@pytest.mark.parametrize("y_dtype,ypad", [("f32", 0), ("f32", 1)], ids=["TMA", "unaligned"])
def test_a_pair_whose_wait_runs_out(built, r, n, k, y_dtype, ypad):
    """One block of a pair has loads in flight that the other never matches: both end once those have come."""
    import torch
    pk = built
    rng = np.random.default_rng(k)
    w = rng.standard_normal((n, k)).astype(np.float32)
    x = rng.standard_normal((r, k)).astype(np.float32)
    layer = pk.Mx4Linear(w)
    dx, y = torch.from_numpy(x).cuda(), torch.zeros(r, n + ypad, device="cuda")
    ws = torch.zeros(layer.workspace(r), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(2):
        layer.set_option(pk.abi.PK_OPT_TIMEOUT_US, 20_000)
        layer.set_option(pk.abi.PK_OPT_TEST_STALL, 1)
        layer.forward(dx.data_ptr(), r, y.data_ptr(), y_stride=n + ypad, workspace=ws.data_ptr(), workspace_bytes=ws.numel())
        layer.set_option(pk.abi.PK_OPT_TIMEOUT_US, 2_000_000)
        torch.cuda.synchronize()
        with pytest.raises(pk.PkError) as e:
            layer.forward(dx.data_ptr(), r, y.data_ptr(), y_stride=n + ypad, workspace=ws.data_ptr(), workspace_bytes=ws.numel())
        assert e.value.status == pk.abi.PK_ERR_TIMEOUT
        check_product(ref_quantize(w)[2], *product(pk, w, x, None, "f32", y_dtype, 0, ypad, layer=layer))


@pytest.mark.gpu
def test_timeouts_reach_their_own_caller(built):
    """A decode through a shared head neither takes nor gets the report of somebody else's product; its own product's
    goes to it alone. Replays of a captured product count."""
    import torch
    pk = built
    rng = np.random.default_rng(0)
    r, n, k = 300, 65, 96
    w = rng.integers(-2, 3, (n, k)).astype(np.float32)     # exact whichever kernel takes it
    x = rng.integers(-2, 3, (r, k)).astype(np.float32)
    head, ctc, other = pk.Mx4Linear(w), pk.CtcGreedy(n, 0), pk.CtcGreedy(n, 0)
    dx, y = torch.from_numpy(x).cuda(), torch.zeros(r, n, device="cuda")
    ws = torch.zeros(head.workspace(r), dtype=torch.uint8, device="cuda")
    want = ctc.decode_frames(x, [0], [r], head=head)[0][0]
    timeout = pk.abi.PK_ERR_TIMEOUT

    def refused(f):
        with pytest.raises(pk.PkError) as e:
            f()
        assert e.value.status == timeout
        return str(e.value)

    def forward():
        head.forward(dx.data_ptr(), r, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel())

    stalled(pk, head, dx, y, ws)                           # somebody's product, still waiting or done
    for i in range(2):
        assert np.array_equal(ctc.decode_frames(x, [0], [r], head=head)[0][0], want)
        torch.cuda.synchronize()
    assert head.timeouts() == 1 and head.timeouts() == 1   # asking does not take the report
    assert "did not run" in refused(forward)
    forward()
    assert head.timeouts() == 1
    # a decode's own product; other handles and forward() hear nothing of it
    head.set_option(pk.abi.PK_OPT_TIMEOUT_US, 20_000)
    head.set_option(pk.abi.PK_OPT_TEST_STALL, 1)
    prev = np.array([3], np.int32)
    assert "pk_ctc_decode" in refused(lambda: ctc.decode_frames(x, [0], [r], head=head, prev=prev))
    head.set_option(pk.abi.PK_OPT_TIMEOUT_US, 2_000_000)
    forward()
    assert head.timeouts() == 1
    for c in (other, ctc):
        assert np.array_equal(c.decode_frames(x, [0], [r], head=head)[0][0], want)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        stalled(pk, head, dx, y, ws)
    assert head.timeouts() == 1
    for i in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert head.timeouts() == 2 + i
    refused(forward)
    forward()
    torch.cuda.synchronize()
    assert head.timeouts() == 3 and torch.equal(y.cpu(), torch.from_numpy(x @ w.T))
    ctc.close()
    other.close()


@pytest.mark.gpu
@pytest.mark.parametrize("r", [3, 40, 700, 2600])
def test_nonfinite_weights_stay_in_their_outputs(built, r):
    rng = np.random.default_rng(r)
    n, k = 1300, 1601
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[0, 5], w[700, k - 1], w[n - 1, 900] = np.nan, np.inf, -np.inf
    seen, y = product(built, w, rng.standard_normal((r, k)))
    assert np.isnan(y[:, [0, 700, n - 1]]).all()
    check_product(ref_quantize(w)[2], seen, y)
