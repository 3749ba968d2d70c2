"""8-bit rows and layers: quantisation in blocks of 128, the values back, the product, CTC through an
8-bit head, and their refusals.

The reference restates the format in numpy: the scale is the smallest power of two that brings the block's
largest magnitude to 448 or below, the code the nearest of the 127 magnitudes with ties to the even code,
products in f64.
"""
import ctypes as C
import subprocess
import sys
import time

import numpy as np
import pytest

from test_mx4 import EPS, cuda, values_like

GRID = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119])
assert len(GRID) == 127 and GRID[-1] == 448


@pytest.fixture(scope="module")
def built(pk):
    pk.build()
    return pk


def ref_quantize(x, block_rows=1):
    """x [rows][K] -> (codes [rows][K], scale bytes [row blocks][nb], values [rows][K]), blocks of block_rows x 128."""
    x = np.asarray(x, np.float64)
    r, k = x.shape
    nr, nb = -(-r // block_rows), -(-k // 128)
    v = np.zeros((nr * block_rows, nb * 128))
    v[:r, :k] = x
    v = v.reshape(nr, block_rows, nb, 128)
    bad = ~np.isfinite(v).all((1, 3))
    a = np.abs(np.where(np.isfinite(v), v, 0)).max((1, 3))
    f, e = np.frexp(np.where(a > 0, a, 1.0))
    e = np.where(a > 0, np.maximum(e - np.where(f <= 0.875, 9, 8), -127), -127)     # 448 = 0.875 * 2^9
    at = (slice(None), None, slice(None), None)
    scale, bad_at = np.exp2(e.astype(np.float64))[at], np.broadcast_to(bad[at], v.shape)
    m = np.abs(np.where(bad_at, 0, v)) / scale
    up = np.minimum(np.searchsorted(GRID, m), 126)
    down = np.maximum(up - 1, 0)
    far, near = GRID[up] - m, m - GRID[down]
    code = np.where((far < near) | ((far == near) & (up % 2 == 0)), up, down)
    val = np.where(bad_at, np.nan, np.copysign(GRID[code], v) * scale)
    code = np.where(bad_at, 0, code + 128 * np.signbit(v))

    def flat(q):
        return q.reshape(nr * block_rows, nb * 128)[:r, :k]

    return flat(code).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8), flat(val)


def pack(code):
    """Codes as rows of whole 16 bytes."""
    r, k = code.shape
    c = np.zeros((r, -(-k // 16) * 16), np.uint8)
    c[:, :k] = code
    return c


# ---- CPU -----------------------------------------------------------------------

def test_reference_known_answers():
    x = np.array([[448.0, -449.0, 17.0, 19.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, -0.0, 432.0, 1.0625]])
    code, byte, val = ref_quantize(np.where(x == -449.0, -448.0, x))
    assert byte.tolist() == [[127]]
    assert val.tolist() == [[448, -448, 16, 20, 2.0 ** -9, 0, 2.0 ** -8, 0, 448, 1]]
    assert code.tolist() == [[126, 254, 88, 90, 1, 0, 2, 128, 126, 56]]
    _, byte, val = ref_quantize(x)                       # 449: the next scale
    assert byte.tolist() == [[128]] and val[0, :2].tolist() == [448, -448]
    _, byte, val = ref_quantize(np.array([[2.0 ** -140, 0.0], [np.inf, 1.0], [0.0, 0.0], [np.finfo(np.float32).max, 1.0]]))
    assert byte[:, 0].tolist() == [0, 255, 0, 247] and val[0, 0] == 0 and np.isnan(val[1]).all()
    w = np.ones((130, 130))
    w[0, 0], w[129, 129] = 448.0, 7.0
    assert ref_quantize(w, 128)[1].tolist() == [[127, 119], [119, 121]]


def test_refusals(built):
    pk, L, abi = built, built.lib(), built.abi
    p = 1 << 20                                         # never read: refused or no device before that
    ok = [0, p, 0, 4, 64, 64, p, p, None]
    for at, bad in ((2, 8), (2, 39), (3, -1), (3, 1 << 31), (4, 0), (4, (1 << 20) + 1), (5, 63), (5, 1 << 40),
                    (1, None), (6, None), (7, None), (1, p + 2), (6, p + 4)):
        a = list(ok)
        a[at] = bad
        assert L.pk_fp8_quantize(*a) == abi.PK_ERR_INVALID, (at, bad)
        assert b"pk_fp8_quantize" in L.pk_last_error()
    assert L.pk_fp8_quantize(99, *ok[1:]) == abi.PK_ERR_NO_DEVICE
    okd = [0, p, p, 4, 64, p, 1, 64, None]
    for at, bad in ((6, 2), (3, -1), (4, 0), (7, 63), (1, None), (2, None), (5, None), (5, p + 1), (1, p + 1)):
        a = list(okd)
        a[at] = bad
        assert L.pk_fp8_dequantize(*a) == abi.PK_ERR_INVALID, (at, bad)
    w = np.zeros((4, 64), np.float32)
    h = C.c_void_p()

    def create(**kw):
        d = dict(data=w.ctypes.data, type=0, ne0=64, ne1=4, nbytes=w.nbytes, device=99, on_device=0, bias=None)
        d.update(kw)
        t = abi.pk_tensor(d["data"], d["type"], 0, d["ne0"], d["ne1"], d["nbytes"])
        return L.pk_fp8_create(d["device"], C.byref(t), d["on_device"], d["bias"], C.byref(h))

    assert create() == abi.PK_ERR_NO_DEVICE
    assert create(data=None) == abi.PK_ERR_INVALID
    assert create(on_device=1, data=p + 1) == abi.PK_ERR_INVALID
    assert create(on_device=1, bias=p + 2) == abi.PK_ERR_INVALID
    for kw in (dict(type=2), dict(type=39, nbytes=4 * 2 * 17), dict(ne0=0), dict(ne1=0), dict(ne1=(1 << 20) + 1),
               dict(nbytes=w.nbytes - 4), dict(type=8, ne0=33, nbytes=4 * 34)):
        assert create(**kw) == abi.PK_ERR_MODEL, kw
    t = abi.pk_tensor(w.ctypes.data, 0, 0, 64, 4, w.nbytes)
    assert L.pk_fp8_create(0, C.byref(t), 0, None, None) == abi.PK_ERR_INVALID
    assert L.pk_fp8_create(0, None, 0, None, C.byref(h)) == abi.PK_ERR_INVALID
    assert L.pk_fp8_workspace(None, 5) == -1 and L.pk_fp8_timeouts(None) == -1
    assert L.pk_fp8_set_option(None, abi.PK_OPT_TIMEOUT_US, 5) == abi.PK_ERR_INVALID
    assert L.pk_fp8_linear(None, p, 0, 1, 64, p, 0, 4, p, 1 << 20, None) == abi.PK_ERR_INVALID
    L.pk_fp8_destroy(None)


# ---- GPU: rows -----------------------------------------------------------------

def run_quantize(pk, a, dtype="f32", pad=0, shift=0):
    import torch
    _, v = cuda(a, dtype, pad, shift)
    r, k = a.shape
    nb, ldc = -(-k // 128), -(-k // 16) * 16
    codes = torch.full((r * ldc + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((r * nb + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    pk.fp8_quantize(v.data_ptr(), r, k, codes.data_ptr(), scales.data_ptr(), dtype=dtype, row_stride=k + pad, stream=s)
    assert (codes[r * ldc:] == 0xA5).all() and (scales[r * nb:] == 0xA5).all()
    return v[:, :k].float().cpu().numpy(), codes, scales


def check_rows(pk, x, dtype, pad, shift, outs):
    import torch
    r, k = x.shape
    seen, codes, scales = run_quantize(pk, x, dtype, pad, shift)
    code, byte, val = ref_quantize(seen)
    assert np.array_equal(codes[:r * (-(-k // 16) * 16)].view(r, -1).cpu().numpy(), pack(code))
    assert np.array_equal(scales[:byte.size].view(r, -1).cpu().numpy(), byte)
    s = torch.cuda.current_stream().cuda_stream
    for out, opad, oshift in outs:
        buf, y = cuda(np.full((r, k), 5.0), out, opad, oshift)
        before = buf.clone()
        pk.fp8_dequantize(codes.data_ptr(), scales.data_ptr(), r, k, y.data_ptr(), dtype=out, row_stride=k + opad, stream=s)
        want = torch.from_numpy(val).to(y.dtype).float().numpy()     # torch rounds f64 once to nearest even
        assert np.array_equal(y[:, :k].float().cpu().numpy(), want, equal_nan=True)
        y[:, :k] = 5.0
        assert torch.equal(buf, before)                              # nothing else was written


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("f32", 3, 1), ("f32", 4, 0), ("f16", 0, 0), ("f16", 1, 3), ("bf16", 8, 0), ("bf16", 5, 1)])
@pytest.mark.parametrize("r,k", [(1, 1), (1, 128), (3, 129), (5, 255), (2, 256), (7, 257), (65, 640), (4, 1000), (129, 1024), (2, 4099)])
def test_quantize_and_back(built, dtype, pad, shift, r, k):
    x = values_like(np.random.default_rng(r * 1000 + k), r, k)
    if dtype == "f16":
        x = np.clip(x, -6e4, 6e4)
    check_rows(built, x, dtype, pad, shift, (("f32", 0, 0), ("f32", 1, 1), ("bf16", 8, 0), ("f16", 3, 0)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("f32", 3, 1), ("f16", 1, 3), ("bf16", 0, 0), ("bf16", 2, 1)])
@pytest.mark.parametrize("k", [1, 7, 16, 31, 32, 33, 49, 64, 65, 127, 128, 129, 250, 256])
def test_many_short_rows(built, k, dtype, pad, shift):
    """Several rows a warp and several warps' rounds of them, every phase of a row's start; a NaN and an
    infinity stay with their own row's block."""
    x = values_like(np.random.default_rng(k), 3001, k)
    if dtype == "f16":
        x = np.clip(x, -6e4, 6e4)
    x[5, k // 2], x[900, 0], x[3000, k - 1] = np.nan, np.inf, -np.inf
    check_rows(built, x, dtype, pad, shift, (("f32", 0, 0), ("f32", 1, 1), ("f32", 2, 2), ("bf16", 0, 0), ("bf16", 7, 5), ("f16", 3, 7)))


@pytest.mark.gpu
def test_quantize_borders(built):
    """Every tie and neighbour of a tie, at the lowest, middle and highest scales; magnitudes around the one
    where the scale steps up; special blocks."""
    mids = (GRID[1:] + GRID[:-1]) / 2
    pts = np.concatenate([GRID, mids, np.nextafter(mids.astype(np.float32), 999).astype(float),
                          np.nextafter(mids.astype(np.float32), 0).astype(float)])
    pts = np.concatenate([pts, -pts])
    pts = np.concatenate([pts, np.zeros(-len(pts) % 127)]).reshape(-1, 127)
    pts = np.concatenate([np.full((len(pts), 1), 448.0), pts], 1)
    rows = [pts * 2.0 ** e for e in (-127, -126, -60, 0, 31, 119)]
    top = []
    for e in (-130, -127, -126, -30, 0, 60, 119):
        for m in (447.99998, 448.0, 448.00003, 511.99997, 512.0, 256.0):
            top.append(np.concatenate([[m], np.linspace(-m, m, 127)]) * 2.0 ** e)
    rows.append(np.array(top))
    for v in (0.0, -0.0, 2.0 ** -149, np.finfo(np.float32).max):
        rows.append(np.full((1, 128), v))
    x = np.concatenate(rows).astype(np.float32).astype(np.float64)
    x = np.concatenate([x, x[::-1]], 1)                 # two blocks a row
    for i, v in enumerate((np.inf, -np.inf, np.nan)):
        x[i, 200] = v                                   # the first block stays a number
    check_rows(built, x, "f32", 0, 0, (("f32", 0, 0), ("bf16", 0, 0)))


@pytest.mark.gpu
def test_values_at_the_ends(built):
    """Every code at every scale byte, in each type: subnormal, infinite and NaN values as rounding the exact
    value gives them."""
    import torch
    pk = built
    byte = np.arange(256, dtype=np.uint8)
    code = np.tile(np.arange(256, dtype=np.uint8), (256, 1))                    # two blocks a row
    mag = np.append(GRID, np.nan)
    val = np.where(code & 128, -1.0, 1.0) * mag[code & 127] * np.exp2(byte.astype(np.float64) - 127)[:, None]
    val[255] = np.nan
    codes, scales = torch.from_numpy(code).cuda(), torch.from_numpy(np.stack([byte, byte], 1)).cuda()
    s = torch.cuda.current_stream().cuda_stream
    for name, t in (("f32", torch.float32), ("f16", torch.float16), ("bf16", torch.bfloat16)):
        out = torch.empty(256, 256, dtype=t, device="cuda")
        pk.fp8_dequantize(codes.data_ptr(), scales.data_ptr(), 256, 256, out.data_ptr(), dtype=name, stream=s)
        assert np.array_equal(out.float().cpu().numpy(), torch.from_numpy(val).to(t).float().numpy(), equal_nan=True), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_quantize_half_precision_borders(built, dtype):
    """All magnitudes of half precision from 2^-11 up under one block maximum of 448, at several scales."""
    step = 2.0 ** -7 if dtype == "bf16" else 2.0 ** -10
    m = np.concatenate([(1 + np.arange(0, 1, step)) * 2.0 ** e for e in range(-11, 9)])
    m = m[m <= 448]
    m = np.concatenate([m, np.zeros(-len(m) % 127)]).reshape(-1, 127)
    x = np.concatenate([np.full((len(m), 1), 448.0), m], 1)
    x = np.concatenate([x, -x])
    for e in ((-126, -30, 0, 100) if dtype == "bf16" else (-13, 0, 7)):
        check_rows(built, np.ldexp(x, e), dtype, 0, 0, ((dtype, 0, 0),))


# ---- GPU: the product -----------------------------------------------------------

def product(pk, w, x, bias=None, x_dtype="f32", y_dtype="f32", xpad=0, ypad=0, shift=0, layer=None, stream=None):
    import torch
    r, k = x.shape
    n = w.shape[0] if layer is None else layer.n
    layer = pk.Fp8Linear(w, bias=bias) if layer is None else layer
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


def weight_values(w):
    return ref_quantize(w, 128)[2]


def check_product(w_val, x_seen, y, bias=None, y_dtype="f32"):
    """Products of two e4m3 values and their powers of two are exact in 32 bits; what rounds is one addition
    per 32 values, each by 2^-24 of the partial sums at most, four times that for sums cut rather than rounded
    in the tensor cores, and at most seven additions of a cluster's sums: (K / 32 + 9) 2^-22 sum |q w|, and y's
    own type."""
    q = ref_quantize(x_seen)[2]
    want = q @ w_val.T + (0 if bias is None else np.asarray(bias, np.float64))
    mass = np.abs(q) @ np.abs(w_val).T + (0 if bias is None else np.abs(bias))
    tol = (q.shape[1] / 32 + 9) * 2.0 ** -22 * mass + EPS[y_dtype] * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -126
    assert np.array_equal(np.isnan(want), np.isnan(y))
    bad = ~np.isnan(want) & ~(np.abs(y - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], y[bad][:5], want[bad][:5])


SHAPES = [(1, 1), (7, 33), (64, 32), (65, 128), (128, 640), (129, 257), (193, 96), (640, 1024), (1025, 512), (1030, 640), (300, 4099), (20, 8200)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("r", [1, 2, 9, 16, 17, 32, 33, 64, 65, 128, 129, 300])
def test_product(built, n, k, r):
    rng = np.random.default_rng(n * 7 + k * 3 + r)
    w = rng.standard_normal((n, k)) * np.exp2(rng.integers(-3, 3, (n, 1)))
    x = values_like(rng, r, k) * 2.0 ** -5
    b = rng.standard_normal(n).astype(np.float32) if (n + r) % 2 else None
    seen, y = product(built, w.astype(np.float32), x, bias=b)
    check_product(weight_values(w.astype(np.float32)), seen, y, b)


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype,y_dtype,xpad,ypad,shift", [("f32", "f32", 1, 1, 1), ("f32", "f32", 4, 4, 0), ("f16", "f32", 0, 3, 0),
                                                             ("bf16", "bf16", 0, 0, 0), ("bf16", "bf16", 3, 1, 1), ("f16", "f16", 8, 8, 0), ("f32", "f16", 2, 5, 3)])
@pytest.mark.parametrize("r,n,k", [(5, 130, 200), (1, 1025, 640), (260, 321, 512), (64, 96, 70)])
def test_product_types_and_strides(built, x_dtype, y_dtype, xpad, ypad, shift, r, n, k):
    rng = np.random.default_rng(r + n + k)
    w = rng.standard_normal((n, k)).astype(np.float32)
    seen, y = product(built, w, rng.standard_normal((r, k)), None, x_dtype, y_dtype, xpad, ypad, shift)
    check_product(weight_values(w), seen, y, None, y_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("bf16", 3, 1)])
@pytest.mark.parametrize("k", [1, 24, 64, 65, 128, 129, 256])
def test_product_of_short_rows(built, k, dtype, pad, shift):
    """Rows whose scales do not fill the words that the product reads, next to a row of NaN."""
    rng = np.random.default_rng(k)
    w = rng.standard_normal((70, k)).astype(np.float32)
    x = rng.standard_normal((515, k)).astype(np.float32)
    x[11] = np.nan
    seen, y = product(built, w, x, x_dtype=dtype, xpad=pad, shift=shift)
    assert np.isnan(y[11]).all()
    keep = np.arange(515) != 11
    check_product(weight_values(w), seen[keep], y[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("r,n,k", [(40001, 96, 320), (2600, 1300, 320), (2561, 1152, 1030), (2700, 1147, 96), (2561, 1152, 1600),
                                   (5200, 2500, 2055), (9000, 300, 128), (19000, 700, 130), (4500, 640, 517)])
@pytest.mark.parametrize("y_dtype,ypad", [("f32", 0), ("f32", 1), ("bf16", 0)])
def test_product_many_tiles(built, r, n, k, y_dtype, ypad):
    """Tiles for every pair of SMs several times over, all tile widths, ragged at each end, K of one to seventeen
    blocks."""
    rng = np.random.default_rng(r + n)
    w = rng.standard_normal((n, k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    x = rng.standard_normal((r, k)).astype(np.float32)
    x[:, : k // 3] *= 2.0 ** 9                            # blocks of unlike scales
    seen, y = product(built, w, x, b, "f32", y_dtype, 0, ypad)
    check_product(weight_values(w), seen, y, b, y_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [3, 40, 200, 2600])
def test_product_nonfinite_stays_apart(built, r):
    """Rows of x with an infinity or a NaN, and weight blocks with one: their own rows and their own 128 outputs."""
    rng = np.random.default_rng(r)
    n, k = 1300, 1601
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[5, 5], w[700, k - 1], w[n - 1, 900] = np.nan, np.inf, -np.inf
    x = rng.standard_normal((r, k))
    x[1, 50], x[r - 1, 3] = np.inf, np.nan
    seen, y = product(built, w, x)
    assert np.isnan(y[[1, r - 1]]).all()
    keep = [i for i in range(r) if i not in (1, r - 1)]
    nan = np.isin(np.arange(n) // 128, (0, 5, 10))
    assert np.isnan(y[:, nan]).all()
    check_product(weight_values(w)[~nan], seen[keep], y[keep][:, ~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("r", [3, 50, 300])
def test_product_at_the_ends_of_the_scales(built, r):
    """Scales far apart from block to block, whose product is an ordinary number."""
    rng = np.random.default_rng(r)
    w = rng.standard_normal((130, 384)).astype(np.float32)
    x = rng.standard_normal((r, 384)).astype(np.float32)
    for i, e in enumerate((-100, 0, 105)):
        x[:, i * 128:(i + 1) * 128] *= np.float32(2.0 ** e)
        w[:, i * 128:(i + 1) * 128] *= np.float32(2.0 ** -e)
    seen, y = product(built, w, x)
    check_product(weight_values(w), seen, y)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("r", [1, 33, 150])
def test_layer_from_gguf_blocks(built, kind, r):
    gguf = pytest.importorskip("gguf")
    pk = built
    rng = np.random.default_rng(r)
    n, k = 277, 160
    w = rng.standard_normal((n, k)).astype(np.float32)
    if kind == "q8_0":
        raw = gguf.quants.quantize(w, gguf.GGMLQuantizationType.Q8_0)
        val = weight_values(gguf.quants.dequantize(raw, gguf.GGMLQuantizationType.Q8_0))
        t = pk.synth.Tensor(np.ascontiguousarray(raw.reshape(-1)), 8, k, n)
    else:
        t = pk.synth.Tensor(np.ascontiguousarray(w.astype(np.float16)).view(np.uint8).reshape(-1), 1, k, n)
        val = weight_values(w.astype(np.float16))
    layer = pk.Fp8Linear(t)
    seen, y = product(pk, w, rng.standard_normal((r, k)), layer=layer)
    check_product(val, seen, y)


@pytest.mark.gpu
def test_layer_on_device_weight_and_refusals(built):
    """A weight written on a stream just before the layer is made, as device memory; calls that are refused."""
    import torch
    pk = built
    w = torch.randn(200, 300, device="cuda").to(torch.bfloat16)
    b = torch.randn(200, device="cuda")
    layer = pk.Fp8Linear(w.data_ptr(), 200, 300, bias=b.data_ptr(), dtype="bf16", on_device=True)
    for r in (9, 90):
        seen, y = product(pk, None, np.random.default_rng(0).standard_normal((r, 300)), layer=layer)
        check_product(weight_values(w.float().cpu().numpy()), seen, y, b.cpu().numpy())
    L, bad, ws = pk.lib(), pk.abi.PK_ERR_INVALID, layer.workspace(90)
    ok = [layer.h, 256, 0, 90, 300, 256, 0, 200, 256, ws, None]
    for at, v in ((1, None), (1, 258), (2, 8), (3, -1), (3, 1 << 31), (4, 299), (4, 1 << 40), (5, None), (5, 257), (6, 8), (7, 199),
                  (7, 1 << 40), (8, None), (8, 128 + 16), (9, ws - 1)):
        a = list(ok)
        a[at] = v
        assert L.pk_fp8_linear(*a) == bad, (at, v)
    assert L.pk_fp8_linear(layer.h, None, 0, 0, 300, None, 0, 200, None, 0, None) == pk.abi.PK_OK
    for option, value in ((pk.abi.PK_OPT_TIMEOUT_US, 0), (pk.abi.PK_OPT_TIMEOUT_US, -1), (pk.abi.PK_OPT_MATH, 1)):
        with pytest.raises(pk.PkError):
            layer.set_option(option, value)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [1, 20, 60, 700])
def test_captured_and_replayed(built, r):
    """Two graphs of one layer, each with its own workspace, replayed on two streams with new inputs."""
    import torch
    pk = built
    rng = np.random.default_rng(r)
    n, k = 333, 640
    w = rng.standard_normal((n, k)).astype(np.float32)
    layer = pk.Fp8Linear(w)
    sides = []
    for _ in range(2):
        x, y = torch.zeros(r, k, device="cuda"), torch.zeros(r, n, device="cuda")
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
            check_product(weight_values(w), v, y.cpu().numpy())


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_batch(built):
    """A row's result for row counts on either side of every kernel's range stays within the bound, and equal
    calls give equal bits; workspace never falls with more rows, and none is needed up to some count."""
    pk = built
    rng = np.random.default_rng(3)
    for n, k in ((257, 384), (8198, 640), (130, 4099)):
        w = rng.standard_normal((n, k)).astype(np.float32)
        layer = pk.Fp8Linear(w)
        need = [layer.workspace(r) for r in range(0, 300)]
        assert need == sorted(need) and need[1] == 0 and need[-1] > 0
        x = rng.standard_normal((300, k)).astype(np.float32)
        val = weight_values(w)
        for r in (1, 4, 16, 31, 32, 33, 48, 64, 96, 128, 129, 300):
            seen, y = product(pk, w, x[:r], layer=layer)
            check_product(val, seen, y)
            assert np.array_equal(y, product(pk, w, x[:r], layer=layer)[1])


@pytest.mark.gpu
def test_first_call_may_be_captured(built):
    """A process whose first products are captured into a graph."""
    code = """
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("parakeet_b200", sys.argv[1] + "/__init__.py", submodule_search_locations=[sys.argv[1]])
pk = importlib.util.module_from_spec(spec); sys.modules["parakeet_b200"] = pk; spec.loader.exec_module(pk)
w = torch.randn(200, 2100, device="cuda")
layer = pk.Fp8Linear(w.data_ptr(), 200, 2100, on_device=True)
x = torch.randn(300, 2100, device="cuda"); y = torch.zeros(300, 200, device="cuda"); z = torch.zeros(2, 200, device="cuda")
ws = torch.empty(layer.workspace(300), dtype=torch.uint8, device="cuda")
g = torch.cuda.CUDAGraph(); torch.cuda.synchronize()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    layer.forward(x.data_ptr(), 300, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=s)
    layer.forward(x.data_ptr(), 2, z.data_ptr(), stream=s)
g.replay(); torch.cuda.synchronize()
a, b = y.clone(), z.clone()
layer.forward(x.data_ptr(), 300, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel())
layer.forward(x.data_ptr(), 2, z.data_ptr())
torch.cuda.synchronize()
assert torch.equal(a, y) and torch.equal(b, z) and (y != 0).any() and (z != 0).any()
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code, built.PKG_DIR], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_an_error_stays_with_its_call(built):
    """A layer too large for the device is refused for memory; neither the next call nor torch finds that error again."""
    import torch
    pk, L, abi = built, built.lib(), built.abi
    x, y = torch.randn(4, 64, device="cuda"), torch.zeros(4, 8, device="cuda")
    small = pk.Fp8Linear(np.ones((8, 64), np.float32))
    n = 1 << 20                                            # 1 TiB of codes: never laid out, the weight never read
    for _ in range(2):
        t = abi.pk_tensor(x.data_ptr(), abi.PK_GGML_F32, 0, n, n, n * n * 4)
        h = C.c_void_p()
        assert L.pk_fp8_create(0, C.byref(t), 1, None, C.byref(h)) == abi.PK_ERR_OOM and not h.value
        small.forward(x.data_ptr(), 4, y.data_ptr())
        torch.cuda.synchronize()
        assert torch.ones(3, device="cuda").sum().item() == 3


def stalled(pk, layer, x, y, ws):
    """Queues a product whose first block's (or pair's second block's) loads never come, its waits bounded to 20 ms."""
    import torch
    layer.set_option(pk.abi.PK_OPT_TIMEOUT_US, 20_000)
    layer.set_option(pk.abi.PK_OPT_TEST_STALL, 1)
    layer.forward(x.data_ptr(), x.shape[0], y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                  stream=torch.cuda.current_stream().cuda_stream)
    layer.set_option(pk.abi.PK_OPT_TIMEOUT_US, 2_000_000)


@pytest.mark.gpu
@pytest.mark.parametrize("r,n,k", [(5, 333, 640), (5, 20000, 640), (60, 333, 640), (60, 333, 4099), (200, 64, 640), (3000, 640, 512), (2600, 1300, 2055)])
def test_a_wait_that_runs_out_is_reported(built, r, n, k):
    """The call after it says so, once; the layer then works as before. Kernels with and without clusters, blocks of a
    pair of which one has loads in flight that the other never matches."""
    import torch
    pk = built
    rng = np.random.default_rng(r)
    w = rng.standard_normal((n, k)).astype(np.float32)
    x = rng.standard_normal((r, k)).astype(np.float32)
    layer = pk.Fp8Linear(w)
    dx, y = torch.from_numpy(x).cuda(), torch.zeros(r, n, device="cuda")
    ws = torch.zeros(max(1, layer.workspace(r)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for i in range(2):
        t0 = time.perf_counter()
        stalled(pk, layer, dx, y, ws)
        torch.cuda.synchronize()
        assert 0.015 < time.perf_counter() - t0 < 1.0
        with pytest.raises(pk.PkError) as e:
            product(pk, w, x, layer=layer)
        assert e.value.status == pk.abi.PK_ERR_TIMEOUT and layer.timeouts() == i + 1
        check_product(weight_values(w), *product(pk, w, x, layer=layer))


# ---- GPU: CTC through an 8-bit head ----------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("frames", [1, 20, 90, 3000])
def test_ctc_through_a_head(built, orc, frames):
    """Whole-number weights and frames: the head's logits are exact, so the path is the argmax of them, and the drawn
    path that of pk_ctc_decode on the same logits."""
    pk = built
    rng = np.random.default_rng(frames)
    n, k = 65, 96
    w, x = rng.integers(-2, 3, (n, k)).astype(np.float32), rng.integers(-2, 3, (frames, k)).astype(np.float32)
    head, ctc = pk.Fp8Linear(w), pk.CtcGreedy(n, 0)
    want = (x @ w.T).astype(np.float32)
    half = frames // 2
    toks, fr, prev = ctc.decode_frames(x, [0, half], [half, frames - half], head=head, with_frames=True)
    for (a, b), t, p in zip(((0, half), (half, frames)), toks, prev):
        if a == b:
            assert len(t) == 0 and p == -1
            continue
        et, _, ep = orc.ctc_greedy_window(want[a:b], 0, -1)
        assert np.array_equal(t, et) and p == ep
    u = rng.random(frames).astype(np.float32)
    drawn = ctc.decode_frames(x, [0], [frames], head=head, uniforms=u, temperature=4.0, top_p=0.9)[0][0]
    assert np.array_equal(drawn, ctc.decode_frames(want, [0], [frames], uniforms=u, temperature=4.0, top_p=0.9)[0][0])
    with pytest.raises(pk.PkError):
        pk.CtcGreedy(n + 1, 0).decode_frames(x, [0], [frames], head=head)
    # a decode's own wait that runs out is reported by the decode
    head.set_option(pk.abi.PK_OPT_TIMEOUT_US, 20_000)
    head.set_option(pk.abi.PK_OPT_TEST_STALL, 1)
    with pytest.raises(pk.PkError) as e:
        ctc.decode_frames(x, [0], [frames], head=head)
    assert e.value.status == pk.abi.PK_ERR_TIMEOUT and "pk_ctc_decode_fp8" in str(e.value) and head.timeouts() == 0
    head.set_option(pk.abi.PK_OPT_TIMEOUT_US, 2_000_000)
    assert np.array_equal(ctc.decode_frames(x, [0, half], [half, frames - half], head=head)[0][1], toks[1])
    head.close()
    with pytest.raises(ValueError):
        ctc.decode_frames(x, [0], [frames], head=head)
    ctc.close()


@pytest.mark.gpu
def test_products_on_many_streams_at_once(built):
    """Products of every kind, in clusters and in pairs of blocks, in 8 bits and in 4, that share the device's SMs and
    their tensor memory: each gives what it gives by itself."""
    import torch
    pk = built
    rng = np.random.default_rng(12)
    jobs = []
    for i, (kind, r, n, k) in enumerate([(pk.Fp8Linear, 1, 1000, 1024), (pk.Fp8Linear, 16, 512, 1024), (pk.Fp8Linear, 30, 384, 1000), (pk.Fp8Linear, 60, 333, 4099),
                                         (pk.Fp8Linear, 128, 700, 4096), (pk.Fp8Linear, 700, 640, 512), (pk.Fp8Linear, 5, 200, 300), (pk.Mx4Linear, 2600, 1300, 512),
                                         (pk.Mx4Linear, 7, 2000, 640), (pk.Mx4Linear, 100, 320, 1024), (pk.Fp8Linear, 3000, 300, 640), (pk.Fp8Linear, 2, 1024, 900)]):
        layer = kind(rng.standard_normal((n, k)).astype(np.float32))
        x, y = torch.from_numpy(rng.standard_normal((r, k)).astype(np.float32)).cuda(), torch.zeros(r, n, device="cuda")
        ws = torch.zeros(max(1, layer.workspace(r)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        layer.forward(x.data_ptr(), r, y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel())
        torch.cuda.synchronize()
        jobs.append((layer, x, y, ws, torch.cuda.Stream(), y.clone()))
        y.zero_()
    torch.cuda.synchronize()
    for _ in range(100):
        for layer, x, y, ws, st, _ in jobs:
            layer.forward(x.data_ptr(), x.shape[0], y.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    for layer, _, y, _, _, want in jobs:
        assert torch.equal(y, want) and layer.timeouts() == 0
