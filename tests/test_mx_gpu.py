"""4-bit block-scaled operands on the GPU against their definition in 64 bits."""
import numpy as np
import pytest
import torch

from rocwmma_b200 import BF16, COL_MAJOR, F16, F32, MXF4, NVF4, ROW_MAJOR, api
from tests import mx_reference as R

pytestmark = pytest.mark.gpu
TYPES = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}
FORMATS = pytest.mark.parametrize("fmt", [MXF4, NVF4], ids=["mxf4", "nvf4"])
KINDS = pytest.mark.parametrize("kind", [F16, BF16, F32], ids=["f16", "bf16", "f32"])


def _values(rows, k, kind, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    return x.to(TYPES[kind])


def _host(x):
    return x.double().cpu().numpy()


def _check_operand(fmt, rows, k, operand, x, exponent=0):
    codes, scales = (t.cpu().numpy() for t in operand)
    want_codes, want_scales, want_values = R.quantize(fmt, _host(x), exponent)
    got_codes, got_scales = R.unpack(fmt, rows, k, codes, scales)
    np.testing.assert_array_equal(got_scales, want_scales)
    # the sign of a zero is nobody's business
    np.testing.assert_array_equal(np.where(got_codes == 8, 0, got_codes), np.where(want_codes == 8, 0, want_codes))
    # nothing but zeros behind the last column, row and block
    plain = R.pack(fmt, got_codes, got_scales)
    np.testing.assert_array_equal(codes, plain[0])
    np.testing.assert_array_equal(scales, plain[1])
    return want_values


@FORMATS
@KINDS
@pytest.mark.parametrize("layout", [ROW_MAJOR, COL_MAJOR], ids=["rows", "columns"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 8192), (3, 31), (2, 33), (127, 64), (128, 128), (129, 257), (300, 1000),
                                    (40, 1204), (1100, 4152)])
def test_quantize(fmt, kind, layout, rows, k):
    x = _values(rows, k, kind, rows * 1000 + k)
    if rows > 2:
        x[1] = 0
    dev = (x.t().contiguous() if layout == COL_MAJOR else x).cuda()
    q = api.mx_quantize(fmt, kind, rows, k, dev, layout=layout)
    want = _check_operand(fmt, rows, k, q, x)
    # and back: codes and scales stand for numbers of at most seven bits
    for out in TYPES:
        got = api.mx_dequantize(fmt, out, rows, k, *q).view(rows, k)
        np.testing.assert_array_equal(_host(got), _host(torch.from_numpy(want).to(TYPES[out])))


@FORMATS
@KINDS
def test_quantize_borders(fmt, kind):
    """Values on and next to every border between two codes, for every scale mantissa."""
    block = R.BLOCK[fmt]
    mids = (R.E2M1[:-1] + R.E2M1[1:]) / 2
    eps = torch.finfo(TYPES[kind]).eps
    rows = []
    for s in np.arange(8, 16) / 8:  # the scale that the largest value makes: 6 s
        for m in mids:
            row = np.zeros(block)
            row[:4] = [m * s, m * s * (1 + eps), -m * s * (1 - eps), -m * s]
            row[4] = 6 * s
            rows.append(row)
    x = torch.tensor(np.array(rows)).to(TYPES[kind])
    for e in (0, -5, 3):
        q = api.mx_quantize(fmt, kind, *x.shape, x.cuda(), exponent=e)
        _check_operand(fmt, *x.shape, q, x, e)


@FORMATS
def test_quantize_extremes(fmt):
    """The smallest and largest values, infinities and NaN, one block each, in 32 bits."""
    block = R.BLOCK[fmt]
    x = torch.zeros(12, 2 * block)
    top = torch.finfo(torch.float32).max
    for i, v in enumerate([top, -top, 2.0 ** -126, 2.0 ** -149, 2.0 ** -127 * 1.5, 448 * 6, 449 * 6, 1e30,
                           2.0 ** -10 * 6, float("inf"), float("-inf"), float("nan")]):
        x[i, 3] = v
        x[i, 4] = v / 3 if np.isfinite(v) else 1.0
        x[i, block] = 1.0  # the neighbouring block is not concerned
    q = api.mx_quantize(fmt, F32, *x.shape, x.cuda())
    want = _check_operand(fmt, *x.shape, q, x)
    got = _host(api.mx_dequantize(fmt, F32, *x.shape, *q).view(x.shape))
    np.testing.assert_array_equal(got, want.astype(np.float32))
    assert np.isnan(got[9:, :block]).all() and np.isfinite(got[:, block:]).all()


@FORMATS
@pytest.mark.parametrize("kind", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layout", [ROW_MAJOR, COL_MAJOR], ids=["rows", "columns"])
def test_quantize_tiny_values_with_an_exponent(fmt, kind, layout):
    """Down to fp32's subnormals, brought into range by the exponent: factor / scale may overflow."""
    rows = torch.arange(-148, -90, dtype=torch.float64)
    x = (torch.rand(rows.numel(), 64, generator=torch.Generator().manual_seed(1), dtype=torch.float64) - 0.5)
    x = (x * 2.0 ** rows[:, None]).to(TYPES[kind])
    dev = (x.t().contiguous() if layout == COL_MAJOR else x).cuda()
    for e in (-64, -60, -31):
        q = api.mx_quantize(fmt, kind, *x.shape, dev, layout=layout, exponent=e)
        _check_operand(fmt, *x.shape, q, x, e)


@FORMATS
@pytest.mark.parametrize("layout", [ROW_MAJOR, COL_MAJOR], ids=["rows", "columns"])
def test_quantize_strides_and_offsets(fmt, layout):
    """A view inside a larger matrix that starts anywhere, into codes with room behind each row."""
    rows, k, ldx, ldq = 37, 75, 131, 96
    big = _values(140 if layout == ROW_MAJOR else k + 3, ldx, BF16, 5)
    flat = big.reshape(-1)[3:]
    x = (flat.as_strided((rows, k), (ldx, 1)) if layout == ROW_MAJOR else flat.as_strided((rows, k), (1, ldx)))
    dev = big.cuda().reshape(-1)[3:]
    codes = torch.full((rows * ldq,), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((api.mx_scale_bytes(fmt, rows, k),), 0x77, dtype=torch.uint8, device="cuda")
    api.mx_quantize(fmt, BF16, rows, k, dev, layout=layout, ldx=ldx, ldq=ldq, out=(codes, scales))
    codes = codes.view(rows, ldq)
    assert (codes[:, api.mx_pitch(k):] == 0x77).all()
    want = _check_operand(fmt, rows, k, (codes[:, :api.mx_pitch(k)].reshape(-1), scales), x)
    out = torch.full((rows * (k + 4),), 7.0, device="cuda")
    api.mx_dequantize(fmt, F32, rows, k, codes.view(-1), scales, ldq=ldq, ldo=k + 4, out=out)
    out = out.view(rows, k + 4)
    np.testing.assert_array_equal(_host(out[:, :k]), want)
    assert (out[:, k:] == 7).all()


@FORMATS
@pytest.mark.parametrize("exponent", [-64, -10, 0, 5, 64])
def test_dequantize_every_code_and_scale(fmt, exponent):
    """All codes under all scales, those no quantisation writes among them: 6 * 2^127 times a small power
    of two is a number again."""
    block, scales = R.BLOCK[fmt], np.arange(256 if fmt == MXF4 else 128, dtype=np.uint8)
    codes = np.tile(np.arange(16, dtype=np.uint8), (scales.size, block // 16))
    packed = [torch.from_numpy(t).cuda() for t in R.pack(fmt, codes, scales[:, None])]
    want = torch.from_numpy(R.values(fmt, codes, scales[:, None]) * 2.0 ** exponent)
    for out in (F32, BF16):
        got = api.mx_dequantize(fmt, out, scales.size, block, *packed, exponent=exponent).view(want.shape)
        # (at most seven bits: fp32, and then bf16, round what lies below their subnormals' steps alike)
        np.testing.assert_array_equal(_host(got), _host(want.float().to(TYPES[out])))


# ---- products ------------------------------------------------------------------------------------

def _small(fmt, rows, k, g):
    """An operand whose products and their sums fit 24 bits: any order of summation is exact."""
    codes = torch.randint(0, 16, (rows, k), generator=g).numpy()
    blocks = -(-k // R.BLOCK[fmt])
    if fmt == MXF4:
        scales = torch.randint(126, 129, (rows, blocks), generator=g).numpy().astype(np.uint8)  # 1/2, 1, 2
    else:
        pick = torch.randint(0, 4, (rows, blocks), generator=g).numpy()
        scales = np.array([48, 56, 60, 64], np.uint8)[pick]  # 1/2, 1, 3/2, 2
    packed = R.pack(fmt, codes.astype(np.uint8), scales)
    return tuple(torch.from_numpy(p).cuda() for p in packed), R.values(fmt, codes, scales)


def _product(fmt, out, m, n, k, seed, alpha=1.0, beta=0.0, c=None, ld=None):
    g = torch.Generator().manual_seed(seed)
    (a, av), (b, bv) = _small(fmt, m, k, g), _small(fmt, n, k, g)
    ld = ld or (n + 7) // 8 * 8
    dev = torch.full((m * ld,), 7.0, dtype=TYPES[out], device="cuda")
    if c is not None:
        c = torch.randint(-64, 64, (m, ld), generator=g).to(TYPES[out])
    api.mx_gemm(fmt, out, m, n, k, a, b, c.cuda() if c is not None else None, alpha, beta, ldc=ld, ldd=ld, out=dev)
    api.check_device()
    want = alpha * (av @ bv.T)
    if c is not None:
        want = want + beta * _host(c)[:, :n]
    dev = dev.view(m, ld)
    assert (dev[:, n:] == 7).all(), "written behind the last column"
    np.testing.assert_array_equal(_host(dev[:, :n]), _host(torch.from_numpy(want).to(TYPES[out])))


@FORMATS
@KINDS
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 64), (1, 1000, 520), (3, 130, 33), (16, 128, 256), (17, 257, 320),
                                   (64, 512, 512), (65, 100, 290), (128, 128, 128), (129, 384, 264), (200, 72, 1000),
                                   (257, 513, 72), (520, 300, 96)])
def test_gemm_exact(fmt, kind, m, n, k):
    _product(fmt, kind, m, n, k, m + n + k)


@FORMATS
@pytest.mark.parametrize("kind", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 264, 200), (40, 130, 96), (300, 260, 300)])
def test_gemm_alpha_beta(fmt, kind, m, n, k):
    _product(fmt, kind, m, n, k, 1, alpha=0.5, beta=-2.0, c=True)
    _product(fmt, kind, m, n, k, 2, alpha=-4.0, beta=1.0, c=True, ld=(n + 7) // 8 * 8 + 16)


@FORMATS
@KINDS
@pytest.mark.parametrize("m,n,k", [(1, 264, 4096), (33, 260, 2100), (16, 1000, 1100), (100, 500, 3000), (300, 9, 4096),
                                   (200, 72, 2100), (1030, 33, 1290)])
def test_gemm_thin_in_parts_with_c(fmt, kind, m, n, k):
    """K in two to eight parts, whose blocks each finish a share of the thin rows: C is read where D is written."""
    _product(fmt, kind, m, n, k, 3, alpha=0.5, beta=-2.0, c=True)
    _product(fmt, kind, m, n, k, 4, alpha=1.0, beta=1.0, c=True, ld=(n + 7) // 8 * 8 + 24)


@FORMATS
@KINDS
@pytest.mark.parametrize("m,n,k", [(2570, 5000, 200), (300, 20001, 328)])
def test_gemm_many_tiles(fmt, kind, m, n, k):
    """More tiles than the device has SMs: several to a block, the last ones ragged."""
    _product(fmt, kind, m, n, k, 5)
    _product(fmt, kind, m, n, k, 6, alpha=0.5, beta=-2.0, c=True)


@FORMATS
@pytest.mark.parametrize("m,n,k", [(1, 500, 4096), (33, 260, 2100), (300, 400, 1111)])
def test_gemm_rounding(fmt, m, n, k):
    """Full-range operands.  Each of the k products enters a fp32 sum that the tensor core may
    truncate instead of rounding: off by at most 2^-23 of the sum of magnitudes, k times."""
    x, w = _values(m, k, F32, 11), _values(n, k, F32, 12, 0.3)
    qa, qb = (api.mx_quantize(fmt, F32, *t.shape, t.cuda()) for t in (x, w))
    d = api.mx_gemm(fmt, F32, m, n, k, qa, qb, None, 1.0, 0.0, ldd=(n + 3) // 4 * 4)
    got = _host(d.view(m, -1)[:, :n])
    av, bv = R.quantize(fmt, _host(x))[2], R.quantize(fmt, _host(w))[2]
    bound = k * 2.0 ** -23 * (np.abs(av) @ np.abs(bv).T)
    assert (np.abs(got - av @ bv.T) <= bound).all()


@FORMATS
def test_gemm_not_a_number_stays_in_its_row_and_column(fmt):
    m, n, k = 40, 200, 300
    x, w = _values(m, k, BF16, 1), _values(n, k, BF16, 2)
    x[5, 7], w[140, 290] = float("inf"), float("nan")
    qa, qb = (api.mx_quantize(fmt, BF16, *t.shape, t.cuda()) for t in (x, w))
    d = api.mx_gemm(fmt, F32, m, n, k, qa, qb, None, 1.0, 0.0).view(m, n).cpu()
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[5], nan[:, 140] = True, True
    assert torch.equal(torch.isnan(d), nan)


@FORMATS
def test_gemm_beta_in_place_and_pitch(fmt):
    """D may be C; operands may have room behind each row of codes."""
    m, n, k, ld = 20, 136, 100, 112
    g = torch.Generator().manual_seed(3)
    (a, av), (b, bv) = _small(fmt, m, k, g), _small(fmt, n, k, g)
    wide = torch.full((m, ld), 0x55, dtype=torch.uint8, device="cuda")
    wide[:, :api.mx_pitch(k)] = a[0].view(m, -1)
    d = torch.randint(-8, 8, (m * n,), generator=g).float().cuda()
    want = av @ bv.T + _host(d).reshape(m, n)
    api.mx_gemm(fmt, F32, m, n, k, (wide.view(-1), a[1]), b, d, 1.0, 1.0, lda=ld, out=d)
    np.testing.assert_array_equal(_host(d).reshape(m, n), want)


@FORMATS
@pytest.mark.parametrize("m,n,k", [(1, 264, 4096), (300, 12, 4096), (100, 500, 3000), (1300, 2600, 200)])
def test_gemm_in_place(fmt, m, n, k):
    """D is C, in parts of K and over several tiles to a block."""
    g = torch.Generator().manual_seed(4)
    (a, av), (b, bv) = _small(fmt, m, k, g), _small(fmt, n, k, g)
    d = torch.randint(-8, 8, (m * n,), generator=g).float().cuda()
    want = 2 * (av @ bv.T) - _host(d).reshape(m, n)
    api.mx_gemm(fmt, F32, m, n, k, a, b, d, 2.0, -1.0, out=d)
    api.check_device()
    np.testing.assert_array_equal(_host(d).reshape(m, n), want)


@FORMATS
def test_gemm_of_an_operand_with_itself(fmt):
    g = torch.Generator().manual_seed(6)
    for rows, k in ((24, 600), (400, 600)):
        a, av = _small(fmt, rows, k, g)
        d = api.mx_gemm(fmt, F32, rows, rows, k, a, a, None, 1.0, 0.0)
        np.testing.assert_array_equal(_host(d).reshape(rows, rows), av @ av.T)


@FORMATS
@pytest.mark.parametrize("layout", [ROW_MAJOR, COL_MAJOR], ids=["rows", "columns"])
def test_quantize_behind_four_billion_values(fmt, layout):
    """Offsets that 32 bits do not hold; the last rows against the definition."""
    rows, k, tail = 70001, 62000, 70
    x = torch.zeros((rows, k) if layout == ROW_MAJOR else (k, rows), dtype=torch.bfloat16, device="cuda")
    end = _values(tail, k, BF16, 1)
    if layout == ROW_MAJOR:
        x[-tail:] = end.cuda()
    else:
        x[:, -tail:] = end.cuda().t()
    codes, scales = api.mx_quantize(fmt, BF16, rows, k, x, layout=layout)
    want = R.quantize(fmt, _host(end))[2]
    del x
    got = api.mx_dequantize(fmt, BF16, rows, k, codes, scales).view(rows, k)
    np.testing.assert_array_equal(_host(got[-tail:]), _host(torch.from_numpy(want).bfloat16()))
    for r in range(0, rows - tail, 5000):
        assert not got[r:min(r + 5000, rows - tail)].any()


@FORMATS
@pytest.mark.parametrize("m,n,k", [(70001, 62000, 96), (3, 2 ** 21 + 5, 4096), (2 ** 21 + 5, 20, 4096)])
def test_gemm_behind_four_billion_values(fmt, m, n, k):
    """D, or the codes of the streamed operand, of more than 2^32 values (4096 x 2^21 codes are 2^32 bytes)."""
    g = torch.Generator().manual_seed(9)
    tail = 40

    def operand(rows):
        """All rows zero but the last ones."""
        last = min(rows, tail)
        pitch, groups = api.mx_pitch(k), -(-k // (4 * R.BLOCK[fmt]))
        codes = torch.zeros(rows, pitch, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(-(-rows // 128), groups, 32, 4, 4, dtype=torch.uint8, device="cuda")
        (c, s), v = _small(fmt, last, k, g)
        codes[-last:] = c.view(last, pitch)
        plain = R.unpack(fmt, last, k, c.cpu().numpy(), s.cpu().numpy())[1]
        for i in range(last):
            r = rows - last + i
            row = np.zeros(groups * 4, np.uint8)
            row[:plain.shape[1]] = plain[i]
            scales[r // 128, :, r % 32, r // 32 % 4] = torch.from_numpy(row.reshape(groups, 4)).cuda()
        return (codes.view(-1), scales.view(-1)), v

    (a, av), (b, bv) = operand(m), operand(n)
    ld = (n + 7) // 8 * 8
    d = api.mx_gemm(fmt, F16, m, n, k, a, b, None, 0.125, 0.0, ldd=ld).view(m, ld)
    api.check_device()
    want = torch.from_numpy(0.125 * (av @ bv.T)).half()
    assert torch.equal(d[-av.shape[0]:, n - bv.shape[0]:n].cpu(), want)
    if m > tail:
        assert not d[:-tail, n - bv.shape[0]:n].any()
    if n > tail:
        assert not d[-av.shape[0]:, :n - tail].any()


def test_quantize_and_product_in_a_graph_and_on_a_stream():
    """Captured once, replayed on new inputs; the same on a stream of its own."""
    m, n, k = 5, 640, 1024
    w = _values(n, k, BF16, 3).cuda()
    qb = api.mx_quantize(MXF4, BF16, n, k, w)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")

    def step(stream=None):
        return api.mx_gemm(MXF4, BF16, m, n, k, api.mx_quantize(MXF4, BF16, m, k, x, stream=stream), qb, None, 1.0, 0.0,
                           stream=stream)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = step()
    for seed in (4, 5):
        x.copy_(_values(m, k, BF16, seed))
        graph.replay()
        xv, wv = R.quantize(MXF4, _host(x))[2], R.quantize(MXF4, _host(w))[2]
        want = xv @ wv.T
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        other = step(side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, d)
        # half a step of bf16 behind the fp32 sum's error
        bound = k * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)
        bound += 2.0 ** -8 * (np.abs(want) + bound)
        assert (np.abs(_host(d).reshape(m, n) - want) <= bound).all()


def test_products_on_several_streams_at_once():
    """Thin products, whose clusters hold tensor memory and wait for each other, and large ones beside
    them: every block that fits an SM finds the columns it needs."""
    g = torch.Generator().manual_seed(7)
    work = []
    for fmt, m, n, k in ((MXF4, 1, 4096, 1024), (NVF4, 100, 8192, 1024), (NVF4, 20, 2048, 2048), (MXF4, 400, 700, 512)):
        (a, av), (b, bv) = _small(fmt, m, k, g), _small(fmt, n, k, g)
        ld = (n + 7) // 8 * 8
        want = torch.from_numpy(av @ bv.T).float().cuda()
        work.append((fmt, m, n, k, a, b, ld, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        for fmt, m, n, k, a, b, ld, want, stream in work:
            results.append((m, n, api.mx_gemm(fmt, F32, m, n, k, a, b, None, 1.0, 0.0, ldd=ld, stream=stream), want))
    torch.cuda.synchronize()
    api.check_device()
    for m, n, d, want in results:
        assert torch.equal(d.view(m, -1)[:, :n], want)


@pytest.mark.parametrize("split", [0, 16, 31, 32])
def test_a_warp_gives_up_as_one(split):
    """Where a wait's limit passes for some lanes only, the warp that drains an accumulator has one answer."""
    import ctypes as C
    from rocwmma_b200 import _lib as L
    wait = C.CDLL(L.TEST_LIB_PATH).b200wmma_test_warp_wait
    wait.argtypes = [C.c_void_p, C.c_uint32, C.c_void_p]
    out = torch.full((64,), 7, dtype=torch.int32, device="cuda")
    assert wait(out.data_ptr(), split, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert out[:32].tolist() == [1] * split + [0] * (32 - split)
    assert out[32:].tolist() == [int(split == 32)] * 32


def test_clusters_beside_blocks_that_take_other_widths_of_tensor_memory():
    """Thin products of 64, 128 and 256 columns a block, K in one to eight parts, and a large one, all on
    streams of their own: ranges of every size come and go on an SM while the blocks of a cluster start."""
    g = torch.Generator().manual_seed(8)
    work = []
    for fmt, m, n, k in ((MXF4, 1, 2048, 4096), (MXF4, 40, 2048, 2048), (MXF4, 100, 2048, 4096), (MXF4, 3, 9000, 512),
                         (NVF4, 20, 4096, 2048), (NVF4, 50, 20000, 512), (NVF4, 128, 1024, 4096), (NVF4, 500, 600, 512)):
        (a, av), (b, bv) = _small(fmt, m, k, g), _small(fmt, n, k, g)
        out = [torch.full((m, n), 7.0, device="cuda") for _ in range(30)]
        work.append((fmt, m, n, k, a, b, torch.from_numpy(av @ bv.T).float().cuda(), out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(30):
        for fmt, m, n, k, a, b, _, out, stream in work:
            api.mx_gemm(fmt, F32, m, n, k, a, b, None, 1.0, 0.0, out=out[i], stream=stream)
    torch.cuda.synchronize()
    api.check_device()
    for *_, want, out, _ in work:
        for d in out:
            assert torch.equal(d, want)


@FORMATS
def test_linear_layer_and_its_gradients(fmt):
    """y = x W^T, dx = dy W and dW = dy^T x, each from operands quantised along the index it sums over."""
    m, n, k = 150, 200, 330
    x, w, dy = _values(m, k, BF16, 1), _values(n, k, BF16, 2, 0.2), _values(m, n, BF16, 3)

    def both(t, columns):
        """(operand, its values): the rows of t, or its columns."""
        rows, length = t.shape[::-1] if columns else t.shape
        q = api.mx_quantize(fmt, BF16, rows, length, t.cuda(), layout=COL_MAJOR if columns else ROW_MAJOR)
        return q, R.quantize(fmt, _host(t).T if columns else _host(t))[2]

    for a, b in ((both(x, False), both(w, False)), (both(dy, False), both(w, True)), (both(dy, True), both(x, True))):
        rows, cols, length = a[1].shape[0], b[1].shape[0], a[1].shape[1]
        ld = (cols + 3) // 4 * 4
        d = api.mx_gemm(fmt, F32, rows, cols, length, a[0], b[0], None, 1.0, 0.0, ldd=ld)
        bound = length * 2.0 ** -23 * (np.abs(a[1]) @ np.abs(b[1]).T)
        assert (np.abs(_host(d.view(rows, ld)[:, :cols]) - a[1] @ b[1].T) <= bound).all()
