"""What the 4-bit and embedding entry points refuse, and their sizes: needs no device."""
import ctypes as C

import numpy as np
import pytest
import torch

from rocwmma_b200 import MXF4, NVF4
from rocwmma_b200 import _lib as L
from rocwmma_b200 import api
from tests import mx_reference as R

P = C.c_void_p(256)
ODD = C.c_void_p(257)


def test_sizes():
    for k, pitch in ((1, 16), (32, 16), (33, 32), (8192, 4096), (2 ** 32 - 1, 2 ** 31)):
        assert L.lib().b200wmma_mx_pitch(k) == pitch == api.mx_pitch(k)
    for fmt in (MXF4, NVF4):
        for rows, k in ((1, 1), (128, 128), (129, 129), (300, 1000), (2 ** 31, 65536)):
            blocks = -(-k // R.BLOCK[fmt])
            assert api.mx_scale_bytes(fmt, rows, k) == -(-rows // 128) * -(-blocks // 4) * 512
    assert L.lib().b200wmma_mx_scale_bytes(L.F16, 128, 128) == 0


def test_reference_packing():
    """The test's own packing turns around, and puts one known scale where the header says."""
    rng = np.random.default_rng(0)
    for fmt in (MXF4, NVF4):
        rows, k = 200, 300
        codes = rng.integers(0, 16, (rows, k), dtype=np.uint8)
        scales = rng.integers(0, 255, (rows, -(-k // R.BLOCK[fmt])), dtype=np.uint8)
        c, s = R.pack(fmt, codes, scales)
        assert c.size == rows * api.mx_pitch(k) and s.size == api.mx_scale_bytes(fmt, rows, k)
        back = R.unpack(fmt, rows, k, c, s)
        assert np.array_equal(back[0], codes) and np.array_equal(back[1], scales)
        groups = s.size // 512 // 2
        assert s[(1 * groups + 1) * 512 + 5 * 16 + 1 * 4 + 3] == scales[128 + 32 + 5, 4 + 3]


def _quantize(fmt=MXF4, kind=L.BF16, rows=8, k=64, x=P, ldx=64, layout=0, exponent=0, codes=P, ldq=32, scales=P):
    return L.lib().b200wmma_mx_quantize(fmt, kind, rows, k, x, ldx, layout, exponent, codes, ldq, scales, None)


def test_quantize_refusals():
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(k=0), dict(ldx=63), dict(ldq=16),
                dict(layout=1, ldx=7), dict(layout=2), dict(exponent=65), dict(exponent=-65)):
        assert _quantize(**bad) == L.ERR_INVALID_ARG, bad
    for bad in (dict(fmt=L.E4M3), dict(fmt=11), dict(kind=L.F64), dict(kind=L.XF32), dict(kind=MXF4)):
        assert _quantize(**bad) == L.ERR_UNSUPPORTED, bad
    for bad in (dict(codes=C.c_void_p(8)), dict(scales=C.c_void_p(8)), dict(ldq=40), dict(x=ODD)):
        assert _quantize(**bad) == L.ERR_ALIGNMENT, bad
    assert _quantize(rows=2 ** 32 - 1, k=2 ** 20, ldx=2 ** 20, ldq=2 ** 19) == L.ERR_TOO_LARGE


def _gemm(fmt=MXF4, kind=L.F32, m=8, n=8, k=64, a=P, sa=P, b=P, sb=P, c=None, d=P, lda=32, ldb=32, ldc=8, ldd=8, beta=0.0):
    return L.lib().b200wmma_mx_gemm(fmt, kind, m, n, k, a, sa, b, sb, c, d, lda, ldb, ldc, ldd, 1.0, beta, None)


def test_gemm_refusals():
    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(d=None), dict(m=0), dict(n=0), dict(k=0),
                dict(lda=16), dict(ldb=16), dict(ldd=4), dict(beta=1.0), dict(beta=1.0, c=P, ldc=4)):
        assert _gemm(**bad) == L.ERR_INVALID_ARG, bad
    for bad in (dict(fmt=L.F16), dict(kind=L.I32), dict(kind=L.F64)):
        assert _gemm(**bad) == L.ERR_UNSUPPORTED, bad
    for bad in (dict(a=ODD), dict(sa=ODD), dict(b=ODD), dict(sb=ODD), dict(d=ODD), dict(lda=40), dict(ldb=40), dict(ldd=9),
                dict(beta=1.0, c=ODD), dict(beta=1.0, c=P, ldc=9)):
        assert _gemm(**bad) == L.ERR_ALIGNMENT, bad
    for bad in (dict(m=2 ** 31), dict(n=2 ** 31, ldd=2 ** 31), dict(k=2 ** 31, lda=2 ** 30, ldb=2 ** 30)):
        assert _gemm(**bad) == L.ERR_TOO_LARGE, bad


def _lookup(table_t=L.F16, out_t=L.F16, rows=9, dim=8, outer=3, inner=2, table=P, ldt=8, ids=P, id_bytes=8, first=None, out=P):
    return L.lib().b200wmma_embedding(table_t, out_t, rows, dim, outer, inner, table, ldt, ids, id_bytes, inner, 1, first,
                                      out, inner * dim, dim, 1.0, None)


def _gradient(table_t=L.F16, out_t=L.F16, rows=9, dim=8, outer=3, inner=2, table=P, ldt=8, ids=P, id_bytes=8, first=None, out=P,
              work=P, size=2 ** 40):
    return L.lib().b200wmma_embedding_grad(out_t, table_t, rows, dim, outer, inner, out, inner * dim, dim, ids, id_bytes, inner, 1,
                                           first, table, ldt, 1.0, 0, work, size, None)


def _rows_share_an_element(outer, a, inner, b, dim):
    starts = np.sort((np.arange(outer)[:, None] * a + np.arange(inner) * b).reshape(-1))
    return bool((np.diff(starts) < dim).any())


def test_lookup_refuses_rows_that_overlap():
    """Every small layout, against the rows written out; only those that overlap are called (there is no
    device to write to)."""
    def call(outer, a, inner, b, dim):
        return L.lib().b200wmma_embedding(L.F32, L.F32, 9, dim, outer, inner, P, dim, P, 8, inner, 1, None, P, a, b, 1.0, None)

    seen = 0
    for outer in (1, 2, 3, 7):
        for inner in (1, 2, 5):
            for a in range(0, 31):
                for b in range(0, 31):
                    if _rows_share_an_element(outer, a, inner, b, 4):
                        assert call(outer, a, inner, b, 4) == L.ERR_INVALID_ARG, (outer, a, inner, b)
                        seen += 1
    assert seen > 1000
    for outer, a, inner, b in ((2 ** 30, 3, 1, 0), (2, 2 ** 63, 2, 2 ** 63), (2 ** 15, 2 ** 15 * 4 - 1, 2 ** 15, 4),
                               (2 ** 15, 4, 2 ** 15, 2 ** 15 * 4 - 1)):
        assert call(outer, a, inner, b, 4) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("call", [_lookup, _gradient])
def test_embedding_refusals(call):
    for bad in (dict(table=None), dict(ids=None), dict(out=None), dict(rows=0), dict(dim=0), dict(outer=0), dict(inner=0),
                dict(ldt=7), dict(id_bytes=2)):
        assert call(**bad) == L.ERR_INVALID_ARG, bad
    for bad in (dict(table_t=L.F64), dict(out_t=L.E4M3), dict(table_t=MXF4)):
        assert call(**bad) == L.ERR_UNSUPPORTED, bad
    for bad in (dict(table=ODD), dict(out=ODD), dict(ids=C.c_void_p(4)), dict(first=C.c_void_p(4))):
        assert call(**bad) == L.ERR_ALIGNMENT, bad
    for bad in (dict(rows=2 ** 31 - 1), dict(outer=2 ** 31, inner=1), dict(outer=2 ** 20, inner=2 ** 11), dict(dim=2 ** 21, ldt=2 ** 21),
                dict(outer=2 ** 63, inner=2 ** 31)):
        assert call(**bad) == L.ERR_TOO_LARGE, bad


def test_gradient_workspace():
    need = api.embedding_grad_workspace(9, 8, 3, 2)
    assert need > 0
    assert _gradient(size=need - 1) == L.ERR_INVALID_ARG
    assert _gradient(work=None) == L.ERR_INVALID_ARG
    assert _gradient(work=C.c_void_p(16), size=need) == L.ERR_ALIGNMENT
    assert api.embedding_grad_workspace(9, 8, 2 ** 31) == 0 == api.embedding_grad_workspace(0, 8, 4)
    sizes = [api.embedding_grad_workspace(1000, 128, n) for n in (1, 100, 10000, 1000000, 2 ** 30)]
    assert sizes == sorted(sizes)


def test_wrappers_refuse_what_does_not_fit():
    cpu = torch.zeros(64, dtype=torch.uint8)
    with pytest.raises(ValueError):
        api.mx_quantize(MXF4, L.BF16, 1, 64, torch.zeros(64, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        api.mx_gemm(MXF4, L.F32, 1, 1, 1, (cpu, cpu), (cpu, cpu), None, 1.0, 0.0)
    with pytest.raises(ValueError):
        api.embedding(torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        api.embedding_grad(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), 4)
    with pytest.raises(ValueError):
        api.embedding_grad(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), 4, accumulate=True)
