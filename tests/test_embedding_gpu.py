"""Embedding lookup and its gradient on the GPU against sums in 64 bits."""
import numpy as np
import pytest
import torch

from rocwmma_b200 import BF16, F16, F32, api

pytestmark = pytest.mark.gpu
TYPES = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}
KINDS = pytest.mark.parametrize("kind", [F16, BF16, F32], ids=["f16", "bf16", "f32"])


def _ids(shape, rows, seed, skew=1.0, padding=0.2, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(shape, generator=g, dtype=torch.float64) ** skew * rows).long().clamp(max=rows - 1)
    ids = torch.where(torch.rand(shape, generator=g) < padding, -1, ids)
    return ids.to(dtype)


def _randn(shape, kind, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[kind])


@KINDS
@pytest.mark.parametrize("out_t", [F16, BF16, F32], ids=["to_f16", "to_bf16", "to_f32"])
@pytest.mark.parametrize("tokens,rows,dim", [(1, 1, 1), (1, 7, 8), (5, 3, 3), (63, 100, 96), (64, 1000, 1001),
                                             (1000, 50, 128), (257, 300, 2056), (20000, 40, 16),
                                             (3, 5, 4954), (700, 9, 1030), (2, 3, 40000), (2500, 30, 2304)])
def test_lookup(kind, out_t, tokens, rows, dim):
    table, ids = _randn((rows, dim), kind, 1), _ids((tokens,), rows, 2)
    for scale in (1.0, 0.3):
        got = api.embedding(table.cuda(), ids.cuda(), scale=scale, out_t=out_t)
        # a value of at most 24 bits times a 24-bit scale, rounded to fp32 and then to the output
        want = table.float()[ids.clamp(min=0)] * np.float32(scale)
        want = torch.where(ids[:, None] >= 0, want, 0.0).to(TYPES[out_t])
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=["int32", "int64"])
@pytest.mark.parametrize("dim", [128, 30])
def test_lookup_of_several_tables_into_the_interaction(dtype, dim):
    """Ids count within each table; the dense row in front of the picked ones is left alone."""
    outer, sizes = 100, [3, 1, 50, 7]
    first = torch.tensor([0, 3, 4, 54, 61])
    table = _randn((61, dim), F16, 1)
    ids = torch.stack([_ids((outer,), n, 3 + i) for i, n in enumerate(sizes)], 1)
    ids[0], ids[1] = torch.tensor([3, 1, 50, 7]), torch.tensor([2, 0, 49, 6])  # one behind the end, the last
    x = torch.full((outer, 5, dim), 7.0, dtype=torch.float16, device="cuda")
    api.embedding(table.cuda(), ids.to(dtype).cuda(), first=first.cuda(), out=x[:, 1:])
    want = torch.full((outer, 5, dim), 7.0, dtype=torch.float16)
    for i, n in enumerate(sizes):
        has = (ids[:, i] >= 0) & (ids[:, i] < n)
        rows = table[first[i] + ids[:, i].clamp(0, n - 1)]
        want[:, 1 + i] = torch.where(has[:, None], rows, 0.0)
    assert torch.equal(x.cpu(), want)


def test_tables_that_run_backwards_or_past_the_end_have_no_rows():
    """Their ids read as zeros and have no gradient; also where the length would wrap in 64 bits."""
    least, most = -2 ** 63, 2 ** 63 - 1
    for first in ([10, least, 0, 30], [10, 5, 31, 12], [least, most, least, 30], [most, least, 1, most]):
        legal = [0 <= a <= b <= 30 for a, b in zip(first, first[1:])]
        table, ids = _randn((30, 8), F32, 1), torch.tensor([[0, 1, 2], [5, -1, 7], [most, least, 2 ** 40]])
        at = torch.tensor(first, device="cuda")
        got = api.embedding(table.cuda(), ids.cuda(), first=at).cpu()
        grad = api.embedding_grad(torch.ones(3, 3, 8, device="cuda"), ids.cuda(), 30, first=at).cpu()
        want, sums = torch.zeros(3, 3, 8), torch.zeros(30, 8)
        for o in range(3):
            for i in range(3):
                if legal[i] and 0 <= int(ids[o, i]) < first[i + 1] - first[i]:
                    want[o, i] = table[first[i] + ids[o, i]]
                    sums[first[i] + ids[o, i]] += 1
        assert torch.equal(got, want) and torch.equal(grad, sums)


def test_lookup_strides():
    """Rows of a wider table, transposed ids, an output with room between its rows."""
    wide = _randn((40, 37), F32, 1)
    ids = _ids((6, 10), 40, 2)
    out = torch.full((6, 10, 20), 7.0, device="cuda")
    api.embedding(wide.cuda()[:, 3:19], ids.t().contiguous().cuda().t(), out=out[:, :, 2:18], scale=2.0)
    want = torch.full((6, 10, 20), 7.0)
    want[:, :, 2:18] = torch.where(ids[..., None] >= 0, 2 * wide[ids.clamp(min=0), 3:19], 0.0)
    assert torch.equal(out.cpu(), want)
    # an id of any size outside the table picks nothing
    far = torch.tensor([2 ** 31, 2 ** 32 + 1, -2 ** 40, 40, 39], device="cuda")
    got = api.embedding(wide.cuda(), far).cpu()
    assert torch.equal(got[:4], torch.zeros(4, 37)) and torch.equal(got[4], wide[39])


def test_lookup_into_rows_that_interleave_and_rows_that_overlap():
    """Any layout whose rows share no element is written; the others are refused."""
    table, dim = _randn((9, 4), F32, 1), 4
    for outer, inner in ((1, 5), (2, 3), (3, 2), (7, 2), (4, 1)):
        ids = _ids((outer, inner), 9, outer)
        want = torch.where(ids[..., None] >= 0, table[ids.clamp(min=0)], 0.0)
        for a in range(0, 25):
            for b in range(0, 25):
                flat = torch.full((400,), 7.0, device="cuda")
                out = flat.as_strided((outer, inner, dim), (a, b, 1))
                starts = (torch.arange(outer)[:, None] * a + torch.arange(inner) * b).reshape(-1).sort().values
                if (starts.diff() < dim).any():
                    with pytest.raises(ValueError):
                        api.embedding(table.cuda(), ids.cuda(), out=out)
                    assert (flat == 7).all()
                else:
                    api.embedding(table.cuda(), ids.cuda(), out=out)
                    assert torch.equal(out.cpu(), want)
                    assert int((flat != 7).sum()) <= outer * inner * dim


def _grad_reference(grad, ids, rows, scale=1.0, old=None):
    """(sum, sum of magnitudes, tokens) of every row in 64 bits."""
    flat, g = ids.reshape(-1).numpy(), grad.double().reshape(-1, grad.shape[-1]).numpy()
    total, size, count = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1])), np.zeros(rows)
    ok = (flat >= 0) & (flat < rows)
    np.add.at(total, flat[ok], g[ok])
    np.add.at(size, flat[ok], np.abs(g[ok]))
    np.add.at(count, flat[ok], 1)
    return total, size, count


def _check_grad(got, grad, ids, rows, kind, scale=1.0, old=None):
    """Each of a row's n additions and the scaling round to fp32 (2^-24 of a partial sum, which is
    no larger than the sum of magnitudes); one more rounding to the result's type."""
    total, size, count = _grad_reference(grad, ids, rows)
    scale = float(np.float32(scale))
    want, bound = total * scale, (count + 1)[:, None] * 2.0 ** -24 * size * abs(scale)
    if old is not None:
        want = want + old
        bound = bound + 2.0 ** -24 * (np.abs(old) + size * abs(scale))
    got = got.double().cpu().numpy()
    step = torch.finfo(TYPES[kind]).eps / 2
    tiny = torch.finfo(TYPES[kind]).smallest_normal * torch.finfo(TYPES[kind]).eps  # subnormal results
    err = np.abs(got - want)
    assert (err <= bound + step * (np.abs(want) + bound) + tiny / 2).all(), err.max()
    assert np.array_equal(got[count == 0], (old if old is not None else np.zeros_like(want))[count == 0])


@KINDS
@pytest.mark.parametrize("out_t", [F16, BF16, F32], ids=["to_f16", "to_bf16", "to_f32"])
@pytest.mark.parametrize("tokens,rows,dim,skew", [(1, 1, 1, 1), (1, 5, 8, 1), (40, 1, 3, 1), (33, 70, 264, 1), (513, 90, 1001, 4),
                                                  (4097, 300, 64, 4), (5000, 70000, 24, 1), (9000, 2, 40, 1),
                                                  (4096, 300, 64, 4), (4100, 40000, 400, 2)])
def test_gradient(kind, out_t, tokens, rows, dim, skew):
    grad, ids = _randn((tokens, dim), kind, 1), _ids((tokens,), rows, 2, skew)
    for scale in (1.0, 0.3):
        got = api.embedding_grad(grad.cuda(), ids.cuda(), rows, out_t=out_t, scale=scale)
        _check_grad(got, grad, ids, rows, out_t, scale)


@pytest.mark.parametrize("tokens,rows,dim", [(300000, 40, 8), (70000, 1, 16), (200000, 100000, 3), (60000, 5000, 8),
                                             (16385, 300, 520), (65536, 5000, 8), (65537, 5000, 8),
                                             (700000, 3000, 4), (2000001, 3000, 4)])
def test_gradient_of_long_runs(tokens, rows, dim):
    """Rows that most tokens share: runs over many chunks and levels; every bit the same again."""
    grad, ids = _randn((tokens, dim), BF16, 1), _ids((tokens,), rows, 2, 6.0)
    got = api.embedding_grad(grad.cuda(), ids.cuda(), rows, out_t=F32)
    _check_grad(got, grad, ids, rows, F32)
    for _ in range(3):
        assert torch.equal(api.embedding_grad(grad.cuda(), ids.cuda(), rows, out_t=F32), got)


def test_gradient_of_nothing():
    """No token has a row: zeros, or what was there."""
    grad, ids = _randn((50, 24), F32, 1).cuda(), torch.full((50,), -1, device="cuda")
    assert not api.embedding_grad(grad, ids, 30).any()
    old = _randn((30, 24), F32, 2).cuda()
    got = api.embedding_grad(grad, ids, 30, out=old.clone(), accumulate=True)
    assert torch.equal(got, old)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert not api.embedding_grad(grad[:0], none, 30).any()
    assert api.embedding(old, none).shape == (0, 24)


@pytest.mark.parametrize("dim", [64, 50])
def test_gradient_accumulates_into_views(dim):
    """Into the first columns of a wider gradient, from the rows behind the interaction's dense one."""
    outer, inner, rows = 70, 3, 25
    grad = _randn((outer, inner + 1, dim), F16, 1)
    sizes, first = [5, 12, 8], torch.tensor([0, 5, 17, 25])
    ids = torch.stack([_ids((outer,), n, 3 + i) for i, n in enumerate(sizes)], 1)
    old = _randn((rows, dim + 8), F32, 9)
    wide = old.cuda()
    got = api.embedding_grad(grad.cuda()[:, 1:], ids.int().cuda(), rows, first=first.cuda(), scale=0.5,
                             out=wide[:, :dim], accumulate=True)
    assert torch.equal(wide[:, dim:].cpu(), old[:, dim:])
    flat = torch.where(ids >= 0, ids + first[:-1], -1)
    _check_grad(got, grad[:, 1:], flat, rows, F32, 0.5, old[:, :dim].double().numpy())


@pytest.mark.parametrize("tokens,rows,dim,skew", [(70000, 300, 64, 6.0), (30000, 2000, 520, 2.0), (5000, 40, 1032, 4.0),
                                                  (3000, 7, 2304, 1.0)])
@pytest.mark.parametrize("grad_off,grad_ld,out_off,out_ld", [(1, 0, 0, 0), (0, 0, 1, 0), (0, 1, 0, 0), (0, 0, 0, 1), (4, 0, 2, 4),
                                                             (2, 2, 1, 3)])
def test_gradient_off_the_boundary(tokens, rows, dim, skew, grad_off, grad_ld, out_off, out_ld):
    """Rows of a multiple of eight that start or follow each other off the boundary: pieces narrower than the
    workspace is planned for, of the gradient and of the table apart, over many parts."""
    grad, ids = _randn((tokens, dim), BF16, 1), _ids((tokens,), rows, 2, skew)
    g = torch.full((grad_off + tokens * (dim + grad_ld),), float("nan"), dtype=torch.bfloat16, device="cuda")
    g = g[grad_off:].view(tokens, dim + grad_ld)[:, :dim]
    g.copy_(grad)
    for kind in (F32, F16):
        flat = torch.full((out_off + rows * (dim + out_ld) + 8,), 7.0, dtype=TYPES[kind], device="cuda")
        out = flat[out_off:out_off + rows * (dim + out_ld)].view(rows, dim + out_ld)[:, :dim]
        api.embedding_grad(g, ids.cuda(), rows, out=out)
        _check_grad(out, grad, ids, rows, kind)
        old = out.clone()
        api.embedding_grad(g, ids.cuda(), rows, out=out, accumulate=True, scale=0.5)
        _check_grad(out, grad, ids, rows, kind, 0.5, old.double().cpu().numpy())
        out.fill_(7.0)
        assert (flat == 7).all()


def test_gradient_is_the_lookups():
    """<grad, embedding(table)> grows with the table as the gradient says: differences in 64 bits of a
    function that is linear in the table."""
    rows, dim = 30, 16
    table, ids, g = _randn((rows, dim), F32, 1), _ids((200,), rows, 2), _randn((200, dim), F32, 3)
    grad = api.embedding_grad(g.cuda(), ids.cuda(), rows, scale=1.5).double().cpu()
    step = _randn((rows, dim), F32, 4)
    up = api.embedding((table + step).cuda(), ids.cuda(), scale=1.5).double().cpu()
    down = api.embedding((table - step).cuda(), ids.cuda(), scale=1.5).double().cpu()
    moved = (((table + step).double() - (table - step).double()) * grad).sum()
    # fp32 roundings: of each looked-up value (2^-24), and those of the gradient's sums (at most 200 a row)
    size = (g.abs().double() * (up.abs() + down.abs())).sum()
    assert abs(((up - down) * g.double()).sum() - moved) <= 202 * 2.0 ** -24 * size


def test_values_of_tokens_without_a_row_reach_nothing():
    """Infinities and NaN beside ids of no row, in the gradient and in rows that nothing picks."""
    for tokens, rows, dim in ((70, 9, 24), (5000, 40, 33), (20000, 3000, 64)):
        ids = _ids((tokens,), rows, 1, 2.0, 0.3)
        ids[3], ids[5] = rows, -2 ** 40
        grad = _randn((tokens, dim), F32, 2)
        grad[(ids < 0) | (ids >= rows)] = torch.tensor([float("nan"), float("inf")]).repeat(dim)[:dim]
        got = api.embedding_grad(grad.cuda(), ids.cuda(), rows)
        _check_grad(got, torch.nan_to_num(grad, 0, 0, 0), ids, rows, F32)
        table = _randn((rows, dim), F32, 3)
        table[rows // 2] = float("nan")
        ids[ids == rows // 2] = -1
        out = api.embedding(table.cuda(), ids.cuda(), scale=0.0)
        assert not out.any()


def test_gradients_and_lookups_on_several_streams_at_once():
    """Calls that overlap, each with the workspace it allocates, give what they give alone."""
    work = []
    for i, (tokens, rows, dim) in enumerate(((300, 50, 64), (40000, 900, 40), (9000, 70000, 24), (2000, 3000, 128))):
        grad, ids = _randn((tokens, dim), BF16, i).cuda(), _ids((tokens,), rows, i, 3.0).cuda()
        table = _randn((rows, dim), F16, i).cuda()
        alone = api.embedding_grad(grad, ids, rows, out_t=F32), api.embedding(table, ids, scale=3.0)
        work.append((grad, ids, rows, table, alone, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for grad, ids, rows, table, alone, stream in work:
            got.append((alone, api.embedding_grad(grad, ids, rows, out_t=F32, stream=stream),
                        api.embedding(table, ids, scale=3.0, stream=stream)))
    torch.cuda.synchronize()
    for alone, total, picked in got:
        assert torch.equal(total, alone[0]) and torch.equal(picked, alone[1])


def test_rows_behind_four_billion_values():
    """Offsets that 32 bits do not hold: of the table, the output, the gradient and the table's gradient."""
    rows, dim = 1050000, 4104
    ids = torch.tensor([0, rows - 1, -1, rows - 2, rows - 1], device="cuda")
    some = _randn((5, dim), F16, 1).cuda()
    table = torch.zeros(rows, dim, dtype=torch.float16, device="cuda")
    table[ids[[0, 1, 3]]] = some[:3]
    picked = api.embedding(table, ids)
    assert torch.equal(picked, torch.stack([some[0], some[1], torch.zeros_like(some[0]), some[2], some[1]]))
    grad = api.embedding_grad(some, ids, rows, out=table)
    want = torch.stack([some[0].float(), some[1].float() + some[4].float(), some[3].float()]).half()
    assert torch.equal(grad[ids[[0, 1, 3]]], want)
    grad[ids[[0, 1, 3]]] = 0
    for r in range(0, rows, 50000):
        assert not grad[r:r + 50000].any()
    # as many tokens: the output, and the gradient that is read
    many = torch.full((rows,), -1, device="cuda")
    many[0], many[-1], many[-2] = 1, 2, 1
    out = api.embedding(some, many, out=table)
    assert torch.equal(out[[0, -2, -1]], some[[1, 1, 2]]) and not out[1:-2:1000].any()
    total = api.embedding_grad(out, many, 5, out_t=F32)
    want = torch.zeros(5, dim, device="cuda")
    want[1], want[2] = 2 * some[1].float(), some[2].float()
    assert torch.equal(total, want)


def test_dlrm_step():
    """Lookup -> interaction -> 4-bit product, and back through the interaction to the tables."""
    from rocwmma_b200 import MXF4
    from tests import mx_reference as R

    batch, dim, sizes = 48, 32, [4, 30, 9]
    m = len(sizes) + 1
    first = torch.tensor([0, 4, 34, 43])
    table, dense = _randn((43, dim), F16, 1), _randn((batch, dim), F16, 2)
    ids = torch.stack([_ids((batch,), n, 3 + i, padding=0) for i, n in enumerate(sizes)], 1)
    x = torch.empty(batch, m, dim, dtype=torch.float16, device="cuda")
    x[:, 0] = dense.cuda()
    api.embedding(table.cuda(), ids.cuda(), first=first.cuda(), out=x[:, 1:])
    width = dim + m * (m - 1) // 2
    z = api.dlrm_fwd(x, m, dim, batch).view(batch, width)
    weight = _randn((64, width), F16, 7)
    qz = api.mx_quantize(MXF4, F16, batch, width, z)
    qw = api.mx_quantize(MXF4, F16, 64, width, weight.cuda())
    y = api.mx_gemm(MXF4, F32, batch, 64, width, qz, qw, None, 1.0, 0.0).view(batch, 64)
    zv, wv = (R.quantize(MXF4, t.double().cpu().numpy())[2] for t in (z, weight))
    bound = width * 2.0 ** -23 * (np.abs(zv) @ np.abs(wv).T)
    assert (np.abs(y.double().cpu().numpy() - zv @ wv.T) <= bound).all()

    upstream = _randn((batch, width), F16, 8).cuda()
    _, grad = api.dlrm_bwd(x, upstream, m, dim, batch)
    grad = grad.view(batch, m, dim)
    total = api.embedding_grad(grad[:, 1:], ids.cuda(), 43, out_t=F32, first=first.cuda())
    _check_grad(total, grad[:, 1:].cpu(), ids + first[:-1], 43, F32)


def test_graph_replays_with_new_tokens_and_shares_a_workspace():
    """Two captured gradients, one workspace, replayed one after the other."""
    rows, dim, n = 500, 48, 3000
    ids, grad = _ids((n,), rows, 1).cuda(), _randn((n, dim), BF16, 2).cuda()
    work = torch.empty(api.embedding_grad_workspace(rows, dim, n), dtype=torch.uint8, device="cuda")
    outs, graphs = [torch.empty(rows, dim, device="cuda") for _ in range(2)], []
    api.embedding_grad(grad, ids, rows, out=outs[0], workspace=work)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            api.embedding_grad(grad, ids, rows, out=out, workspace=work, scale=1.0 + i)
        graphs.append(g)
    for seed in (3, 4):
        ids.copy_(_ids((n,), rows, seed, 3.0))
        grad.copy_(_randn((n, dim), BF16, seed))
        for g in graphs:
            g.replay()
        for i, out in enumerate(outs):
            _check_grad(out, grad.cpu(), ids.cpu(), rows, F32, 1.0 + i)
