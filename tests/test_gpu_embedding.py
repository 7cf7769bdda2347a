"""GPU (-m gpu): the row lookup and its gradients against the formula in 64 bits.

u = 2^-24 (fp32), t = half a step of the table's or the result's type (bf16 2^-8, fp16 2^-11, fp32 0 once u is counted).
out: the product of scale and row: u, and t.  d_table: k entries added in fp32 in whatever pieces: at most k u sum|terms|, one
u more for the term of a plain product, and t.  d_scale: the same over the width.  Where the data are small whole numbers
every sum is exact and the results have to be equal, however often a row is hit."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
T = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}
u = 2.0 ** -24


def _ids(kind, n, rows, rng):
    if kind == "uniform":
        return rng.integers(0, rows, n)
    if kind == "same":
        return np.full(n, rows // 2)
    if kind == "hot":                                       # half of the entries in one row
        return np.where(rng.uniform(size=n) < 0.5, rows // 3, rng.integers(0, rows, n))
    if kind == "runs":                                      # sorted already, long runs
        return np.sort(rng.integers(0, max(rows // 8, 1), n))
    if kind == "ends":
        return np.where(rng.uniform(size=n) < 0.5, 0, rows - 1)
    if kind == "none":
        return np.full(n, -1)
    ids = rng.integers(0, rows, n)                          # "holes": no row, in every way there is
    bad = rng.uniform(size=n) < 0.4
    return np.where(bad, rng.choice([-1, rows, rows + 1, -2 ** 31, 2 ** 31 - 1], n), ids)


def _inputs(n, rows, width, kind="uniform", dtype=F32, out=None, scale="row", index=torch.int64, seed=0, whole=False):
    rng = np.random.default_rng(seed)
    draw = (lambda *s: rng.integers(-3, 4, s).astype(np.float64)) if whole else (lambda *s: rng.normal(size=s))
    table = torch.tensor(draw(rows, width)).to(dtype).to(DEV)
    g = torch.tensor(draw(n, width)).to(out or dtype).to(DEV)
    ids = torch.tensor(_ids(kind, n, rows, rng), dtype=index, device=DEV)
    if scale == "row":
        scale = torch.tensor(rng.choice([0.5, 1.0, 2.0, -1.0], n) if whole else rng.normal(size=n), dtype=F32, device=DEV)
    return table, ids, scale, g


def _run(table, ids, scale, g, dtype=None):
    from vegs_amd import embedding
    table = table.detach().requires_grad_(True)
    wanted = [table]
    if isinstance(scale, torch.Tensor):
        scale = scale.detach().requires_grad_(True)
        wanted.append(scale)
    out = embedding.lookup(table, ids, scale, dtype=dtype)
    grads = torch.autograd.grad(out, wanted, g)
    return out.detach(), grads[0], grads[1] if len(grads) > 1 else None


def _formula(table, ids, scale, g):
    """(out, d_table, sum of the terms' magnitudes, entries per row, d_scale, its terms' magnitudes) in 64 bits on the CPU"""
    table, g, ids = table.detach().double().cpu(), g.double().cpu(), ids.cpu().long()
    rows, width = table.shape
    there = (ids >= 0) & (ids < rows)
    at = ids[there]
    s = scale.detach().double().cpu() if isinstance(scale, torch.Tensor) else torch.full((len(ids),), 1.0 if scale is None else float(scale)).double()
    out, d_scale, m_scale = torch.zeros(len(ids), width).double(), torch.zeros(len(ids)).double(), torch.zeros(len(ids)).double()
    out[there] = s[there, None] * table[at]
    terms = s[there, None] * g[there]
    d_table, m_table = torch.zeros(rows, width).double(), torch.zeros(rows, width).double()
    d_table.index_add_(0, at, terms)
    m_table.index_add_(0, at, terms.abs())
    d_scale[there] = (g[there] * table[at]).sum(1)
    m_scale[there] = (g[there] * table[at]).abs().sum(1)
    return out, d_table, m_table, torch.bincount(at, minlength=rows).double(), d_scale, m_scale


def _check(table, ids, scale, g, dtype=None, exact=False):
    out, d_table, d_scale = _run(table, ids, scale, g, dtype)
    w_out, w_table, m_table, k, w_scale, m_scale = _formula(table, ids, scale, g)
    assert out.dtype == (dtype or table.dtype) and d_table.dtype == table.dtype and d_table.shape == table.shape
    out, d_table = out.double().cpu(), d_table.double().cpu()
    if exact:
        assert torch.equal(out, w_out) and torch.equal(d_table, w_table.to(table.dtype).double())
    assert ((out - w_out).abs() <= (2 * u + T[g.dtype]) * w_out.abs() + TINY[g.dtype]).all()
    off = (k[:, None] + 2) * u * m_table
    assert ((d_table - w_table).abs() <= off + T[table.dtype] * (w_table.abs() + off) + TINY[table.dtype]).all()
    assert (d_table[k == 0] == 0).all() and (out[(ids.cpu() < 0) | (ids.cpu() >= len(table))] == 0).all()
    if d_scale is not None:
        assert d_scale.dtype == F32
        if exact:
            assert torch.equal(d_scale.double().cpu(), w_scale)
        assert ((d_scale.double().cpu() - w_scale).abs() <= (table.shape[1] + 2) * u * m_scale).all()


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 8, 9, 10, 15, 16, 17, 31, 32, 33, 45, 48, 63, 64, 65, 127, 128, 129, 255, 256,
                                   257, 300, 511, 512, 513, 1000, 1025, 2048, 2051, 5000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_widths(width, dtype):
    _check(*_inputs(300, 41, width, "holes", dtype, seed=width))
    _check(*_inputs(700, 200, width, "hot", dtype, seed=width + 1, scale=0.25))


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("width", [3, 8, 45, 130, 600])
@pytest.mark.parametrize("scale", ["row", None, -1.75])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_types(dtype, out, width, scale, index):
    table, ids, scale, g = _inputs(1000, 77, width, "holes", dtype, out, scale, index, seed=3)
    _check(table, ids, scale, g, out)


# more entries than one workgroup sorts alone (1024), and more than sixteen sort by ranges of rows (16384): sums in chunks
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 33, 45, 48, 64, 65, 128, 129, 255, 257, 512, 513, 1025, 2051])
@pytest.mark.parametrize("n,kind", [(1500, "holes"), (5000, "hot"), (17000, "holes"), (17000, "ends")])
def test_widths_in_chunks(width, n, kind):
    _check(*_inputs(n, 300, width, kind, seed=width, whole=True), exact=True)
    _check(*_inputs(n, 300, width, kind, BF16, seed=width + 1))


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("width", [3, 8, 45, 600])
@pytest.mark.parametrize("scale", ["row", None, -1.75])
@pytest.mark.parametrize("n", [3000, 20000])
def test_types_in_chunks(dtype, out, width, scale, n):
    for index in (torch.int32, torch.int64):
        table, ids, scale_, g = _inputs(n, 700, width, "holes", dtype, out, scale, index, seed=3)
        _check(table, ids, scale_, g, out)


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 255, 256, 4095, 4096, 70000])
@pytest.mark.parametrize("n", [1025, 16384, 16385])
@pytest.mark.parametrize("kind", ["uniform", "same", "holes"])
def test_rows_at_the_borders_of_the_sorts(rows, n, kind):
    _check(*_inputs(n, rows, 6, kind, seed=rows, whole=True), exact=True)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096,
                               4097, 8193, 20011])
@pytest.mark.parametrize("kind", ["uniform", "same", "hot", "runs", "ends", "holes", "none"])
def test_lengths_and_patterns(n, kind):
    _check(*_inputs(n, 500, 12, kind, seed=n, whole=True), exact=True)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 255, 256, 257, 511, 512, 513, 8192, 65535, 65536, 65537, 300007])
@pytest.mark.parametrize("n", [5, 3000])
def test_numbers_of_rows(rows, n):
    _check(*_inputs(n, rows, 5, "holes", seed=rows, whole=True), exact=True)


@pytest.mark.parametrize("kind", ["same", "hot", "uniform", "ends", "runs"])
@pytest.mark.parametrize("width", [1, 45, 300])
def test_rows_hit_a_hundred_thousand_times(kind, width):
    """Whole numbers: equal, so that no entry is lost or taken twice where a row's sum goes through many pieces."""
    n = 250007 if width < 300 else 100003
    _check(*_inputs(n, 900, width, kind, seed=8, whole=True), exact=True)


def test_long_sums_keep_their_precision():
    """250007 entries of one row: pieces that are joined, not one running sum (whose bound is thousands of times as wide).  A
    piece adds at most 64 entries, and the pieces are joined in at most 64 + 64 + 64 further additions on any path."""
    table, ids, scale, g = _inputs(250007, 900, 45, "same", seed=8)
    _, d_table, _ = _run(table, ids, scale, g)
    _, want, terms, _, _, _ = _formula(table, ids, scale, g)
    assert ((d_table.double().cpu() - want).abs() <= 256 * u * terms).all()


def test_the_same_bits_every_time():
    args = _inputs(50000, 300, 45, "hot", seed=4)
    first = _run(*args)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _run(*args)))


def test_gradients_against_differences():
    """The result is linear in the table and in the scales: with whole numbers the differences are exact."""
    from vegs_amd import embedding
    table, ids, scale, g = _inputs(500, 30, 45, "holes", seed=6, whole=True)
    _, d_table, d_scale = _run(table, ids, scale, g)
    rng = np.random.default_rng(1)
    dt = torch.tensor(rng.integers(-3, 4, tuple(table.shape)), dtype=F32, device=DEV)
    ds = torch.tensor(rng.integers(-3, 4, tuple(scale.shape)), dtype=F32, device=DEV)
    value = lambda t, s: (embedding.lookup(t, ids, s).double() * g.double()).sum().item()
    assert value(table + dt, scale) - value(table, scale) == (d_table.double() * dt.double()).sum().item()
    assert value(table, scale + ds) - value(table, scale) == (d_scale.double() * ds.double()).sum().item()


def test_what_stands_where_there_is_no_row_does_not_matter():
    table, ids, scale, g = _inputs(400, 30, 20, "holes", seed=7)
    gone = (ids < 0) | (ids >= 30)
    want = _run(table, ids, scale, g)
    g[gone] = math.nan
    scale[gone] = math.inf
    for a, b in zip(want, _run(table, ids, scale, g)):
        assert torch.equal(a, b)
    far = torch.tensor([2 ** 40, -2 ** 63, 2 ** 63 - 1, 2 ** 32, 2 ** 32 + 3, 3], device=DEV)        # 64-bit ids are not cut
    out, d_table, d_scale = _run(table, far, scale[:6].nan_to_num(posinf=1.0), torch.ones(6, 20, device=DEV))
    assert (out[:5] == 0).all() and (out[5] != 0).any() and (d_scale[:5] == 0).all()
    assert (d_table[3] != 0).all() and d_table.count_nonzero().item() == 20


def test_infinities_and_nans_reach_their_rows_only():
    table, ids, scale, g = _inputs(600, 25, 9, "uniform", seed=9)
    table[4, 2] = math.inf
    g[17, 5] = math.nan
    out, d_table, d_scale = _run(table, ids, scale, g)
    assert out.isfinite().all(1).logical_not().equal(ids == 4)
    at = ids[17].item()
    assert d_table[at, 5].isnan() and d_table.isnan().sum().item() == 1
    bad = (ids == 4)
    bad[17] = True
    assert d_scale.isfinite().logical_not().equal(bad)


def test_shapes_and_layouts():
    from vegs_amd import embedding
    rng = np.random.default_rng(2)
    whole = torch.tensor(rng.normal(size=(50, 16, 3)), dtype=F32, device=DEV)
    ids = torch.tensor(rng.integers(-1, 50, (6, 40)), device=DEV)
    # a part of wider rows; ids and scales that do not lie in order; more than one dimension of ids
    table = whole[:, 1:]
    scale = torch.tensor(rng.normal(size=(40, 6)), dtype=F32, device=DEV).t()
    out = embedding.lookup(table, ids, scale)
    want = torch.where((ids >= 0)[..., None, None], table[ids.clamp(min=0)] * scale[..., None, None], 0.0)
    assert out.shape == (6, 40, 15, 3) and torch.equal(out, want)
    assert torch.equal(embedding.lookup(table, ids.t()), torch.where((ids >= 0).t()[..., None, None], table[ids.t().clamp(min=0)], 0.0))
    # the gradient through a view of the parameter, and one that arrives as a part of wider rows
    leaf = whole.clone().requires_grad_(True)
    flat = ids.reshape(-1)
    wide = torch.cat((torch.zeros(240, 1, 3, device=DEV), embedding.lookup(leaf[:, 1:], flat)), 1)
    g = torch.tensor(rng.normal(size=(240, 16, 3)), dtype=F32, device=DEV)
    wide.backward(g)
    _, want, terms, k, _, _ = _formula(whole[:, 1:].reshape(50, 45), flat, None, g[:, 1:].reshape(240, 45))
    assert (leaf.grad[:, 0] == 0).all()
    assert ((leaf.grad[:, 1:].reshape(50, 45).double().cpu() - want).abs() <= (k[:, None] + 2) * u * terms).all()
    # one value for all, expanded: .sum()'s gradient
    leaf.grad = None
    embedding.lookup(leaf, flat).sum().backward()
    hits = torch.bincount(flat[flat >= 0], minlength=50).float()
    assert torch.equal(leaf.grad, hits[:, None, None].expand(50, 16, 3))
    # rows of one value
    assert torch.equal(embedding.lookup(whole[:, 0, 0].contiguous(), flat.clamp(min=0)), whole[:, 0, 0][flat.clamp(min=0)])


@pytest.mark.parametrize("n", [100, 5000, 30000])
@pytest.mark.parametrize("how", ["recomputed", "offloaded"])
@pytest.mark.parametrize("by_row", [False, True])
def test_saved_tensors_that_move(n, how, by_row):
    """What the gradient reads comes back from the hooks on saved tensors, not from where the forward had it: there something
    else stands by then.  Whole numbers: every sum is exact."""
    from torch.utils.checkpoint import checkpoint
    from vegs_amd import embedding
    table, ids, scale, g = _inputs(n, 301, 12, "holes", scale="row" if by_row else 2.0, whole=True)
    table.requires_grad_(True)
    wanted = [table] + ([scale.requires_grad_(True)] if by_row else [])

    def rows():
        # ids, scales and a table that live no longer than the call, the table as rows with a gap
        wide = torch.zeros((301, 16), device=DEV)
        wide[:, :12] = table
        return embedding.lookup(wide[:, :12], ids + 0, 1.0 * scale if by_row else scale)

    want = torch.autograd.grad(rows(), wanted, g)
    if how == "recomputed":
        out = checkpoint(rows, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            out = rows()
    over = [torch.full((k,), 3, dtype=torch.int64, device=DEV) for k in (n, n // 2, 301 * 8, 301 * 6) for _ in range(8)]
    for x, y in zip(torch.autograd.grad(out, wanted, g), want):
        assert torch.equal(x, y)
    _check(table.detach(), ids, scale.detach() if by_row else scale, g, exact=True)
    del over


def test_only_one_of_the_gradients_is_wanted():
    from vegs_amd import embedding
    table, ids, scale, g = _inputs(300, 30, 45, "holes", seed=11)
    out, d_table, d_scale = _run(table, ids, scale, g)
    t, s = table.clone().requires_grad_(True), scale.clone().requires_grad_(True)
    a, = torch.autograd.grad(embedding.lookup(t, ids, scale), [t], g)
    b, = torch.autograd.grad(embedding.lookup(table, ids, s), [s], g)
    assert torch.equal(a, d_table) and torch.equal(b, d_scale)
    # the table may change between the forward and the backward that does not read it, not before one that does
    y = embedding.lookup(t, ids, scale)
    with torch.no_grad():
        t.mul_(2.0)
    assert torch.equal(torch.autograd.grad(y, [t], g)[0], d_table)
    y = embedding.lookup(t, ids, s)
    with torch.no_grad():
        t.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [s], g)
    with torch.no_grad():
        assert not embedding.lookup(t, ids, s).requires_grad


def test_empty_inputs():
    from vegs_amd import embedding
    for n, rows, width in ((0, 5, 3), (4, 0, 3), (4, 5, 0), (0, 0, 0)):
        t = torch.ones(rows, width, device=DEV, requires_grad=True)
        s = torch.ones(n, device=DEV, requires_grad=True)
        out = embedding.lookup(t, torch.zeros(n, dtype=torch.int64, device=DEV), s)
        assert out.shape == (n, width) and (out == 0).all()
        out.sum().backward()
        assert t.grad.shape == (rows, width) and (t.grad == 0).all() and (s.grad == 0).all()


def test_refusals():
    from vegs_amd import embedding
    t, ids = torch.ones(5, 3, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for table, i, scale, dtype in ((t.double(), ids, None, None), (t, ids.cpu(), None, None), (t, ids.float(), None, None),
                                   (t, ids.short(), None, None), (t, [0, 1], None, None), (t, ids, torch.ones(3, device=DEV), None),
                                   (t, ids, torch.ones(4), None), (t, ids, torch.ones(4, device=DEV, dtype=BF16), None),
                                   (t, ids, None, BF16), (t.bfloat16(), ids, None, F16), (torch.tensor(1.0, device=DEV), ids, None, None)):
        with pytest.raises(ValueError):
            embedding.lookup(table, i, scale, dtype=dtype)
    t.requires_grad_(True)
    y = embedding.lookup(t, ids)
    d, = torch.autograd.grad(y, [t], torch.ones_like(y, requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()                                  # (once differentiable)


def test_more_values_than_31_bits_count():
    """The result and the table both past 2^31 elements: the last rows are where an offset would be cut."""
    from vegs_amd import embedding
    rows, width, n = 1100000, 2048, 1100003
    table = torch.empty((rows, width), dtype=BF16, device=DEV)
    step = torch.arange(width, device=DEV) % 7
    for at in range(0, rows, 100000):
        table[at:at + 100000] = ((torch.arange(at, min(at + 100000, rows), device=DEV)[:, None] % 251) + step).to(BF16)
    ids = (rows - 1 - torch.arange(n, device=DEV)).to(torch.int32)              # the last three: no row
    table.requires_grad_(True)
    out = embedding.lookup(table, ids, 0.5)
    for i in (0, 1, 1048575, 1048576, 1048577, rows - 1, rows, n - 1):
        want = torch.zeros(width, dtype=BF16, device=DEV) if i >= rows else 0.5 * table[rows - 1 - i]
        assert torch.equal(out[i], want.detach()), i
    g = torch.zeros_like(out)
    g[0], g[5], g[rows - 1], g[n - 1] = 4.0, 6.0, 8.0, math.nan
    d, = torch.autograd.grad(out, [table], g)
    assert (d[rows - 1] == 2.0).all() and (d[rows - 6] == 3.0).all() and (d[0] == 4.0).all()
    assert d[1:rows - 6].abs().max().item() == 0.0


def test_more_threads_than_32_bits_count():
    """The scales' gradient alone takes a wave for each of 67 million entries, the forward a quarter of one.  Whole numbers: exact."""
    from vegs_amd import embedding
    n, rows, width = (1 << 26) + 3, 5, 129
    table = ((torch.arange(rows * width, device=DEV) * 7) % 5 - 2.0).reshape(rows, width)
    ids = (torch.arange(n, dtype=torch.int32, device=DEV) % (rows + 1))                # one in six: no row
    scale = (1.0 + torch.arange(n, device=DEV) % 3).float().requires_grad_(True)
    out = embedding.lookup(table, ids, scale)
    d, = torch.autograd.grad(out, [scale], out.detach())                              # s |T[id]|^2
    square = torch.cat((table.square().sum(1), table.new_zeros(1)))
    assert torch.equal(d, scale.detach() * square[ids.long()])
    assert torch.equal(out[-7:].detach(), scale.detach()[-7:, None] * torch.cat((table, table.new_zeros(1, width)))[ids[-7:].long()])


def test_on_another_stream():
    """Forward and backward run where the caller's stream is; their workspaces are used again at once."""
    side = torch.cuda.Stream()
    sets = [_inputs(40000, 500, 45, "hot", seed=k) for k in range(4)]
    want = [_run(*s) for s in sets]
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for k in range(8):
        if k % 2:
            with torch.cuda.stream(side):
                got.append(_run(*sets[k % 4]))
        else:
            got.append(_run(*sets[k % 4]))
    torch.cuda.synchronize()
    for k in range(8):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k % 4]))


@pytest.mark.parametrize("n", [100, 5000, 30000])
def test_captured_and_replayed(n):
    """A training step's lookup and gradients in a graph, twice, replayed with other inputs and eager work between."""
    from vegs_amd import embedding
    graphs = []
    for seed in (1, 2):
        table, ids, scale, g = _inputs(n, 300, 45, "holes", seed=seed)
        table, scale = table.requires_grad_(True), scale.requires_grad_(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(embedding.lookup(table, ids, scale), [table, scale], g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = embedding.lookup(table, ids, scale)
            grads = torch.autograd.grad(out, [table, scale], g)
        graphs.append((graph, (table, ids, scale, g), (out,) + grads))
    for k in range(3):
        for i, (graph, inputs, results) in enumerate(graphs):
            fresh = _inputs(n, 300, 45, ("hot", "uniform", "same")[k], seed=10 + 2 * k + i)
            with torch.no_grad():
                for a, b in zip(inputs, fresh):
                    a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(results, _run(*fresh)):
                assert torch.equal(a, b)


# ---- together: codebook -> render -> loss -> the table's gradient -> one norm with everything else -> clipped Adam
@pytest.mark.parametrize("by_row", [False, True])
def test_codebook_through_the_rasterizer_into_a_clipped_step(by_row):
    from vegs_amd import embedding, harness, optim, rasterizer, scenes
    dev = torch.device(DEV)
    sc, deg = scenes.scene_street(P=20000, length=60.0, sh_degree=3, seed=12)
    cam = scenes.kitti_camera(0.0, 0.3, 344, 94)
    cam_t = harness.cam_tensors(cam, dev)
    rng = np.random.default_rng(0)
    gt = torch.tensor(rng.uniform(0, 1, (3, 94, 344)).astype(np.float32), device=dev)
    P, K = len(sc["means3D"]), 64
    ids = torch.tensor(rng.integers(0, K, P), device=dev)
    book = torch.nn.Parameter(torch.tensor(0.2 * rng.normal(size=(K, 15, 3)), dtype=F32, device=dev))
    gain = torch.nn.Parameter(torch.tensor(rng.uniform(0.5, 1.5, P), dtype=F32, device=dev))
    t = {k: torch.tensor(v, device=dev, requires_grad=True) for k, v in sc.items()}
    dc = torch.nn.Parameter(t["shs"][:, :1].detach().clone().contiguous())

    def loss_of(rest):
        inputs = dict(t, shs=(dc, rest))
        return (harness.render(cam, inputs, deg, torch.zeros(3, device=dev), cam_t=cam_t)["render"] - gt).abs().mean()

    with rasterizer.flags(rasterizer.get_flags() | rasterizer.FLAG_DETERMINISTIC):
        rest = embedding.lookup(book, ids, gain if by_row else None)
        loss_of(rest).backward()
        # the dense model that the codebook stands for
        dense = (book[ids] * gain[:, None, None] if by_row else book[ids]).detach().requires_grad_(True)
        assert torch.equal(rest, dense)
        g, = torch.autograd.grad(loss_of(dense), [dense])
    _, d_book, terms, k, d_gain, m_gain = _formula(book.reshape(K, 45), ids, gain if by_row else None, g.reshape(P, 45))
    assert g.abs().max().item() > 0
    assert ((book.grad.reshape(K, 45).double().cpu() - d_book).abs() <= (k[:, None] + 2) * u * terms).all()
    if by_row:
        assert ((gain.grad.double().cpu() - d_gain).abs() <= 47 * u * m_gain).all()
    # the step: two optimizers, one norm; torch's own clipping and Adam on copies
    params = [book, dc] + ([gain] if by_row else [])
    copies = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    for p, q in zip(params, copies):
        q.grad = p.grad.double().cpu()
    bound = 0.5 * optim.grad_norm(params).item()
    norm = optim.step_many([optim.Adam([book], lr=1e-2, eps=1e-15), optim.Adam(params[1:], lr=1e-3)], max_grad_norm=bound)
    want = torch.nn.utils.clip_grad_norm_(copies, bound)
    torch.optim.Adam([copies[0]], lr=1e-2, eps=1e-15).step()
    torch.optim.Adam(copies[1:], lr=1e-3).step()
    assert abs(norm.item() - want.item()) <= 2 * u * want.item()
    for p, q, lr in zip(params, copies, (1e-2, 1e-3, 1e-3)):
        # a first step moves every value by lr g / (|g| + eps): the factor cancels but for eps, 1e-8 beside clipped gradients:
        # the step's own roundings (at most 16 u) plus eps' share of an 8 u error, and the value's rounding
        assert ((p.detach().double().cpu() - q.detach()).abs() <= 24 * u * lr + u * q.detach().abs() * 1.01).all()


@pytest.mark.parametrize("dtype,width", [(0, 3), (0, 256), (0, 257), (0, 1000), (1, 600)])
def test_no_entries_at_the_c_entry(dtype, width):
    """The table's gradient is zeros, and the scales' gradient, which has no elements, is left alone."""
    import ctypes as C
    from vegs_amd import _capi
    table = torch.ones(7, width, device=DEV, dtype=(F32, BF16)[dtype])
    d_table, d_scale = torch.full_like(table, 3.0), torch.full((4,), 5.0, device=DEV)
    empty = _capi.VrLookup(table.data_ptr(), None, None, 0, 7, width, width, dtype, dtype, 0, 1.0)
    stream = torch.cuda.current_stream().cuda_stream
    for scales in (d_scale.data_ptr(), None):
        d_table.fill_(3.0)
        assert _capi.load().vr_lookup_backward(C.byref(empty), None, width, d_table.data_ptr(), scales, None, 0, stream) == 0
        assert (d_table == 0).all() and (d_scale == 5.0).all()


def test_forward_mode_tangents_are_refused():
    """A dual tensor requires no gradient and has an address like any other: its tangent may not get lost on the way."""
    import torch.autograd.forward_ad as fwd
    from vegs_amd import embedding
    table, ids, scale, _ = _inputs(50, 9, 5, "holes", seed=2)
    want = embedding.lookup(table, ids, scale)
    with fwd.dual_level():
        dual, dual_scale = fwd.make_dual(table, torch.ones_like(table)), fwd.make_dual(scale, torch.ones_like(scale))
        for t, s in ((dual, None), (dual, 2.0), (dual, scale), (table, dual_scale), (dual, dual_scale)):
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(NotImplementedError, match="jvp"):
                    embedding.lookup(t, ids, s)
        assert torch.equal(embedding.lookup(table, ids, scale), want)             # no tangent: nothing to refuse
        with torch.no_grad():
            out = embedding.lookup(table.clone().requires_grad_(True), ids, scale)
            assert torch.equal(out, want) and not out.requires_grad
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: embedding.lookup(t, ids, scale), (table,), (table,))
    assert torch.equal(embedding.lookup(table, ids, scale), want)


@pytest.mark.parametrize("clipped", [False, True])
def test_a_step_between_forward_and_backward_is_noticed(clipped):
    """The scales' gradient reads the table: stepped in between, it is not the table that the result was looked up in."""
    from vegs_amd import embedding, optim
    table, ids, scale, g = _inputs(300, 30, 45, "holes", seed=11)
    t, s = torch.nn.Parameter(table), scale.requires_grad_(True)
    t.grad = torch.ones_like(t)
    y = embedding.lookup(t, ids, s)
    optim.step_many([optim.Adam([t], lr=0.1)], max_grad_norm=1.0 if clipped else None)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [s], g)


@pytest.mark.parametrize("value", [1.9876709, 1.02771, 0.1, 1.0])
def test_equal_entries_of_one_row_add_up(value):
    """2^21 entries of one row, equal values, whose roundings do not cancel.  At this width a chunk has 64 entries (64 additions), 16
    groups join 2048 pieces each, 128 in a row and then 16 such sums, and are added pairwise: 64 + 128 + 16 + 4, and one for the product."""
    from vegs_amd import embedding
    n, width = 1 << 21, 130
    table = torch.zeros((3, width), device=DEV, requires_grad=True)
    g = torch.full((n, width), value, device=DEV)
    out = embedding.lookup(table, torch.ones(n, dtype=torch.int32, device=DEV))
    d, = torch.autograd.grad(out, [table], g)
    want = n * float(torch.tensor(value, dtype=F32))
    assert (d[0] == 0).all() and (d[2] == 0).all()
    assert ((d[1].double() - want).abs() <= (64 + 128 + 16 + 4 + 1) * u * want).all()


@pytest.mark.parametrize("n", [100, 5000])
def test_saved_tensors_in_another_order_of_strides(n):
    """A hook may give back the values laid out otherwise: the gradients are laid out as their inputs' shapes say."""
    from vegs_amd import embedding
    table, ids, scale, g = _inputs(n, 40, 12, "holes", whole=True)
    ids, scale, g = ids.reshape(n // 4, 4), scale.reshape(n // 4, 4), g.reshape(n // 4, 4, 12)
    want = _run(table, ids, scale, g)
    turned = lambda x: x.t().contiguous().t()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: turned(x) if x.dim() == 2 else x):
        got = _run(table, ids, scale, g)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # only the table's: the type of the result is not the table's
    t = table.bfloat16().requires_grad_(True)
    d, = torch.autograd.grad(embedding.lookup(t, ids, scale, dtype=F32), [t], g)
    assert d.dtype == BF16 and d.is_contiguous() and torch.equal(d, want[1].bfloat16())


@pytest.mark.parametrize("wanted", [False, True])
def test_numbers_as_scales(wanted):
    """Float32's range and what float32 has beyond numbers; not what it would have to round to infinity."""
    from vegs_amd import embedding
    t, ids = torch.ones(5, 3, device=DEV, requires_grad=wanted), torch.tensor([1, -1], device=DEV)
    for scale in (0.0, -2, True, 2.0 ** -149, torch.finfo(F32).max, -torch.finfo(F32).max, math.inf, -math.inf, math.nan, np.float32(0.25)):
        out = embedding.lookup(t, ids, scale).detach()
        assert torch.equal(out[0].nan_to_num(7.0), torch.full((3,), float(scale), device=DEV).nan_to_num(7.0)) and (out[1] == 0).all()
    for scale in (1e39, -1e39, 3.5e38, "x"):
        with pytest.raises(ValueError):
            embedding.lookup(t, ids, scale)


@pytest.mark.parametrize("by_row", [False, True])
def test_tangents_that_arrive_in_the_backward_are_refused(by_row):
    """Forward over reverse: what follows the lookup carries a tangent, and so does the gradient that reaches it."""
    import torch.autograd.forward_ad as fwd
    from vegs_amd import embedding
    table, ids, scale, g = _inputs(50, 9, 5, "holes", scale="row" if by_row else 2.0, seed=2)
    table.requires_grad_(True)
    with fwd.dual_level():
        out = embedding.lookup(table, ids, scale)
        weighted = (out * fwd.make_dual(g, torch.ones_like(g))).sum()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(weighted, [table])
        d, = torch.autograd.grad((embedding.lookup(table, ids, scale) * g).sum(), [table])
    assert torch.equal(d, torch.autograd.grad((embedding.lookup(table, ids, scale) * g).sum(), [table])[0])
