"""GPU (-m gpu): the global gradient norm, clipping in place, and the clipped Adam steps, against the formula in 64 bits.

Roundings counted in u = half a step of a type (fp32 2^-24, bf16 2^-8, fp16 2^-11).  The norm: sums in 64 bits, one rounding:
u.  The factor max_norm / (norm + 1e-6): norm, sum, quotient: 3 u.  A clipped fp32 value: 4 u, doubled once more below for
second-order terms; in 16 bits plus that type's u, and plus half its smallest subnormal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
# one element; ends of vectors, waves, workgroups and units on either side
SIZES = [1, 3, 4, 63, 255, 256, 1023, 4095, 4096, 4097, 8191, 8192, 8193, 16385]


def _param(g):
    p = torch.empty_like(g)
    p.grad = g
    return p


def _norm64(grads, norm_type=2.0):
    flat = torch.cat([g.detach().double().cpu().reshape(-1) for g in grads])
    return float(flat.abs().max()) if norm_type == math.inf else math.sqrt(math.fsum((flat * flat).tolist()))


def _make(shapes, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=g)).to(dtype).to(DEV) for s in shapes]


def _check_clipped(before, after, norm64, max_norm):
    c = min(1.0, max_norm / (norm64 + 1e-6))
    for b, a in zip(before, after):
        want = b.double().cpu() * c
        u = 8 * 2.0 ** -24 + (0 if b.dtype == torch.float32 else U[b.dtype])
        assert a.dtype == b.dtype and a.shape == b.shape
        assert ((a.double().cpu() - want).abs() <= u * want.abs() + TINY[b.dtype]).all()


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_and_clipping_of_many_sizes(dtype, norm_type):
    from vegs_amd import optim
    grads = _make([(n,) for n in SIZES], dtype)
    before = [g.clone() for g in grads]
    params = [_param(g) for g in grads]
    want = _norm64(before, norm_type)
    for max_norm in (0.25 * want, 4.0 * want):
        for p, b in zip(params, before):
            p.grad.copy_(b)
        only = optim.grad_norm(params, norm_type)
        norm = optim.clip_grad_norm_(params, max_norm, norm_type)
        assert norm.dtype == torch.float32 and norm.shape == () and norm.device == grads[0].device
        assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want and norm.item() == only.item()
        _check_clipped(before, grads, want, max_norm)
        if max_norm > want:
            assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_one_gradient_of_each_size(n, dtype):
    from vegs_amd import optim
    g, = _make([(n,)], dtype, seed=n)
    before = g.clone()
    norm = optim.clip_grad_norm_(_param(g), 0.1)
    want = _norm64([before])
    assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
    _check_clipped([before], [g], want, 0.1)


@pytest.mark.parametrize("offset", [1, 2, 3, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_that_start_off_a_vector_boundary(offset, dtype):
    from vegs_amd import optim
    buf, = _make([(60000,)], dtype, seed=9)
    whole = buf.clone()
    params = [_param(buf[offset:offset + 40001]), _param(buf[offset + 40001:offset + 40005])]
    want = _norm64([buf[offset:offset + 40005]])
    norm = optim.clip_grad_norm_(params, 1.0)
    assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
    _check_clipped([whole[offset:offset + 40005]], [buf[offset:offset + 40005]], want, 1.0)
    assert torch.equal(buf[:offset], whole[:offset]) and torch.equal(buf[offset + 40005:], whole[offset + 40005:])


@pytest.mark.parametrize("count", [127, 128, 129, 300])
def test_more_tensors_than_a_launch_takes_and_empty_ones(count):
    from vegs_amd import optim
    shapes = [((i * 37) % 90, 3) if i % 11 else (0, 3) for i in range(count)]
    grads = _make(shapes, seed=count)
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_([_param(g) for g in grads] + [torch.nn.Parameter(torch.zeros(3, device=DEV))], 2.0)
    want = _norm64(before)
    assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
    _check_clipped(before, grads, want, 2.0)


def test_mixed_types_and_layouts():
    from vegs_amd import optim
    a, b, c, d = _make([(64, 31), (45, 77), (1000,), (33, 40)], seed=4)
    grads = [a.t(), b.bfloat16(), c.half(), d[:, ::2]]            # transposed, two 16-bit types, every other column
    before = [g.clone() for g in grads]
    left = d[:, 1::2].clone()
    params = []
    for g in grads:
        p = torch.empty(g.shape, dtype=g.dtype, device=DEV)
        p.grad = g
        params.append(p)
    assert params[0].grad.stride() == (1, 31) and params[3].grad.stride() == (40, 2)
    norm = optim.clip_grad_norm_(params, 3.0)
    want = _norm64(before)
    assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
    _check_clipped(before, [p.grad for p in params], want, 3.0)
    assert torch.equal(d[:, 1::2], left)                          # what lies between the elements is not touched


def test_refusals_on_the_gpu():
    from vegs_amd import optim
    p = torch.empty(4, 5, device=DEV)
    p.grad = torch.ones(1, device=DEV).expand(4, 5)
    assert abs(optim.grad_norm(p).item() - math.sqrt(20.0)) <= 2.0 ** -24 * 1.01 * math.sqrt(20.0)
    with pytest.raises(ValueError, match="expanded"):
        optim.clip_grad_norm_(p, 1.0)
    q = torch.empty(3, device=DEV, dtype=torch.float64)
    q.grad = torch.ones_like(q)
    with pytest.raises(ValueError, match="float32"):
        optim.grad_norm([q])
    cpu = torch.empty(3)
    cpu.grad = torch.ones(3)
    r = _param(torch.ones(3, device=DEV))
    with pytest.raises(ValueError, match="one device"):
        optim.clip_grad_norm_([r, cpu], 1.0)
    assert torch.equal(r.grad, torch.ones(3, device=DEV))
    opt = optim.Adam([torch.nn.Parameter(torch.zeros(3, device=DEV))])
    opt.param_groups[0]["params"][0].grad = torch.ones(3, device=DEV)
    for bad in (torch.tensor(1.0), torch.ones(2, device=DEV), 1.0):
        with pytest.raises(ValueError, match="grad_norm"):
            optim.step_many([opt], max_grad_norm=1.0, grad_norm=bad)
    assert not opt.state


@pytest.mark.parametrize("value", [1e30, 3e38, 1e-30, 1e-42, 0.0])
def test_magnitudes_whose_squares_leave_fp32(value):
    from vegs_amd import optim
    x = torch.full((5001,), value, device=DEV)
    want = float(x[0].double()) * math.sqrt(5001.0)
    p = _param(x)
    norm = optim.clip_grad_norm_(p, 1.0).item()
    if want > torch.finfo(torch.float32).max:
        assert norm == math.inf and (p.grad == 0).all()
    else:
        assert abs(norm - want) <= 2.0 ** -24 * 1.01 * want + TINY[torch.float32]
        _check_clipped([torch.full((5001,), value, device=DEV)], [p.grad], want, 1.0)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("place", [0, 700, 20000])
def test_nan_and_infinity(place, norm_type):
    from vegs_amd import optim
    for bad in (math.nan, math.inf, -math.inf):
        a, b = _make([(20001,), (30,)], seed=1)
        a[place] = bad
        before = [a.clone(), b.clone()]
        with pytest.raises(RuntimeError, match="not finite"):
            optim.clip_grad_norm_([_param(a), _param(b)], 1.0, norm_type, error_if_nonfinite=True)
        assert torch.equal(a.nan_to_num(7.0), before[0].nan_to_num(7.0)) and torch.equal(b, before[1])
        norm = optim.clip_grad_norm_([_param(a), _param(b)], 1.0, norm_type)
        want = [x.cpu() for x in before]
        torch_norm = torch.nn.utils.clip_grad_norm_([_param(x) for x in want], 1.0, norm_type)
        assert str(norm.item()) == str(torch_norm.item())         # nan or inf
        for mine, its in zip((a, b), want):
            assert torch.equal(mine.cpu().isnan(), its.isnan()) and torch.equal(mine.cpu().nan_to_num(7.0), its.nan_to_num(7.0))


def test_a_bound_of_zero_and_of_infinity():
    from vegs_amd import optim
    g, = _make([(3000,)])
    keep = g.clone()
    optim.clip_grad_norm_(_param(g), math.inf)
    assert torch.equal(g, keep)
    optim.clip_grad_norm_(_param(g), 0.0)
    assert (g == 0).all()


def test_one_gradient_of_more_values_than_31_bits_count():
    """3, 4 and 12 at the borders where an offset would be cut: the norm is 13, half of it the factor one half of powers of two."""
    from vegs_amd import optim
    n = 2 ** 31 + 2 ** 17 + 5
    p = torch.empty(n, dtype=torch.bfloat16, device=DEV)
    p.grad = torch.zeros_like(p)
    places = (0, 2 ** 31 - 1, 2 ** 31, n - 1)
    for at, x in zip(places, (3.0, 4.0, 0.0, 12.0)):
        p.grad[at] = x
    assert optim.grad_norm(p).item() == 13.0 and optim.grad_norm(p, math.inf).item() == 12.0
    assert optim.clip_grad_norm_(p, 6.5).item() == 13.0
    assert [p.grad[at].item() for at in places] == [1.5, 2.0, 0.0, 6.0]           # (6.5 / (13 + 1e-6) rounds to a half of them in 8 bits)
    assert p.grad.count_nonzero().item() == 3


def test_a_gradient_met_twice_counts_once():
    from vegs_amd import optim
    g, = _make([(5000,)])
    keep = g.clone()
    p = _param(g)
    want = _norm64([keep])
    norm = optim.clip_grad_norm_([p, p, p], 1.0)
    assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
    _check_clipped([keep], [g], want, 1.0)


def test_the_same_bits_every_time_and_in_every_layout_of_streams():
    from vegs_amd import optim
    grads = _make([(300001, 3), (17,), (40000, 45)], seed=2)
    params = [_param(g) for g in grads]
    first = optim.grad_norm(params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [optim.grad_norm(params) for _ in range(3)]
    again = optim.grad_norm(params)
    torch.cuda.synchronize()
    assert all(x.item() == first.item() for x in other + [again])


def test_captured_and_replayed():
    """Two graphs with workspaces of their own, replayed in turn with eager work between: every replay reads the gradients
    that are there then."""
    from vegs_amd import optim
    sets = [_make([(50000, 3), (7,)], seed=5), _make([(21, 3)], seed=6)]      # the launches of large sets and of small ones
    graphs, norms = [], []
    side = torch.cuda.Stream()
    for grads in sets:
        params = [_param(g) for g in grads]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            optim.clip_grad_norm_(params, 1.0)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(optim.clip_grad_norm_(params, 1.0))
        graphs.append(graph)
    for k in range(4):
        for i, grads in enumerate(sets):
            fresh = _make([tuple(g.shape) for g in grads], seed=50 + 2 * k + i, scale=2.0 ** k)
            for g, f in zip(grads, fresh):
                g.copy_(f)
            graphs[i].replay()
            eager = [_param(f.clone()) for f in fresh]
            want = optim.clip_grad_norm_(eager, 1.0)
            assert norms[i].item() == want.item()
            assert all(torch.equal(g, e.grad) for g, e in zip(grads, eager))


# ---- the clipped Adam step
def _optimizers(seed=0, rows=(3000, 70), poses=3):
    from vegs_amd import optim
    g = torch.Generator().manual_seed(seed)
    opts = []
    for n in rows:
        opts.append(optim.Adam([{"params": [torch.nn.Parameter(torch.randn((n,) + s, generator=g).to(DEV))], "lr": lr}
                                for s, lr in (((3,), 1e-3), ((15, 3), 1e-4), ((1,), 5e-2), ((4,), 1e-3))], lr=0.0, eps=1e-15))
    for _ in range(poses):
        opts.append(optim.Adam([torch.nn.Parameter(torch.randn((k,), generator=g).to(DEV)) for k in (4, 3, 3)], lr=5e-3))
    return opts


def _params(opts):
    return [p for o in opts for g in o.param_groups for p in g["params"]]


def _give_grads(opts, seed, scale=1.0):
    for p, g in zip(_params(opts), _make([tuple(p.shape) for p in _params(opts)], seed=seed, scale=scale)):
        p.grad = g


@pytest.mark.parametrize("factor", [0.1, 50.0])
def test_clipped_step_is_clipping_and_stepping(factor):
    """Bit for bit: the factor meets the gradient in the same fp32 product.  .grad stays as it was."""
    from vegs_amd import optim
    a, b = _optimizers(), _optimizers()
    for step in range(3):
        _give_grads(a, step); _give_grads(b, step)
        bound = factor * _norm64([p.grad for p in _params(a)])
        keep = [p.grad.clone() for p in _params(a)]
        got = optim.step_many(a, max_grad_norm=bound)
        want = optim.clip_grad_norm_(b, bound)
        assert optim.step_many(b) is None
        assert got.item() == want.item()
        for p, q, g in zip(_params(a), _params(b), keep):
            assert torch.equal(p, q) and torch.equal(p.grad, g)
    for oa, ob in zip(a, b):
        for p, q in zip(_params([oa]), _params([ob])):
            sa, sb = oa.state[p], ob.state[q]
            assert torch.equal(sa["exp_avg"], sb["exp_avg"]) and torch.equal(sa["exp_avg_sq"], sb["exp_avg_sq"])
            assert float(sa["step"]) == float(sb["step"]) == 3


def test_clipped_step_against_64_bits():
    """One step from random moments.  With u = 2^-24, clipped g = c g is 8 u off (see above); m' = m + (g - m) (1 - b1): at most
    8 u g + 4 u (|m| + |g|); v' = b2 v + (1 - b2) g g: 3 u b2 v + (2 * 8 + 4) u (1 - b2) g^2 <= 20 u v'; the step
    lr_t m' / (sqrt(v') / c2 + eps): m's error, plus (20 / 2 + 6) u of itself; p': one rounding more."""
    from vegs_amd import optim
    opts = _optimizers(seed=3)
    _give_grads(opts, 8)
    for i, o in enumerate(opts):
        for p in _params([o]):
            m, v = _make([tuple(p.shape)] * 2, seed=int(p.numel()) + i)
            o.state[p] = {"step": torch.tensor(11.0), "exp_avg": m, "exp_avg_sq": v * v + 0.01}
    c = 0.3
    norm = _norm64([p.grad for p in _params(opts)])
    old = [(p.detach().double(), o.state[p]["exp_avg"].double(), o.state[p]["exp_avg_sq"].double()) for o in opts for p in _params([o])]
    got = optim.step_many(opts, max_grad_norm=c * norm)
    assert abs(got.item() - norm) <= 2.0 ** -24 * 1.01 * norm
    c, u, k = c * norm / (norm + 1e-6), 2.0 ** -24, 0
    for o in opts:
        for grp in o.param_groups:
            for p in grp["params"]:
                p0, m0, v0 = old[k]
                k += 1
                g = p.grad.double() * c
                m = m0 + (g - m0) * (1 - 0.9)
                v = 0.999 * v0 + (1 - 0.999) * g * g
                denom = v.sqrt() / math.sqrt(1 - 0.999 ** 12) + grp["eps"]
                lr = grp["lr"] / (1 - 0.9 ** 12)
                m_off = 8 * u * g.abs() + 4 * u * (m0.abs() + g.abs())
                st = o.state[p]
                assert float(st["step"]) == 12
                assert ((st["exp_avg"].double() - m).abs() <= m_off).all()
                assert ((st["exp_avg_sq"].double() - v).abs() <= 20 * u * v).all()
                p1 = p0 - lr * m / denom
                assert ((p.detach().double() - p1).abs() <= lr * m_off / denom + 16 * u * lr * m.abs() / denom + u * p1.abs() * 1.01).all()


def test_an_infinite_and_a_nan_norm_in_the_step():
    """As after torch's clipping: an infinite norm zeroes the finite gradients, a NaN reaches every parameter."""
    from vegs_amd import optim
    for bad in (math.inf, math.nan):
        a, b = _optimizers(rows=(40,), poses=1), _optimizers(rows=(40,), poses=1)
        for o in (a, b):
            _give_grads(o, 1)
            _params(o)[0].grad[3, 1] = bad
        optim.step_many(a, max_grad_norm=1.0)
        optim.clip_grad_norm_(b, 1.0)
        optim.step_many(b)
        for p, q in zip(_params(a), _params(b)):
            assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.nan_to_num(7.0), q.nan_to_num(7.0))


@pytest.mark.parametrize("P,deg,views,split", [(1, 0, 1, False), (63, 1, 2, True), (257, 2, 3, True), (5000, 3, 2, True), (700, 3, 1, False)])
def test_factored_gradients_in_the_norm_and_the_step(P, deg, views, split):
    """The norm with a gradient given as factors is the norm with the dense gradient they stand for, and the clipped factored
    step is the clipped dense one, bit for bit: the dense row comes from the same function."""
    from vegs_amd import optim
    g = torch.Generator().manual_seed(P)
    M = 16
    means, campos = torch.randn((P, 3), generator=g).to(DEV) * 3, torch.randn((views, 3), generator=g).to(DEV)
    factors = torch.randn((views, P, 3), generator=g) * (torch.rand((views, P, 1), generator=g) > 0.3)
    factors = factors.to(DEV)

    def models():
        gg = torch.Generator().manual_seed(7)
        shapes = [(P, 1, 3), (P, M - 1, 3)] if split else [(P, M, 3)]
        ps = [torch.nn.Parameter(torch.randn(s, generator=gg).to(DEV)) for s in shapes]
        other = torch.nn.Parameter(torch.randn((P, 3), generator=gg).to(DEV))
        opt = optim.Adam([{"params": [p], "lr": 1e-2} for p in ps + [other]], lr=0.0, eps=1e-15)
        other.grad = torch.randn((P, 3), generator=gg).to(DEV)
        return ps, other, opt

    (ps, other, opt), (qs, other_q, opt_q) = models(), models()
    scale = 0.37
    dense = optim.sh_grad_from_factors(means, campos, factors, deg, M, scale, split=split)
    for q, d in zip(qs, dense if split else [dense]):
        q.grad = d
    sh = [(means, campos, factors, deg, scale)]
    for norm_type in (2.0, math.inf):
        mine, its = optim.grad_norm([opt], norm_type, sh_factors=sh), optim.grad_norm([opt_q], norm_type)
        want = _norm64([d for d in (dense if split else [dense])] + [other.grad], norm_type)
        assert abs(mine.item() - want) <= 2.0 ** -24 * 1.01 * want and abs(its.item() - want) <= 2.0 ** -24 * 1.01 * want
    norm = optim.grad_norm([opt], sh_factors=sh)
    bound = 0.21 * norm.item()
    assert optim.adam_step_sh_factored(opt, ps[0], ps[1] if split else None, means, campos, factors, deg, scale,
                                       max_grad_norm=bound, grad_norm=norm) is norm
    optim.step_many([opt], max_grad_norm=bound, grad_norm=norm)
    optim.step_many([opt_q], max_grad_norm=bound, grad_norm=norm)
    for p, q in zip(ps + [other], qs + [other_q]):
        assert torch.equal(p, q)
        assert torch.equal(opt.state[p]["exp_avg"], opt_q.state[q]["exp_avg"])
    # its own norm where none is given
    own = optim.adam_step_sh_factored(opt, ps[0], ps[1] if split else None, means, campos, factors, deg, scale, max_grad_norm=1e9)
    want = _norm64(list(dense) if split else [dense])
    assert abs(own.item() - want) <= 2.0 ** -24 * 1.01 * want


def test_factored_gradients_of_as_many_points_as_31_bits_count():
    """Degree 0: the row is scale x 0.28209479 x the factor, wherever its point stands.  One fp32 rounding of the constant, of each
    of the two products and of the norm itself: 4 x 2^-24."""
    from vegs_amd import optim
    P = 2 ** 31 - 1
    means, factors = torch.zeros((P, 3), device=DEV), torch.zeros((1, P, 3), device=DEV)
    for at, x in ((0, 3.0), (2 ** 31 - 2 ** 18 - 2, 4.0), (P - 1, 12.0)):
        factors[0, at, at % 3] = x
    sh = [(means, torch.ones((1, 3), device=DEV), factors, 0, 0.5)]
    for norm_type, want in ((2.0, 13.0), (math.inf, 12.0)):
        want *= 0.5 * 0.28209479177387814
        assert abs(optim.grad_norm([], norm_type, sh_factors=sh).item() - want) <= 4.01 * 2.0 ** -24 * want


@pytest.mark.parametrize("n_boxes,factored", [(0, False), (0, True), (2, False), (2, True)])
def test_trainer_clips_all_its_optimizers_by_one_norm(n_boxes, factored):
    """One iteration: the trainer's norm is that of every gradient its optimizers hold, and what it steps with is theirs
    times the factor -- seen in the first moments, (1 - beta1) c g after the first step."""
    from vegs_amd import harness, iteration, rasterizer, scenes
    dev = torch.device(DEV)
    sc, deg = scenes.scene_street(P=20000, length=60.0, sh_degree=3, seed=12)
    cam = scenes.kitti_camera(0.0, 0.3, 344, 94)
    rng = np.random.default_rng(0)
    gt = torch.tensor(rng.uniform(0, 1, (3, 94, 344)).astype(np.float32), device=dev)
    normal = torch.tensor(rng.normal(size=(3, 94, 344)).astype(np.float32), device=dev)
    runs = []
    with rasterizer.flags(rasterizer.get_flags() | rasterizer.FLAG_DETERMINISTIC):
        for bound in (None, 1e-3):
            tr = iteration.Trainer(sc, dev, n_boxes=n_boxes, fused=True, box_points=500, factored_sh=factored,
                                   optimise_boxes=n_boxes > 0, max_grad_norm=bound)
            tr.step(cam, harness.cam_tensors(cam, dev), deg, torch.zeros(3, device=dev), gt, normal)
            runs.append((tr, {k: v for k, v in tr.state_tensors().items() if k.endswith("exp_avg")}))
    (plain, m0), (clipped, m1) = runs
    assert plain.last["grad_norm"] is None
    norm = clipped.last["grad_norm"].item()
    # the pose corrections have stepped a second time, on their regulariser, and hold no plain (1 - beta1) g
    names = [k for k in m0 if not k.startswith("box")]
    assert norm > 1e-3 and len(names) >= 6
    size = math.sqrt(sum(float((m0[k].double() ** 2).sum()) for k in names)) / 0.1
    assert size <= norm * (1 + 1e-6)
    if n_boxes == 0:                    # m = (g - 0) 0.1f: 2 u each and 0.1's own rounding, and the norm's: 4 u
        assert abs(size - norm) <= 4 * 2.0 ** -24 * norm
    c = 1e-3 / (norm + 1e-6)
    for k in names:                     # both sides (1 - beta1) times a gradient: 2 u and 8 u + 2 u
        want = m0[k].double() * c
        assert ((m1[k].double() - want).abs() <= 12 * 2.0 ** -24 * want.abs() + 2.0 ** -148).all(), k


def test_gradients_that_begin_at_one_address():
    """b[:n] and b[::2] of one buffer: other elements, so both enter the norm; each value in memory is scaled once."""
    from vegs_amd import optim
    n = 4000
    b, = _make([(2 * n,)], seed=3)
    before = b.clone()
    dense, apart = _param(b[:n]), torch.empty(n, device=DEV)
    apart.grad = b[::2]
    want = _norm64([before[:n], before[::2]])
    assert abs(optim.grad_norm([dense, apart]).item() - want) <= 2.0 ** -24 * 1.01 * want
    opts = [optim.Adam([torch.nn.Parameter(torch.zeros(n, device=DEV))]) for _ in range(2)]
    for o, g in zip(opts, (b[:n], b[::2])):
        o.param_groups[0]["params"][0].grad = g
    assert abs(optim.step_many(opts, max_grad_norm=1.0).item() - want) <= 2.0 ** -24 * 1.01 * want
    for params in ([dense, apart], [apart, dense]):
        b.copy_(before)
        norm = optim.clip_grad_norm_(params, 0.25 * want)
        assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
        held = torch.zeros(2 * n, dtype=torch.bool, device=DEV)
        held[:n] = held[::2] = True
        _check_clipped([before[held]], [b[held]], want, 0.25 * want)
        assert torch.equal(b[~held], before[~held])


def test_columns_of_one_buffer_are_clipped_as_they_are():
    from vegs_amd import optim
    b, = _make([(700, 9)], seed=4)
    before = b.clone()
    left, right = torch.empty(700, 3, device=DEV), torch.empty(700, 6, device=DEV)
    left.grad, right.grad = b[:, :3], b[:, 3:]
    want = _norm64([before])
    norm = optim.clip_grad_norm_([left, right], 0.5 * want)
    assert abs(norm.item() - want) <= 2.0 ** -24 * 1.01 * want
    _check_clipped([before], [b], want, 0.5 * want)


@pytest.mark.parametrize("error_if_nonfinite", [False, True])
def test_gradients_that_share_a_part_of_their_memory_are_refused(error_if_nonfinite):
    from vegs_amd import optim
    b, = _make([(9000,)], seed=5)
    before = b.clone()
    with pytest.raises(ValueError, match="share memory"):
        optim.clip_grad_norm_([_param(b[:6000]), _param(b[5999:])], 1.0, error_if_nonfinite=error_if_nonfinite)
    assert torch.equal(b, before)
    want = _norm64([before[:6000], before[5999:]])
    assert abs(optim.grad_norm([_param(b[:6000]), _param(b[5999:])]).item() - want) <= 2.0 ** -24 * 1.01 * want


def test_what_the_kernels_write_has_a_new_version():
    """As after torch's own clipping and Adam: a graph that needs the old values raises."""
    from vegs_amd import optim
    g, = _make([(40, 3)], seed=1)
    for grad in (g, _make([(40, 6)], seed=1)[0][:, ::2]):
        p = torch.empty((40, 3), device=DEV)
        p.grad = grad
        w = torch.ones((40, 3), device=DEV, requires_grad=True)
        y = (p.grad * w).sum()                        # its backward reads p.grad
        optim.grad_norm(p)
        assert torch.autograd.grad(y, [w], retain_graph=True)[0].equal(p.grad)
        optim.clip_grad_norm_(p, 0.5)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, [w])
    opt = optim.Adam([{"params": [torch.nn.Parameter(torch.ones(s, device=DEV))], "name": n}
                      for n, s in (("a", (50, 1, 3)), ("b", (50, 15, 3)), ("c", (50, 3)))], lr=1e-2)
    a, b, c = _params([opt])

    def raises(p, step):
        before = p.detach().clone()
        y = (p * p).sum()
        step()
        assert not torch.equal(p, before)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()

    for kw in ({}, {"max_grad_norm": 1.0}):
        c.grad = torch.ones_like(c)
        raises(c, lambda: optim.step_many([opt], **kw))
        raises(c, opt.step)
        c.grad = None
        means, factors = torch.zeros(50, 3, device=DEV), torch.ones(1, 50, 3, device=DEV)
        campos = torch.ones(1, 3, device=DEV)
        for p in (a, b):
            raises(p, lambda: optim.adam_step_sh_factored(opt, a, b, means, campos, factors, 3, **kw))
            versions = [opt.state[p][k]._version for k in ("exp_avg", "exp_avg_sq")]
            optim.adam_step_sh_factored(opt, a, b, means, campos, factors, 3, **kw)
            assert all(opt.state[p][k]._version > v for k, v in zip(("exp_avg", "exp_avg_sq"), versions))


def test_gradients_and_parameters_of_inference_mode():
    """They have no version to raise.  (The factor is not a half: 0.5 norm / (norm + 1e-6), 6.5e-8 less of it.)"""
    from vegs_amd import optim
    with torch.inference_mode():
        p = torch.ones(30, device=DEV)
        p.grad = torch.full((30,), 2.0, device=DEV)
        plain = _param(torch.full((30,), 2.0, device=DEV))
        optim.clip_grad_norm_([p, plain], 0.5 * math.sqrt(240.0))
    before = torch.full((30,), 2.0, device=DEV)
    _check_clipped([before, before], [p.grad, plain.grad], math.sqrt(240.0), 0.5 * math.sqrt(240.0))


@pytest.mark.parametrize("bound", [None, 1.0])
def test_a_parameter_met_twice_is_not_stepped_at_all(bound):
    """One launch would read, step and write it from two workgroups."""
    from vegs_amd import optim
    p, q = (torch.nn.Parameter(torch.ones(5000, device=DEV)) for _ in range(2))
    a, b, c = optim.Adam([p], lr=0.1), optim.Adam([q, p], lr=0.1), optim.Adam([q], lr=0.1)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    for opts in ([a, a], [a, b], [c, b, a]):
        with pytest.raises(ValueError, match="twice"):
            optim.step_many(opts, max_grad_norm=bound)
    assert (p == 1).all() and (q == 1).all() and not a.state and not b.state and not c.state
    optim.step_many([a, c], max_grad_norm=bound)
    assert (p < 1).all() and (q < 1).all()
    q.grad = None                                   # without a gradient it is not stepped, and may be in both
    optim.step_many([b, c], max_grad_norm=bound)
    assert float(b.state[p]["step"]) == 1
