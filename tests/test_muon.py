"""Orthogonalised updates (muon_ops, optim.Muon, csrc/muon.hip) against the definition in 64 bits: shapes on both sides of every
tile, stacks and lists, storage types, strides, zero / non-finite / huge / tiny matrices, other coefficients, repeatability,
streams, captured graphs, the optimiser's step and a model's training step, and the refusals."""
import math

import pytest
import torch

C = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def iterate(x, steps=5, coef=C, eps=EPS):
    """(result, bound of the kernel's error in the 2-norm): float64."""
    x = x.double()
    wide = x.shape[-2] <= x.shape[-1]
    x = x if wide else x.mT
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    rows = [coef] * steps if not isinstance(coef[0], (tuple, list)) else coef
    # What a step adds: X is held to 2^-22 of each entry, and so are G and P, whose errors reach X through a product; the fp32
    # sums of a product over k terms take a rounding for each 16 of them and each of the three parts.  Together at most
    # (3 + sqrt(k) / 4) 2^-22 |X|_F.  What a later step makes of it: at most its polynomial's largest slope on [0, 1.3].
    s = torch.linspace(0, 1.3, 200, dtype=torch.float64)
    slopes = [float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()) for a, b, c in rows]
    bound = 2.0 ** -22 * (1 + x.norm())
    for (a, b, c), slope in zip(rows, slopes):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
        bound = bound * slope + (3 + math.sqrt(x.shape[-2]) / 4) * 2.0 ** -22 * x.norm()
    return (x if wide else x.mT), float(bound)


def matrix(*shape, dtype=torch.float32, device="cuda", seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(shape[-1], generator=g)) + 0.3
    return (1e-2 * x).to(dtype).to(device)


def close(got, x, **kw):
    ref, bound = iterate(x, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    err = float((got.double() - ref).norm())
    tol = bound + torch.finfo(x.dtype).eps / 2 * float(ref.norm())
    assert err <= tol, (err, tol, float(ref.norm()))


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 200), (16, 16), (33, 31), (63, 64), (64, 64), (64, 65), (65, 300), (128, 128),
          (130, 129), (191, 700), (255, 256), (256, 1000), (257, 515), (4, 64), (512, 32), (2, 5000), (1029, 64), (1728, 64),
          (1000, 300), (640, 640), (20000, 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(device, shape):
    from dpcr_agb_amd.muon_ops import orthogonalize
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = matrix(*shape, dtype=dtype, device=device, seed=shape[0])
        close(orthogonalize(x), x)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 3, 4), (27, 64, 64), (2, 3, 70, 130), (343, 3, 64), (3, 300, 260)])
def test_stacks(device, shape):
    """Every matrix of a stack by itself."""
    from dpcr_agb_amd.muon_ops import orthogonalize
    x = matrix(*shape, device=device)
    got = orthogonalize(x)
    flat, out = x.reshape(-1, *shape[-2:]), got.reshape(-1, *shape[-2:])
    for i in range(0, flat.shape[0], max(1, flat.shape[0] // 9)):
        close(out[i], flat[i])


@pytest.mark.gpu
def test_large_kernel_matrix(device):
    from dpcr_agb_amd.muon_ops import orthogonalize
    x = matrix(13824, 512, device=device)
    close(orthogonalize(x), x)


@pytest.mark.gpu
def test_more_than_31_bits_of_elements(device):
    """A polynomial of X X^T times X is X times a small matrix, which is taken in 64 bits here: rows at both ends, and where the
    offsets pass 2^31."""
    from dpcr_agb_amd.muon_ops import orthogonalize
    rows, cols = 16_000_000, 136
    x = torch.randn(rows, cols, device=device) * torch.exp(0.5 * torch.randn(cols, device=device))
    got = orthogonalize(x)
    g = torch.zeros(cols, cols, dtype=torch.float64, device=device)
    for part in x.split(1 << 20):
        g += part.double().T.contiguous() @ part.double()
    norm = float(g.trace().sqrt()) + EPS
    g = g / norm ** 2
    q, s2 = torch.eye(cols, dtype=torch.float64, device=device), g
    for a, b, c in [C] * 5:
        step = a * torch.eye(cols, dtype=torch.float64, device=device) + b * s2 + c * (s2 @ s2)
        q, s2 = q @ step, s2 @ step @ step
    bound = iterate(torch.linalg.cholesky(g).T)[1]       # (the same singular values)
    at = (1 << 31) // cols
    for first in (0, at - 500, rows - 1000):
        want = (x[first:first + 1000].double() / norm) @ q
        # the bound is of all rows together; a thousand of them take their part of it, and five times that
        err = float((got[first:first + 1000].double() - want).norm())
        assert err <= 5 * (1000 / rows) ** 0.5 * bound + 2.0 ** -24 * float(want.norm()), (first, err)


@pytest.mark.gpu
def test_lists_equal_single_calls(device):
    """A list of unlike matrices (more than one table's worth, empty ones among them) gives what single calls give, bit for bit."""
    from dpcr_agb_amd.muon_ops import orthogonalize
    shapes = [(64, 4), (4, 64), (1728, 64), (0, 5), (3, 0, 4), (300, 290), (2, 33, 65), (512, 512), (70, 7)] * 9
    xs = [matrix(*s, device=device, seed=i) if math.prod(s) else torch.zeros(s, device=device) for i, s in enumerate(shapes)]
    many = orthogonalize(xs)
    assert orthogonalize([]) == []
    for x, y in zip(xs, many):
        assert torch.equal(y, orthogonalize(x))


@pytest.mark.gpu
@pytest.mark.parametrize("small", [(2, 512, 64), (5, 300, 40), (2, 128, 128)])
@pytest.mark.parametrize("large", [(64, 700), (300, 700)])
def test_stacks_beside_tiles(device, small, large):
    """Matrices taken whole in the last launch of others, up to the most shared memory that one takes."""
    from dpcr_agb_amd.muon_ops import orthogonalize
    xs = [matrix(*large, device=device), matrix(*small, device=device, seed=1)]
    for got, x in zip(orthogonalize(xs), xs):
        assert torch.equal(got, orthogonalize(x))
        for g, m in zip(got.reshape(-1, *got.shape[-2:]), x.reshape(-1, *x.shape[-2:])):
            close(g, m)


@pytest.mark.gpu
def test_strided_rows(device):
    from dpcr_agb_amd.muon_ops import orthogonalize
    wide = matrix(90, 200, device=device)
    for x in (wide[:, 3:70], wide[::2, :100], wide.t(), wide[:1].expand(4, 200), wide[:, :1], wide[5:6, 1:],
              matrix(4, 30, 40, device=device)[1::2, 2:, :33], matrix(3, 30, 40, device=device).transpose(0, 1)):
        assert torch.equal(orthogonalize(x), orthogonalize(x.contiguous()))


@pytest.mark.gpu
def test_zero_huge_tiny_and_non_finite(device):
    from dpcr_agb_amd.muon_ops import orthogonalize
    x = matrix(70, 90, device=device)
    assert torch.equal(orthogonalize(torch.zeros_like(x)), torch.zeros_like(x))
    for scale in (1e30, 1e-30):          # (squares leave the fp32 range both ways)
        y = x * scale
        close(orthogonalize(y, eps=0.0), y, eps=0.0)
    one = orthogonalize(torch.stack([x, torch.zeros_like(x)]))
    assert torch.equal(one[0], orthogonalize(x)) and torch.equal(one[1], torch.zeros_like(x))
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[3, 5] = bad
        both = orthogonalize(torch.stack([y, x]))
        assert torch.isnan(both[0]).all() and torch.equal(both[1], one[0])


@pytest.mark.gpu
def test_rank_one_and_repeated_rows(device):
    from dpcr_agb_amd.muon_ops import orthogonalize
    u, v = matrix(100, 1, device=device, seed=1), matrix(1, 300, device=device, seed=2)
    close(orthogonalize(u @ v), u @ v)
    x = matrix(1, 80, device=device).expand(80, 80).contiguous()
    close(orthogonalize(x), x)
    close(orthogonalize(torch.eye(128, device=device)), torch.eye(128, device=device))


@pytest.mark.gpu
@pytest.mark.parametrize("steps,coef", [(1, C), (2, C), (8, C), (10, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375)),
                                        (3, [C, (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)])])
def test_other_steps_and_coefficients(device, steps, coef):
    from dpcr_agb_amd.muon_ops import orthogonalize
    x = matrix(150, 90, device=device)
    close(orthogonalize(x, steps=steps, coefficients=coef), x, steps=steps, coef=coef)


@pytest.mark.gpu
def test_converges_to_orthogonal(device):
    """With the convergent cubic the result is orthogonal: X^T X = 1."""
    from dpcr_agb_amd.muon_ops import orthogonalize
    q = orthogonalize(matrix(300, 40, device=device), steps=40, coefficients=(1.5, -0.5, 0.0)).double()
    # entries of X^T X: sums of 300 products of entries held to 2^-22 (and the fp32 result's 2^-24)
    assert float((q.T @ q - torch.eye(40, device=device).double()).abs().max()) < 8 * 2.0 ** -22


@pytest.mark.gpu
def test_repeats_on_streams_and_in_graphs(device):
    from dpcr_agb_amd.muon_ops import orthogonalize
    xs = [matrix(300, 520, device=device), matrix(64, 48, device=device), matrix(6000, 256, dtype=torch.bfloat16, device=device)]
    want = orthogonalize(xs)
    assert all(torch.equal(a, b) for a, b in zip(want, orthogonalize(xs)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = orthogonalize(xs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = orthogonalize(xs)
        graphs.append((g, out))
    for step in range(4):
        for i, x in enumerate(xs):
            x.copy_(matrix(*x.shape, device=device, seed=10 * step + i))
        want = orthogonalize(xs)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, out)), step


def update64(p, g, m, lr, mu, nesterov, wd, clip=None, **kw):
    p, g, m = p.double(), g.double(), m.double()
    if clip:
        g = g.clamp(-clip, clip)
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    o, bound = iterate(u.reshape(-1, u.shape[-1]), **kw)
    step = lr * 0.2 * math.sqrt(max(o.shape))
    return p * (1 - lr * wd) - step * o.reshape(p.shape), m, step * bound


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16, torch.float16])
def test_update(device, nesterov, gdtype):
    """Three steps of a list of weights; every step from the state the kernels left."""
    from dpcr_agb_amd.muon_ops import muon_update
    shapes = [(27, 64, 64), (64, 4), (4, 64), (343, 3, 64), (200, 300), (27, 64, 128), (2, 2)]
    ps = [matrix(*s, device=device, seed=i) for i, s in enumerate(shapes)]
    ms = [torch.zeros_like(p) for p in ps]
    for step in range(3):
        gs = [matrix(*s, dtype=gdtype, device=device, seed=100 * step + i) for i, s in enumerate(shapes)]
        clip = 0.02 if step == 2 else None
        want = [update64(p, g, m, 0.02, 0.9, nesterov, 0.1, clip) for p, g, m in zip(ps, gs, ms)]
        kept = [g.clone() for g in gs]
        muon_update(ps, gs, ms, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, clip_value=clip)
        for p, m, g, k, (rp, rm, bound) in zip(ps, ms, gs, kept, want):
            assert torch.equal(g, k)
            assert float((m.double() - rm).abs().max()) <= 4 * 2.0 ** -24 * float(rm.abs().max() + 1e-3)
            assert float((p.double() - rp).norm()) <= 2 * bound + 4 * 2.0 ** -24 * float(rp.norm())


# tall ones whose rows are read eight elements at a time, and those that just miss it: widths, ends, types, strides
WHOLE = [(200, 40), (100, 8), (129, 64), (250, 24), (97, 96), (128, 120), (128, 104), (64, 8), (256, 56), (8, 8), (200, 36), (130, 7),
         (128, 100), (40, 200), (104, 128), (9, 256), (512, 64), (300, 48), (321, 5), (60, 400), (257, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", WHOLE)
def test_matrices_taken_whole(device, shape, dtype):
    from dpcr_agb_amd.muon_ops import muon_update, orthogonalize
    x = matrix(3, *shape, dtype=dtype, device=device)
    for got, want in zip(orthogonalize(x), x):
        close(got, want)
    wide = torch.full((3, shape[0] + 1, shape[1] + 24), float("nan"), dtype=dtype, device=device)
    for first in (8, 1):           # aligned rows further apart, and rows off the grid
        v = wide[:, :shape[0], first:first + shape[1]]
        v.copy_(x)
        assert torch.equal(orthogonalize(v), orthogonalize(x))
    p, m = matrix(*shape, device=device, seed=1), matrix(*shape, device=device, seed=2)
    rp, rm, bound = update64(p, x[0], m, 0.02, 0.9, True, 0.1)
    muon_update([p], [x[0]], [m], lr=0.02, momentum=0.9, weight_decay=0.1)
    assert float((m.double() - rm).abs().max()) <= 4 * 2.0 ** -24 * float(rm.abs().max() + 1e-3)
    assert float((p.double() - rp).norm()) <= 2 * bound + 4 * 2.0 ** -24 * float(rp.norm())


@pytest.mark.gpu
def test_optimiser_splits_matrices_and_vectors(device):
    """optim.Muon: matrices by the update above, vectors and groups with muon=False exactly as AdaBelief alone."""
    from dpcr_agb_amd.optim import AdaBelief, Muon
    shapes = [(27, 64, 64), (64,), (1, 64), (64, 32), (33, 2), (7,)]
    a = [torch.nn.Parameter(matrix(*s, device=device, seed=i)) for i, s in enumerate(shapes)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    opt = Muon([{"params": a[:4]}, {"params": a[4:], "muon": False, "lr": 0.003}], lr=0.01, weight_decay=0.05, fused=True,
               clip_value=1.0)
    ref = AdaBelief([{"params": [b[1], b[2]]}, {"params": b[4:], "lr": 0.003}], lr=0.01, weight_decay=0.05, fused=True,
                    clip_value=1.0)
    mom = {i: torch.zeros_like(a[i]) for i in (0, 3)}
    for step in range(3):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = matrix(*shapes[i], device=device, seed=50 * step + i)
            q.grad = p.grad.clone()
        want = {i: update64(a[i].detach(), a[i].grad, mom[i], 0.01, 0.95, True, 0.05) for i in mom}
        opt.step()
        ref.step()
        for i in (1, 2, 4, 5):
            assert torch.equal(a[i], b[i]), i
        for i, (rp, rm, bound) in want.items():
            assert float((a[i].detach().double() - rp).norm()) <= 2 * bound + 4 * 2.0 ** -24 * float(rp.norm())
            mom[i] = opt.state[a[i]]["momentum_buffer"].clone()
    state = opt.state_dict()
    again = Muon([{"params": a[:4]}, {"params": a[4:], "muon": False, "lr": 0.003}], lr=0.01, fused=True)
    again.load_state_dict(state)
    assert torch.equal(again.state[a[0]]["momentum_buffer"], mom[0]) and again.param_groups[0]["weight_decay"] == 0.05


@pytest.mark.gpu
def test_update_captured(device):
    """An update captured into a graph and replayed equals eager steps."""
    from dpcr_agb_amd.muon_ops import muon_update
    shapes = [(27, 64, 64), (64, 4), (300, 100)]
    ps = [matrix(*s, device=device, seed=i) for i, s in enumerate(shapes)]
    ms, gs = [torch.zeros_like(p) for p in ps], [matrix(*s, device=device, seed=9 + i) for i, s in enumerate(shapes)]
    eager = [[p.clone() for p in ps], [m.clone() for m in ms]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_update(ps, gs, ms, lr=0.02)
    for step in range(3):
        for i, g in enumerate(gs):
            g.copy_(matrix(*g.shape, device=device, seed=30 * step + i))
        muon_update(eager[0], gs, eager[1], lr=0.02)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps + ms, eager[0] + eager[1])), step


def test_refusals():
    from dpcr_agb_amd import _lib
    from dpcr_agb_amd.muon_ops import muon_update, orthogonalize
    x = torch.zeros(4, 8)
    with pytest.raises(_lib.AgbError):
        orthogonalize(x)                                                         # host tensors
    with pytest.raises(_lib.AgbError):
        orthogonalize(x.double())
    with pytest.raises(ValueError):
        orthogonalize(torch.zeros(8))
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(x, steps=0)
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(x, steps=65)
    with pytest.raises(ValueError, match="coefficients"):
        orthogonalize(x, coefficients=(1.0, 2.0))
    with pytest.raises(ValueError, match="coefficients"):
        orthogonalize(x, coefficients=[C, C])
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(x, eps=float("nan"))
    with pytest.raises(ValueError, match="differentiable"):
        orthogonalize(torch.zeros(4, 8, requires_grad=True))
    with pytest.raises(ValueError, match="shorter"):
        orthogonalize(torch.zeros(1, 1).expand(20000, 20000))
    ok = [torch.zeros(4, 8)]
    for args, err in (((ok, ok, []), ValueError), (([torch.zeros(8)],) * 3, ValueError), (([torch.zeros(1, 8)],) * 3, ValueError),
                      ((ok, [torch.zeros(8, 4)], ok), ValueError), (([x.double()], [x.double()], [x.double()]), _lib.AgbError),
                      (([x], [x], [x]), _lib.AgbError), (([torch.zeros(8, 4).t()], [x], [x]), _lib.AgbError)):
        with pytest.raises(err):
            muon_update(*args, lr=0.1)
    for kw in ({"momentum": 1.0}, {"clip_value": 0.0}, {"eps": -1.0}, {"steps": 0}):
        with pytest.raises(ValueError):
            muon_update(ok, ok, ok, lr=0.1, **kw)
    from dpcr_agb_amd.optim import Muon
    p = torch.nn.Parameter(x)
    for kw in ({"momentum": 1.5}, {"ns_steps": 0}, {"adjust": "fan"}, {"lr": -1.0}):
        with pytest.raises(ValueError):
            Muon([p], **kw)


@pytest.mark.gpu
def test_refuses_what_is_listed_twice(device):
    from dpcr_agb_amd.muon_ops import muon_update
    p, m = matrix(8, 8, device=device), torch.zeros(8, 8, device=device)
    with pytest.raises(ValueError, match="twice"):
        muon_update([p, p], [p.clone()] * 2, [m, m.clone()], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_update([p, p.clone()], [p.clone()] * 2, [m, m], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_update([p], [p.clone()], [p], lr=0.1)
    with pytest.raises(ValueError, match="gradient"):
        muon_update([p], [m], [m], lr=0.1)
    with pytest.raises(ValueError, match="gradient"):
        muon_update([p, p.clone()], [m.clone(), p], [m, m.clone()], lr=0.1)


def test_optimiser_refuses_what_no_step_could_take():
    from dpcr_agb_amd.optim import Muon
    wide = torch.nn.Parameter(torch.empty(16385, 16385, device="meta"))
    with pytest.raises(ValueError, match="muon=False"):
        Muon([wide])
    opt = Muon([{"params": [wide], "muon": False}])
    with pytest.raises(ValueError, match="muon=False"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.empty(2, 1 << 25, device="meta"))]})
    with pytest.raises(ValueError, match="momentum"):
        Muon([torch.nn.Parameter(torch.zeros(2, 2))], momentum=1.0)
    with pytest.raises(ValueError, match="steps"):
        Muon([torch.nn.Parameter(torch.zeros(2, 2))], ns_steps=0)
    with pytest.raises(ValueError, match="adjust"):
        Muon([torch.nn.Parameter(torch.zeros(2, 2))], adjust="spectral")


def test_entry_points_validate_before_any_launch():
    import ctypes
    from dpcr_agb_amd import _lib, muon_ops
    L = _lib.load()
    assert L.agb_ns_fields() == muon_ops._FIELDS

    def fields(rows=8, cols=8, batch=1, ld=8, typ=0, inp=256, mom=0):
        return (ctypes.c_longlong * 11)(inp, 512, mom, rows, cols, batch, ld, 64, ld, 64, typ)

    size = _lib.size_call("agb_ns_workspace_bytes", fields(), 1)
    assert size > 0 and _lib.size_call("agb_ns_workspace_bytes", fields(rows=0), 1) == 0
    assert _lib.size_call("agb_ns_workspace_bytes", fields(rows=17000, cols=17000), 1) == 0
    good, steps = (ctypes.c_float * 15)(*C * 5), 5

    def run(f=None, count=1, steps=5, coef=good, eps=1e-7, ws=ctypes.c_void_p(256), nbytes=size):
        return L.agb_orthogonalize(f or fields(), count, steps, coef, ctypes.c_double(eps), ws, ctypes.c_size_t(nbytes), None)

    for kw, word in (({"steps": 0}, b"steps"), ({"steps": 65}, b"steps"), ({"coef": None}, b"steps"), ({"eps": -1.0}, b"eps"),
                     ({"coef": (ctypes.c_float * 15)(*(9.0, 0.0, 0.0) * 5)}, b"coefficients"),
                     ({"coef": (ctypes.c_float * 15)(*(float("nan"), 0.0, 0.0) * 5)}, b"coefficients"),
                     ({"f": fields(rows=0)}, b"not taken"), ({"f": fields(batch=0)}, b"not taken"),
                     ({"f": fields(ld=7)}, b"row stride"), ({"f": fields(typ=3)}, b"type"), ({"f": fields(inp=0)}, b"null"),
                     ({"ws": None}, b"workspace"), ({"nbytes": size - 1}, b"workspace")):
        assert run(**kw) == -1 and word in L.agb_last_error(), (kw, L.agb_last_error())
    assert run(count=0) == 0
    d = ctypes.c_double
    step = (ctypes.c_float * 1)(0.1)
    assert L.agb_muon_update(fields(), 1, 5, good, d(1e-7), None, d(1), d(0.9), 1, 0.0, None, 0, None) == -1
    assert L.agb_muon_update(fields(), 1, 5, good, d(1e-7), step, d(1), d(1.0), 1, 0.0, None, 0, None) == -1
    assert b"momentum" in L.agb_last_error()
    assert L.agb_muon_update(fields(), 1, 5, good, d(1e-7), step, d(1), d(0.9), 1, 0.0, None, 0, None) == -1
    assert b"null pointer" in L.agb_last_error()
    assert L.agb_muon_update(fields(batch=2, mom=768), 1, 5, good, d(1e-7), step, d(1), d(0.9), 1, 0.0, None, 0, None) == -1
    assert b"one matrix" in L.agb_last_error()
