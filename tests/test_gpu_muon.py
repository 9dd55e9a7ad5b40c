"""GPU parity of the orthogonalised updates against the definition in float64, and of their refusals.

Tolerances (set before the first run). Up to 64 on the shorter side the steps run in float64 on the Gram matrix: singular values'
squares are off by about 2^-52 of the largest, which the product of the steps' polynomials (at most 485, no steeper than 1e6) turns
into 1e-9 of |X| = 1; the result is rounded to float32, then to its type. A momentum's update u is formed in float32, three roundings
of 2^-24, and an error in u grows by 485 at most: 485 * 3 * 2^-24 of |X| = 1.

Above, float16 operands round X, A and B by 2^-11, and how much that moves the result depends on the spectrum. So the oracle takes the same
steps in float64 with those roundings, each where the kernels make it (`rounded`), and its distance from the definition is what the
kernels are allowed, half as much again in norm for the luck of the roundings, three times at a single place; their
float32 sums add a thirtieth of that. That distance itself has to stay below 5e-3 of the norm for the spectra here."""
import math

import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu
fm = sub("enhancers.fused_muon")
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ABC = fm.COEFFICIENTS


def definition(u, steps=5, abc=ABC, eps=1e-7):
    a, b, c = abc
    x = u.double() / u.double().norm().clamp(min=eps)
    flip = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if flip else x
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T.contiguous() if flip else x


def rounded(u, steps=5, abc=ABC, eps=1e-7):
    """The definition with the roundings of the float16 path."""
    a, b, c = abc
    h = lambda t: t.half().double()                                                             # noqa: E731
    u = u.double()
    flip = u.shape[0] > u.shape[1]
    u = u.T.contiguous() if flip else u
    s = 2.0 ** (math.floor(0.5 * math.log2(u.shape[0])) - 1)
    f = u * (s / u.norm().clamp(min=eps))
    eye = torch.eye(u.shape[0], dtype=torch.float64, device=u.device)
    x = h(f)
    lo = h((f - x) * 2048) / 2048
    for k in range(steps):
        g = h(x @ x.T)
        carry = k < steps - 2
        q = h(c / s ** 2 * (g @ g) + b * g + (0 if carry else a * s ** 2) * eye)
        f = q @ x / s ** 2 + (a * (x + lo) if carry else 0)
        if k + 1 == steps:
            x = f / s
            break
        x = h(f)
        lo = h((f - x) * 2048) / 2048
    return x.T.contiguous() if flip else x


def matrix(rows, cols, kind, g):
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                                # noqa: E731
    x = rnd(rows, cols)
    if kind == "falling":                                       # strong directions whose sizes fall off, in noise
        r = max(1, min(32, rows // 2, cols // 2))
        x = 0.1 * x + (rnd(rows, r) / torch.arange(1, r + 1, device="cuda")) @ rnd(r, cols)
    return x * 1e-3


def hold(got, u, what):
    """`got` against the orthogonalised `u`, by the rules above."""
    want, unit = definition(u), UNIT[got.dtype]
    err = (got.double() - want).abs()
    if min(u.shape) <= 64:
        # (float16 below 2^-14 is in steps of 2^-24, so a rounding is off by up to 2^-25 there, more than 2^-11 of the value)
        tol = (unit + 2.0 ** -23) * want.abs() + 1e-8 + (2.0 ** -25 if got.dtype == torch.float16 else 0)
        over = float((err - tol).max())
        assert over <= 0, (what, over)
        return
    sim = (rounded(u) - want).abs()
    assert float(sim.norm()) < 5e-3 * float(want.norm()), what
    rel = float(err.norm() / want.norm())
    assert rel <= 1.5 * float(sim.norm() / want.norm()) + unit, (what, rel, float(sim.norm() / want.norm()))
    over = float((err - 3 * sim.max() - unit * want.abs()).max())
    assert over <= 0, (what, over, float(err.max()), float(sim.max()))


# both sides of the border at 64, one value, odd sizes, wide and tall, every tiling of both products and slices of the sum
SHAPES = [(1, 1, 1, 1), (2, 1, 300, 1), (3, 300, 1, 1), (1, 7, 5, 1), (5, 16, 16, 1), (4, 17, 1000, 0), (3, 1000, 31, 0),
          (2, 33, 4097, 0), (2, 5000, 64, 0), (70, 32, 512, 0), (66, 64, 40, 0), (1, 64, 64, 1), (1, 65, 65, 0), (2, 65, 1531, 0),
          (3, 1531, 67, 0), (2, 128, 128, 0), (1, 129, 257, 0), (3, 255, 200, 0), (2, 1021, 333, 0), (1, 640, 2048, 0),
          (1, 2048, 640, 0), (70, 96, 104, 0), (2, 1000, 1000, 0), (1, 1536, 1536, 0), (1, 2051, 1029, 0), (5, 1100, 2200, 0),
          (1, 4096, 1300, 0)]


@pytest.mark.parametrize("i", range(len(SHAPES)), ids=["x".join(map(str, s[:3])) for s in SHAPES])
def test_orthogonalize(native, i):
    count, rows, cols, _ = SHAPES[i]
    dtype = (torch.bfloat16, torch.float16, torch.float32)[i % 3]
    g = torch.Generator(device="cuda").manual_seed(100 + i)
    print(f"case orthogonalize {count} x {rows} x {cols} {dtype}", flush=True)
    x = torch.stack([matrix(rows, cols, ("falling", "flat")[k % 2], g) for k in range(count)]).to(dtype)
    got = fm.orthogonalize(x)
    assert got.shape == x.shape and got.dtype == dtype
    for k in range(0, count, max(1, count // 3)):
        hold(got[k], x[k], (i, k))
    assert torch.equal(got, fm.orthogonalize(x))
    assert torch.equal(fm.orthogonalize(x[count - 1]), got[count - 1]) or min(rows, cols) > 64      # (another batch may be sliced otherwise)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("nesterov,adjust", [(True, "spectral"), (False, "rms")])
def test_steps(native, dtype, nesterov, adjust):
    """Two steps of matrices of several shapes, some of one shape, one without values."""
    dt, g = getattr(torch, dtype), torch.Generator(device="cuda").manual_seed(4)
    shapes = [(48, 200), (200, 48), (48, 200), (300, 130), (130, 300), (300, 130), (1, 9), (0, 5), (129, 129)]
    p = [(0.02 * torch.randn(s, generator=g, device="cuda")).to(dt) for s in shapes]
    m = fm.muon_momenta(p)
    mu, lr, decay = 0.9, 0.05, 0.2
    for step in range(2):
        grads = [matrix(*s, "falling", g).to(dt) if min(s) else torch.zeros(s, dtype=dt, device="cuda") for s in shapes]
        before = [(a.double(), b.double()) for a, b in zip(p, m)]
        fm.muon_step(p, grads, m, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, adjust=adjust)
        for i, s in enumerate(shapes):
            if not min(s):
                continue
            q, old = before[i]
            d = grads[i].double()
            want_m = mu * old + (1 - mu) * d
            assert bool(((m[i].double() - want_m).abs() <= 2.0 ** -22 * (mu * old.abs() + d.abs())).all()), (step, i)
            u = mu * want_m + (1 - mu) * d if nesterov else want_m
            o = definition(u)
            rate = lr * (math.sqrt(max(1, s[0] / s[1])) if adjust == "spectral" else 0.2 * math.sqrt(max(s)))
            want = (1 - lr * decay) * q - rate * o
            off = 485 * 3 * 2.0 ** -24 + (3 * float((rounded(u) - o).abs().max()) if min(s) > 64 else 0)
            tol = UNIT[dt] * want.abs() + rate * off + 2.0 ** -22 * (q.abs() + rate * o.abs()) + (2.0 ** -25 if dt == torch.float16 else 0)
            err = (p[i].double() - want).abs()
            assert bool((err <= tol).all()), (step, i, float((err - tol).max()))


def test_zeros_ranks_sizes_and_nan(native):
    for rows, cols in ((40, 90), (90, 40), (200, 90), (90, 200)):
        x = torch.zeros(4, rows, cols, device="cuda")
        x[1, 3, 5] = -2.5                                       # one value: rank one
        x[2] = torch.randn(rows, 1, device="cuda") @ torch.randn(1, cols, device="cuda")
        x[3, 0, 0] = float("nan")
        got = fm.orthogonalize(x)
        top = definition(torch.ones(1, 1, device="cuda"))[0, 0]          # what a singular value of one becomes
        assert (got[0] == 0).all() and got[3].isnan().any() and got[:3].isfinite().all()
        one = torch.zeros(rows, cols, dtype=torch.float64, device="cuda")
        one[3, 5] = -top
        assert float((got[1] - one).abs().max()) < 2e-3
        sv = torch.linalg.svdvals(got[2].double())
        assert abs(float(sv[0] - top)) < 4e-3
        # a tenth of 2^-11, at 90 places, times 485: what rounding noise may make of directions that are not there
        assert float(sv[1]) < 0.05
    # sizes far from one
    g = torch.Generator(device="cuda").manual_seed(1)
    for size in (1e-30, 1e25):
        for rows, cols in ((50, 70), (100, 70)):
            x = torch.randn(rows, cols, generator=g, device="cuda")
            got = fm.orthogonalize(x * size, eps=1e-37)
            assert float((got.double() - definition(x)).norm()) < 5e-3 * float(definition(x).norm())
    x = torch.full((70, 70), 1e-12, device="cuda")
    assert float(fm.orthogonalize(x).abs().max()) < 0.1         # far below eps: divided by eps


def test_other_polynomials(native):
    g = torch.Generator(device="cuda").manual_seed(2)
    for rows, cols in ((30, 80), (150, 200)):
        x = torch.randn(rows, cols, generator=g, device="cuda")
        for steps, abc in ((1, ABC), (2, ABC), (3, ABC), (8, (1.5, -0.5, 0.0)), (12, (2.0, -1.5, 0.5)), (32, (1.5, -0.5, 0.0))):
            got, want = fm.orthogonalize(x, steps, abc).double(), definition(x, steps, abc)
            assert float((got - want).norm()) < 5e-3 * float(want.norm()), (rows, steps, abc)
    # enough cubic steps give the nearest orthogonal matrix
    u, _, v = torch.linalg.svd(x.double(), full_matrices=False)
    assert float((got - u @ v).norm()) < 2e-3 * float((u @ v).norm())


def test_strides_streams_and_two_at_once(native):
    g = torch.Generator(device="cuda").manual_seed(3)
    for rows, cols in ((40, 300), (140, 200)):
        x = torch.randn(3, rows, cols, generator=g, device="cuda").bfloat16()
        want = fm.orthogonalize(x)
        assert torch.equal(fm.orthogonalize(x.transpose(0, 1).contiguous().transpose(0, 1)), want)
        assert torch.equal(fm.orthogonalize(x.view(3, 1, rows, cols)).view_as(x), want)
        odd = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view_as(x).copy_(x)
        assert torch.equal(fm.orthogonalize(odd), want)
        sides = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for _ in range(3):
            for s in sides:
                with torch.cuda.stream(s):
                    got.append(fm.orthogonalize(x))
        torch.cuda.synchronize()
        assert all(torch.equal(v, want) for v in got)
    assert fm.orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert fm.orthogonalize(torch.empty(2, 0, 5, device="cuda")).shape == (2, 0, 5)
    leaf = torch.randn(8, 8, device="cuda", requires_grad=True)
    assert not fm.orthogonalize(leaf).requires_grad


def test_captured_and_replayed(native):
    g = torch.Generator(device="cuda").manual_seed(6)
    for rows, cols in ((40, 300), (200, 1000)):
        x = torch.randn(2, rows, cols, generator=g, device="cuda").bfloat16()
        fm.orthogonalize(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fm.orthogonalize(x)
        for k in range(4):
            x.copy_(torch.randn(2, rows, cols, generator=g, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, fm.orthogonalize(x)), k
        p = [x[0].clone()]
        m = fm.muon_momenta(p)
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fm.muon_step(p, [x[0]], m)
        torch.cuda.synchronize()


def test_optimizer_and_its_state(native):
    g = torch.Generator(device="cuda").manual_seed(8)
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(k)).cuda().bfloat16())   # noqa: E731
                    for k, s in enumerate(((80, 100), (20, 30), (80, 100)))]
    a, b = make(), make()
    one, two = fm.Muon(a, lr=0.1), fm.Muon(b, lr=0.1)
    grads = [[torch.randn(p.shape, generator=g, device="cuda").bfloat16() for p in a] for _ in range(4)]

    def run(params, optimizer, steps):
        for k in steps:
            for i, p in enumerate(params):
                p.grad = None if (k, i) == (1, 2) else grads[k][i].clone()
            kept = params[2].detach().clone()
            optimizer.step()
            assert torch.equal(params[2], kept) == ((k, 2) == (1, 2))
    run(a, one, range(4))
    run(b, two, range(2))
    saved = two.state_dict()
    c = [torch.nn.Parameter(p.detach().clone()) for p in b]
    three = fm.Muon(c, lr=0.1)
    three.load_state_dict(saved)
    assert three.state[c[0]]["momentum"].dtype == torch.float32
    run(c, three, range(2, 4))
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    version = c[0]._version
    run(c, three, range(2, 3))
    assert c[0]._version > version


def test_refused_steps_change_nothing(native):
    p = [torch.randn(70, 80, device="cuda"), torch.randn(8, 9, device="cuda")]
    m, g = fm.muon_momenta(p), [torch.randn_like(t) for t in p]
    kept = [t.clone() for t in p + m]
    vector = torch.randn(5, device="cuda")
    bad = [((p, g[:1], m), {}), ((p, g, [m[0], m[1].double()]), {}), ((p, [g[0], g[1].t().contiguous().t()], m), {}),
           ((p, [g[0], g[1].bfloat16()], m), {}), ((p + [vector], g + [vector], m + [vector]), {}), ((p, g, m), {"momentum": 1.0}),
           ((p, g, m), {"lr": float("nan")}), ((p, g, m), {"steps": 0}), ((p, g, m), {"steps": 33}), ((p, g, m), {"adjust": "none"}),
           ((p, g, m), {"coefficients": (4.0, 0.0, 0.0)}), ((p, g, m), {"eps": 0.0}), ((p + p[:1], g + g[:1], m + m[:1]), {}),
           ((p, g, [m[0], m[1].cpu()]), {}), ((p, [g[0], g[1].view(9, 8)], m), {})]
    for args, options in bad:
        with pytest.raises(ValueError):
            fm.muon_step(*args, **options)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, p + m))
    assert fm.orthogonalize(p[0].cpu()) is None and fm.orthogonalize(p[0].double()) is None
    with pytest.raises(ValueError):
        fm.orthogonalize(vector)
    with pytest.raises(ValueError):
        fm.orthogonalize(p[0], coefficients=(3.0, 1.0, 1.0))
    with pytest.raises(ValueError):
        fm.Muon([torch.nn.Parameter(vector)])
    fm.muon_step([], [], [])


def test_zeros_below_any_eps(native):
    # 1 / eps^2 is infinite from 1e-155 down, and 0 times that no number
    for rows, cols in ((40, 90), (90, 40), (200, 90), (1, 1)):
        zeros = torch.zeros(rows, cols, device="cuda")
        for eps in (1e-100, 1e-200, 5e-324):
            assert torch.equal(fm.orthogonalize(zeros, eps=eps), zeros)
        p, m = torch.ones_like(zeros), torch.zeros_like(zeros)
        fm.muon_step([p], [zeros], [m], lr=0.5, weight_decay=0.5, eps=1e-200)
        assert torch.equal(p, torch.full_like(p, 0.75)) and torch.equal(m, zeros)


def test_a_gradient_in_a_momentums_memory(native):
    p = [torch.randn(70, 80, device="cuda"), torch.randn(8, 9, device="cuda"), torch.randn(0, 9, device="cuda")]
    g = [torch.randn_like(t) for t in p]
    m = fm.muon_momenta(p)
    kept = [t.clone() for t in p]
    for momenta in ([m[0], g[1], m[2]], [g[0], m[1], g[2]]):
        with pytest.raises(ValueError):
            fm.muon_step(p, g, momenta)
    assert all(torch.equal(a, b) for a, b in zip(kept, p))
    fm.muon_step(p, [g[0], g[1], p[2]], m)                          # (nothing shares no memory, and one gradient may serve two)
    q = [torch.randn(70, 80, device="cuda") for _ in range(2)]
    fm.muon_step(q, [g[0], g[0]], fm.muon_momenta(q))


def test_the_largest_shorter_side(native):
    # 16384 x 16384: the powers of two that keep X and its products in float16's range are at their largest
    g = torch.Generator(device="cuda").manual_seed(9)
    x = matrix(16384, 16384, "falling", g).bfloat16()
    x[:, 0] *= 40                                               # one column, and so one entry of X^T X, far above the others
    got = fm.orthogonalize(x)
    assert got.isfinite().all()
    sv = torch.linalg.svdvals(got[:, :64].double())
    # 64 of the columns of a matrix whose singular values all lie below 1.21 (the polynomial's largest, plus 1 % for the roundings)
    assert float(sv[0]) < 1.22
    a, b, c = ABC
    want = x.float() / x.float().norm()
    for _ in range(5):                                          # float32 products: 2^-24 against 2^-11
        s = want @ want.T
        want = a * want + (b * s + c * (s @ s)) @ want
    assert float((got.float() - want).norm() / want.norm()) < 5e-3
